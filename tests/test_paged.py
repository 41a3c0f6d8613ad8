"""The paged KV cache: vc4_paged_append and vc4_paged_attention against their
definitions in 64 bits, and what they refuse."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import vc4b200
from paged_ref import GRID, POOL, TORCH, Cache, attention, attention_bound, decode, half_step, swap16

EINVAL = 1


# ---- refusals, before any GPU is asked for -------------------------------------------

class _NoGpu:
    _h = None


def _host_batch(**over):
    a = dict(cu=64, length=64, table=64, seqs=2, tokens=4, max_new=2, max_len=32, table_stride=2)
    a.update(over)
    return vc4b200.PagedBatch(**a)


def _host_pages(fmt="q8", **over):
    a = dict(data=256, pages=4, page_len=16, kv_heads=2, head_dim=64)
    a.update(over)
    return vc4b200.PagedKV(_NoGpu(), a["data"], fmt, a["pages"], a["page_len"], a["kv_heads"], a["head_dim"])


def _refused(call, words):
    with pytest.raises(vc4b200.EngineError) as e:
        call()
    assert "error %d" % EINVAL in str(e.value) and words in str(e.value), str(e.value)


@pytest.mark.parametrize("over,words", [
    (dict(page_len=24), "page_len"), (dict(page_len=512), "page_len"), (dict(head_dim=72), "head_dim"),
    (dict(head_dim=144), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(pages=0), "positive"),
    (dict(kv_heads=0), "positive"), (dict(data=0), "address"), (dict(data=264), "address"),
    (dict(pages=2 ** 25, page_len=32), "2^31 - 1 rows"), (dict(pages=2 ** 31 - 1), "2^31 - 1 rows")])
def test_pages_are_refused(over, words):
    _refused(lambda: _host_pages(**over).append(_host_batch(), 64, "f32", 4, 64, "bf16"), words)
    _refused(lambda: _host_pages(**over).attend(_host_batch(), 64, "bf16", 4, 64, "bf16"), words)


@pytest.mark.parametrize("over,words", [
    (dict(seqs=0), "seqs"), (dict(tokens=-1), "not negative"), (dict(max_new=-1), "not negative"),
    (dict(table_stride=0), "table_stride"), (dict(max_len=33), "page table"), (dict(cu=0), "required"),
    (dict(length=0), "required"), (dict(table=0), "required"), (dict(table_stride=2 ** 26 + 1), "2^30 positions")])
def test_batches_are_refused(over, words):
    _refused(lambda: _host_pages().append(_host_batch(**over), 64, "f32", 4, 64, "bf16"), words)
    _refused(lambda: _host_pages().attend(_host_batch(**over), 64, "bf16", 4, 64, "bf16"), words)
    _refused(lambda: _host_pages().attend_bytes(_host_batch(**over), 4), words)


@pytest.mark.parametrize("fmt,args,more,words", [
    ("q8", (64, "f32", 3, 64, "bf16"), {}, "multiple of kv_heads"),
    ("q8", (64, "q16", 4, 64, "bf16"), {}, "VC4_F32"), ("q8", (64, "f32", 4, 64, "q16"), {}, "VC4_F32"),
    ("q8", (72, "f32", 4, 64, "bf16"), {}, "qkv's address"), ("q8", (64, "f32", 4, 0, "bf16"), {}, "q's address"),
    ("q8", (64, "f32", 4, 64, "bf16"), dict(qkv_stride=504), "stride"),
    ("q8", (64, "f32", 4, 64, "bf16"), dict(q_stride=260), "stride"),
    ("q8", (64, "f32", 4, 64, "bf16"), dict(q_norm=64), "go together"),
    ("q8", (64, "f32", 4, 64, "bf16"), dict(q_norm=64, k_norm=68), "norm weights"),
    ("q8", (64, "f32", 4, 64, "bf16"), dict(q_norm=64, k_norm=64, eps=-1.0), "eps"),
    ("q8", (64, "f32", 4, 64, "bf16"), dict(cos=64), "go together"),
    ("q8", (64, "f32", 4, 64, "bf16"), dict(cos=64, sin=64), "rotation tables"),
    ("q8", (64, "f32", 4, 64, "bf16"), {}, "gpu is null")])
def test_append_refuses(fmt, args, more, words):
    _refused(lambda: _host_pages(fmt).append(_host_batch(), *args, **more), words)


@pytest.mark.parametrize("fmt,args,more,words", [
    ("q8", (64, "f32", 4, 64, "bf16"), {}, "q is VC4_BF16 or VC4_F16"),
    ("bf16", (64, "f16", 4, 64, "bf16"), {}, "pages' type"), ("f16", (64, "bf16", 4, 64, "bf16"), {}, "pages' type"),
    ("q8", (64, "bf16", 4, 64, "q16"), {}, "out is"), ("q8", (64, "bf16", 5, 64, "bf16"), {}, "multiple of kv_heads"),
    ("q8", (66, "bf16", 4, 64, "bf16"), {}, "q's address"), ("q8", (64, "bf16", 4, 72, "bf16"), {}, "out's address"),
    ("q8", (64, "bf16", 4, 64, "bf16"), dict(out_stride=8), "stride"),
    ("q8", (64, "bf16", 4, 64, "bf16"), dict(scale=-0.5), "scale"),
    ("q8", (64, "bf16", 4, 64, "bf16"), dict(scale=math.nan), "scale"),
    ("q8", (64, "bf16", 4, 64, "bf16"), dict(scale=1e-38), "float's range"),
    ("bf16", (64, "bf16", 4, 64, "bf16"), dict(scale=3e38), "float's range"),
    ("q8", (64, "bf16", 4, 64, "bf16"), {}, "gpu is null")])
def test_attend_refuses(fmt, args, more, words):
    _refused(lambda: _host_pages(fmt).attend(_host_batch(), *args, **more), words)


def test_unknown_names_are_refused():
    for call in (lambda: _host_pages("q4"), lambda: _host_pages().append(_host_batch(), 64, "f64", 4, 64, "bf16")):
        with pytest.raises(vc4b200.EngineError, match="unknown"):
            call()


# ---- append -------------------------------------------------------------------------

def _append_case(cache, heads, kind, out_kind, norm, half, rope=True, pad=0, seed=1):
    g = torch.Generator().manual_seed(seed)
    kv, dim = cache.kv, cache.dim
    width = (heads + 2 * kv) * dim
    qkv = torch.randn(cache.rows, width + pad, generator=g).to(TORCH[kind]).cuda()
    q = torch.full((cache.rows, heads * dim + pad), 7.0, dtype=TORCH[out_kind], device="cuda")
    n = max(cache.length + [1]) + 2
    cos, sin = vc4b200.rope_tables(1e4, dim, n)
    t = {"qkv": qkv, "q": q, "cos": torch.from_numpy(cos).cuda(), "sin": torch.from_numpy(sin).cuda(),
         "qn": (1 + 0.3 * torch.randn(dim, generator=g)).cuda(), "kn": (1 + 0.3 * torch.randn(dim, generator=g)).cuda()}
    kw = dict(rope_half=half, qkv_stride=width + pad, q_stride=heads * dim + pad)
    if norm:
        kw.update(q_norm=t["qn"].data_ptr(), k_norm=t["kn"].data_ptr(), eps=1e-6)
    if rope:
        kw.update(cos=t["cos"].data_ptr(), sin=t["sin"].data_ptr(), rope_len=n)
    return t, kw


def _append_ref(cache, t, heads, norm, half, rope):
    """(q, k, v, bound) of every token in doubles; bound: what the float steps may be off."""
    kv, dim = cache.kv, cache.dim
    x = t["qkv"][: cache.tokens, : (heads + 2 * kv) * dim].double().view(-1, heads + 2 * kv, dim)
    y = x.clone()
    if norm:
        r = 1 / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        w = torch.cat([t["qn"].expand(heads, dim), t["kn"].expand(kv, dim)]).double()
        y[:, : heads + kv] = w * (r * x)[:, : heads + kv]
    size = y.abs()
    if rope:
        pos = torch.cat([torch.arange(n - m, n) for n, m in zip(cache.length, cache.new)]).cuda()
        c, s = t["cos"].double()[pos][:, None], t["sin"].double()[pos][:, None]
        z = y[:, : heads + kv]
        a, b = (z[..., : dim // 2], z[..., dim // 2:]) if half else (z[..., 0::2], z[..., 1::2])
        u, v, m = a * c - b * s, a * s + b * c, a.abs() + b.abs()
        if half:
            z, m = torch.cat([u, v], -1), torch.cat([m, m], -1)
        else:
            z, m = torch.stack([u, v], -1).flatten(-2), torch.stack([m, m], -1).flatten(-2)
        y[:, : heads + kv], size[:, : heads + kv] = z, m
    # at most: square sum, quotient, + eps, root, reciprocal, two products, rotation product and sum
    return y[:, :heads], y[:, heads: heads + kv], y[:, heads + kv:], 9 * 2.0 ** -24 * size


SHAPES = [  # heads, kv, dim, page
    (8, 4, 96, 16), (16, 2, 64, 32), (4, 2, 16, 16), (7, 1, 128, 64), (3, 3, 80, 128), (2, 1, 48, 256), (4, 4, 112, 16),
    (6, 2, 32, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["q8", "q16", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,page", SHAPES)
@pytest.mark.parametrize("kind,out_kind,norm,half,rope", [
    ("f32", "bf16", True, True, True), ("bf16", "f32", False, False, True), ("f16", "f16", True, False, True),
    ("f32", "f32", False, True, False)])
def test_append(fmt, heads, kv, dim, page, kind, out_kind, norm, half, rope):
    length, new = [1, 0, page + 3, 5, page, 40], [1, 0, 7, 5, 1, 0]
    cache = Cache(length, new, fmt, page, kv, dim, rows=20)
    t, kw = _append_case(cache, heads, kind, out_kind, norm, half, rope, pad=8)
    before, gpu = cache.pool.clone(), vc4b200.GPU(0)
    handle, batch = cache.handles(vc4b200, gpu)
    torch.cuda.synchronize()
    handle.append(batch, t["qkv"].data_ptr(), kind, heads, t["q"].data_ptr(), out_kind, **kw)
    gpu.sync()
    assert int(cache.status) == 0
    q, k, v, off = _append_ref(cache, t, heads, norm, half, rope)
    n = cache.tokens
    got = t["q"][:n, : heads * dim].double().view(n, heads, dim)
    tiny = 2.0 ** -25 if out_kind == "f16" else 0.0   # below f16's normal range a half step is 2^-25
    assert bool(((got - q).abs() <= off[:, :heads] * 1.01 + half_step(out_kind) * q.abs() * 1.001 + tiny).all())
    assert bool((t["q"][n:] == 7).all()) and bool((t["q"][:, heads * dim:] == 7).all())   # rows and columns behind
    now, was = decode(cache.pool, fmt), decode(before, fmt)
    written = torch.zeros(cache.pages, page, dtype=torch.bool, device="cuda")
    for s in range(len(length)):
        for j in range(new[s]):
            row, pos = int(cache.host_cu[s]) + j, length[s] - new[s] + j
            pg = int(cache.host_table[s, pos // page])
            written[pg, pos % page] = True
            for sel, want, o in ((0, k[row], off[row, heads: heads + kv]), (1, v[row], 0 * off[row, heads + kv:])):
                have = now[pg, sel, :, pos % page]
                if fmt in GRID:
                    low, high = (-8, 127 / 16) if fmt == "q8" else (-16, 32767 / 2048)
                    bound = 0.5 / GRID[fmt] + o * 1.01 + 2.0 ** -23 * want.abs()   # + the scaled value's 1/2 added
                    assert bool(((have - want.clamp(low, high)).abs() <= bound).all())
                else:
                    tiny = 2.0 ** -25 if fmt == "f16" else 0.0
                    assert bool(((have - want).abs() <= o * 1.01 + half_step(fmt) * want.abs() * 1.001 + tiny).all())
    keep = ~written[:, None, None, :, None].expand_as(now)
    assert torch.equal(now[keep], was[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["q8", "q16"])
@pytest.mark.parametrize("kind,half", [("f32", True), ("bf16", False), ("f16", True)])
def test_append_levels_are_the_slot_caches_arithmetic(fmt, kind, half):
    """Every level and q value of many tokens: the float operations one by one
    (squares in double), as the slot cache's kernels round them."""
    heads, kv, dim, n = 16, 8, 96, 4000
    cache = Cache([n], [n], fmt, 32, kv, dim)
    t, kw = _append_case(cache, heads, kind, "f32", True, half)
    gpu = vc4b200.GPU(0)
    handle, batch = cache.handles(vc4b200, gpu)
    torch.cuda.synchronize()
    handle.append(batch, t["qkv"].data_ptr(), kind, heads, t["q"].data_ptr(), "f32", **kw)
    gpu.sync()
    x = t["qkv"].float().view(n, heads + 2 * kv, dim)
    y = x[:, : heads + kv]
    mean = y.double().square().sum(-1, keepdim=True).float() / torch.full((), float(dim), device="cuda")
    y = torch.cat([t["qn"].expand(heads, dim), t["kn"].expand(kv, dim)]) * ((1 / (mean + 1e-6).sqrt()) * y)
    c, s = t["cos"][:n, None], t["sin"][:n, None]
    a, b = (y[..., : dim // 2], y[..., dim // 2:]) if half else (y[..., 0::2], y[..., 1::2])
    u, v = a * c - b * s, a * s + b * c
    y = torch.cat([u, v], -1) if half else torch.stack([u, v], -1).flatten(-2)
    assert torch.equal(t["q"].view(n, heads, dim), y[:, :heads])
    want = torch.stack([y[:, heads:], x[:, heads + kv:]], 1)
    grid, low, high = (16, -128, 127) if fmt == "q8" else (2048, -32768, 32767)
    want = (want * grid + 0.5).floor().clamp(low, high) / grid
    have = cache.rows_of(0).permute(2, 0, 1, 3).float()
    assert torch.equal(have, want)


@pytest.mark.gpu
def test_append_codec_borders_and_rails():
    """The codec's ties, rails and infinities, value by value, as the slot cache's own encoder gives them."""
    dim = 16
    x = np.array([0.03125, -0.03125, 7.96875, 7.97, 8.0, -8.03125, -8.04, np.inf, -np.inf, 1e30, 0.0, -0.0,
                  15.99951171875, 15.9998, 16.0, -16.1], np.float32)
    gpu = vc4b200.GPU(0)
    for fmt, bits in (("q8", 8), ("q16", 16)):
        cache = Cache([1], [1], fmt, 16, 1, dim)
        handle, batch = cache.handles(vc4b200, gpu)
        qkv = torch.from_numpy(np.concatenate([x, x, x])).cuda()
        q = torch.empty(dim, device="cuda")
        torch.cuda.synchronize()
        handle.append(batch, qkv.data_ptr(), "f32", 1, q.data_ptr(), "f32")
        gpu.sync()
        want = np.empty(dim * bits // 8, np.uint8)
        assert vc4b200.lib().vc4_kv_codec_probe(0, bits, x.ctypes.data_as(C.c_void_p), dim, want.ctypes.data_as(C.c_void_p)) == 0
        pg = int(cache.host_table[0, 0])
        for sel in (0, 1):
            assert cache.pool[pg, sel, 0, 0].cpu().contiguous().view(torch.uint8).numpy().tobytes() == want.tobytes()
        assert torch.equal(q, qkv[:dim])


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["page high", "page negative", "length short", "table short", "rotation short", "max_new"])
def test_append_flags_bad_entries_and_skips_them(what):
    cache = Cache([20, 9], [4, 2], "bf16", 16, 2, 64, spare=2)
    t, kw = _append_case(cache, 4, "f32", "bf16", False, True)
    good_row = slice(4, 6)      # sequence 1 stays good
    over = {}
    if what.startswith("page"):
        cache.table[0, 1] = cache.pages if what == "page high" else -1
    elif what == "length short":
        cache.len[0] = 3
    elif what == "table short":
        cache.len[0] = 16 * cache.width + 2
    elif what == "rotation short":
        kw["rope_len"] = 19
    else:
        over["max_new"] = 3
    gpu = vc4b200.GPU(0)
    handle, batch = cache.handles(vc4b200, gpu, **over)
    before = cache.pool.clone()
    torch.cuda.synchronize()
    handle.append(batch, t["qkv"].data_ptr(), "f32", 4, t["q"].data_ptr(), "bf16", **kw)
    gpu.sync()
    assert int(cache.status) == EINVAL
    assert not bool((t["q"][good_row] == 7).any())
    changed = (cache.pool != before).any(-1).any(-1).any(-1).any(-1)
    mine = {int(cache.host_table[0, 0]), int(cache.host_table[0, 1]), int(cache.host_table[1, 0])}
    assert set(torch.nonzero(changed).flatten().tolist()) <= mine


# ---- attention ------------------------------------------------------------------------

def _attend(cache, heads, kind, out_kind, q, scale=0.0, pad=0, stream=0, gpu=None, **bounds):
    gpu = gpu or vc4b200.GPU(0)
    handle, batch = cache.handles(vc4b200, gpu, **bounds)
    width = heads * cache.dim
    out = torch.full((cache.rows, width + pad), 7.0, dtype=TORCH[out_kind], device="cuda")
    need = handle.attend_bytes(batch, heads)
    work = torch.full((max(16, need),), 255, dtype=torch.uint8, device="cuda")   # NaN, should anything stale be read
    torch.cuda.synchronize()
    handle.attend(batch, q.data_ptr(), kind, heads, out.data_ptr(), out_kind, work.data_ptr(), need, scale=scale,
                  q_stride=q.stride(0), out_stride=width + pad, stream=stream)
    torch.cuda.synchronize()
    return out, width


def _check_attend(cache, heads, kind, out_kind, scale=0.0, pad=0, gain=1.5, seed=3, hidden=(), **bounds):
    g = torch.Generator().manual_seed(seed)
    width = heads * cache.dim
    q = (gain * torch.randn(cache.rows, width + pad, generator=g)).to(TORCH[kind]).cuda()
    out, _ = _attend(cache, heads, kind, out_kind, q, scale, pad, **bounds)
    want, mass, top = attention(cache, q[:, :width], heads, scale or None, hidden)
    have = out[: cache.tokens, :width].double().view_as(want)
    bound = attention_bound(cache.fmt, out_kind, want, mass, top, cache.dim)
    far = (have - want).abs() / bound
    assert bool(torch.isfinite(have).all()) and float(far.max() if far.numel() else 0) <= 1, float(far.max())
    assert bool((out[cache.tokens:] == 7).all()) and bool((out[:, width:] == 7).all())
    return out


def _kind(fmt, other="bf16"):
    return fmt if fmt in ("bf16", "f16") else other


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["q8", "q16", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,page", SHAPES)
@pytest.mark.parametrize("new", [1, 3, 37])
def test_attend(fmt, heads, kv, dim, page, new):
    """Every format, head size and page length; lengths around tiles and pages,
    sequences without new tokens, rows and columns behind the batch."""
    length = [new, new + 1, 15 + new, 64, 65 + new, 130 + new, 40, 257 + new, 700]
    cache = Cache(length, [new, new, new, new, new, new, 0, new, min(new, 2)], fmt, page, kv, dim, rows=9 * new + 5,
                  fill=float("nan") if fmt in ("bf16", "f16") else 127)
    _check_attend(cache, heads, _kind(fmt), {1: "bf16", 3: "f32", 37: "f16"}[new], pad=8)
    assert int(cache.status) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,kind", [("q8", "f16"), ("q16", "f16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("heads,kv,dim,new,length", [
    (8, 4, 96, 1, 9000), (32, 8, 128, 1, 5000), (16, 2, 64, 5, 4097), (12, 12, 64, 2, 2047), (64, 8, 128, 3, 3001)])
def test_attend_long(fmt, kind, heads, kv, dim, new, length):
    """Few rows over many positions: the positions are split over blocks, a
    short sequence beside the long one leaves splits empty."""
    cache = Cache([length, new, 70 + new], [new, new, new], fmt, 32, kv, dim)
    _check_attend(cache, heads, kind, "f32", scale=0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["q8", "q16", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,page,new,past", [
    (8, 4, 96, 16, 300, 500), (32, 8, 128, 128, 129, 64), (16, 2, 64, 32, 513, 0), (7, 1, 128, 16, 200, 1), (4, 4, 64, 64, 1000, 333),
    (28, 4, 128, 32, 90, 1000)])
def test_attend_chunk(fmt, heads, kv, dim, page, new, past):
    """Prompt chunks: many rows, the diagonal inside tiles; a second ragged one beside it."""
    cache = Cache([past + new, past // 2 + new - 7], [new, new - 7], fmt, page, kv, dim, rows=2 * new,
                  fill=float("nan") if fmt in ("bf16", "f16") else 127)
    _check_attend(cache, heads, _kind(fmt), _kind(fmt))


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 150])
def test_attend_large_scores_and_one_position(new):
    """Scores of a few hundred (one weight takes all) and a single position."""
    cache = Cache([new, 400 + new], [new, new], "bf16", 16, 2, 64)
    _check_attend(cache, 8, "bf16", "f32", gain=40.0)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_attend_bad_pages_are_not_read(fmt, new):
    """A page id outside the pool hides its positions and sets the status."""
    cache = Cache([200 + new, 64 + new], [new, new], fmt, 16, 2, 64)
    good = cache.host_table.copy()
    cache.table[0, 3] = cache.pages + 5
    cache.table[0, 7] = -2
    assert (cache.host_table == good).all()
    _check_attend(cache, 4, "bf16", "f32", hidden=list(range(48, 64)) + list(range(112, 128)))
    assert int(cache.status) == EINVAL


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_attend_rows_that_see_nothing_are_zero(fmt):
    """Every page bad, or fewer positions than new tokens: zero, and the status says so."""
    cache = Cache([40, 90], [2, 2], fmt, 16, 2, 64)
    cache.table[0] = -1
    q = torch.randn(4, 4 * 64, device="cuda").to(torch.bfloat16)
    out, _ = _attend(cache, 4, "bf16", "f32", q)
    assert bool((out[:2] == 0).all()) and bool((out[2:] != 0).any()) and int(cache.status) == EINVAL
    cache = Cache([40, 90], [3, 2], fmt, 16, 2, 64)
    cache.len[0] = 2
    q = torch.randn(5, 4 * 64, device="cuda").to(torch.bfloat16)
    out, _ = _attend(cache, 4, "bf16", "f32", q)
    assert bool((out[0] == 0).all()) and bool(torch.isfinite(out).all()) and int(cache.status) == EINVAL


@pytest.mark.gpu
@pytest.mark.parametrize("new", [2, 100])
@pytest.mark.parametrize("cu", [(0, "all", "more"), (-1, "all", "all"), (0, "all", 1)])
def test_attend_flags_bad_offsets(new, cu):
    """Offsets past the batch's rows, below them or running backwards: flagged, nothing outside the rows touched."""
    cache = Cache([300, 200], [new, new], "bf16", 16, 1, 64)
    cache.cu.copy_(torch.tensor([{"all": new, "more": 2 * new + 1}.get(c, c) for c in cu], dtype=torch.int32))
    if cu[2] == "all":
        cache.cu[2] = 2 * new
    q = torch.randn(cache.rows, 64, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    _attend(cache, 1, "bf16", "f32", q)
    assert int(cache.status) == EINVAL


@pytest.mark.gpu
def test_attend_infinite_and_nan_values_reach_only_rows_that_see_them():
    """Positions no row sees may hold anything; a NaN score is not hidden."""
    cache = Cache([50], [1], "bf16", 16, 1, 64, fill=float("nan"))
    q = torch.randn(1, 128, device="cuda").to(torch.bfloat16)
    out, _ = _attend(cache, 2, "bf16", "f32", q)
    assert bool(torch.isfinite(out).all())
    cache.pool[int(cache.host_table[0, 1]), 0, 0, 4, 3] = float("nan")     # K of position 20
    out, _ = _attend(cache, 2, "bf16", "f32", q)
    assert bool(torch.isnan(out).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,new,past", [(2, 1, 64, 5, 40), (8, 2, 128, 9, 300), (4, 4, 96, 7, 5000), (4, 1, 128, 100, 60),
                                                   (2, 2, 64, 300, 200), (8, 1, 80, 90, 3000), (4, 1, 48, 100, 60),
                                                   (2, 1, 32, 200, 3000), (8, 2, 16, 70, 129)])
def test_attend_wild_values_of_later_tokens_stay_there(fmt, heads, kv, dim, new, past):
    """A new token whose K and V are infinite or NaN: the rows before it come out as
    without it, it and those after it are not finite."""
    at = new * 2 // 3
    cache = Cache([past + new, 33], [new, 1], fmt, 16, kv, dim)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(new + 1, heads * dim, generator=g).to(TORCH[fmt]).cuda()
    clean, _ = _attend(cache, heads, fmt, "f32", q)
    pos = past + at
    pg = int(cache.host_table[0, pos // 16])
    for k_value, v_value in ((None, float("inf")), (None, float("nan")), (float("nan"), float("-inf"))):
        pool = cache.pool.clone()
        cache.pool[pg, 1, kv - 1, pos % 16, dim - 1] = v_value
        cache.pool[pg, 1, kv - 1, pos % 16, 0] = v_value
        if k_value is not None:
            cache.pool[pg, 0, :, pos % 16] = k_value
        out, _ = _attend(cache, heads, fmt, "f32", q)
        assert torch.equal(out[:at], clean[:at]) and torch.equal(out[new:], clean[new:])
        mine = out[at:new].view(new - at, heads, dim)[:, -1]     # the last query head reads the last KV head
        assert not bool(torch.isfinite(mine[:, [0, dim - 1]]).any())
        cache.pool.copy_(pool)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,new", [("q8", 2), ("q8", 150), ("bf16", 2), ("bf16", 150), ("q16", 150)])
def test_pool_beyond_32_bits(fmt, new):
    """Pages whose bytes and values lie past 2^32: append and attention find them."""
    kv, dim, page, heads = 4, 64, 64, 8
    cache = Cache([300 + new, 70 + new], [new, new], fmt, page, kv, dim)
    small_pool, small_table, per = cache.pool, cache.host_table, 2 * kv * page * dim
    shift = (1 << 32) // per + 7
    big = torch.empty((shift + cache.pages) * per, dtype=POOL[fmt], device="cuda")
    big = big.view(-1, 2, kv, page, dim)
    big[shift:] = small_pool
    cache.table += shift * (cache.table >= 0).int()
    t, kw = _append_case(cache, heads, "bf16", _kind(fmt), True, True)
    gpu = vc4b200.GPU(0)
    handle, batch = cache.handles(vc4b200, gpu)
    handle = vc4b200.PagedKV(gpu, big.data_ptr(), fmt, big.shape[0], page, kv, dim)
    out = torch.zeros(2 * new, heads * dim, device="cuda")
    need = handle.attend_bytes(batch, heads)
    work = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    handle.append(batch, t["qkv"].data_ptr(), "bf16", heads, t["q"].data_ptr(), _kind(fmt), **kw)
    handle.attend(batch, t["q"].data_ptr(), _kind(fmt), heads, out.data_ptr(), "f32", work.data_ptr(), need)
    gpu.sync()
    assert int(cache.status) == 0
    cache.pool = big[shift:]
    q, k, v, off = _append_ref(cache, t, heads, True, True, True)
    row, pos = new - 1, cache.length[0] - 1
    have = decode(cache.pool, fmt)[int(small_table[0, pos // page]), 0, :, pos % page]
    step = 0.5 / GRID[fmt] if fmt in GRID else half_step(fmt) * float(k[row].abs().max())
    assert bool(((have - k[row].clamp(-16, 16)).abs() <= step * 1.01 + off[row, heads: heads + kv] + 1e-6).all())
    want, mass, top = attention(cache, t["q"], heads)
    assert bool(((out.double().view_as(want) - want).abs() <= attention_bound(fmt, "f32", want, mass, top, dim)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt,kind", [("q8", "bf16"), ("bf16", "bf16")])
def test_attend_same_bits_twice_and_on_another_stream(fmt, kind):
    cache = Cache([3000, 77], [2, 2], fmt, 32, 2, 128)
    q = torch.randn(4, 8 * 128, device="cuda").to(TORCH[kind])
    a, _ = _attend(cache, 8, kind, "f32", q)
    side = torch.cuda.Stream()
    b, _ = _attend(cache, 8, kind, "f32", q, stream=side.cuda_stream)
    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("new", [1, 90])
def test_captured_step_follows_its_arrays(new):
    """Append and attend captured once: replays follow lengths and tables that
    change within the bounds, and two graphs with buffers of their own overlap."""
    heads, kv, dim, page = 8, 2, 64, 16
    gpu = vc4b200.GPU(0)
    graphs = []
    for seed in (0, 1):
        cache = Cache([500 + new, 300 + new], [new, new], "bf16", page, kv, dim, seed=seed, width=60)
        t, kw = _append_case(cache, heads, "bf16", "bf16", True, True, seed=seed)
        handle, batch = cache.handles(vc4b200, gpu, max_len=900)
        out = torch.zeros(2 * new, heads * dim, device="cuda")
        need = handle.attend_bytes(batch, heads)
        work = torch.empty(max(16, need), dtype=torch.uint8, device="cuda")
        cos, sin = vc4b200.rope_tables(1e4, dim, 900)
        t["cos"], t["sin"] = torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda()
        kw.update(cos=t["cos"].data_ptr(), sin=t["sin"].data_ptr(), rope_len=900)

        def step(stream):
            handle.append(batch, t["qkv"].data_ptr(), "bf16", heads, t["q"].data_ptr(), "bf16", stream=stream, **kw)
            handle.attend(batch, t["q"].data_ptr(), "bf16", heads, out.data_ptr(), "f32", work.data_ptr(), need,
                          stream=stream)
        torch.cuda.synchronize()
        step(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(torch.cuda.current_stream().cuda_stream)
        graphs.append((graph, cache, t, out, work, step))
    for grow in (0, 37):
        for graph, cache, t, out, *_ in graphs:
            spare = [p for p in range(cache.pages) if p not in set(cache.host_table[cache.host_table >= 0].tolist())]
            for s in (0,):    # sequence 0 grows into spare pages
                cache.length[s] += grow
                for e in range((cache.length[s] + page - 1) // page):
                    if cache.host_table[s, e] < 0:
                        cache.host_table[s, e] = spare.pop()
            cache.len.copy_(torch.tensor(cache.length, dtype=torch.int32))
            cache.table.copy_(torch.from_numpy(cache.host_table))
            out.zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, *_), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for graph, cache, t, out, *_ in graphs:
            assert int(cache.status) == 0
            want, mass, top = attention(cache, t["q"], heads)
            bound = attention_bound("bf16", "f32", want, mass, top, dim)
            assert bool(((out.double().view_as(want) - want).abs() <= bound).all())


@pytest.mark.gpu
def test_no_tokens_and_work_buffer():
    gpu = vc4b200.GPU(0)
    cache = Cache([5000], [100], "q8", 16, 2, 64)
    handle, batch = cache.handles(vc4b200, gpu)
    need = handle.attend_bytes(batch, 4)
    assert need > 0
    q = torch.randn(100, 256, device="cuda").to(torch.bfloat16)
    out = torch.zeros(100, 256, device="cuda")
    _refused(lambda: handle.attend(batch, q.data_ptr(), "bf16", 4, out.data_ptr(), "f32", out.data_ptr(), need - 1), "work buffer")
    _refused(lambda: handle.attend(batch, q.data_ptr(), "bf16", 4, out.data_ptr(), "f32", 0, need), "work buffer")
    empty = vc4b200.PagedBatch(cache.cu.data_ptr(), cache.len.data_ptr(), cache.table.data_ptr(), 1, 0, 0, 0, cache.width)
    handle.attend(empty, q.data_ptr(), "bf16", 4, out.data_ptr(), "f32")
    handle.append(empty, q.data_ptr(), "bf16", 4, out.data_ptr(), "f32")
    torch.cuda.synchronize()
    assert bool((out == 0).all())


# ---- offsets of any kind ------------------------------------------------------------------

OFFSETS = [  # offsets of two or three sequences over 6 rows, those that stand
    ([0, 3, 9], [0]), ([0, 3, 2], [0]), ([-1, 3, 6], [1]), ([-2, -1, 6], []), ([4, 2, 6], [1]), ([0, 3, 1, 6], []),
    ([0, 2, 7, 7], [0]), ([0, 6, 4], [0])]


@pytest.mark.gpu
@pytest.mark.parametrize("cu,good", OFFSETS)
@pytest.mark.parametrize("fmt", ["q8", "bf16"])
def test_append_flags_bad_offsets(fmt, cu, good):
    """Offsets that start below 0, run backwards or end past the rows: flagged; a sequence
    with such an offset writes nothing, the others what they write alone.  (Rows of two
    sequences that overlap belong to one of them.)"""
    seqs, heads, kv, dim = len(cu) - 1, 4, 2, 64
    cache = Cache([40] * seqs, [3] * seqs, fmt, 16, kv, dim, rows=6)
    cache.new = [6] * seqs                       # max_new of the batch: no bound of its own here
    t, kw = _append_case(cache, heads, "f32", "bf16", True, True)
    gpu = vc4b200.GPU(0)
    cache.cu.copy_(torch.tensor(cu, dtype=torch.int32))
    handle, batch = cache.handles(vc4b200, gpu)
    before = cache.pool.clone()
    torch.cuda.synchronize()
    handle.append(batch, t["qkv"].data_ptr(), "f32", heads, t["q"].data_ptr(), "bf16", **kw)
    gpu.sync()
    assert int(cache.status) == EINVAL
    pages = lambda s: torch.from_numpy(cache.host_table[s, :3].astype(np.int64)).cuda()  # noqa: E731
    for s in range(seqs):
        now, was = cache.pool[pages(s)], before[pages(s)]
        if 0 <= cu[s] <= cu[s + 1] <= 6 and s in good:
            n = cu[s + 1] - cu[s]
            alone = Cache([40], [n], fmt, 16, kv, dim, rows=6)
            alone.pool, alone.pages = before.clone(), cache.pages
            alone.table.copy_(cache.table[s: s + 1])
            alone.cu.copy_(torch.tensor([cu[s], cu[s + 1]], dtype=torch.int32))
            h, b = alone.handles(vc4b200, gpu)
            q = torch.full_like(t["q"], 7.0)
            torch.cuda.synchronize()
            h.append(b, t["qkv"].data_ptr(), "f32", heads, q.data_ptr(), "bf16", **kw)
            gpu.sync()
            assert int(alone.status) == 0 and torch.equal(now, alone.pool[pages(s)])
            assert torch.equal(t["q"][cu[s]: cu[s + 1]], q[cu[s]: cu[s + 1]])
        elif not (0 <= cu[s] <= cu[s + 1] <= 6):
            assert torch.equal(now, was)
    inside = torch.zeros(6, dtype=torch.bool, device="cuda")
    for s in range(seqs):
        if 0 <= cu[s] <= cu[s + 1] <= 6:
            inside[cu[s]: cu[s + 1]] = True
    assert bool((t["q"][~inside] == 7).all())


@pytest.mark.gpu
def test_append_flags_a_bad_offset_among_many_sequences():
    """The offset that runs backwards lies past every row: no token's look-up meets it."""
    seqs = 3000
    cache = Cache([20] * 2, [1] * 2, "q8", 16, 1, 16, rows=2)
    cu = torch.full((seqs + 1,), 2, dtype=torch.int32, device="cuda")
    cu[0], cu[1] = 0, 1
    length = torch.full((seqs,), 20, dtype=torch.int32, device="cuda")
    table = cache.table[:1].repeat(seqs, 1).contiguous()
    t, kw = _append_case(cache, 1, "f32", "f32", False, True)
    gpu = vc4b200.GPU(0)
    handle, _ = cache.handles(vc4b200, gpu)
    for bad in (False, True):
        if bad:
            cu[2900] = 1
        batch = vc4b200.PagedBatch(cu.data_ptr(), length.data_ptr(), table.data_ptr(), seqs, 2, 1, 20, cache.width,
                                   status=cache.status.data_ptr())
        torch.cuda.synchronize()
        handle.append(batch, t["qkv"].data_ptr(), "f32", 1, t["q"].data_ptr(), "f32", **kw)
        gpu.sync()
        assert int(cache.status) == (EINVAL if bad else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("cu,good", [((0, 100, 201), [0]), ((-1, 100, 200), [1]), ((0, 100, 1), [0]), ((100, 100, 200), [0, 1]),
                                     ((-5, -1, 200), []), ((0, 2 ** 31 - 1, 200), []), ((-2 ** 31, 100, 200), [1])])
@pytest.mark.parametrize("heads,length", [(1, 300), (4, 3000), (8, 130)])
def test_attend_leaves_rows_of_bad_offsets(heads, length, cu, good):
    """Many rows, their positions split or not: a sequence that starts below 0, ends
    before it starts or past the rows is skipped, its rows and those behind the batch stay;
    the others are the definition's."""
    new, dim = 100, 64
    cache = Cache([length, length - 90], [new, new], "bf16", 16, 1, dim, rows=2 * new)
    # (a length below the new tokens is flagged too: 40 positions for 100 tokens)
    bad = not 0 <= cu[0] <= cu[1] <= cu[2] <= 2 * new or length - 90 < cu[2] - cu[1]
    cache.cu.copy_(torch.tensor(cu, dtype=torch.int32))
    q = torch.randn(2 * new, heads * dim, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16).cuda()
    out, _ = _attend(cache, heads, "bf16", "f32", q)
    assert int(cache.status) == (EINVAL if bad else 0)
    left = torch.ones(2 * new, dtype=torch.bool, device="cuda")
    cache.host_cu = np.maximum(0, np.minimum(cu, 2 * new))
    cache.new = [max(0, int(n)) if s in good else 0 for s, n in enumerate(cache.host_cu[1:] - cache.host_cu[:-1])]
    cache.tokens = 2 * new
    want, mass, top = attention(cache, q, heads)
    bound = attention_bound("bf16", "f32", want, mass, top, dim)
    for s in good:
        rows = slice(int(cache.host_cu[s]), int(cache.host_cu[s]) + cache.new[s])
        assert bool(((out[rows].double().view_as(want[rows]) - want[rows]).abs() <= bound[rows]).all())
        left[rows] = False
    assert bool((out[left] == 7).all())


@pytest.mark.parametrize("name", ["cu", "length", "table", "status"])
@pytest.mark.parametrize("off", [1, 2])
def test_batches_off_their_elements_are_refused(name, off):
    batch = _host_batch(**{name: 64 + off})
    _refused(lambda: _host_pages().append(batch, 64, "f32", 4, 64, "bf16"), "aligned to their elements")
    _refused(lambda: _host_pages().attend(batch, 64, "bf16", 4, 64, "bf16"), "aligned to their elements")
    _refused(lambda: _host_pages().attend_bytes(batch, 4), "aligned to their elements")


# ---- buffers that overlap -----------------------------------------------------------------

class _SomeGpu:
    """A handle that a refusal does not look into."""
    _h = 1


@pytest.mark.parametrize("q,kw,words", [
    (0x10000, {}, "q overlaps qkv"), (0x10000 + 4 * 512 * 4 - 16, {}, "q overlaps qkv"), (0x10000 - 16, {}, "q overlaps qkv"),
    (0x10000 - 4 * 256 * 2 + 16, {}, "q overlaps qkv"),                       # the last row's end
    (0x10000 + 512 * 4, dict(qkv_stride=600, q_stride=1200), None),            # in the rows' gaps: 88 floats < 256 bf16
    (0x10000 + 512 * 4, dict(qkv_stride=1024, q_stride=2048), "pool"),         # fits the gaps
    (0x10000 - 512, dict(qkv_stride=640, q_stride=1280), "pool"),              # ahead of each row
    (0x10000 - 528, dict(qkv_stride=640, q_stride=1280), "q overlaps qkv"),    # and round into the row before
    (0x10000 + 512 * 4, dict(qkv_stride=1024, q_stride=2040), "q overlaps qkv"),
    (0x10000 + 4 * 512 * 4, {}, "pool"), (0x10000 - 4 * 256 * 2, {}, "pool")])
def test_append_refuses_overlaps(q, kw, words):
    """Rows of 512 f32 (4 + 2 * 2 heads of 64) and 256 bf16, four tokens; the pool lies over all."""
    pages = _host_pages("q8", data=0x8000, pages=64)
    pages.gpu = _SomeGpu()
    _refused(lambda: pages.append(_host_batch(), 0x10000, "f32", 4, q, "bf16", **kw), words or "q overlaps qkv")


@pytest.mark.parametrize("out,kw,words", [
    (0x10000, {}, "out overlaps q"), (0x10000 + 2032, {}, "out overlaps q"), (0x10000 - 4080, {}, "out overlaps q"),
    (0x10000 + 512, dict(q_stride=512, out_stride=256), "out overlaps q"),
    (0x10000 + 512, dict(q_stride=768, out_stride=384), "out overlaps the pool"),
    (0x10000 + 2048, {}, "out overlaps the pool"), (0x10000 - 4096, {}, "out overlaps the pool")])
def test_attend_refuses_overlaps(out, kw, words):
    """Rows of 256 bf16 and 256 f32, four tokens."""
    pages = _host_pages("q8", data=0x8000, pages=64)
    pages.gpu = _SomeGpu()
    _refused(lambda: pages.attend(_host_batch(), 0x10000, "bf16", 4, out, "f32", **kw), words)


@pytest.mark.gpu
def test_rows_side_by_side_and_a_work_buffer_that_overlaps():
    """q and out as columns of one buffer; the work buffer over q, out or the pool is refused."""
    heads, dim, new = 4, 64, 90
    gpu = vc4b200.GPU(0)
    cache = Cache([3000], [new], "bf16", 16, 2, dim)
    handle, batch = cache.handles(vc4b200, gpu)
    need = handle.attend_bytes(batch, heads)
    assert need > 0
    both = torch.randn(new, 2 * heads * dim, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    q, out = both[:, : heads * dim], both[:, heads * dim:]
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    kw = dict(q_stride=both.stride(0), out_stride=both.stride(0))
    for at in (q, out, cache.pool):
        _refused(lambda: handle.attend(batch, q.data_ptr(), "bf16", heads, out.data_ptr(), "bf16", at.data_ptr(), need, **kw), "overlaps")
    torch.cuda.synchronize()
    handle.attend(batch, q.data_ptr(), "bf16", heads, out.data_ptr(), "bf16", work.data_ptr(), need, **kw)
    gpu.sync()
    want, mass, top = attention(cache, q, heads)
    bound = attention_bound("bf16", "bf16", want, mass, top, dim)
    assert int(cache.status) == 0 and bool(((out.double().reshape(want.shape) - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["q8", "q16", "bf16", "f16"])
@pytest.mark.parametrize("new", [1, 100])
@pytest.mark.parametrize("length", [-1, -2 ** 31 + 1, -2 ** 31])
def test_negative_lengths_see_nothing(fmt, new, length):
    """However far below 0 a length lies: nothing is appended, the rows are zero, the others stand."""
    cache = Cache([50 + new, 70 + new], [new, new], fmt, 16, 1, 64)
    _check_attend(cache, 2, _kind(fmt), _kind(fmt))
    cache.len[0] = length
    before = cache.pool.clone()
    t, kw = _append_case(cache, 2, "f32", "f32", False, True)
    gpu = vc4b200.GPU(0)
    handle, batch = cache.handles(vc4b200, gpu)
    torch.cuda.synchronize()
    handle.append(batch, t["qkv"].data_ptr(), "f32", 2, t["q"].data_ptr(), "f32", **kw)
    gpu.sync()
    mine = torch.from_numpy(cache.host_table[0][cache.host_table[0] >= 0].astype(np.int64)).cuda()
    assert int(cache.status) == EINVAL and torch.equal(cache.pool[mine], before[mine]) and bool((t["q"][:new] == 7).all())
    cache.status.zero_()
    q = torch.randn(2 * new, 128, generator=torch.Generator().manual_seed(2)).to(TORCH[_kind(fmt)]).cuda()
    out, _ = _attend(cache, 2, _kind(fmt), _kind(fmt), q)
    want, mass, top = attention(cache, q, 2)
    bound = attention_bound(fmt, _kind(fmt), want, mass, top, 64)
    assert int(cache.status) == EINVAL and bool((out[:new] == 0).all())
    assert bool(((out[new:].double().view_as(want[new:]) - want[new:]).abs() <= bound[new:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv", [(4, 4), (64, 1)])
@pytest.mark.parametrize("new,max_new", [(1, 1000), (3, 2 ** 31 - 1), (100, 2 ** 31 - 1)])
def test_attend_bounds_far_above_the_tokens(heads, kv, new, max_new):
    """max_new is a bound: one beyond the batch's rows asks for no more work than they are."""
    cache = Cache([500 + new] * 40, [new] * 40, "q8", 16, kv, 64)
    gpu = vc4b200.GPU(0)
    (handle, tight), (_, wide) = cache.handles(vc4b200, gpu, max_new=40 * new), cache.handles(vc4b200, gpu, max_new=max_new)
    assert handle.attend_bytes(tight, heads) == handle.attend_bytes(wide, heads)
    _check_attend(cache, heads, "bf16", "bf16", max_new=max_new)
    assert int(cache.status) == 0


def test_bytes_of_too_many_rows_are_refused():
    _refused(lambda: _host_pages().attend_bytes(_host_batch(tokens=2 ** 29, max_new=2 ** 29), 4), "too many rows")


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,new,past", [
    (2, 1, 64, 5, 40), (8, 2, 128, 9, 300), (4, 4, 96, 7, 5000), (4, 1, 128, 100, 60), (2, 2, 64, 300, 200), (8, 1, 80, 90, 3000),
    (4, 1, 48, 100, 60), (2, 1, 32, 200, 3000), (8, 2, 16, 70, 129), (1, 1, 16, 64, 0), (2, 2, 128, 513, 1000)])
@pytest.mark.parametrize("out_kind", ["f32", "bf16"])
def test_attend_wild_values_stay_in_their_columns(fmt, heads, kv, dim, new, past, out_kind):
    """Infinite and NaN V of new tokens: their columns of the rows that see them are what the
    sum is, infinite or NaN, every other value as without them, however many tokens are fed together."""
    first, second = new // 3, new * 2 // 3
    cache = Cache([33, past + new], [1, new], fmt, 16, kv, dim)
    g = torch.Generator().manual_seed(6)
    q = torch.randn(new + 1, heads * dim, generator=g).to(TORCH[fmt]).cuda()
    clean, _ = _attend(cache, heads, fmt, out_kind, q)
    inf, nan = float("inf"), float("nan")
    plants = [(first, 0, inf), (second, 0, -inf), (second, dim - 1, nan), (first, dim // 2 + 1, -inf), (second, dim // 2 + 1, -inf)]
    want = clean.view(new + 1, heads, dim).clone()
    for at, d, value in plants:
        pg, off = int(cache.host_table[1, (past + at) // 16]), (past + at) % 16
        cache.pool[pg, 1, kv - 1, off, d] = value
        want[1 + at:, heads - heads // kv:, d] = value
    want[1 + second:, heads - heads // kv:, 0] = nan             # both infinities
    out, _ = _attend(cache, heads, fmt, out_kind, q)
    assert torch.equal(torch.nan_to_num(out, nan=7.5).view_as(want), torch.nan_to_num(want, nan=7.5))
    for at in (first, second, new - 1):                          # the same row fed alone
        one = Cache([past + at + 1], [1], fmt, 16, kv, dim)
        one.pool, one.pages = cache.pool, cache.pages
        one.table.copy_(cache.table[1:, : one.width])
        alone, _ = _attend(one, heads, fmt, out_kind, q[1 + at: 2 + at])
        a, b = alone.view(heads, dim), want[1 + at]
        assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
        assert torch.equal(a[torch.isinf(a)], b[torch.isinf(b)])


# ---- q16 levels whole ---------------------------------------------------------------------

def _levels(cache, sel, pos, levels):
    """Plants int16 levels ([kv][dim] or one number) of K (0) or V (1) at a position of sequence 0."""
    x = torch.as_tensor(levels).expand(cache.kv, cache.dim).to(torch.int16).contiguous()
    cache.pool[int(cache.host_table[0, pos // 16]), sel, :, pos % 16] = swap16(x).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [16, 48, 64, 128])
@pytest.mark.parametrize("heads", [2, 32, 64, 128, 300])
@pytest.mark.parametrize("kind,out_kind", [("f16", "f32"), ("bf16", "f32"), ("f16", "f16")])
def test_attend_q16_scores_use_all_bits_of_a_level(dim, heads, kind, out_kind):
    """f16 and float outputs: two positions whose levels, 16391 and 16393, an f16 operand rounds
    8 times as far apart.  The bound is the definition's for exact operands (twice the products)."""
    cache = Cache([2], [1], "q16", 16, 2, dim)
    for pos, k, v in ((0, 16391, 16384), (1, 16393, -16384)):
        _levels(cache, 0, pos, k)
        _levels(cache, 1, pos, v)
    q = torch.full((1, heads * dim), 8.0, dtype=TORCH[kind], device="cuda")
    out, _ = _attend(cache, heads, kind, out_kind, q)
    want, mass, top = attention(cache, q, heads)
    bound = attention_bound("f16", out_kind, want, mass, top, 2 * dim)
    rounded = 8 * math.tanh(-8 * 8 / 2048 * math.sqrt(dim))     # 16384 and 16400
    assert float((rounded - want).abs().min()) > 4 * float(bound.max())
    assert bool(((out.double().view_as(want) - want).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [16, 64, 80, 128])
@pytest.mark.parametrize("heads", [2, 32, 64, 128, 300])
def test_attend_q16_values_use_all_bits_of_a_level(dim, heads):
    """Float outputs of one position are its V: 2^-21 for the exponential and the quotient, a
    128th of what an f16 operand drops of an odd level near 2^14 (7 of 16391)."""
    cache = Cache([1], [1], "q16", 16, 2, dim)
    g = torch.Generator().manual_seed(dim)
    v = torch.randint(-32768, 32768, (2, dim), generator=g)
    v[:, :6] = torch.tensor([16391, -16391, 32767, -32768, 1, -1])
    _levels(cache, 1, 0, v)
    out, _ = _attend(cache, heads, "f16", "f32", torch.zeros(1, heads * dim, dtype=torch.float16, device="cuda"))
    want = (v.double() / 2048).repeat_interleave(heads // 2, 0).cuda()
    assert bool(((out.double().view_as(want) - want).abs() <= 2.0 ** -21 * want.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["q8", "q16", "bf16", "f16"])
@pytest.mark.parametrize("seqs,new,length", [(2, 100, 3000), (40, 200, 900), (2, 700, 900)])
def test_attend_many_rows_same_bits_twice(fmt, seqs, new, length):
    """Split positions or not, on one stream and another: the same inputs, the same bits."""
    cache = Cache([length - 3 * s for s in range(seqs)], [new] * seqs, fmt, 32, 2, 64)
    q = torch.randn(cache.rows, 8 * 64, generator=torch.Generator().manual_seed(1)).to(TORCH[_kind(fmt)]).cuda()
    a, _ = _attend(cache, 8, _kind(fmt), _kind(fmt), q)
    side = torch.cuda.Stream()
    for stream in (0, side.cuda_stream, 0):
        b, _ = _attend(cache, 8, _kind(fmt), _kind(fmt), q, stream=stream)
        assert torch.equal(a, b)
