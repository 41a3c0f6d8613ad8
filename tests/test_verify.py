"""vc4_verify_draft against its definition in 64 bits, vc4_step_draft against the
serial steps, and the paged operators and the verification run together."""
import math

import numpy as np
import pytest
import torch

import vc4b200
from paged_ref import TORCH, Cache, attention, attention_bound
from vc4b200 import mmcf_writer, synth

EINVAL, ERANGE = 1, 6


def reference(counts, fed, logits, probs, u, u_sample, temperature):
    """(next, accepted, prob, clear) by the definition, row by row in doubles.
    clear: no decision is nearer to its border than the operator's arithmetic
    reaches: 2^-18 of p for a draft (p stands over a float sum, 2^-20 an
    exponential), 1e-12 of the total for a sample (sums in double)."""
    nxt, acc, prob, clear = [], [], [], True
    row = d = 0
    for s, n in enumerate(counts):
        mine, pr = [], []
        for i in range(n):
            l = np.where(np.isnan(logits[row + i]), -np.inf, logits[row + i].astype(np.float64))
            top = l.max()
            if top == -np.inf:
                p = None
            elif temperature == 0:
                p = np.zeros_like(l)
                p[int(np.argmax(l))] = 1
            else:
                with np.errstate(invalid="ignore"):
                    e = np.where(l == top, 1.0, np.exp((l - top) / temperature))
                p = e / e.sum()
            last = i == n - 1
            x = -1 if last else int(fed[row + i + 1])
            known = 0 <= x < l.size
            if not last:
                px = p[x] if p is not None and known else 0.0
                dx = 1.0 if probs is None or not known else float(probs[d + i, x])
                clear &= px == 0 or abs(float(u[row + i]) * dx - px) > 2.0 ** -18 * px
                if float(u[row + i]) * dx < px:
                    mine.append(x)
                    pr.append(px)
                    continue
            if p is None:
                mine.append(-1)
                pr.append(0.0)
                break
            r = p.copy()
            if not last and probs is not None:
                r = np.maximum(p - probs[d + i].astype(np.float64), 0)
            elif not last and known:
                r[x] = 0
            if not r.sum() > 0:
                r = p
            c = np.cumsum(r)
            goal = float(u_sample[s]) * c[-1]
            v = int(np.argmax(c > goal)) if (c > goal).any() else int(np.nonzero(r)[0][-1])
            clear &= min(abs(c[v] - goal), abs(goal - (c[v - 1] if v else -1.0))) > 1e-12 * c[-1]
            mine.append(v)
            pr.append(p[v])
            break
        acc.append(len(mine) - 1 if n else 0)
        nxt += mine + [-1] * (n - len(mine))
        prob += pr + [0.0] * (n - len(pr))
        row += n
        d += max(0, n - 1)
    return np.array(nxt, np.int64), np.array(acc, np.int64), np.array(prob), clear


def call(counts, fed, logits, kind, probs, u, u_sample, temperature, pad=0, rows=None, shift=0):
    """The operator on device copies; (next, accepted, prob, status) of every row and sequence."""
    gpu = vc4b200.GPU(0)
    vocab, n = logits.shape[1], sum(counts)
    rows = rows or max(1, n)
    store = torch.int32 if kind == "q16" else TORCH[kind]
    buf = torch.zeros(rows * (vocab + pad) + shift, dtype=store, device="cuda")
    lg = buf[shift: shift + rows * (vocab + pad)].view(rows, vocab + pad)
    lg[:n, :vocab] = logits.cuda()
    cu = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    dev = lambda x, t: torch.as_tensor(np.resize(x, rows) if len(x) < rows else x).to(t).cuda()  # noqa: E731
    f, uu, us = dev(fed, torch.int32), dev(u, torch.float32), torch.as_tensor(u_sample).float().cuda()
    dp = None if probs is None else torch.nn.functional.pad(probs.cuda(), (0, pad)).contiguous()
    nxt = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
    acc = torch.full((len(counts),), -9, dtype=torch.int32, device="cuda")
    pr, status = torch.full((rows,), -9.0, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    need = gpu.verify_bytes(len(counts), rows, vocab)
    work = torch.full((max(16, need),), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    gpu.verify_draft(len(counts), rows, vocab, cu.data_ptr(), f.data_ptr(), lg.data_ptr(), kind, temperature,
                     uu.data_ptr(), us.data_ptr(), nxt.data_ptr(), acc.data_ptr(), pr.data_ptr(), work.data_ptr(), need,
                     probs=0 if dp is None else dp.data_ptr(), logits_stride=vocab + pad, probs_stride=vocab + pad,
                     status=status.data_ptr())
    gpu.sync()
    assert bool((nxt[n:] == -9).all()) and bool((pr[n:] == -9).all())
    return nxt[:n].cpu().numpy(), acc.cpu().numpy(), pr[:n].cpu().numpy(), int(status)


def make(counts, vocab, kind, with_probs, seed, spread=2.0):
    """Logits and drafts sampled from a neighbouring distribution."""
    g = torch.Generator().manual_seed(seed)
    n = sum(counts)
    logits = spread * torch.randn(n, vocab, generator=g)
    logits = (logits * 256).round().to(torch.int32) if kind == "q16" else logits.to(TORCH[kind])
    value = logits.double() / 256 if kind == "q16" else logits.double()
    judged, row = [], 0
    for c in counts:
        judged += range(row, row + max(0, c - 1))
        row += c
    draft = (value[judged] + 0.5 * torch.randn(len(judged), vocab, generator=g).double()).softmax(-1).float()
    fed = torch.randint(0, vocab, (n,), generator=g)
    if judged:
        fed[torch.tensor(judged) + 1] = torch.multinomial(draft.double(), 1, generator=g)[:, 0]
    u, us = torch.rand(n, generator=g).numpy(), torch.rand(len(counts), generator=g).numpy()
    return logits, value.numpy(), fed.numpy(), draft if with_probs else None, u, us


def check(counts, vocab, kind, with_probs, temperature, seed=0, **kw):
    logits, value, fed, probs, u, us = make(counts, vocab, kind, with_probs, seed)
    want = reference(counts, fed, value, None if probs is None else probs.numpy(), u, us, temperature)
    assert want[3]
    got = call(counts, fed, logits, kind, probs, u, us, temperature, **kw)
    assert got[3] == 0
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    # p: exp in double over a float sum (2^-20 an exponential, the additions below that)
    assert np.all(np.abs(got[2] - want[2]) <= 2.0 ** -19 * want[2] + 1e-30)
    return got


# ---- refusals, before any GPU is asked for --------------------------------------------

class _Host(vc4b200.GPU):
    def __init__(self):
        self._h = None


@pytest.mark.parametrize("over,words", [
    (dict(seqs=0), "seqs"), (dict(vocab=0), "vocab"), (dict(rows=-1), "not negative"), (dict(rows=2 ** 31 - 1, vocab=100000), "too many"), (dict(seqs=2 ** 25), "too many"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=math.nan), "temperature"), (dict(temperature=math.inf), "temperature"), (dict(temperature=1e-6), "temperature"),
    (dict(cu=0), "null"), (dict(fed=0), "null"), (dict(logits=0), "null"), (dict(u=0), "null"), (dict(u_sample=0), "null"),
    (dict(next_tokens=0), "null"), (dict(accepted=0), "null"), (dict(logits=66), "aligned"), (dict(probs=66), "aligned"),
    (dict(logits_stride=99), "stride"), (dict(probs_stride=99), "stride"), (dict(work=0), "work buffer"), (dict(work=72), "work buffer"),
    (dict(work_bytes=1), "work buffer"),
    (dict(next_tokens=0x2004), "output overlaps an input"), (dict(accepted=0x1004), "output overlaps an input"),
    (dict(prob=0x4008), "output overlaps an input"), (dict(work=0x10010), "output overlaps an input"),
    (dict(next_tokens=0x20100, probs=0x20000), "output overlaps an input"), (dict(status=0x5000), "output overlaps an input"),
    (dict(accepted=0x6008), "two outputs overlap"), (dict(prob=0x6000), "two outputs overlap"), ({}, "gpu is null"),
    # neighbours are none of each other's
    (dict(next_tokens=0x200c, probs=0x20000, prob=0x20000 + 400), "gpu is null")])
def test_verify_refuses(over, words):
    a = dict(seqs=1, rows=3, vocab=100, cu=0x1000, fed=0x2000, logits=0x10000, logits_type="f32", temperature=1.0, u=0x4000,
             u_sample=0x5000, next_tokens=0x6000, accepted=0x7000, prob=0, work=0x30000, work_bytes=1 << 20)
    if "probs" in over and "next_tokens" in over:
        a["rows"] = 2 if "prob" in over else 3
    a.update(over)
    with pytest.raises(vc4b200.EngineError) as e:
        _Host().verify_draft(**a)
    assert "error %d" % EINVAL in str(e.value) and words in str(e.value), str(e.value)


def test_unknown_logits_type_is_refused():
    with pytest.raises(vc4b200.EngineError, match="unknown element type"):
        _Host().verify_draft(1, 1, 8, 64, 64, 64, "f64", 1.0, 64, 64, 64, 64, 0, 64, 1 << 20)


def test_reference_walk_by_hand():
    """The definition itself on numbers done by hand."""
    lg = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.8, 0.1], [0.2, 0.2, 0.6]]))
    # draft 0: u * 1 = 0.4 < 0.5 accepted; draft 1 at row 1: 0.9 > 0.8 refused, rest (0.1, 0, 0.1), goal 0.15 -> id 2
    got = reference([3], [9, 0, 1], lg, None, [0.4, 0.9, 0.0], [0.75], 1.0)
    assert got[0].tolist() == [0, 2, -1] and got[1].tolist() == [1]
    assert np.allclose(got[2], [0.5, 0.1, 0])


# ---- the operator ---------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 7, 33, 1025, 6400, 8191, 8192, 8193, 73448])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16", "q16"])
@pytest.mark.parametrize("with_probs", [False, True])
def test_verify(vocab, kind, with_probs):
    counts = [5, 1, 0, 3, 8, 2]
    check(counts, vocab, kind, with_probs, 0.8, seed=vocab)
    check(counts, vocab, kind, with_probs, 0.0, seed=vocab + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,pad,shift", [("f32", 3, 1), ("bf16", 5, 3), ("f16", 1, 7), ("q16", 2, 3)])
def test_verify_strides_and_alignment(kind, pad, shift):
    check([4, 4, 4], 9001, kind, True, 1.0, seed=5, pad=pad, shift=shift, rows=17)


@pytest.mark.gpu
def test_verify_rows_beyond_32_bits():
    """Rows 2^27 values apart: the last ones start past 2^32."""
    vocab, stride, counts = 700, 1 << 27, [20, 21]
    logits, value, fed, _, u, us = make(counts, vocab, "bf16", False, 12)
    want = reference(counts, fed, value, None, u, us, 0.9)
    assert want[3]
    buf = torch.empty(40 * stride + vocab, dtype=torch.bfloat16, device="cuda")
    torch.as_strided(buf, (41, vocab), (stride, 1)).copy_(logits)
    gpu = vc4b200.GPU(0)
    ints = lambda x: torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()  # noqa: E731
    cu, f, uu, uz = ints([0, 20, 41]), ints(fed), torch.from_numpy(u).cuda(), torch.from_numpy(us).cuda()
    nxt, acc = ints(np.zeros(41)), ints(np.zeros(2))
    need = gpu.verify_bytes(2, 41, vocab)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    gpu.verify_draft(2, 41, vocab, cu.data_ptr(), f.data_ptr(), buf.data_ptr(), "bf16", 0.9, uu.data_ptr(), uz.data_ptr(),
                     nxt.data_ptr(), acc.data_ptr(), 0, work.data_ptr(), need, logits_stride=stride)
    gpu.sync()
    assert np.array_equal(nxt.cpu().numpy(), want[0]) and np.array_equal(acc.cpu().numpy(), want[1])


@pytest.mark.gpu
def test_verify_captured_and_on_two_streams():
    """A captured call follows its arrays; two calls with buffers of their own overlap."""
    gpu, runs = vc4b200.GPU(0), []
    for seed in (1, 2):
        counts = [4, 6]
        logits, value, fed, probs, u, us = make(counts, 3001, "f32", True, seed)
        t = {"cu": torch.tensor([0, 4, 10], dtype=torch.int32).cuda(), "fed": torch.from_numpy(fed).int().cuda(),
             "logits": logits.cuda(), "probs": probs.cuda(), "u": torch.from_numpy(u).cuda(), "us": torch.from_numpy(us).cuda(),
             "next": torch.zeros(10, dtype=torch.int32).cuda(), "acc": torch.zeros(2, dtype=torch.int32).cuda()}
        need = gpu.verify_bytes(2, 10, 3001)
        t["work"] = torch.empty(need, dtype=torch.uint8, device="cuda")

        def step(t=t, need=need):
            gpu.verify_draft(2, 10, 3001, t["cu"].data_ptr(), t["fed"].data_ptr(), t["logits"].data_ptr(), "f32", 1.0,
                             t["u"].data_ptr(), t["us"].data_ptr(), t["next"].data_ptr(), t["acc"].data_ptr(), 0,
                             t["work"].data_ptr(), need, probs=t["probs"].data_ptr(),
                             stream=torch.cuda.current_stream().cuda_stream)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        runs.append((graph, t, counts, value, fed, probs, u, us))
    for change in (False, True):
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, t, *_), st in zip(runs, streams):
            if change:
                t["us"].copy_(1 - t["us"])
                torch.cuda.synchronize()
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for graph, t, counts, value, fed, probs, u, us in runs:
            want = reference(counts, fed, value, probs.numpy(), u, t["us"].cpu().numpy(), 1.0)
            assert want[3] and np.array_equal(t["next"].cpu().numpy(), want[0])


@pytest.mark.gpu
def test_verify_many_drafts_and_many_sequences():
    check([70, 33, 32, 31], 200, "f32", True, 1.3, seed=2)     # the walk takes 32 rows at a time
    check([2] * 500, 300, "bf16", True, 1.0, seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 3])
def test_verify_accepts_and_refuses_everywhere(n):
    """u of 0 accepts every draft with any probability; u of 1 refuses all but certain ones."""
    logits, value, fed, probs, u, us = make([n], 500, "f32", True, 9)
    nxt, acc, prob, _ = call([n], fed, logits, "f32", probs, np.zeros(n), us, 1.0)
    assert acc[0] == n - 1 and np.array_equal(nxt[: n - 1], fed[1:])
    nxt, acc, prob, _ = call([n], fed, logits, "f32", None, np.ones(n), us, 1.0)
    assert acc[0] == 0 and nxt[0] != fed[1] and np.all(nxt[1:] == -1) and np.all(prob[1:] == 0)


@pytest.mark.gpu
def test_verify_ends_of_the_sum():
    """u_sample of 0 gives the first id with any weight, one just below 1 the last; ids of -inf never."""
    lg = torch.zeros(1, 1000)
    lg[0, :10] = -math.inf
    lg[0, 990:] = -math.inf
    for us, want in ((0.0, 10), (np.float32(1 - 2.0 ** -24), 989), (1.0, 989), (0.5, 500)):
        nxt, acc, prob, st = call([1], [0], lg, "f32", None, [0.0], [us], 1.0)
        assert nxt[0] == want and acc[0] == 0 and st == 0 and abs(prob[0] - 1 / 980) < 1e-8


@pytest.mark.gpu
def test_verify_equal_distributions_fall_back_to_the_target():
    """Nothing is left of p - d: the refused row is sampled from p."""
    lg = torch.zeros(2, 4)
    d = torch.full((1, 4), 0.25)
    nxt, acc, prob, st = call([2], [0, 3], lg, "f32", d, [1.0, 0.0], [0.3], 1.0)
    assert acc[0] == 0 and nxt.tolist() == [1, -1] and prob[0] == 0.25 and st == 0


@pytest.mark.gpu
def test_verify_greedy_takes_the_first_maximum():
    lg = torch.zeros(3, 20000)
    lg[:, 5] = 3
    lg[:, 9000] = 3
    lg[2] = 0
    nxt, acc, prob, st = call([3], [0, 5, 9000], lg, "f32", None, [0.999, 0.999, 0], [0.99], 0.0)
    assert acc[0] == 1 and nxt.tolist() == [5, 5, -1]
    nxt, acc, prob, st = call([3], [0, 5, 5], lg, "f32", None, [0.999, 0.999, 0], [0.99], 0.0)
    assert acc[0] == 2 and nxt.tolist() == [5, 5, 0] and prob.tolist() == [1, 1, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_verify_nan_infinite_and_unknown_ids(temperature):
    counts = [2, 2, 2, 2, 1]
    lg = torch.randn(9, 300, generator=torch.Generator().manual_seed(4))
    lg[0] = -math.inf                      # nothing finite: no token
    lg[2, 7] = math.nan                    # counts as -inf
    lg[4, 11] = math.inf                   # takes all
    fed = np.array([0, 1, 0, 7, 0, 11, 0, 300, 0])
    u = np.full(9, 0.5, np.float32)
    want = reference(counts, fed, lg.numpy(), None, u, np.full(5, 0.4), temperature)
    nxt, acc, prob, st = call(counts, fed, lg, "f32", None, u, np.full(5, 0.4, np.float32), temperature)
    assert nxt[0] == -1 and acc[0] == 0 and acc[2] == 1 and acc[3] == 0
    assert np.array_equal(nxt, want[0]) and np.array_equal(acc, want[1]) and np.allclose(prob, want[2], rtol=2.0 ** -19)
    assert st == ERANGE
    _, _, _, st = call([2], [0, -5], lg[3:5], "f32", None, [0.5, 0.5], [0.4], temperature)
    assert st == EINVAL


@pytest.mark.gpu
@pytest.mark.parametrize("cu,good", [([0, 3, 2], [0]), ([-1, 3, 6], [1]), ([0, 3, 9], [0]), ([4, 2, 6], [1])])
def test_verify_flags_bad_offsets(cu, good):
    """Offsets that run backwards, start below 0 or end past the rows: flagged, the other sequences stand."""
    g = torch.Generator().manual_seed(2)
    gpu, vocab, rows = vc4b200.GPU(0), 500, 6
    lg = torch.randn(rows, vocab, generator=g).cuda()
    fed = lg.argmax(-1).roll(1).int()
    ints = torch.full((rows + 4,), -9, dtype=torch.int32, device="cuda")
    nxt, acc, status = ints[:rows], ints[rows: rows + 2], ints[rows + 2: rows + 3]
    status.zero_()
    u, offs = torch.full((rows + 2,), 0.5, device="cuda"), torch.tensor(cu, dtype=torch.int32, device="cuda")
    need = gpu.verify_bytes(2, rows, vocab)
    work = torch.zeros(max(16, need), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    gpu.verify_draft(2, rows, vocab, offs.data_ptr(), fed.data_ptr(), lg.data_ptr(), "f32", 0.0, u.data_ptr(),
                     u[rows:].data_ptr(), nxt.data_ptr(), acc.data_ptr(), 0, work.data_ptr(), need, status=status.data_ptr())
    gpu.sync()
    assert int(status) == EINVAL and int(ints[-1]) == -9
    for s in good:      # every draft is the first maximum of the row before it
        at = slice(cu[s], cu[s + 1])
        assert int(acc[s]) == cu[s + 1] - cu[s] - 1 and torch.equal(nxt[at].long(), lg[at].argmax(-1))


@pytest.mark.gpu
def test_verify_follows_the_target_distribution():
    """Whatever the draft model, the accepted or sampled id of a row has the
    target's distribution: frequencies over many random numbers."""
    n, vocab = 20000, 6
    p = np.array([0.4, 0.25, 0.15, 0.1, 0.06, 0.04])
    d = np.array([0.1, 0.5, 0.1, 0.1, 0.1, 0.1])
    rng = np.random.default_rng(8)
    x = rng.choice(vocab, n, p=d)
    fed = np.stack([np.zeros(n, int), x], 1).ravel()
    lg = torch.from_numpy(np.log(p)).float().repeat(2 * n, 1)
    nxt, acc, _, _ = call([2] * n, fed, lg, "f32", torch.from_numpy(d).float().repeat(n, 1), rng.random(2 * n), rng.random(n), 1.0)
    count = np.bincount(nxt[0::2], minlength=vocab)
    assert np.all(np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p)))          # five standard deviations
    share = np.minimum(p, d).sum()
    assert abs(acc.mean() - share) <= 5 * math.sqrt(share * (1 - share) / n)


# ---- the session's speculative step -----------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("key", ["tiny_q8", "tiny_moe_q4", "tiny_t3"])
@pytest.mark.parametrize("hd64", [False, True])
def test_step_draft_is_the_serial_steps(tiny_paths, tmp_path, key, hd64):
    """Greedy: drafts taken from the serial decode are accepted up to the planted
    wrong one, the tokens gained are the serial ones, and the cache rows of the
    decoded positions are the serial ones.  Sampled: the walk over the serial logits."""
    cfg = synth.TINY_CONFIGS[key]
    path = tiny_paths[key]
    if hd64:       # head size 64: the batched pass; 16 steps position by position
        shape = synth.Shape("tiny-hd64", 256, 1056, 2, 4, 2, 1600, 1e6, True)
        if key != "tiny_q8":
            pytest.skip("one model of this head size")
        path = str(tmp_path / "m.mmcf")
        with open(path, "wb") as f:
            f.write(mmcf_writer.pack(shape, synth.hf_tensors(shape, 3), "q8", 64))
    gpu = vc4b200.GPU(0)
    model = vc4b200.Model(gpu, path)
    kv = "q16" if cfg.kv_bits == 16 else "q8"
    a, b = (vc4b200.Session(model, slots=8, seq=48, kv=kv) for _ in range(2))
    rng = np.random.default_rng(3)
    prompt = [int(v) for v in rng.integers(0, model.info.vocab, 6)]
    for s in (a, b):
        s.prefill(prompt[:-1], 0, slot=1)
    toks, logits = [prompt[-1]], []
    for i in range(9):
        logits.append(a.step(toks[-1], 5 + i, slot=1))
        toks.append(int(np.argmax(logits[-1])))
    serial = [a.kv_rows(l, 9, slot=1) for l in range(model.info.layers)]
    # four right drafts, then a wrong one and another
    wrong = (toks[5] + 1) % model.info.vocab
    got, prob = b.step_draft([toks[0]] + toks[1:5] + [wrong, 0], 5, slot=1)
    assert got == toks[1:6] and prob.tolist() == [1.0] * 5
    assert [b.kv_rows(l, 9, slot=1) for l in range(model.info.layers)] == serial
    more, _ = b.step_draft([got[-1]], 10, slot=1)      # no drafts: a plain step
    assert more == [toks[6]]
    # sampled, with a draft distribution
    lg = np.stack(logits[6:9]).astype(np.float64)
    d = np.full((2, model.info.vocab), 1.0 / model.info.vocab, np.float32)
    u, us = np.array([0.3, 0.9], np.float32), 0.37
    want = reference([3], toks[6:9], lg, d, np.append(u, 0), [np.float32(us)], 0.9)
    assert want[3]
    got, prob = b.step_draft(toks[6:9], 11, d, 0.9, u, us, slot=1)
    assert got == want[0][: want[1][0] + 1].tolist()
    assert np.allclose(prob, want[2][: want[1][0] + 1], rtol=2.0 ** -19)


@pytest.mark.gpu
def test_step_draft_refuses(tiny_paths):
    model = vc4b200.Model(vc4b200.GPU(0), tiny_paths["tiny_q8"])
    s = vc4b200.Session(model, slots=3, seq=16)
    for call_, words in ((lambda: s.step_draft([], 0), "fed tokens"), (lambda: s.step_draft([1] * 4, 0), "fed tokens"),
                         (lambda: s.step_draft([1, 2, 3], 14), "sequence length"),
                         (lambda: s.step_draft([1, 1600], 0), "token id"), (lambda: s.step_draft([1], 0, slot=3), "slot"),
                         (lambda: s.step_draft([1], 0, temperature=-1.0), "temperature"),
                         (lambda: s.step_draft([1, 2], 0, temperature=1.0), "random number"),
                         (lambda: s.step_draft([1, 2], 0, np.zeros((2, 5)), u=[0.5]), "drafts x vocab")):
        with pytest.raises(vc4b200.EngineError, match=words):
            call_()
    assert s.step_draft([1], 0)[0] == [s.step_greedy(1, 0)]


# ---- together ---------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("key", ["tiny_q8", "tiny_flat_q8", "tiny_t3"])
def test_pages_hold_the_slot_caches_rows(tiny_paths, key):
    """A layer's projection appended to pages gives the slot cache's bytes, and
    attention over them the attention block's output to its own grid; with the
    second layer's on top, and the drafts judged on the logits, a whole step."""
    cfg = synth.TINY_CONFIGS[key]
    gpu = vc4b200.GPU(0)
    model = vc4b200.Model(gpu, tiny_paths[key])
    info = model.info
    fmt = "q16" if cfg.kv_bits == 16 else "q8"
    seq, n, heads, kv, dim = 32, 21, info.heads, info.kv_heads, info.head_dim
    s = vc4b200.Session(model, slots=2, seq=seq, kv=fmt)
    rng = np.random.default_rng(5)
    toks = [int(v) for v in rng.integers(0, info.vocab, n)]
    L = vc4b200.lib()
    width = info.dim + 2 * info.kv_dim
    qkv, att = np.empty((n, width), np.float32), np.empty((n, info.dim), np.float32)
    for i, t in enumerate(toks):
        assert L.vc4_embedding(s._h, 0, t, 0) == 0
        assert L.vc4_rmsnorm(s._h, 0, 0, 0, 0, 2) == 0
        assert L.vc4_matvec_from(s._h, 0, 0, 0, 0, 2, 1, qkv[i].ctypes.data) == 0
        assert L.vc4_attention_block(s._h, 0, 0, i, 2, 5) == 0
        assert L.vc4_read_buffer(s._h, 0, 5, info.dim, att[i].ctypes.data) == 0
    slot_rows = np.frombuffer(s.kv_rows(0, n), np.uint8).reshape(n, 2, kv, -1)
    cos, sin = (torch.from_numpy(x).cuda() for x in vc4b200.rope_tables(info.rope_theta, dim, seq))
    ones = torch.ones(dim, device="cuda")
    x = torch.from_numpy(qkv).cuda()
    norm = dict(q_norm=ones.data_ptr(), k_norm=ones.data_ptr(), eps=1e-6) if info.qk_norm else {}
    # two chunks of one sequence, as a prompt arrives
    cache = Cache([n], [n], fmt, 16, kv, dim)
    handle, _ = cache.handles(vc4b200, gpu)
    q = torch.empty(n, heads * dim, dtype=torch.float16, device="cuda")
    out = torch.empty(n, heads * dim, device="cuda")
    for lo, hi in ((0, 13), (13, n)):
        cu = torch.tensor([0, hi - lo], dtype=torch.int32, device="cuda")
        ln = torch.tensor([hi], dtype=torch.int32, device="cuda")
        batch = vc4b200.PagedBatch(cu.data_ptr(), ln.data_ptr(), cache.table.data_ptr(), 1, hi - lo, hi - lo, n, cache.width,
                                   status=cache.status.data_ptr())
        torch.cuda.synchronize()
        handle.append(batch, x[lo].data_ptr(), "f32", heads, q[lo].data_ptr(), "f16", cos=cos.data_ptr(), sin=sin.data_ptr(),
                      rope_len=seq, rope_half=bool(info.rope_half), **norm)
        assert handle.attend_bytes(batch, heads) == 0
        handle.attend(batch, q[lo].data_ptr(), "f16", heads, out[lo].data_ptr(), "f32")
        gpu.sync()
    assert int(cache.status) == 0
    rows = cache.pool[torch.from_numpy(cache.host_table[0].astype(np.int64)).cuda()].permute(0, 3, 1, 2, 4).contiguous()
    mine = rows.view(torch.uint8).cpu().numpy().reshape(-1, 2, kv, slot_rows.shape[-1])[:n]
    assert np.array_equal(mine, slot_rows)
    # the attention block's float q rounded to f16 (2^-11 of every product, twice in a weight) and its q16 output
    want, mass, top = attention(cache, q, heads)
    bound = attention_bound(fmt, "f32", want, mass, top, dim) + 2 * top * 2.0 ** -11 * mass * 1.01 + 0.5 / 256 + 1e-6
    ref = torch.from_numpy(att).cuda().double().view_as(want)
    assert bool(((out.double().view_as(want) - ref).abs() <= bound).all())
    assert bool(((out.double().view_as(want) - want).abs() <= attention_bound(fmt, "f32", want, mass, top, dim)).all())
    # the same step whole: the drafts of the last four positions judged on the engine's logits
    s.prefill(toks[:-4], 0, slot=1)
    lg = np.stack([s.step(t, n - 4 + i, slot=1) for i, t in enumerate(toks[-4:])])
    u = np.array([0.2, 0.4, 0.6, 0], np.float32)
    ints = torch.from_numpy(np.rint(lg * 256).astype(np.int32))
    want = reference([4], toks[-4:], lg, None, u, [0.5], 1.0)
    got = call([4], np.array(toks[-4:]), ints, "q16", None, u, np.array([0.5], np.float32), 1.0)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


# ---- ends of the ranges -----------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("kind,top", [("f32", -3.4e38), ("f32", 1e20), ("f32", -65504.0), ("f32", 3e38), ("bf16", None), ("f16", None)])
@pytest.mark.parametrize("temperature", [0.7, 1.0, 1e-5, 50.0])
def test_verify_rows_of_huge_finite_logits(kind, top, temperature):
    """A row's largest logit is weighed 1 wherever it lies: all ids masked with the
    type's lowest value are equally likely, and one that stands out takes all."""
    vocab, low = 1500, torch.finfo(TORCH[kind]).min
    lg = torch.full((4, vocab), low if top is None else top, dtype=TORCH[kind])     # rows 0, 1: equal
    lg[2:, :] = low
    lg[2:, 700] = low / 2 if top is None or top == -3.4e38 else top      # rows 2, 3: one stands out, by far
    counts, fed, u, us = [1, 1, 2], [0, 0, 0, 700], np.full(4, 0.999, np.float32), np.array([0.2501, 0.9, 0.5], np.float32)
    want = reference(counts, fed, lg.double().numpy(), None, u, us, temperature)
    assert want[3] and want[0].tolist() == [375, 1349, 700, 700]
    got = call(counts, fed, lg, kind, None, u, us, temperature)
    assert got[3] == 0 and np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    assert np.all(np.abs(got[2] - want[2]) <= 2.0 ** -19 * want[2])
    # what is left of p behind draft probabilities: the row's own p below them at one id
    d = torch.full((1, vocab), 1 / vocab)
    d[0, :vocab // 2] = 0
    want = reference([2], [0, 1000], lg[:2].double().numpy(), d.numpy(), [1.5, 0], us[:1], temperature)
    got = call([2], [0, 1000], lg[:2], kind, d, [1.5, 0], us[:1], temperature)
    assert want[3] and got[3] == 0 and np.array_equal(got[0], want[0]) and want[0][0] < vocab // 2


def _offsets(cu, rows, vocab, drafts, seed=2):
    """One greedy call over `rows` rows with offsets of any kind and `drafts` rows of draft
    probabilities: all 1 at the draft, so a draft is accepted where u < p.  Returns (logits,
    next, accepted, status)."""
    g = torch.Generator().manual_seed(seed)
    gpu, seqs = vc4b200.GPU(0), len(cu) - 1
    lg = torch.randn(rows, vocab, generator=g).cuda()
    fed = lg.argmax(-1).roll(1).int()
    nxt, acc = (torch.full((n,), -9, dtype=torch.int32, device="cuda") for n in (rows, seqs))
    status, offs = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor(cu, dtype=torch.int32, device="cuda")
    u, us = torch.full((rows,), 0.5, device="cuda"), torch.full((seqs,), 0.5, device="cuda")
    need = gpu.verify_bytes(seqs, rows, vocab)
    work = torch.zeros(max(16, need), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    gpu.verify_draft(seqs, rows, vocab, offs.data_ptr(), fed.data_ptr(), lg.data_ptr(), "f32", 0.0, u.data_ptr(), us.data_ptr(),
                     nxt.data_ptr(), acc.data_ptr(), 0, work.data_ptr(), need, probs=drafts.data_ptr(), status=status.data_ptr())
    gpu.sync()
    return lg, nxt, acc, int(status)


@pytest.mark.gpu
@pytest.mark.parametrize("first", [0, 1, 5])
def test_verify_draft_rows_count_from_the_first_offset(first):
    """A batch whose first sequence starts at row `first`: its draft probabilities are rows
    0, 1, .. of the array, which ends with the last draft."""
    vocab, counts = 300, [3, 0, 1, 4]
    cu = np.concatenate([[0], np.cumsum(counts)]) + first
    drafts = torch.zeros(5, vocab, device="cuda")
    drafts[[0, 2, 3]] = 1.0            # rows 1 and 4: d is 3, so u * d is above any p
    drafts[[1, 4]] = 3.0
    lg, nxt, acc, status = _offsets(cu.tolist(), first + 8, vocab, drafts)
    assert status == 0 and acc.tolist() == [1, 0, 0, 2]
    want = lg.argmax(-1).int()
    assert nxt[:first].tolist() == [-9] * first
    # (a refused row's p is one at its maximum, where d is above it: the rest falls back to p)
    for at, n, a in ((first, 3, 1), (first + 3, 1, 0), (first + 4, 4, 2)):
        assert torch.equal(nxt[at: at + a + 1], want[at: at + a + 1]) and bool((nxt[at + a + 1: at + n] == -1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cu,good,drafts", [([0, 3, 2], [0], 2), ([-1, 3, 6], [], 5), ([0, 3, 9], [0], 2), ([4, 2, 6], [], 3),
                                            ([0, 9, 3, 6], [], 5), ([0, 2, 1, 4, 6], [0], 4)])
def test_verify_skips_draft_rows_behind_bad_offsets(cu, good, drafts):
    """With draft probabilities: sequences behind offsets that start below 0 or run backwards,
    and one that ends past the rows, are flagged and skipped, those before them stand."""
    rows, vocab = 6, 300
    lg, nxt, acc, status = _offsets(cu, rows, vocab, torch.ones(drafts, vocab, device="cuda"))
    assert status == EINVAL
    touched = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for s in range(len(cu) - 1):
        at = slice(max(0, cu[s]), max(0, min(cu[s + 1], rows)))
        if s in good:       # every draft is the first maximum of the row before it
            assert int(acc[s]) == at.stop - at.start - 1 and torch.equal(nxt[at].long(), lg[at].argmax(-1))
            touched[at] = True
        else:
            assert int(acc[s]) == 0
    assert bool((nxt[~touched] == -9).all())


@pytest.mark.gpu
def test_verify_without_any_row_accepts_nothing():
    """No sequence has a row: the counts are 0 all the same, captured too."""
    gpu = vc4b200.GPU(0)
    ints = lambda n, v: torch.full((n,), v, dtype=torch.int32, device="cuda")  # noqa: E731
    cu, fed, nxt, acc, lg = ints(4, 0), ints(4, 0), ints(4, -9), ints(4, -9), torch.zeros(4, 100, device="cuda")
    u = torch.zeros(4, device="cuda")
    assert gpu.verify_bytes(3, 0, 100) == 0

    def step():
        gpu.verify_draft(3, 0, 100, cu.data_ptr(), fed.data_ptr(), lg.data_ptr(), "f32", 1.0, u.data_ptr(), u.data_ptr(),
                         nxt.data_ptr(), acc.data_ptr(), 0, 0, 0, stream=torch.cuda.current_stream().cuda_stream)
    step()
    torch.cuda.synchronize()
    assert acc.tolist() == [0, 0, 0, -9] and nxt.tolist() == [-9] * 4
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    acc.fill_(5)
    graph.replay()
    torch.cuda.synchronize()
    assert acc.tolist() == [0, 0, 0, 5]


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("x", [300, 2 ** 31 - 1, -1, -2 ** 31])
def test_verify_never_accepts_an_unknown_id(x, temperature):
    """An id outside the vocabulary is refused whatever u says, and not handed on."""
    lg = torch.randn(3, 300, generator=torch.Generator().manual_seed(4))
    nxt, acc, prob, st = call([3], [0, x, 1], lg, "f32", None, [-1.0, 0.5, 0], [0.4], temperature)
    want = reference([3], [0, x, 1], lg.numpy(), None, [1.0, 0.5, 0], [np.float32(0.4)], temperature)
    assert st == EINVAL and acc[0] == 0 and np.array_equal(nxt, want[0]) and 0 <= nxt[0] < 300


@pytest.mark.parametrize("name", ["cu", "fed", "probs", "u", "u_sample", "next_tokens", "accepted", "prob", "status"])
@pytest.mark.parametrize("off", [1, 2])
def test_verify_refuses_arrays_off_their_elements(name, off):
    a = dict(seqs=1, rows=3, vocab=100, cu=0x1000, fed=0x2000, logits=0x10000, logits_type="f32", temperature=1.0, u=0x4000,
             u_sample=0x5000, next_tokens=0x6000, accepted=0x7000, prob=0x8000, work=0x30000, work_bytes=1 << 20, probs=0x20000,
             status=0x9000)
    a[name] += off
    with pytest.raises(vc4b200.EngineError, match="error %d.*aligned" % EINVAL):
        _Host().verify_draft(**a)
