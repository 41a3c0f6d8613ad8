"""The operators of a paged speculative decoding step, as cases: appending a
projection's rows to a paged KV cache (QK-norm and RoPE on the way), attention
of some new tokens over the pages, and the verification of drafted tokens.

`own` False computes each in elementary torch operations; True makes the calls
a user makes of vc4b200.
"""
import functools
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_FLOAT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_POOL = {"q8": torch.int8, "q16": torch.int16, "bf16": torch.bfloat16, "f16": torch.float16}
_GRID = {"q8": 16.0, "q16": 2048.0}


# ---- cases -----------------------------------------------------------------------

def _append(name, seqs, new, past, heads, kv, dim, kind, fmt, page, norm, half):
    return {"name": name, "op": "append", "seqs": seqs, "new": new, "past": past, "heads": heads, "kv": kv,
            "dim": dim, "in": kind, "fmt": fmt, "page": page, "norm": norm, "half": half}


def _attend(name, seqs, new, length, heads, kv, dim, kind, fmt, page):
    return {"name": name, "op": "attend", "seqs": seqs, "new": new, "len": length, "heads": heads, "kv": kv,
            "dim": dim, "in": kind, "fmt": fmt, "page": page}


def _verify(name, seqs, drafts, vocab, kind, probs, temperature):
    return {"name": name, "op": "verify", "seqs": seqs, "drafts": drafts, "vocab": vocab, "in": kind,
            "probs": probs, "temperature": temperature}


def listed():
    return [
        # one decode step of 64 MiniMind3 sequences: where the call itself counts
        _append("append decode 64 q8", 64, 1, 700, 8, 4, 96, "f32", "q8", 16, True, True),
        # ragged prompts of a ternary decoder without QK-norm, neighbouring pairs rotated
        _append("append ragged 5.9k q16", 23, 257, 0, 16, 2, 64, "bf16", "q16", 32, False, False),
        # a long prompt chunk in a wide decoder
        _append("append chunk 16k bf16", 4, 4096, 4096, 32, 8, 128, "bf16", "bf16", 64, True, True),
        # one user's next token: latency
        _attend("attend one 777 q16", 1, 1, 777, 8, 4, 96, "bf16", "q16", 16),
        # the many-sequence decode of the benchmark: 1024 sequences of up to 768 positions
        _attend("attend decode 1024 q8", 1024, 1, 768, 8, 4, 96, "bf16", "q8", 32),
        # few long conversations: the work is split over the positions
        _attend("attend long 12x40k bf16", 12, 1, 40000, 32, 8, 128, "bf16", "bf16", 64),
        # five fed tokens (four drafts) of 61 sequences, the target's verification pass
        _attend("attend drafts 61x5 f16", 61, 5, 2000, 16, 2, 64, "f16", "f16", 16),
        # prompt chunks of several sequences over a quantised cache
        _attend("attend chunk 6x700 q8", 6, 700, 5000, 8, 4, 96, "bf16", "q8", 16),
        # a long prompt's chunk: bound by the products
        _attend("attend chunk 4k of 16k bf16", 1, 4096, 16384, 32, 8, 128, "bf16", "bf16", 128),
        # one user's four drafts on the small vocabulary: latency
        _verify("verify 1x4 v6400", 1, 4, 6400, "f32", True, 1.0),
        # a batch of users on the large vocabulary, prompt-lookup drafts (no probabilities)
        _verify("verify 61x5 v73448 bf16", 61, 5, 73448, "bf16", False, 0.7),
        # a full server
        _verify("verify 256x7 v73448", 256, 7, 73448, "f32", True, 0.9),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "attend", "verify"])
    heads, kv = rng.choice([(8, 4), (16, 2), (32, 8), (7, 1), (12, 12), (28, 4), (64, 8)])
    dim = rng.choice([64, 96, 128, 128, 80, 32])
    page = rng.choice([16, 32, 64, 128])
    fmt = rng.choice(["q8", "q16", "bf16", "f16"])
    kind = fmt if fmt in ("bf16", "f16") else rng.choice(["bf16", "f16"])
    if op == "append":
        tokens = _log(rng, 1, 16384 * 48 // (heads + 2 * kv))
        seqs = min(tokens, _log(rng, 1, 300))
        return {"op": op, "seqs": seqs, "new": max(1, tokens // seqs), "past": _log(rng, 1, 4000), "heads": heads,
                "kv": kv, "dim": dim, "in": rng.choice(["f32", "bf16", "f16"]), "fmt": fmt, "page": page,
                "norm": rng.random() < 0.6, "half": rng.random() < 0.6}
    if op == "attend":
        new = 1 if rng.random() < 0.4 else rng.randint(2, 16) if rng.random() < 0.4 else _log(rng, 17, 2000)
        length = new + _log(rng, 1, 16000)
        length = max(new, min(length, int(1.6e9 / (new * heads))))
        most = min(8e6 / (length * kv), 1.6e9 / (new * length * heads))  # cached rows, scores
        return {"op": op, "seqs": _log(rng, 1, max(1, min(500, most))), "new": new, "len": length, "heads": heads,
                "kv": kv, "dim": dim, "in": kind, "fmt": fmt, "page": page}
    vocab = _log(rng, 500, 160000)
    seqs = _log(rng, 1, max(1, min(256, 150e6 / (8 * vocab))))
    return {"op": op, "seqs": seqs, "drafts": rng.randint(0, 7), "vocab": vocab,
            "in": rng.choice(["f32", "bf16", "f16"]), "probs": rng.random() < 0.6,
            "temperature": rng.choice([0.0, 0.6, 0.8, 1.0, 1.3])}


# ---- inputs ----------------------------------------------------------------------

def _lengths(case):
    """New tokens and total length of each sequence: the largest as the case
    says, the others spread below it (at least one new token each).  They are
    the case's own, so that outputs of two seeds have one shape."""
    g = torch.Generator().manual_seed(case["seqs"])
    seqs = case["seqs"]
    new = torch.full((seqs,), case["new"], dtype=torch.int64)
    if case["op"] == "append":
        past = torch.randint(0, case["past"] + 1, (seqs,), generator=g)
        past[0] = case["past"]
    else:
        past = torch.randint((case["len"] - case["new"]) // 2, case["len"] - case["new"] + 1, (seqs,), generator=g)
        past[0] = case["len"] - case["new"]
    if seqs > 1 and case["new"] > 8:  # ragged chunks
        new[1:] = torch.randint(max(1, case["new"] // 2), case["new"] + 1, (seqs - 1,), generator=g)
    return new, past + new


def _cache(case, seed):
    """A pool of pages, the page table in a shuffled order, and the batch's offsets."""
    g = torch.Generator().manual_seed(seed)
    d = torch.Generator(device="cuda").manual_seed(seed)
    new, length = _lengths(case)
    page, seqs = case["page"], case["seqs"]
    need = (length + page - 1) // page
    pages, width = int(need.sum()) + 3, int(need.max())
    order = torch.randperm(pages, generator=g)[: int(need.sum())].to(torch.int32)
    table = torch.zeros(seqs, width, dtype=torch.int32)
    live = torch.arange(width)[None] < need[:, None]
    table[live] = order
    shape = (pages, 2, case["kv"], page, case["dim"])
    dt = _POOL[case["fmt"]]
    if case["op"] == "append":  # what was there: an empty pool, but for a pattern that shows stray writes
        pool = torch.ones(shape, dtype=dt, device="cuda")
    elif dt == torch.int8:
        pool = torch.randn(shape, device="cuda", generator=d).mul_(16).round_().clamp_(-128, 127).to(dt)
    elif dt == torch.int16:
        pool = torch.randn(shape, device="cuda", generator=d).mul_(2048).round_().clamp_(-32768, 32767).to(dt)
        pool = pool.view(torch.uint8).view(*shape, 2).flip(-1).contiguous().view(dt).view(shape)
    else:
        pool = torch.randn(shape, device="cuda", generator=d).to(dt)
    cu = torch.zeros(seqs + 1, dtype=torch.int32)
    cu[1:] = new.cumsum(0)
    return {"pool": pool, "table": table.cuda(), "cu": cu.cuda(), "len": length.to(torch.int32).cuda(),
            "tokens": int(cu[-1]), "max_new": int(new.max()), "max_len": int(length.max()),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda")}, d


def prepare(case, seed):
    op, heads = case["op"], case.get("heads")
    if op == "verify":
        return _prepare_verify(case, seed)
    st, d = _cache(case, seed)
    st["case"] = case
    kv, dim, tokens = case["kv"], case["dim"], st["tokens"]
    if op == "append":
        kind = _FLOAT[case["in"]]
        st["qkv"] = torch.randn(tokens, (heads + 2 * kv) * dim, device="cuda", generator=d).to(kind)
        st["q"] = torch.empty(tokens, heads * dim, device="cuda", dtype=_FLOAT[_q_type(case)])
        st["q_norm"] = 1 + 0.2 * torch.randn(dim, device="cuda", generator=d)
        st["k_norm"] = 1 + 0.2 * torch.randn(dim, device="cuda", generator=d)
        freq = 1e6 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
        angle = torch.arange(st["max_len"], device="cuda", dtype=torch.float64)[:, None] * freq
        st["cos"], st["sin"] = angle.cos().float(), angle.sin().float()
    else:
        kind = _FLOAT[case["in"]]
        st["q"] = (1.5 * torch.randn(tokens, heads * dim, device="cuda", generator=d)).to(kind)
        st["out"] = torch.empty_like(st["q"])
    return st


def _q_type(case):
    return case["fmt"] if case["fmt"] in ("bf16", "f16") else "bf16"


def _prepare_verify(case, seed):
    """Logits of a trained model's spread, a draft model near the target's
    distribution, drafts sampled from it."""
    d = torch.Generator(device="cuda").manual_seed(seed)
    seqs, k, vocab = case["seqs"], case["drafts"], case["vocab"]
    rows = seqs * (k + 1)
    target = torch.randn(rows, vocab, device="cuda", generator=d).mul_(2.5)
    top = torch.randint(0, vocab, (rows, 8), device="cuda", generator=d)
    target.scatter_add_(1, top, 9 + 2 * torch.randn(rows, 8, device="cuda", generator=d))
    st = {"case": case, "rows": rows}
    near = target.view(seqs, k + 1, vocab)[:, :k].reshape(seqs * k, vocab)
    probs = torch.empty_like(near).normal_(generator=d).mul_(0.5).add_(near).softmax(-1)
    fed = torch.randint(0, vocab, (seqs, k + 1), device="cuda", generator=d)
    if k:
        # drafts drawn from the draft model: a position of its cumulative sums
        at = torch.rand(seqs * k, 1, device="cuda", generator=d)
        cdf = probs.cumsum(-1)
        fed[:, 1:] = torch.searchsorted(cdf, at * cdf[:, -1:]).clamp_(max=vocab - 1).view(seqs, k)
        del cdf
    st["logits"] = target.to(_FLOAT[case["in"]])
    st["probs"] = probs if case["probs"] else None
    st["fed"] = fed.reshape(rows).to(torch.int32)
    st["cu"] = torch.arange(0, rows + 1, k + 1, dtype=torch.int32, device="cuda")
    st["u"] = torch.rand(rows, device="cuda", generator=d)
    st["u_sample"] = torch.rand(seqs, device="cuda", generator=d)
    st["tokens"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    st["accepted"] = torch.empty(seqs, dtype=torch.int32, device="cuda")
    st["prob"] = torch.empty(rows, device="cuda")
    st["status"] = torch.zeros(1, dtype=torch.int32, device="cuda")
    return st


# ---- one pass --------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "verify": _own_verify}[op](state)
    return {"append": _plain_append, "attend": _plain_attend, "verify": _plain_verify}[op](state)


@functools.lru_cache(maxsize=None)
def _library():
    sys.path.insert(0, os.path.join(_ROOT, "vc4-gles2-inference_b200"))
    import vc4b200
    return vc4b200, vc4b200.GPU(torch.cuda.current_device())


def _paged(st):
    """The pool and batch descriptions, kept with the state as a server keeps them."""
    if "paged" not in st:
        lib, gpu = _library()
        case, pool = st["case"], st["pool"]
        st["paged"] = (lib.PagedKV(gpu, pool.data_ptr(), case["fmt"], pool.shape[0], case["page"], case["kv"], case["dim"]),
                       lib.PagedBatch(st["cu"].data_ptr(), st["len"].data_ptr(), st["table"].data_ptr(), case["seqs"],
                                      st["tokens"], st["max_new"], st["max_len"], st["table"].shape[1],
                                      status=st["status"].data_ptr()))
    return st["paged"]


def _own_append(st):
    case = st["case"]
    cache, batch = _paged(st)
    norm = case["norm"]
    cache.append(batch, st["qkv"].data_ptr(), case["in"], case["heads"], st["q"].data_ptr(), _q_type(case),
                 q_norm=st["q_norm"].data_ptr() if norm else 0, k_norm=st["k_norm"].data_ptr() if norm else 0, eps=1e-6,
                 cos=st["cos"].data_ptr(), sin=st["sin"].data_ptr(), rope_len=st["max_len"], rope_half=case["half"],
                 stream=torch.cuda.current_stream().cuda_stream)
    return {"q": st["q"], "pool": st["pool"]}


def _own_attend(st):
    case = st["case"]
    cache, batch = _paged(st)
    if "work" not in st:
        st["work"] = torch.empty(max(1, cache.attend_bytes(batch, case["heads"])), dtype=torch.uint8, device="cuda")
    cache.attend(batch, st["q"].data_ptr(), case["in"], case["heads"], st["out"].data_ptr(), case["in"],
                 st["work"].data_ptr(), st["work"].numel(), stream=torch.cuda.current_stream().cuda_stream)
    return st["out"]


def _own_verify(st):
    case = st["case"]
    lib, gpu = _library()
    if "work" not in st:
        st["work"] = torch.empty(max(1, gpu.verify_bytes(case["seqs"], st["rows"], case["vocab"])), dtype=torch.uint8,
                                 device="cuda")
    gpu.verify_draft(case["seqs"], st["rows"], case["vocab"], st["cu"].data_ptr(), st["fed"].data_ptr(),
                     st["logits"].data_ptr(), case["in"], case["temperature"], st["u"].data_ptr(),
                     st["u_sample"].data_ptr(), st["tokens"].data_ptr(), st["accepted"].data_ptr(),
                     st["prob"].data_ptr(), st["work"].data_ptr(), st["work"].numel(),
                     probs=0 if st["probs"] is None else st["probs"].data_ptr(), status=st["status"].data_ptr(),
                     stream=torch.cuda.current_stream().cuda_stream)
    return {"tokens": st["tokens"], "accepted": st["accepted"], "prob": st["prob"]}


# ---- plain forms -----------------------------------------------------------------

def _places(st):
    """Sequence, position and (page, offset) of every new token."""
    case, cu = st["case"], st["cu"].long()
    n = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), n, output_size=st["tokens"])
    nth = torch.arange(st["tokens"], device="cuda") - cu[seq]
    pos = st["len"].long()[seq] - n[seq] + nth
    return seq, nth, pos, st["table"].long()[seq, pos // case["page"]], pos % case["page"]


def _rotate(x, c, s, half):
    if half:
        a, b = x[..., : x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
        return torch.cat([a * c - b * s, a * s + b * c], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)


def _encode(x, fmt):
    if fmt == "q8":
        return (x * 16 + 0.5).floor().clamp(-128, 127).to(torch.int8)
    if fmt == "q16":
        level = (x * 2048 + 0.5).floor().clamp(-32768, 32767).to(torch.int16)
        return level.view(torch.uint8).view(*x.shape, 2).flip(-1).contiguous().view(torch.int16).view(x.shape)
    return x.to(_POOL[fmt])


def _decode(pool, fmt):
    if fmt == "q8":
        return pool.float() / 16
    if fmt == "q16":
        pair = pool.contiguous().view(torch.uint8).view(*pool.shape, 2)
        return (pair[..., 0].view(torch.int8).float() * 256 + pair[..., 1].float()) / 2048
    return pool.float()


def _plain_append(st):
    case = st["case"]
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    _, _, pos, page, off = _places(st)
    x = st["qkv"].float().view(-1, heads + 2 * kv, dim)
    qk, v = x[:, : heads + kv], x[:, heads + kv:]
    if case["norm"]:
        # the sum of squares in 64 bits: a level next to a border goes by its last bit
        mean = qk.double().square().sum(-1, keepdim=True).float() / torch.full((), float(dim), device="cuda")
        weight = torch.cat([st["q_norm"].expand(heads, dim), st["k_norm"].expand(kv, dim)])
        qk = weight * (1 / (mean + 1e-6).sqrt() * qk)
    qk = _rotate(qk, st["cos"][pos][:, None], st["sin"][pos][:, None], case["half"])
    st["q"].copy_(qk[:, :heads].reshape(-1, heads * dim))
    st["pool"][page, 0, :, off] = _encode(qk[:, heads:], case["fmt"])
    st["pool"][page, 1, :, off] = _encode(v, case["fmt"])
    return {"q": st["q"], "pool": st["pool"]}


def _plain_attend(st):
    case = st["case"]
    seqs, heads, kv, dim, group = case["seqs"], case["heads"], case["kv"], case["dim"], case["heads"] // case["kv"]
    seq, nth, pos, _, _ = _places(st)
    rows = _decode(st["pool"][st["table"].long()], case["fmt"])  # seqs, pages, 2, kv, page, dim
    k, v = rows.permute(2, 0, 3, 1, 4, 5).reshape(2, seqs, kv, -1, dim)
    q = torch.zeros(seqs, st["max_new"], heads, dim, device="cuda")
    q[seq, nth] = st["q"].float().view(-1, heads, dim)
    last = torch.zeros(seqs, st["max_new"], dtype=torch.int64, device="cuda")
    last[seq, nth] = pos
    q = q.view(seqs, st["max_new"], kv, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, dim)
    score = q @ k.transpose(-1, -2)
    score = score.mul_(1 / math.sqrt(dim)).view(seqs, kv, group, st["max_new"], -1)
    seen = torch.arange(k.shape[2], device="cuda") <= last[:, None, None, :, None]
    score = score.masked_fill_(~seen, -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = score.view(seqs, kv, group * st["max_new"], -1) @ v
    out = out.view(seqs, kv, group, st["max_new"], dim) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, st["max_new"], heads * dim)
    st["out"].copy_(out[seq, nth])
    return st["out"]


def _plain_verify(st):
    case = st["case"]
    seqs, vocab, rows, t = case["seqs"], case["vocab"], st["rows"], case["temperature"]
    cu = st["cu"].long()
    n = cu[1:] - cu[:-1]
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), n, output_size=rows)
    row = torch.arange(rows, device="cuda")
    judged = row + 1 < cu[1:][seq]  # the last row of a sequence judges no draft
    draft = st["fed"].long()[(row + 1).clamp(max=rows - 1)]
    x = st["logits"].float()
    top, first = x.max(-1)
    if t > 0:
        e = ((x - top[:, None]) / t).exp_()
        total = e.sum(-1)
        p = e.gather(1, draft[:, None])[:, 0] / total
    else:
        first = (x == top[:, None]).to(torch.uint8).argmax(-1)  # the lowest index of the maximum
        p = (first == draft).float()
    at = (row - seq).clamp(max=max(0, rows - seqs - 1))  # this row's draft probabilities
    ratio = st["u"] if st["probs"] is None or rows == seqs else st["u"] * st["probs"][at, draft]
    stop = torch.where(judged & (ratio < p), rows, row)
    stop = torch.full((seqs,), rows, device="cuda").scatter_reduce(0, seq, stop, "amin")
    # the row that is sampled from, in 64 bits: its cumulative sums decide between neighbours
    l = st["logits"][stop].double()
    if t > 0:
        w = ((l - l.amax(-1, keepdim=True)) / t).exp_()
        w = w / w.sum(-1, keepdim=True)
    else:
        w = torch.zeros_like(l).scatter_(1, first[stop][:, None], 1.0)
    refused = judged[stop]
    if st["probs"] is not None and rows > seqs:
        minus = st["probs"][at[stop]].double() * refused[:, None]
    else:
        minus = torch.zeros_like(w).scatter_(1, draft[stop][:, None], refused.double()[:, None])
    rest = (w - minus).clamp_(min=0)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    cdf = rest.cumsum(-1)
    goal = st["u_sample"].double()[:, None] * cdf[:, -1:]
    token = (cdf > goal).to(torch.uint8).argmax(-1)
    last = stop[seq]
    st["tokens"].copy_(torch.where(row < last, draft, torch.where(row == last, token[seq], -1)))
    own_p = w.gather(1, token[:, None])[:, 0].float()
    st["prob"].copy_(torch.where(row < last, p, torch.where(row == last, own_p[seq], 0.0)))
    st["accepted"].copy_(stop - cu[:-1])
    return {"tokens": st["tokens"], "accepted": st["accepted"], "prob": st["prob"]}


# ---- what a pass needs -----------------------------------------------------------

def work(case):
    size = {"q8": 1, "q16": 2, "bf16": 2, "f16": 2, "f32": 4}
    if case["op"] == "verify":
        rows = case["seqs"] * (case["drafts"] + 1)
        read = rows * case["vocab"] * size[case["in"]]
        if case["probs"] and case["drafts"]:
            read += case["seqs"] * case["vocab"] * 4  # one refused row of each
        return {"bytes": read + rows * 16, "flops": 4 * rows * case["vocab"]}
    new, length = _lengths(case)
    tokens, heads, kv, dim = int(new.sum()), case["heads"], case["kv"], case["dim"]
    if case["op"] == "append":
        each = (heads + 2 * kv) * dim * size[case["in"]] + heads * dim * 2 + 2 * kv * dim * size[case["fmt"]] + 8 * dim // 2
        return {"bytes": tokens * each, "flops": 6 * tokens * (heads + kv) * dim}
    seen = int((new * (length - new) + new * (new + 1) // 2).sum())
    return {"bytes": int(length.sum()) * 2 * kv * dim * size[case["fmt"]] + 4 * tokens * heads * dim,
            "flops": 4 * seen * heads * dim}


# ---- the definitions in 64 bits ----------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "verify": _exact_verify}[case["op"]](st)


def _exact_append(st):
    case = st["case"]
    heads, kv, dim, page, half = case["heads"], case["kv"], case["dim"], case["page"], case["half"]
    x = st["qkv"].double().view(-1, heads + 2 * kv, dim)
    cu, length = st["cu"].tolist(), st["len"].tolist()
    place = torch.cat([torch.arange(e - (b - a), e, device="cuda") for a, b, e in zip(cu, cu[1:], length)])
    if case["norm"]:
        size = (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
        x = torch.cat([x[:, :heads] / size[:, :heads] * st["q_norm"].double(),
                       x[:, heads: heads + kv] / size[:, heads: heads + kv] * st["k_norm"].double(), x[:, heads + kv:]], 1)
    turn = torch.complex(st["cos"].double(), st["sin"].double())[place][:, None]
    y = x[:, : heads + kv]
    z = torch.complex(y[..., : dim // 2], y[..., dim // 2:]) if half else torch.view_as_complex(y.reshape(*y.shape[:-1], -1, 2))
    z = z * turn
    y = torch.cat([z.real, z.imag], -1) if half else torch.view_as_real(z).flatten(-2)
    if case["fmt"] in _GRID:  # whole levels have no value in 64 bits that they are near to
        return {"q": y[:, :heads].reshape(-1, heads * dim), "pool": None}
    pool = st["pool"].double()
    for s in range(case["seqs"]):
        at = place[cu[s]: cu[s + 1]]
        ids = st["table"][s][at // page].long()
        pool[ids, 0, :, at % page] = y[cu[s]: cu[s + 1], heads:]
        pool[ids, 1, :, at % page] = x[cu[s]: cu[s + 1], heads + kv:]
    return {"q": y[:, :heads].reshape(-1, heads * dim), "pool": pool}


def _exact_attend(st):
    case = st["case"]
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    out = torch.empty(st["tokens"], heads, dim, dtype=torch.float64, device="cuda")
    q = st["q"].double().view(-1, heads, dim)
    cu, length = st["cu"].tolist(), st["len"].tolist()
    for s in range(case["seqs"]):
        a, b, n = cu[s], cu[s + 1], length[s]
        rows = _decode(st["pool"][st["table"][s, : -(-n // page)].long()], case["fmt"]).double()
        hide = torch.ones(b - a, n, dtype=torch.bool, device="cuda").triu(n - (b - a) + 1)
        for h in range(kv):
            k, v = (rows[:, i, h].reshape(-1, dim)[:n] for i in (0, 1))
            mine = slice(h * heads // kv, (h + 1) * heads // kv)
            p = torch.einsum("tgd,nd->gtn", q[a:b, mine], k) / dim ** 0.5
            p = p.masked_fill_(hide, -math.inf).softmax(-1)
            out[a:b, mine] = torch.einsum("gtn,nd->tgd", p, v)
    return out.view(-1, heads * dim)


def _exact_verify(st):
    """The probabilities; the whole numbers have to be equal anyway."""
    case = st["case"]
    k, t = case["drafts"], case["temperature"]
    prob = torch.zeros(st["rows"], dtype=torch.float64, device="cuda")
    for s in range(case["seqs"]):
        base = s * (k + 1)
        l = st["logits"][base: base + k + 1].double()
        if t:
            p = (l / t).softmax(-1)
        else:
            p = (l.argmax(-1, keepdim=True) == torch.arange(case["vocab"], device="cuda")).double()
        fed, u = st["fed"][base: base + k + 1].tolist(), st["u"][base: base + k + 1].double().tolist()
        i = 0
        while i < k:
            px = float(p[i, fed[i + 1]])
            qx = 1.0 if st["probs"] is None else float(st["probs"][s * k + i, fed[i + 1]])
            if not u[i] * qx < px:
                break
            prob[base + i] = px
            i += 1
        r = p[i].clone()
        if i < k:
            if st["probs"] is None:
                r[fed[i + 1]] = 0
            else:
                r = (r - st["probs"][s * k + i].double()).clamp(min=0)
            r = r if float(r.sum()) > 0 else p[i]
        c = r.cumsum(0)
        x = int((c <= float(st["u_sample"][s]) * c[-1]).sum())
        prob[base + i] = p[i, min(x, case["vocab"] - 1)]
    return {"tokens": None, "accepted": None, "prob": prob}
