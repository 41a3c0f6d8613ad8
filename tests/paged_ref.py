"""The paged operators' definitions in 64 bits, and the buffers their tests use."""
import math

import numpy as np
import torch

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
POOL = {"q8": torch.int8, "q16": torch.int16, "bf16": torch.bfloat16, "f16": torch.float16}
GRID = {"q8": 16.0, "q16": 2048.0}


def half_step(kind: str) -> float:
    """The largest relative rounding error of an activation type."""
    return torch.finfo(TORCH[kind]).eps / 2


def swap16(t):
    """int16 levels to and from their big-endian bytes in memory."""
    return t.contiguous().view(torch.uint8).view(*t.shape, 2).flip(-1).contiguous().view(torch.int16).view(t.shape)


def decode(pool, fmt):
    """Cached values as doubles."""
    if fmt == "q8":
        return pool.double() / 16
    if fmt == "q16":
        return swap16(pool).double() / 2048
    return pool.double()


class Cache:
    """A pool with shuffled pages for sequences of the given total lengths, of
    which the last `new` are the batch's new tokens.  Rows no sequence uses
    (whole spare pages, the ends of last pages) hold `fill`."""

    def __init__(self, length, new, fmt, page, kv, dim, seed=0, spare=3, width=None, rows=None, fill=None, device="cuda"):
        self.length, self.new, self.fmt, self.page, self.kv, self.dim = list(length), list(new), fmt, page, kv, dim
        g = torch.Generator().manual_seed(seed)
        seqs = len(self.length)
        need = [(n + page - 1) // page for n in self.length]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=g)[: sum(need)].tolist()
        self.width = width or max(1, max(need))
        self.host_table = np.full((seqs, self.width), -7, np.int32)   # entries behind a sequence's pages are never read
        at = 0
        for s, n in enumerate(need):
            self.host_table[s, :n] = order[at: at + n]
            at += n
        shape = (self.pages, 2, kv, page, dim)
        x = torch.randn(shape, generator=g)
        if fmt == "q8":
            pool = (x * 16).round().clamp(-128, 127).to(torch.int8)
        elif fmt == "q16":
            pool = swap16((x * 2048).round().clamp(-32768, 32767).to(torch.int16))
        else:
            pool = x.to(POOL[fmt])
        if fill is not None:
            used = torch.zeros(self.pages, page, dtype=torch.bool)
            for s, n in enumerate(self.length):
                for t in range(n):
                    used[self.host_table[s, t // page], t % page] = True
            pool = pool.permute(0, 3, 1, 2, 4).contiguous()
            pool[~used] = fill
            pool = pool.permute(0, 2, 3, 1, 4).contiguous()
        self.pool = pool.to(device)
        self.host_cu = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.tokens = int(self.host_cu[-1])
        self.rows = rows or max(1, self.tokens)     # rows of the activations, some behind the last sequence
        self.cu = torch.from_numpy(self.host_cu).to(device)
        self.len = torch.tensor(self.length, dtype=torch.int32, device=device)
        self.table = torch.from_numpy(self.host_table).to(device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)

    def handles(self, lib, gpu, max_len=None, max_new=None):
        cache = lib.PagedKV(gpu, self.pool.data_ptr(), self.fmt, self.pages, self.page, self.kv, self.dim)
        batch = lib.PagedBatch(self.cu.data_ptr(), self.len.data_ptr(), self.table.data_ptr(), len(self.length), self.rows,
                               max_new or max(self.new + [1]), max_len or max(self.length + [1]), self.width,
                               status=self.status.data_ptr())
        return cache, batch

    def rows_of(self, s):
        """K and V of sequence s in order, as doubles: [2][kv][len][dim]."""
        n = self.length[s]
        ids = torch.from_numpy(self.host_table[s, : (n + self.page - 1) // self.page]).long().to(self.pool.device)
        x = decode(self.pool[ids], self.fmt).permute(1, 2, 0, 3, 4)
        return x.reshape(2, self.kv, -1, self.dim)[:, :, :n]


def attention(cache, q, heads, scale=None, hidden=()):
    """(out, sum p |v|, the largest sum |q k| * scale) per row, in doubles.
    hidden: positions of sequence 0 that nobody sees."""
    kv, dim = cache.kv, cache.dim
    group, scale = heads // kv, scale or 1 / math.sqrt(dim)
    out = torch.zeros(cache.tokens, heads, dim, dtype=torch.float64, device=q.device)
    mass, top = torch.zeros_like(out), torch.zeros(cache.tokens, heads, 1, dtype=torch.float64, device=q.device)
    x = q[: cache.tokens].double().view(-1, heads, dim)
    for s in range(len(cache.length)):
        a, n, new = int(cache.host_cu[s]), cache.length[s], cache.new[s]
        if not new or not n:
            continue
        k, v = cache.rows_of(s)
        k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
        y = x[a: a + new].transpose(0, 1)
        score = y @ k.transpose(1, 2) * scale
        hide = torch.arange(n, device=q.device)[None] > torch.arange(n - new, n, device=q.device)[:, None]
        if s == 0 and len(hidden):
            hide[:, list(hidden)] = True
        p = score.masked_fill(hide, -math.inf).softmax(-1)
        p = torch.nan_to_num(p, nan=0.0) if bool(hide.all(-1).any()) else p
        out[a: a + new] = (p @ v).transpose(0, 1)
        mass[a: a + new] = (p @ v.abs()).transpose(0, 1)
        top[a: a + new, :, 0] = ((y.abs() @ k.abs().transpose(1, 2)) * scale).masked_fill(hide, 0).amax(-1).transpose(0, 1)
    return out, mass, top


def attention_bound(fmt, out_kind, out, mass, top, dim):
    """How far a row may be from `out`.  A weight p is off by half a step of the
    operand type (its rounding) and by a score's error twice (its own and the
    sum's): dim products added in float, 2^-24 each of sum |q k|, for q16 the f16
    rounding of a level (2^-12) as well, and 2^-20 for the exponential and the
    float sums; a q16 value of V is rounded by 2^-12 too.  A weight below f16's
    normal range is off by half of its last step instead: the weights are held
    times 2^15, so by 2^-40 of the largest weight, which is at most the sum; the
    positions (at most 2^14 here) times |v| (below 16) of those.  Then the
    output's own half step."""
    operand = torch.finfo(torch.bfloat16 if fmt == "bf16" else torch.float16).eps / 2
    level = 2.0 ** -12 if fmt == "q16" else 0.0
    rel = operand + level + 2 * top * (dim * 2.0 ** -24 + level) + 2.0 ** -20
    small = 1e-12 if fmt == "bf16" else 2.0 ** (14 + 4 - 40)
    least = torch.finfo(TORCH[out_kind]).smallest_normal * torch.finfo(TORCH[out_kind]).eps
    return rel * mass * 1.01 + half_step(out_kind) * out.abs() * 1.01 + least + small
