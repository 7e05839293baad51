"""The operators of the paged key/value cache from their definitions, in 64 bits, and how far a result in fewer may be from them.

A case is laid out here as a test needs it: sequences of given lengths on pages scattered over a pool, tables on the GPU."""
import math

import torch

ROWS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CACHE = {"f32": torch.float16, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}      # finfo.eps / 2: the most that one rounding is off by
# what is lost of a query or a probability on its way to the tensor cores: one rounding, or with f32 rows that of a (hi, lo) pair
PAIR = {"f32": 2.0 ** -22, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -25, "f16": 2.0 ** -25, "bf16": 0.0}                 # half a step of the smallest f16 numbers


class Layout:
    """rows new rows and lens keys per sequence (rows None: one row each); n_rows rows in the buffers."""

    def __init__(self, lens, page, rows=None, extra_rows=0, extra_pages=2, seed=0, drop=None, max_pages=None):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.step = list(lens), page, rows is None
        self.rows = [1] * len(self.lens) if rows is None else list(rows)
        self.begin = [sum(self.rows[:s]) for s in range(len(self.rows))]
        self.real = sum(self.rows)
        self.n_rows = self.real + extra_rows
        width = max_pages or max(1, max((n + page - 1) // page for n in self.lens))
        self.table = torch.full((len(self.lens), width), -1, dtype=torch.int32)
        need = [(s, p) for s, n in enumerate(self.lens) for p in range((n + page - 1) // page) if not (drop and drop(s, p))]
        self.n_pages = len(need) + extra_pages
        order = torch.randperm(self.n_pages, generator=g)[:len(need)]
        for (s, p), at in zip(need, order.tolist()):
            self.table[s, p] = at
        self.table_dev = self.table.cuda()
        self.len_dev = torch.tensor(self.lens, dtype=torch.int32).cuda()
        self.off_dev = None if self.step else torch.tensor([0] + self.rows).cumsum(0).to(torch.int32).cuda()

    def batch(self, cache):
        return cache.batch(self.len_dev, self.table_dev, row_off=self.off_dev, n_rows=self.n_rows)


def pools(cache, fmt):
    """The cache's own pools as tensors."""
    return [torch.as_tensor(p, device="cuda").view(CACHE[fmt]) for p in cache.pages()]


def keys_of(pool, lay, s, positions):
    """Rows [positions, kv heads, dim] of a sequence, in 64 bits."""
    at = torch.tensor(positions, dtype=torch.long)
    return pool[lay.table[s].long()[at // lay.page].cuda(), :, (at % lay.page).cuda()].double()


def visible(pos, window, sinks):
    return [j for j in range(pos + 1) if not window or j > pos - window or j < sinks]


def attend(lay, q, k_pool, v_pool, kv_heads, window=0, sinks=0, scale=0.0, fmt="bf16"):
    """Result and bound for every row that belongs to a sequence: [rows, heads * dim] each."""
    d = k_pool.shape[-1]
    scale = scale or 1 / math.sqrt(d)
    out, bound = torch.zeros(lay.real, q.shape[1], dtype=torch.float64, device="cuda"), torch.zeros(lay.real, q.shape[1], dtype=torch.float64, device="cuda")
    h = q.shape[1] // d
    for s, (n, length) in enumerate(zip(lay.rows, lay.lens)):
        if n == 0 or length <= 0:
            continue
        seen = sorted(set().union(*(visible(p, window, sinks) for p in ({length - n, length - 1} if not window else range(length - n, length)) if p >= 0)))
        if not seen:
            continue
        k, v = keys_of(k_pool, lay, s, seen), keys_of(v_pool, lay, s, seen)
        j = torch.tensor(seen, device="cuda")
        p = torch.arange(length - n, length, device="cuda")[:, None]
        mask = (j <= p) & ((j > p - window) | (j < sinks) if window else True)
        mask &= p >= 0
        part = slice(lay.begin[s], lay.begin[s] + n)
        x = q[part].double().reshape(n, h, d).transpose(0, 1)
        kk, vv = (t.transpose(0, 1).repeat_interleave(h // kv_heads, 0) for t in (k, v))
        score = (scale * (x @ kk.transpose(1, 2))).masked_fill(~mask, -math.inf)
        top = score.amax(-1, keepdim=True).clamp_min(-1e300)
        e = torch.exp(score - top)
        total = e.sum(-1, keepdim=True)
        w = torch.where(total > 0, e / total, 0.0)
        o = w @ vv
        # a score: the query's own loss (f32 rows only: those of 16 bits are taken as they are) and d products in f32. It moves the
        # logarithm of a probability, so twice (numerator and sum) the probability itself, with some room for the second order
        lost = (PAIR[fmt] if fmt == "f32" else 0.0) + d * 2.0 ** -24
        off = scale * (x.abs() @ kk.abs().transpose(1, 2)) * lost + (scale * TINY[fmt] * kk.abs().sum(-1)[:, None, :] if fmt == "f32" else 0.0)
        off = off + 2.0 ** -22 * (1 + (score - top).abs().clamp_max(200))     # scaling and exponential: an f32 argument of that size
        off = torch.where(mask, off, 0.0).amax(-1, keepdim=True)
        wide = w @ vv.abs()
        seen_abs = mask.double() @ vv.abs()
        b = wide * (2.2 * off + PAIR[fmt] + (len(seen) + 64) * 2.0 ** -24) + TINY[fmt] * seen_abs
        b = b + HALF_STEP[fmt] * (o.abs() + b) + TINY[fmt]
        out[part] = o.transpose(0, 1).reshape(n, h * d)
        bound[part] = b.transpose(0, 1).reshape(n, h * d)
    return out, bound


def turn(x, pos, rotary, theta=1e4, inv_freq=None, interleaved=False):
    """x [rows, heads, dim] in 64 bits turned by its positions; and the sum of magnitudes that each value was made of."""
    size = x.abs()
    if not rotary:
        return x, size
    f = torch.tensor([theta ** (-2.0 * i / rotary) for i in range(rotary // 2)] if inv_freq is None else list(inv_freq), dtype=torch.float64, device="cuda")
    angle = torch.tensor(pos, dtype=torch.float64, device="cuda")[:, None, None] * f
    i = torch.arange(rotary // 2, device="cuda")
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
    y, size = x.clone(), size.clone()
    y[..., a] = x[..., a] * angle.cos() - x[..., b] * angle.sin()
    y[..., b] = x[..., a] * angle.sin() + x[..., b] * angle.cos()
    both = x[..., a].abs() + x[..., b].abs()
    size[..., a] = both
    size[..., b] = both
    return y, size


def heads_of(rows, d, weight, eps, pos, **rope):
    """q or k heads [rows, heads, dim] as append leaves them, in 64 bits, and a bound without the last rounding."""
    x = rows.double().reshape(rows.shape[0], -1, d)
    if weight is not None:
        x = weight.double() * x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps)
    y, size = turn(x, pos, **rope)
    # norm: the sum's and three more roundings, products with it and the weight; rotation: two products and a sum, and an angle that is
    # off by half a step of its turns in f32 (2^-25 of a turn: 2e-7) and sine and cosine by two steps
    return y, size * ((d / 8 + 12) * 2.0 ** -24 + 4e-7)


def fits(bound, value, fmt):
    """Bound with the rounding to the type on top."""
    return bound + HALF_STEP[fmt] * (value.abs() + bound) + TINY[fmt]


def check(got, want, bound):
    got = got.double()
    off = (got - want).abs()
    assert torch.isfinite(got).all()
    worst = (off / bound.clamp_min(1e-300)).max().item() if off.numel() else 0.0
    assert (off <= bound).all(), "off by %.3g of what rounding explains" % worst
    return worst
