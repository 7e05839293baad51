"""The paged key/value cache where numbers are far apart or large: each expectation from the definition in 64 bits, each tolerance from the
arithmetic that the header states."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import kv_plain as P  # noqa: E402
from test_kv_gpu import here, number, randn  # noqa: E402

pytestmark = pytest.mark.gpu

FLOOR = {"f32": 2.0 ** -39, "f16": 2.0 ** -32}            # how finely a probability is held, relative to the largest (the header)


def led(pkg, lens, rows, dim, fmt, lead, spread, heads=1, seed=3):
    """Sequences whose first key leads by `lead` units and has the value 0; the others are `spread` around 0, their values around 1."""
    lay = P.Layout(lens, 256, rows)
    cache = pkg.KvCache(heads, heads, dim, 256, lay.n_pages, fmt=number(pkg, fmt), scale=1.0)
    k, v = P.pools(cache, fmt)
    k.copy_(randn(seed, *k.shape))
    v.copy_(1 + 0.25 * randn(seed + 1, *v.shape))
    k[..., 0] = 0
    k[..., 1] = (spread * randn(seed + 2, *k.shape[:3])).to(k.dtype)
    for s in range(len(lens)):
        first = lay.table[s, 0].item()
        k[first, :, 0, 0], k[first, :, 0, 1], v[first, :, 0] = lead, 0, 0
    q = torch.zeros(lay.n_rows, heads, dim, device="cuda")
    q[..., :2] = 1
    return lay, cache, k, v, q.reshape(lay.n_rows, heads * dim).to(P.ROWS[fmt])


@pytest.mark.parametrize("fmt", ["f32", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [None, 3, 200])
def test_small_probabilities(gpu_pkg, fmt, dim, rows):
    # A tail whose keys each have 3e-4 to 2e-9 of the leader's weight, and whose values alone make the result. A tail key's probability is off by
    # PAIR of itself or FLOOR of the leader's, by 2^-22 (1 + its distance in units) of itself from an f32 argument of that size and its exponential
    # (as kv_plain), sums by 1e-6 (test_long_sums_of_f32_rows; f16 rows, whose sums stay in the tensor core: 2e-8 per 16 keys); then a rounding.
    for lens in ([64, 700], [9000], [100000], [1300] * 40):
        if rows and len(lens) > 2 and rows > 3:
            continue
        for lead in (8.0, 12.0, 16.0, 20.0):
            for spread in (0.0, 1.0):
                lay, cache, k, v, q = led(gpu_pkg, lens, None if rows is None else [min(rows, n) for n in lens], dim, fmt, lead, spread)
                out = torch.zeros_like(q)
                cache.attend(lay.batch(cache), q, out, stream=here())
                cache.sync(here())
                for s in {0, len(lens) - 1}:
                    n, m, at = lens[s], lay.rows[s], lay.begin[s]
                    kk, vv = (P.keys_of(p, lay, s, list(range(n)))[:, 0] for p in (k, v))
                    score = (kk[:, 0] + kk[:, 1]).expand(m, n).clone()
                    score.masked_fill_(torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda")[:, None], -math.inf)
                    w = torch.softmax(score, -1)
                    want = w @ vv
                    wide = w @ vv.abs()
                    rel = P.PAIR[fmt] + 2.0 ** -22 * (1 + lead + 5 * spread) + (1e-6 if fmt == "f32" else 2e-8 * (n / 16 + 4))
                    bound = wide * rel + FLOOR[fmt] * w.amax(-1, keepdim=True) * ((score > -math.inf).double() @ vv.abs())
                    P.check(out[at:at + m], want, bound + P.HALF_STEP[fmt] * (want.abs() + bound) + 2.0 ** -25 * (fmt == "f16"))
