"""The paged key/value cache where numbers are far apart or large: each expectation from the definition in 64 bits, each tolerance from the
arithmetic that the header states."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import kv_plain as P  # noqa: E402
from test_kv_gpu import attend_case, here, number, randn  # noqa: E402

pytestmark = pytest.mark.gpu

FMTS = ("f32", "f16", "bf16")
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


def settled(pkg, lay, fmt, heads, dim, scale, q, k_of, seed=5, more=0.0):
    """Results of all rows, and softmax of the exact scores times the values: k_of(position) gives the first two values of a key, the others are 0."""
    cache = pkg.KvCache(heads, heads, dim, lay.page, lay.n_pages, fmt=number(pkg, fmt), scale=scale)
    k, v = P.pools(cache, fmt)
    v.copy_(1 + 0.25 * randn(seed, *v.shape))
    for s, n in enumerate(lay.lens):
        at = torch.arange(n)
        page, slot = lay.table[s].long()[at // lay.page].cuda(), (at % lay.page).cuda()
        a, b = k_of(at.double())
        k[page, :, slot, 0], k[page, :, slot, 1] = (t.cuda()[:, None].expand(n, heads).to(k.dtype) for t in (a, b))
    rows = torch.zeros(lay.n_rows, heads, dim, device="cuda")
    rows[..., 0], rows[..., 1] = q
    rows = rows.reshape(lay.n_rows, heads * dim).to(P.ROWS[fmt])
    out = torch.zeros_like(rows)
    cache.attend(lay.batch(cache), rows, out, stream=here())
    cache.sync(here())
    for s, (n, m) in enumerate(zip(lay.lens, lay.rows)):
        kk, vv = (P.keys_of(p, lay, s, list(range(n)))[:, 0] for p in (k, v))
        x = rows[lay.begin[s], :2].double()
        score = (scale * (kk[:, 0] * x[0] + kk[:, 1] * x[1])).expand(m, n).clone()
        score.masked_fill_(torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda")[:, None], -math.inf)
        w = torch.softmax(score, -1)
        want = w @ vv
        # weights as in test_small_probabilities, of distances up to 6 units (others are exact or nothing); values all near 1
        rel = P.PAIR[fmt] + 2.0 ** -22 * 7 + (1e-6 if fmt == "f32" else 2e-8 * (n / 16 + 4) + more)
        bound = rel * (w @ vv.abs()) + 2.0 ** -32 * n
        P.check(out[lay.begin[s]:lay.begin[s] + m].double().reshape(m, heads, dim)[:, 0], want, bound + P.HALF_STEP[fmt] * (want.abs() + bound))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,rows", [([1, 40, 700, 9000], None), ([300] * 80, None), ([1, 40, 3000], [1, 9, 70]), ([700, 900], [700, 333])])
def test_scores_far_from_zero(gpu_pkg, fmt, dim, lens, rows):
    lay = P.Layout(lens, 16, rows)
    top = 1e16 if fmt == "bf16" else 6e4
    scale = 1.0 if fmt == "bf16" else 1e20
    flat, heads = torch.zeros_like, 2
    for sign in (1.0, -1.0):
        # all alike, 1e30 and more away from 0: the average
        settled(gpu_pkg, lay, fmt, heads, dim, scale, (top, 0.0), lambda at: (flat(at) + sign * top, flat(at)))
        # far apart from one another: the largest takes all
        settled(gpu_pkg, lay, fmt, heads, dim, scale, (top, 0.0), lambda at: (sign * top * (0.25 + (at * 7 % 32) / 64), flat(at)))
        # small steps on a large common part: 2^22 + {0, 0.5, ... 5}, exact in f32
        settled(gpu_pkg, lay, fmt, heads, dim, 2.0 ** -7, (32768.0, 64.0), lambda at: (flat(at) + sign * 16384, at * 5 % 11))
        settled(gpu_pkg, lay, fmt, heads, dim, 2.0 ** -7, (512.0, 64.0), lambda at: (flat(at) + sign * 1024, at * 5 % 11))
        # rising slowly past the scores from where on 16-bit rows take differences (2^10 to powers of two): an exponent there is off by 2^-14
        settled(gpu_pkg, lay, fmt, heads, dim, 1 / 8, (8.0, 64.0), lambda at: (at // 64, flat(at) + (87.5 if sign > 0 else -90)), more=2.0 ** -14)
        # rising by more than any distance that a probability survives
        settled(gpu_pkg, lay, fmt, heads, dim, scale, (top / 64, 0.0), lambda at: (sign * ((at // 64) * 64 - 8192), flat(at)))


@pytest.mark.parametrize("fmt", ["bf16", "f16"])
@pytest.mark.parametrize("lens,rows", [([1, 2, 3, 40, 700, 9000], None), ([300] * 80, None), ([1, 40, 3000], [1, 9, 70]), ([700, 900], [700, 333])])
def test_average_of_the_largest_values(gpu_pkg, fmt, lens, rows):
    """Values that are the largest numbers of the type: no sum of them ends at infinity, and no average beyond them."""
    top = torch.finfo(P.CACHE[fmt]).max
    lay = P.Layout(lens, 16, rows)
    for dim in (64, 128):
        cache = gpu_pkg.KvCache(4, 2, dim, 16, lay.n_pages, fmt=number(gpu_pkg, fmt))
        k, v = P.pools(cache, fmt)
        k.copy_(randn(1, *k.shape))
        v[..., ::2], v[..., 1::2] = top, -top
        q = (2 * randn(2, lay.n_rows, 4 * dim)).to(P.ROWS[fmt])
        out = torch.zeros_like(q)
        cache.attend(lay.batch(cache), q, out, stream=here())
        cache.sync(here())
        want = v[0, 0, 0].double().repeat(4).expand(lay.n_rows, -1)
        # weights off by one rounding each (the rest of their error is the same in the sum), sums as above; then a rounding
        rel = P.PAIR[fmt] + 2.0 ** -20 + 2e-8 * (max(lens) / 16 + 4)
        P.check(out, want, top * (rel + P.HALF_STEP[fmt] * (1 + rel)) * torch.ones_like(want))
        assert (out.abs() <= top).all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (2, 1, 128)])
@pytest.mark.parametrize("lens,rows", [([40, 300, 9], None), ([40, 300, 9] * 60, None), ([40, 5000, 9], [9, 70, 9]), ([700, 900, 700] * 3, [700, 333, 600] * 3)])
def test_scores_that_are_no_numbers_are_reported(gpu_pkg, fmt, heads, kv_heads, dim, lens, rows):
    """A row whose scores are NaN or infinite is an error of the next sync; the other rows keep their bits, and what no row sees, rows that see no key
    and rows behind the last sequence are no errors."""
    lay = P.Layout(lens, 16, rows, extra_rows=3)
    cache = gpu_pkg.KvCache(heads, kv_heads, dim, 16, lay.n_pages, fmt=number(gpu_pkg, fmt))
    k, v = P.pools(cache, fmt)
    k.copy_(randn(1, *k.shape))
    v.copy_(randn(2, *v.shape))
    good = randn(3, lay.n_rows, heads * dim).to(P.ROWS[fmt])
    good[lay.real:] = math.nan
    out, plain = torch.zeros_like(good), torch.zeros_like(good)
    batch = lay.batch(cache)
    cache.attend(batch, good, plain, stream=here())
    cache.sync(here())
    at = lay.begin[1] + lay.rows[1] - 1                   # the last row of sequence 1, its last head
    first = lay.table[1, 0].item()
    cases = [("nan", math.nan, None), ("inf", math.inf, None)]
    if fmt == "bf16":                                     # finite numbers whose products are not
        cases += [("above", 1e30, 1e30), ("below", 1e30, -1e30)]
    for name, value, key in cases:
        q = good.clone()
        q[at, (heads - 1) * dim:] = value
        kept = k.clone()
        if key is not None:                               # all keys of sequence 1, or the first one
            some = lay.table[1] if name == "below" else lay.table[1, :1]
            k[some[some >= 0].long().cuda(), kv_heads - 1] = key
        cache.attend(batch, q, out, stream=here())
        with pytest.raises(gpu_pkg.BackendError, match="finite"):
            cache.sync(here())
        cache.sync(here())
        others = [i for i in range(lay.real) if not lay.begin[1] <= i < lay.begin[1] + lay.rows[1]]
        assert torch.equal(out[others], plain[others]) and (out[lay.real:] == 0).all()
        if key is None:
            assert out[at, (heads - 1) * dim:].isnan().all()
            assert torch.equal(out[at, :(heads - 1) * dim], plain[at, :(heads - 1) * dim])
        k.copy_(kept)
    if fmt == "bf16":                                     # one key at minus infinity among others is none
        q = good.clone()
        q[at, (heads - 1) * dim:] = 1e30
        kept = k.clone()
        k[:, kv_heads - 1] = 0
        k[first, kv_heads - 1, 0] = -1e30
        cache.attend(batch, q, out, stream=here())
        cache.sync(here())
        k.copy_(kept)


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_without_keys_are_no_errors(gpu_pkg, fmt):
    for lens, rows in (([0, 3, 0], None), ([0, 3, 2], [4, 5, 300])):
        lay = P.Layout(lens, 16, rows)
        cache = gpu_pkg.KvCache(4, 2, 64, 16, lay.n_pages, fmt=number(gpu_pkg, fmt))
        q = torch.ones(lay.n_rows, 256, device="cuda").to(P.ROWS[fmt])
        blind = [lay.begin[s] + i for s, n in enumerate(lay.rows) for i in range(n) if lay.lens[s] - n + i < 0]
        q[blind] = math.nan
        out = torch.ones_like(q)
        cache.attend(lay.batch(cache), q, out, stream=here())
        cache.sync(here())
        assert (out == 0).all()


def test_reports_are_neither_hidden_nor_lost(gpu_pkg):
    """Two findings before one sync are both named; findings of a stream while another thread syncs a second one are all seen."""
    import threading
    import time
    lay = P.Layout([30, 45], 16)
    cache = gpu_pkg.KvCache(2, 2, 32, 16, lay.n_pages, fmt=gpu_pkg.F32)
    good, table = torch.ones(2, 64, device="cuda"), lay.table_dev.clone()
    large, out = 1e6 * good, torch.zeros_like(good)
    table[1, 2] = lay.n_pages
    fine, broken = lay.batch(cache), cache.batch(lay.len_dev, table)
    calls = {"page": lambda st: cache.append(broken, good, good, good, out, stream=st), "16 bits": lambda st: cache.append(fine, good, large, good, out, stream=st)}
    for order in (["page", "16 bits"], ["16 bits", "page"], ["page", "page"], ["16 bits"]):
        for name in order:
            calls[name](here())
        with pytest.raises(gpu_pkg.BackendError) as said:
            cache.sync(here())
        assert all((name in str(said.value)) == (name in order) for name in calls)
        cache.sync(here())
    seen, stop, streams = [], threading.Event(), [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def look():
        while not stop.is_set():
            try:
                cache.sync(streams[1].cuda_stream)
            except gpu_pkg.BackendError as e:
                seen.append(str(e))

    thread = threading.Thread(target=look)
    thread.start()
    try:
        for i in range(300):
            seen.clear()
            for name in ("page", "16 bits"):
                calls[name](streams[0].cuda_stream)
                until = time.perf_counter() + i % 20 * 5e-6
                while time.perf_counter() < until:
                    pass
            until = time.perf_counter() + 5
            while not all(any(name in text for text in seen) for name in calls):
                assert time.perf_counter() < until, "round %d: %s" % (i, seen)
    finally:
        stop.set()
        thread.join()


@pytest.mark.parametrize("fmt", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 128), (8, 8, 64), (3, 1, 80), (5, 5, 16)])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_norms_of_large_and_small_heads(gpu_pkg, fmt, heads, kv_heads, dim, eps):
    """Heads whose squares f32 does not hold are reported, and no numbers in q_out, 0 in the cache; those beside them are as they should."""
    lay = P.Layout([40, 7], 16, [40, 7])
    w = 1 + 0.3 * randn(5, dim)
    cache = gpu_pkg.KvCache(heads, kv_heads, dim, 16, lay.n_pages, fmt=number(gpu_pkg, fmt), rotary_dim=dim // 8 * 8, q_norm=w.cpu().numpy(), k_norm=w.cpu().numpy(), norm_eps=eps)
    k, v = P.pools(cache, fmt)
    batch = lay.batch(cache)
    pos = [n - r + i for n, r in zip(lay.lens, lay.rows) for i in range(r)]
    fine, large, small = [0.0, 1e18, 1.0, 1e9, 1e-3], [3e38, 1e25, 1e20], [1e-38, 1e-25, 1e-30]
    if eps == 0:
        fine[0] = 1e-18                                   # (0 / 0 otherwise)
    for odd in ([], large, small):
        def rows(seed, n):
            x = randn(seed, lay.n_rows, n, dim)
            x = x / x.abs().amax(-1, keepdim=True)        # the largest value of a head is 1
            power = torch.tensor(fine + odd, device="cuda")
            which = (torch.arange(lay.n_rows * n, device="cuda") % len(power)).reshape(lay.n_rows, n)
            return (x * power[which][..., None]).reshape(lay.n_rows, n * dim).to(P.ROWS[fmt]), which >= len(fine)

        (q, odd_q), (kr, odd_k) = rows(1, heads), rows(2, kv_heads)
        vr, out = randn(3, lay.n_rows, kv_heads * dim).to(P.ROWS[fmt]), torch.zeros_like(q)
        lost = bool(odd) and (odd is large or eps == 0)
        cache.append(batch, q, kr, vr, out, stream=here())
        if lost:
            with pytest.raises(gpu_pkg.BackendError, match="finite"):
                cache.sync(here())
        else:
            cache.sync(here())
            odd_q, odd_k = torch.zeros_like(odd_q), torch.zeros_like(odd_k)
        got_q = out.double().reshape(lay.n_rows, heads, dim)
        got_k = torch.cat([P.keys_of(k, lay, s, list(range(n - r, n))) for s, (n, r) in enumerate(zip(lay.lens, lay.rows))])
        assert not got_q[odd_q].isfinite().any() and (got_k[odd_k] == 0).all()
        for got, x, bad, to in ((got_q, q, odd_q, fmt), (got_k, kr, odd_k, "bf16" if fmt == "bf16" else "f16")):
            want, bound = P.heads_of(x, dim, w, float(np.float32(eps)), pos, rotary=dim // 8 * 8)
            # (2^-134: half a step of the smallest bf16 numbers, where a head of 1e-38 turned by a small angle ends up)
            P.check(got[~bad], want[~bad], P.fits(bound, want, to)[~bad] + 2.0 ** -134)


def test_largest_f16_values(gpu_pkg):
    """65504 is an f16 number: rows of it go into the cache as they are. What norm or rotation brings beyond it is reported."""
    lay = P.Layout([3], 8, [3])
    top = 65504.0
    x = torch.tensor([top, -top, 0.0, 1.0], device="cuda").repeat(8)[None].repeat(3, 1).half()
    cache = gpu_pkg.KvCache(2, 2, 16, 8, lay.n_pages, fmt=gpu_pkg.F16)
    out = torch.zeros_like(x)
    cache.append(lay.batch(cache), x, x, x, out, stream=here())
    cache.sync(here())
    assert torch.equal(out, x)
    for pool in P.pools(cache, "f16"):
        assert torch.equal(P.keys_of(pool, lay, 0, [0, 1, 2]).reshape(3, 32), x.double())
    one = torch.ones_like(x)
    for weight, fits in ((65504.0, True), (65519.0, True), (65521.0, False), (1e6, False)):
        w = np.full(16, weight, np.float32)               # (a head of ones: the weight itself, off by 2^-22 of it at most)
        for which in ("q_norm", "k_norm"):
            cache = gpu_pkg.KvCache(2, 2, 16, 8, lay.n_pages, fmt=gpu_pkg.F16, norm_eps=0.0, **{which: w})
            cache.append(lay.batch(cache), one, one, one, out, stream=here())
            if fits:
                cache.sync(here())
            else:
                with pytest.raises(gpu_pkg.BackendError, match="16 bits"):
                    cache.sync(here())
            got = out if which == "q_norm" else P.keys_of(P.pools(cache, "f16")[0], lay, 0, [0, 1, 2])
            assert (got == (top if fits else math.inf if which == "q_norm" else 0.0)).all()


@pytest.mark.parametrize("rows", [None, 3])
def test_scale_of_scores_is_the_one_given(gpu_pkg, rows):
    # 14 x 0.7419... units between the first key and 64 others, all products exact, the scale to powers of two itself an f32 number (to 3e-12). A tail
    # probability is off by 2^-25 from its exponent, 2^-22 from the exponential, 2^-22 from its pair; the sum of 64 equal ones by 2^-23 (its hi parts
    # add up exactly, the cut is that of adding them to the lo parts), that of all probabilities by 2^-23; a rounding: 8e-7
    scale = 0.7419314384460449
    lay, cache, k, v, q = led(gpu_pkg, [65], None if rows is None else [rows], 128, "f32", 14.0, 0.0)
    cache = gpu_pkg.KvCache(1, 1, 128, 256, lay.n_pages, fmt=gpu_pkg.F32, scale=scale)
    for to, of in zip(P.pools(cache, "f32"), (k, torch.ones_like(v))):
        to.copy_(of)
    P.pools(cache, "f32")[1][lay.table[0, 0].item(), :, 0] = 0
    out = torch.zeros_like(q)
    cache.attend(lay.batch(cache), q, out, stream=here())
    cache.sync(here())
    for i in range(lay.n_rows):
        tail = (65 - lay.n_rows + i) * math.exp(-14 * scale)
        want = tail / (1 + tail)
        assert abs(out[i].double() - want).max() <= 8e-7 * want


@pytest.mark.parametrize("n", [257, 600, 3000])
@pytest.mark.parametrize("fmt,heads,kv_heads,dim", [("bf16", 4, 2, 64), ("f32", 2, 1, 128)])
def test_many_sequences(gpu_pkg, n, fmt, heads, kv_heads, dim):
    """Steps and prompts of more sequences than a warp counts through, some of them empty, in a table with room for far longer ones."""
    lens = [(i * 37) % 90 + (700 if i % 97 == 5 else 0) for i in range(n)]
    for rows in (None, [min((i * 13) % 7 + (150 if i % 101 == 9 else 0), m) if i % 5 else 0 for i, m in enumerate(lens)]):
        lay = P.Layout(lens, 16, rows, extra_rows=3, max_pages=400)
        cache = gpu_pkg.KvCache(heads, kv_heads, dim, 16, lay.n_pages, fmt=number(gpu_pkg, fmt))
        k, v = P.pools(cache, fmt)
        k.copy_(randn(1, *k.shape))
        v.copy_(randn(2, *v.shape))
        q, kr, vr = (randn(s, lay.n_rows, w * dim).to(P.ROWS[fmt]) for s, w in ((3, heads), (4, kv_heads), (5, kv_heads)))
        turned, out = torch.full_like(q, 7.0), torch.full_like(q, 7.0)
        cache.append(lay.batch(cache), q, kr, vr, turned, stream=here())
        cache.attend(lay.batch(cache), q, out, stream=here())
        cache.sync(here())
        full = [i for s, m in enumerate(lay.rows) for i in range(lay.begin[s], lay.begin[s] + m) if lens[s]]
        assert torch.equal(turned[full], q[full]) and (turned[lay.real:] == 7).all() and (out[lay.real:] == 7).all()
        want, bound = P.attend(lay, q, k, v, kv_heads, fmt=fmt)
        P.check(out[:lay.real], want, bound)
        for s in range(0, n, 41):
            m = min(lay.rows[s], lens[s])
            got = P.keys_of(v, lay, s, list(range(lens[s] - m, lens[s])))
            assert torch.equal(got, vr[lay.begin[s]:lay.begin[s] + m].to(v.dtype).double().reshape(got.shape))


@pytest.mark.parametrize("n", [6, 30, 200, 300])
def test_rows_that_many_sequences_claim(gpu_pkg, n):
    """Offsets that go back and forth, so that every second sequence has all rows: reported, no more work than a table in order has, and the next
    call as if nothing had been."""
    lay = P.Layout([500] * n, 16, [1] * n, extra_rows=900)
    cache = gpu_pkg.KvCache(4, 2, 64, 16, lay.n_pages, fmt=gpu_pkg.BF16)
    k, v = P.pools(cache, "bf16")
    k.copy_(randn(1, *k.shape))
    v.copy_(randn(2, *v.shape))
    wide = randn(3, lay.n_rows + 40, 256).bfloat16()
    q, out = wide[20:-20], torch.full_like(wide, 7.0)
    off = torch.tensor([lay.n_rows * (i % 2) for i in range(n + 1)], dtype=torch.int32, device="cuda")
    batch = cache.batch(lay.len_dev, lay.table_dev, row_off=off, n_rows=lay.n_rows)
    cache.attend(batch, q, out[20:-20], stream=here())
    with pytest.raises(gpu_pkg.BackendError, match="does not exist"):
        cache.sync(here())
    assert (out[:20] == 7).all() and (out[-20:] == 7).all()
    cache.append(batch, q, q[:, :128], q[:, :128], out[20:-20], stream=here())
    with pytest.raises(gpu_pkg.BackendError, match="does not exist"):
        cache.sync(here())
    assert (out[:20] == 7).all() and (out[-20:] == 7).all()
    cache.attend(lay.batch(cache), q, out[20:-20], stream=here())
    cache.sync(here())
    want, bound = P.attend(lay, q, k, v, 2, fmt="bf16")
    P.check(out[20:20 + lay.real], want, bound)


def test_prompts_in_buffers_of_many_rows(gpu_pkg):
    lay = P.Layout([300, 0, 4000], 16, [300, 0, 700], extra_rows=2 ** 22)
    cache = gpu_pkg.KvCache(2, 1, 16, 16, lay.n_pages, fmt=gpu_pkg.BF16)
    k, v = P.pools(cache, "bf16")
    k.copy_(randn(1, *k.shape))
    v.copy_(randn(2, *v.shape))
    q = randn(3, lay.n_rows, 32).bfloat16()
    out = torch.full_like(q, 7.0)
    cache.attend(lay.batch(cache), q, out, stream=here())
    cache.sync(here())
    want, bound = P.attend(lay, q, k, v, 1, fmt="bf16")
    P.check(out[:lay.real], want, bound)
    assert (out[lay.real:] == 7).all()


def test_calls_without_a_stream_follow_the_tensors(gpu_pkg):
    """Without a stream, a call is one of torch's current stream: it waits for what writes its rows, and its results are there for what comes next."""
    lay = P.Layout([300, 40], 16, [64, 40])
    cache, side = gpu_pkg.KvCache(4, 2, 64, 16, lay.n_pages, fmt=gpu_pkg.BF16, rotary_dim=64), torch.cuda.Stream()
    k, v = P.pools(cache, "bf16")
    k.copy_(randn(1, *k.shape))
    v.copy_(randn(2, *v.shape))
    x = randn(3, lay.n_rows, 512).bfloat16()
    batch, want, turned, out, late = lay.batch(cache), torch.zeros_like(x[:, :256]), torch.zeros_like(x[:, :256]), torch.zeros_like(x[:, :256]), torch.zeros_like(x)
    cache.append(batch, x[:, :256], x[:, 256:384], x[:, 384:], turned, stream=here())
    cache.attend(batch, turned, want, stream=here())
    cache.sync(here())
    for pool in (k, v):
        pool[lay.table[1, :3].long().cuda()] = 0
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)                     # 10 ms
        late.copy_(x)
        cache.append(batch, late[:, :256], late[:, 256:384], late[:, 384:], turned)
        cache.attend(batch, turned, out)
        copy = out.clone()
        cache.sync()
        assert torch.equal(out, want)                     # (the sync has waited)
    assert torch.equal(copy, want)
    graph = torch.cuda.CUDAGraph()
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        cache.attend(batch, turned, out)
    torch.cuda.synchronize()
    assert (out == 0).all()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("fmt", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,rows", [([3000] * 4, None), ([3000] * 70, None), ([900, 2100], [40, 300]), ([1500] * 6, [1500] * 6)])
def test_roundings_of_16_bit_rows(gpu_pkg, fmt, dim, lens, rows):
    # Two roundings, of each probability and of the result, independent of one another: the mean square of what is off is that of
    # h^2 / 3 (w . v)^2 over the keys and h^2 / 3 o^2, h half a step relative to the lower end of its binade, times 0.541 for numbers spread evenly over the
    # logarithm of a binade ((1 - 1 / 4) / (2 ln 2)). Its root may be 10 % above that; one bit less in a probability makes it 58 % more.
    lay = P.Layout(lens, 16, rows)
    cache = gpu_pkg.KvCache(4, 2, dim, 16, lay.n_pages, fmt=number(gpu_pkg, fmt))
    k, v = P.pools(cache, fmt)
    k.copy_(randn(1, *k.shape))
    v.copy_(randn(2, *v.shape))
    q = randn(3, lay.n_rows, 4 * dim).to(P.ROWS[fmt])
    out = torch.zeros_like(q)
    cache.attend(lay.batch(cache), q, out, stream=here())
    cache.sync(here())
    off, square, count = 0.0, 0.0, 0
    for s, (n, m) in enumerate(zip(lens, lay.rows)):
        kk, vv = (P.keys_of(p, lay, s, list(range(n))).transpose(0, 1).repeat_interleave(2, 0) for p in (k, v))
        rows_of = slice(lay.begin[s], lay.begin[s] + m)
        score = q[rows_of].double().reshape(m, 4, dim).transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(dim)
        score.masked_fill_(torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda")[:, None], -math.inf)
        w = torch.softmax(score, -1)
        o = w @ vv
        off += (out[rows_of].double().reshape(m, 4, dim).transpose(0, 1) - o).square().sum().item()
        square += (w.square() @ vv.square() + o.square()).sum().item()
        count += o.numel()
    want = P.HALF_STEP[fmt] * math.sqrt(0.541 / 3 * square / count)
    assert math.sqrt(off / count) <= 1.1 * want


def test_first_call_of_a_thread(gpu_pkg):
    """A thread that has not touched CUDA before."""
    import threading
    for fmt in FMTS:
        for rows in (None, [30, 129, 300]):
            lay = P.Layout([900, 2000, 333], 16, rows)
            cache = gpu_pkg.KvCache(4, 2, 64, 16, lay.n_pages, fmt=number(gpu_pkg, fmt))
            q = randn(3, lay.n_rows, 256).to(P.ROWS[fmt])
            kr, turned, out, want, failed = q[:, :128], torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q), []
            batch, stream = lay.batch(cache), torch.cuda.Stream()
            cache.append(batch, q, kr, kr, turned, stream=here())
            cache.attend(batch, turned, want, stream=here())
            cache.sync(here())
            for call in (lambda: cache.attend(batch, turned, out, stream=stream.cuda_stream), lambda: cache.append(batch, q, kr, kr, turned, stream=stream.cuda_stream),
                         lambda: cache.sync(stream.cuda_stream)):
                def run():
                    try:
                        call()
                    except Exception as e:
                        failed.append(e)
                thread = threading.Thread(target=run)
                thread.start()
                thread.join()
            assert not failed and torch.equal(out, want)


def test_calls_beside_another_threads_recording(gpu_pkg):
    """While one thread records, another one calls and syncs on its own stream: neither disturbs the other."""
    from concurrent.futures import ThreadPoolExecutor
    for rows in (None, [30, 129, 300]):
        lay = P.Layout([900, 2000, 333], 16, rows)
        cache = gpu_pkg.KvCache(6, 3, 48, 16, lay.n_pages, fmt=gpu_pkg.F16)
        k, v = P.pools(cache, "f16")
        k.copy_(randn(1, *k.shape))
        v.copy_(randn(2, *v.shape))
        q = randn(3, lay.n_rows, 288).half()
        batch, outs, side = lay.batch(cache), [torch.zeros_like(q) for _ in range(2)], torch.cuda.Stream()
        torch.cuda.synchronize()

        def other():
            cache.attend(batch, q, outs[1], stream=side.cuda_stream)
            cache.sync(side.cuda_stream)
            return True

        graph = torch.cuda.CUDAGraph()
        with ThreadPoolExecutor(1) as pool:
            with torch.cuda.graph(graph):
                cache.attend(batch, q, outs[0], stream=here())
                assert pool.submit(other).result()
                cache.attend(batch, q, outs[0], stream=here())
        graph.replay()
        torch.cuda.synchronize()
        want, bound = P.attend(lay, q, k, v, 3, fmt="f16")
        for out in outs:
            P.check(out, want, bound)


@pytest.mark.parametrize("fmt,heads,kv_heads,dim", [("bf16", 4, 2, 64), ("f32", 2, 1, 128), ("f16", 8, 1, 128)])
def test_few_rows_among_many_sequences(gpu_pkg, fmt, heads, kv_heads, dim):
    """Nearly all sequences of a prompts' call bring no rows: clusters share the keys of those that do."""
    n = 700
    lens = [3000 if i in (0, 13, 350, 698, 699) else i % 5 for i in range(n)]
    lay = P.Layout(lens, 16, [9 if m == 3000 else 0 for m in lens], extra_rows=3)
    attend_case(gpu_pkg, lay, heads, kv_heads, dim, fmt)


def test_a_cache_made_beside_a_recording(gpu_pkg):
    """On a stream that waits for the legacy default stream, as cudaStreamCreate makes them."""
    import ctypes
    from concurrent.futures import ThreadPoolExecutor
    runtime = ctypes.CDLL("libcudart.so.12")
    raw = ctypes.c_void_p()
    assert runtime.cudaStreamCreate(ctypes.byref(raw)) == 0
    stream, x, graph = torch.cuda.ExternalStream(raw.value), torch.ones(1000, device="cuda"), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def make():
        cache = gpu_pkg.KvCache(2, 2, 16, 16, 8, fmt=gpu_pkg.F16, rotary_dim=16, q_norm=np.ones(16), k_norm=np.ones(16))
        return cache.close() is None

    with ThreadPoolExecutor(1) as pool:
        with torch.cuda.graph(graph, stream=stream):
            x.add_(1)
            assert pool.submit(make).result()
            x.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert (x == 3).all()
    del graph
    torch.cuda.synchronize()
    assert runtime.cudaStreamDestroy(raw) == 0


@pytest.mark.parametrize("rows", [None, [200]])
def test_small_bf16_values(gpu_pkg, rows):
    """Values down to 1e-30 come out as exactly as others."""
    lay = P.Layout([700], 16, rows)
    for dim in (64, 128):
        cache = gpu_pkg.KvCache(4, 2, dim, 16, lay.n_pages, fmt=gpu_pkg.BF16)
        k, v = P.pools(cache, "bf16")
        k.copy_(randn(1, *k.shape))
        q = randn(3, lay.n_rows, 4 * dim).bfloat16()
        out = torch.zeros_like(q)
        for size in (1.0, 1e-20, 1e-28, 1e-30):
            v.copy_((1 + 0.1 * randn(5, *v.shape)) * size)
            cache.attend(lay.batch(cache), q, out, stream=here())
            cache.sync(here())
            want, bound = P.attend(lay, q, k, v, 2, fmt="bf16")
            P.check(out, want, bound)
