"""The paged key/value cache on the GPU: append and attend against their definitions in 64 bits (kv_plain), at the sizes, masks and
tables where they can go wrong. Bounds are those of the arithmetic, worked out in kv_plain."""
import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import kv_plain as P  # noqa: E402

pytestmark = pytest.mark.gpu

FMTS = ("f32", "f16", "bf16")


def number(pkg, fmt):
    return {"f32": pkg.F32, "f16": pkg.F16, "bf16": pkg.BF16}[fmt]


def here():
    return torch.cuda.current_stream().cuda_stream


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def filled(pkg, lay, heads, kv_heads, dim, fmt, seed=1, **more):
    """A cache whose pools hold random keys and values, stale ones in the slots that no sequence has."""
    cache = pkg.KvCache(heads, kv_heads, dim, lay.page, lay.n_pages, fmt=number(pkg, fmt), **more)
    k, v = P.pools(cache, fmt)
    k.copy_(randn(seed, *k.shape))
    v.copy_(randn(seed + 1, *v.shape))
    return cache, k, v


def attend_case(pkg, lay, heads, kv_heads, dim, fmt, seed=1, sharp=1.0, **more):
    cache, k, v = filled(pkg, lay, heads, kv_heads, dim, fmt, seed, **more)
    q = (sharp * randn(seed + 2, lay.n_rows, heads * dim)).to(P.ROWS[fmt])
    out = torch.full_like(q, 7.0)
    cache.attend(lay.batch(cache), q, out, stream=here())
    cache.sync(here())
    want, bound = P.attend(lay, q, k, v, kv_heads, more.get("window", 0), more.get("n_sinks", 0), more.get("scale", 0.0), fmt)
    P.check(out[:lay.real], want, bound)
    assert (out[lay.real:] == 7.0).all()                  # rows behind the last sequence
    return cache, q, out


# ------------------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,kv_heads,dim,page,rotary,interleaved", [
    (4, 2, 128, 16, 128, False), (8, 8, 64, 32, 64, True), (5, 5, 64, 8, 32, False), (3, 1, 80, 16, 40, False), (6, 3, 112, 64, 56, True),
    (7, 1, 96, 128, 48, False), (2, 2, 16, 256, 16, False), (12, 4, 32, 16, 8, False), (4, 4, 48, 16, 0, False), (64, 1, 128, 16, 72, False)])
def test_append(gpu_pkg, fmt, heads, kv_heads, dim, page, rotary, interleaved):
    for norm, rows, lens in ((True, [1, 17, 0, 40, 3], [1, 17, 9, 1000, 33]), (False, None, [5, 0, 300, 1])):
        lay = P.Layout(lens, page, rows, extra_rows=3, seed=heads)
        wq, wk = (1 + 0.3 * randn(s, dim) for s in (5, 6))
        cache, k, v = filled(gpu_pkg, lay, heads, kv_heads, dim, fmt, rotary_dim=rotary, interleaved=interleaved, rope_theta=1e6,
                             q_norm=wq.cpu().numpy() if norm else None, k_norm=wk.cpu().numpy() if norm else None, norm_eps=1e-5)
        k0, v0 = k.clone(), v.clone()
        width = (heads + 2 * kv_heads) * dim
        x = (2 * randn(3, lay.n_rows, width)).to(P.ROWS[fmt])           # one projection's output
        q, kr, vr = x[:, :heads * dim], x[:, heads * dim:(heads + kv_heads) * dim], x[:, (heads + kv_heads) * dim:]
        out = torch.full((lay.n_rows, heads * dim), 7.0, dtype=q.dtype, device="cuda")
        batch = lay.batch(cache)
        cache.append(batch, q, kr, vr, out, stream=here())
        cache.sync(here())
        seq = [s for s, n in enumerate(lay.rows) for _ in range(n) if lay.lens[s] > 0]
        at = [lay.begin[s] + i for s, n in enumerate(lay.rows) for i in range(n) if lay.lens[s] > 0]
        pos = [lay.lens[s] - n + i for s, n in enumerate(lay.rows) for i in range(n) if lay.lens[s] > 0]
        rope = dict(rotary=rotary, theta=1e6, interleaved=interleaved)
        want, bound = P.heads_of(q[at], dim, wq if norm else None, 1e-5, pos, **rope)
        P.check(out[at].reshape(want.shape), want, P.fits(bound, want, fmt))
        rest = sorted(set(range(lay.n_rows)) - set(at))
        assert (out[rest] == 7.0).all()
        page_of = torch.stack([lay.table[s, p // page] for s, p in zip(seq, pos)]).long().cuda()
        slot = torch.tensor([p % page for p in pos]).cuda()
        cfmt = "bf16" if fmt == "bf16" else "f16"
        want, bound = P.heads_of(kr[at], dim, wk if norm else None, 1e-5, pos, **rope)
        P.check(k[page_of, :, slot], want, P.fits(bound, want, cfmt))
        assert torch.equal(v[page_of, :, slot], vr[at].reshape(len(at), kv_heads, dim).to(v.dtype))
        for pool, old in ((k, k0), (v, v0)):              # nothing else has changed
            pool[page_of, :, slot] = old[page_of, :, slot]
            assert torch.equal(pool, old)
        # in place, and without the graph's help: the same bits
        again = q.clone()
        cache.append(batch, again, kr, vr, again, stream=here())
        cache.sync(here())
        assert torch.equal(again[at], out[at]) and torch.equal(again[rest], q[rest])


def test_append_many_rows(gpu_pkg):
    """Whole rows per warp: more rows than the SMs hold warps."""
    rows = [1 + (i * 37) % 61 for i in range(333)]
    lay = P.Layout([r + i % 7 for i, r in enumerate(rows)], 16, rows, extra_rows=100)
    cache, k, v = filled(gpu_pkg, lay, 4, 2, 64, "f16", rotary_dim=64)
    q, kr, vr = (randn(s, lay.n_rows, n * 64).half() for s, n in ((1, 4), (2, 2), (3, 2)))
    out = torch.zeros_like(q)
    cache.append(lay.batch(cache), q, kr, vr, out, stream=here())
    cache.sync(here())
    pos = [n - r + i for n, r in zip(lay.lens, rows) for i in range(r)]
    want, bound = P.heads_of(q[:lay.real], 64, None, 0, pos, rotary=64)
    P.check(out[:lay.real].reshape(want.shape), want, P.fits(bound, want, "f16"))
    assert (out[lay.real:] == 0).all()
    got = torch.cat([P.keys_of(v, lay, s, list(range(n - r, n))) for s, (n, r) in enumerate(zip(lay.lens, rows))])
    assert torch.equal(got, vr[:lay.real].double().reshape(got.shape))


def test_append_far_positions(gpu_pkg):
    """Positions of a million, frequencies that the caller gives; a table whose other pages were given back."""
    lens = [1_000_003, 2 ** 20, 777_777]
    lay = P.Layout(lens, 256, drop=lambda s, p: p < (lens[s] - 1) // 256)
    freq = np.array([1.0, 0.731, 0.0123, -0.5])
    cache, k, v = filled(gpu_pkg, lay, 2, 1, 32, "f32", rotary_dim=8, inv_freq=freq)
    q, kr, vr = (randn(s, 3, n * 32) for s, n in ((1, 2), (2, 1), (3, 1)))
    out = torch.zeros_like(q)
    cache.append(lay.batch(cache), q, kr, vr, out, stream=here())
    cache.sync(here())
    want, bound = P.heads_of(q, 32, None, 0, [n - 1 for n in lens], rotary=8, inv_freq=freq)
    P.check(out.reshape(want.shape), want, P.fits(bound, want, "f32"))
    want, bound = P.heads_of(kr, 32, None, 0, [n - 1 for n in lens], rotary=8, inv_freq=freq)
    P.check(torch.cat([P.keys_of(k, lay, s, [n - 1]) for s, n in enumerate(lens)]), want, P.fits(bound, want, "f16"))


def test_append_more_rows_than_keys(gpu_pkg):
    lay = P.Layout([3, 4], 16, [5, 4])
    cache, k, v = filled(gpu_pkg, lay, 2, 2, 16, "f16")
    q = randn(1, 9, 32).half()
    out = torch.full_like(q, 7.0)
    cache.append(lay.batch(cache), q, q, q, out, stream=here())
    cache.sync(here())
    assert (out[:2] == 7.0).all() and torch.equal(out[2:], q[2:])
    assert torch.equal(P.keys_of(v, lay, 0, [0, 1, 2]), q[2:5].double().reshape(3, 2, 16))


@pytest.mark.parametrize("fmt", FMTS)
def test_append_reports_values_that_do_not_fit(gpu_pkg, fmt):
    lay = P.Layout([3, 9], 16)
    cache, k, v = filled(gpu_pkg, lay, 2, 2, 32, fmt)
    batch = lay.batch(cache)
    good = torch.ones(2, 64, device="cuda").to(P.ROWS[fmt])
    out = torch.zeros_like(good)
    bad = [math.inf, -math.inf, math.nan] + ([70000.0, 65504.0] if fmt == "f32" else [])
    for value in bad:
        for which in range(3):
            rows = [good.clone() for _ in range(3)]
            rows[which][1, 37] = value
            cache.append(batch, *rows, out, stream=here())
            if which == 0 and fmt == "f32" and math.isfinite(value):
                cache.sync(here())                        # an f32 query may be that large
                continue
            with pytest.raises(gpu_pkg.BackendError, match="16 bits"):
                cache.sync(here())
            cache.sync(here())                            # reported once
            if which:
                got = P.keys_of(k if which == 1 else v, lay, 1, [8]).reshape(-1)
                assert got[37] == 0 and (got[:37] == 1).all() and (got[38:] == 1).all()


# ------------------------------------------------------------------------------------------------------------ one row per sequence
EDGES = [1, 0, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 1000]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 8, 128, 16), (16, 2, 128, 16), (32, 4, 64, 32), (6, 2, 80, 8), (20, 1, 96, 64), (64, 1, 112, 16),
                                                     (3, 3, 16, 16), (16, 1, 32, 128), (33, 1, 48, 256), (17, 17, 64, 8)])
def test_step_lengths(gpu_pkg, fmt, heads, kv_heads, dim, page):
    lay = P.Layout(EDGES, page, extra_rows=2, seed=dim)
    attend_case(gpu_pkg, lay, heads, kv_heads, dim, fmt, sharp=2.0)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window,sinks,page", [(1, 0, 16), (5, 1, 8), (32, 4, 16), (33, 33, 32), (100, 64, 16), (64, 200, 64), (2000, 7, 16)])
def test_step_window(gpu_pkg, fmt, window, sinks, page):
    lay = P.Layout(EDGES + [100, 101, 132, 133, 137, 264, 1234], page, seed=window)
    attend_case(gpu_pkg, lay, 8, 4, 64, fmt, window=window, n_sinks=sinks)


@pytest.mark.parametrize("lens", [[1], [33], [700], [9000], [20001], [40000, 3], [0, 0], [12345] * 3, [5] * 150, [300] * 40 + [6000]])
def test_step_batches(gpu_pkg, lens):
    """Every way to split a length, from one sequence to many."""
    lay = P.Layout(lens, 16, seed=len(lens))
    attend_case(gpu_pkg, lay, 8, 2, 128, "bf16", sharp=1.5)


def test_step_scale_and_sharp_scores(gpu_pkg):
    lay = P.Layout([1, 40, 300, 1025], 16)
    attend_case(gpu_pkg, lay, 4, 2, 64, "f16", scale=1.0)                 # scores of +-30: one key takes all
    attend_case(gpu_pkg, lay, 4, 2, 64, "f32", scale=0.7)
    attend_case(gpu_pkg, lay, 4, 2, 64, "bf16", scale=1e-3)


def test_dropped_pages_are_not_read(gpu_pkg):
    """Pages between the first tokens and the window: no entry in the table."""
    lens = [500, 1600, 90, 129, 8000]
    for rows in (None, [3, 130, 90, 1, 257]):
        n = rows or [1] * 5
        lay = P.Layout(lens, 16, rows, drop=lambda s, p: p > 0 and (p + 1) * 16 <= lens[s] - n[s] - 64 + 1)
        assert (lay.table[4] == -1).sum() > 400
        for fmt in FMTS:
            attend_case(gpu_pkg, lay, 4, 2, 128, fmt, window=64, n_sinks=5)


# ------------------------------------------------------------------------------------------------------------ rows per sequence
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 8, 128, 16), (8, 2, 128, 64), (6, 2, 64, 16), (5, 1, 80, 8), (16, 1, 112, 256), (3, 3, 16, 32),
                                                     (64, 1, 48, 128), (33, 1, 96, 16)])
def test_chunk_lengths(gpu_pkg, fmt, heads, kv_heads, dim, page):
    rows = [1, 5, 0, 16, 33, 64, 127, 128, 129, 260, 31]
    lens = [1, 5, 7, 300, 33, 70, 127, 500, 129, 260, 1027]
    lay = P.Layout(lens, page, rows, extra_rows=5, seed=dim)
    attend_case(gpu_pkg, lay, heads, kv_heads, dim, fmt, sharp=2.0)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 2), (64, 4), (128, 128), (129, 1), (300, 140), (5000, 3)])
def test_chunk_window(gpu_pkg, fmt, window, sinks):
    lay = P.Layout([200, 700, 1, 1300, 130], 16, [200, 513, 1, 90, 129], seed=window)
    attend_case(gpu_pkg, lay, 8, 2, 64, fmt, window=window, n_sinks=sinks)
    attend_case(gpu_pkg, lay, 2, 2, 128, fmt, window=window, n_sinks=sinks)


def test_chunk_rows_without_keys(gpu_pkg):
    """More rows than keys: the rows in front of the first position see nothing and come out as 0."""
    lay = P.Layout([0, 3, 2, 100], 16, [4, 5, 300, 100])
    for fmt in FMTS:
        _, _, out = attend_case(gpu_pkg, lay, 4, 1, 64, fmt)
        assert (out[:6] == 0).all() and (out[9:9 + 298] == 0).all()


def test_chunk_many_sequences(gpu_pkg):
    rows = [(i * 7) % 40 for i in range(150)]
    lay = P.Layout([r + (i * 11) % 50 for i, r in enumerate(rows)], 16, rows, extra_rows=64)
    attend_case(gpu_pkg, lay, 4, 4, 64, "bf16")
    attend_case(gpu_pkg, lay, 12, 2, 128, "f16")


def test_chunk_scores_that_grow(gpu_pkg):
    """Keys whose scores rise along the sequence, by steps small and large: the running maximum moves again and again."""
    for fmt in FMTS:
        lay = P.Layout([1500], 16, [1500])
        cache, k, v = filled(gpu_pkg, lay, 2, 1, 128, fmt)
        q = torch.zeros(1500, 256, device="cuda")
        q[:, 0], q[:, 128] = 1.0, -0.25
        q = q.to(P.ROWS[fmt])
        ramp = torch.arange(1500, dtype=torch.float32, device="cuda") * 0.125 + (torch.arange(1500, device="cuda") // 500) * 256.0
        at = torch.arange(1500)
        k[lay.table[0].long()[at // 16].cuda(), :, (at % 16).cuda(), 0] = ramp[:, None].to(k.dtype)
        out = torch.zeros_like(q)
        cache.attend(lay.batch(cache), q, out, stream=here())
        cache.sync(here())
        want, bound = P.attend(lay, q, k, v, 1, fmt=fmt)
        P.check(out, want, bound)


# ------------------------------------------------------------------------------------------------------------ masked places, tables
@pytest.mark.parametrize("rows", [None, [1, 40, 30]])
def test_what_is_masked_has_no_say(gpu_pkg, rows):
    """The slots behind a sequence's keys and outside of its window hold the largest numbers there are; results keep their bits."""
    for fmt in FMTS:
        for window in (0, 20):
            lay = P.Layout([1, 45, 130], 16, rows)
            cache, k, v = filled(gpu_pkg, lay, 4, 2, 64, fmt, window=window)
            q = randn(9, lay.n_rows, 256).to(P.ROWS[fmt])
            out, other = torch.zeros_like(q), torch.zeros_like(q)
            cache.attend(lay.batch(cache), q, out, stream=here())
            hidden = torch.ones(k.shape[0], 16, dtype=torch.bool)
            for s, (n, length) in enumerate(zip(lay.rows, lay.lens)):
                for j in range(max(0, length - n - window + 1) if window else 0, length):
                    hidden[lay.table[s, j // 16], j % 16] = False
            big = 65472.0 if fmt != "bf16" else 1e30          # f16 scores reach 1e10
            where = hidden.cuda().nonzero(as_tuple=True)
            k[where[0], :, where[1]] = big
            v[where[0], :, where[1]] = -big
            cache.attend(lay.batch(cache), q, other, stream=here())
            cache.sync(here())
            assert torch.equal(out, other)


def bad_tables(lay, what):
    table, lens, off = lay.table_dev.clone(), lay.len_dev.clone(), None if lay.off_dev is None else lay.off_dev.clone()
    if what == "page":
        table[1, 1] = lay.n_pages
    elif what == "negative page":
        table[1, 0] = -5
    elif what == "large page":
        table[1, 1] = 2 ** 31 - 1
    elif what == "length":
        lens[1] = lay.table.shape[1] * lay.page + 1
    elif what == "negative length":
        lens[1] = -1
    elif what == "huge length":
        lens[1] = 2 ** 31 - 1
    elif what == "rows":
        off[2] = lay.n_rows + 1
    elif what == "negative rows":
        off[2] = off[1] - 1
    elif what == "huge rows":
        off[2] = 2 ** 31 - 1
    return table, lens, off


@pytest.mark.parametrize("rows,what", [(r, w) for r in (None, [1, 40, 30, 6]) for w in (
    "page", "negative page", "large page", "length", "negative length", "huge length") + (("rows", "negative rows", "huge rows") if r else ())])
def test_bad_tables_are_reported(gpu_pkg, rows, what):
    """What names a page, a length or a row that does not exist is an error of the next sync; sequences that are in order keep their
    results, and nothing outside of the buffers is touched."""
    lay = P.Layout([30, 45, 130, 17], 16, rows, extra_rows=4)
    for fmt in ("f16", "f32"):
        cache, k, v = filled(gpu_pkg, lay, 4, 2, 64, fmt)
        q = randn(9, lay.n_rows, 256).to(P.ROWS[fmt])
        out, other, kept = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
        cache.attend(lay.batch(cache), q, out, stream=here())
        table, lens, off = bad_tables(lay, what)
        batch = cache.batch(lens, table, row_off=off, n_rows=lay.n_rows)
        cache.sync(here())
        cache.attend(batch, q, other, stream=here())
        with pytest.raises(gpu_pkg.BackendError, match="does not exist"):
            cache.sync(here())
        first = lay.begin[1]                              # sequence 0, and where the rows are in order those behind sequence 1
        if what != "negative rows":                       # (offsets 0, 1, 0, 71: row 0 is sequence 0's and sequence 2's)
            assert torch.equal(out[:first], other[:first])
        if "rows" not in what:
            assert torch.equal(out[lay.begin[2]:lay.real], other[lay.begin[2]:lay.real])
        kr = q[:, :128].contiguous()
        if what in ("page", "large page") and rows is None:
            lens[1] = 20                                  # the new key itself lies in that page
        cache.append(batch, q, kr, kr, kept, stream=here())
        if what != "negative page" or rows:
            with pytest.raises(gpu_pkg.BackendError, match="does not exist"):
                cache.sync(here())
        else:
            cache.sync(here())                            # (a step writes its last page only)
        cache.attend(lay.batch(cache), q, out, stream=here())
        cache.sync(here())


# ------------------------------------------------------------------------------------------------------------ together
def layer(cache, batch, x, heads, kv_heads, dim, stream):
    """One decoder layer's attention on a projection's output."""
    q, k, v = x[:, :heads * dim], x[:, heads * dim:(heads + kv_heads) * dim], x[:, (heads + kv_heads) * dim:]
    turned = torch.empty(x.shape[0], heads * dim, dtype=x.dtype, device="cuda")
    out = torch.zeros_like(turned)
    cache.append(batch, q, k, v, turned, stream=stream)
    cache.attend(batch, turned, out, stream=stream)
    return turned, out


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_prompts_pieces_and_steps(gpu_pkg, fmt, window, sinks):
    """Three sequences: prompts at once, then a piece, then steps of which every row is checked against a cache kept in 64 bits' stead."""
    heads, kv_heads, dim, page, most = 8, 2, 64, 16, 400
    g = torch.Generator().manual_seed(3)
    table = torch.randperm(3 * 25, generator=g).reshape(3, 25).to(torch.int32).cuda()
    w = (1 + 0.2 * randn(8, dim))
    cache = gpu_pkg.KvCache(heads, kv_heads, dim, page, 75, fmt=number(gpu_pkg, fmt), rotary_dim=dim, q_norm=w.cpu().numpy(), k_norm=w.cpu().numpy(),
                            window=window, n_sinks=sinks)
    k_pool, v_pool = P.pools(cache, fmt)
    lens = [0, 0, 0]
    for turn, rows in enumerate(([130, 17, 1], [0, 5, 64], [1, 1, 1], [1, 1, 1], [100, 1, 9], [1, 1, 1])):
        step = rows == [1, 1, 1]
        lens = [n + r for n, r in zip(lens, rows)]
        lay = P.Layout(lens, page, None if step else rows, extra_rows=2 * (not step), max_pages=25)
        lay.table, lay.table_dev = table.cpu(), table
        x = randn(50 + turn, lay.n_rows, (heads + 2 * kv_heads) * dim).to(P.ROWS[fmt])
        turned, out = layer(cache, lay.batch(cache), x, heads, kv_heads, dim, here())
        cache.sync(here())
        pos = [n - r + i for n, r in zip(lens, rows) for i in range(r)]
        want, bound = P.heads_of(x[:lay.real, :heads * dim], dim, w, 1e-6, pos, rotary=dim)
        P.check(turned[:lay.real].reshape(want.shape), want, P.fits(bound, want, fmt))
        want, bound = P.heads_of(x[:lay.real, heads * dim:(heads + kv_heads) * dim], dim, w, 1e-6, pos, rotary=dim)
        got = torch.cat([P.keys_of(k_pool, lay, s, list(range(n - r, n))) for s, (n, r) in enumerate(zip(lens, rows))])
        P.check(got, want, P.fits(bound, want, "bf16" if fmt == "bf16" else "f16"))
        want, bound = P.attend(lay, turned, k_pool, v_pool, kv_heads, window, sinks, fmt=fmt)
        P.check(out[:lay.real], want, bound)


def test_beside_the_resident_linears(gpu_pkg, synth):
    """A layer as a host runs it: projection (QMat), append, attend, output projection, all on device rows."""
    import ctypes
    heads, kv_heads, dim, d = 8, 2, 64, 256
    rng = np.random.default_rng(5)
    L = gpu_pkg.lib()
    L.mynah_b200_qmat_mul_device.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_int]
    wide = (heads + 2 * kv_heads) * dim
    w_in, w_out = rng.standard_normal((wide, d)).astype(np.float32) * 0.1, rng.standard_normal((d, heads * dim)).astype(np.float32) * 0.1
    qkv, o = gpu_pkg.QMat(gpu_pkg.F32, w_in, wide, d), gpu_pkg.QMat(gpu_pkg.F32, w_out, d, heads * dim)
    lay = P.Layout([40, 200], 16, [40, 33])
    cache, k, v = filled(gpu_pkg, lay, heads, kv_heads, dim, "f32", rotary_dim=dim)
    x = randn(1, lay.n_rows, d)
    rows, y = torch.zeros(lay.n_rows, wide, device="cuda"), torch.zeros(lay.n_rows, d, device="cuda")
    torch.cuda.synchronize()
    assert L.mynah_b200_qmat_mul_device(qkv.h, x.data_ptr(), rows.data_ptr(), lay.n_rows, 0) == 0
    assert L.mynah_b200_qmat_sync(qkv.h) == 0
    turned, out = layer(cache, lay.batch(cache), rows, heads, kv_heads, dim, here())
    cache.sync(here())
    assert L.mynah_b200_qmat_mul_device(o.h, out.data_ptr(), y.data_ptr(), lay.n_rows, 0) == 0
    assert L.mynah_b200_qmat_sync(o.h) == 0
    want, bound = P.attend(lay, turned, k, v, kv_heads, fmt="f32")
    P.check(out, want, bound)
    wt = torch.from_numpy(w_out).cuda().double()
    P.check(y, want @ wt.T, bound @ wt.abs().T + 4e-6 * (want.abs() @ wt.abs().T))


def test_captured_steps(gpu_pkg):
    """A step recorded once and launched for growing lengths, its tables written between the launches."""
    heads, kv_heads, dim, n = 8, 4, 128, 5
    table = torch.arange(n * 8, dtype=torch.int32).reshape(n, 8).flip(0).contiguous().cuda()
    cache = gpu_pkg.KvCache(heads, kv_heads, dim, 16, n * 8, fmt=gpu_pkg.BF16, rotary_dim=dim)
    k, v = P.pools(cache, "bf16")
    kv_len = torch.zeros(n, dtype=torch.int32, device="cuda")
    batch = cache.batch(kv_len, table)
    x = torch.zeros(n, (heads + 2 * kv_heads) * dim, dtype=torch.bfloat16, device="cuda")
    parts = x[:, :heads * dim], x[:, heads * dim:(heads + kv_heads) * dim], x[:, (heads + kv_heads) * dim:]
    turned, out = (torch.zeros(n, heads * dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(batch, *parts, turned, stream=here())
        cache.attend(batch, turned, out, stream=here())
    lens = [0, 3, 15, 30, 100]
    for s, length in enumerate(lens):                     # what came before the steps
        for p in range((length + 15) // 16):
            k[table[s, p]] = randn(s * 9 + p, kv_heads, 16, dim).bfloat16()
            v[table[s, p]] = randn(s * 9 + p + 99, kv_heads, 16, dim).bfloat16()
    for i in range(20):
        lens = [m + (s != 2) for s, m in enumerate(lens)]
        kv_len.copy_(torch.tensor([m if s != 2 else 0 for s, m in enumerate(lens)], dtype=torch.int32))
        x.copy_(randn(1000 + i, *x.shape))
        graph.replay()
        cache.sync(here())
        lay = P.Layout([m if s != 2 else 0 for s, m in enumerate(lens)], 16, max_pages=8)
        lay.table, lay.table_dev = table.cpu(), table
        want, bound = P.attend(lay, turned, k, v, kv_heads, fmt="bf16")
        P.check(out, want, bound)


@pytest.mark.parametrize("rows", [None, [300, 100]])
def test_two_graphs_and_streams_at_once(gpu_pkg, rows):
    """Two recordings of one handle's calls, launched side by side again and again: no workspace that they could share."""
    lays = [P.Layout([5000, 700], 16, rows, seed=s) for s in (1, 2)]
    cache, k, v = filled(gpu_pkg, lays[0], 8, 2, 128, "bf16")
    streams = [torch.cuda.Stream() for _ in range(2)]
    q = [randn(s, lay.n_rows, 1024).bfloat16() for s, lay in enumerate(lays)]
    alone = [torch.zeros_like(t) for t in q]
    outs = [torch.zeros_like(t) for t in q]
    batches = [lay.batch(cache) for lay in lays]
    for b, t, o in zip(batches, q, alone):
        cache.attend(b, t, o, stream=here())
    torch.cuda.synchronize()
    graphs = []
    for b, t, o, st in zip(batches, q, outs, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=st):
            for _ in range(4):
                cache.attend(b, t, o, stream=st.cuda_stream)
    for _ in range(30):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, o) for a, o in zip(alone, outs))
    cache.sync()


def test_same_bits_every_time_and_beside_others(gpu_pkg):
    """No atomics in sums: a call gives its bits again, from any stream and thread, and a sequence gives the same bits beside others."""
    from concurrent.futures import ThreadPoolExecutor
    for rows in (None, [30, 129, 300]):
        lay = P.Layout([900, 2000, 333], 16, rows)
        cache, k, v = filled(gpu_pkg, lay, 8, 2, 64, "f32")
        q = randn(1, lay.n_rows, 512)
        first = torch.zeros_like(q)
        batch = lay.batch(cache)
        cache.attend(batch, q, first, stream=here())
        cache.sync(here())

        def one(i):
            st = torch.cuda.Stream()
            out = torch.zeros_like(q)
            st.wait_stream(torch.cuda.default_stream())
            for _ in range(10):
                cache.attend(batch, q, out, stream=st.cuda_stream)
            cache.sync(st.cuda_stream)
            return torch.equal(out, first)

        torch.cuda.synchronize()
        with ThreadPoolExecutor(4) as pool:
            assert all(pool.map(one, range(8)))
        # beside other sequences, in a call of as many rows and sequences: how a sequence is cut does not depend on the others
        order, other = [2, 1, 0], P.Layout([333, 2000, 7], 16, [300, 129, 7] if rows else None, seed=5)
        table = other.table.clone()
        table[:, :] = -1
        for to, (at, keep) in enumerate(((2, True), (1, True), (0, False))):
            n = min(table.shape[1], lay.table.shape[1])
            table[to, :n] = lay.table[at, :n] if keep else lay.table[0, :n]
        n_rows = lay.n_rows
        q2 = torch.zeros(n_rows, 512, device="cuda")
        begin2 = other.begin
        for to, at in enumerate(order[:2]):
            q2[begin2[to]:begin2[to] + lay.rows[at]] = q[lay.begin[at]:lay.begin[at] + lay.rows[at]]
        out2 = torch.zeros_like(q2)
        b2 = cache.batch(other.len_dev, table.cuda(), row_off=other.off_dev, n_rows=n_rows)
        cache.attend(b2, q2, out2, stream=here())
        cache.sync(here())
        for to, at in enumerate(order[:2]):
            assert torch.equal(out2[begin2[to]:begin2[to] + lay.rows[at]], first[lay.begin[at]:lay.begin[at] + lay.rows[at]])


def test_offsets_beyond_32_bits(gpu_pkg):
    """Pools of 5.4 GB each: the last pages lie behind 2^31 values."""
    heads, kv_heads, dim, page, n_pages = 8, 8, 128, 64, 41000
    cache = gpu_pkg.KvCache(heads, kv_heads, dim, page, n_pages, fmt=gpu_pkg.BF16)
    k, v = P.pools(cache, "bf16")
    for rows in (None, [100, 70]):
        lay = P.Layout([100, 70], page, rows)
        lay.table = torch.tensor([[40999, 3], [40998, 40997]], dtype=torch.int32)
        lay.table_dev = lay.table.cuda()
        x = [randn(s, lay.n_rows, 1024).bfloat16() for s in range(3)]
        if rows is None:
            for s, length in enumerate(lay.lens):
                for p in range(2):
                    k[lay.table[s, p]] = randn(s + 2 * p, kv_heads, page, dim).bfloat16()
                    v[lay.table[s, p]] = randn(s + 2 * p + 9, kv_heads, page, dim).bfloat16()
        turned, out = torch.zeros_like(x[0]), torch.zeros_like(x[0])
        cache.append(lay.batch(cache), *x, turned, stream=here())
        cache.attend(lay.batch(cache), turned, out, stream=here())
        cache.sync(here())
        want, bound = P.attend(lay, turned, k, v, kv_heads, fmt="bf16")
        P.check(out, want, bound)
        got = torch.cat([P.keys_of(k, lay, s, list(range(m - r, m))) for s, (m, r) in enumerate(zip(lay.lens, lay.rows))])
        assert torch.equal(got, x[1].double().reshape(got.shape))
    cache.close()


# ------------------------------------------------------------------------------------------------------------ refusals
def test_refusals(gpu_pkg):
    lay = P.Layout([30, 45], 16)
    cache, k, v = filled(gpu_pkg, lay, 4, 2, 64, "f16")
    batch = lay.batch(cache)
    q, kr = torch.ones(2, 256, device="cuda").half(), torch.ones(2, 128, device="cuda").half()
    out = torch.zeros_like(q)
    wide = torch.zeros(3, 264, device="cuda").half()
    for bad in (q.float(), q.bfloat16(), q[:1], q[:, :128], q.t().contiguous().t(), q.cpu()):
        with pytest.raises(ValueError):
            cache.attend(batch, bad, out, stream=here())
        with pytest.raises(ValueError):
            cache.attend(batch, q, bad, stream=here())
    with pytest.raises(gpu_pkg.BackendError, match="16-byte"):
        cache.attend(batch, wide[:, 1:257], out, stream=here())
    with pytest.raises(gpu_pkg.BackendError, match="16-byte"):
        cache.attend(batch, torch.zeros(3 * 260, device="cuda").half().as_strided((2, 256), (260, 1)), out, stream=here())
    with pytest.raises(gpu_pkg.BackendError, match="row stride"):
        cache.append(batch, q, kr[:1].expand(2, 128), kr, out, stream=here())
    with pytest.raises(ValueError):
        cache.batch(lay.len_dev.long(), lay.table_dev)
    with pytest.raises(ValueError):
        cache.batch(lay.len_dev, lay.table_dev, row_off=lay.len_dev, n_rows=2)
    L, b = gpu_pkg.lib(), batch.at
    host = torch.zeros(2, 256).half()                    # pageable memory of the host, through the C entry
    assert L.mynah_b200_kv_attend(cache.h, b, host.data_ptr(), 256, out.data_ptr(), 256, 1) == -1
    assert b"device" in L.mynah_b200_last_error()
    assert L.mynah_b200_kv_attend(cache.h, b, q.data_ptr(), 255, out.data_ptr(), 256, 1) == -1
    assert L.mynah_b200_kv_attend(cache.h, None, q.data_ptr(), 256, out.data_ptr(), 256, 1) == -1
    cache.sync(here())
    assert (out == 0).all()
    cache.attend(cache.batch(lay.len_dev[:0], lay.table_dev[:0]), q, out, stream=here())      # no sequences: nothing happens
    cache.sync(here())
    assert (out == 0).all()


@pytest.mark.parametrize("kind,dim", [("chunk", 128), ("chunk", 64), ("chunk", 48), ("step", 128), ("step", 64)])
def test_long_sums_of_f32_rows(gpu_pkg, kind, dim):
    # Values that share a mean, so that their sum grows with every key. A product's sum is cut, not rounded: a loss of 2^-23 at most and of
    # half as much on average, and half of that again while the sum grows to its end. With at most 10 such cuts (8 of 16 keys, and two small
    # products between them) before a sum is put away: 10 * 2^-23 / 4 = 3e-7. Scores of |s| <= 4 that are off by D / 16 cuts each on their way
    # up, 8 * 2^-24 * 4 / 2 = 1e-6 of a weight at most, average over the keys; 32-bit sums of 64 tiles: 2^-24 * sqrt(64). Together below 1e-6; a
    # sum that stays in the tensor core for 8192 keys loses 512 * 2 * 2^-25 = 3e-5.
    lay = P.Layout([8192, 8190], 64, [400, 150]) if kind == "chunk" else P.Layout([8192] * 40, 64)
    heads = 40 if kind == "chunk" else 4                  # (so many that no kernel splits the keys)
    cache, k, v = filled(gpu_pkg, lay, heads, heads, dim, "f32")
    v.copy_((1 + randn(7, *v.shape)).to(v.dtype))
    q = 0.5 * randn(3, lay.n_rows, heads * dim)
    out = torch.zeros_like(q)
    cache.attend(lay.batch(cache), q, out, stream=here())
    cache.sync(here())
    some = [0, heads // 2, heads - 1]
    for s in range(0, len(lay.lens), 13):
        n, m, at = lay.lens[s], lay.rows[s], lay.begin[s]
        keys, values = (P.keys_of(p, lay, s, list(range(n)))[:, some].transpose(0, 1) for p in (k, v))
        pick = slice(at, at + m)
        scores = q[pick].double().reshape(m, heads, dim)[:, some].transpose(0, 1) @ keys.transpose(1, 2) / dim ** 0.5
        scores.masked_fill_(torch.arange(n, device="cuda") > torch.arange(n - m, n, device="cuda")[:, None], -float("inf"))
        want = (torch.softmax(scores, -1) @ values).transpose(0, 1)
        got = out[pick].double().reshape(m, heads, dim)[:, some]
        assert (got - want).norm() <= 1e-6 * want.norm()


@pytest.mark.parametrize("more", [["--T", "1"], ["--T", "70", "--rows", "f32", "--kv-heads", "2"], ["--T", "5", "--rows", "f16", "--dim", "64", "--window", "100", "--sinks", "3"]])
def test_kernel_case(gpu_pkg, more):
    got = subprocess.run([sys.executable, os.path.join(os.path.dirname(gpu_pkg.__file__), "kernel_case.py"), "kv", "--batch", "3", "--keys", "333", "--iters", "1"] + more,
                         capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, got.stderr
    said = json.loads(got.stdout)
    assert said["kernel"] == "kv" and 0 < said["append_ms"] < 100 and 0 < said["attend_ms"] < 100


# ------------------------------------------------------------------------------------------------------------ the ends of what is allowed
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("rows", [None, [200, 300, 1]])
@pytest.mark.parametrize("window,sinks", [(MOST, 0), (MOST, MOST), (1, MOST), (1, MOST - 31), (2, 2 ** 26 + 1), (1, 0)])
def test_largest_windows_and_sinks(gpu_pkg, rows, window, sinks):
    lay = P.Layout([200, 700, 1], 16, rows)
    for dim, fmt in ((64, "bf16"), (128, "f32")):
        _, q, got = attend_case(gpu_pkg, lay, 4, 2, dim, fmt, window=window, n_sinks=sinks)
        if window + sinks > 700:                          # everything in front is seen, as without a window
            cache, _, _ = filled(gpu_pkg, lay, 4, 2, dim, fmt)
            plain = torch.full_like(q, 7.0)
            cache.attend(lay.batch(cache), q, plain, stream=here())
            cache.sync(here())
            assert torch.allclose(plain.float(), got.float(), rtol=0.02, atol=0.02)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lens,rows", [([5000, 40, 0], None), ([300] * 60, None), ([3000, 40], [130, 40]), ([800, 700, 900], [700, 650, 900])])
def test_attend_in_place(gpu_pkg, fmt, lens, rows):
    """out may be q: with few blocks, whose parts several CTAs share, and with many."""
    lay = P.Layout(lens, 16, rows, extra_rows=3)
    for heads, kv_heads, dim in ((8, 2, 64), (32, 8, 128), (40, 1, 128)):
        cache, _, _ = filled(gpu_pkg, lay, heads, kv_heads, dim, fmt)
        q = randn(3, lay.n_rows, heads * dim).to(P.ROWS[fmt])
        out, same = torch.zeros_like(q), q.clone()
        out[lay.real:] = q[lay.real:]
        cache.attend(lay.batch(cache), q, out, stream=here())
        cache.attend(lay.batch(cache), same, same, stream=here())
        cache.sync(here())
        assert torch.equal(out, same)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dim,heads", [(128, 1), (128, 4), (64, 1), (32, 8)])
def test_chunk_clusters_of_many_sequences(gpu_pkg, fmt, dim, heads):
    """More sequences than lanes, few blocks: clusters, whose CTAs share long blocks and leave short ones to the first of them."""
    rows = [(i * 5) % 9 for i in range(37)]
    lens = [r + (0 if i % 3 else 1700 + 90 * i) for i, r in enumerate(rows)]
    attend_case(gpu_pkg, P.Layout(lens, 16, rows, extra_rows=5), heads, 1, dim, fmt)
    attend_case(gpu_pkg, P.Layout(lens, 16, rows), heads, 1, dim, fmt, window=700, n_sinks=150)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("rows", [None, [150, 300]])
def test_rows_far_apart(gpu_pkg, fmt, rows):
    """Rows of a wider tensor, in and out: what lies between them stays."""
    lay = P.Layout([400, 310], 16, rows)
    cache, k, v = filled(gpu_pkg, lay, 6, 2, 48, fmt)
    wide = randn(3, lay.n_rows, 288 * 3 + 8).to(P.ROWS[fmt])
    q, out = wide[:, 288:576], torch.full_like(wide, 7.0)
    cache.attend(lay.batch(cache), q, out[:, 576:864], stream=here())
    cache.sync(here())
    want, bound = P.attend(lay, q.contiguous(), k, v, 2, fmt=fmt)
    P.check(out[:, 576:864], want, bound)
    assert (out[:, :576] == 7).all() and (out[:, 864:] == 7).all()


def test_largest_values(gpu_pkg):
    """The largest finite numbers of the rows' type go into the cache as they are (f16: below 65504)."""
    for fmt, top in (("bf16", torch.finfo(torch.bfloat16).max), ("f16", 65472.0), ("f32", 65472.0)):
        lay = P.Layout([3], 8, [3])
        cache, k, v = filled(gpu_pkg, lay, 2, 2, 16, fmt)
        x = torch.tensor([top, -top, 0.0, 1.0], device="cuda").repeat(8)[None].repeat(3, 1).to(P.ROWS[fmt])
        out = torch.zeros_like(x)
        cache.append(lay.batch(cache), x, x, x, out, stream=here())
        cache.sync(here())
        assert torch.equal(out, x)
        for pool in (k, v):
            assert torch.equal(P.keys_of(pool, lay, 0, [0, 1, 2]).reshape(3, 32), x.double())


FIRST = """
import importlib.util, os, sys
spec = importlib.util.spec_from_file_location("mynah_asr_b200", sys.argv[1], submodule_search_locations=[os.path.dirname(sys.argv[1])])
pkg = importlib.util.module_from_spec(spec); sys.modules["mynah_asr_b200"] = pkg; spec.loader.exec_module(pkg)
import torch
for fmt, t in ((pkg.F32, torch.float32), (pkg.BF16, torch.bfloat16)):
    for dim in (64, 128):
        cache = pkg.KvCache(4, 2, dim, 16, 64, fmt=fmt)
        table = torch.arange(64, dtype=torch.int32, device="cuda").reshape(2, 32)
        lens = torch.full((2,), 300, dtype=torch.int32, device="cuda")
        off = torch.tensor([0, 40, 80], dtype=torch.int32, device="cuda")
        x = torch.randn(80, 8 * dim, device="cuda").to(t)
        q, k, v = x[:, :4 * dim], x[:, 4 * dim:6 * dim], x[:, 6 * dim:]
        turned, a, b = (torch.zeros(80, 4 * dim, device="cuda", dtype=t) for _ in range(3))
        batch, step = cache.batch(lens, table, row_off=off, n_rows=80), cache.batch(lens, table)
        def calls(out):
            s = torch.cuda.current_stream().cuda_stream
            cache.append(batch, q, k, v, turned, stream=s)
            cache.attend(batch, turned, out, stream=s)
            cache.attend(step, turned, out, stream=s)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            calls(a)
        graph.replay()
        torch.cuda.synchronize()
        calls(b)
        torch.cuda.synchronize()
        cache.sync()
        assert torch.equal(a, b) and a.abs().sum() > 0
print("same")
"""


def test_first_calls_of_a_process_are_captured(gpu_pkg):
    got = subprocess.run([sys.executable, "-c", FIRST, gpu_pkg.__file__], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "same" in got.stdout, got.stderr


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dim,window,sinks", [(64, 0, 0), (128, 0, 0), (64, 200, 5), (128, 333, 70)])
def test_chunk_more_blocks_than_places(gpu_pkg, fmt, dim, window, sinks):
    """More blocks than run at a time: the longest first, then there and back. Sequences without rows, with more rows than keys, alike ones."""
    rows = [640, 1, 0, 640, 129, 900, 700, 640, 128, 64, 257, 500, 0, 333, 640]
    lens = [640, 700, 50, 640, 2000, 900, 300, 800, 1500, 64, 1280, 500, 0, 0, 640]
    attend_case(gpu_pkg, P.Layout(lens, 32, rows, extra_rows=9), 16, 16, dim, fmt, window=window, n_sinks=sinks)
    attend_case(gpu_pkg, P.Layout(lens[::-1], 32, rows[::-1]), 20, 5, dim, fmt, window=window, n_sinks=sinks)
