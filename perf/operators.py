"""The operators of a text decoder's attention over a paged key/value cache, as cases that can be timed.

  append  the rows of a step or of prompts go into the cache: root-mean-square norm of every query and key head, rotation by
          the position, keys and values into the pages of their sequences (KvCache.append)
  step    attention of one new row per sequence over the sequence's pages (KvCache.attend)
  chunk   attention of many rows per sequence, prompts or pieces of prompts behind cached keys (KvCache.attend)

A case is a dict of plain values. Heads: `heads` query heads share `kv_heads` key/value heads of `dim` values. `fmt` is the type
of the rows; the cache holds f16 for f32 and f16 rows and bf16 for bf16 rows. `seqs` sequences have lengths spread over
[lo, hi] (and new rows over [rows_lo, rows_hi]); `pad` sequences or rows more stand empty behind them, as in a captured graph
of a fixed size. window > 0: a row at position p sees the positions above p - window and the first `sinks` ones.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _package():
    if "mynah_asr_b200" not in sys.modules:
        folder = os.path.join(os.getcwd(), "mynah-asr_b200")
        spec = importlib.util.spec_from_file_location("mynah_asr_b200", os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        sys.modules["mynah_asr_b200"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["mynah_asr_b200"])
    return sys.modules["mynah_asr_b200"]


def _case(kind, heads, kv_heads, dim, fmt, page, seqs, lo, hi, rows_lo=1, rows_hi=1, pad=0, window=0, sinks=0, **more):
    return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, fmt=fmt, page=page, seqs=seqs, lo=lo, hi=hi, rows_lo=rows_lo,
                rows_hi=rows_hi, pad=pad, window=window, sinks=sinks, **more)


def listed():
    rope = dict(rotary=128, interleaved=False, theta=1e6, norm=True, fused=True)
    return [
        # one user's next token: the smallest append there is, latency alone
        dict(_case("append", 16, 8, 128, "bf16", 16, 1, 700, 700, **rope), name="append_one"),
        # a server's step: the next token of 120 users in a graph captured for 128
        dict(_case("append", 32, 8, 128, "bf16", 16, 120, 5, 3000, pad=8, **rope), name="append_step"),
        # ragged transcripts behind a decoder with the heads of this repository's small models, f32 rows, rotated in part
        dict(_case("append", 8, 8, 64, "f32", 32, 23, 200, 1900, 3, 1500, pad=5, rotary=32, interleaved=True, theta=1e4, norm=False, fused=False),
             name="append_ragged"),
        # a recording's worth of context as one prompt: the largest append
        dict(_case("append", 32, 8, 128, "bf16", 64, 1, 32768, 32768, 32768, 32768, **rope), name="append_prompt"),
        # one user's next token
        dict(_case("step", 16, 8, 128, "bf16", 16, 1, 700, 700), name="step_one"),
        # one user with hours of context
        dict(_case("step", 32, 8, 128, "bf16", 64, 1, 131071, 131071), name="step_long"),
        # a server's step over ragged contexts
        dict(_case("step", 32, 8, 128, "bf16", 16, 60, 40, 9000, pad=4), name="step_batch"),
        # captioning without end: a window and the first tokens, f32 rows, the pages in between given back
        dict(_case("step", 8, 8, 64, "f32", 32, 200, 300, 20000, window=1000, sinks=4), name="step_window"),
        # short turns of a dialogue behind their history
        dict(_case("chunk", 32, 8, 128, "bf16", 16, 4, 300, 1500, 5, 61), name="chunk_short"),
        # one long prompt: the largest case
        dict(_case("chunk", 32, 8, 128, "bf16", 64, 1, 16384, 16384, 16384, 16384), name="chunk_long"),
        # ragged transcripts under a window, 64-wide heads
        dict(_case("chunk", 16, 4, 64, "f16", 32, 7, 400, 5000, 301, 4000, pad=9, window=512, sinks=4), name="chunk_window"),
        # the attention decoder's heads on f32 rows, as the resident linears give them
        dict(_case("chunk", 8, 8, 128, "f32", 16, 9, 150, 1700, 40, 1300), name="chunk_f32"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(("append", "step", "chunk"))
    heads, kv_heads = rng.choice(((8, 8), (16, 8), (32, 8), (16, 2), (12, 4), (20, 5), (8, 1), (32, 4)))
    dim = rng.choice((64, 64, 128, 128, 128, 80, 96, 112))
    fmt = rng.choice(("bf16", "bf16", "f16", "f32"))
    page = rng.choice((16, 16, 32, 64, 128))
    window, sinks = (log(64, 2048), rng.choice((0, 1, 4, 16))) if rng.random() < 0.35 else (0, 0)
    pad = rng.choice((0, 0, 1, 7))
    if kind == "append":
        seqs = log(1, 128)
        rows = sorted(log(1, min(8192, 16384 // seqs)) for _ in range(2)) if rng.random() < 0.6 else (1, 1)
        past = log(1, 2000)
        rotary = rng.choice((dim, dim, dim // 2, 0))
        return _case(kind, heads, kv_heads, dim, fmt, page, seqs, rows[1], rows[1] + past, rows[0], rows[1], pad, rotary=rotary,
                     interleaved=rng.random() < 0.3, theta=rng.choice((1e4, 5e5, 1e6)), norm=rng.random() < 0.7, fused=rng.random() < 0.6)
    if kind == "step":
        seqs = log(1, 256)
        lens = sorted(log(1, min(60000, 500000 // seqs // kv_heads)) for _ in range(2))
        return _case(kind, heads, kv_heads, dim, fmt, page, seqs, lens[0], lens[1], 1, 1, pad, window, sinks)
    seqs = log(1, 12)
    rows = sorted(log(1, min(5000, 14000 // seqs)) for _ in range(2))
    past = log(1, 2000)
    return _case(kind, heads, kv_heads, dim, fmt, page, seqs, rows[1], rows[1] + past, rows[0], rows[1], pad, window, sinks)


# ------------------------------------------------------------------------------------------------------------ lengths
def _spread(lo, hi, i, step):
    """The i-th of a row of whole numbers spread over [lo, hi], evenly over their logarithm."""
    u = (0.5 + i * step) % 1.0
    return min(hi, max(lo, int(round(lo * (hi / lo) ** u))))


def _lengths(case):
    """New rows and keys (with the new ones) of every sequence."""
    rows = [_spread(case["rows_lo"], case["rows_hi"], i, 0.618034) for i in range(case["seqs"])]
    lens = [max(r, _spread(case["lo"], case["hi"], i, 0.414214)) for i, r in enumerate(rows)]
    return rows, lens


def _visible(case, n, length):
    """Keys that the last n rows of a sequence of `length` see: pairs of row and key, and keys that any of them sees."""
    w, s = case["window"], case["sinks"]
    if not w:
        return sum(range(length - n + 1, length + 1)), length
    pairs = sum(min(p + 1, w + min(s, max(0, p + 1 - w))) for p in range(length - n, length))
    first = max(0, length - n - w + 1)
    return pairs, length - first + min(s, first)


def work(case):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    rows, lens = _lengths(case)
    size = 4 if case["fmt"] == "f32" else 2
    total = sum(rows)
    if case["kind"] == "append":
        move = total * ((2 * h + 2 * kv) * d * size + 2 * kv * d * 2)
        return {"bytes": move, "flops": total * d * ((6 if case["norm"] else 0) + (3 if case["rotary"] else 0)) * (h + kv)}
    seen = [_visible(case, n, length) for n, length in zip(rows, lens)]
    return {"bytes": 2 * total * h * d * size + sum(k for _, k in seen) * kv * d * 4, "flops": sum(p for p, _ in seen) * 4 * h * d}


# ------------------------------------------------------------------------------------------------------------ inputs
def _make(case, seed):
    """Inputs on the GPU: rows as a decoder's projections give them, caches whose pages lie scattered over a pool."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = TYPES[case["fmt"]]
    ct = torch.bfloat16 if case["fmt"] == "bf16" else torch.float16
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rows, lens = _lengths(case)
    step = case["kind"] == "step" or case["rows_hi"] == 1
    real = sum(rows)
    n_rows = real + case["pad"]
    seqs = case["seqs"] + (case["pad"] if step else 0)
    kv_len = torch.tensor(lens + [0] * (seqs - len(lens)), dtype=torch.int32)
    row_off = torch.tensor([0] + rows, dtype=torch.int32).cumsum(0).to(torch.int32)
    # the pages of a sequence: those of its keys, without the ones that a window has left behind
    most = max(lens)
    table = torch.full((seqs, (most + page - 1) // page + 1), -1, dtype=torch.int32)
    need = []
    for s, (n, length) in enumerate(zip(rows, lens)):
        first = max(0, length - n - case["window"] + 1) if case["window"] else 0
        need += [(s, p) for p in range((length + page - 1) // page) if p * page < case["sinks"] or (p + 1) * page > first]
    n_pages = len(need) + 3
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(int(seed)))[:len(need)].to(torch.int32)
    at = torch.tensor(need, dtype=torch.int64)
    table[at[:, 0], at[:, 1]] = order
    make = lambda *shape: torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)  # noqa: E731
    state = dict(case=case, real=real, most=most, rows_most=max(rows), step=step, n_rows=n_rows, n_pages=n_pages,
                 kv_len=kv_len.cuda(), table=table.cuda(), row_off=None if step else row_off.cuda(),
                 k_pages=make(n_pages, kv, page, d).to(ct), v_pages=make(n_pages, kv, page, d).to(ct))
    if case["kind"] == "append":
        if case["fused"]:                                 # one projection's output
            x = make(n_rows, (h + 2 * kv) * d).to(t)
            state.update(q=x[:, :h * d], k=x[:, h * d:(h + kv) * d], v=x[:, (h + kv) * d:])
        else:
            state.update(q=make(n_rows, h * d).to(t), k=make(n_rows, kv * d).to(t), v=make(n_rows, kv * d).to(t))
        if case["norm"]:
            state.update(q_norm=1 + 0.2 * make(d), k_norm=1 + 0.2 * make(d))
    else:
        sharp = torch.linspace(0.3, 2.5, h, device="cuda")[None, :, None]     # heads that look everywhere and heads that look at little
        state.update(q=(make(n_rows, h, d) * sharp).to(t).reshape(n_rows, h * d))
    state["out"] = torch.zeros(n_rows, h * d, dtype=t, device="cuda")
    return state


def prepare(case, seed):
    state = _make(case, seed)
    if own:
        pkg = _package()
        append = case["kind"] == "append"
        cache = pkg.KvCache(case["heads"], case["kv_heads"], case["dim"], case["page"], state["n_pages"],
                            fmt={"f32": pkg.F32, "f16": pkg.F16, "bf16": pkg.BF16}[case["fmt"]],
                            rotary_dim=case["rotary"] if append else 0, interleaved=append and case["interleaved"],
                            rope_theta=case["theta"] if append else 1e4,
                            q_norm=state["q_norm"].cpu().numpy() if "q_norm" in state else None,
                            k_norm=state["k_norm"].cpu().numpy() if "k_norm" in state else None, norm_eps=EPS,
                            window=case["window"], n_sinks=case["sinks"])
        pools = [torch.as_tensor(p, device="cuda").view(state["k_pages"].dtype) for p in cache.pages()]
        pools[0].copy_(state["k_pages"])
        pools[1].copy_(state["v_pages"])
        state.update(cache=cache, k_pages=pools[0], v_pages=pools[1],
                     batch=cache.batch(state["kv_len"], state["table"], row_off=state["row_off"], n_rows=state["n_rows"]))
    return state


# ------------------------------------------------------------------------------------------------------------ the operators
def run(state):
    append = state["case"]["kind"] == "append"
    if own:
        stream = torch.cuda.current_stream().cuda_stream
        if append:
            state["cache"].append(state["batch"], state["q"], state["k"], state["v"], state["out"], stream=stream)
        else:
            state["cache"].attend(state["batch"], state["q"], state["out"], stream=stream)
    elif append:
        _append(state)
    else:
        _attend(state)
    return (state["out"], state["k_pages"], state["v_pages"]) if append else state["out"]


def _places(state):
    """Sequence, place among its rows and position of every row that belongs to a sequence."""
    row = torch.arange(state["real"], device="cuda")
    if state["step"]:
        return row, torch.zeros_like(row), state["kv_len"][:state["real"]].long() - 1
    off = state["row_off"].long()
    seq = torch.searchsorted(off[1:], row, right=True)
    return seq, row - off[seq], state["kv_len"].long()[seq] - (off[1:] - off[:-1])[seq] + row - off[seq]


def _append(state):
    case, real = state["case"], state["real"]
    d, r = case["dim"], case["rotary"]
    seq, _, pos = _places(state)

    def heads(x, weight):
        x = x[:real].float().reshape(real, -1, d)
        if weight is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
        if not r:
            return x
        freq = case["theta"] ** (torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / -r)
        angle = (pos.double()[:, None] * freq)[:, None, :]
        cos, sin = angle.cos().float(), angle.sin().float()
        y = x.clone()
        a, b = (x[..., 0:r:2], x[..., 1:r:2]) if case["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
        u, w = (y[..., 0:r:2], y[..., 1:r:2]) if case["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
        u.copy_(a * cos - b * sin)
        w.copy_(a * sin + b * cos)
        return y

    page, slot = state["table"][seq, pos // case["page"]].long(), pos % case["page"]
    ct = state["k_pages"].dtype
    state["out"][:real] = heads(state["q"], state.get("q_norm")).reshape(real, -1).to(state["out"].dtype)
    state["k_pages"][page, :, slot] = heads(state["k"], state.get("k_norm")).to(ct)
    state["v_pages"][page, :, slot] = state["v"][:real].reshape(real, -1, d).to(ct)


def _softmax_sum(score, seen, v):
    """softmax(score) v over the last axis where `seen`; 0 where nothing is."""
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, (p @ v) / total, 0.0)


def _attend(state):
    case, real = state["case"], state["real"]
    h, kv, d, w, sinks, n = case["heads"], case["kv_heads"], case["dim"], case["window"], case["sinks"], case["seqs"]
    length = state["kv_len"][:n].long()
    scale = 1 / math.sqrt(d)
    if state["step"]:
        # keys that the new row can see: all, or the first ones and those of the window
        if w:
            near = length[:, None] - w + torch.arange(w, device="cuda")
            first = torch.arange(sinks, device="cuda").expand(n, sinks)
            pos = torch.cat((first, near), 1)
            seen = torch.cat((first < length[:, None], near >= sinks), 1)
        else:
            pos = torch.arange(state["most"], device="cuda").expand(n, -1)
            seen = pos < length[:, None]
        at = pos.clamp(0, state["most"] - 1)
        page, slot = state["table"][:n].long().gather(1, at // case["page"]).clamp_min(0), at % case["page"]
        k, v = (x[page, :, slot].float().transpose(1, 2) for x in (state["k_pages"], state["v_pages"]))
        q = state["q"][:n].float().reshape(n, kv, h // kv, d)
        out = _softmax_sum(scale * (q @ k.transpose(2, 3)), seen[:, None, None], v)
        state["out"][:n] = out.reshape(n, h * d).to(state["out"].dtype)
        return
    seq, place, _ = _places(state)
    off = state["row_off"].long()
    count = off[1:] - off[:-1]
    rank = torch.arange(state["rows_most"], device="cuda")
    q = state["q"][(off[:-1, None] + rank).clamp_max(real - 1)].float().reshape(n, len(rank), kv, h // kv, d)
    j = torch.arange(state["most"], device="cuda")
    p = (length - count)[:, None, None] + rank[:, None]
    seen = (j <= p) & ((j > p - w) | (j < sinks)) if w else j <= p
    page, slot = state["table"].long()[:, j // case["page"]].clamp_min(0), j % case["page"]
    out = torch.empty(real, kv, h // kv, d, device="cuda")
    for i in range(kv):                                   # the scores of all heads at once do not fit the card
        k, v = (x[page, i, slot].float()[:, None] for x in (state["k_pages"], state["v_pages"]))
        o = _softmax_sum(scale * (q[:, :, i].transpose(1, 2) @ k.transpose(2, 3)), seen[:, None], v)
        out[:, i] = o.transpose(1, 2)[seq, place]
    state["out"][:real] = out.reshape(real, h * d).to(state["out"].dtype)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    state = _make(case, seed)
    rows, lens = _lengths(case)
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out, begin = state["out"].double(), 0
    table = state["table"].cpu().long()
    if case["kind"] == "append":
        k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
        for s, (n, length) in enumerate(zip(rows, lens)):
            pos = torch.arange(length - n, length)
            where, slot = table[s, pos // page].cuda(), (pos % page).cuda()
            part = slice(begin, begin + n)
            turn = torch.zeros(n, d // 2, dtype=torch.complex128, device="cuda") + 1
            if case["rotary"]:
                freq = torch.tensor([case["theta"] ** (-2.0 * i / case["rotary"]) for i in range(case["rotary"] // 2)], dtype=torch.float64, device="cuda")
                angle = pos.cuda().double()[:, None] * freq
                turn[:, :case["rotary"] // 2] = torch.complex(torch.cos(angle), torch.sin(angle))
            for name, count, weight in (("q", h, state.get("q_norm")), ("k", kv, state.get("k_norm"))):
                x = state[name][part].double().reshape(n, count, d)
                if weight is not None:
                    x = weight.double() * x / torch.sqrt(x.square().sum(-1, keepdim=True) / d + EPS)
                if case["rotary"]:
                    half = case["rotary"] // 2
                    pairs = list(range(half))
                    one = torch.tensor([2 * i for i in pairs] if case["interleaved"] else pairs, device="cuda")
                    two = one + (1 if case["interleaved"] else half)
                    z = torch.complex(x[..., one], x[..., two]) * turn[:, None, :half]
                    x[..., one], x[..., two] = z.real, z.imag
                if name == "q":
                    out[part] = x.reshape(n, h * d)
                else:
                    k_pages[where, :, slot] = x
            v_pages[where, :, slot] = state["v"][part].double().reshape(n, kv, d)
            begin += n
        return out, k_pages, v_pages
    for s, (n, length) in enumerate(zip(rows, lens)):
        j = torch.arange(length)
        if case["window"]:                                # keys that no row of this sequence sees may have no page
            j = j[(j < case["sinks"]) | (j > length - n - case["window"])]
        where, slot = table[s, j // page].cuda(), (j % page).cuda()
        k, v = state["k_pages"][where, :, slot].double(), state["v_pages"][where, :, slot].double()
        j = j.cuda()
        for lo in range(0, n, 2048):
            hi = min(n, lo + 2048)
            p = torch.arange(length - n + lo, length - n + hi, device="cuda")[:, None]
            hidden = j[None, :] > p
            if case["window"]:
                hidden |= (j[None, :] <= p - case["window"]) & (j[None, :] >= case["sinks"])
            for head in range(h):
                a = state["q"][begin + lo:begin + hi, head * d:(head + 1) * d].double() @ k[:, head * kv // h].T / math.sqrt(d)
                out[begin + lo:begin + hi, head * d:(head + 1) * d] = torch.softmax(a.masked_fill_(hidden, -math.inf), -1) @ v[:, head * kv // h]
        begin += n
    return out
