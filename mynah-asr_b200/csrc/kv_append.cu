// Rows of a decoder layer into its paged cache: for every row and head
//   y = w x / sqrt(mean(x^2) + eps)                               (q and k heads, where a norm is set)
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t), t = p f_i   (the first `rot` values of q and k heads, p the row's position)
// then q heads go to q_out, k and v heads to their slot of the cache, each rounded once.
//
// HBM-bound: every value is read once and written once. A head is spread over D / 8 lanes (rounded up to a power of two), eight values
// each as two quads: where halves turn against one another, lane l of the first rot / 8 holds the values 4 l of both halves, so that a
// pair meets in one lane and nothing but the sum of squares crosses lanes; elsewhere the quads are neighbours. A warp takes a run of a
// row's heads, all of which turn by the same angles: a lane keeps the cosines and sines of its four pairs and its norm weights in
// registers, and has 2 KB of reads in flight. Sums of squares, norms and rotation are in f32; the angle is formed as turns in
// f64 and reduced there (a position of 10^6 times a frequency near 1 has no correct digit behind the point in f32), its sine and
// cosine then in f32.
// Measured (norm and rotation, 32 query and 8 kv heads of 128, bf16): 32768 rows 165 us = 4.9 TB/s, issue slots 62 % and ALU 55 % taken (the
// 64 registers that 32 warps leave spill 36 bytes); 120 rows 4.9 us, one 2.8; 23 sequences of f32 rows, 8 heads of 64, half of each turned, 14.1 us = 3.5 TB/s. With pairs exchanged between
// lanes instead, and all kinds of heads in one loop, the first took 441 us.
#include "kv.h"

namespace mb {

__device__ __forceinline__ float2 ka_unpack(uint32_t u, bool bf) {
    if (bf) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&u));
    return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}
// Four values of a row, as they lie in memory
template <int FMT> struct KaQuad { typedef uint2 type; };
template <> struct KaQuad<KV_F32> { typedef float4 type; };
template <int FMT>
__device__ __forceinline__ void ka_open(const typename KaQuad<FMT>::type &r, float *v) {
    if constexpr (FMT == KV_F32) { v[0] = r.x; v[1] = r.y; v[2] = r.z; v[3] = r.w; }
    else {
        const float2 a = ka_unpack(r.x, FMT == KV_BF16), b = ka_unpack(r.y, FMT == KV_BF16);
        v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
    }
}
template <int FMT>
__device__ __forceinline__ typename KaQuad<FMT>::type ka_close(const float *v) {
    if constexpr (FMT == KV_F32) return make_float4(v[0], v[1], v[2], v[3]);
    else return make_uint2(kv_pack<FMT == KV_BF16>(v[0], v[1]), kv_pack<FMT == KV_BF16>(v[2], v[3]));
}

// The mean of squares, below 2^-126 (where f32 loses digits of it) 0. At 0 and at infinity the factor rsqrt(mean) + (mean - mean) is no
// number, and so are the head's values: out of range, not 0. (Such heads taken again with their values scaled, in the loop or behind it, cost the
// heads of ordinary size 7 to 24 % of 32768 rows' time.)
__device__ __forceinline__ float ka_mean(float squares, float inv_d, float eps) {
    float r;
    asm("fma.rn.ftz.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(squares), "f"(inv_d), "f"(eps));
    return r;
}

static constexpr int KA_WARPS = 8;
// Below what a value lies: from (2 - 2^-8) 2^127 on, halfway behind the largest bf16, and from 65520 on, halfway behind the largest f16, it would
// round to infinity. F32 rows end where the library's operand planes do.
static constexpr float KA_BF16_MAX = 0x1.ffp127f, KA_F16_MAX = 65520.f;

enum { KA_Q, KA_K, KA_V };
// What a lane knows of its row: where its quads begin, cosines and sines of its pairs, the row's slot
struct KaLane {
    int sub, qa, qb;
    bool on, turns;
    float2 cs[2], sn[2], nsn[2];                     // pairs (0, 1) and (2, 3)
};
template <int FMT> struct KaAhead { static constexpr int N = FMT == KV_F32 ? 2 : 4; };   // head groups in flight: 2 KB of a warp's reads

// The heads [h0 + sub, end) of one kind in steps of a warp's heads, from rows at `from` to `to` (elements of a head apart: step)
template <int FMT, int LPH, int KIND>
__device__ __forceinline__ bool ka_heads(const KvAppendArgs &p, const KaLane &w, const char *from, int g, int g_end, int heads, void *to, size_t step,
                                         typename KaQuad<FMT>::type (&in)[KaAhead<FMT>::N][2], bool fetched) {
    typedef typename KaQuad<FMT>::type Quad;
    constexpr int HPI = 32 / LPH, SIZE = FMT == KV_F32 ? 4 : 2, N = KaAhead<FMT>::N;
    constexpr int OUT = KIND == KA_Q ? FMT : FMT == KV_BF16 ? KV_BF16 : KV_F16;
    typedef typename KaQuad<OUT>::type Out;
    const float *norm = KIND == KA_Q ? p.q_norm : KIND == KA_K ? p.k_norm : nullptr;
    const float top = KIND == KA_Q && FMT == KV_F32 ? INFINITY : FMT == KV_BF16 ? KA_BF16_MAX : FMT == KV_F16 ? KA_F16_MAX : H16_MAX;
    float2 wt[4];
    if (KIND != KA_V && norm && w.on) {
        *reinterpret_cast<float4 *>(wt) = *reinterpret_cast<const float4 *>(norm + w.qa);
        *reinterpret_cast<float4 *>(wt + 2) = *reinterpret_cast<const float4 *>(norm + w.qb);
    }
    const float inv_d = 1.f / (float)p.a.D;
    bool bad = false;
    for (; g < g_end; g += N) {
        if (!fetched) {
#pragma unroll
            for (int u = 0; u < N; u++) {
                const int h = (g + u) * HPI + w.sub;
                in[u][0] = in[u][1] = Quad();
                if (w.on && h < heads && g + u < g_end) {
                    const char *s = from + (size_t)h * (p.a.D * SIZE);
                    in[u][0] = *reinterpret_cast<const Quad *>(s + w.qa * SIZE);
                    in[u][1] = *reinterpret_cast<const Quad *>(s + w.qb * SIZE);
                }
            }
        }
        fetched = false;
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int h = (g + u) * HPI + w.sub;
            if (g + u >= g_end) break;               // the same for the whole warp
            float2 x[4];
            ka_open<FMT>(in[u][0], reinterpret_cast<float *>(x));
            ka_open<FMT>(in[u][1], reinterpret_cast<float *>(x + 2));
            if (KIND != KA_V && norm) {              // the same for the whole launch
                float2 s2 = kv_mul2(x[0], x[0]);
#pragma unroll
                for (int i = 1; i < 4; i++) s2 = kv_fma2(x[i], x[i], s2);
                float ss = s2.x + s2.y;
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float mean = ka_mean(ss, inv_d, p.eps), r = rsqrtf(mean) + (mean - mean);
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] = kv_mul2(kv_mul2(x[i], wt[i]), make_float2(r, r));
            }
            if (KIND != KA_V && w.turns) {
                if (p.interleaved) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float c = i & 1 ? w.cs[i >> 1].y : w.cs[i >> 1].x, n = i & 1 ? w.sn[i >> 1].y : w.sn[i >> 1].x, b = x[i].x;
                        x[i].x = fmaf(b, c, -x[i].y * n);
                        x[i].y = fmaf(b, n, x[i].y * c);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float2 b = x[i];
                        x[i] = kv_fma2(b, w.cs[i], kv_mul2(x[i + 2], w.nsn[i]));
                        x[i + 2] = kv_fma2(b, w.sn[i], kv_mul2(x[i + 2], w.cs[i]));
                    }
                }
            }
            if (w.on && h < heads) {
                bool over = false;
#pragma unroll
                for (int i = 0; i < 4; i++) over |= !(fabsf(x[i].x) < top) | !(fabsf(x[i].y) < top);
                if (over) {
                    bad = true;
                    if (KIND != KA_Q) {
                        // the cache holds finite values only: what a mask hides is multiplied by a probability of 0
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            x[i].x = fabsf(x[i].x) < top ? x[i].x : 0.f;
                            x[i].y = fabsf(x[i].y) < top ? x[i].y : 0.f;
                        }
                    }
                }
                char *d = static_cast<char *>(to) + (size_t)h * step * (KIND == KA_Q ? SIZE : 2);
                *reinterpret_cast<Out *>(d + w.qa * (KIND == KA_Q ? SIZE : 2)) = ka_close<OUT>(reinterpret_cast<const float *>(x));
                *reinterpret_cast<Out *>(d + w.qb * (KIND == KA_Q ? SIZE : 2)) = ka_close<OUT>(reinterpret_cast<const float *>(x + 2));
            }
        }
    }
    return bad;
}

// Warp = row x of 8 per block, and the block's part of the row's head groups: q's, then k's, then v's
template <int FMT, int LPH>
__global__ void __launch_bounds__(KA_WARPS * 32, FMT == KV_F32 ? 3 : 4)
kv_append_kernel(const KvAppendArgs p, int per_part) {
    typedef typename KaQuad<FMT>::type Quad;
    constexpr int HPI = 32 / LPH, SIZE = FMT == KV_F32 ? 4 : 2, N = KaAhead<FMT>::N;
    const KvArgs &a = p.a;
    const int lane = threadIdx.x & 31;
    chain_trigger();
    chain_wait();
    const int row = (int)blockIdx.x * KA_WARPS + (int)(threadIdx.x >> 5);
    if (blockIdx.y == 0 && a.row_off) kv_look_over(a, lane, row, (int)gridDim.x * KA_WARPS);
    if (row >= a.n_rows) return;
    KaLane w;
    const int l = lane % LPH;
    w.sub = lane / LPH;
    w.on = l * 8 < a.D;
    w.turns = l * 8 < p.rot;
    w.qa = w.turns && !p.interleaved ? 4 * l : 8 * l;
    w.qb = w.turns && !p.interleaved ? p.rot / 2 + 4 * l : 8 * l + 4;
    const int gq = (a.H + HPI - 1) / HPI, gk = (a.Hkv + HPI - 1) / HPI;
    const int g0 = (int)blockIdx.y * per_part, g1 = g0 + per_part;
    const char *q = static_cast<const char *>(a.q) + row * a.ldq * SIZE, *k = static_cast<const char *>(p.k_rows) + row * p.ldk * SIZE,
               *v = static_cast<const char *>(p.v_rows) + row * p.ldv * SIZE;
    // the first reads are under way while the tables are looked up (rows that turn out to have no place are within the buffers, too)
    Quad in[N][2];
    {
        const int kind = g0 < gq ? KA_Q : g0 < gq + gk ? KA_K : KA_V, g = kind == KA_Q ? g0 : kind == KA_K ? g0 - gq : g0 - gq - gk;
        const int heads = kind == KA_Q ? a.H : a.Hkv, end = min(g1 - g0 + g, kind == KA_Q ? gq : gk);
        const char *from = kind == KA_Q ? q : kind == KA_K ? k : v;
#pragma unroll
        for (int u = 0; u < N; u++) {
            const int h = (g + u) * HPI + w.sub;
            in[u][0] = in[u][1] = Quad();
            if (w.on && h < heads && g + u < end) {
                const char *s = from + (size_t)h * (a.D * SIZE);
                in[u][0] = *reinterpret_cast<const Quad *>(s + w.qa * SIZE);
                in[u][1] = *reinterpret_cast<const Quad *>(s + w.qb * SIZE);
            }
        }
    }
    const int seq = kv_find_seq(a, row, lane);
    if (seq < 0) return;                             // behind the last sequence: everything stays as it was
    KvSeq s;
    if (!kv_seq(a.row_off, a.kv_len, seq, a.n_rows, kv_capacity(a), &s) || row < s.begin || row >= s.begin + s.n) {
        if (lane == 0) kv_report(a, ST_PAGE);
        return;
    }
    const int pos = s.len - s.n + (row - s.begin);
    if (pos < 0) return;                             // in front of the first position
    const int page = a.table[(size_t)seq * a.max_pages + (pos >> a.page_shift)], slot = pos & ((1 << a.page_shift) - 1);
    if (w.turns) {
        float c4[4], s4[4];                          // of the lane's pairs: values (i, i + 4), or (2 i, 2 i + 1) where interleaved
#pragma unroll
        for (int i = 0; i < 4; i++) {
            double t = (double)pos * p.turns[4 * l + i];
            t -= rint(t);
            sincospif(2.f * (float)t, &s4[i], &c4[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            w.cs[i] = make_float2(c4[2 * i], c4[2 * i + 1]);
            w.sn[i] = make_float2(s4[2 * i], s4[2 * i + 1]);
            w.nsn[i] = make_float2(-s4[2 * i], -s4[2 * i + 1]);
        }
    }
    if ((unsigned)page >= (unsigned)a.n_pages) {
        if (lane == 0) kv_report(a, ST_PAGE);
        return;
    }
    const size_t step = (size_t)a.D << a.page_shift, base = kv_row(a, page, 0, slot) * a.D;
    bool bad = false, fetched = true;
    if (g0 < gq) {
        bad |= ka_heads<FMT, LPH, KA_Q>(p, w, q, g0, min(g1, gq), a.H, static_cast<char *>(a.out) + row * a.ldo * SIZE, (size_t)a.D, in, fetched);
        fetched = false;
    }
    if (g0 < gq + gk && g1 > gq) {
        bad |= ka_heads<FMT, LPH, KA_K>(p, w, k, max(g0 - gq, 0), min(g1 - gq, gk), a.Hkv, a.k + base, step, in, fetched);
        fetched = false;
    }
    if (g1 > gq + gk) bad |= ka_heads<FMT, LPH, KA_V>(p, w, v, max(g0 - gq - gk, 0), min(g1 - gq - gk, gk), a.Hkv, a.v + base, step, in, fetched);
    if (bad) kv_report(a, ST_RANGE);
}

template <int FMT>
static int append_fmt(const KvAppendArgs &p, cudaStream_t st) {
    const KvArgs &a = p.a;
    const int lph = a.D <= 16 ? 2 : a.D <= 32 ? 4 : a.D <= 64 ? 8 : 16, hpi = 32 / lph;
    const int groups = cdiv(a.H, hpi) + 2 * cdiv(a.Hkv, hpi);
    // A warp takes a whole row where there are rows enough to fill the SMs (32 warps each), a part of one otherwise
    const int64_t want = 32ll * device_sm_count();
    int parts = (int)((want + a.n_rows - 1) / a.n_rows);
    if (parts > groups) parts = groups;
    const int per_part = cdiv(groups, parts);
    parts = cdiv(groups, per_part);
    auto kernel = lph == 2 ? kv_append_kernel<FMT, 2> : lph == 4 ? kv_append_kernel<FMT, 4> : lph == 8 ? kv_append_kernel<FMT, 8> : kv_append_kernel<FMT, 16>;
    MB_CUDA(launch_kernel(kernel, dim3((unsigned)((a.n_rows - 1) / KA_WARPS + 1), (unsigned)parts), dim3(KA_WARPS * 32), 0, st, true, 1, p, per_part));
    note_launch();
    return 0;
}

int kv_append(const KvAppendArgs &p, int fmt, cudaStream_t st) {
    return fmt == KV_F32 ? append_fmt<KV_F32>(p, st) : fmt == KV_F16 ? append_fmt<KV_F16>(p, st) : append_fmt<KV_BF16>(p, st);
}

}  // namespace mb
