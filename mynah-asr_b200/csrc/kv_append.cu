// Rows of a decoder layer into its paged cache: for every row and head
//   y = w x / sqrt(mean(x^2) + eps)                               (q and k heads, where a norm is set)
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t), t = p f_i   (the first `rot` values of q and k heads, p the row's position)
// then q heads go to q_out, k and v heads to their slot of the cache, each rounded once.
//
// HBM-bound: every value is read once and written once. A head is spread over D / 8 lanes (rounded up to a power of two), eight values
// each as two quads: where halves turn against one another, lane l of the first rot / 8 holds the values 4 l of both halves, so that a
// pair meets in one lane and nothing but the sum of squares crosses lanes; elsewhere the quads are neighbours. A warp takes a run of a
// row's heads, all of which turn by the same angles: a lane keeps the cosines and sines of its four pairs and its norm weights in
// registers, and has KA_AHEAD head groups in flight. Sums of squares, norms and rotation are in f32; the angle is formed as turns in
// f64 and reduced there (a position of 10^6 times a frequency near 1 has no correct digit behind the point in f32), its sine and
// cosine then in f32.
#include "kv.h"
#include <cuda_bf16.h>

namespace mb {

__device__ __forceinline__ uint32_t ka_pack(float x, float y, bool bf) {
    if (bf) { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t *>(&h); }
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
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
    else return make_uint2(ka_pack(v[0], v[1], FMT == KV_BF16), ka_pack(v[2], v[3], FMT == KV_BF16));
}

static constexpr int KA_WARPS = 8, KA_AHEAD = 4;     // head groups that a warp has in flight
// The largest magnitude that a cache value may have: beyond it a bf16 would round to infinity; f16 as the operand planes
static constexpr float KA_BF16_MAX = 3.3895313e38f;

template <int FMT, int LPH>
__global__ void __launch_bounds__(KA_WARPS * 32)
kv_append_kernel(const KvAppendArgs p, int parts, int per_part) {
    typedef typename KaQuad<FMT>::type Quad;
    constexpr int HPI = 32 / LPH, SIZE = FMT == KV_F32 ? 4 : 2;        // heads side by side in a warp; bytes of a row's value
    const KvArgs &a = p.a;
    const int lane = threadIdx.x & 31;
    chain_trigger();
    chain_wait();
    const int64_t unit = (int64_t)blockIdx.x * KA_WARPS + (threadIdx.x >> 5);
    const int row = (int)(unit / parts), part = (int)(unit % parts);
    if (unit == 0 && a.row_off) kv_look_over(a, lane);
    if (row >= a.n_rows) return;
    const int sub = lane / LPH, l = lane % LPH;
    const bool on = l * 8 < a.D, pairs = !p.interleaved && l * 8 < p.rot;
    const int qa = pairs ? 4 * l : 8 * l, qb = pairs ? p.rot / 2 + 4 * l : 8 * l + 4;         // first values of the lane's quads
    const int heads = a.H + 2 * a.Hkv, g0 = part * per_part, g_end = min(g0 + per_part, (heads + HPI - 1) / HPI);
    const char *q = static_cast<const char *>(a.q) + row * a.ldq * SIZE, *k = static_cast<const char *>(p.k_rows) + row * p.ldk * SIZE,
               *v = static_cast<const char *>(p.v_rows) + row * p.ldv * SIZE;
    Quad in[KA_AHEAD][2];
    auto fetch = [&](int g) {
#pragma unroll
        for (int u = 0; u < KA_AHEAD; u++) {
            const int h = (g + u) * HPI + sub;
            if (on && g + u < g_end && h < heads) {
                const char *s = h < a.H ? q + (size_t)h * a.D * SIZE : h < a.H + a.Hkv ? k + (size_t)(h - a.H) * a.D * SIZE : v + (size_t)(h - a.H - a.Hkv) * a.D * SIZE;
                in[u][0] = *reinterpret_cast<const Quad *>(s + qa * SIZE);
                in[u][1] = *reinterpret_cast<const Quad *>(s + qb * SIZE);
            } else {
                in[u][0] = in[u][1] = Quad();
            }
        }
    };
    fetch(g0);                                       // (rows that turn out to have no place are within the buffers, too)
    float wq[8], wk[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int e = (i < 4 ? qa : qb - 4) + i;
        wq[i] = p.q_norm && on ? p.q_norm[e] : 1.f;
        wk[i] = p.k_norm && on ? p.k_norm[e] : 1.f;
    }
    const int seq = kv_find_seq(a, row, lane);
    if (seq < 0) return;                             // behind the last sequence: everything stays as it was
    KvSeq s;
    if (!kv_seq(a.row_off, a.kv_len, seq, a.n_rows, kv_capacity(a), &s) || row < s.begin || row >= s.begin + s.n) {
        if (lane == 0) atomicExch(a.status, ST_PAGE);
        return;
    }
    const int pos = s.len - s.n + (row - s.begin);
    if (pos < 0) return;                             // in front of the first position
    const int page = a.table[(size_t)seq * a.max_pages + (pos >> a.page_shift)], slot = pos & ((1 << a.page_shift) - 1);
    float cs[4], sn[4];                              // of the lane's pairs: values (i, i + 4), or (2 i, 2 i + 1) where interleaved
    if (p.rot) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            cs[i] = 1.f; sn[i] = 0.f;
            if (l * 8 < p.rot) {
                double t = (double)pos * p.turns[4 * l + i];
                t -= rint(t);
                sincospif(2.f * (float)t, &sn[i], &cs[i]);
            }
        }
    }
    if ((unsigned)page >= (unsigned)a.n_pages) {
        if (lane == 0) atomicExch(a.status, ST_PAGE);
        return;
    }
    const size_t head_step = (size_t)a.D << a.page_shift, base = kv_row(a, page, 0, slot) * a.D;
    char *out = static_cast<char *>(a.out) + row * a.ldo * SIZE;
    const float top = FMT == KV_BF16 ? KA_BF16_MAX : H16_MAX, inv_d = 1.f / (float)a.D;
    bool bad = false;
    for (int g = g0; g < g_end; g += KA_AHEAD) {
        if (g > g0) fetch(g);
#pragma unroll
        for (int u = 0; u < KA_AHEAD; u++) {
            const int h = (g + u) * HPI + sub;
            if (g + u >= g_end) break;               // the same for the whole warp
            float x[8];
            ka_open<FMT>(in[u][0], x);
            ka_open<FMT>(in[u][1], x + 4);
            const bool turns = h < a.H + a.Hkv;      // (v heads pass as they are)
            if (p.q_norm || p.k_norm) {              // the same for the whole launch
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
                for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float r = rsqrtf(fmaf(ss, inv_d, p.eps));
                if (h < a.H ? p.q_norm != nullptr : turns && p.k_norm != nullptr) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] *= r * (h < a.H ? wq[i] : wk[i]);
                }
            }
            if (p.rot && turns) {
                if (p.interleaved) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float c = x[2 * i], d = x[2 * i + 1];
                        x[2 * i] = fmaf(c, cs[i], -d * sn[i]);
                        x[2 * i + 1] = fmaf(c, sn[i], d * cs[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float c = x[i], d = x[i + 4];
                        x[i] = fmaf(c, cs[i], -d * sn[i]);
                        x[i + 4] = fmaf(c, sn[i], d * cs[i]);
                    }
                }
            }
            if (!on || h >= heads) continue;
            if (h < a.H) {
#pragma unroll
                for (int i = 0; i < 8; i++) bad |= !(fabsf(x[i]) < (FMT == KV_F32 ? INFINITY : top));
                char *to = out + (size_t)h * a.D * SIZE;
                *reinterpret_cast<Quad *>(to + qa * SIZE) = ka_close<FMT>(x);
                *reinterpret_cast<Quad *>(to + qb * SIZE) = ka_close<FMT>(x + 4);
            } else {
                // the cache holds finite values only: what a mask hides is multiplied by a probability of 0
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const bool fits = fabsf(x[i]) < top;
                    bad |= !fits;
                    x[i] = fits ? x[i] : 0.f;
                }
                uint16_t *to = (turns ? a.k : a.v) + base + (size_t)(h - a.H - (turns ? 0 : a.Hkv)) * head_step;
                *reinterpret_cast<uint2 *>(to + qa) = ka_close<FMT == KV_BF16 ? KV_BF16 : KV_F16>(x);
                *reinterpret_cast<uint2 *>(to + qb) = ka_close<FMT == KV_BF16 ? KV_BF16 : KV_F16>(x + 4);
            }
        }
    }
    if (bad) atomicExch(a.status, ST_RANGE);
}

template <int FMT>
static int append_fmt(const KvAppendArgs &p, cudaStream_t st) {
    const KvArgs &a = p.a;
    const int lph = a.D <= 16 ? 2 : a.D <= 32 ? 4 : a.D <= 64 ? 8 : 16;
    const int groups = cdiv(a.H + 2 * a.Hkv, 32 / lph);
    // A warp takes a whole row where there are rows enough to fill the SMs (32 warps each), a part of one otherwise
    const int64_t want = 32ll * device_sm_count();
    int parts = (int)((want + a.n_rows - 1) / a.n_rows);
    if (parts > groups) parts = groups;
    const int per_part = cdiv(groups, parts);
    parts = cdiv(groups, per_part);
    const int64_t blocks = ((int64_t)a.n_rows * parts + KA_WARPS - 1) / KA_WARPS;
    if (blocks > 0x7fffffff) { set_error("kv_append: too many rows in one call"); return -1; }
    auto kernel = lph == 2 ? kv_append_kernel<FMT, 2> : lph == 4 ? kv_append_kernel<FMT, 4> : lph == 8 ? kv_append_kernel<FMT, 8> : kv_append_kernel<FMT, 16>;
    MB_CUDA(launch_kernel(kernel, dim3((unsigned)blocks), dim3(KA_WARPS * 32), 0, st, true, 1, p, parts, per_part));
    note_launch();
    return 0;
}

int kv_append(const KvAppendArgs &p, int fmt, cudaStream_t st) {
    return fmt == KV_F32 ? append_fmt<KV_F32>(p, st) : fmt == KV_F16 ? append_fmt<KV_F16>(p, st) : append_fmt<KV_BF16>(p, st);
}

}  // namespace mb
