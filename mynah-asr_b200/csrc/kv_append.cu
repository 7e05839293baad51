// Rows of a decoder layer into its paged cache: for every row and head
//   y = w x / sqrt(mean(x^2) + eps)                               (q and k heads, where a norm is set)
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t), t = p f_i   (the first `rot` values of q and k heads, p the row's position)
// then q heads go to q_out, k and v heads to their slot of the cache, each rounded once.
//
// HBM-bound: every value is read once and written once. A head is spread over D / 8 lanes (rounded up to a power of two), eight
// values each, so that 16-bit rows move by 16-byte accesses; a warp takes a run of a row's heads, all of which turn by the same
// angles: a lane keeps the cosines and sines of its eight values in registers. Sums of squares, norms and rotation are in f32; the
// angle is formed as turns in f64 and reduced there (a position of 10^6 times a frequency near 1 has no correct digit behind the point
// in f32), its sine and cosine then in f32.
#include "kv.h"
#include <cuda_bf16.h>

namespace mb {

template <int FMT> struct KvRow;                     // eight values of a row, and of a 16-bit cache row
template <> struct KvRow<KV_F32> {
    static __device__ __forceinline__ void load(const void *p, int64_t i, float *v) {
        const float4 *s = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
        const float4 a = s[0], b = s[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void store(void *p, int64_t i, const float *v) {
        float4 *d = reinterpret_cast<float4 *>(static_cast<float *>(p) + i);
        d[0] = make_float4(v[0], v[1], v[2], v[3]); d[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
};
__device__ __forceinline__ uint4 kv_pack8(const float *v, bool bf) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (bf) { const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]); r[i] = *reinterpret_cast<const uint32_t *>(&h); }
        else { const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]); r[i] = *reinterpret_cast<const uint32_t *>(&h); }
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
template <bool BF> struct KvRow16 {
    static __device__ __forceinline__ void load(const void *p, int64_t i, float *v) {
        const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + i);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float2 f;
            if (BF) f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w[e]));
            else f = __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
            v[2 * e] = f.x; v[2 * e + 1] = f.y;
        }
    }
    static __device__ __forceinline__ void store(void *p, int64_t i, const float *v) {
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + i) = kv_pack8(v, BF);
    }
};
template <> struct KvRow<KV_F16> : KvRow16<false> {};
template <> struct KvRow<KV_BF16> : KvRow16<true> {};

static constexpr int KA_WARPS = 8, KA_AHEAD = 4;     // head groups that a warp has in flight
// The largest magnitude that a cache value may have: beyond it a bf16 would round to infinity; f16 as the operand planes
static constexpr float KA_BF16_MAX = 3.3895313e38f;

template <int FMT, int LPH>
__global__ void __launch_bounds__(KA_WARPS * 32)
kv_append_kernel(const KvAppendArgs p, int parts, int per_part) {
    constexpr int HPI = 32 / LPH;                    // heads side by side in a warp
    const KvArgs &a = p.a;
    const int lane = threadIdx.x & 31;
    chain_trigger();
    chain_wait();
    const int64_t unit = (int64_t)blockIdx.x * KA_WARPS + (threadIdx.x >> 5);
    const int row = (int)(unit / parts), part = (int)(unit % parts);
    if (unit == 0 && a.row_off) kv_look_over(a, lane);
    if (row >= a.n_rows) return;
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
    if ((unsigned)page >= (unsigned)a.n_pages) {
        if (lane == 0) atomicExch(a.status, ST_PAGE);
        return;
    }
    const int sub = lane / LPH, e0 = (lane % LPH) * 8, half = p.rot / 2;
    const bool on = e0 < a.D;
    float cs[8], sn[8];                              // value i becomes v[i] cs[i] + partner sn[i]
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int e = e0 + i;
        cs[i] = 1.f; sn[i] = 0.f;
        if (e < p.rot) {
            const int f = p.interleaved ? e >> 1 : (e < half ? e : e - half);
            double t = (double)pos * p.turns[f];
            t -= rint(t);
            float sv, cv;
            sincospif(2.f * (float)t, &sv, &cv);
            cs[i] = cv;
            sn[i] = (p.interleaved ? (e & 1) : e >= half) ? sv : -sv;
        }
    }
    const int heads = a.H + 2 * a.Hkv;
    const float top = FMT == KV_BF16 ? KA_BF16_MAX : H16_MAX;
    bool bad = false;
    const int g_end = min((part + 1) * per_part, (heads + HPI - 1) / HPI);
    for (int g0 = part * per_part; g0 < g_end; g0 += KA_AHEAD) {
        float v[KA_AHEAD][8];
#pragma unroll
        for (int u = 0; u < KA_AHEAD; u++) {
            const int h = (g0 + u) * HPI + sub;
#pragma unroll
            for (int i = 0; i < 8; i++) v[u][i] = 0.f;
            if (on && g0 + u < g_end && h < heads) {
                if (h < a.H) KvRow<FMT>::load(a.q, row * a.ldq + h * a.D + e0, v[u]);
                else if (h < a.H + a.Hkv) KvRow<FMT>::load(p.k_rows, row * p.ldk + (h - a.H) * a.D + e0, v[u]);
                else KvRow<FMT>::load(p.v_rows, row * p.ldv + (h - a.H - a.Hkv) * a.D + e0, v[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < KA_AHEAD; u++) {
            const int h = (g0 + u) * HPI + sub;
            if (g0 + u >= g_end) break;              // the same for the whole warp
            float *x = v[u];
            const float *w = h < a.H ? p.q_norm : p.k_norm;
            const bool turns = h < a.H + a.Hkv;      // (v heads pass as they are)
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (turns && w && on) {
                const float r = 1.f / sqrtf(ss / (float)a.D + p.eps);
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] *= r * w[e0 + i];
            }
            if (p.rot) {                             // the same for the whole launch
                float y[8];
                if (p.interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] = x[i ^ 1];
                } else {
                    // value e turns with e + half or e - half: eight values further on a lane boundary, or four (half % 8 is 0 or 4)
                    const bool split = half & 4;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int e = e0 + i, other = e < half ? e + half : e < p.rot ? e - half : e;
                        const float mine = split ? x[i ^ 4] : x[i];
                        y[i] = __shfl_sync(0xffffffffu, mine, (sub * LPH) + ((other >> 3) & (LPH - 1)));
                    }
                }
                if (turns) {
#pragma unroll
                    for (int i = 0; i < 8; i++) x[i] = e0 + i < p.rot ? fmaf(x[i], cs[i], y[i] * sn[i]) : x[i];
                }
            }
            if (!on || h >= heads) continue;
            if (h < a.H) {
#pragma unroll
                for (int i = 0; i < 8; i++) bad |= !(fabsf(x[i]) < (FMT == KV_F32 ? INFINITY : top));
                KvRow<FMT>::store(a.out, row * a.ldo + h * a.D + e0, x);
            } else {
                // the cache holds finite values only: what a mask hides is multiplied by a probability of 0
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const bool fits = fabsf(x[i]) < top;
                    bad |= !fits;
                    x[i] = fits ? x[i] : 0.f;
                }
                const bool key = h < a.H + a.Hkv;
                const size_t at = kv_row(a, page, h - a.H - (key ? 0 : a.Hkv), slot) * a.D + e0;
                *reinterpret_cast<uint4 *>((key ? a.k : a.v) + at) = kv_pack8(x, FMT == KV_BF16);
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
