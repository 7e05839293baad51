// Attention over a paged cache in its plainest form: a warp per row and head, keys one after the other with the running maximum
// and sum of their softmax.
#include "kv.h"
#include <cuda_bf16.h>

namespace mb {

template <int FMT>
__device__ __forceinline__ float kp_row(const void *p, int64_t i) {
    if (FMT == KV_F32) return static_cast<const float *>(p)[i];
    if (FMT == KV_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

template <int FMT>
__global__ void __launch_bounds__(256)
kv_plain_kernel(const KvArgs a) {
    const int lane = threadIdx.x & 31;
    chain_trigger();
    chain_wait();
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int row = (int)(unit / a.H), h = (int)(unit % a.H);
    if (unit == 0 && a.row_off) kv_look_over(a, lane);
    if (row >= a.n_rows) return;
    const int seq = kv_find_seq(a, row, lane);
    if (seq < 0) return;
    KvSeq s;
    if (!kv_seq(a.row_off, a.kv_len, seq, a.n_rows, kv_capacity(a), &s) || row < s.begin || row >= s.begin + s.n) {
        if (lane == 0) atomicExch(a.status, ST_PAGE);
        return;
    }
    const int pos = s.len - s.n + (row - s.begin);
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
    for (int i = 0; i < 4; i++) {
        const int e = lane + 32 * i;
        q[i] = e < a.D ? kp_row<FMT>(a.q, row * a.ldq + (int64_t)h * a.D + e) : 0.f;
    }
    for (int j = 0; j <= pos; j++) {
        if (!kv_sees(pos, j, a.window, a.sinks)) continue;
        const size_t at = kv_row(a, kv_page(a, seq, j >> a.page_shift), h / a.G, j & ((1 << a.page_shift) - 1)) * a.D;
        constexpr int CF = FMT == KV_BF16 ? KV_BF16 : KV_F16;
        float d = 0.f;
        for (int i = 0; i < 4; i++) if (lane + 32 * i < a.D) d = fmaf(q[i], kp_row<CF>(a.k, at + lane + 32 * i), d);
        d = warp_sum(d) * a.scale;
        const float m2 = fmaxf(m, d), c = expf(m - m2), w = expf(d - m2);
        l = l * c + w;
        for (int i = 0; i < 4; i++) o[i] = o[i] * c + (lane + 32 * i < a.D ? w * kp_row<CF>(a.v, at + lane + 32 * i) : 0.f);
        m = m2;
    }
    for (int i = 0; i < 4; i++) {
        const int e = lane + 32 * i;
        if (e >= a.D) continue;
        const float v = l > 0.f ? o[i] / l : 0.f;
        const int64_t at = row * a.ldo + (int64_t)h * a.D + e;
        if (FMT == KV_F32) static_cast<float *>(a.out)[at] = v;
        else if (FMT == KV_F16) static_cast<__half *>(a.out)[at] = __float2half_rn(v);
        else static_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
    }
}

int kv_attend_plain(const KvArgs &a, int fmt, cudaStream_t st) {
    const int64_t blocks = ((int64_t)a.n_rows * a.H + 7) / 8;
    if (blocks > 0x7fffffff) { set_error("kv_attend: too many rows in one call"); return -1; }
    auto kernel = fmt == KV_F32 ? kv_plain_kernel<KV_F32> : fmt == KV_F16 ? kv_plain_kernel<KV_F16> : kv_plain_kernel<KV_BF16>;
    MB_CUDA(launch_kernel(kernel, dim3((unsigned)blocks), dim3(256), 0, st, true, 1, a));
    note_launch();
    return 0;
}

}  // namespace mb
