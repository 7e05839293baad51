// Paged key/value cache of one decoder layer: what the kernels of kv_append.cu, kv_step.cu and kv_chunk.cu get.
#pragma once
#include <cuda_bf16.h>

#include "kernels.h"
#include "kv_index.h"

namespace mb {

enum { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };       // rows; the cache holds f16 for the first two, bf16 for the third

// Positions of a sequence: sums with a window, a tile or a page stay in 32 bits, and a block's work within the kernels' limit on waits
static constexpr int KV_MOST = 1 << 26;
// Sequences of a call: what a warp that looks for its work passes over stays within the limit on waits, too
static constexpr int KV_MOST_SEQ = 1 << 16;

// Pools are [page][kv head][slot][D], 16 bits a value: the keys of one head in one page are one run of memory.
struct KvArgs {
    int H, Hkv, G, D;                                // G = H / Hkv query heads share a kv head
    int page_shift, n_pages;
    int window, sinks;
    float scale2;                                    // of scores, for powers of two
    uint16_t *k, *v;                                 // pools
    int *status;                                     // bits 1 << ST_...
    // the call
    int n_seq, n_rows, max_pages;
    const int *row_off, *kv_len, *table;
    const void *q;
    void *out;
    int64_t ldq, ldo;                                // row strides in values
};
struct KvAppendArgs {
    KvArgs a;
    const void *k_rows, *v_rows;
    int64_t ldk, ldv;
    const float *q_norm, *k_norm;                    // [D] or null
    float eps;
    const double *turns;                             // [rot / 2]: turns of a pair per position
    int rot, interleaved;
};

#ifdef __CUDACC__
// ---- distributed shared memory of a cluster
__device__ __forceinline__ uint32_t kv_peer(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 kv_peer4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float2 kv_peer2(uint32_t addr) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void kv_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// ---- small arithmetic
__device__ __forceinline__ float kv_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A running maximum is that of the scores as the products leave them, -infinity before the first key, and an exponent is (x - m) scale2: the
// difference of neighbours is exact, where x scale2 - m scale2 has lost its digits for scores of 2^24 and more. What was summed under the
// maximum m counts 2^((m - top) scale2) under a larger one.
__device__ __forceinline__ float kv_weight(float m, float top, float scale2) { return m == top ? 1.f : kv_ex2((m - top) * scale2); }
// The sum of a row's probabilities, of which the largest is not small: where it is nothing or no number, the scores were not finite
__device__ __forceinline__ bool kv_sound(float l) { return l > 0.f && l < INFINITY; }
// Near 0, x scale2 + kv_base(m) is the same in one operation, to 2^-14 of a probability: less than the rounding of 16-bit rows (16384 bf16 rows 2012
// us, with the difference for all 2044)
__device__ __forceinline__ float kv_base(float m, float scale2, float up) { return m == -INFINITY ? up : fmaf(-m, scale2, up); }
__device__ __forceinline__ bool kv_far(float base) { return !(fabsf(base) < 1024.f); }
template <bool BF>
__device__ __forceinline__ uint32_t kv_pack(float x, float y) {
    if (BF) { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t *>(&h); }
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// Two results. They are averages, so what rounding has brought beyond the type's largest number is that number (a NaN stays one)
template <bool BF>
__device__ __forceinline__ uint32_t kv_pack_result(float x, float y) {
    uint32_t r;
    if (BF) asm("cvt.rn.satfinite.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(x), "f"(y));
    else asm("cvt.rn.satfinite.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(x), "f"(y));
    return r;
}
// x, y as f16 pairs: hi and what it leaves. The rest stays unscaled (it may be subnormal): both products go into one accumulator.
__device__ __forceinline__ void kv_split(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
// two f32 operations in one instruction
__device__ __forceinline__ float2 kv_twice(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 kv_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 kv_mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmul.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 kv_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// ---- what a kernel has found: a bit of the handle's word for each code, so that none hides another
__device__ __forceinline__ void kv_report(const KvArgs &a, int code) { atomicOr(a.status, 1 << code); }
// ---- tables
__device__ __forceinline__ int64_t kv_capacity(const KvArgs &a) { return (int64_t)a.max_pages << a.page_shift; }
// Index of a cache row (one head at one slot)
__device__ __forceinline__ size_t kv_row(const KvArgs &a, int page, int head, int slot) {
    return ((((size_t)page * a.Hkv + head) << a.page_shift) + slot);
}
// The sequence that row r belongs to, found by a whole warp: the last s with row_off[s] <= r; -1 where there is none, or the row lies
// behind the last sequence. Each round looks at 32 places of what is left.
__device__ __forceinline__ int kv_find_seq(const KvArgs &a, int r, int lane) {
    if (!a.row_off) return r < a.n_seq ? r : -1;
    int lo = 0, hi = a.n_seq + 1;                    // the answer lies in [lo, hi)
    bool first = true;
    while (first || hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned below = __ballot_sync(0xffffffffu, at < hi && a.row_off[at < hi ? at : lo] <= r);
        if (below == 0) return -1;
        lo += (31 - __clz(below)) * step;
        if (hi > lo + step) hi = lo + step;
        first = false;
    }
    return lo < a.n_seq ? lo : -1;
}
// Reports sequences whose tables contradict the call (rows are found from the offsets, so a row may miss that they decrease): the warp's share of
// them, one of `of`
__device__ __forceinline__ void kv_look_over(const KvArgs &a, int lane, int which, int of) {
    bool bad = false;
    for (int64_t s = (int64_t)which * 32 + lane; s < a.n_seq; s += (int64_t)of * 32) {
        KvSeq q;
        bad |= !kv_seq(a.row_off, a.kv_len, (int)s, a.n_rows, kv_capacity(a), &q);
    }
    if (bad) kv_report(a, ST_PAGE);
}
#endif

int kv_append(const KvAppendArgs &a, int fmt, cudaStream_t st);
// Attention of one row per sequence, and of many. Maps of the two pools as [rows][D] with boxes of 64 columns and kv_box slots (prompts:
// box_rows, a page or 32 of them).
int kv_box(int D, int page_size);
int kv_step(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, int fmt, cudaStream_t st);
// 16-bit query rows as [rows][H][D]: boxes of 64 columns, G heads and 128 / G rows
bool kv_rows_map(CUtensorMap *m, const KvArgs &a, bool bf);
int kv_chunk(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, int box_rows, int fmt, cudaStream_t st);

}  // namespace mb
