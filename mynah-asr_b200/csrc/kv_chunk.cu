// Attention of many rows per sequence over the pages of its cache: prompts, or pieces of prompts behind cached keys,
//   o_p = sum_j softmax_j(scale q_p . k_j) v_j  over j <= p, with a window also j > p - window or j < sinks.
//
// Bound by the tensor cores and, as much, by the exponentials (4 D operations and one exponential per pair of row and key). A CTA
// owns one kv head and two tiles of 128 rows: the G query heads of 128 / G positions each (row r is head r % G of position r / G), so
// that short pieces fill a tile and all heads share the keys' tiles. Keys and values come in tiles of 128 by TMA, from their pages
// straight into the swizzled operand layout.
//   tensor memory  S0, S1: scores of the two tiles (128 columns each; the probabilities overwrite them as 16-bit operands),
//                  O0, O1: results (D columns each)
//   warps          0-3 and 4-7: softmax of tile 0 and 1, a thread per row; 8: TMA; 9: MMA
//   order of MMAs  P0 V(i), S0(i + 1), P1 V(i), S1(i + 1): one tile's exponentials run under the other's products. MMAs run in the
//                  order of their issue, so S(i + 1) does not overwrite the P(i) that P V(i) reads, and whoever sees S(i + 1) finished
//                  finds O at rest.
// The softmax keeps a running maximum per row; O is rescaled only when it has grown by more than 2^8 (what is stale cancels in the
// final division). F32 rows: queries and probabilities as (hi, lo) f16 pairs, two products each.
#include "kv.h"
#include <cuda_bf16.h>

namespace mb {

static constexpr int KC_ROWS = 128, KC_KEYS = 128, KC_HALF = 128 * 128;      // a 128-row x 64-column box of 16-bit values: 16 KB
static constexpr int KC_SOFT = 8, KC_W_TMA = 8, KC_W_MMA = 9, KC_THREADS = 320;
static constexpr int KC_HEAD = 1024;
static constexpr int KC_PART = 6;                    // P V begins when the first 6 x 16 keys' probabilities are there
static constexpr float KC_NONE = -1e30f;             // "maximum" of no keys

template <int DP, int FMT> struct ChunkShape {
    static constexpr int HALVES = DP / 64, PLANES = FMT == KV_F32 ? 2 : 1;
    static constexpr int OPERAND = HALVES * KC_HALF;           // a tile of queries (one plane), of keys, or of values
    static constexpr int Q = 2 * PLANES * OPERAND;
    static constexpr int STAGES = DP == 64 ? 6 : PLANES == 1 ? 5 : 3;
    static constexpr int SMEM = KC_HEAD + Q + STAGES * OPERAND + 1024;
    static_assert(SMEM <= 232448, "shared memory");
    static constexpr int COL_S = 0, COL_O = 256;
};

struct KcPlace { int seq, block; };

__device__ __forceinline__ void kc_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) { tc_mma_f16(d, a, b, idesc, acc); }
__device__ __forceinline__ void kc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void kc_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void kc_st8(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void kc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float kc_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two f32 operations in one instruction
__device__ __forceinline__ float2 kc_fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 kc_add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 ra, rb, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tadd.rn.f32x2 rd, ra, rb;\n\tmov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
// Waits for loads from tensor memory; the values that they bring are not to be touched before (nor their use moved up)
__device__ __forceinline__ void kc_wait_ld32(float *x) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7]), "+f"(x[8]), "+f"(x[9]), "+f"(x[10]),
                   "+f"(x[11]), "+f"(x[12]), "+f"(x[13]), "+f"(x[14]), "+f"(x[15]), "+f"(x[16]), "+f"(x[17]), "+f"(x[18]), "+f"(x[19]), "+f"(x[20]),
                   "+f"(x[21]), "+f"(x[22]), "+f"(x[23]), "+f"(x[24]), "+f"(x[25]), "+f"(x[26]), "+f"(x[27]), "+f"(x[28]), "+f"(x[29]), "+f"(x[30]), "+f"(x[31])
                 :: "memory");
}
template <bool BF>
__device__ __forceinline__ uint32_t kc_pack(float x, float y) {
    if (BF) { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); return *reinterpret_cast<const uint32_t *>(&h); }
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
// x, y as f16 pairs: hi and what it leaves, unscaled: both products go into one accumulator
__device__ __forceinline__ void kc_split(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
// Instruction descriptor: f32 accumulators, A and B both f16 (or both bf16: formats 1 << 7 and 1 << 10), M x N
__host__ __device__ constexpr uint32_t kc_idesc(bool bf, int N) { return umma_idesc_f16(KC_ROWS, N) | (bf ? (1u << 7) | (1u << 10) : 0u); }
// B operand [keys][D] with D contiguous: eight-key groups 1024 bytes apart, 64-wide blocks of D one half apart
__device__ __forceinline__ uint64_t kc_desc_mn(uint32_t addr) {
    return umma_desc_sw128(addr) | ((uint64_t)(KC_HALF >> 4) << 16);
}

// The block of positions that CTA x of a kv head works on: the call's blocks from the last to the first, since later positions see more
// keys and what takes longest should begin first. By one warp; false where there is none.
__device__ __forceinline__ bool kc_place(const KvArgs &a, int x, int per_block, int lane, KcPlace *at) {
    int total = 0;
    bool bad = false;
    for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
        KvSeq q = {0, 0, 0};
        if (s0 + lane < a.n_seq) bad |= !kv_seq(a.row_off, a.kv_len, s0 + lane, a.n_rows, kv_capacity(a), &q);
        total += __reduce_add_sync(0xffffffffu, (q.n + per_block - 1) / per_block);
    }
    if (bad) atomicExch(a.status, ST_PAGE);
    int nth = total - 1 - x;
    if (nth < 0) return false;
    for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
        KvSeq q = {0, 0, 0};
        if (s0 + lane < a.n_seq) kv_seq(a.row_off, a.kv_len, s0 + lane, a.n_rows, kv_capacity(a), &q);
        const int n = (q.n + per_block - 1) / per_block;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const unsigned in = __ballot_sync(0xffffffffu, nth < upto);
        if (in) {
            const int who = __ffs(in) - 1;
            at->seq = s0 + who;
            at->block = nth - __shfl_sync(0xffffffffu, upto - n, who);
            return true;
        }
        nth -= __shfl_sync(0xffffffffu, upto, 31);
    }
    return false;
}

template <int DP, int FMT>
__global__ void __launch_bounds__(KC_THREADS, 1)
kv_chunk_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const KvArgs a, int box_rows) {
    using Sh = ChunkShape<DP, FMT>;
    constexpr bool BF = FMT == KV_BF16, F32 = FMT == KV_F32;
    constexpr int STAGES = Sh::STAGES;
    extern __shared__ uint8_t kc_raw[];
    uint8_t *head = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(kc_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *qst = head + KC_HEAD, *ring = qst + Sh::Q;
    uint64_t *full = reinterpret_cast<uint64_t *>(head), *empty = full + STAGES, *q_full = empty + STAGES, *s_full = q_full + 1,
             *p_part = s_full + 2, *p_full = p_part + 2, *o_full = p_full + 2, *drain = o_full + 2;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
    volatile int *place = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int warp = warp_index(), lane = threadIdx.x & 31;

    chain_trigger();
    chain_wait();
    const int tq = KC_ROWS / a.G;                              // positions of a tile
    if (warp == 0) {
        KcPlace at = {-1, 0};
        if (!kc_place(a, (int)blockIdx.x, 2 * tq, lane, &at)) at.seq = -1;
        if (lane == 0) { place[0] = at.seq; place[1] = at.block; }
    }
    if (threadIdx.x == 32) {
        tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
        for (int s = 0; s < STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(q_full, KC_SOFT);
        for (int t = 0; t < 2; t++) { mbar_init(&s_full[t], 1); mbar_init(&p_part[t], KC_SOFT / 2); mbar_init(&p_full[t], KC_SOFT / 2); mbar_init(&o_full[t], 1); }
        mbar_init(drain, 1);
        mbar_fence_init();
    }
    __syncthreads();
    const int seq = place[0], block = place[1];
    if (seq < 0) return;                                       // the whole CTA
    if (warp == KC_W_MMA) { tc_alloc(tmem_slot, 512); tc_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    KvSeq sq;
    kv_seq(a.row_off, a.kv_len, seq, a.n_rows, kv_capacity(a), &sq);
    const int kvh = blockIdx.y, t0 = block * 2 * tq;           // first position's place among the sequence's rows
    const int base_pos = sq.len - sq.n;
    const int last = min(t0 + 2 * tq, sq.n) - 1;
    const KvTiles tiles = kv_tiles(base_pos + t0 > 0 ? base_pos + t0 : 0, base_pos + last, a.window, a.sinks, KC_KEYS);
    const int n = tiles.count;

    if (warp == KC_W_TMA) {
        // ---- lane = one box of a tile: 64 of the D columns, the slots of one page. Item 2 i of the ring is K(i), 2 i + 1 V(i).
        const int shift = a.page_shift, boxes = KC_KEYS / box_rows * Sh::HALVES;
        const int b_half = lane % Sh::HALVES, b_sub = lane / Sh::HALVES;
        const uint32_t b_at = b_half * KC_HALF + b_sub * box_rows * 128;
        const int top = base_pos + last, low = base_pos + t0;  // what the CTA's rows see between them
        auto seen = [&](int j) { return j <= top && (a.window <= 0 || j + box_rows - 1 > low - a.window || j < a.sinks); };
        auto entry_of = [&](int i) -> int {
            const int j = tiles.at(i) * KC_KEYS + b_sub * box_rows;
            return lane < boxes && i < n && seen(j) ? a.table[(size_t)seq * a.max_pages + (j >> shift)] : -1;
        };
        int entry = entry_of(0), s = 0, ph = 0, r = 0;
        bool ok = true;
        for (int i = 0; i < n && ok; i++) {
            const int next = entry_of(i + 1);
            const int j = tiles.at(i) * KC_KEYS + b_sub * box_rows;
            if (lane < boxes && (unsigned)entry >= (unsigned)a.n_pages) {
                if (seen(j)) atomicExch(a.status, ST_PAGE);
                entry = 0;                                     // any finite rows do
            }
            const int y = (int)kv_row(a, entry, kvh, j & ((1 << shift) - 1));
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                if (r >= STAGES && !mbar_wait_warp(&empty[s], (uint32_t)(ph ^ 1))) { ok = false; break; }
                if (lane == 0) mbar_expect_tx(&full[s], Sh::OPERAND);
                __syncwarp();
                if (lane < boxes) tma_load_2d(ring + s * Sh::OPERAND + b_at, kv ? &tmV : &tmK, b_half * 64, y, &full[s]);
                r++;
                if (++s == STAGES) { s = 0; ph ^= 1; }
            }
            entry = next;
        }
        if (!ok && lane == 0) atomicExch(a.status, ST_TIMEOUT_PRODUCER);
        for (int t = 0; t < STAGES && t < r; t++) {            // what was asked for has to land before the CTA leaves
            if (s == 0) { s = STAGES; ph ^= 1; }
            if (!mbar_wait_warp(&full[--s], (uint32_t)ph)) break;
        }
    } else if (warp == KC_W_MMA) {
        const uint32_t idesc_s = kc_idesc(BF, KC_KEYS), idesc_o = kc_idesc(BF, a.D) | (1u << 16);       // V: MN-major
        const uint64_t qdesc = umma_desc_sw128(smem_u32(qst)), kdesc = umma_desc_sw128(smem_u32(ring)), vdesc = kc_desc_mn(smem_u32(ring));
        const int steps = a.D / 16;
        bool ok = n > 0 ? mbar_wait_warp(q_full, 0) : true;
        auto issue_s = [&](int t, int s) {                     // by one lane
            const uint64_t kd = kdesc + (uint64_t)((s * Sh::OPERAND) >> 4);
            for (int plane = 0; plane < Sh::PLANES; plane++) {
                const uint64_t qd = qdesc + (uint64_t)(((t * Sh::PLANES + plane) * Sh::OPERAND) >> 4);
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk++) {
                    const uint64_t ko = (uint64_t)(((kk >> 2) * KC_HALF + (kk & 3) * 32) >> 4);
                    if (kk < steps) kc_mma(tmem + Sh::COL_S + t * 128, qd + ko, kd + ko, idesc_s, (kk | plane) != 0);
                }
            }
        };
        auto issue_o = [&](int t, int s, bool first, int k0, int k1) {
            const uint64_t vd = vdesc + (uint64_t)((s * Sh::OPERAND) >> 4);
#pragma unroll
            for (int plane = 0; plane < Sh::PLANES; plane++) {
#pragma unroll
                for (int kk = k0; kk < k1; kk++)
                    kc_mma_ts(tmem + Sh::COL_O + t * DP, tmem + Sh::COL_S + t * 128 + plane * 64 + 8 * kk, vd + (uint64_t)((kk * 2048) >> 4), idesc_o,
                              !first || (kk | plane) != 0);
            }
        };
        int s = 0, ph = 0;                                     // ring place of the next item
        auto take = [&](int *at) {                             // waits for the next item
            *at = s;
            const bool got = mbar_wait_warp(&full[s], (uint32_t)ph);
            if (++s == STAGES) { s = 0; ph ^= 1; }
            return got;
        };
        int sk = 0, sv = 0;
        if (ok && n > 0 && (ok = take(&sk))) {
            tc_fence_after();
            if (elect_one()) {
                issue_s(0, sk); tc_commit(&s_full[0]);
                issue_s(1, sk); tc_commit(&s_full[1]);
                tc_commit(&empty[sk]);
            }
            __syncwarp();
            ok = take(&sv);
        }
        // An issued product keeps the pipe busy for 60 clocks, a wait that has come true costs as much: the waits stand where
        // products are still under way.
        for (int i = 0; i < n && ok; i++) {
            const bool more = i + 1 < n;
            const int v = sv;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                if (!mbar_wait_warp(&p_part[t], (uint32_t)(i & 1))) { ok = false; break; }
                tc_fence_after();
                if (elect_one()) issue_o(t, v, i == 0, 0, KC_PART);
                __syncwarp();
                if (more && !take(t == 0 ? &sk : &sv)) { ok = false; break; }      // K(i + 1), V(i + 1)
                if (!mbar_wait_warp(&p_full[t], (uint32_t)(i & 1))) { ok = false; break; }
                tc_fence_after();
                if (elect_one()) {
                    issue_o(t, v, i == 0, KC_PART, KC_KEYS / 16);
                    if (more) { issue_s(t, sk); tc_commit(&s_full[t]); }
                    else tc_commit(&o_full[t]);
                    if (t == 1) { tc_commit(&empty[v]); if (more) tc_commit(&empty[sk]); }
                }
                __syncwarp();
            }
        }
        if (!ok) {                                             // nothing may run on when tensor memory is given back
            if (lane == 0) atomicExch(a.status, ST_TIMEOUT_MMA);
            if (elect_one()) tc_commit(drain);
            __syncwarp();
            mbar_wait_warp(drain, 0);
        }
    } else {
        // ---- softmax: thread = row of tile t
        const int t = warp >> 2, r = (warp & 3) * 32 + lane;
        const int tok = t0 + t * tq + r / a.G, h = kvh * a.G + r % a.G;
        const bool valid = r < tq * a.G && tok < sq.n;
        // rows that do not exist take the last one's position, so that they need no mask of their own
        const int pos = base_pos + min(r < tq * a.G ? tok : t0 + t * tq, sq.n - 1);
        const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        if (n > 0) {
            uint8_t *qt = qst + t * Sh::PLANES * Sh::OPERAND + r * 128;
            const int64_t at = (int64_t)(sq.begin + tok) * a.ldq + (int64_t)h * a.D;
            bool bad = false;
#pragma unroll 4
            for (int c = 0; c < DP / 8; c++) {
                const uint32_t to = (c >> 3) * KC_HALF + (((c & 7) ^ (r & 7)) << 4);
                const bool on = valid && c * 8 < a.D;
                if (F32) {
                    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
                    if (on) {
                        const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + at + c * 8);
                        x = p[0]; y = p[1];
                    }
                    bad |= !(fabsf(x.x) < H16_MAX) | !(fabsf(x.y) < H16_MAX) | !(fabsf(x.z) < H16_MAX) | !(fabsf(x.w) < H16_MAX) |
                           !(fabsf(y.x) < H16_MAX) | !(fabsf(y.y) < H16_MAX) | !(fabsf(y.z) < H16_MAX) | !(fabsf(y.w) < H16_MAX);
                    uint4 hi, lo;
                    kc_split(x.x, x.y, hi.x, lo.x); kc_split(x.z, x.w, hi.y, lo.y); kc_split(y.x, y.y, hi.z, lo.z); kc_split(y.z, y.w, hi.w, lo.w);
                    *reinterpret_cast<uint4 *>(qt + to) = hi;
                    *reinterpret_cast<uint4 *>(qt + Sh::OPERAND + to) = lo;
                } else {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (on) x = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(a.q) + at + c * 8);
                    *reinterpret_cast<uint4 *>(qt + to) = x;
                }
            }
            if (bad) atomicExch(a.status, ST_RANGE);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // generic-proxy stores -> visible to the tensor core
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const float sc = a.scale * 1.4426950408889634f;
        float m = KC_NONE;
        float2 l2[2] = {{0.f, 0.f}, {0.f, 0.f}};
        bool ok = true;
        for (int i = 0; i < n && ok; i++) {
            if (!mbar_wait_warp(&s_full[t], (uint32_t)(i & 1))) { ok = false; break; }
            tc_fence_after();
            float x[KC_KEYS];
            const uint32_t s_at = trow + Sh::COL_S + t * 128;
            tc_ld32(s_at, x);
            tc_ld32(s_at + 32, x + 32);
            kc_wait_ld32(x); kc_wait_ld32(x + 32);
            tc_ld32(s_at + 64, x + 64);
            tc_ld32(s_at + 96, x + 96);
            float m4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int c = 4; c < 60; c += 8)
#pragma unroll
                for (int e = 0; e < 4; e++) m4[e] = fmaxf(m4[e], fmaxf(x[c + e], x[c + 4 + e]));
#pragma unroll
            for (int e = 0; e < 4; e++) m4[e] = fmaxf(m4[e], x[60 + e]);
            kc_wait_ld32(x + 64); kc_wait_ld32(x + 96);
#pragma unroll
            for (int c = 64; c < 128; c += 8)
#pragma unroll
                for (int e = 0; e < 4; e++) m4[e] = fmaxf(m4[e], fmaxf(x[c + e], x[c + 4 + e]));
            const int j0 = tiles.at(i) * KC_KEYS, d = pos - j0;
            const bool whole = d >= KC_KEYS - 1 && (a.window <= 0 || d < a.window || j0 + KC_KEYS - 1 < a.sinks);
            if (!__all_sync(0xffffffffu, whole)) {
                const int low = a.window > 0 ? d - a.window : -1, keep = a.sinks - j0;       // hidden: above d; up to low, from keep on
                m4[0] = m4[1] = m4[2] = m4[3] = -INFINITY;
#pragma unroll
                for (int c = 0; c < KC_KEYS; c++) {
                    if (c > d || (c <= low && c >= keep)) x[c] = -INFINITY;
                    m4[c & 3] = fmaxf(m4[c & 3], x[c]);
                }
            }
            const float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * sc;
            const bool grow = mt > m + 8.f;
            if (__any_sync(0xffffffffu, grow)) {
                const float alpha = grow ? kc_ex2(m - mt) : 1.f;
                if (grow) m = mt;
                l2[0].x *= alpha; l2[0].y *= alpha; l2[1].x *= alpha; l2[1].y *= alpha;
                if (i > 0) {
#pragma unroll 1
                    for (int c = 0; c < DP / 16; c++) {
                        float o[16];
                        tc_ld16(trow + Sh::COL_O + t * DP + 16 * c, o);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] *= alpha;
                        kc_st16(trow + Sh::COL_O + t * DP + 16 * c, reinterpret_cast<const uint32_t *>(o));
                    }
                }
            }
            const float2 sc2 = make_float2(sc, sc), neg = make_float2(-m, -m);
            // groups of 16 keys: a group's exponentials are under way while the one before is summed, packed and stored
#pragma unroll
            for (int c = 0; c <= 8; c++) {
                if (c < 8) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        float *v = x + c * 16 + 2 * e;
                        const float2 y = kc_fma2(make_float2(v[0], v[1]), sc2, neg);
                        v[0] = kc_ex2(y.x); v[1] = kc_ex2(y.y);
                    }
                }
                if (c > 0) {
                    uint32_t hi[8], lo[F32 ? 8 : 1];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float *v = x + (c - 1) * 16 + 2 * e;
                        l2[e & 1] = kc_add2(l2[e & 1], make_float2(v[0], v[1]));
                        if (F32) kc_split(v[0], v[1], hi[e], lo[F32 ? e : 0]);
                        else hi[e] = kc_pack<BF>(v[0], v[1]);
                    }
                    kc_st8(trow + Sh::COL_S + t * 128 + 8 * (c - 1), hi);
                    if (F32) kc_st8(trow + Sh::COL_S + t * 128 + 64 + 8 * (c - 1), lo);
                    if (c == KC_PART) {
                        kc_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_part[t]);
                    }
                }
            }
            kc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[t]);
        }
        if (n > 0 && ok) ok = mbar_wait_warp(&o_full[t], 0);
        if (!ok && lane == 0) atomicExch(a.status, ST_TIMEOUT_EPILOGUE);
        tc_fence_after();
        const float l = (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y), inv = l != 0.f ? 1.f / l : 0.f;
        const int64_t to = (int64_t)(sq.begin + tok) * a.ldo + (int64_t)h * a.D;
#pragma unroll 1
        for (int c = 0; c < DP / 32; c++) {
            float o[32];
            if (n > 0) {
                tc_ld32(trow + Sh::COL_O + t * DP + 32 * c, o);
                tc_wait_ld();
            }
#pragma unroll
            for (int e = 0; e < 32; e++) o[e] = inv != 0.f ? o[e] * inv : 0.f;
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
                if (!valid || c * 32 + e >= a.D) continue;
                if (F32) {
                    float *p = static_cast<float *>(a.out) + to + c * 32 + e;
                    *reinterpret_cast<float4 *>(p) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    *reinterpret_cast<float4 *>(p + 4) = make_float4(o[e + 4], o[e + 5], o[e + 6], o[e + 7]);
                } else {
                    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(a.out) + to + c * 32 + e) =
                        make_uint4(kc_pack<BF>(o[e], o[e + 1]), kc_pack<BF>(o[e + 2], o[e + 3]), kc_pack<BF>(o[e + 4], o[e + 5]), kc_pack<BF>(o[e + 6], o[e + 7]));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == KC_W_MMA) tc_dealloc(tmem, 512);
}

template <int DP, int FMT>
static int chunk_launch(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, int box_rows, cudaStream_t st) {
    using Sh = ChunkShape<DP, FMT>;
    auto kernel = kv_chunk_kernel<DP, FMT>;
    static PerDevice configured = {};
    int dev = 0;
    if (configured.below((size_t)Sh::SMEM, &dev)) {
        MB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
        configured.record(dev, (size_t)Sh::SMEM);
    }
    const int per_block = 2 * (KC_ROWS / a.G);
    const int64_t blocks = (int64_t)a.n_rows / per_block + (a.n_seq < a.n_rows ? a.n_seq : a.n_rows);      // the last block of each may be short
    if (blocks > 0x7fffffff) { set_error("kv_attend: too many rows in one call"); return -1; }
    MB_CUDA(launch_kernel(kernel, dim3((unsigned)blocks, (unsigned)a.Hkv), dim3(KC_THREADS), (size_t)Sh::SMEM, st, true, 1, k, v, a, box_rows));
    note_launch();
    return 0;
}

int kv_chunk(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, int box_rows, int fmt, cudaStream_t st) {
    if (a.D <= 64)
        return fmt == KV_F32 ? chunk_launch<64, KV_F32>(k, v, a, box_rows, st) : fmt == KV_F16 ? chunk_launch<64, KV_F16>(k, v, a, box_rows, st)
                                                                                          : chunk_launch<64, KV_BF16>(k, v, a, box_rows, st);
    return fmt == KV_F32 ? chunk_launch<128, KV_F32>(k, v, a, box_rows, st) : fmt == KV_F16 ? chunk_launch<128, KV_F16>(k, v, a, box_rows, st)
                                                                                       : chunk_launch<128, KV_BF16>(k, v, a, box_rows, st);
}

}  // namespace mb
