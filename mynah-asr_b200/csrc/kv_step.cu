// Attention of one new row per sequence over the pages of its cache:
//   o = sum_j softmax_j(scale q . k_j) v_j  over the visible keys of the sequence,
// for the G query heads that share a kv head at once.
//
// HBM-bound: 4 D bytes of keys and values per key and kv head, 4 G D operations. Up to 16 CTAs of a cluster share a (sequence, kv
// head) and up to 16 of its query heads (StepPlan). One warp of a CTA asks for tiles of 32 KB (64 keys of 128 values) by TMA, two or
// three ahead: the slots of a page and head are a run of rows of a 2-D map, with the 128-byte swizzle. Four warps take a quarter of a
// tile's keys each and keep the running maximum, sum and weighted values of their keys in registers. The products are mma.sync
// m16n8k16 with 16 keys (then 16 values of D) as rows and eight query heads as columns, so that the usual groups of up to eight heads
// waste least: a tcgen05 tile would have 128 rows for them, and mma.sync takes its operands from registers, where the probabilities
// are already (movmatrix turns them). F32 rows: queries and probabilities as (hi, lo) f16 pairs, two products each, which the memory's
// pace hides. The partial results are joined in shared memory, then in the cluster's distributed shared memory, in a fixed order,
// each CTA for its slice of the values: no workspace, no second launch, no atomics.
// Measured (32 query and 8 kv heads of 128, bf16): 131071 keys 99 us = 5.4 TB/s (128 CTAs of 148 SMs: a cluster has at most 16), 60
// ragged sequences of 40 to 9000 keys 76 us = 5.9 TB/s, 700 keys (16 query heads) 6.4 us; 200 sequences of F32 rows, 8 heads of 64, window 1000, 65 us = 5.6 TB/s
// (61 without any arithmetic, as are 98 of the 99: what is left is the pace of the copies). A warp that asks for its own tiles took
// 128 us for the first (each TMA instruction of a diverged lane waits for its operands, in front of the products), query heads as the
// 16 rows of the products 192 us.
#include "kv.h"

namespace mb {

// Probabilities are 2^V of the warp's largest, which the final division takes out again: f16 ends at 2^-24, so that what is held of them, and
// with F32 rows of their rest, is 2^-40 of the largest and not 2^-25 (100 000 keys 17 units below the first one were lost, all but 0.2 %). bf16 has
// the range, but its values end where f32 does: 2^26 of them, the most that a sequence has, do not add up to infinity.
template <int FMT> struct StepTop { static constexpr float V = FMT == KV_BF16 ? -27.f : 15.f; };
static constexpr int KS_MOST_STAGES = 3, KS_HEAD = 1024;                  // barriers in front of the ring
static constexpr int KS_WARPS = 4, KS_THREADS = (KS_WARPS + 1) * 32;      // warps that compute, and one that asks for the tiles
// DP: D rounded up to 64 or 128
template <int DP> struct StepShape {
    static constexpr int HALVES = DP / 64;           // 128-byte wide boxes of a row
    static constexpr int TILE = 64 * 128 / DP;
    static constexpr int OPERAND = TILE * DP * 2;    // keys, or values, of a tile
    static constexpr int STAGE = 2 * OPERAND;
    static constexpr int LDO = DP + 4;               // partial values [heads][LDO], so that a warp's stores touch all banks
};

__device__ __forceinline__ void ks_ldsm(uint32_t addr, uint32_t *r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ks_ldsm_t(uint32_t addr, uint32_t *r) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 8 x 8 of 16 bits, transposed between the lanes
__device__ __forceinline__ uint32_t ks_turn(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool BF>
__device__ __forceinline__ void ks_mma(float *c, const uint32_t *a, uint32_t b0, uint32_t b1) {
    if (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Who does what. A sequence's tiles are cut for 2^k CTAs by its own length: for as many as 2^log_even (what fills the GPU once with the
// call's units) down to a tile each, for more, up to a cluster, as long as each has over half of KS_CHUNK tiles. The units (sequence,
// kv head, head tile) of one k stand side by side in clusters, those of the largest k first, so that what takes longest begins first;
// every warp finds its place from the lengths. Ragged batches need the long sequences cut finer than the others: 32 sequences of 100
// to 16000 keys (8 kv heads of 128) take 72 us this way and 187 with a CTA per unit, 32 of 4096 keys 92 and 83.
static constexpr int KS_CHUNK = 16, KS_MANY = 256;
struct StepPlan {
    int log_size, log_even, per_seq;                 // CTAs of a cluster, see above, units of a sequence
};
__device__ __forceinline__ int ks_log(int v) { return v <= 1 ? 0 : 32 - __clz(v - 1); }
__device__ __forceinline__ int ks_class(const KvArgs &a, const StepPlan &p, int s, int tile) {
    KvSeq q;
    kv_seq(nullptr, a.kv_len, s, a.n_rows, kv_capacity(a), &q);
    const int t = kv_tiles(q.len - 1, q.len - 1, a.window, a.sinks, tile).count;
    return max(min(ks_log(t), p.log_even), min(ks_log((t + KS_CHUNK - 1) / KS_CHUNK), p.log_size));
}
// What CTA `rank` of cluster v works on: a sequence (-1: nothing), its place among the sequence's units, and k. False for a cluster
// behind the last one. (All numbers of units are below 2^31.)
__device__ __forceinline__ bool ks_place(const KvArgs &a, const StepPlan &p, int v, int rank, int tile, int lane, int *seq, int *unit, int *log_parts) {
    if (p.log_size == 0) {                           // a CTA is a unit
        *seq = v / p.per_seq; *unit = v - *seq * p.per_seq; *log_parts = 0;
        return true;
    }
    int count[5] = {0, 0, 0, 0, 0};                  // sequences of each k
    int first = -1;                                  // k of the lane's one of the first 32
#pragma unroll 4
    for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
        const int c = s0 + lane < a.n_seq ? ks_class(a, p, s0 + lane, tile) : -1;
        if (s0 == 0) first = c;
#pragma unroll
        for (int k = 0; k < 5; k++) count[k] += __popc(__ballot_sync(0xffffffffu, c == k));
    }
    int k = -1, have = 0;
#pragma unroll
    for (int c = 4; c >= 0; c--)
        if (k < 0 && c <= p.log_size) {
            const int share = p.log_size - c;        // a cluster holds 2^share units
            const int n = (int)(((unsigned)count[c] * p.per_seq + (1u << share) - 1) >> share);
            if (v < n) { k = c; have = count[c]; } else v -= n;
        }
    if (k < 0) return false;
    const unsigned u = ((unsigned)v << (p.log_size - k)) + (unsigned)(rank >> k);
    int nth = (int)(u / (unsigned)p.per_seq);
    *log_parts = k;
    *unit = (int)(u - (unsigned)nth * p.per_seq);
    *seq = -1;
    for (int s0 = 0; nth < have && s0 < a.n_seq; s0 += 32) {
        const unsigned in = __ballot_sync(0xffffffffu, s0 == 0 ? first == k : s0 + lane < a.n_seq && ks_class(a, p, s0 + lane, tile) == k);
        const int c = __popc(in);
        if (nth < c) {
            *seq = s0 + __ffs(__ballot_sync(0xffffffffu, (in >> lane & 1) && __popc(in & ((1u << lane) - 1)) == nth)) - 1;
            break;
        }
        nth -= c;
    }
    return true;
}

template <int N_> struct KsBatch { static constexpr int N = N_; };

// CTAs that the registers leave room for on an SM
template <int DP, int FMT, int NT> struct StepRoom { static constexpr int CTAS = NT == 1 && (FMT != KV_F32 || DP == 64) ? 3 : 2; };

template <int DP, int FMT, int NT>
__global__ void __launch_bounds__(KS_THREADS, StepRoom<DP, FMT, NT>::CTAS)
kv_step_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const KvArgs a, int log_size, int log_even,
               int stages, int head_tiles) {
    using Sh = StepShape<DP>;
    constexpr bool BF = FMT == KV_BF16, F32 = FMT == KV_F32;
    constexpr int KK = DP / 16, TILE = Sh::TILE, OWN = TILE / KS_WARPS, MT = OWN / 16, HEADS = 8 * NT;
    extern __shared__ uint8_t ks_raw[];
    // (the base has the same offset in every CTA of a cluster)
    uint8_t *head = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(ks_raw) + 1023) & ~uintptr_t(1023)), *smem = head + KS_HEAD;
    uint64_t *full = reinterpret_cast<uint64_t *>(head), *empty = full + KS_MOST_STAGES;
    const int warp = warp_index(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
        for (int s = 0; s < stages; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], KS_WARPS); }
        mbar_fence_init();
    }
    __syncthreads();
    chain_trigger();
    chain_wait();

    const int rank = (int)(blockIdx.x & ((1u << log_size) - 1));
    int seq, unit, log_parts;
    if (!ks_place(a, StepPlan{log_size, log_even, a.Hkv * head_tiles}, (int)(blockIdx.x >> log_size), rank, TILE, lane, &seq, &unit, &log_parts)) return;
    const int parts_n = 1 << log_parts, part_no = rank & (parts_n - 1);
    const int g0 = (unit % head_tiles) * HEADS, kvh = unit / head_tiles;
    const int rows = seq < 0 ? 0 : min(HEADS, a.G - g0);
    KvSeq sq = {0, 0, 0};
    if (seq >= 0 && !kv_seq(nullptr, a.kv_len, seq, a.n_rows, kv_capacity(a), &sq) && threadIdx.x == 0) kv_report(a, ST_PAGE);
    const int pos = sq.len - 1;
    const KvTiles tiles = kv_tiles(pos, pos, a.window, a.sinks, TILE);
    const int n = part_no < tiles.count ? (tiles.count - part_no + parts_n - 1) >> log_parts : 0;        // tiles of this CTA

    // o[nt][dt]: values 16 dt + lane / 4 (+ 8) of the heads 8 nt + 2 (lane % 4) + {0, 1}; m, l of these two heads
    float o[NT][DP / 16][4], m[NT][2], l[NT][2];
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    if (warp == KS_WARPS) {
        // ---- requests: lane = one box of a tile (keys or values, 64 of the D columns, the slots of one page). The table's entry is
        // fetched a tile ahead of its use.
        const int shift = a.page_shift, box_rows = min(1 << shift, TILE), boxes = TILE / box_rows * Sh::HALVES * 2;
        const int b_kv = lane & 1, b_half = (lane >> 1) % Sh::HALVES, b_sub = (lane >> 1) / Sh::HALVES;
        const uint32_t b_at = b_kv * Sh::OPERAND + b_half * (TILE * 128) + b_sub * box_rows * 128;
        const CUtensorMap *map = b_kv ? &tmV : &tmK;
        auto key_of = [&](int i) { return tiles.at(part_no + (i << log_parts)) * TILE + b_sub * box_rows; };
        auto seen = [&](int j) { return j <= pos && (a.window <= 0 || j + box_rows - 1 > pos - a.window || j < a.sinks); };
        // page of this lane's box of tile i; -1 where none of its keys is visible (and the table may say anything)
        auto entry_of = [&](int i) -> int {
            const int j = key_of(i);
            return lane < boxes && i < n && seen(j) ? a.table[(size_t)seq * a.max_pages + (j >> shift)] : -1;
        };
        int entry = entry_of(0), s = 0, ph = 0, i = 0;
        for (; i < n; i++) {
            const int next = entry_of(i + 1);
            if (i >= stages && !mbar_wait_warp(&empty[s], (uint32_t)(ph ^ 1))) {
                if (lane == 0) kv_report(a, ST_TIMEOUT_PRODUCER);
                break;
            }
            if (lane == 0) mbar_expect_tx(&full[s], Sh::STAGE);
            __syncwarp();
            if (lane < boxes) {
                const int j = key_of(i);
                if ((unsigned)entry >= (unsigned)a.n_pages) {
                    if (seen(j)) kv_report(a, ST_PAGE);
                    entry = 0;                                 // any finite rows do
                }
                tma_load_2d(smem + s * Sh::STAGE + b_at, map, b_half * 64, (int)kv_row(a, entry, kvh, j & ((1 << shift) - 1)), &full[s]);
            }
            entry = next;
            if (++s == stages) { s = 0; ph ^= 1; }
        }
        // what was asked for has to land before the ring serves another purpose or the CTA leaves, whatever becomes of the other warps
        for (int t = 0; t < stages && t < i; t++) {
            if (s == 0) { s = stages; ph ^= 1; }
            if (!mbar_wait_warp(&full[--s], (uint32_t)ph)) break;
        }
    } else {
        // ---- the query heads as the B operand [D][heads]: head lane / 4, values 2 (lane % 4) and 8 further
        uint32_t qh[NT][KK][2], ql[F32 ? NT : 1][F32 ? KK : 1][2];
        bool bad = false;
        const int64_t row = (int64_t)seq * a.ldq + (int64_t)(kvh * a.G + g0) * a.D;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int r = nt * 8 + r0;
                    const bool on = r < rows && kk * 16 < a.D && n > 0;
                    const int64_t at = row + (int64_t)r * a.D + kk * 16 + c0 + e * 8;
                    qh[nt][kk][e] = 0;
                    if (F32) {
                        float2 f = make_float2(0.f, 0.f);
                        if (on) f = *reinterpret_cast<const float2 *>(static_cast<const float *>(a.q) + at);
                        bad |= !(fabsf(f.x) < H16_MAX) | !(fabsf(f.y) < H16_MAX);
                        kv_split(f.x, f.y, qh[nt][kk][e], ql[F32 ? nt : 0][F32 ? kk : 0][e]);
                    } else if (on) {
                        qh[nt][kk][e] = *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(a.q) + at);
                    }
                }
        if (bad) kv_report(a, ST_RANGE);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int i = 0; i < DP / 16; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }
        const float sc = a.scale2;
        const int g = lane >> 3, rr = lane & 7;                // ldmatrix: lane group = 8 x 8 matrix, row in it
        const uint32_t base = smem_u32(smem) + warp * OWN * 128;
        const uint32_t k_row = ((g & 1) * 8 + rr) * 128, v_row = ((g >> 1) * 8 + rr) * 128;
        int s = 0, ph = 0;
        for (int i = 0; i < n; i++) {
            const int j0 = tiles.at(part_no + (i << log_parts)) * TILE + warp * OWN;
            if (!mbar_wait_warp(&full[s], (uint32_t)ph)) {
                if (lane == 0) kv_report(a, ST_TIMEOUT_EPILOGUE);
                break;
            }
            const uint32_t kt = base + s * Sh::STAGE, vt = kt + Sh::OPERAND;
            const bool whole = j0 + OWN - 1 <= pos && (a.window <= 0 || j0 > pos - a.window || j0 + OWN - 1 < a.sinks);
            if (whole || (j0 <= pos && (a.window <= 0 || j0 + OWN - 1 > pos - a.window || j0 < a.sinks))) {
                // ---- scores: rows = keys, columns = heads. Two sums per score, of the even and the odd steps: half the chain
                float x[NT][MT][4], y[NT][MT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) x[nt][mt][e] = y[nt][mt][e] = 0.f;
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    if (kk * 16 < a.D) {
#pragma unroll
                        for (int mt = 0; mt < MT; mt++) {
                            uint32_t k4[4];
                            ks_ldsm(kt + (kk >> 2) * (TILE * 128) + mt * 2048 + k_row + ((((kk & 3) * 2 + (g >> 1)) ^ rr) << 4), k4);
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                float *acc = (kk & 1) ? y[nt][mt] : x[nt][mt];
                                ks_mma<BF>(acc, k4, qh[nt][kk][0], qh[nt][kk][1]);
                                if (F32) ks_mma<BF>(acc, k4, ql[F32 ? nt : 0][F32 ? kk : 0][0], ql[F32 ? nt : 0][F32 ? kk : 0][1]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int e = 0; e < 4; e++) x[nt][mt][e] += y[nt][mt][e];
                if (!whole) {
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (!kv_sees(pos, j0 + mt * 16 + r0 + (e >> 1) * 8, a.window, a.sinks)) {
#pragma unroll
                                for (int nt = 0; nt < NT; nt++) x[nt][mt][e] = -INFINITY;
                            }
                }
                // ---- running maximum of each head, over the keys: the lanes of a column
                uint32_t pb[NT][MT][2], pl[F32 ? NT : 1][F32 ? MT : 1][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float t[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        t[0] = fmaxf(t[0], fmaxf(x[nt][mt][0], x[nt][mt][2]));
                        t[1] = fmaxf(t[1], fmaxf(x[nt][mt][1], x[nt][mt][3]));
                    }
#pragma unroll
                    for (int w = 4; w < 32; w *= 2) {
                        t[0] = fmaxf(t[0], __shfl_xor_sync(0xffffffffu, t[0], w));
                        t[1] = fmaxf(t[1], __shfl_xor_sync(0xffffffffu, t[1], w));
                    }
                    const float n0 = fmaxf(m[nt][0], t[0]), n1 = fmaxf(m[nt][1], t[1]);
                    if (__any_sync(0xffffffffu, n0 > m[nt][0] || n1 > m[nt][1])) {
                        const float a0 = kv_weight(m[nt][0], n0, sc), a1 = kv_weight(m[nt][1], n1, sc);
                        l[nt][0] *= a0; l[nt][1] *= a1;
#pragma unroll
                        for (int d = 0; d < DP / 16; d++) { o[nt][d][0] *= a0; o[nt][d][1] *= a1; o[nt][d][2] *= a0; o[nt][d][3] *= a1; }
                        m[nt][0] = n0; m[nt][1] = n1;
                    }
                    const float off[2] = {m[nt][0] == -INFINITY ? 0.f : m[nt][0], m[nt][1] == -INFINITY ? 0.f : m[nt][1]};
                    // ---- probabilities, turned from [key][head] to the B operand's layout
#pragma unroll
                    for (int mt = 0; mt < MT; mt++) {
                        float p[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) p[e] = kv_ex2(fmaf(x[nt][mt][e] - off[e & 1], sc, StepTop<FMT>::V));
                        l[nt][0] += p[0] + p[2]; l[nt][1] += p[1] + p[3];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            if (F32) {
                                uint32_t hi, lo;
                                kv_split(p[2 * e], p[2 * e + 1], hi, lo);
                                pb[nt][mt][e] = ks_turn(hi);
                                pl[F32 ? nt : 0][F32 ? mt : 0][e] = ks_turn(lo);
                            } else {
                                pb[nt][mt][e] = ks_turn(kv_pack<BF>(p[2 * e], p[2 * e + 1]));
                            }
                        }
                    }
                }
                // ---- values: rows = D (V transposed on its way out of shared memory), columns = heads
                // F32 rows: the tensor cores cut sums toward zero, which over 1000 keys costs 5e-6 of a result, so each tile's sum is one of its
                // own, the small products first, and added here
                auto values = [&](int dt, int mt, auto &&sum) {
                    uint32_t v4[4];
                    ks_ldsm_t(vt + (dt >> 2) * (TILE * 128) + mt * 2048 + v_row + ((((dt & 3) * 2 + (g & 1)) ^ rr) << 4), v4);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) sum(nt, v4);
                };
                if (F32) {
#pragma unroll
                    for (int dt = 0; dt < DP / 16; dt++) {
                        if (dt * 16 < a.D) {
                            float f[NT][4] = {};
#pragma unroll
                            for (int mt = 0; mt < MT; mt++)
                                values(dt, mt, [&](int nt, const uint32_t *v4) {
                                    ks_mma<BF>(f[nt], v4, pl[F32 ? nt : 0][F32 ? mt : 0][0], pl[F32 ? nt : 0][F32 ? mt : 0][1]);
                                    ks_mma<BF>(f[nt], v4, pb[nt][mt][0], pb[nt][mt][1]);
                                });
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                for (int e = 0; e < 4; e++) o[nt][dt][e] += f[nt][e];
                        }
                    }
                } else {
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int dt = 0; dt < DP / 16; dt++)
                            if (dt * 16 < a.D) values(dt, mt, [&](int nt, const uint32_t *v4) { ks_mma<BF>(o[nt][dt], v4, pb[nt][mt][0], pb[nt][mt][1]); });
                }
            }
            __syncwarp();                                      // every lane has read the stage
            if (lane == 0) mbar_arrive(&empty[s]);
            if (++s == stages) { s = 0; ph ^= 1; }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int w = 4; w < 32; w *= 2) {
                l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], w);
                l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], w);
            }
    }
    // ---- join. Parts are values [heads][LDO] and (maximum, sum) of each head: first those of the CTA's warps, where the tiles were
    constexpr int PART = HEADS * Sh::LDO + 2 * HEADS;
    float *parts = reinterpret_cast<float *>(smem), *mine = parts + KS_WARPS * PART;
    __syncthreads();                                           // nobody reads a tile any more
    if (warp < KS_WARPS) {
        float *part = parts + warp * PART;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int h = nt * 8 + c0;
#pragma unroll
            for (int d = 0; d < DP / 16; d++)
#pragma unroll
                for (int e = 0; e < 4; e++) part[(h + (e & 1)) * Sh::LDO + d * 16 + r0 + (e >> 1) * 8] = o[nt][d][e];
            if (lane < 4) *reinterpret_cast<float4 *>(part + HEADS * Sh::LDO + 2 * h) = make_float4(m[nt][0], l[nt][0], m[nt][1], l[nt][1]);
        }
    }
    __syncthreads();
    const int quads = a.D / 4;
    auto store = [&](int r, int c, float4 v, float total) {
        const float inv = total != 0.f ? 1.f / total : 0.f;
        const int64_t at = (int64_t)seq * a.ldo + (int64_t)(kvh * a.G + g0 + r) * a.D + c;
        if (F32) *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        else *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + at) = make_uint2(kv_pack_result<BF>(v.x * inv, v.y * inv), kv_pack_result<BF>(v.z * inv, v.w * inv));
        if (!kv_sound(total) && c == 0 && pos >= 0) kv_report(a, ST_RANGE);
    };
    for (int q = threadIdx.x; q < rows * quads; q += KS_THREADS) {
        const int r = q / quads, c = (q % quads) * 4;
        float2 e[KS_WARPS];
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < KS_WARPS; w++) {
            e[w] = *reinterpret_cast<const float2 *>(parts + w * PART + HEADS * Sh::LDO + 2 * r);
            top = fmaxf(top, e[w].x);
        }
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KS_WARPS; w++) {
            const float4 v = *reinterpret_cast<const float4 *>(parts + w * PART + r * Sh::LDO + c);
            const float f = kv_weight(e[w].x, top, a.scale2);
            total = fmaf(f, e[w].y, total);
            sum.x = fmaf(f, v.x, sum.x); sum.y = fmaf(f, v.y, sum.y); sum.z = fmaf(f, v.z, sum.z); sum.w = fmaf(f, v.w, sum.w);
        }
        if (log_parts == 0) {
            store(r, c, sum, total);
        } else {
            *reinterpret_cast<float4 *>(mine + r * Sh::LDO + c) = sum;
            if (c == 0) *reinterpret_cast<float2 *>(mine + HEADS * Sh::LDO + 2 * r) = make_float2(top, total);
        }
    }
    // then those of the CTAs that share the unit, in their order, each CTA for its slice of the values
    if (log_parts > 0) {
        kv_cluster_sync();
        const uint32_t at0 = smem_u32(mine);
        const int base = rank - part_no;
        // (up to eight parts' reads are under way at a time: one after the other, sixteen took 3800 of a short call's 12900 clocks)
        auto join = [&](auto at_a_time) {                      // a divisor of parts_n
            constexpr int N = decltype(at_a_time)::N;
            for (int q = part_no * KS_THREADS + (int)threadIdx.x; q < rows * quads; q += parts_n * KS_THREADS) {
                const int r = q / quads, c = (q % quads) * 4;
                float top = -INFINITY, total = 0.f;
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                for (int p0 = 0; p0 < parts_n; p0 += N) {
                    float2 e[N];
                    float4 v[N];
#pragma unroll
                    for (int p = 0; p < N; p++) {
                        e[p] = kv_peer2(kv_peer(at0 + (HEADS * Sh::LDO + 2 * r) * 4, base + p0 + p));
                        v[p] = kv_peer4(kv_peer(at0 + (r * Sh::LDO + c) * 4, base + p0 + p));
                    }
                    float m = top;
#pragma unroll
                    for (int p = 0; p < N; p++) m = fmaxf(m, e[p].x);
                    const float old = kv_weight(top, m, a.scale2);
                    total *= old; sum.x *= old; sum.y *= old; sum.z *= old; sum.w *= old;
                    top = m;
#pragma unroll
                    for (int p = 0; p < N; p++) {
                        const float f = kv_weight(e[p].x, m, a.scale2);
                        total = fmaf(f, e[p].y, total);
                        sum.x = fmaf(f, v[p].x, sum.x); sum.y = fmaf(f, v[p].y, sum.y); sum.z = fmaf(f, v[p].z, sum.z); sum.w = fmaf(f, v[p].w, sum.w);
                    }
                }
                store(r, c, sum, total);
            }
        };
        if (parts_n == 2) join(KsBatch<2>()); else if (parts_n == 4) join(KsBatch<4>()); else join(KsBatch<8>());
        kv_cluster_sync();                                     // nobody leaves while its part is being read
    }
}

template <int DP, int FMT, int NT>
static int step_launch(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, cudaStream_t st) {
    using Sh = StepShape<DP>;
    auto kernel = kv_step_kernel<DP, FMT, NT>;
    static PerDevice configured = {};
    int dev = 0;
    const size_t most = (size_t)KS_MOST_STAGES * Sh::STAGE + KS_HEAD + 1024;
    if (configured.below(most, &dev)) {
        MB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
        MB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        configured.record(dev, most);
    }
    const int head_tiles = cdiv(a.G, 8 * NT);
    const int64_t units = (int64_t)a.n_seq * a.Hkv * head_tiles;
    // log_even: two CTAs per SM at most; a cluster is up to four times that, where the table has room for sequences that need it
    const int64_t sms = device_sm_count();
    int log_even = 0, log_size, most_tiles = 0;
    {
        const int64_t keys = (int64_t)a.max_pages << a.page_shift, seen = (int64_t)a.window + a.sinks + 2 * Sh::TILE;
        most_tiles = (int)(((a.window > 0 && seen < keys ? seen : keys) + Sh::TILE - 1) / Sh::TILE);
    }
    while (log_even < 4 && units << (log_even + 1) <= 2 * sms && 1 << log_even < most_tiles) log_even++;
    log_size = log_even;
    // (Not where the units alone keep the GPU busy, or the lengths that every warp looks through are many: bf16, 4 query heads of 128 per kv head, a
    // table for 32768 keys, us, cut and not: 32 sequences of 8 kv heads, 100 to 16000 keys 70, 186, 20 to 300 keys 8.4, 7.4; 192 357, 430 and 52, 22;
    // 256 473, 517 and 77, 28, of 2 kv heads 121, 229 and 22, 11; 2048 with 2 query heads of 64 each 4918, 1643 and 2622, 145.)
    const bool cut = a.n_seq <= KS_MANY && units <= 12 * sms;
    while (cut && log_size < 4 && log_size < log_even + 2 && KS_CHUNK << log_size < most_tiles) log_size++;
    // Tiles ahead: two, so that three CTAs fit an SM, where there are more than two for each; three otherwise. us, with two and with three tiles
    // ahead: 20 sequences of 2000 keys (16 and 8 heads of 64, f16) 18.6, 16.3, 18 of 500 (32 and 8 of 128, bf16) 11.9, 10.9; 60 of 100 to
    // 4230 (8 heads of 64, F32 rows) 51, 60, 200 under a window of 1000 64, 68
    const int stages = StepRoom<DP, FMT, NT>::CTAS == 2 || units << log_size <= 2 * sms ? 3 : 2;
    if (units << log_size > 0x7fffffff) { set_error("kv_attend: too many sequences in one call"); return -1; }
    const size_t smem = (size_t)stages * Sh::STAGE + KS_HEAD + 1024;
    MB_CUDA(launch_kernel(kernel, dim3((unsigned)(units << log_size)), dim3(KS_THREADS), smem, st, true, 1 << log_size, k, v, a, log_size, log_even, stages, head_tiles));
    note_launch();
    return 0;
}

template <int DP, int FMT>
static int step_heads(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, cudaStream_t st) {
    return a.G <= 8 ? step_launch<DP, FMT, 1>(k, v, a, st) : step_launch<DP, FMT, 2>(k, v, a, st);
}

int kv_box(int D, int page_size) {
    const int tile = D <= 64 ? StepShape<64>::TILE : StepShape<128>::TILE;
    return page_size < tile ? page_size : tile;
}

int kv_step(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, int fmt, cudaStream_t st) {
    if (a.D <= 64) return fmt == KV_F32 ? step_heads<64, KV_F32>(k, v, a, st) : fmt == KV_F16 ? step_heads<64, KV_F16>(k, v, a, st) : step_heads<64, KV_BF16>(k, v, a, st);
    return fmt == KV_F32 ? step_heads<128, KV_F32>(k, v, a, st) : fmt == KV_F16 ? step_heads<128, KV_F16>(k, v, a, st) : step_heads<128, KV_BF16>(k, v, a, st);
}

}  // namespace mb
