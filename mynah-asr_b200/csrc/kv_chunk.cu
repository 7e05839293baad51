// Attention of many rows per sequence over the pages of its cache: prompts, or pieces of prompts behind cached keys,
//   o_p = sum_j softmax_j(scale q_p . k_j) v_j  over j <= p, with a window also j > p - window or j < sinks.
//
// Bound by the tensor cores and, as much, by the exponentials (4 D operations and one exponential per pair of row and key: with D = 128
// both take about 1024 clocks of an SM for 128 rows and 128 keys). A CTA owns one kv head and one or two tiles of 128 rows: the G query
// heads of 128 / G positions each (row r is head r % G of position r / G), so that short pieces fill a tile and all heads share the
// keys' tiles. Keys and values come in tiles of 128 by TMA, from their pages straight into the swizzled operand layout: groups of 32
// keys, those that some row sees, side by side (KvGroups; with a tile of their own for a window's first tokens the third case below took 75 us instead of 63).
//   tensor memory  16-bit rows: scores S (128 columns a tile) and results O. D > 64: two tiles of rows, whose probabilities P overwrite
//                  their scores. D <= 64: one tile, two CTAs an SM, columns of their own for P, so that S(i + 1) is computed under the
//                  exponentials of tile i. F32 rows: one tile, and F, the products of one tile of keys (see ChunkShape)
//   warps          0-3 (and 4-7): softmax of tile 0 (and 1), a thread per row; then TMA, and MMA
//   order of MMAs  P0 V(i), S0(i + 1), P1 V(i), S1(i + 1): one tile's exponentials run under the other's products. MMAs run in the
//                  order of their issue, so S(i + 1) does not overwrite the P(i) that P V(i) reads, and whoever sees S(i + 1) finished
//                  finds O at rest. With columns of their own for P: S(i + 1) in front of P V(i).
// A CTA stays and takes block after block (heads of a block side by side, long blocks first, KcFinder): the next block's place, queries
// and first keys are looked up, fetched and multiplied while the results of the one before are written.
// The softmax keeps a running maximum per row; O is rescaled only when it has grown by more than ChunkTop says (what is stale cancels
// in the final division). F32 rows: queries and probabilities as (hi, lo) f16 pairs, two products each.
// A call with few blocks is launched as clusters: the CTAs of a cluster take a block's tiles in turn, two at least each, and join their
// results through distributed shared memory.
//
// Measured (us): 16384 rows of 32 query and 8 kv heads of 128, bf16, 2045 = 1.1 PFLOP/s under the power cap (1.72 GHz; a library's
// product of matrices holds 1.42 there); 4 pieces of 5 to 61 rows behind 300 to 1500 keys 14.0; 7 prompts of 301 to 4000 rows, 16 and 4
// heads of 64, f16, window 512, 59.7; 9 of 40 to 1300 F32 rows, 8 heads of 128, 37.4. A tile of D = 128 goes through 1190 clocks of
// waiting for its scores, 245 + 220 of their maximum, 1550 of exponentials and packing, 250 of signals; the other tile's take turns with
// it. Tensor cores and exponential units are busy half of the time each. What was tried against that: steps of 64 keys with two score
// buffers, so that no softmax waits (2210: products 64 columns wide take as long as 128 wide ones), a part of the exponentials as
// polynomials (no gain), two threads a row (none), one tile and two CTAs an SM (slower), six stages (none).
#include "kv.h"

namespace mb {

static constexpr int KC_ROWS = 128, KC_KEYS = 128, KC_HALF = 128 * 128;      // a 128-row x 64-column box of 16-bit values: 16 KB
static constexpr int KC_HEAD = 1024, KC_STAY = 3000;
static constexpr int KC_PART = 3;                    // P V begins when the first 3 x 32 keys' probabilities are there

// The maximum of a row may lag by 2^LAG, and a probability is 2^TOP of it, which the final division takes out again: together below f16's 2^16,
// and what is held of a probability (with F32 rows: of its rest) is 2^-25 / 2^TOP of the largest, where it was 2^-25 without. bf16 has the
// range, but its values end where f32 does: 2^26 of them, the most that a sequence has, do not add up to infinity. A smaller LAG rescales O more
// often: f16, 8192 rows of 32 heads of 128, scores spread by 2.5 units: 481 us, with a LAG of 4 518, of 2 540. F32 rows of
// 128 rescale for every tile in any case; 8 heads of 64 take 41.8 us, with a LAG of 8 40.3.
template <int FMT> struct ChunkTop {
    static constexpr float LAG = FMT == KV_F32 ? 1.f : 8.f, TOP = FMT == KV_F32 ? 14.f : FMT == KV_F16 ? 7.f : -35.f;
};

template <int DP, int FMT> struct ChunkShape {
    static constexpr int HALVES = DP / 64, PLANES = FMT == KV_F32 ? 2 : 1;
    // F32 rows: the tensor cores cut every sum toward zero, which over 1000 keys costs 5e-6 of a result; so a tile's P V is a sum of its
    // own, in columns F, that the softmax warps add to O
    static constexpr bool FRESH = FMT == KV_F32;
    static constexpr int TILES = DP == 64 || FRESH ? 1 : 2, PER_SM = DP == 64 ? 2 : 1;         // tiles of rows of a CTA, CTAs of an SM
    // two threads a row, 64 of a tile's keys and half of O each, where the SM has no other softmax warps
    static constexpr int SPLIT = TILES * PER_SM == 1 ? 2 : 1, OWN = KC_KEYS / SPLIT;
    static constexpr int SOFT = 4 * TILES * SPLIT, W_TMA = SOFT, W_MMA = SOFT + 1;             // warps
    // The launch's registers are dealt out anew between the softmax warps and the four warps of TMA and MMA, two of which have no other
    // work than to lend theirs
    static constexpr int THREADS = 32 * (SOFT + 4), REGS = SOFT == 8 ? 168 : 128, MORE = SOFT == 8 ? 208 : 200, LESS = SOFT == 8 ? 88 : 56;
    static_assert(32 * SOFT * MORE + 128 * LESS <= THREADS * REGS, "a share beyond the launch's registers waits for good");
    static constexpr int OPERAND = HALVES * KC_HALF;           // a tile of queries (one plane), of keys, or of values
    static constexpr int Q = TILES * PLANES * OPERAND;
    static constexpr int STAGES = 6 - PLANES;
    static constexpr int HEAD = KC_HEAD + (SPLIT == 2 ? 2048 : 0);     // barriers, blocks' words; what the two threads of a row tell one another
    static constexpr int SMEM = HEAD + Q + STAGES * OPERAND + 1024;
    static_assert(PER_SM * (SMEM + 1024) <= 233472, "shared memory");
    static constexpr bool OWN_P = TILES == 1 && (DP == 64) == (PLANES == 1);   // columns of their own for the probabilities
    static constexpr int COL_S = 0, COL_P = OWN_P ? 128 * TILES : 0, STEP_P = OWN_P ? 64 * PLANES : 128, COL_O = 128 * TILES + (OWN_P ? STEP_P * TILES : 0);
    static constexpr int COL_F = COL_O + (FRESH ? TILES * DP : 0);     // where P V goes
    static constexpr int TMEM = 512 / PER_SM;
    static_assert(COL_F + TILES * DP <= TMEM, "tensor memory");
    static constexpr int LDO = DP + 4;                         // a part of a row's result in shared memory
    static_assert(TILES * 128 * (LDO * 4 + 8 + 64) <= Q + STAGES * OPERAND, "parts");
};

__device__ __forceinline__ void kc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void kc_load_3d(void *dst, const CUtensorMap *m, int x, int y, int z, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
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
// Waits for loads from tensor memory; the values that they bring are not to be touched before (nor their use moved up)
__device__ __forceinline__ void kc_wait_ld32(float *x) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(x[0]), "+f"(x[1]), "+f"(x[2]), "+f"(x[3]), "+f"(x[4]), "+f"(x[5]), "+f"(x[6]), "+f"(x[7]), "+f"(x[8]), "+f"(x[9]), "+f"(x[10]),
                   "+f"(x[11]), "+f"(x[12]), "+f"(x[13]), "+f"(x[14]), "+f"(x[15]), "+f"(x[16]), "+f"(x[17]), "+f"(x[18]), "+f"(x[19]), "+f"(x[20]),
                   "+f"(x[21]), "+f"(x[22]), "+f"(x[23]), "+f"(x[24]), "+f"(x[25]), "+f"(x[26]), "+f"(x[27]), "+f"(x[28]), "+f"(x[29]), "+f"(x[30]), "+f"(x[31])
                 :: "memory");
}
template <int N> __device__ __forceinline__ void kc_regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void kc_regs_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// Instruction descriptor: f32 accumulators, A and B both f16 (or both bf16: formats 1 << 7 and 1 << 10), M x N
__host__ __device__ constexpr uint32_t kc_idesc(bool bf, int N) { return umma_idesc_f16(KC_ROWS, N) | (bf ? (1u << 7) | (1u << 10) : 0u); }
// B operand [keys][D] with D contiguous: eight-key groups 1024 bytes apart, 64-wide blocks of D one half apart
__device__ __forceinline__ uint64_t kc_desc_mn(uint32_t addr) {
    return umma_desc_sw128(addr) | ((uint64_t)(KC_HALF >> 4) << 16);
}

// Where the TMA warp finds the call's blocks: all their number, and the x-th from the last, since later positions see more keys and
// what takes longest should begin first. With up to 32 sequences a lane keeps one, and the x-th longest is found, too: by bisection of
// the length that more than x blocks have (with it the third and fourth case above took 58.8 and 37.6 us, with the order of the sequences
// 63.4 and 46.2). Up to 256 are counted through, 32 at a time; with more, see KcMany.
static constexpr int KC_LANES = 32, KC_COUNT = 256;
struct KcFinder {
    int per_block, total, mine;                      // rows of a block, blocks of the call, blocks of the lane's sequence
    KvSeq q;
    __device__ __forceinline__ void look(const KvArgs &a, int s, bool *bad) {
        q = {0, 0, 0};
        if (s < a.n_seq) *bad |= !kv_seq(a.row_off, a.kv_len, s, a.n_rows, kv_capacity(a), &q);
        mine = (q.n + per_block - 1) / per_block;
    }
    // most: blocks of tables that are in order. Rows that several sequences claim make no more than that.
    __device__ __forceinline__ void init(const KvArgs &a, int per, int most, int lane) {
        per_block = per; total = 0;
        bool bad = false;
        for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
            look(a, s0 + lane, &bad);
            total += __reduce_add_sync(0xffffffffu, mine);
        }
        if (bad) kv_report(a, ST_PAGE);
        total = min(total, most);
    }
    // Blocks of the lane's sequence with `tiles` tiles of keys at least: those from some place on (a window bounds all alike)
    __device__ __forceinline__ int as_long(const KvArgs &a, int tiles) const {
        const int need = (tiles - 1) * KC_KEYS + 1 - (q.len - q.n);            // rows that the block's last one has in front of it, and itself
        if (need > q.n || (a.window > 0 && (tiles - 1) * KC_KEYS >= a.window + a.sinks + per_block)) return 0;
        return mine - (need <= per_block ? 0 : (need + per_block - 1) / per_block - 1);
    }
    __device__ __forceinline__ void find_longest(const KvArgs &a, int x, int lane, int *seq, int *block, KvSeq *at) {
        *seq = -1; *block = 0; *at = {0, 0, 0};
        if (x >= total) return;
        int lo = 0, hi = __reduce_max_sync(0xffffffffu, q.n > 0 ? (max(q.len, 0) + KC_KEYS - 1) / KC_KEYS : 0) + 1;         // x < blocks of lo tiles, not of hi
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (__reduce_add_sync(0xffffffffu, as_long(a, mid)) > x) lo = mid; else hi = mid;
        }
        const int longer = as_long(a, lo + 1), some = lo > 0 ? as_long(a, lo) : mine, n = some - longer;
        int nth = x - __reduce_add_sync(0xffffffffu, longer), upto = n;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const int who = __ffs(__ballot_sync(0xffffffffu, nth < upto)) - 1;
        if (who < 0) return;
        *seq = who;
        *block = __shfl_sync(0xffffffffu, mine - some - (upto - n), who) + nth;
        at->begin = __shfl_sync(0xffffffffu, q.begin, who);
        at->n = __shfl_sync(0xffffffffu, q.n, who);
        at->len = __shfl_sync(0xffffffffu, q.len, who);
    }
    __device__ __forceinline__ void find(const KvArgs &a, int x, int lane, int *seq, int *block, KvSeq *at) {
        int nth = total - 1 - x;
        *seq = -1; *block = 0; *at = {0, 0, 0};
        if (nth < 0) return;
        bool bad = false;
        for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
            if (a.n_seq > KC_LANES) look(a, s0 + lane, &bad);
            const int n = mine;
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned in = __ballot_sync(0xffffffffu, nth < upto);
            if (in) {
                const int who = __ffs(in) - 1;
                *seq = s0 + who;
                *block = nth - __shfl_sync(0xffffffffu, upto - n, who);
                at->begin = __shfl_sync(0xffffffffu, q.begin, who);
                at->n = __shfl_sync(0xffffffffu, q.n, who);
                at->len = __shfl_sync(0xffffffffu, q.len, who);
                return;
            }
            nth -= __shfl_sync(0xffffffffu, upto, 31);
        }
    }
};

// The same where counting takes long: block i of sequence s has the number row_off[s] / per_block + s + i, which no other block has, so a sequence is
// found by bisection of the offsets, and numbers without a block are passed over. (Sequences of 5 to 40 rows, us, counted through and this
// way: 300 65, 66, 1000 302, 192, 4000 3600, 740.)
struct KcMany {
    int per_block, total;
    __device__ __forceinline__ void init(const KvArgs &, int per, int most, int) { per_block = per; total = most; }
    __device__ __forceinline__ void find(const KvArgs &a, int x, int lane, int *seq, int *block, KvSeq *at) const {
        const int nth = total - 1 - x;
        *seq = -1; *block = 0; *at = {0, 0, 0};
        if (nth < 0) return;
        // the last sequence whose first number is nth at most: each round looks at 32 places of what is left
        int lo = 0, hi = a.n_seq;
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) / 32, place = min(lo + lane * step, hi - 1);
            const unsigned below = __ballot_sync(0xffffffffu, lo + lane * step < hi && a.row_off[place] / per_block + place <= nth);
            if (below == 0) return;
            lo += (31 - __clz(below)) * step;
            hi = min(hi, lo + step);
        }
        KvSeq s;
        const int i = nth - a.row_off[lo] / per_block - lo;
        if (!kv_seq(a.row_off, a.kv_len, lo, a.n_rows, kv_capacity(a), &s) || i < 0 || i >= (s.n + per_block - 1) / per_block) return;
        *seq = lo; *block = i; *at = s;
    }
};

template <bool MANY> struct KcFind { typedef KcFinder Type; };
template <> struct KcFind<true> { typedef KcMany Type; };

// What a block is to those who work on it. The TMA warp finds it out and leaves it as words in shared memory.
struct KcBlock {
    static constexpr int WORDS = 12;
    int seq, kvh, begin, rows, t0, base_pos;         // its sequence (-1: no block, -2: the wait for one ran out), head, the sequence's rows; the block's
                                                     // first one among them, the position of row 0 of the sequence
    int n, nt, rank, shares;                         // tiles of keys of this CTA, tiles that have rows, CTAs that share the block
    KvGroups keys;
    __device__ __forceinline__ void make(const KvArgs &a, int seq_, int block, int kvh_, const KvSeq &q, int tq, int n_tiles, int size, int rank_) {
        seq = seq_; kvh = kvh_; begin = q.begin; rows = q.n;
        t0 = block * n_tiles * tq;
        base_pos = q.len - q.n;
        keys = {0, 0, 0};
        if (seq >= 0) keys = kv_groups(base_pos + t0 > 0 ? base_pos + t0 : 0, top(tq, n_tiles), a.window, a.sinks);
        // CTAs that share the block: two tiles each at least, by the block's own tiles
        const int tiles = (keys.count + 3) / 4, log_shares = min(31 - __clz(size), tiles < 4 ? 0 : 30 - __clz(tiles));
        rank = rank_; shares = 1 << log_shares;
        n = rank < shares ? (tiles - rank + shares - 1) >> log_shares : 0;
        nt = n_tiles == 2 && t0 + tq < rows ? 2 : 1;
    }
    __device__ __forceinline__ int top(int tq, int n_tiles) const { return base_pos + min(t0 + n_tiles * tq, rows) - 1; }      // last key that any row sees
    __device__ __forceinline__ void write(volatile int *w) const {
        w[0] = seq; w[1] = kvh; w[2] = begin; w[3] = rows; w[4] = t0; w[5] = base_pos; w[6] = n; w[7] = nt; w[8] = shares;
        w[9] = keys.first; w[10] = keys.start; w[11] = keys.count;
    }
    __device__ __forceinline__ void read(const volatile int *w, int lane, int rank_) {
        // (one lane's values for all, so that the compiler keeps them and what follows from them in uniform registers)
        const int v = w[lane < WORDS ? lane : 0];
        auto word = [&](int i) { return __shfl_sync(0xffffffffu, v, i); };
        seq = word(0); kvh = word(1); begin = word(2); rows = word(3); t0 = word(4); base_pos = word(5); n = word(6); nt = word(7); shares = word(8);
        keys.first = word(9); keys.start = word(10); keys.count = word(11);
        rank = rank_;
    }
    __device__ __forceinline__ int tile_at(int i) const { return 4 * (rank + i * shares); }        // first group of the CTA's i-th tile,
    __device__ __forceinline__ int groups(int g0) const { return min(4, keys.count - g0); }        // and how many it has
};

// Four lanes' 16 words each, turned so that a lane's words 4 k to 4 k + 3 are its quarter of the words of the four lanes' k-th: lane q of
// the four gets words 4 q ... of lane k. Stores of rows then touch eight lines an instruction instead of 32.
__device__ __forceinline__ void kc_quads(uint32_t *w, int lane) {
#pragma unroll
    for (int step = 1; step < 4; step *= 2) {
        const bool up = lane & step;
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (!(k & step)) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t &lo = w[4 * k + e], &hi = w[4 * (k + step) + e];
                    const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? lo : hi, step);
                    if (up) lo = got; else hi = got;
                }
            }
    }
}

template <int DP, int FMT, bool MANY>
__global__ void __launch_bounds__(ChunkShape<DP, FMT>::THREADS, ChunkShape<DP, FMT>::PER_SM)
kv_chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const KvArgs a,
                int box_rows, int log_size, int longest_first, int tq, uint32_t inv_g, int most) {
    using Sh = ChunkShape<DP, FMT>;
    constexpr bool BF = FMT == KV_BF16, F32 = FMT == KV_F32, OWN_P = Sh::OWN_P;
    constexpr int STAGES = Sh::STAGES, TILES = Sh::TILES, SPLIT = Sh::SPLIT, OWN = Sh::OWN, GROUPS = OWN / 32;
    extern __shared__ uint8_t kc_raw[];
    uint8_t *head = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(kc_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *qst = head + Sh::HEAD, *ring = qst + Sh::Q;
    uint64_t *full = reinterpret_cast<uint64_t *>(head), *empty = full + STAGES, *q_full = empty + STAGES, *q_empty = q_full + 1, *s_full = q_empty + 1,
             *s_free = s_full + 2, *p_part = s_free + 2, *p_full = p_part + 2, *o_full = p_full + 2, *i_full = o_full + 2, *i_empty = i_full + 2,
             *drain = i_empty + 2, *pair = drain + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(pair + 4);
    volatile int *items = reinterpret_cast<volatile int *>(tmem_slot + 1);     // two blocks' words
    const int warp = warp_index(), lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
        if (!F32) tma_prefetch_desc(&tmQ);
        for (int s = 0; s < STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(q_full, F32 ? Sh::SOFT : 1); mbar_init(q_empty, 1);
        for (int t = 0; t < TILES; t++) {
            mbar_init(&s_full[t], 1); mbar_init(&o_full[t], 1);
            mbar_init(&s_free[t], 4 * SPLIT); mbar_init(&p_part[t], 4 * SPLIT); mbar_init(&p_full[t], 4 * SPLIT);
        }
        if (SPLIT == 2) for (int i = 0; i < 4; i++) mbar_init(&pair[i], 2);
        for (int i = 0; i < 2; i++) { mbar_init(&i_full[i], 1); mbar_init(&i_empty[i], Sh::SOFT + 1); }
        mbar_init(drain, 1);
        mbar_fence_init();
    }
    if (warp == Sh::W_MMA) { tc_alloc(tmem_slot, Sh::TMEM); tc_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    chain_trigger();
    chain_wait();
    const uint32_t tmem = *tmem_slot;
    auto by_g = [&](int x) { return (int)(((uint32_t)x * inv_g) >> 16); };
    const int size = 1 << log_size, rank = (int)blockIdx.x & (size - 1);
    const bool once = log_size > 0;                            // a cluster's CTAs work on one block and join their results
    // Everybody but the TMA warp: the CTA's j-th block, -1 as its sequence behind the last one, and -2 where it does not come
    auto next_block = [&](int j) {
        const bool got = mbar_wait_warp(&i_full[j & 1], (uint32_t)((j >> 1) & 1));
        KcBlock b;
        b.read(items + (j & 1) * KcBlock::WORDS, lane, rank);
        if (!got) { b.seq = -2; b.n = 0; }
        return b;
    };
    auto leave_block = [&](int j) {                            // its words are not needed any more
        __syncwarp();
        if (lane == 0) mbar_arrive(&i_empty[j & 1]);
    };
    // row of a softmax thread, in tile t; its keys and columns of a tile are those from half * OWN (half * DP / SPLIT) on
    const int t = TILES == 2 ? (warp >> 2) & 1 : 0, half = SPLIT == 2 ? (warp >> 2) & 1 : 0, r = (warp & 3) * 32 + lane;
    const bool soft = warp < Sh::SOFT;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16), s_at = trow + Sh::COL_S + t * 128, p_at = trow + Sh::COL_P + t * Sh::STEP_P,
                   o_at = trow + Sh::COL_O + t * DP, f_at = trow + Sh::COL_F + t * DP;
    float m = -INFINITY, l = 0.f;                              // of the row: running maximum and sum
    constexpr int COLS = F32 ? 16 : 32;                        // columns in 16 words
    auto result = [&](int n, int c, float *o) {                // COLS columns of the row's result over n tiles
        if constexpr (F32) {
            float f[32];
            tc_ld16(f_at + c, f);
            tc_ld16(n > 1 ? o_at + c : f_at + c, f + 16);
            kc_wait_ld32(f);
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] = n > 1 ? f[e] + f[e + 16] : f[e];
        } else {
            tc_ld32(f_at + c, o);
            kc_wait_ld32(o);
        }
    };

    if (!soft) {
    kc_regs_less<Sh::LESS>();                                  // (one instruction for the four warps)
    if (warp == Sh::W_TMA) {
        // ---- lane = one box of a tile: 64 of the D columns, the slots of one page. Item 2 i of the ring is K(i), 2 i + 1 V(i).
        const int shift = a.page_shift, boxes = (KC_KEYS >> (__ffs(box_rows) - 1)) * Sh::HALVES;
        const int b_half = lane % Sh::HALVES, b_sub = lane / Sh::HALVES;
        const uint32_t b_at = b_half * KC_HALF + b_sub * box_rows * 128;
        int x = (int)(blockIdx.x >> log_size), nth = x / a.Hkv;
        typename KcFind<MANY>::Type finder;
        finder.init(a, TILES * tq, most, lane);
        int s = 0, ph = 0, r = 0, queries = 0;                 // place in the ring, its parity, requests; blocks with queries so far
        bool ok = true;
        for (int j = 0, x0 = 0; ok; j++) {
            if (j >= 2 && !mbar_wait_warp(&i_empty[j & 1], (uint32_t)(((j >> 1) & 1) ^ 1))) { ok = false; break; }
            int seq, block;
            KvSeq sq;
            if constexpr (MANY) {
                for (;;) {
                    finder.find(a, nth, lane, &seq, &block, &sq);
                    if (seq >= 0 || nth >= most || once) break;
                    x0 += (int)gridDim.x;                      // a number without a block
                    x = x0 + (int)blockIdx.x;
                    nth = x / a.Hkv;
                }
            } else if (longest_first) finder.find_longest(a, nth, lane, &seq, &block, &sq);
            else finder.find(a, nth, lane, &seq, &block, &sq);
            KcBlock b;
            b.make(a, seq, block, x - nth * a.Hkv, sq, tq, TILES, size, rank);
            if (lane == 0) {
                b.write(items + (j & 1) * KcBlock::WORDS);
                mbar_arrive(&i_full[j & 1]);
            }
            __syncwarp();
            if (b.seq < 0) break;
            const int top = b.top(tq, TILES), low = b.base_pos + b.t0 - a.window + 1;       // last key that any row sees, and first that a window shows
            auto seen = [&](int j) { return j <= top && (a.window <= 0 || j + box_rows - 1 >= low || j < a.sinks); };
            auto key_of = [&](int i) { return b.keys.at(b.tile_at(i) + (b_sub * box_rows >> 5)) + (b_sub * box_rows & 31); };
            auto entry_of = [&](int i) -> int {
                const int j = key_of(i);
                return lane < boxes && i < b.n && seen(j) ? a.table[(size_t)b.seq * a.max_pages + (j >> shift)] : -1;
            };
            int entry = entry_of(0);
            if (!F32 && b.n > 0) {                             // 16-bit queries: rows as they lie are the tile's rows
                if (queries > 0 && !mbar_wait_warp(q_empty, (uint32_t)((queries - 1) & 1))) { ok = false; break; }
                if (lane == 0) mbar_expect_tx(q_full, (uint32_t)(b.nt * Sh::HALVES * 128 * tq * a.G));
                __syncwarp();
                if (lane < b.nt * Sh::HALVES)
                    kc_load_3d(qst + (lane / Sh::HALVES) * Sh::OPERAND + (lane % Sh::HALVES) * KC_HALF, &tmQ, (lane % Sh::HALVES) * 64, b.kvh * a.G,
                               b.begin + b.t0 + lane / Sh::HALVES * tq, q_full);
                queries++;
            }
            for (int i = 0; i < b.n && ok; i++) {
                const int next = entry_of(i + 1);
                const int j = key_of(i);
                if (lane < boxes && (unsigned)entry >= (unsigned)a.n_pages) {
                    if (seen(j)) kv_report(a, ST_PAGE);
                    entry = 0;                                 // any finite rows do
                }
                const int y = (int)kv_row(a, entry, b.kvh, j & ((1 << shift) - 1));
#pragma unroll
                for (int kv = 0; kv < 2; kv++) {
                    if (r >= STAGES && !mbar_wait_warp(&empty[s], (uint32_t)(ph ^ 1))) { ok = false; break; }
                    if (lane == 0) mbar_expect_tx(&full[s], Sh::OPERAND);
                    __syncwarp();
                    if (lane < boxes) tma_load_2d(ring + s * Sh::OPERAND + b_at, kv ? &tmV : &tmK, b_half * 64, y, &full[s]);
                    if (r < STAGES) r++;
                    if (++s == STAGES) { s = 0; ph ^= 1; }
                }
                entry = next;
            }
            if (once) break;
            // (there and back: a CTA whose block was the longest of its round gets the shortest of the next)
            x0 += (int)gridDim.x;
            x = x0 + (longest_first && !(j & 1) ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x);
            nth = x / a.Hkv;
        }
        if (!ok && lane == 0) kv_report(a, ST_TIMEOUT_PRODUCER);
        if (MANY) kv_look_over(a, lane, (int)blockIdx.x, (int)gridDim.x);
        for (int u = 0; u < STAGES && u < r; u++) {            // what was asked for has to land before the CTA leaves
            if (s == 0) { s = STAGES; ph ^= 1; }
            if (!mbar_wait_warp(&full[--s], (uint32_t)ph)) break;
        }
        if (!F32 && queries > 0) mbar_wait_warp(q_full, (uint32_t)((queries - 1) & 1));
    } else if (warp == Sh::W_MMA) {
        const uint32_t idesc_o = kc_idesc(BF, a.D) | (1u << 16);       // V: MN-major
        const uint64_t qdesc = umma_desc_sw128(smem_u32(qst)), kdesc = umma_desc_sw128(smem_u32(ring)), vdesc = kc_desc_mn(smem_u32(ring));
        const int steps = a.D / 16;
        auto issue_s = [&](int t, int s, int hi) {             // by one lane: the scores of the first 32 hi keys
            const uint64_t kd = kdesc + (uint64_t)((s * Sh::OPERAND) >> 4);
            const uint32_t idesc = kc_idesc(BF, 32 * hi);
#pragma unroll
            for (int plane = Sh::PLANES - 1; plane >= 0; plane--) {            // (the small products first: every sum is cut to the accumulator's bits)
                const uint64_t qd = qdesc + (uint64_t)(((t * Sh::PLANES + plane) * Sh::OPERAND) >> 4);
#pragma unroll
                for (int kk = 0; kk < DP / 16; kk++) {
                    const uint64_t ko = (uint64_t)(((kk >> 2) * KC_HALF + (kk & 3) * 32) >> 4);
                    if (kk < steps) tc_mma_f16(tmem + Sh::COL_S + t * 128, qd + ko, kd + ko, idesc, kk != 0 || plane != Sh::PLANES - 1);
                }
            }
        };
        // groups [k0, k1) of P V, again the small products first; the first one begins the sum
        auto issue_o = [&](int t, int s, int k0, int k1, bool begins) {
            const uint64_t vd = vdesc + (uint64_t)((s * Sh::OPERAND) >> 4);
#pragma unroll
            for (int plane = Sh::PLANES - 1; plane >= 0; plane--)
                for (int k = k0; k < k1; k++) {
#pragma unroll
                    for (int b = 0; b < 2; b++)
                        kc_mma_ts(tmem + Sh::COL_F + t * DP, tmem + Sh::COL_P + t * Sh::STEP_P + plane * 64 + 16 * k + 8 * b,
                                  vd + (uint64_t)((k * 4096 + b * 2048) >> 4), idesc_o, !begins || k != 0 || b != 0 || plane != Sh::PLANES - 1);
                }
        };
        int s = 0, ph = 0;                                     // ring place of the next item
        auto take = [&](int *at) {                             // waits for the next item
            *at = s;
            const bool got = mbar_wait_warp(&full[s], (uint32_t)ph);
            if (++s == STAGES) { s = 0; ph ^= 1; }
            return got;
        };
        int done0 = 0, done1 = 0, queries = 0;                 // tiles of keys behind each tile of rows; blocks with queries so far
        bool ok = true;
        for (int j = 0; ok; j++) {
            const KcBlock b = next_block(j);
            if (b.seq < 0) { ok = b.seq == -1; break; }
            leave_block(j);
            const int n = b.n, nt = b.nt;
            if (n > 0) {
                int sk = 0, sv = 0, hi = b.groups(b.tile_at(0));
                ok = mbar_wait_warp(q_full, (uint32_t)(queries & 1)) && take(&sk);
                queries++;
                if (ok) {
                    tc_fence_after();
                    if (elect_one()) {
                        for (int t = 0; t < nt; t++) { issue_s(t, sk, hi); tc_commit(&s_full[t]); }
                        tc_commit(&empty[sk]);
                    }
                    __syncwarp();
                    ok = take(&sv);
                }
                // An issued product keeps the pipe busy for 60 clocks, a wait that has come true costs as much: the waits stand where
                // products are still under way.
                for (int i = 0; i < n && ok; i++) {
                    const bool more = i + 1 < n;
                    const int v = sv, hi2 = more ? b.groups(b.tile_at(i + 1)) : 4;
                    const bool begins = i == 0 || Sh::FRESH;
                    if (OWN_P && more) {
                        ok = take(&sk);
                        for (int t = 0; t < nt && ok; t++) {
                            if (!mbar_wait_warp(&s_free[t], (uint32_t)(((t ? done1 : done0) + i) & 1))) { ok = false; break; }
                            tc_fence_after();
                            if (elect_one()) {
                                issue_s(t, sk, hi2); tc_commit(&s_full[t]);
                                if (t == nt - 1) tc_commit(&empty[sk]);
                            }
                            __syncwarp();
                        }
                    }
                    for (int t = 0; t < nt && ok; t++) {
                        if (!mbar_wait_warp(&p_part[t], (uint32_t)(((t ? done1 : done0) + i) & 1))) { ok = false; break; }
                        tc_fence_after();
                        if (elect_one()) issue_o(t, v, 0, min(hi, KC_PART), begins);
                        __syncwarp();
                        if (more && !OWN_P && t == 0 && !take(&sk)) { ok = false; break; }     // K(i + 1)
                        if (more && t == nt - 1 && !take(&sv)) { ok = false; break; }          // V(i + 1)
                        if (!mbar_wait_warp(&p_full[t], (uint32_t)(((t ? done1 : done0) + i) & 1))) { ok = false; break; }
                        tc_fence_after();
                        if (elect_one()) {
                            issue_o(t, v, KC_PART, hi, begins);
                            if (OWN_P || !more) tc_commit(&o_full[t]);
                            if (more && !OWN_P) { issue_s(t, sk, hi2); tc_commit(&s_full[t]); }
                            if (t == nt - 1) {
                                tc_commit(&empty[v]);
                                if (more && !OWN_P) tc_commit(&empty[sk]);
                                if (!more) tc_commit(q_empty);
                            }
                        }
                        __syncwarp();
                    }
                    hi = hi2;
                }
                done0 += n;
                if (nt == 2) done1 += n;
            }
            if (once) break;
        }
        if (!ok) {                                             // nothing may run on when tensor memory is given back
            if (lane == 0) kv_report(a, ST_TIMEOUT_MMA);
            if (elect_one()) tc_commit(drain);
            __syncwarp();
            mbar_wait_warp(drain, 0);
        }
    }
    } else {
    // ---- softmax: thread = row
    kc_regs_more<Sh::MORE>();
    const float sc = a.scale2;
    bool ok = true;
    int done = 0, blocks = 0;                                  // tiles of keys, and blocks, behind this tile of rows
    // The two threads of a row exchange a value; false where the other one's does not come
    float *told = reinterpret_cast<float *>(head + KC_HEAD);
    int turn = 0;
    auto exchange = [&](float mine, float *other) {
        float *at = told + (turn & 1) * 256 + r;
        at[half * 128] = mine;
        __syncwarp();
        if (lane == 0) mbar_arrive(&pair[warp & 3]);
        const bool got = mbar_wait_warp(&pair[warp & 3], (uint32_t)(turn & 1));
        *other = at[(half ^ 1) * 128];
        turn++;
        return got;
    };
    for (int j = 0; ok; j++) {
        const KcBlock b = next_block(j);
        if (b.seq < 0) { ok = b.seq == -1; break; }
        const int n = b.n, tok = b.t0 + t * tq + by_g(r);
        if (F32 && n > 0) {
                // the warp's 32 (or 16) rows, neighbouring lanes on neighbouring pieces of eight values
                constexpr int PIECES = DP / 8, ROWS = 32 / PIECES, ROUNDS = 32 / SPLIT / ROWS, BATCH = 8;
                uint8_t *qt = qst + t * Sh::PLANES * Sh::OPERAND;
                const int c = lane % PIECES, row0 = (warp & 3) * 32 + half * (32 / SPLIT);
                bool bad = false;
                if (t < b.nt) {
#pragma unroll 1
                    for (int u = 0; u < ROUNDS; u += BATCH) {
                        float4 in[BATCH][2];
#pragma unroll
                        for (int i = 0; i < BATCH; i++) {
                            const int row = row0 + (u + i) * ROWS + lane / PIECES, pl = by_g(row), at = b.t0 + t * tq + pl;
                            in[i][0] = in[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (row < tq * a.G && at < b.rows && c * 8 < a.D) {
                                const float4 *p = reinterpret_cast<const float4 *>(static_cast<const float *>(a.q) + (int64_t)(b.begin + at) * a.ldq +
                                                                                   (int64_t)(b.kvh * a.G + row - pl * a.G) * a.D + c * 8);
                                in[i][0] = p[0]; in[i][1] = p[1];
                            }
                        }
#pragma unroll
                        for (int i = 0; i < BATCH; i++) {
                            const int row = row0 + (u + i) * ROWS + lane / PIECES;
                            uint8_t *to = qt + (c >> 3) * KC_HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4);
                            const float *f = reinterpret_cast<const float *>(in[i]);
                            uint4 hi, lo;
#pragma unroll
                            for (int e = 0; e < 8; e++) bad |= !(fabsf(f[e]) < H16_MAX) && b.base_pos + b.t0 + t * tq + by_g(row) >= 0;
                            kv_split(f[0], f[1], hi.x, lo.x); kv_split(f[2], f[3], hi.y, lo.y); kv_split(f[4], f[5], hi.z, lo.z); kv_split(f[6], f[7], hi.w, lo.w);
                            *reinterpret_cast<uint4 *>(to) = hi;
                            *reinterpret_cast<uint4 *>(to + Sh::OPERAND) = lo;
                        }
                    }
                    if (bad) kv_report(a, ST_RANGE);
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // generic-proxy stores -> visible to the tensor core
                }
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        m = -INFINITY; l = 0.f;
        float base = ChunkTop<FMT>::TOP;                       // 16-bit rows: that of m; and whether one of the warp's is far
        bool far = false;
        if (t < b.nt) {
            // rows that do not exist take the last one's position, so that they need no mask of their own
            const int pos = b.base_pos + min(r < tq * a.G ? tok : b.t0 + t * tq, b.rows - 1);
            auto gather = [&](int i, float alpha) {                // O = (O + P(i - 1) V) alpha
#pragma unroll 1
                for (int c = half * (DP / 32 / SPLIT); c < (half + 1) * (DP / 32 / SPLIT); c++) {
                    float f[32], o[32];
                    tc_ld32(f_at + 32 * c, f);
                    tc_ld32(i > 1 ? o_at + 32 * c : f_at + 32 * c, o);
                    kc_wait_ld32(f); kc_wait_ld32(o);
#pragma unroll
                    for (int e = 0; e < 32; e++) f[e] = (i > 1 ? f[e] + o[e] : f[e]) * alpha;
                    kc_st16(o_at + 32 * c, reinterpret_cast<const uint32_t *>(f));
                    kc_st16(o_at + 32 * c + 16, reinterpret_cast<const uint32_t *>(f + 16));
                }
            };
            for (int i = 0; i < n && ok; i++) {
                if (!mbar_wait_warp(&s_full[t], (uint32_t)((done + i) & 1))) { ok = false; break; }
                tc_fence_after();
                if (Sh::FRESH && !OWN_P && i > 0) gather(i, 1.f);  // (while the scores take no registers)
                float x[OWN], m4[4];
                const uint32_t x_at = s_at + half * OWN;
                tc_ld32(x_at, x);
                tc_ld32(x_at + 32, x + 32);
                kc_wait_ld32(x); kc_wait_ld32(x + 32);
                if (OWN == 128) { tc_ld32(x_at + 64, x + OWN - 64); tc_ld32(x_at + 96, x + OWN - 32); }
#pragma unroll
                for (int e = 0; e < 4; e++) m4[e] = x[e];
#pragma unroll
                for (int c = 4; c < 60; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; e++) m4[e] = fmaxf(m4[e], fmaxf(x[c + e], x[c + 4 + e]));
#pragma unroll
                for (int e = 0; e < 4; e++) m4[e] = fmaxf(m4[e], x[60 + e]);
                if (OWN == 128) { kc_wait_ld32(x + OWN - 64); kc_wait_ld32(x + OWN - 32); }
                if (OWN_P) {                                       // the scores are in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_free[t]);
                }
#pragma unroll
                for (int c = 64; c < OWN; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; e++) m4[e] = fmaxf(m4[e], fmaxf(x[c + e], x[c + 4 + e]));
                const int g0 = b.tile_at(i), j0 = b.keys.at(g0), d = pos - j0;
                const bool whole = d >= KC_KEYS - 1 && (a.window <= 0 || (d < a.window && (g0 >= b.keys.first || g0 + 4 <= b.keys.first)) || j0 + KC_KEYS - 1 < a.sinks);
                if (!__all_sync(0xffffffffu, whole)) {             // (columns that have no scores are hidden, too)
                    // 32 columns at a time, where some row of the warp does not see them all: a bit per column, visible up to the row's
                    // position, and with a window behind its lower end or among the first tokens
                    auto upto = [](int c) -> uint32_t { return c < 0 ? 0u : c >= 31 ? 0xffffffffu : (2u << c) - 1u; };      // bits 0 to c
                    m4[0] = m4[1] = m4[2] = m4[3] = -INFINITY;
#pragma unroll
                    for (int w = 0; w < GROUPS; w++) {
                        const int jw = b.keys.at(g0 + half * GROUPS + w), dw = pos - jw;
                        const uint32_t see = upto(dw) & (~upto(a.window > 0 ? dw - a.window : -1) | upto(a.sinks - 1 - jw));
                        if (!__all_sync(0xffffffffu, see == 0xffffffffu)) {
#pragma unroll
                            for (int c = 0; c < 32; c++)
                                if (!(see >> c & 1)) x[32 * w + c] = -INFINITY;
                        }
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
#pragma unroll
                            for (int e = 0; e < 4; e++) m4[e] = fmaxf(m4[e], fmaxf(x[32 * w + c + e], x[32 * w + c + 4 + e]));
                    }
                }
                float mt = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                if (SPLIT == 2) {
                    float other;
                    if (!exchange(mt, &other)) { ok = false; break; }
                    mt = fmaxf(mt, other);
                }
                if (OWN_P && i > 0) {                              // P(i - 1) has been read, and O is at rest
                    if (!mbar_wait_warp(&o_full[t], (uint32_t)((done + i - 1) & 1))) { ok = false; break; }
                    tc_fence_after();
                }
                const bool grow = (mt - m) * sc > ChunkTop<FMT>::LAG;      // (not where both are -infinity)
                const bool any = __any_sync(0xffffffffu, grow);
                if (any || (Sh::FRESH && OWN_P)) {
                    const float alpha = grow ? kv_ex2((m - mt) * sc) : 1.f;
                    if (grow) m = mt;
                    l *= alpha;
                    if (!F32) {
                        base = kv_base(m, sc, ChunkTop<FMT>::TOP);
                        far = __any_sync(0xffffffffu, kv_far(base));
                    }
                    if (Sh::FRESH && OWN_P && i > 0) {
                        gather(i, alpha);
                    } else if (i > 0) {
                        if (Sh::FRESH) kc_wait_st();
#pragma unroll 1
                        for (int c = 0; c < DP / 16; c++) {
                            float o[16];
                            tc_ld16(o_at + 16 * c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] *= alpha;
                            kc_st16(o_at + 16 * c, reinterpret_cast<const uint32_t *>(o));
                        }
                    }
                }
                const float off = m == -INFINITY ? 0.f : -m;       // (no key yet: all are hidden)
                const float2 sc2 = kv_twice(sc), off2 = kv_twice(off);
                float2 top2 = kv_twice(F32 ? ChunkTop<FMT>::TOP : base);
                if (__builtin_expect(!F32 && far, 0)) {
                    const float2 o = kv_twice(kv_far(base) ? off : 0.f);
#pragma unroll
                    for (int c = 0; c < OWN; c += 2) {
                        const float2 y = kv_add2(make_float2(x[c], x[c + 1]), o);
                        x[c] = y.x; x[c + 1] = y.y;
                    }
                    if (kv_far(base)) top2 = kv_twice(ChunkTop<FMT>::TOP);
                }
                float2 l2[2] = {{0.f, 0.f}, {0.f, 0.f}};           // the tile's sum: small terms are not lost one by one in a large l
                auto open = [&](int c) {                           // the exponentials of 16 keys, in place
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        float *v = x + c * 16 + 2 * e;
                        const float2 y = kv_fma2(F32 ? kv_add2(make_float2(v[0], v[1]), off2) : make_float2(v[0], v[1]), sc2, top2);
                        v[0] = kv_ex2(y.x); v[1] = kv_ex2(y.y);
                    }
                };
                auto close = [&](int c) {                          // summed, packed and stored
                    uint32_t hi[8], lo[F32 ? 8 : 1];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const float *v = x + c * 16 + 2 * e;
                        l2[e & 1] = kv_add2(l2[e & 1], make_float2(v[0], v[1]));
                        if (F32) kv_split(v[0], v[1], hi[e], lo[F32 ? e : 0]);
                        else hi[e] = kv_pack<BF>(v[0], v[1]);
                    }
                    kc_st8(p_at + half * (OWN / 2) + 8 * c, hi);
                    if (F32) kc_st8(p_at + 64 + half * (OWN / 2) + 8 * c, lo);
                };
                auto ready = [&](uint64_t *bar) {
                    kc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar);
                };
                // some keys' exponentials are under way while those before are summed, packed and stored
                const int hi = b.groups(g0) - half * GROUPS, part = KC_PART - half * GROUPS;      // of the thread's groups: those with keys; the first signal's
                if (hi >= GROUPS) {
#pragma unroll
                    for (int c = 0; c <= 2 * GROUPS; c++) {
                        if (c < 2 * GROUPS) open(c);
                        if (c > 0) close(c - 1);
                        if (c == 2 * min(part, GROUPS)) ready(&p_part[t]);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c <= GROUPS; c++) {
                        if (c < GROUPS && c < hi) { open(2 * c); open(2 * c + 1); }
                        if (c > 0 && c <= hi) { close(2 * c - 2); close(2 * c - 1); }
                        if (c == min(part, GROUPS)) ready(&p_part[t]);
                    }
                }
                ready(&p_full[t]);
                l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
            }
            if (n > 0 && ok) ok = mbar_wait_warp(&o_full[t], (uint32_t)(OWN_P ? (done + n - 1) & 1 : blocks & 1));
            if (n > 0) { done += n; blocks++; }
            tc_fence_after();
            if (SPLIT == 2 && n > 0 && ok) {
                float other;
                ok = exchange(l, &other);
                l += other;
            }
            // (what the results need of the block is read again, so that it takes no registers above)
            const volatile int *w = items + (j & 1) * KcBlock::WORDS;
            if (w[8] == 1 && rank == 0 && ok) {
                const float inv = l != 0.f ? 1.f / l : 0.f;
                if (!kv_sound(l)) {
                    const int mine = w[4] + t * tq + by_g(r);  // the thread's row in its sequence
                    if (r < tq * a.G && mine < w[3] && w[5] + mine >= 0) kv_report(a, ST_RANGE);
                }
                // after the turn a lane stores a quarter of 16 words of each of the four rows of its lanes: where they lie, -1 for rows that are not
                const int begin = w[2], last = w[3] - w[4] - t * tq, kvh = w[1];       // (rows of the tile: below last)
                const int64_t first = (int64_t)(begin + w[4] + t * tq) * a.ldo + (int64_t)kvh * a.G * a.D;
                int64_t to[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int row = (r & ~3) + k, pl = by_g(row);
                    to[k] = row < tq * a.G && pl < last ? first + pl * a.ldo + (row - pl * a.G) * a.D : -1;
                }
#pragma unroll 1
                for (int c = half * (DP / COLS / SPLIT); c < (half + 1) * (DP / COLS / SPLIT); c++) {
                    float o[COLS];
                    if (n > 0) result(n, c * COLS, o);
                    uint32_t v[16];
#pragma unroll
                    for (int u = 0; u < 16; u++) {
                        if (F32) v[u] = __float_as_uint(inv != 0.f ? o[u] * inv : 0.f);
                        else v[u] = inv != 0.f ? kv_pack_result<BF>(o[2 * u] * inv, o[2 * u + 1] * inv) : 0u;
                    }
                    kc_quads(v, lane);
                    const int col = c * COLS + (lane & 3) * (COLS / 4);
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        if (to[k] >= 0 && col < a.D)
                            *reinterpret_cast<uint4 *>(static_cast<uint8_t *>(a.out) + (to[k] + col) * (F32 ? 4 : 2)) = make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
                }
                tc_fence_before();                             // (the next block's products are ordered behind these loads by its P)
            }
        }
        leave_block(j);
        if (once) break;
    }
    if (!ok && lane == 0) kv_report(a, ST_TIMEOUT_EPILOGUE);
    }
    __syncwarp();
    if (once) {
        __syncthreads();                                       // (the TMA warp has written the block's words)
        KcBlock b;
        b.read(items, lane, rank);
        if (b.shares > 1) {
            // parts of the rows' results and (maximum, sum) of each, where queries and tiles were; then the weights of the parts, and their sum
            // by all CTAs of the cluster, each for its rows
            float *part = reinterpret_cast<float *>(qst), *weight = part + TILES * 128 * (Sh::LDO + 2);
            float2 *ml = reinterpret_cast<float2 *>(part + TILES * 128 * Sh::LDO);
            __syncthreads();                                       // (both tiles' products have been waited for)
            if (soft && t < b.nt && b.n > 0) {
                float *row = part + (t * 128 + r) * Sh::LDO;
#pragma unroll 1
                for (int c = half * (DP / SPLIT); c < (half + 1) * (DP / SPLIT); c += COLS) {
                    float o[COLS];
                    result(b.n, c, o);
#pragma unroll
                    for (int e = 0; e < COLS; e += 4) *reinterpret_cast<float4 *>(row + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
                if (half == 0) ml[t * 128 + r] = make_float2(m, l);
            }
            kv_cluster_sync();
            const uint32_t part0 = smem_u32(part), ml0 = smem_u32(ml);
            const int per_tile = tq * a.G, rows = min((min(b.t0 + TILES * tq, b.rows) - b.t0) * a.G, b.nt * per_tile), share = (rows + size - 1) >> log_size;
            const int v0 = rank * share, mine = max(0, min(share, rows - v0)), quads = a.D / 4;
            auto place_of = [&](int v) { return v < per_tile ? v : 128 + v - per_tile; };
            for (int v = threadIdx.x; v < mine; v += Sh::THREADS) {
                const int at = place_of(v0 + v);
                float2 e[16];
                float top_m = -INFINITY, total = 0.f;
#pragma unroll
                for (int p = 0; p < 16; p++) {
                    e[p] = make_float2(-INFINITY, 0.f);
                    if (p < b.shares) e[p] = kv_peer2(kv_peer(ml0 + at * 8, p));
                }
#pragma unroll
                for (int p = 0; p < 16; p++) top_m = fmaxf(top_m, e[p].x);
#pragma unroll
                for (int p = 0; p < 16; p++) {
                    e[p].x = kv_weight(e[p].x, top_m, a.scale2);
                    total = fmaf(e[p].x, e[p].y, total);
                }
                const float inv = total != 0.f ? 1.f / total : 0.f;
                if (!kv_sound(total) && b.base_pos + b.t0 + by_g(v0 + v) >= 0) kv_report(a, ST_RANGE);
#pragma unroll
                for (int p = 0; p < 16; p++)
                    if (p < b.shares) weight[v * 16 + p] = e[p].x * inv;
            }
            __syncthreads();
            for (int u = threadIdx.x; u < mine * quads; u += Sh::THREADS) {
                const int v = u / quads, c = (u - v * quads) * 4, at = place_of(v0 + v);
                float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int p0 = 0; p0 < b.shares; p0 += 4) {
                    float4 o[4];
#pragma unroll
                    for (int p = 0; p < 4; p++) {
                        o[p] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (p0 + p < b.shares) o[p] = kv_peer4(kv_peer(part0 + (at * Sh::LDO + c) * 4, p0 + p));
                    }
#pragma unroll
                    for (int p = 0; p < 4; p++)
                        if (p0 + p < b.shares) {
                            const float w = weight[v * 16 + p0 + p];
                            sum.x = fmaf(w, o[p].x, sum.x); sum.y = fmaf(w, o[p].y, sum.y); sum.z = fmaf(w, o[p].z, sum.z); sum.w = fmaf(w, o[p].w, sum.w);
                        }
                }
                const int pl = by_g(v0 + v);
                const int64_t to = (int64_t)(b.begin + b.t0 + pl) * a.ldo + (int64_t)(b.kvh * a.G + v0 + v - pl * a.G) * a.D + c;
                if (F32) *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + to) = sum;
                else *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.out) + to) = make_uint2(kv_pack_result<BF>(sum.x, sum.y), kv_pack_result<BF>(sum.z, sum.w));
            }
            kv_cluster_sync();                                     // nobody leaves while its part is being read
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == Sh::W_MMA) tc_dealloc(tmem, Sh::TMEM);
}

// Clusters of 2^k CTAs that run at a time on the current device with a CTA per SM; -1 with the error set
template <int DP, int FMT, bool MANY>
static int most_clusters(int k) {
    using Sh = ChunkShape<DP, FMT>;
    static PerDevice known[5] = {};                            // (the number and one)
    int dev = 0;
    if (!known[k].below(1, &dev)) return (int)known[k].v[dev] - 1;
    cudaLaunchConfig_t lc = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 1u << k; at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    lc.gridDim = dim3(1u << k); lc.blockDim = dim3(Sh::THREADS); lc.dynamicSmemBytes = Sh::SMEM;
    lc.attrs = at; lc.numAttrs = 1;
    int n = 0;
    MB_CUDA(cudaOccupancyMaxActiveClusters(&n, kv_chunk_kernel<DP, FMT, MANY>, &lc));
    known[k].record(dev, (size_t)n + 1);
    return n;
}

template <int DP, int FMT, bool MANY>
static int chunk_launch(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, int box_rows, cudaStream_t st) {
    using Sh = ChunkShape<DP, FMT>;
    auto kernel = kv_chunk_kernel<DP, FMT, MANY>;
    static PerDevice configured = {};
    int dev = 0;
    if (configured.below((size_t)Sh::SMEM, &dev)) {
        cudaFuncAttributes at;
        MB_CUDA(cudaFuncGetAttributes(&at, kernel));
        if (at.numRegs < Sh::REGS) { set_error("kv_attend: the kernel was built with %d registers, not %d", at.numRegs, Sh::REGS); return -1; }
        MB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM));
        MB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        configured.record(dev, (size_t)Sh::SMEM);
    }
    const int tq = KC_ROWS / a.G, per_block = Sh::TILES * tq;                  // positions of a tile of rows, of a block
    const uint32_t inv_g = (65536u + a.G - 1) / a.G;           // x / G = x inv_g / 2^16 for x < 256, G <= 64
    const int64_t full = ((int64_t)a.n_rows + per_block - 1) / per_block, seqs = a.n_seq < a.n_rows ? a.n_seq : a.n_rows;
    const int64_t most = a.n_rows / per_block + (MANY ? a.n_seq : seqs), blocks = most * a.Hkv;      // the last block of each sequence may be short
    // Clusters where the blocks that are likely (whole ones, or one per sequence) leave SMs without work: the largest of which as many
    // run at a time (with one CTA per SM a GPU of 148 has room for fewer than eight clusters of 16)
    const int64_t likely = (full > seqs ? full : seqs) * a.Hkv;
    int log_size = 0;
    for (int k = 1; k <= 4 && (int64_t)KC_KEYS << k < ((int64_t)a.max_pages << a.page_shift); k++) {
        const int most = most_clusters<DP, FMT, MANY>(k);
        if (most < 0) return -1;
        if (likely <= (int64_t)Sh::PER_SM * most) log_size = k;
    }
    if (blocks << log_size > 0x3fffffff) { set_error("kv_attend: too many rows in one call"); return -1; }
    // As many CTAs as fit take one block after the other, the longest first (us, that way and with a CTA per block, heads of 128: 4 x 2000 rows
    // 141, 172, 2 x 4000 237, 270, 8000 440, 460, 9 of 300 to 8000 550, 640). With more sequences than lanes, where the lengths are not
    // put in order, only blocks that are short: the hardware deals out long ones better (40 of 100 to 8000 F32 rows 1723, 1645)
    const int64_t keys = (int64_t)a.max_pages << a.page_shift, seen = (int64_t)a.window + a.sinks + per_block;
    const bool stay = a.n_seq <= KC_LANES || (a.window > 0 && seen < keys ? seen : keys) <= KC_STAY;
    const int64_t room = (int64_t)Sh::PER_SM * device_sm_count();
    const int64_t ctas = log_size ? blocks << log_size : stay && blocks > room ? room : blocks;
    const bool longest_first = !MANY && blocks > room && a.n_seq <= KC_LANES;
    CUtensorMap q = k;
    if (FMT != KV_F32 && !kv_rows_map(&q, a, FMT == KV_BF16)) { set_error("kv_attend: no tensor map of the rows"); return -1; }
    MB_CUDA(launch_kernel(kernel, dim3((unsigned)ctas), dim3(Sh::THREADS), (size_t)Sh::SMEM, st, true, 1 << log_size, q, k, v, a, box_rows, log_size, longest_first ? 1 : 0,
                          tq, inv_g, (int)most));
    note_launch();
    return 0;
}

template <int DP, int FMT>
static int chunk_find(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, int box_rows, cudaStream_t st) {
    // (up to here 256 sequences that all claim all rows have fewer blocks than 31 bits)
    const bool many = a.n_seq > KC_COUNT || a.n_rows >= 1 << 22;
    return many ? chunk_launch<DP, FMT, true>(k, v, a, box_rows, st) : chunk_launch<DP, FMT, false>(k, v, a, box_rows, st);
}

int kv_chunk(const CUtensorMap &k, const CUtensorMap &v, const KvArgs &a, int box_rows, int fmt, cudaStream_t st) {
    if (a.D <= 64)
        return fmt == KV_F32 ? chunk_find<64, KV_F32>(k, v, a, box_rows, st) : fmt == KV_F16 ? chunk_find<64, KV_F16>(k, v, a, box_rows, st)
                                                                                        : chunk_find<64, KV_BF16>(k, v, a, box_rows, st);
    return fmt == KV_F32 ? chunk_find<128, KV_F32>(k, v, a, box_rows, st) : fmt == KV_F16 ? chunk_find<128, KV_F16>(k, v, a, box_rows, st)
                                                                                     : chunk_find<128, KV_BF16>(k, v, a, box_rows, st);
}

}  // namespace mb
