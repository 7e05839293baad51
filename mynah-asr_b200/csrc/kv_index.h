// Where the rows of a call lie in a paged key/value cache: index arithmetic of the kv kernels, free of CUDA so that the tests
// can compile it for the host. Tables come from the caller's device memory; nothing here trusts them.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define MB_HD __host__ __device__ __forceinline__
#else
#define MB_HD inline
#endif

namespace mb {

// One sequence of a call: its rows [begin, begin + n) stand at the positions [len - n, len).
struct KvSeq {
    int begin, n, len;
};
// Rows and keys of sequence s as its tables say; false where they contradict the call's sizes (n = len = 0 then).
// row_off null: one row per sequence.
MB_HD bool kv_seq(const int *row_off, const int *kv_len, int s, int n_rows, int64_t capacity, KvSeq *q) {
    int64_t begin = s, n = 1;
    if (row_off) { begin = row_off[s]; n = row_off[s + 1] - begin; }
    const int len = kv_len[s];
    const bool ok = begin >= 0 && n >= 0 && begin + n <= n_rows && len >= 0 && (int64_t)len <= capacity;
    q->begin = ok ? (int)begin : 0;
    q->n = ok ? (int)n : 0;
    q->len = ok ? len : 0;
    return ok;
}

// The positions a row sees: j <= pos, and with a window j > pos - window or j < sinks.
MB_HD bool kv_sees(int pos, int j, int window, int sinks) {
    return j <= pos && (window <= 0 || j > pos - window || j < sinks);
}

// The tiles of `tile` keys that rows at the positions [pos0, pos1] look at between them, as one row of numbers: tiles [0, head) of
// the first tokens, then those from `from` on. count = 0 where no key is visible.
struct KvTiles {
    int head, from, count;
    MB_HD int at(int i) const { return i < head ? i : from + (i - head); }
};
MB_HD KvTiles kv_tiles(int pos0, int pos1, int window, int sinks, int tile) {
    KvTiles t = {0, 0, 0};
    if (pos1 < 0) return t;
    const int last = pos1 / tile;
    if (window > 0) {
        const int64_t low = (int64_t)pos0 - window + 1;
        if (low > 0) {
            t.from = (int)(low / tile);
            if (t.from > last) t.from = last;
            const int s = sinks < pos1 + 1 ? sinks : pos1 + 1;
            t.head = s > 0 ? (s - 1) / tile + 1 : 0;
            if (t.head >= t.from) { t.head = 0; t.from = 0; }      // the two meet: one run of tiles
        }
    }
    t.count = t.head + last + 1 - t.from;
    return t;
}

// The same in groups of 32 keys: groups [0, first) of the first tokens, then those from the position `start` on. Tiles are cut from the
// row of groups, so that a few first tokens take no tile of their own, and a window's first tile begins where the window does.
struct KvGroups {
    int first, start, count;
    MB_HD int at(int g) const { return g < first ? 32 * g : start + 32 * (g - first); }     // first position of group g
};
MB_HD KvGroups kv_groups(int pos0, int pos1, int window, int sinks) {
    KvGroups t = {0, 0, 0};
    if (pos1 < 0) return t;
    if (window > 0) {
        const int64_t low = (int64_t)pos0 - window + 1;
        if (low > 0) {
            const int s = sinks < pos1 + 1 ? sinks : pos1 + 1;
            t.start = (int)(low < pos1 ? low : pos1) & ~31;
            t.first = s > 0 ? (s - 1) / 32 + 1 : 0;
            if (t.first >= t.start / 32) { t.first = 0; t.start = 0; }             // the two meet
        }
    }
    t.count = t.first + (pos1 - t.start) / 32 + 1;
    return t;
}

}  // namespace mb
