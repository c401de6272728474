// kv4_index.h -- where the paged 4-bit KV cache keeps a value, which position a batch row stands for, and the page
// bookkeeping.  Plain C++ (no CUDA headers): the kernels use the index functions on the device, the C entries the page
// table of reference counts on the host, and both are checked on the CPU by the tests.
//
// A unit holds 64 positions of one (page, layer, KV head); a page is its layers' and heads' units one after the other, so
// that a page is one contiguous piece of memory.  A unit of head width hd (a multiple of 32, at most 256; NG = hd / 32
// groups) is 72 hd bytes:
//     K codes  64 rows of hd / 2 bytes       row t: four chunks of 4 NG bytes, chunk j word g = dims 32 g + 8 j .. + 7,
//                                            dim 32 g + 8 j + i in nibble i
//     K steps  64 x NG f16                   [t][g]
//     V codes  4 blocks of 16 positions      [block][half][lane = 4 r + j][g] words: positions 16 block + 8 half + 2 j (low
//                                            16 bits) and + 1 (high 16 bits), dims 32 g + 4 r + i in nibble i
//     V steps  64 x NG f16                   [t][g]
// Both orders are the operand fragments of the 16-bit matrix instruction: lane 4 r + j of a warp reads consecutive bytes
// (16 of them for hd = 128), and one mask of such a word leaves two operand values, two dims of a key row or the same
// dim of two positions.  A position owns its 16-bit pieces alone, so storing one never touches a neighbour's bits.
#pragma once
#include <stdint.h>
#include <stddef.h>
#include <algorithm>
#include <vector>
#ifdef __CUDACC__
#define KV4_HD __host__ __device__ __forceinline__
#else
#define KV4_HD inline
#endif

constexpr int KV4_PAGE = 64;

struct Kv4Geom {
    int layers, KV, hd, pages;
};
KV4_HD size_t kv4_unit_bytes(int hd) { return (size_t)72 * hd; }
KV4_HD size_t kv4_page_bytes(const Kv4Geom &g) { return kv4_unit_bytes(g.hd) * g.KV * g.layers; }
// first byte of the unit of (page, layer, head); page must have passed kv4_page_ok
KV4_HD size_t kv4_unit_off(const Kv4Geom &g, int page, int layer, int head) {
    return (size_t)page * kv4_page_bytes(g) + (size_t)(layer * g.KV + head) * kv4_unit_bytes(g.hd);
}
KV4_HD bool kv4_page_ok(const Kv4Geom &g, int page) { return page >= 0 && page < g.pages; }

KV4_HD int kv4_k_step_off(int hd) { return 32 * hd; }
KV4_HD int kv4_v_code_off(int hd) { return 36 * hd; }
KV4_HD int kv4_v_step_off(int hd) { return 68 * hd; }
// byte (within the unit) of the 32-bit word that holds dims 32 g + 8 j .. + 7 of key row t
KV4_HD int kv4_k_word(int hd, int t, int g, int j) { return t * (hd >> 1) + j * (hd >> 3) + 4 * g; }
// byte of the 16-bit piece that holds dims 32 g + 4 r .. + 3 of value row t
KV4_HD int kv4_v_piece(int hd, int t, int g, int r) {
    return kv4_v_code_off(hd) + (t >> 4) * (8 * hd) + ((t >> 3) & 1) * (4 * hd) + (r * 4 + ((t >> 1) & 3)) * (hd >> 3) + 4 * g + 2 * (t & 1);
}

// A ragged batch as the kernels see it (the device arrays of MotyKv4Batch).
struct Kv4Batch {
    int nseq, rows, ld;
    const int *row0, *len, *table;       // [nseq + 1], [nseq], [nseq][ld]
};
// KV4_ROW_STRAY: a row that no sequence has, found beside arrays that do not describe one.
enum { KV4_ROW_NONE = 0, KV4_ROW_OK = 1, KV4_ROW_BAD = 2, KV4_ROW_STRAY = 3 };
// The row range, first position and length of sequence s.  KV4_ROW_NONE: it has no rows.  KV4_ROW_BAD: the device arrays
// do not describe one (rows outside the buffers, more rows than positions, positions past the table).
KV4_HD int kv4_seq(const Kv4Batch &b, int s, int *r0, int *n, int *len) {
    const int a = b.row0[s], e = b.row0[s + 1];
    *r0 = a; *n = e - a; *len = b.len[s];
    if (a < 0 || e < a || e > b.rows) return KV4_ROW_BAD;
    if (e == a) return KV4_ROW_NONE;
    if (*len < *n || (long long)*len > (long long)b.ld * KV4_PAGE) return KV4_ROW_BAD;
    return KV4_ROW_OK;
}
// The last sequence s with row0[s] <= r (0 when there is none), found by W probes at a time: count(lo, step) = how many of
// the sequences lo, lo + step, .. lo + (W - 1) step below nseq begin at row r or before it.  (Offsets that do not ascend give some
// sequence below nseq.)
template <int W, class Count> KV4_HD int kv4_find_seq(int nseq, Count count) {
    int lo = 0;
    for (int n = nseq; n > 1;) {
        const int step = (n + W - 1) / W, c = count(lo, step);
        lo += c > 1 ? (c - 1) * step : 0;
        n = step;
    }
    return lo;
}
// The position of row r if it belongs to sequence s.  KV4_ROW_NONE: it does not.  KV4_ROW_BAD: it is a row of a sequence that
// is refused.  KV4_ROW_STRAY: it lies outside such a one's rows, and is nobody's.
KV4_HD int kv4_row_in(const Kv4Batch &b, int s, int r, int *pos) {
    int r0, n, len;
    const int st = kv4_seq(b, s, &r0, &n, &len);
    *pos = 0;
    if (st == KV4_ROW_BAD) return b.row0[s] <= r && r < b.row0[s + 1] ? KV4_ROW_BAD : KV4_ROW_STRAY;
    if (st == KV4_ROW_NONE || r < r0 || r >= r0 + n) return KV4_ROW_NONE;
    *pos = len - n + (r - r0);
    return KV4_ROW_OK;
}
// The sequence and position of row r (0 <= r < rows).  KV4_ROW_NONE: the row lies behind the last sequence.  On the device W lanes
// side by side look for a row of theirs (the whole warp calls it), so that 64 sequences take two loads one after the
// other with W = 16 and not six: 64 rows of as many sequences stored and fetched 6.7 us, 7.8 us with a bisection.
#ifdef __CUDACC__
template <int W> __device__ __forceinline__ int kv4_row(const Kv4Batch &b, int r, int *seq, int *pos) {
    const int lane = threadIdx.x & 31, sub = lane % W;
    *seq = kv4_find_seq<W>(b.nseq, [&](int lo, int step) {
        const int s = lo + sub * step;
        const unsigned m = __ballot_sync(0xffffffffu, s < b.nseq && b.row0[s] <= r);
        return W == 32 ? __popc(m) : __popc(m >> (lane & ~(W - 1)) & (unsigned)((1ull << W) - 1));
    });
    return kv4_row_in(b, *seq, r, pos);
}
#else
inline int kv4_row(const Kv4Batch &b, int r, int *seq, int *pos) {
    *seq = kv4_find_seq<16>(b.nseq, [&](int lo, int step) {
        int c = 0;
        for (int i = 0; i < 16 && lo + i * step < b.nseq; i++) c += b.row0[lo + i * step] <= r;
        return c;
    });
    return kv4_row_in(b, *seq, r, pos);
}
#endif

// Reference counts of the pages (host).  The lowest free ids are handed out first, ascending.
struct Kv4Pages {
    std::vector<int> refs, heap;                               // heap: free ids, a min-heap
    void init(int n) {
        refs.assign(n, 0); heap.resize(n);
        for (int i = 0; i < n; i++) heap[i] = i;               // ascending order is a heap
    }
    int free_count() const { return (int)heap.size(); }
    bool alloc(int n, int *out) {
        if (n > (int)heap.size()) return false;
        for (int i = 0; i < n; i++) {
            std::pop_heap(heap.begin(), heap.end(), [](int a, int b) { return a > b; });
            out[i] = heap.back(); heap.pop_back(); refs[out[i]] = 1;
        }
        return true;
    }
    bool live(int id) const { return id >= 0 && id < (int)refs.size() && refs[id] > 0; }
    // one more owner for each id (-1 entries are skipped); all or nothing
    bool retain(const int *ids, int n) {
        for (int i = 0; i < n; i++) if (ids[i] != -1 && (!live(ids[i]) || refs[ids[i]] > (1 << 30))) return false;
        for (int i = 0; i < n; i++) if (ids[i] != -1) refs[ids[i]]++;
        return true;
    }
    // one owner less; a page without owners is free again.  All or nothing: an id listed more often than it has owners fails.
    bool release(const int *ids, int n) {
        for (int i = 0; i < n; i++) {
            if (ids[i] == -1) continue;
            if (!live(ids[i])) {
                for (int k = 0; k < i; k++) if (ids[k] != -1) refs[ids[k]]++;
                return false;
            }
            refs[ids[i]]--;
        }
        for (int i = 0; i < n; i++)
            if (ids[i] != -1 && refs[ids[i]] == 0) {
                refs[ids[i]] = -1;                             // (listed twice: pushed once)
                heap.push_back(ids[i]); std::push_heap(heap.begin(), heap.end(), [](int a, int b) { return a > b; });
            }
        for (int i = 0; i < n; i++) if (ids[i] != -1 && refs[ids[i]] == -1) refs[ids[i]] = 0;
        return true;
    }
    // the moves that bring the live pages to ids 0 .. live - 1: src[i] -> dst[i], both ascending, no id in both
    void plan(std::vector<int> *src, std::vector<int> *dst) const {
        int nlive = 0;
        for (int r : refs) nlive += r > 0;
        src->clear(); dst->clear();
        for (int i = 0; i < nlive; i++) if (refs[i] <= 0) dst->push_back(i);
        for (int i = nlive; i < (int)refs.size(); i++) if (refs[i] > 0) src->push_back(i);
    }
    void moved(const std::vector<int> &src, const std::vector<int> &dst) {
        for (size_t i = 0; i < src.size(); i++) { refs[dst[i]] = refs[src[i]]; refs[src[i]] = 0; }
        heap.clear();
        for (int i = 0; i < (int)refs.size(); i++) if (refs[i] <= 0) heap.push_back(i);
    }
};
