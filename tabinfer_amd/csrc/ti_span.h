// ti_span.h — which keys of the int8 KV cache a query sees under a sliding window with sinks, and where a position's
// row lies in a contiguous cache or in pages. Plain C++ beside the HIP keywords, so that a host compiler can test it.
#pragma once
#include <stdint.h>
#include <stddef.h>
#ifdef __HIPCC__
#define TI_HD __host__ __device__
#else
#define TI_HD
#endif

// One type on both sides: the toolkit's host min and max take int.
template <class N> TI_HD inline N ti_min(N a, N b) { return b < a ? b : a; }
template <class N> TI_HD inline N ti_max(N a, N b) { return a < b ? b : a; }

// Positions of the attention calls end here, so that a block of keys past the last one has 32-bit positions too.
constexpr int TI_POS_END = 0x7fffff00;

// The keys a query at position p sees: [0, first) and [low, p + 1), in order; first <= low. window < 0: all of them.
struct TiSpan {
    int first, low, end;
    TI_HD int count() const { return first + (end - low); }
};
TI_HD inline TiSpan ti_span(int p, int window, int sinks) {
    TiSpan s;
    s.end = p + 1;
    s.low = window < 0 || window > p ? 0 : p + 1 - window;
    s.first = sinks < s.low ? sinks : s.low;
    return s;
}

// Position -> row of the cache. Pages are a power of two of positions long (page = 1 << shift); table == nullptr: the
// positions are the rows, pages * page of them. -1: no such row.
struct TiPages {
    const int32_t* table;
    int shift, pages, width;
    TI_HD long row(int seq, int pos) const {
        if (pos < 0) return -1;
        const int k = pos >> shift;
        if (!table) return k < pages ? (long)pos : -1;
        if (k >= width) return -1;
        const int id = table[(size_t)seq * width + k];
        return id >= 0 && id < pages ? ((long)id << shift) + (pos & ((1 << shift) - 1)) : -1;
    }
};
// Position of a sequence's last query: of `len` keys, taken as at most `most` of them; -1 where there is none, whatever the length
TI_HD inline int ti_last_pos(int len, long most) { return len <= 0 ? -1 : (int)ti_min((long)len, most) - 1; }

// Groups of sequences that share their first positions: group g holds the sequences [starts[g], starts[g + 1]) of B. One of a single
// sequence shares nothing: it counts as empty. Whatever `starts` holds, members are of [0, B).
struct TiMembers {
    int first, count;
};
TI_HD inline TiMembers ti_group_members(const int32_t* starts, int B, int g) {
    const int lo = ti_max(0, ti_min((int)starts[g], B)), n = ti_max(lo, ti_min((int)starts[g + 1], B)) - lo;
    return TiMembers{lo, n > 1 ? n : 0};
}
// The group of sequence b, with something to share, and what that is: -1 and 0 for none
struct TiGroup {
    int g, first, shared;
};
TI_HD inline TiGroup ti_group_at(int g, int s0, int s1, int shared, int B, int b) {   // group g = [s0, s1), if b is in it
    const int32_t s[2] = {s0, s1};
    const TiMembers m = ti_group_members(s, B, 0);
    return b < s0 || b >= s1 || shared <= 0 || m.count == 0 ? TiGroup{-1, 0, 0} : TiGroup{g, m.first, shared};
}
TI_HD inline TiGroup ti_group_of(const int32_t* starts, const int32_t* shared, int P, int B, int b) {
    int lo = 0, hi = P;                      // the first group that begins behind b is in [lo, hi]
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (starts[mid] <= b) lo = mid + 1;
        else hi = mid;
    }
    const int g = lo - 1;
    return g < 0 ? TiGroup{-1, 0, 0} : ti_group_at(g, starts[g], starts[g + 1], shared[g], B, b);
}
// A number for tile `tile` of `rows` rows of group g, whose first sequence is `first` and whose sequences have G rows each: larger for
// later tiles and later groups (a group of n G rows has at most one tile more than n G / rows, and takes one number more: groups with
// something to share are at least two sequences apart). Below ti_group_tile(B, P, 0, G, rows) for those of P groups.
TI_HD inline int ti_group_tile(int first, int g, int tile, int G, int rows) {
    return (int)((long)first * G / rows) + ti_min(g, first / 2) + tile;
}
// a / b of numbers that are rarely as large as 64 bits, whose division takes four times as long
TI_HD inline long ti_quotient(long a, long b) { return (a | b) >> 31 ? a / b : (long)((uint32_t)a / (uint32_t)b); }
// Into how many runs a tile's or sequence's nb blocks are cut, where all units of `tiles` tiles each have `total` together: its share
// of wgs workgroups, of a block for each of a run's BW waves at least. `many` (2 wgs or one less) instead where a wave would have more than
// 8 blocks: a second workgroup a CU hides the first one's loads and waits, but doubles the partials and the operands, which short runs feel (32
// sequences of 16 heads over 8 behind 8192 shared keys 33.8 us with one, 38.5 with two; 16384 47.3 / 45.6; 32768 71.0 / 62.2; 128 sequences of
// 32768 241 / 172). Of several tiles a multiple of the XCDs, so that a part's workgroups are on one XCD for all of them and its keys come
// into that L2 once (48 sequences of three tiles behind 12288 keys 63.0 us, 47.3 so). All units' runs are many plus their tiles at most: rounding
// up concerns units of nine runs and more, eight times as many in all as there are such tiles, and makes them 16/9 as many
constexpr int TI_XCDS = 8, TI_LONG_RUN = 8;
TI_HD inline int ti_group_parts(long total, int nb, int tiles, int wgs, int many, int BW) {
    const bool more = many > wgs && total > (long)TI_LONG_RUN * BW * wgs;
    const int n = more ? many : wgs;
    const long chunk = ti_max(ti_quotient(total + n - 1, n), (long)BW);
    const int parts = (int)ti_quotient(nb + chunk - 1, chunk);
    return tiles < 2 || parts <= TI_XCDS ? parts : (more ? parts : parts + TI_XCDS - 1) / TI_XCDS * TI_XCDS;
}
inline bool ti_pow2(int v) { return v > 0 && (v & (v - 1)) == 0; }
inline int ti_log2(int v) { return 31 - __builtin_clz((unsigned)v); }
static inline bool ti_al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
