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
inline bool ti_pow2(int v) { return v > 0 && (v & (v - 1)) == 0; }
inline int ti_log2(int v) { return 31 - __builtin_clz((unsigned)v); }
static inline bool ti_al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
