// ti_evict.h — what an eviction keeps in the partials' scratch, and how many slots fit. Plain C++, so that a host compiler
// can test it.
#pragma once
#include "ti_limits.h"

constexpr int TI_EVICT_FORMED = 2048;        // up to so many slots a head's workgroup forms their keys itself
constexpr long TI_EVICT_WORDS = (long)TI_ATTN_ROWSPLITS * TI_ATTN_HD_MAX;      // 32-bit words of the scratch

// n slots a KV head cut to kept <= n of them: a bit a slot below `kept` that stays, the moves' counts, the moves (from, to), the
// keys of many slots. Offsets in 32-bit words; the bits lie first, on 8 bytes
struct TiEvictScratch {
    int room, words;                         // moves of a head, at most; 64-bit words of its bits
    long count, moves, keys, total;
    constexpr TiEvictScratch(int n, int kept, int nKv)
        : room(kept < n - kept ? kept : n - kept), words(kept / 64 + (kept % 64 != 0)), count(2L * nKv * words), moves(count + nKv),
          keys(moves + 2L * nKv * room), total(keys + (n > TI_EVICT_FORMED ? (long)nKv * n : 0)) {}
    constexpr bool fits() const { return total <= TI_EVICT_WORDS; }
};
