// k_kv_evict.hip — an int8 KV cache cut, per KV head, to the slots whose keys received the most attention.
//
// A slot's key is an unsigned word that orders as (protected, mass): the k-th largest is found by a radix select, eight
// bits a pass, by one workgroup a head; ties go to the lower slot. The kept slots at and above `keep` then move into the
// freed ones below it, the i-th into the i-th: no slot is both read and written, so the moves run in any order, a cache
// that frees one slot moves one row, and what stays below `keep` stays where it is.
#include "ti_dev.h"
#include "ti_span.h"

namespace {

constexpr int SEL = 1024;

struct EvictArgs {
    uint8_t* kq;
    float* ks;
    uint8_t* vq;
    float* vs;
    const float* mass;
    const int32_t* where;
    float* mass_out;
    int32_t* where_out;
    int32_t* moves;          // [nKv][room][2]: (from, to)
    int32_t* count;          // [nKv]
    int n, known, keep, sinks, late, next, nKv, hd, room;   // late: positions from here on are protected
};

// the position of a slot: as `where` says, or of the last tokens in order
__device__ __forceinline__ int slot_pos(const EvictArgs& a, int i, int h) {
    return i < a.known ? a.where[(size_t)i * a.nKv + h] : a.next - (a.n - i);
}
// larger: kept sooner. NaN below everything, -0 equal to 0
__device__ __forceinline__ uint32_t slot_key(const EvictArgs& a, int i, int h) {
    const int p = slot_pos(a, i, h);
    if (p < a.sinks || p >= a.late) return 0xffffffffu;
    const float m = a.mass[(size_t)i * a.nKv + h] + 0.0f;
    const uint32_t b = __builtin_bit_cast(uint32_t, m);
    return m != m ? 0u : (b >> 31 ? ~b : b | 0x80000000u);
}

// exclusive count of the flags of the lanes and waves before this thread, and the total, over 1024 threads
__device__ __forceinline__ int flag_scan(bool f, int* s16, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t b = __ballot(f);
    if (lane == 0) s16[wave] = __popcll(b);
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < SEL / 64; w++) {
        const int v = s16[w];
        before += w < wave ? v : 0;
        all += v;
    }
    total = all;
    __syncthreads();
    return before + __popcll(b & ((1ull << lane) - 1));
}

__global__ __launch_bounds__(SEL) void k_evict_select(EvictArgs a) {
    __shared__ uint32_t hist[256];
    __shared__ uint32_t s_prefix, s_need;
    __shared__ int s16[SEL / 64];
    const int tid = threadIdx.x, h = blockIdx.x;
    uint32_t prefix = 0, need = (uint32_t)a.keep;        // the need-th largest among the keys that share the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < a.n; i += SEL) {
            const uint32_t k = slot_key(a, i, h);
            if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t left = need;
            int d = 255;
            for (; d > 0 && hist[d] < left; d--) left -= hist[d];
            s_prefix = (prefix << 8) | (uint32_t)d;
            s_need = left;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
    }
    // kept: above the threshold, and the first `need` slots at it
    int ties = 0, holes = 0, tails = 0;
    for (int i0 = 0; i0 < a.n; i0 += SEL) {
        const int i = i0 + tid;
        const uint32_t k = i < a.n ? slot_key(a, i, h) : 0u;
        const bool tie = i < a.n && k == prefix;
        int all;
        const int rank = ties + flag_scan(tie, s16, all);
        ties += all;
        const bool kept = i < a.n && (k > prefix || (tie && rank < (int)need));
        const bool hole = i < a.keep && !kept, tail = i >= a.keep && kept;
        const int hr = holes + flag_scan(hole, s16, all);
        holes += all;
        const int tr = tails + flag_scan(tail, s16, all);
        tails += all;
        int32_t* mv = a.moves + (size_t)h * a.room * 2;
        if (hole) mv[2 * hr + 1] = i;
        if (tail) mv[2 * tr] = i;
    }
    if (tid == 0) a.count[h] = holes;
}

// The bookkeeping of the slots that stay where they are, then the moves: a wave a (move, KV head)
__global__ __launch_bounds__(256) void k_evict_stay(EvictArgs a) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long)a.keep * a.nKv) return;
    a.mass_out[i] = a.mass[i];
    a.where_out[i] = slot_pos(a, (int)(i / a.nKv), (int)(i % a.nKv));
}
__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a) {
    const int h = blockIdx.y, lane = threadIdx.x & 63;
    const int count = a.count[h];
    for (int m = blockIdx.x * 4 + (threadIdx.x >> 6); m < count; m += gridDim.x * 4) {
        const int32_t* mv = a.moves + ((size_t)h * a.room + m) * 2;
        const int from = mv[0], to = mv[1];
        const size_t src = (size_t)from * a.nKv + h, dst = (size_t)to * a.nKv + h;
        const int w4 = a.hd / 16, ng = a.hd / 32;
        if (lane < w4) {
            reinterpret_cast<uint4*>(a.kq)[dst * w4 + lane] = reinterpret_cast<const uint4*>(a.kq)[src * w4 + lane];
            reinterpret_cast<uint4*>(a.vq)[dst * w4 + lane] = reinterpret_cast<const uint4*>(a.vq)[src * w4 + lane];
        }
        if (lane < ng) {
            a.ks[dst * ng + lane] = a.ks[src * ng + lane];
            a.vs[dst * ng + lane] = a.vs[src * ng + lane];
        }
        if (lane == 0) {
            a.mass_out[dst] = a.mass[src];
            a.where_out[dst] = slot_pos(a, from, h);
        }
    }
}

}  // namespace

extern "C" int ti_kv_evict_q8(ti_ctx* c, uint32_t* kq, float* ks, uint32_t* vq, float* vs, const float* mass, const int32_t* where,
                              float* mass_out, int32_t* where_out, int n, int known, int keep, int sinks, int recent, int next,
                              int nKv, int hd) {
    TI_CHECK_CTX(c);
    TI_REQUIRE(kq && ks && vq && vs && mass && mass_out && where_out, "ti_kv_evict_q8: null buffer");
    TI_REQUIRE(ti_al16(kq) && ti_al16(vq), "ti_kv_evict_q8: kq/vq must be 16-byte aligned");
    TI_REQUIRE(n > 0 && keep > 0 && nKv > 0 && nKv <= TI_ATTN_HEADS_MAX && hd > 0 && hd % 32 == 0 && hd <= TI_ATTN_HD_MAX,
               "ti_kv_evict_q8: bad shape (n=%d keep=%d nKv=%d hd=%d)", n, keep, nKv, hd);
    TI_REQUIRE(known >= 0 && known <= n && (where || known == 0), "ti_kv_evict_q8: %d slots with a known position of %d", known, n);
    TI_REQUIRE(sinks >= 0 && recent >= 0 && (long)sinks + recent <= keep, "ti_kv_evict_q8: %d sinks and %d recent tokens do not fit %d slots",
               sinks, recent, keep);
    TI_REQUIRE(next >= n - known, "ti_kv_evict_q8: %d slots without a known position before position %d", n - known, next);
    const int kept = keep < n ? keep : n;
    const int room = kept < n - kept ? kept : n - kept;      // moves of a head, at most
    TI_REQUIRE((long)nKv * room * 2 + nKv <= (long)TI_ATTN_ROWSPLITS * TI_ATTN_HD_MAX, "ti_kv_evict_q8: %d moves a head exceed the scratch", room);
    EvictArgs a = {reinterpret_cast<uint8_t*>(kq), ks, reinterpret_cast<uint8_t*>(vq), vs, mass, where, mass_out, where_out,
                   reinterpret_cast<int32_t*>(c->attn_po) + nKv, reinterpret_cast<int32_t*>(c->attn_po), n, known, kept, sinks,
                   recent > next ? 0 : next - recent, next, nKv, hd, room};
    if (room > 0) {
        k_evict_select<<<nKv, SEL, 0, c->stream>>>(a);
        TI_LAUNCHED("k_evict_select");
    }
    k_evict_stay<<<(unsigned)(((long)kept * nKv + 255) / 256), 256, 0, c->stream>>>(a);
    TI_LAUNCHED("k_evict_stay");
    if (room > 0) {
        const int blocks = (room + 3) / 4 < 256 ? (room + 3) / 4 : 256;
        k_evict_move<<<dim3(blocks, nKv), 256, 0, c->stream>>>(a);
        TI_LAUNCHED("k_evict_move");
    }
    return TI_OK;
}
