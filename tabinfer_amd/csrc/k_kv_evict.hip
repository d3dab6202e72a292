// k_kv_evict.hip — an int8 KV cache cut, per KV head, to the slots whose keys received the most attention.
//
// A slot's key is an unsigned word that orders as (protected, mass): the keep-th largest is found by a radix select, by one
// workgroup a head; ties go to the lower slot. The kept slots at and above `keep` then move into the freed ones below it, the
// i-th into the i-th: no slot is both read and written, so the moves run in any order, a cache that frees one slot moves one
// row, and what stays below `keep` stays where it is.
//
// Bound by its launches and by the select's chain of barriers, not by bytes: 4097 slots of 8 heads to 4096
// 2.7 + 5.1 + 2.7 us (keys, the one slot, the move and the bookkeeping), 16384 to 4096 2.7 + 19.2 + 5.9 us (keys, select, moves), where the moved
// rows' 13 MB are 2.7 us of a copy. A workgroup a head and not more: the select's steps depend on one another, and counts
// across workgroups would cost a launch a digit (about 5 us each). 1024 threads: of an earlier version for 4097 and
// 16384 slots 512 took 20.1 and 28.1 us where 1024 took 17.2 and 22.2, and 256 29.3 and 54.3 (more keys a thread, in turn).
#include "ti_dev.h"
#include "ti_evict.h"
#include "ti_span.h"

namespace {

constexpr int SEL = 1024;       // threads of a head's workgroup
constexpr int FORMED = TI_EVICT_FORMED;     // see k_evict_keys

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
    uint32_t* keys;          // [nKv][n]: the keys of more than FORMED slots, head by head
    uint64_t* stays;         // [nKv][words]: a bit a slot below keep that stays
    int n, known, keep, sinks, late, next, nKv, hd, room, words;   // late: positions from here on are protected
};

// the position of a slot: as `where` says, or of the last tokens in order
__device__ __forceinline__ int slot_pos(const EvictArgs& a, int i, int h) {
    return i < a.known ? a.where[(size_t)i * a.nKv + h] : a.next - (a.n - i);
}
// larger: kept sooner. NaN below everything, -0 equal to 0
__device__ __forceinline__ uint32_t order_key(const EvictArgs& a, int p, float mass) {
    const float m = mass + 0.0f;
    const uint32_t b = __builtin_bit_cast(uint32_t, m);
    return p < a.sinks || p >= a.late ? 0xffffffffu : m != m ? 0u : (b >> 31 ? ~b : b | 0x80000000u);
}
// the bookkeeping of a slot that stays (nothing to do where it is in place already)
__device__ __forceinline__ void stay(const EvictArgs& a, int i, int h) {
    const size_t at = (size_t)i * a.nKv + h;
    if (a.mass_out != a.mass) a.mass_out[at] = a.mass[at];
    if (a.where_out != a.where || i >= a.known) a.where_out[at] = slot_pos(a, i, h);
}

// a move, 16 lanes: K's and V's pieces and scales, and what the slot holds (read above keep, written below)
__device__ __forceinline__ void move_slot(const EvictArgs& a, int from, int to, int h, int l) {
    const size_t src = (size_t)from * a.nKv + h, dst = (size_t)to * a.nKv + h;
    const int w4 = a.hd / 16, ng = a.hd / 32, p = l & 7;
    const uint4* cs = reinterpret_cast<const uint4*>(l < 8 ? a.kq : a.vq);
    uint4* cd = reinterpret_cast<uint4*>(l < 8 ? a.kq : a.vq);
    float* sc = l < 8 ? a.ks : a.vs;
    if (p < w4) cd[dst * w4 + p] = cs[src * w4 + p];
    if (p < ng) sc[dst * ng + p] = sc[src * ng + p];
    if (l == 0) {
        a.mass_out[dst] = a.mass[src];
        a.where_out[dst] = slot_pos(a, from, h);
    }
}

// nothing to evict: every slot stays
__global__ __launch_bounds__(256) void k_evict_none(EvictArgs a) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i < (long)a.n * a.nKv) stay(a, (int)(i / a.nKv), (int)(i % a.nKv));
}

// The keys of many slots, head by head: rows of all heads are read in whole lines here, where a head's one workgroup would
// take a 4-byte piece of each (8 heads: 16384 slots 9 us against 5.5 with this launch, 4097 slots to all but 99 of them 16.1
// with the select against 14.5; up to 2048 slots the pieces cost less than the launch, 9.7 against 13.1)
__global__ __launch_bounds__(256) void k_evict_keys(EvictArgs a) {
    const long x = (long)blockIdx.x * 256 + threadIdx.x;
    if (x >= (long)a.n * a.nKv) return;
    const int i = (int)(x / a.nKv), h = (int)(x % a.nKv);
    a.keys[(size_t)h * a.n + i] = order_key(a, slot_pos(a, i, h), a.mass[x]);
}

// A workgroup a head. Slot i = 1024 k + tid of a chunk of 1024 x KPT; up to KPT = 16 every key stays in a register, more slots
// go through in chunks of 16, read again for each digit (32 keys a thread spill: 17000 slots to 4096 42.4 us against 34.6 in chunks, 32000
// to 8000 46.8 / 34.8, 100000 to 25000 171 / 121); no more registers than the slots need (4097 slots 11.6 us with 8, 15.2
// with 16). The keep-th largest key by a radix select of 11, 11 and 10 bits: a histogram in LDS, its bins added
// up from the top, and only the keys with the digits so far go on; done as soon
// as all of these are kept (16384 slots of 8 heads to 4096: 22 us, all three digits' passes, to 20). Lanes of a wave that all have one digit count as one, so
// that equal masses do not queue for their bin.
constexpr int BINS = 2048;
template <int KPT>
struct SelLds {
    uint32_t hist[BINS];
    uint32_t digit, need, all;             // the bin that holds the keep-th key, its rank in it, the bin's count
    int part[KPT * (SEL / 64)], tot[SEL / 64];
};

// sum over the threads before this one
__device__ __forceinline__ int thread_scan(int v, int* tot) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;                                             // rows of 16 lanes, then the rows before
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);   // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);   // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);   // row_bcast:31 into rows 2 and 3
    if (lane == 63) tot[wave] = x;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < SEL / 64; w++) before += w < wave ? tot[w] : 0;
    return before + x - v;
}

// exclusive sums of part[] in place; its total
template <int KPT>
__device__ __forceinline__ int part_scan(SelLds<KPT>& L) {
    constexpr int N = KPT * (SEL / 64);
    static_assert(N <= SEL, "a thread a count");
    const int tid = threadIdx.x;
    __syncthreads();
    const int v = tid < N ? L.part[tid] : 0;
    const int before = thread_scan(v, L.tot);
    if (tid < N) L.part[tid] = before;
    __syncthreads();
    int sum = L.tot[0];
#pragma unroll
    for (int w = 1; w < SEL / 64; w++) sum += L.tot[w];
    return sum;
}

// the keys of slots i0 + 1024 k + tid, every load in flight at once; 0 behind the last slot. FORM: else k_evict_keys did
template <int KPT, bool FORM>
__device__ __forceinline__ void load_keys(const EvictArgs& a, int h, int i0, uint32_t (&key)[KPT]) {
    const int tid = threadIdx.x;
    if constexpr (!FORM) {
#pragma unroll
        for (int k = 0; k < KPT; k++) key[k] = a.keys[(size_t)h * a.n + ti_min(i0 + k * SEL + tid, a.n - 1)];
#pragma unroll
        for (int k = 0; k < KPT; k++) key[k] = i0 + k * SEL + tid < a.n ? key[k] : 0u;
        return;
    }
#pragma unroll
    for (int k = 0; k < KPT; k++) key[k] = __builtin_bit_cast(uint32_t, a.mass[(size_t)ti_min(i0 + k * SEL + tid, a.n - 1) * a.nKv + h]);
    int at[KPT];
#pragma unroll
    for (int k = 0; k < KPT; k++) at[k] = a.known ? a.where[(size_t)ti_min(i0 + k * SEL + tid, a.known - 1) * a.nKv + h] : 0;
#pragma unroll
    for (int k = 0; k < KPT; k++) {
        const int i = i0 + k * SEL + tid;
        if (i >= a.known) at[k] = a.next - (a.n - i);
        key[k] = i < a.n ? order_key(a, at[k], __builtin_bit_cast(float, key[k])) : 0u;
    }
}

// One slot too many, a bounded cache's every token: the last slot of the smallest key, by a minimum in place of the select
// (4097 slots of 8 heads: 5.1 us, the select 11.6). In place it moves the one slot too, and nothing follows (with a launch for
// the move 2.8 us more); elsewhere k_evict_move writes what the other slots hold along the rows of all heads (2.9 us; from
// here, a 4-byte piece of each row at a time, 5)
template <bool FORM>
__global__ __launch_bounds__(SEL) void k_evict_one(EvictArgs a, bool placed) {
    constexpr int KPT = FORMED / SEL;
    __shared__ uint64_t s_best[SEL / 64];
    const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.x;
    uint64_t best = ~0ull;                                 // (key, slots behind it)
    for (int i0 = 0; i0 < a.n; i0 += KPT * SEL) {
        uint32_t key[KPT];
        load_keys<KPT, FORM>(a, h, i0, key);
#pragma unroll
        for (int k = 0; k < KPT; k++) {
            const int i = i0 + k * SEL + tid;
            if (i < a.n) best = ti_min(best, (uint64_t)key[k] << 32 | (uint32_t)(a.n - 1 - i));
        }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) best = ti_min(best, (uint64_t)__shfl_xor((unsigned long long)best, o));
    if (lane == 0) s_best[tid >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < SEL / 64; w++) best = ti_min(best, s_best[w]);
    const int out = a.n - 1 - (int)(uint32_t)best;
    if (placed) {
        if (tid < 16 && out < a.keep) move_slot(a, a.keep, out, h, tid);
        return;
    }
    for (int w = tid; w < a.words; w += SEL) a.stays[(size_t)h * a.words + w] = ~(out / 64 == w ? 1ull << (out & 63) : 0ull);
    if (tid > 0) return;
    a.count[h] = out < a.keep;
    a.moves[2 * h] = a.keep;                               // the one slot behind them, and room for one move a head
    a.moves[2 * h + 1] = out;
}

template <int KPT, bool FORM>
__global__ __launch_bounds__(SEL) void k_evict_pick(EvictArgs a) {
    constexpr int W = SEL / 64;
    static_assert(KPT * SEL <= 32768, "counts of 16 bits");
    __shared__ SelLds<KPT> L;
    const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t key[KPT];                                     // 0 behind the last slot
    auto load = [&](int i0) { load_keys<KPT, FORM>(a, h, i0, key); };
    constexpr int CHUNK = KPT * SEL;
    const bool one = a.n <= CHUNK;
    if (one) load(0);
    uint32_t top = 0;                                      // the keep-th largest key, its digits so far (from bit `shift` up)
    int shift = 0;
    int need = a.keep;                                     // which of the keys with those digits, from the largest
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int bits = pass == 2 ? 10 : 11;
        L.hist[tid] = 0;
        L.hist[tid + SEL] = 0;
        __syncthreads();
        for (int i0 = 0; i0 < a.n; i0 += CHUNK) {
            if (!one) load(i0);
#pragma unroll
            for (int k = 0; k < KPT; k++) {
                const bool on = i0 + k * SEL + tid < a.n && (pass == 0 || key[k] >> (shift + bits) == top);
                const uint64_t b = __ballot(on);
                if (b == 0) continue;                      // wave-uniform
                const uint32_t d = key[k] >> shift & ((1u << bits) - 1);
                const uint32_t d0 = (uint32_t)__builtin_amdgcn_readlane((int)d, __builtin_ctzll(b));
                if (__ballot(on && d == d0) == b) {
                    if (lane == __builtin_ctzll(b)) atomicAdd(&L.hist[d0], (uint32_t)__popcll(b));
                } else if (on) {
                    atomicAdd(&L.hist[d], 1u);
                }
            }
        }
        __syncthreads();
        // a thread: two bins, from the top
        static_assert(BINS == 2 * SEL, "two bins a thread");
        const int h0 = (int)L.hist[BINS - 1 - 2 * tid], h1 = (int)L.hist[BINS - 2 - 2 * tid];
        const int before = thread_scan(h0 + h1, L.tot);
        if (before < need && need <= before + h0 + h1) {   // one thread
            const bool second = need > before + h0;
            L.digit = (uint32_t)(BINS - 1 - 2 * tid - (second ? 1 : 0));
            L.need = (uint32_t)(need - before - (second ? h0 : 0));
            L.all = (uint32_t)(second ? h1 : h0);
        }
        __syncthreads();
        top = top << bits | L.digit;
        need = (int)L.need;
        if (L.need == L.all) break;                        // every key with these digits is kept: the other digits do not matter
    }
    // kept: the keys above those digits, and of those equal in them the first `need` slots
    const uint64_t below = (1ull << lane) - 1;
    int32_t* mv = a.moves + (size_t)h * a.room * 2;
    int ties = 0, holes = 0, tails = 0;                    // of the chunks before
    for (int i0 = 0; i0 < a.n; i0 += CHUNK) {
        if (!one) load(i0);
        auto is_tie = [&](int k) { return key[k] >> shift == top && i0 + k * SEL + tid < a.n; };
#pragma unroll
        for (int k = 0; k < KPT; k++) {
            const uint64_t b = __ballot(is_tie(k));
            if (lane == 0) L.part[k * W + wave] = __popcll(b);
        }
        const int chunk_ties = part_scan(L);
        uint32_t kept = 0;                                 // a bit a slot
#pragma unroll
        for (int k = 0; k < KPT; k++) {
            const uint64_t b = __ballot(is_tie(k));
            const int rank = ties + L.part[k * W + wave] + __popcll(b & below);
            const bool st = key[k] >> shift > top || (is_tie(k) && rank < need);
            kept |= st ? 1u << k : 0u;
            const uint64_t stays = __ballot(st);           // for the launch that follows
            const int w0 = i0 + k * SEL + 64 * wave;
            if (lane == 0 && w0 < a.keep) a.stays[(size_t)h * a.words + w0 / 64] = stays;
        }
        ties += chunk_ties;
        __syncthreads();
        // ranks of the freed slots below keep and of the kept ones above: counts side by side in a word
        auto moves = [&](int k) { return (i0 + k * SEL + tid < a.keep) != (bool)(kept >> k & 1u); };
#pragma unroll
        for (int k = 0; k < KPT; k++) {
            const uint64_t b = __ballot(moves(k)), low = __ballot(i0 + k * SEL + tid < a.keep);
            if (lane == 0) L.part[k * W + wave] = __popcll(b & low) | __popcll(b & ~low) << 16;
        }
        const int total = part_scan(L);
#pragma unroll
        for (int k = 0; k < KPT; k++) {
            const int i = i0 + k * SEL + tid;
            const uint64_t b = __ballot(moves(k)), low = __ballot(i < a.keep);
            const uint32_t base = (uint32_t)L.part[k * W + wave];
            if (moves(k)) {
                if (i < a.keep) mv[2 * (holes + (int)(base & 0xffff) + __popcll(b & low & below)) + 1] = i;
                else mv[2 * (tails + (int)(base >> 16) + __popcll(b & ~low & below))] = i;
            }
        }
        holes += total & 0xffff;
        tails += (int)((uint32_t)total >> 16);
        __syncthreads();                                   // the parts are read
    }
    if (tid == 0) a.count[h] = holes;
}

// The moves, 16 lanes each. Behind them (blocks from mblocks on) the bookkeeping of the slots that stay, along the rows of all heads
__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a, int mblocks, int per_head) {
    if ((int)blockIdx.x >= mblocks) {
        const long x = (long)(blockIdx.x - mblocks) * 256 + threadIdx.x;
        const int i = (int)(x / a.nKv), h = (int)(x % a.nKv);
        if (i < a.keep && (a.stays[(size_t)h * a.words + i / 64] >> (i & 63) & 1)) stay(a, i, h);
        return;
    }
    const int h = blockIdx.x / per_head, l = threadIdx.x & 15, m = blockIdx.x % per_head * 16 + (threadIdx.x >> 4);
    if (m >= a.count[h]) return;
    const int32_t* mv = a.moves + ((size_t)h * a.room + m) * 2;
    move_slot(a, mv[0], mv[1], h, l);
}

}  // namespace

extern "C" int ti_kv_evict_q8(ti_ctx* c, uint32_t* kq, float* ks, uint32_t* vq, float* vs, const float* mass, const int32_t* where,
                              float* mass_out, int32_t* where_out, int n, int known, int keep, int sinks, int recent, int next,
                              int nKv, int hd) {
    TI_CHECK_CTX(c);
    TI_REQUIRE(kq && ks && vq && vs && mass && mass_out && where_out, "ti_kv_evict_q8: null buffer");
    TI_REQUIRE(ti_al16(kq) && ti_al16(vq), "ti_kv_evict_q8: kq/vq must be 16-byte aligned");
    TI_REQUIRE_DENSE("ti_kv_evict_q8", kq);
    TI_REQUIRE_DENSE("ti_kv_evict_q8", vq);
    TI_REQUIRE(n > 0 && keep > 0 && nKv > 0 && nKv <= TI_ATTN_HEADS_MAX && hd > 0 && hd % 32 == 0 && hd <= TI_ATTN_HD_MAX,
               "ti_kv_evict_q8: bad shape (n=%d keep=%d nKv=%d hd=%d)", n, keep, nKv, hd);
    TI_REQUIRE(known >= 0 && known <= n && (where || known == 0), "ti_kv_evict_q8: %d slots with a known position of %d", known, n);
    TI_REQUIRE(sinks >= 0 && recent >= 0 && (long)sinks + recent <= keep, "ti_kv_evict_q8: %d sinks and %d recent tokens do not fit %d slots",
               sinks, recent, keep);
    TI_REQUIRE(next >= n - known, "ti_kv_evict_q8: %d slots without a known position before position %d", n - known, next);
    const int kept = keep < n ? keep : n;
    const bool single = n - kept == 1, many = n > FORMED;
    const TiEvictScratch at(n, kept, nKv);
    const int room = at.room;
    TI_REQUIRE(at.fits(), "ti_kv_evict_q8: %d slots and %d moves a head exceed the scratch", n, room);
    int32_t* scratch = reinterpret_cast<int32_t*>(c->attn_po);
    EvictArgs a = {reinterpret_cast<uint8_t*>(kq), ks, reinterpret_cast<uint8_t*>(vq), vs, mass, where, mass_out, where_out,
                   scratch + at.moves, scratch + at.count, reinterpret_cast<uint32_t*>(scratch + at.keys), reinterpret_cast<uint64_t*>(scratch),
                   n, known, kept, sinks, recent > next ? 0 : next - recent, next, nKv, hd, room, at.words};
    if (room == 0) {
        k_evict_none<<<(unsigned)(((long)n * nKv + 255) / 256), 256, 0, c->stream>>>(a);
        TI_LAUNCHED("k_evict_none");
        return TI_OK;
    }
    // in place, the slots that stay already hold what they held
    const bool placed = mass_out == mass && where_out == where && known >= kept;
    if (many) {
        k_evict_keys<<<(unsigned)(((long)n * nKv + 255) / 256), 256, 0, c->stream>>>(a);
        TI_LAUNCHED("k_evict_keys");
    }
    if (single && many) k_evict_one<false><<<nKv, SEL, 0, c->stream>>>(a, placed);
    else if (single) k_evict_one<true><<<nKv, SEL, 0, c->stream>>>(a, placed);
    else if (n <= FORMED) k_evict_pick<FORMED / SEL, true><<<nKv, SEL, 0, c->stream>>>(a);
    else if (n <= 8 * SEL) k_evict_pick<8, false><<<nKv, SEL, 0, c->stream>>>(a);
    else k_evict_pick<16, false><<<nKv, SEL, 0, c->stream>>>(a);
    TI_LAUNCHED("k_evict_pick");
    if (single && placed) return TI_OK;
    const int per_head = (room + 15) / 16, sblocks = placed ? 0 : (int)(((long)kept * nKv + 255) / 256);
    k_evict_move<<<(unsigned)(per_head * nKv + sblocks), 256, 0, c->stream>>>(a, per_head * nKv, per_head);
    TI_LAUNCHED("k_evict_move");
    return TI_OK;
}
