// k_logprobs.hip — log probabilities of given tokens under rows of logits, the rows' entropy and their likeliest tokens, in one pass over
// the logits. The reference has no counterpart: its sampler keeps an index (models/qwen3.js:2624-2740).
//
// With M the row's maximum, C the number of elements equal to it, S = sum e^(x - M) of the others and U = sum e^(x - M) (x - M): log p(x) =
// (x - M) - ln (C + S) and the entropy ln (C + S) - U / (C + S), two terms of one sign. C and S apart, so that the logarithm is that of 1 + (C - 1 + S)
// and a token that is nearly certain keeps its digits. A lane keeps (m, c, s, u) of its own elements and turns them to a larger maximum by
// s' = a (s + c), c' = 0, u' = a (u + (m - m') (s + c)), a = e^(m - m'); lanes, waves and workgroups are joined by the same rule in a fixed order.
//
// The likeliest: a value and its index are one 64-bit key (the float's bits in an order of whole numbers, then the inverted index: the lower
// index wins), so that no two are equal. A wave takes 1024 elements at a time, in registers. Where `top` lanes hold something above its
// limit, as always at first, the limit is raised to the top-th largest of the lanes' maxima, or to the first bits of it that no other lane reaches,
// found bit by bit with ballots; it never falls. What is above it goes to a list in LDS, of at most `top` lanes and so 16 top keys a chunk, whatever the values are. (The first limit is that of all of the
// workgroup's waves together.) Where the list has grown to more than 64 keys, and at the end, it is sorted into the 64 largest that the wave keeps, a lane each, by exchanges between lanes; so all chunks but a wave's first
// cost little more than a comparison. A workgroup sorts once, what is above the largest of its waves' limits.
//
// Bound by the stream where rows are many (400 rows of 151936 logits, 243 MB, 43.4 + 4.7 us: 5.0 TB/s), with tokens kept by the listing of candidates, a
// ballot an element, and the sorts (48 rows with 20 tokens, 29 MB, 21.3 us; without tokens 12), in one row by the chain from its first load to the join (with
// five tokens 10.3).
//
// Long rows are cut into parts. Of up to 128 rows the workgroup that ends last joins a row's parts, of more a second launch does.
#include "ti_dev.h"
#include "ti_span.h"

namespace {

typedef float v4f_u __attribute__((ext_vector_type(4), aligned(4)));   // rows start anywhere

constexpr int EPT = 16, CHUNK = 64 * EPT, WAVES = 4, STEP = WAVES * CHUNK;     // elements of a lane, a wave's chunk, a workgroup's
constexpr int TOP_MAX = 64;                  // one lane a kept key
constexpr int LONG = 64;                     // keys after which a list is sorted
constexpr int SEGS_MAX = 64;                 // workgroups a row: one lane each where they are joined
constexpr int ROWS_MAX = 1 << 17;
constexpr float LOW = -3.402823466e38f;

constexpr int PART = 8;                      // floats a part

struct LpArgs {
    const float* x;
    const int32_t* ids;
    float *lp, *ent;
    int32_t *rank, *top_ids;
    float* top_lp;
    float* part;                             // [row][segs][PART] (m, s, u, c, number of logits above the token's)
    uint64_t* keys;                          // [row][segs][top], from large to small, 0 behind the last
    uint32_t* arrived;                       // a line a row, 0 between launches; or nullptr: a second launch joins the parts
    long ld;
    int T, N, top, segs, per;                // a row is cut into `segs` parts of `per` steps
};

__device__ __forceinline__ uint32_t ordered(float v) {     // 0: no candidate (NaN)
    const uint32_t b = __float_as_uint(v + 0.0f);          // -0 is 0
    return v != v ? 0u : b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t u) { return __uint_as_float(u ^ (u >> 31 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t key_of(uint32_t u, uint32_t index) { return (uint64_t)u << 32 | ~index; }

struct Sum {
    float m, s, u;
    int c;
};
__device__ __forceinline__ float down_to(float d) { return d < -150.0f ? -150.0f : d; }      // e^-150 is 0; NaN stays
// a, at the maximum m of its own or a larger one
__device__ __forceinline__ Sum turned(const Sum& a, float m) {
    const float d = down_to(a.m - m), e = expf(d), all = a.s + (float)a.c;
    const bool same = d == 0.0f;
    return {m, same ? a.s : all * e, e * (a.u + d * all), same ? a.c : 0};
}
__device__ __forceinline__ Sum joined(const Sum& a, const Sum& b) {
    const float m = fmaxf(a.m, b.m);
    const Sum x = turned(a, m), y = turned(b, m);
    return {m, x.s + y.s, x.u + y.u, x.c + y.c};
}
__device__ __forceinline__ Sum wave_joined(const Sum& a) {
    // the maximum first, so that every lane turns its own to it once; the offsets spelled out, as ti_wave_sum's
    const Sum x = turned(a, ti_wave_max(a.m));
    return {x.m, ti_wave_sum(x.s), ti_wave_sum(x.u), ti_wave_sum_i(x.c)};
}

// ---- 64 keys, a lane each, from large to small ---------------------------------------------------------------------
__device__ __forceinline__ uint64_t key_xor(uint64_t k, int o) {
    return (uint64_t)ti_xor((uint32_t)(k >> 32), o) << 32 | ti_xor((uint32_t)k, o);
}
// lanes O apart: the one without bit O takes the larger key where `down`, the smaller elsewhere
template <int O>
__device__ __forceinline__ uint64_t exchange(uint64_t k, bool down) {
    const uint64_t other = key_xor(k, O);
    const bool first = (threadIdx.x & O) == 0;
    return (other > k) == (first == down) ? other : k;
}
// a sequence that rises and falls once (in every 2 O lanes), sorted
template <int O>
__device__ __forceinline__ uint64_t merged(uint64_t k, bool down) {
    k = exchange<O>(k, down);
    if constexpr (O > 1) k = merged<O / 2>(k, down);
    return k;
}
template <int O>
__device__ __forceinline__ uint64_t sorted(uint64_t k) {   // in every 2 O lanes, down and up in turn
    if constexpr (O > 1) k = sorted<O / 2>(k);
    return merged<O>(k, (threadIdx.x & 63 & 2 * O) == 0);
}
// the 64 largest of two sorted 64, the second from small to large
__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t up) { return merged<32>(a > up ? a : up, true); }
// 64 keys in any order into the kept ones
__device__ __forceinline__ uint64_t taken(uint64_t kept, uint64_t k) {
    k = merged<32>(sorted<16>(k), false);                  // from small to large
    return larger(kept, k);
}
// the first keys that are kept: n of them, in the lowest lanes
__device__ __forceinline__ uint64_t taken_first(uint64_t k, int n) {
    k = sorted<8>(k);
    if (n > 16) {
        k = merged<16>(k, (threadIdx.x & 32) == 0);
        if (n > 32) k = merged<32>(k, true);
    }
    return k;
}
// a wave's list into its kept keys
__device__ __forceinline__ uint64_t taken(uint64_t kept, const uint64_t* list, int n) {
    const int lane = threadIdx.x & 63;
    ti_wave_lds_fence();
    for (int j = 0; j < n; j += 64) kept = taken(kept, j + lane < n ? list[j + lane] : 0ull);
    ti_wave_lds_fence();
    return kept;
}
__device__ __forceinline__ uint32_t value_at(uint64_t kept, int i) { return __builtin_amdgcn_readlane((uint32_t)(kept >> 32), i); }

// what a row's numbers come to, and its likeliest tokens' (key of lane i the i-th)
__device__ __forceinline__ void finish(const LpArgs& a, int t, const Sum& r, int above, uint64_t key) {
    const int lane = threadIdx.x & 63;
    const float ln = log1pf((float)(r.c - 1) + r.s);
    if (lane == 0) {
        const int id = a.ids[t];
        const bool there = id >= 0 && id < a.N;
        a.lp[t] = there ? (a.x[t * a.ld + id] - r.m) - ln : -INFINITY;
        if (a.ent) a.ent[t] = ln - r.u / ((float)r.c + r.s);
        if (a.rank) a.rank[t] = there ? above + 1 : 0;
    }
    if (lane < a.top) {
        const size_t at = (size_t)t * a.top + lane;
        a.top_ids[at] = key ? (int32_t)~(uint32_t)key : -1;
        a.top_lp[at] = key ? (value_of((uint32_t)(key >> 32)) - r.m) - ln : -INFINITY;
    }
}

// What `top` lanes of a workgroup's first step reach, of the upper 16 bits of a value: every wave then lists a fourth of what a limit of its own
// would let through. 0 (every wave finds its own) where that is no number, or zero, below which there is no other next to it; or where more of this
// wave's lanes reach it than its list has room for. 48 rows with 5 tokens 20.2 us (each wave with a limit of its own 22.3), with 20 20.8 (24.3), with 64
// 28.8 (36.0), 1000 rows of 30000 with 5 35.9 (41.6); one row with 10 12.8 (11.9), with 64 22.9 (30.2)
__device__ __forceinline__ uint32_t first_limit(const float (&v)[EPT], long there, int top, uint32_t* s_most) {
    const int lane = threadIdx.x & 63, in = (int)ti_max(-256L, ti_min((long)CHUNK, there)) - 4 * lane;
    uint32_t most = 0, reach = 0;
    if (there > 0) {
#pragma unroll
        for (int i = 0; i < EPT; i++) most = max(most, 256 * (i / 4) + i % 4 < in ? ordered(v[i]) : 0u);
    }
    s_most[threadIdx.x] = most;
    __syncthreads();
    uint32_t w[WAVES];
#pragma unroll
    for (int k = 0; k < WAVES; k++) w[k] = s_most[64 * k + lane];
    int held = 64 * WAVES + 1;
    for (uint32_t bit = 0x80000000u; bit > 0x8000u && held > top; bit >>= 1) {
        int n = 0;
#pragma unroll
        for (int k = 0; k < WAVES; k++) n += __builtin_popcountll(__ballot(w[k] >= (reach | bit)));
        if (n >= top) {
            reach |= bit;
            held = n;
        }
    }
    const bool fits = __builtin_popcountll(__ballot(most >= reach)) <= top;
    return fits && reach > ordered(-INFINITY) && reach != ordered(0.0f) ? reach : 0u;
}

// A row's parts, by a workgroup: their numbers, a lane of the first wave each, and their keys, 64 at a time. (Only those above what the parts' j-th
// keys show to be unwanted, in a list: 48 rows with 20 tokens took 2.9 us more, one row 0.7 less.) PUB: other workgroups of
// this launch wrote them
template <bool PUB>
__device__ __forceinline__ void join_parts(const LpArgs& a, int t, uint64_t (*s_waves)[64]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = a.segs * a.top;
    const bool has = lane < a.segs;
    const float* q = a.part + ((size_t)t * a.segs + ti_min(lane, a.segs - 1)) * PART;
    const uint64_t* keys = a.keys + (size_t)t * n;
    auto number = [&](int i) { return PUB ? ti_pub_load(q + i) : q[i]; };
    const float m = number(0), sum = number(1), u = number(2), c = number(3), above = number(4);
    auto load = [&](int j) {
        const uint64_t* k = keys + ti_min(j + lane, n - 1);
        const uint64_t key = PUB ? ti_pub_load(k) : *k;
        return j + lane < n ? key : 0ull;
    };
    uint64_t kept = 0;
    if (64 * wave < n) kept = taken_first(load(64 * wave), ti_min(64, n - 64 * wave));
    for (int j = 64 * (wave + WAVES); j < n; j += 64 * WAVES) kept = taken(kept, load(j));
    if (n > 64) {
        if (wave > 0) s_waves[wave - 1][63 - lane] = kept;
        __syncthreads();
    }
    if (wave != 0) return;
    if (n > 64)
#pragma unroll
        for (int w = 0; w < WAVES - 1; w++) kept = larger(kept, s_waves[w][lane]);
    const Sum r = wave_joined(has ? Sum{m, sum, u, __float_as_int(c)} : Sum{LOW, 0.0f, 0.0f, 0});
    finish(a, t, r, ti_wave_sum_i(has ? __float_as_int(above) : 0), kept);
}

template <bool TOP>
__global__ __launch_bounds__(256) void k_logprobs(LpArgs a) {
    extern __shared__ __align__(16) uint64_t s_keys[];
    __shared__ Sum s_sum[WAVES];
    __shared__ int s_above[WAVES], s_all, s_last;
    __shared__ uint32_t s_limit[WAVES];
    __shared__ uint64_t s_waves[2 * WAVES][64];            // the waves' lists and kept keys; later three waves' parts
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x / a.segs, seg = blockIdx.x % a.segs, top = a.top;
    const float* x = a.x + t * a.ld;
    const int id = a.ids[t];
    const float xi = id >= 0 && id < a.N ? x[id] : INFINITY;
    const long begin = (long)seg * a.per * STEP;
    const int end = (int)ti_min((long)a.N, begin + (long)a.per * STEP);
    uint64_t* list = s_keys + wave * (EPT * top + LONG);   // what a chunk adds at most, behind what is there
    uint64_t kept = 0;
    int listed = 0;
    uint32_t last = 0;                                     // a value that `top` keys so far reach: what comes later has to be larger
    Sum r = {LOW, 0.0f, 0.0f, 0};
    int above = 0;
    auto load = [&](long at, float (&v)[EPT]) {
        const long i0 = at + 4 * lane;
        if (at + CHUNK <= end) {
#pragma unroll
            for (int i = 0; i < EPT / 4; i++) {
                const v4f_u w = __builtin_nontemporal_load(reinterpret_cast<const v4f_u*>(x + i0 + 256 * i));
#pragma unroll
                for (int e = 0; e < 4; e++) v[4 * i + e] = w[e];
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < EPT; i++) v[i] = x[ti_min(i0 + 256 * (i / 4) + i % 4, (long)a.N - 1)];
    };
    float v[EPT], next[EPT];
    long at = begin + wave * CHUNK;
    if (at < end) load(at, v);
    if (at + STEP < end) load(at + STEP, next);
    if constexpr (TOP) last = first_limit(v, end - at, top, reinterpret_cast<uint32_t*>(&s_waves[0][0]));
    for (bool begun = false; at < end; at += STEP, begun = true) {
        if (begun) {
#pragma unroll
            for (int i = 0; i < EPT; i++) v[i] = next[i];
            if (at + STEP < end) load(at + STEP, next);
        }
        const int in = (int)ti_min((long)CHUNK, end - at) - 4 * lane;       // of the lane's elements, those at 256 (i / 4) + i % 4 below it
        if (at + CHUNK > end) {
#pragma unroll
            for (int i = 0; i < EPT; i++) v[i] = 256 * (i / 4) + i % 4 < in ? v[i] : -INFINITY;
        }
        float most = v[0];
#pragma unroll
        for (int i = 1; i < EPT; i++) most = fmaxf(most, v[i]);
        const float m = fmaxf(r.m, most);
        r = turned(r, m);
#pragma unroll
        for (int i = 0; i < EPT; i++) {
            const float z = v[i] - m, e = __builtin_amdgcn_exp2f(z * 1.44269504088896341f);
            r.s += z == 0.0f ? 0.0f : e;
            r.c += z == 0.0f;
            r.u = fmaf(e, fmaxf(z, -150.0f), r.u);         // e^-150 is 0; a NaN is in s
            above += v[i] > xi;
        }
        if constexpr (TOP) {
            const float least = value_of(begun ? last : last - 1);               // what reaches the first step's limit counts in it
            const uint64_t lanes = __ballot(last == 0 || most > least);
            if (lanes == 0) continue;
            if (last != 0 && (!begun || __builtin_popcountll(lanes) < top)) {
#pragma unroll
                for (int i = 0; i < EPT; i++) {
                    const bool take = v[i] > least;        // no NaN, nothing behind the row's end
                    const uint64_t who = __ballot(take);
                    if (who == 0) continue;
                    if (take) list[listed + __builtin_popcountll(who & ((1ull << lane) - 1))] = key_of(ordered(v[i]), (uint32_t)(at + 256 * (i / 4) + 4 * lane + i % 4));
                    listed += __builtin_popcountll(who);
                }
                if (listed > LONG) {
                    kept = taken(kept, list, listed);
                    listed = 0;
                    last = max(last, value_at(kept, top - 1));
                }
                continue;
            }
            uint32_t u[EPT], mine = 0;
#pragma unroll
            for (int i = 0; i < EPT; i++) {
                u[i] = 256 * (i / 4) + i % 4 < in ? ordered(v[i]) : 0u;
                mine = max(mine, u[i]);
            }
            uint32_t limit = last, place = 0xffffffffu;    // listed: above the limit, or at it up to this place in the chunk
            bool ties = false;
            if (__builtin_popcountll(__ballot(mine > last)) >= top) {
                limit = 0;
                int held = 65;                             // lanes at or above the limit
                for (uint32_t bit = 0x80000000u; bit && held > top; bit >>= 1) {
                    const int n = __builtin_popcountll(__ballot(mine >= (limit | bit)));
                    if (n >= top) {
                        limit |= bit;
                        held = n;
                    }
                }
                // a prefix that just `top` lanes reach may be below what was the limit before
                ties = limit > last;
                limit = max(limit, last);
                const int more = __builtin_popcountll(__ballot(mine > limit));
                if (held > top) {
                    // lanes whose maxima are equal: those whose first is at the lowest places
                    uint32_t first = 0xffffffffu;
#pragma unroll
                    for (int i = EPT - 1; i >= 0; i--)
                        if (u[i] == limit) first = 256 * (i / 4) + 4 * lane + i % 4;
                    if (mine != limit) first = 0xffffffffu;
                    place = 0;
                    for (uint32_t bit = CHUNK / 2; bit; bit >>= 1)
                        if (more + __builtin_popcountll(__ballot(first < (place | bit))) < top) place |= bit;
                }
            }
#pragma unroll
            for (int i = 0; i < EPT; i++) {
                const uint32_t p = 256 * (i / 4) + 4 * lane + i % 4;
                const bool take = u[i] > limit || (ties && u[i] == limit && p <= place);
                const uint64_t who = __ballot(take);
                if (take) list[listed + __builtin_popcountll(who & ((1ull << lane) - 1))] = key_of(u[i], (uint32_t)(at + p));
                listed += __builtin_popcountll(who);
            }
            last = limit;
            if (listed > LONG) {
                kept = taken(kept, list, listed);
                listed = 0;
                last = max(last, value_at(kept, top - 1));
            }
        }
    }
    r = wave_joined(r);
    above = ti_wave_sum_i(above);
    if (lane == 0) {
        s_sum[wave] = r;
        s_above[wave] = above;
        s_limit[wave] = last;
        if (wave == 0) s_all = 0;
    }
    __syncthreads();
    r = joined(joined(s_sum[0], s_sum[1]), joined(s_sum[2], s_sum[3]));
    above = (s_above[0] + s_above[1]) + (s_above[2] + s_above[3]);
    uint64_t key = 0;
    if constexpr (TOP) {
        // what reaches the largest of the waves' limits, in any order
        const uint32_t limit = max(max(s_limit[0], s_limit[1]), max(s_limit[2], s_limit[3]));
        uint64_t* all = &s_waves[0][0];
        ti_wave_lds_fence();
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint64_t k = half ? lane < top ? kept : 0ull : lane < listed ? list[lane] : 0ull;
            const bool take = k && (uint32_t)(k >> 32) >= limit;
            const uint64_t who = __ballot(take);
            if (who == 0) continue;
            int first = 0;
            if (lane == 0) first = __hip_atomic_fetch_add(&s_all, __builtin_popcountll(who), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            first = __builtin_amdgcn_readfirstlane(first);
            if (take) all[first + __builtin_popcountll(who & ((1ull << lane) - 1))] = k;
        }
        __syncthreads();
        if (wave == 0) {
            const int n = s_all;
            key = taken_first(lane < n ? all[lane] : 0ull, n);
            if (n > 64) key = taken(key, all + 64, n - 64);
            key = lane < top ? key : 0;
        }
    }
    if (a.segs == 1) {
        if (wave == 0) finish(a, t, r, above, key);
        return;
    }
    const size_t p = (size_t)t * a.segs + seg;
    float* q = a.part + p * PART;
    if (!a.arrived) {
        if (wave != 0) return;
        if (lane == 0) {
            *reinterpret_cast<float4*>(q) = make_float4(r.m, r.s, r.u, __int_as_float(r.c));
            q[4] = __int_as_float(above);
        }
        if (TOP && lane < top) a.keys[p * top + lane] = key;
        return;
    }
    if (wave == 0) {
        const float number = lane == 0 ? r.m : lane == 1 ? r.s : lane == 2 ? r.u : __int_as_float(lane == 3 ? r.c : above);
        if (lane < 5) ti_pub_store(q + lane, number);
        if (TOP && lane < top) ti_pub_store(a.keys + p * top + lane, key);
        ti_stores_done();
        if (lane == 0) s_last = ti_arrive(a.arrived + t * TI_SYNC_LOGPROBS_STRIDE) == (uint32_t)(a.segs - 1);
    }
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0) ti_pub_store(a.arrived + t * TI_SYNC_LOGPROBS_STRIDE, 0u);
    join_parts<true>(a, t, s_waves);
}

__global__ __launch_bounds__(256) void k_logprobs_join(LpArgs a) {
    __shared__ uint64_t s_waves[WAVES - 1][64];
    join_parts<false>(a, blockIdx.x, s_waves);
}

}  // namespace

extern "C" int ti_logprobs(ti_ctx* c, const float* logits, const int32_t* ids, float* lp, float* entropy, int32_t* rank, int32_t* top_ids,
                           float* top_lp, int T, int N, int ld, int top) {
    TI_CHECK_CTX(c);
    TI_REQUIRE(logits && ids && lp, "ti_logprobs: null buffer");
    TI_REQUIRE(T > 0 && T <= ROWS_MAX && N > 0 && N <= TI_POS_END, "ti_logprobs: bad shape (T=%d N=%d)", T, N);
    TI_REQUIRE(top >= 0 && top <= TOP_MAX && top <= N, "ti_logprobs: top = %d of %d logits, at most %d", top, N, TOP_MAX);
    TI_REQUIRE(top == 0 || (top_ids && top_lp), "ti_logprobs: null buffer for the likeliest tokens");
    TI_REQUIRE(ld == 0 || ld >= N, "ti_logprobs: rows of %d logits, %d apart", N, ld);
    LpArgs a = {logits, ids, lp, entropy, rank, top_ids, top_lp, nullptr, nullptr, nullptr, ld ? ld : N, T, N, top, 1, 0};
    // workgroups of whole steps until every CU has four, or two where tokens are kept, which costs most in a wave's first chunk
    // (400 rows with 20 tokens 67.7 us, with four a CU 71.8; 1000 rows of 30000 with 5 36.8 / 41.1; 48 rows with 20 21.0 / 21.5)
    const long steps = ((long)N + STEP - 1) / STEP;
    const long segs = ti_max(1L, ti_min(ti_min((long)SEGS_MAX, steps), ((top ? 2L : 4L) * c->cus + T - 1) / T));
    a.per = (int)((steps + segs - 1) / segs);
    a.segs = (int)((steps + a.per - 1) / a.per);
    // fewer than T + 4 CUs of them
    static_assert((ROWS_MAX + 4L * 4096) * (4 * PART + 8 * TOP_MAX) <= 4L * TI_ATTN_ROWSPLITS * TI_ATTN_HD_MAX, "the parts fit the scratch");
    a.part = c->attn_po;
    a.keys = reinterpret_cast<uint64_t*>(a.part + (size_t)T * a.segs * PART);
    if (T <= TI_LOGPROBS_ROWS) a.arrived = c->sync + TI_SYNC_LOGPROBS;
    const unsigned grid = (unsigned)(T * a.segs);
    if (top) k_logprobs<true><<<grid, 256, WAVES * (EPT * top + LONG) * 8, c->stream>>>(a);
    else k_logprobs<false><<<grid, 256, 0, c->stream>>>(a);
    TI_LAUNCHED("k_logprobs");
    if (a.segs > 1 && !a.arrived) {
        k_logprobs_join<<<T, 256, 0, c->stream>>>(a);
        TI_LAUNCHED("k_logprobs_join");
    }
    return TI_OK;
}
