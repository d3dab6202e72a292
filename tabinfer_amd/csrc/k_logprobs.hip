// k_logprobs.hip — log probabilities of given tokens under rows of logits, the rows' entropy and their likeliest tokens, in one pass over
// the logits. The reference has no counterpart: its sampler keeps an index (models/qwen3.js:2624-2740).
//
// With M the row's maximum, S = sum e^(x - M) and U = sum e^(x - M) (x - M): log p(x) = (x - M) - ln S and the entropy
// ln S - U / S, two terms of one sign. A lane keeps (m, s, u) of its own elements and turns them to a new maximum by
// s' = a s, u' = a (u + (m - m') s), a = e^(m - m'); lanes, waves and workgroups are joined by the same rule in a fixed order.
//
// The likeliest: a value and its index are one 64-bit key (the float's bits in an order of whole numbers, then the inverted index: the lower
// index wins), so that no two are equal. A wave takes 1024 elements at a time, in registers. Where fewer than `top` lanes hold something
// above its last kept key, what is above it goes to a list in LDS; where as many do, as always at first, the limit is raised to the top-th
// largest of the lanes' maxima, found bit by bit with ballots: no more than `top` lanes then hold anything to list, so that the list's room,
// 16 keys a lane, is bounded whatever the values are. List and kept keys are ranked by counting. So all chunks but a wave's first
// cost a comparison and little more.
#include "ti_dev.h"
#include "ti_span.h"

namespace {

typedef float v4f_u __attribute__((ext_vector_type(4), aligned(4)));   // rows start anywhere

constexpr int EPT = 16, CHUNK = 64 * EPT, WAVES = 4, STEP = WAVES * CHUNK;     // elements of a lane, a wave's chunk, a workgroup's
constexpr int TOP_MAX = 64;                  // one lane a kept key
constexpr int SEGS_MAX = 64;                 // workgroups a row: one lane each where they are joined
constexpr int ROWS_MAX = 1 << 17;
constexpr float LOW = -3.402823466e38f;

struct LpArgs {
    const float* x;
    const int32_t* ids;
    float *lp, *ent;
    int32_t *rank, *top_ids;
    float* top_lp;
    float4* part;                            // [row][segs] (m, s, u, number of logits above the token's)
    uint64_t* keys;                          // [row][segs][top], from large to small, 0 behind the last
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
};
__device__ __forceinline__ float down_to(float d) { return d < -150.0f ? -150.0f : d; }      // e^-150 is 0; NaN stays
__device__ __forceinline__ Sum joined(const Sum& a, const Sum& b) {
    const float m = fmaxf(a.m, b.m), da = down_to(a.m - m), db = down_to(b.m - m);
    const float ea = expf(da), eb = expf(db);
    return {m, a.s * ea + b.s * eb, ea * (a.u + da * a.s) + eb * (b.u + db * b.s)};
}
__device__ __forceinline__ Sum wave_joined(Sum a) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = joined(a, Sum{ti_xor(a.m, o), ti_xor(a.s, o), ti_xor(a.u, o)});
    return a;
}

// a wave's keys: kept ones from large to small, 0 behind the last, and a list
struct Kept {
    uint64_t *now, *next, *list;
};
// `n` listed keys into the kept ones
__device__ __forceinline__ void keep(Kept& k, int n, int top) {
    const int lane = threadIdx.x & 63;
    ti_wave_lds_fence();
    if (lane < top) k.next[lane] = 0;
    ti_wave_lds_fence();
    for (int j = lane; j < n + top; j += 64) {
        const uint64_t key = j < top ? k.now[j] : k.list[j - top];
        if (key == 0) continue;
        int rank = 0;
        for (int i = 0; i < top; i++) rank += k.now[i] > key;
        for (int i = 0; i < n; i++) rank += k.list[i] > key;
        if (rank < top) k.next[rank] = key;
    }
    ti_wave_lds_fence();
    uint64_t* t = k.now;
    k.now = k.next;
    k.next = t;
}

// what a row's numbers come to, and its likeliest tokens' (key of lane i the i-th)
__device__ __forceinline__ void finish(const LpArgs& a, int t, const Sum& r, int above, uint64_t key) {
    const int lane = threadIdx.x & 63;
    const float ln = logf(r.s);
    if (lane == 0) {
        const int id = a.ids[t];
        const bool there = id >= 0 && id < a.N;
        a.lp[t] = there ? (a.x[t * a.ld + id] - r.m) - ln : -INFINITY;
        if (a.ent) a.ent[t] = ln - r.u / r.s;
        if (a.rank) a.rank[t] = there ? above + 1 : 0;
    }
    if (lane < a.top) {
        const size_t at = (size_t)t * a.top + lane;
        a.top_ids[at] = key ? (int32_t)~(uint32_t)key : -1;
        a.top_lp[at] = key ? (value_of((uint32_t)(key >> 32)) - r.m) - ln : -INFINITY;
    }
}

template <bool TOP>
__global__ __launch_bounds__(256) void k_logprobs(LpArgs a) {
    extern __shared__ __align__(16) uint64_t s_keys[];
    __shared__ Sum s_sum[WAVES];
    __shared__ int s_above[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = blockIdx.x / a.segs, seg = blockIdx.x % a.segs, top = a.top;
    const float* x = a.x + t * a.ld;
    const int id = a.ids[t];
    const float xi = id >= 0 && id < a.N ? x[id] : INFINITY;
    const long begin = (long)seg * a.per * STEP;
    const int end = (int)ti_min((long)a.N, begin + (long)a.per * STEP);
    Kept kept;
    if constexpr (TOP) {
        kept.now = s_keys + wave * (EPT + 2) * top;
        kept.next = kept.now + top;
        kept.list = kept.next + top;
        if (lane < top) kept.now[lane] = 0;
        ti_wave_lds_fence();
    }
    uint32_t last = 0;                                     // the kept keys' last value: what comes later has to be larger
    Sum r = {LOW, 0.0f, 0.0f};
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
    if (at < end) load(at, next);
    for (; at < end; at += STEP) {
#pragma unroll
        for (int i = 0; i < EPT; i++) v[i] = next[i];
        if (at + STEP < end) load(at + STEP, next);
        const int in = (int)ti_min((long)CHUNK, end - at) - 4 * lane;       // of the lane's elements, those at 256 (i / 4) + i % 4 below it
        if (at + CHUNK > end) {
#pragma unroll
            for (int i = 0; i < EPT; i++) v[i] = 256 * (i / 4) + i % 4 < in ? v[i] : -INFINITY;
        }
        float m = r.m;
#pragma unroll
        for (int i = 0; i < EPT; i++) m = fmaxf(m, v[i]);
        const float d = down_to(r.m - m), f = expf(d);
        r.u = f * (r.u + d * r.s);
        r.s = f * r.s;
        r.m = m;
#pragma unroll
        for (int i = 0; i < EPT; i++) {
            const float z = down_to(v[i] - m), e = __builtin_amdgcn_exp2f(z * 1.44269504088896341f);
            r.s += e;
            r.u = fmaf(e, z, r.u);
            above += v[i] > xi;
        }
        if constexpr (TOP) {
            uint32_t u[EPT], mine = 0;
#pragma unroll
            for (int i = 0; i < EPT; i++) {
                u[i] = 256 * (i / 4) + i % 4 < in ? ordered(v[i]) : 0u;
                mine = max(mine, u[i]);
            }
            if (!__any(mine > last)) continue;
            uint32_t limit = last, place = 0xffffffffu;    // listed: above the limit, or at it up to this place in the chunk
            bool ties = false;
            if (__builtin_popcountll(__ballot(mine > last)) >= top) {
                limit = 0;
                for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
                    if (__builtin_popcountll(__ballot(mine >= (limit | bit))) >= top) limit |= bit;
                ties = true;
                const int more = __builtin_popcountll(__ballot(mine > limit));
                if (__builtin_popcountll(__ballot(mine >= limit)) > top) {
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
            int n = 0;
#pragma unroll
            for (int i = 0; i < EPT; i++) {
                const uint32_t p = 256 * (i / 4) + 4 * lane + i % 4;
                const bool take = u[i] > limit || (ties && u[i] == limit && p <= place);
                const uint64_t who = __ballot(take);
                if (take) kept.list[n + __builtin_popcountll(who & ((1ull << lane) - 1))] = key_of(u[i], (uint32_t)(at + p));
                n += __builtin_popcountll(who);
            }
            keep(kept, n, top);
            last = (uint32_t)(kept.now[top - 1] >> 32);
        }
    }
    r = wave_joined(r);
    above = ti_wave_sum_i(above);
    if (lane == 0) {
        s_sum[wave] = r;
        s_above[wave] = above;
    }
    __syncthreads();
    r = joined(joined(s_sum[0], s_sum[1]), joined(s_sum[2], s_sum[3]));
    above = (s_above[0] + s_above[1]) + (s_above[2] + s_above[3]);
    uint64_t key = 0;
    if constexpr (TOP) {
        // the waves' kept keys, ranked into the first wave's list
        const int tid = threadIdx.x;
        uint64_t* out = s_keys + WAVES * (EPT + 2) * top;
        uint64_t* all = out + top;
        if (tid < top) out[tid] = 0;
        if (lane < top) all[wave * top + lane] = kept.now[lane];
        __syncthreads();
        if (tid < 4 * top && all[tid]) {
            int rank = 0;
            for (int i = 0; i < 4 * top; i++) rank += all[i] > all[tid];
            if (rank < top) out[rank] = all[tid];
        }
        __syncthreads();
        if (lane < top) key = out[lane];
    }
    if (wave != 0) return;
    if (a.segs == 1) return finish(a, t, r, above, key);
    const size_t p = (size_t)t * a.segs + seg;
    if (lane == 0) a.part[p] = make_float4(r.m, r.s, r.u, __int_as_float(above));
    if (TOP && lane < top) a.keys[p * top + lane] = key;
}

// A wave a row: its parts' numbers, a lane each, and of their keys the largest of the heads, `top` times
__global__ __launch_bounds__(256) void k_logprobs_join(LpArgs a) {
    const int lane = threadIdx.x & 63, t = blockIdx.x * WAVES + (threadIdx.x >> 6);
    if (t >= a.T) return;                                  // wave-uniform
    const bool has = lane < a.segs;
    const size_t p = (size_t)t * a.segs + ti_min(lane, a.segs - 1);
    const float4 q = a.part[p];
    const Sum r = wave_joined(has ? Sum{q.x, q.y, q.z} : Sum{LOW, 0.0f, 0.0f});
    const int above = ti_wave_sum_i(has ? __float_as_int(q.w) : 0);
    uint64_t key = 0;
    if (a.top) {
        const uint64_t* mine = a.keys + p * a.top;
        uint64_t head = has ? mine[0] : 0, after = has && a.top > 1 ? mine[1] : 0;
        int at = 1;
        for (int i = 0; i < a.top; i++) {
            uint64_t best = head;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const uint64_t other = (uint64_t)ti_xor((uint32_t)(best >> 32), o) << 32 | ti_xor((uint32_t)best, o);
                best = other > best ? other : best;
            }
            if (best == 0) break;
            if (lane == i) key = best;
            if (head == best) {
                head = after;
                at++;
                after = at < a.top ? mine[at] : 0;
            }
        }
    }
    finish(a, t, r, above, key);
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
    LpArgs a = {logits, ids, lp, entropy, rank, top_ids, top_lp, nullptr, nullptr, ld ? ld : N, T, N, top, 1, 0};
    // four workgroups a CU where the rows are long enough, each of whole steps
    const long steps = ((long)N + STEP - 1) / STEP;
    const long segs = ti_max(1L, ti_min(ti_min((long)SEGS_MAX, steps), (4L * c->cus + T - 1) / T));
    a.per = (int)((steps + segs - 1) / segs);
    a.segs = (int)((steps + a.per - 1) / a.per);
    // fewer than T + 4 CUs of them
    static_assert((ROWS_MAX + 4L * 4096) * (16 + 8 * TOP_MAX) <= 4L * TI_ATTN_ROWSPLITS * TI_ATTN_HD_MAX, "the parts fit the scratch");
    a.part = reinterpret_cast<float4*>(c->attn_po);
    a.keys = reinterpret_cast<uint64_t*>(a.part + (size_t)T * a.segs);
    const unsigned grid = (unsigned)(T * a.segs);
    if (top) k_logprobs<true><<<grid, 256, (WAVES * (EPT + 2) + 5) * top * 8, c->stream>>>(a);
    else k_logprobs<false><<<grid, 256, 0, c->stream>>>(a);
    TI_LAUNCHED("k_logprobs");
    if (a.segs > 1) {
        k_logprobs_join<<<(T + WAVES - 1) / WAVES, 256, 0, c->stream>>>(a);
        TI_LAUNCHED("k_logprobs_join");
    }
    return TI_OK;
}
