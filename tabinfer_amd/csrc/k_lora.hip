// k_lora.hip — low-rank adapters of many requests beside a shared projection: y[t] += s_a B_a (A_a x[t]), a = idx[t]. The reference has no
// counterpart (its projections: models/qwen3.js:1588-1608).
//
// Rows meet adapters in tiles of a few rows: a tile's distinct adapters are taken one behind the other, or dealt out to workgroups ("slots"),
// each for the rows that are its own.
#include "ti_dev.h"
#include "ti_span.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int RANK_MAX = 128;
constexpr int DIM_MAX = 1 << 30;            // of K and N: 32-bit indices step past them, by columns and rounding of all parts, or by stages loaded ahead
constexpr long ROWS_MAX = 1 << 18, SCRATCH = (long)TI_ATTN_ROWSPLITS * TI_ATTN_HD_MAX;
static_assert(ROWS_MAX * RANK_MAX <= SCRATCH, "h of every row fits the scratch");

struct LoraArgs {
    const float* x;
    const int32_t* idx;
    const uint16_t *a, *b;
    const float* scale;
    float* y;
    float* h;                                // prompts: [splits][T][rp]
    long ldx, ldy;
    int T, K, N, r, n, slots, parts, splits, rp;   // parts of N, of K; rp: r in whole tiles of 16
};

// A tile's distinct adapters, one behind the other: `own` is the adapter of the tile's row `lane`, -1 none
template <int ROWS>
struct Adapters {
    uint64_t todo;
    int own, at, id;
    uint32_t rows;                           // of adapter `id`
    __device__ static int fetch(const LoraArgs& a, int row0) {      // ahead of other loads, since they come back in order
        const int lane = threadIdx.x & 63;
        return a.idx[ti_min(row0 + ti_min(lane, ROWS - 1), a.T - 1)];
    }
    __device__ Adapters(const LoraArgs& a, int row0, int fetched) {
        const int lane = threadIdx.x & 63;
        own = lane < ROWS && row0 + lane < a.T && fetched < a.n ? fetched : -1;
        todo = __ballot(own >= 0);
        at = -1;
    }
    __device__ bool next(int slots, int slot) {            // the next one of those dealt to this slot
        while (todo) {
            id = __builtin_amdgcn_readlane(own, __builtin_ctzll(todo));
            const uint64_t m = __ballot(own == id) & todo;
            todo &= ~m;
            rows = (uint32_t)m;
            if (++at % slots == slot) return true;
        }
        return false;
    }
};

// 8 ranks of a row of B from rank k0 on, those behind the last as zeros
template <bool VEC>
__device__ __forceinline__ uint4 b_ranks(const uint16_t* row, int k0, int r) {
    if constexpr (VEC) return k0 < r ? *reinterpret_cast<const uint4*>(row + k0) : make_uint4(0, 0, 0, 0);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t lo = k0 + 2 * i < r ? row[k0 + 2 * i] : 0u, hi = k0 + 2 * i + 1 < r ? row[k0 + 2 * i + 1] : 0u;
        w[i] = lo | hi << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// ---- few rows ---------------------------------------------------------------------------------------------------
// A workgroup: two rows, its slot's adapters, a part of N; a row or two an adapter, so that weights are read once and there is nothing for the
// matrix cores to share: f32 FMAs on weights as they lie in memory, a wave 512 of K of one rank, or 64 / L rows of B, in whole lines. (With matrix
// operands read from memory, 16 rows apart, each of a load's 64 lanes is a cache access of its own: 48 rows over 16 adapters 12.9 us.)
// h = A x first, four waves along K and four along the ranks; the sums over lanes halve the values with every step. Parts of N form h
// again, each for itself, and there is no second launch.
// Bound by its chain of round trips (indices; A and x; B and y): one row of rank 16, 2048 to 2048, 4.8 us; 48 rows of rank 32 over 16 adapters, 2048
// to 4096 (8.3 MB), 8.6.
constexpr int FROWS = 2, FWAVES = 16, RB = 8, ALONG = 4;   // RB: ranks of a wave at a time; ALONG: waves along K

template <bool BF16>
__device__ __forceinline__ void widen(uint4 w, float (&f)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f[2 * i] = BF16 ? __uint_as_float(u[i] << 16) : ti_h2f((uint16_t)u[i]);
        f[2 * i + 1] = BF16 ? __uint_as_float(u[i] & 0xffff0000u) : ti_h2f((uint16_t)(u[i] >> 16));
    }
}

// L: lanes that share a row of B, 8 ranks each
template <bool BF16, int L, bool VEC>
__global__ __launch_bounds__(64 * FWAVES) void k_lora_few(LoraArgs a) {
    constexpr int NPW = 64 / L, NI = L == 1 ? 2 : 4;       // columns of a wave's load; loads at a time
    constexpr int RPL = L >= FROWS ? 1 : FROWS / L;        // rows whose y a lane reads and writes
    __shared__ float s_part[ALONG][FROWS][RANK_MAX], s_h[FROWS][RANK_MAX];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int part = blockIdx.x % a.parts, slot = blockIdx.x / a.parts % a.slots, row0 = FROWS * (blockIdx.x / (a.parts * a.slots));
    const int per = (a.N + a.parts * NPW - 1) / (a.parts * NPW) * NPW, c0 = ti_min(a.N, part * per), c1 = ti_min(a.N, c0 + per);
    const int sub = lane % L, along = wave % ALONG, group = wave / ALONG;
    Adapters<FROWS> ad(a, row0, Adapters<FROWS>::fetch(a, row0));
    while (ad.next(a.slots, slot)) {
        const uint16_t *w = a.a + (size_t)ad.id * a.r * a.K, *b = a.b + (size_t)ad.id * a.N * a.r;
        const float scale = a.scale[ad.id];
        for (int r0 = 0; r0 < a.r; r0 += RB * FWAVES / ALONG) {
            const int j0 = r0 + RB * group;
            float acc[FROWS][RB];
#pragma unroll
            for (int q = 0; q < FROWS; q++)
#pragma unroll
                for (int i = 0; i < RB; i++) acc[q][i] = 0.0f;
            if (j0 < a.r) {                                // wave-uniform
                for (int k0 = 512 * along; k0 < a.K; k0 += 512 * ALONG) {
                    const int k = k0 + 8 * lane, kc = ti_min(k, a.K - 8);
                    uint4 wv[RB];
#pragma unroll
                    for (int i = 0; i < RB; i++) wv[i] = *reinterpret_cast<const uint4*>(w + (size_t)ti_min(j0 + i, a.r - 1) * a.K + kc);
                    float x[FROWS][8];
#pragma unroll
                    for (int q = 0; q < FROWS; q++) {
                        if (!(ad.rows >> q & 1)) continue;
                        const float* p = a.x + (row0 + q) * a.ldx + kc;
#pragma unroll
                        for (int u = 0; u < 2; u++) {
                            const v4f f = *reinterpret_cast<const v4f*>(p + 4 * u);
#pragma unroll
                            for (int e = 0; e < 4; e++) x[q][4 * u + e] = k < a.K ? f[e] : 0.0f;
                        }
                    }
#pragma unroll
                    for (int i = 0; i < RB; i++) {
                        float f[8];
                        widen<BF16>(wv[i], f);
#pragma unroll
                        for (int q = 0; q < FROWS; q++) {
                            if (!(ad.rows >> q & 1)) continue;
#pragma unroll
                            for (int e = 0; e < 8; e++) acc[q][i] = fmaf(f[e], x[q][e], acc[q][i]);
                        }
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < FROWS; q++) {
                if (!(ad.rows >> q & 1)) continue;
                const float v = transpose_reduce<64, RB>(acc[q], lane);
                if ((lane & 7) == 0 && j0 < a.r) s_part[along][q][j0 + lane / 8] = v;
            }
        }
        // a lane's row of B and its values of y, on their way while the parts of h are joined
        uint4 bv[NI];
        float yv[NI][RPL];
        auto load = [&](int c) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int n = ti_min(c + FWAVES * NPW * i, a.N - 1);
                bv[i] = b_ranks<VEC>(b + (size_t)n * a.r, 8 * sub, a.r);
#pragma unroll
                for (int u = 0; u < RPL; u++) {
                    const int q = sub + L * u;
                    if (q < FROWS && (ad.rows >> q & 1)) yv[i][u] = a.y[(row0 + q) * a.ldy + n];
                }
            }
        };
        const int first = c0 + wave * NPW + lane / L;
        load(first);
        __syncthreads();
        if (tid < FROWS * RANK_MAX) {
            const int q = tid / RANK_MAX, j = tid % RANK_MAX;
            s_h[q][j] = j < a.r && (ad.rows >> q & 1) ? ((s_part[0][q][j] + s_part[1][q][j]) + (s_part[2][q][j] + s_part[3][q][j])) * scale : 0.0f;
        }
        __syncthreads();
        float h[FROWS][8];
#pragma unroll
        for (int q = 0; q < FROWS; q++)
#pragma unroll
            for (int e = 0; e < 8; e++) h[q][e] = s_h[q][8 * sub + e];
        for (int c = first; c - lane / L < c1; c += FWAVES * NPW * NI) {
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const int n = c + FWAVES * NPW * i;
                float f[8], d[FROWS];
                widen<BF16>(bv[i], f);
#pragma unroll
                for (int q = 0; q < FROWS; q++) {
                    d[q] = 0.0f;
                    if (!(ad.rows >> q & 1)) continue;
#pragma unroll
                    for (int e = 0; e < 8; e++) d[q] = fmaf(f[e], h[q][e], d[q]);
#pragma unroll
                    for (int o = L / 2; o > 0; o >>= 1) d[q] += ti_xor(d[q], o);
                }
#pragma unroll
                for (int u = 0; u < RPL; u++) {
                    const int q = sub + L * u;
                    float v = 0.0f;
#pragma unroll
                    for (int k = 0; k < FROWS; k++) v = q == k ? d[k] : v;
                    if (n < c1 && q < FROWS && (ad.rows >> q & 1)) a.y[(row0 + q) * a.ldy + n] = yv[i][u] + v;
                }
            }
            if (c - lane / L + FWAVES * NPW * NI < c1) load(c + FWAVES * NPW * NI);
        }
        __syncthreads();                                   // h is read
    }
}

// ---- prompts ----------------------------------------------------------------------------------------------------
// Both products on the matrix cores, weights exact, f32 activations as two f16 (f16 weights: each row scaled by a power of two, an
// element off by 2^-22 of itself or 2^-39 of the largest) or three bf16 (bf16 weights: exactly), sums in f32. 32 rows a workgroup; an adapter
// multiplies all of its tile's rows, and what is another's is zero or not kept. Two launches: h in parts of K, then its sums times B.
// 1500 rows of rank 64, 6144 to 2048, bf16: 13.9 us (37 MB of x, 2.7 TB/s; bound by splitting x into operands between the stages' barriers) and 10.8 (25 MB
// of y in and out, 2.3 TB/s, behind the sums of h's parts that each workgroup forms first).

// 8 f32 of a row as MFMA operands of the weights' type: f16, scaled by `up`, as hi + lo; bf16, as three. An infinity's other pieces are NaN
template <bool BF16> struct Pieces;
template <> struct Pieces<false> {
    ti_h8 p[2];
    __device__ __forceinline__ void set(const float (&v)[8], float up) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float s = v[e] * up;
            const _Float16 hi = (_Float16)s;
            p[0][e] = hi;
            p[1][e] = (_Float16)(s - (float)hi);
        }
    }
    __device__ __forceinline__ v4f right_of(ti_v4u w, v4f acc) const {      // w the first operand
        const ti_h8 a = __builtin_bit_cast(ti_h8, w);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p[1], acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p[0], acc, 0, 0, 0);
    }
    __device__ __forceinline__ v4f left_of(uint4 w, v4f acc) const {
        const ti_h8 a = __builtin_bit_cast(ti_h8, w);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[1], a, acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(p[0], a, acc, 0, 0, 0);
    }
};
template <> struct Pieces<true> {
    ti_b8 p[3];
    __device__ __forceinline__ void set(const float (&v)[8], float) { ti_bf16x3(v, p); }
    __device__ __forceinline__ v4f right_of(ti_v4u w, v4f acc) const {
        const ti_b8 a = __builtin_bit_cast(ti_b8, w);
#pragma unroll
        for (int i = 2; i >= 0; i--) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p[i], acc, 0, 0, 0);
        return acc;
    }
    __device__ __forceinline__ v4f left_of(uint4 w, v4f acc) const {
        const ti_b8 a = __builtin_bit_cast(ti_b8, w);
#pragma unroll
        for (int i = 2; i >= 0; i--) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p[i], a, acc, 0, 0, 0);
        return acc;
    }
};
// 2^k that brings a row's largest magnitude (of the lanes 16 apart) to [2^14, 2^15), where f16 pieces want it
template <bool BF16>
__device__ __forceinline__ int row_exponent(float mx) {
    if constexpr (BF16) return 0;
    mx = fmaxf(mx, ti_xor(mx, 16));
    mx = fmaxf(mx, ti_xor(mx, 32));
    int ex = 15;
    if (mx > 0.0f && mx < INFINITY) (void)frexpf(mx, &ex);
    return ti_min(15 - ex, 100);
}

constexpr int PROWS = 32, RW = PROWS / 16, DWAVES = 8, PWAVES = 4, SPLITS = 4;
constexpr int KC = 128, XP = KC / 4, WP = KC / 8;          // K of a stage; 16-byte pieces of its rows of x and of A

template <bool BF16>
__device__ __forceinline__ float one(uint16_t w) { return BF16 ? __uint_as_float((uint32_t)w << 16) : ti_h2f(w); }
// Ranks j0 .. j0 + 3 of a row's h over K's [k0, k1), element by element: where the pieces came to NaN, as they do beside an infinity, whose other
// pieces have no value. 1500 rows of rank 64, 6144 to 2048: one such row 0.15 ms a call, all of them 0.4 (NaN) to 0.95 (infinities)
template <bool BF16>
__device__ __forceinline__ v4f sums(const LoraArgs& a, const uint16_t* w, int row, int j0, int k0, int k1) {
    v4f h = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = k0; k < k1; k++) {
        const float x = a.x[row * a.ldx + k];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint16_t u = w[(size_t)ti_min(j0 + e, a.r - 1) * a.K + k];
            h[e] = fmaf(one<BF16>(u), x, h[e]);
        }
    }
    return h;
}

// A workgroup: 32 rows, a part of K in stages of 128, read in whole lines and put into LDS, pieces permuted so that 16 rows' are in different
// banks; three stages are on their way. A wave takes 16 rows and one 32-step of each stage, so that a value of x is split once.
template <bool BF16, int RT>
__global__ __launch_bounds__(64 * DWAVES, 1) void k_lora_down(LoraArgs a) {
    constexpr int NX = PROWS * XP / (64 * DWAVES), NW = (RT * 16 * WP + 64 * DWAVES - 1) / (64 * DWAVES), AHEAD = 3;
    struct Stage {
        v4f x[PROWS * XP];
        ti_v4u w[RT * 16 * WP];
    };
    __shared__ union {
        Stage s[2];
        v4f part[DWAVES][RT][64];
    } L;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m16 = lane & 15, j = lane >> 4, q = wave % RW, ks = wave / RW;
    const int ptiles = (a.T + PROWS - 1) / PROWS, slot = blockIdx.x / (a.splits * ptiles);
    const int split = blockIdx.x % a.splits, row0 = PROWS * (blockIdx.x / a.splits % ptiles);
    const int stages = (a.K + KC - 1) / KC, per = (stages + a.splits - 1) / a.splits, g0 = split * per, g1 = ti_min(stages, g0 + per);
    const int fetched = Adapters<PROWS>::fetch(a, row0);
    // this thread's pieces of a stage
    const float* xp[NX];
    int xk[NX], wk[NW], wr[NW], wp[NW];
#pragma unroll
    for (int i = 0; i < NX; i++) {
        const int p = 64 * DWAVES * i + tid, row = p / XP;
        xp[i] = a.x + (long)ti_min(row0 + row, a.T - 1) * a.ldx;
        xk[i] = 4 * ((p % XP) ^ (row & 15));
    }
#pragma unroll
    for (int i = 0; i < NW; i++) {
        wp[i] = (64 * DWAVES * i + tid) % (RT * 16 * WP);  // one tile of ranks: twice the same, each half of the threads
        wr[i] = ti_min(wp[i] / WP, a.r - 1);
        wk[i] = 8 * ((wp[i] % WP) ^ (wp[i] / WP & 15));
    }
    v4f xv[AHEAD][NX];
    ti_v4u wv[AHEAD][NW];
    auto load_x = [&](int u, int g) {
#pragma unroll
        for (int i = 0; i < NX; i++) xv[u][i] = *reinterpret_cast<const v4f*>(xp[i] + ti_min(KC * g + xk[i], a.K - 4));
    };
#pragma unroll
    for (int u = 0; u < AHEAD; u++) load_x(u, g0 + u);
    Adapters<PROWS> ad(a, row0, fetched);
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    bool again = false;
    while (ad.next(a.slots, slot)) {
        const uint16_t* w = a.a + (size_t)ad.id * a.r * a.K;
        auto load_w = [&](int u, int g) {
#pragma unroll
            for (int i = 0; i < NW; i++) wv[u][i] = *reinterpret_cast<const ti_v4u*>(w + (size_t)wr[i] * a.K + ti_min(KC * g + wk[i], a.K - 8));
        };
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            if (again) load_x(u, g0 + u);
            load_w(u, g0 + u);
        }
        again = true;
        const bool in = ad.rows >> (16 * q + m16) & 1;     // rows of other adapters may hold anything
        v4f acc[RT];
#pragma unroll
        for (int k = 0; k < RT; k++) acc[k] = zero;
        for (int g = g0; g < g1; g += AHEAD) {
#pragma unroll
            for (int u = 0; u < AHEAD; u++) {
                Stage& S = L.s[(g - g0 + u) & 1];
#pragma unroll
                for (int i = 0; i < NX; i++) S.x[64 * DWAVES * i + tid] = xv[u][i];
#pragma unroll
                for (int i = 0; i < NW; i++) S.w[wp[i]] = wv[u][i];
                __syncthreads();                           // this stage is there; the one before the last has been read
                load_x(u, g + u + AHEAD);
                load_w(u, g + u + AHEAD);
                float v[8], mx = 0.0f;
                const bool there = in && g + u < g1 && KC * (g + u) + 32 * ks < a.K;   // stages behind the last count nothing
#pragma unroll
                for (int z = 0; z < 2; z++) {
                    const v4f f = S.x[(16 * q + m16) * XP + ((8 * ks + 2 * j + z) ^ m16)];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        v[4 * z + e] = there ? f[e] : 0.0f;
                        mx = fmaxf(mx, fabsf(v[4 * z + e]));
                    }
                }
                const int ex = row_exponent<BF16>(mx);
                const float up = ldexpf(1.0f, ex), down = ldexpf(1.0f, -ex);
                Pieces<BF16> p;
                p.set(v, up);
#pragma unroll
                for (int k = 0; k < RT; k++) {
                    const ti_v4u f = S.w[(16 * k + m16) * WP + ((4 * ks + j) ^ m16)];
                    if constexpr (BF16) acc[k] = p.right_of(f, acc[k]);
                    else {
                        const v4f d = p.right_of(f, zero);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[k][e] = fmaf(d[e], down, acc[k][e]);
                    }
                }
            }
        }
        // the 32-steps' sums: lane (m16, j) of tile k holds ranks 16 k + 4 j.. of row m16
        __syncthreads();
#pragma unroll
        for (int k = 0; k < RT; k++) L.part[wave][k][lane] = acc[k];
        __syncthreads();
        for (int z = tid; z < RW * RT * 64; z += 64 * DWAVES) {
            const int k = z / 64 % RT, qq = z / (64 * RT), l = z & 63, t = 16 * qq + (l & 15);
            if (!(ad.rows >> t & 1) || 16 * k >= a.rp) continue;
            v4f h = zero;
#pragma unroll
            for (int s = 0; s < DWAVES / RW; s++) h += L.part[RW * s + qq][k][l];
            const int j0 = 16 * k + 4 * (l >> 4);
            if (__builtin_expect(__builtin_isunordered(h[0] + h[1], h[2] + h[3]), 0)) h = sums<BF16>(a, w, row0 + t, j0, KC * g0, ti_min(a.K, KC * g1));
            *reinterpret_cast<v4f*>(a.h + ((size_t)split * a.T + row0 + t) * a.rp + j0) = h;
        }
        __syncthreads();
    }
}

// A workgroup: 32 rows, a part of N; a wave 16 columns at a time, next to each other. h, all parts of K together and times the adapter's
// scale, is formed in LDS; y is read and written 16 columns of four rows at a time
template <bool BF16, bool VEC, int RS>
__global__ __launch_bounds__(64 * PWAVES) void k_lora_up(LoraArgs a) {
    constexpr int NB = 2, HS = 32 * RS + 4;
    __shared__ __align__(16) float s_h[PROWS][HS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m16 = lane & 15, j = lane >> 4;
    const int ptiles = (a.T + PROWS - 1) / PROWS, slot = blockIdx.x / (a.parts * ptiles);
    const int part = blockIdx.x % a.parts, row0 = PROWS * (blockIdx.x / a.parts % ptiles);
    const int tiles = (a.N + 15) / 16, per = (tiles + a.parts - 1) / a.parts, t0 = part * per + NB * wave, t1 = ti_min(tiles, (part + 1) * per);
    Adapters<PROWS> ad(a, row0, Adapters<PROWS>::fetch(a, row0));
    if (!ad.next(a.slots, slot)) return;                   // the same in every wave
    for (int z = tid; z < PROWS * 8 * RS; z += 64 * PWAVES) {
        const int t = z / (8 * RS), k = 4 * (z % (8 * RS)), row = ti_min(row0 + t, a.T - 1), id = a.idx[row];
        v4f h = {0.0f, 0.0f, 0.0f, 0.0f};
        if (k < a.rp) {
            v4f f[SPLITS];
#pragma unroll
            for (int s = 0; s < SPLITS; s++) f[s] = *reinterpret_cast<const v4f*>(a.h + ((size_t)ti_min(s, a.splits - 1) * a.T + row) * a.rp + k);
            const float sc = id >= 0 && id < a.n ? a.scale[id] : 0.0f;
#pragma unroll
            for (int s = 0; s < SPLITS; s++)
                if (s < a.splits) h += f[s];
#pragma unroll
            for (int e = 0; e < 4; e++) h[e] = k + e < a.r ? h[e] * sc : 0.0f;
        }
        *reinterpret_cast<v4f*>(&s_h[t][k]) = h;
    }
    uint4 bv[NB][RS];
    float yv[NB][RW][4];
    auto row_in = [&](int q, int e) { return ad.rows >> (16 * q + 4 * j + e) & 1; };
    float* y = a.y + (row0 + 4 * j) * a.ldy + m16;
    auto load = [&](int t) {
        const uint16_t* b = a.b + (size_t)ad.id * a.N * a.r;
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const int c = 16 * (t + i);
            const uint16_t* br = b + (size_t)ti_min(c + m16, a.N - 1) * a.r;
#pragma unroll
            for (int s = 0; s < RS; s++) bv[i][s] = b_ranks<VEC>(br, 32 * s + 8 * j, a.r);
#pragma unroll
            for (int q = 0; q < RW; q++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (row_in(q, e) && c + m16 < a.N) yv[i][q][e] = y[(16 * q + e) * a.ldy + c];
        }
    };
    load(t0);
    __syncthreads();
    Pieces<BF16> hp[RW][RS];
    float down[RW][4];
    uint32_t infinite = 0;                                 // rows whose h holds an infinity
#pragma unroll
    for (int q = 0; q < RW; q++) {
        float v[RS][8], mx = 0.0f;
#pragma unroll
        for (int s = 0; s < RS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[s][e] = s_h[16 * q + m16][32 * s + 8 * j + e];
                mx = fmaxf(mx, fabsf(v[s][e]));
            }
        const uint64_t some = __ballot(mx == INFINITY);
        infinite |= (uint32_t)((some | some >> 16 | some >> 32 | some >> 48) & 0xffff) << (16 * q);
        const int ex = row_exponent<BF16>(mx);
        const float up = ldexpf(1.0f, ex);
#pragma unroll
        for (int e = 0; e < 4; e++) down[q][e] = BF16 ? 1.0f : ldexpf(1.0f, -__shfl(ex, 4 * j + e));
#pragma unroll
        for (int s = 0; s < RS; s++) hp[q][s].set(v[s], up);
    }
    ad.rows &= ~infinite;
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    for (bool first = true;; first = false) {
        for (int t = t0; t < t1; t += NB * PWAVES) {
            if (!first || t != t0) load(t);
#pragma unroll
            for (int i = 0; i < NB; i++) {
                const int c = 16 * (t + i);
                if (t + i >= t1) break;
#pragma unroll
                for (int q = 0; q < RW; q++) {
                    v4f d = zero;
#pragma unroll
                    for (int s = 0; s < RS; s++) d = hp[q][s].left_of(bv[i][s], d);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (row_in(q, e) && c + m16 < a.N) y[(16 * q + e) * a.ldy + c] = yv[i][q][e] + d[e] * down[q][e];
                }
            }
        }
        if (!ad.next(a.slots, slot)) break;
        ad.rows &= ~infinite;
    }
    if (infinite == 0) return;                             // workgroup-uniform
    // those rows element by element, by all waves
    Adapters<PROWS> all(a, row0, Adapters<PROWS>::fetch(a, row0));
    while (all.next(a.slots, slot))
        for (uint32_t left = all.rows & infinite; left; left &= left - 1) {
            const int t = __builtin_ctz(left);
            for (int n = 16 * part * per + tid; n < ti_min(a.N, 16 * (part + 1) * per); n += 64 * PWAVES) {
                const uint16_t* b = a.b + ((size_t)all.id * a.N + n) * a.r;
                float d = 0.0f;
                for (int k = 0; k < a.r; k++) d = fmaf(one<BF16>(b[k]), s_h[t][k], d);
                a.y[(row0 + t) * a.ldy + n] += d;
            }
        }
}

template <bool BF16, bool VEC>
void launch_prompt(ti_ctx* c, const LoraArgs& a, unsigned down, unsigned up) {
    if (a.r <= 16) k_lora_down<BF16, 1><<<down, 64 * DWAVES, 0, c->stream>>>(a);
    else if (a.r <= 32) k_lora_down<BF16, 2><<<down, 64 * DWAVES, 0, c->stream>>>(a);
    else if (a.r <= 64) k_lora_down<BF16, 4><<<down, 64 * DWAVES, 0, c->stream>>>(a);
    else k_lora_down<BF16, 8><<<down, 64 * DWAVES, 0, c->stream>>>(a);
    if (a.r <= 32) k_lora_up<BF16, VEC, 1><<<up, 64 * PWAVES, 0, c->stream>>>(a);
    else if (a.r <= 64) k_lora_up<BF16, VEC, 2><<<up, 64 * PWAVES, 0, c->stream>>>(a);
    else k_lora_up<BF16, VEC, 4><<<up, 64 * PWAVES, 0, c->stream>>>(a);
}

int lanes_of(int r) { return r <= 8 ? 1 : r <= 16 ? 2 : r <= 32 ? 4 : r <= 64 ? 8 : 16; }

template <bool BF16, bool VEC>
void launch_few(ti_ctx* c, const LoraArgs& a, unsigned grid) {
    const int L = lanes_of(a.r);
    if (L == 1) k_lora_few<BF16, 1, VEC><<<grid, 64 * FWAVES, 0, c->stream>>>(a);
    else if (L == 2) k_lora_few<BF16, 2, VEC><<<grid, 64 * FWAVES, 0, c->stream>>>(a);
    else if (L == 4) k_lora_few<BF16, 4, VEC><<<grid, 64 * FWAVES, 0, c->stream>>>(a);
    else if (L == 8) k_lora_few<BF16, 8, VEC><<<grid, 64 * FWAVES, 0, c->stream>>>(a);
    else k_lora_few<BF16, 16, VEC><<<grid, 64 * FWAVES, 0, c->stream>>>(a);
}

// Few rows: their number times the rank. Rows of one request each / all of one request, 2048 x 2048 and rank 16: 512 rows in 11.3 / 11.2 us (as a
// prompt 41.9 / 10.1), 1000 in 19.1 / 20.8 (48.2 / 12.3); 2048 x 4096 and rank 64: 128 in 14.8 / 15.3 (52.2 / 11.9), 256 in 21.1 / 22.9 (57.8 / 12.4)
constexpr long FEW = 8192;

}  // namespace

extern "C" int ti_lora_add(ti_ctx* c, const float* x, const int32_t* idx, const uint16_t* a, const uint16_t* b, const float* scale, float* y,
                           int T, int K, int N, int r, int n, int ldx, int ldy, int bf16) {
    TI_CHECK_CTX(c);
    TI_REQUIRE(x && idx && a && b && scale && y, "ti_lora_add: null buffer");
    TI_REQUIRE(T > 0 && K > 0 && K % 32 == 0 && N > 0 && n > 0, "ti_lora_add: bad shape (T=%d K=%d N=%d n=%d), K a multiple of 32", T, K, N, n);
    TI_REQUIRE(r > 0 && r <= RANK_MAX, "ti_lora_add: rank %d, at most %d", r, RANK_MAX);
    TI_REQUIRE(bf16 == 0 || bf16 == 1, "ti_lora_add: bf16 is 0 or 1 (%d)", bf16);
    LoraArgs g = {x, idx, a, b, scale, y, nullptr, ldx ? ldx : K, ldy ? ldy : N, T, K, N, r, n, 1, 1, 1, (r + 15) / 16 * 16};
    TI_REQUIRE(g.ldx >= K && g.ldx % 4 == 0 && g.ldy >= N, "ti_lora_add: rows of %ld and %ld floats, of K = %d and N = %d; x's in multiples of 4", g.ldx, g.ldy, K, N);
    TI_REQUIRE(ti_al16(x) && ti_al16(a) && ti_al16(b), "ti_lora_add: x, a and b must be 16-byte aligned");
    TI_REQUIRE((long)T <= ROWS_MAX, "ti_lora_add: %d rows in one call", T);
    TI_REQUIRE(K <= DIM_MAX && N <= DIM_MAX, "ti_lora_add: K = %d, N = %d, at most %d", K, N, DIM_MAX);
    const uintptr_t x0 = (uintptr_t)x, y0 = (uintptr_t)y, x1 = x0 + 4 * ((T - 1) * (size_t)g.ldx + K), y1 = y0 + 4 * ((T - 1) * (size_t)g.ldy + N);
    TI_REQUIRE(x1 <= y0 || y1 <= x0, "ti_lora_add: x and y overlap");
    if ((long)T * r > FEW) {
        // K and N in parts until two workgroups a CU are there. A tile's adapters are dealt out to as many workgroups as make four a CU, since how
        // many it has is known on the device alone; those dealt none end behind three stages' loads of x (1500 rows of four
        // requests: about 200 of 940 have one)
        const long tiles = (T + PROWS - 1) / PROWS, want = ti_max(1L, 2L * c->cus / tiles);
        g.h = c->attn_po;
        g.splits = (int)ti_max(1L, ti_min(ti_min(want, (long)K / (4 * KC)), ti_min((long)SPLITS, SCRATCH / ((long)T * g.rp))));
        g.parts = (int)ti_max(1L, ti_min(want, ((long)N + 32 * PWAVES - 1) / (32 * PWAVES)));
        g.slots = (int)ti_min(16L, ti_max(2L, 4L * c->cus / (tiles * g.splits)));
        const unsigned down = (unsigned)(tiles * g.splits * g.slots), up = (unsigned)(tiles * g.parts * g.slots);
        if (bf16) r % 8 == 0 ? launch_prompt<true, true>(c, g, down, up) : launch_prompt<true, false>(c, g, down, up);
        else r % 8 == 0 ? launch_prompt<false, true>(c, g, down, up) : launch_prompt<false, false>(c, g, down, up);
        TI_LAUNCHED("k_lora_down");
        return TI_OK;
    }
    // a tile's adapters apart, then N in parts of at least one load a wave, as long as every workgroup has a CU of its own
    const long tiles = (T + FROWS - 1) / FROWS, cols = FWAVES * 64 / lanes_of(r);
    g.slots = ti_min(FROWS, ti_min(T, n));
    g.parts = (int)ti_max(1L, ti_min((N + cols - 1) / cols, c->cus / (tiles * g.slots)));
    const unsigned grid = (unsigned)(tiles * g.slots * g.parts);
    if (bf16) r % 8 == 0 ? launch_few<true, true>(c, g, grid) : launch_few<true, false>(c, g, grid);
    else r % 8 == 0 ? launch_few<false, true>(c, g, grid) : launch_few<false, false>(c, g, grid);
    TI_LAUNCHED("k_lora_few");
    return TI_OK;
}
