// k_lora.hip — low-rank adapters of many requests beside a shared projection: y[t] += s_a B_a (A_a x[t]), a = idx[t]. The reference has no
// counterpart (its projections: models/qwen3.js:1588-1608).
//
// Both products on the matrix cores, weights exact, f32 activations as two f16 (f16 weights: each row scaled by a power of two, an
// element off by 2^-22 of itself or 2^-39 of the largest) or three bf16 (bf16 weights: exactly), sums in f32. Rows meet adapters in
// tiles of 16 rows: a tile's distinct adapters are taken one behind the other, each multiplies all 16 columns, and a column is
// kept where the adapter is its row's. A prompt's tile has one adapter, or two at a border; a batch's up to 16, which are dealt out to
// workgroups of their own. k_lora_down leaves h = A x in parts of K in the context's scratch, k_lora_up adds them up.
#include "ti_dev.h"
#include "ti_span.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_u __attribute__((ext_vector_type(4), aligned(4)));   // y's rows start anywhere

constexpr int RANK_MAX = 128, CS = 4;        // CS: 32-steps of K a wave takes at once
constexpr int SPLITS_MAX = 32;
constexpr int H_WORDS = TI_ATTN_ROWSPLITS * TI_ATTN_HD_MAX;            // the scratch

struct LoraArgs {
    const float* x;
    const int32_t* idx;
    const uint16_t *a, *b;
    const float* scale;
    float* y;
    float* h;                                // [splits][T][rp]
    long ldx, ldy;
    int T, K, N, r, n, rp, splits, slots, parts;   // rp: r in whole tiles of 16; slots: workgroups that a tile's adapters are dealt to
};

// 8 f32 of a row as MFMA operands of the weights' type: f16, scaled by `up`, as hi + lo; bf16, as three
template <bool BF16> struct Pieces;
template <> struct Pieces<false> {
    static constexpr int NP = 2;
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
    __device__ __forceinline__ v4f times(uint4 w, v4f acc) const {
        const ti_h8 a = __builtin_bit_cast(ti_h8, w);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p[1], acc, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p[0], acc, 0, 0, 0);
    }
};
template <> struct Pieces<true> {
    static constexpr int NP = 3;
    ti_b8 p[3];
    __device__ __forceinline__ void set(const float (&v)[8], float) { ti_bf16x3(v, p); }
    __device__ __forceinline__ v4f times(uint4 w, v4f acc) const {
        const ti_b8 a = __builtin_bit_cast(ti_b8, w);
#pragma unroll
        for (int i = 2; i >= 0; i--) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p[i], acc, 0, 0, 0);
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

// A tile's distinct adapters, one behind the other: `own` is the adapter of the tile's row `lane` (16 rows), -1 none
struct Adapters {
    uint64_t todo;
    int own, at, id;
    uint32_t rows;                           // of adapter `id`
    __device__ Adapters(const LoraArgs& a, int row0) {
        const int lane = threadIdx.x & 63, t = row0 + lane;
        own = lane < 16 && t < a.T ? a.idx[t] : -1;
        if (own >= a.n) own = -1;
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

// A workgroup: 16 rows, a part of K, its slot's adapters. A wave every fourth chunk of 128 of the part; the waves' sums meet in LDS
template <bool BF16, int RT>
__global__ __launch_bounds__(256) void k_lora_down(LoraArgs a) {
    __shared__ v4f s_acc[3][RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m16 = lane & 15, j = lane >> 4;
    const int split = blockIdx.x % a.splits, slot = blockIdx.x / a.splits % a.slots, row0 = 16 * (blockIdx.x / (a.splits * a.slots));
    const int steps = a.K / 32, per = (steps + a.splits - 1) / a.splits, s0 = split * per, s1 = ti_min(steps, s0 + per);
    const float* x = a.x + ti_min(row0 + m16, a.T - 1) * a.ldx + 8 * j;
    Adapters ad(a, row0);
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    while (ad.next(a.slots, slot)) {
        const uint16_t* w = a.a + (size_t)ad.id * a.r * a.K + 8 * j;
        v4f acc[RT];
#pragma unroll
        for (int k = 0; k < RT; k++) acc[k] = zero;
        for (int s = s0 + wave * CS; s < s1; s += 4 * CS) {
            float v[CS][8];
            uint4 wv[CS][RT];
            float mx = 0.0f;
#pragma unroll
            for (int i = 0; i < CS; i++) {
                const int at = 32 * ti_min(s + i, s1 - 1);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const v4f q = *reinterpret_cast<const v4f*>(x + at + 4 * u);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[i][4 * u + e] = q[e];
                }
#pragma unroll
                for (int k = 0; k < RT; k++)
                    wv[i][k] = *reinterpret_cast<const uint4*>(w + (size_t)ti_min(16 * k + m16, a.r - 1) * a.K + at);
            }
#pragma unroll
            for (int i = 0; i < CS; i++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    v[i][e] = s + i < s1 ? v[i][e] : 0.0f;
                    mx = fmaxf(mx, fabsf(v[i][e]));
                }
            const int ex = row_exponent<BF16>(mx);
            const float up = ldexpf(1.0f, ex), down = ldexpf(1.0f, -ex);
            v4f d[RT];
#pragma unroll
            for (int k = 0; k < RT; k++) d[k] = BF16 ? acc[k] : zero;
#pragma unroll
            for (int i = 0; i < CS; i++) {
                Pieces<BF16> p;
                p.set(v[i], up);
#pragma unroll
                for (int k = 0; k < RT; k++) d[k] = p.times(wv[i][k], d[k]);
            }
#pragma unroll
            for (int k = 0; k < RT; k++) {
                if constexpr (BF16) acc[k] = d[k];
                else
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[k][e] = fmaf(d[k][e], down, acc[k][e]);
            }
        }
        __syncthreads();                                   // the last adapter's sums are read
        if (wave > 0) {
#pragma unroll
            for (int k = 0; k < RT; k++) s_acc[wave - 1][k][lane] = acc[k];
        }
        __syncthreads();
        if (wave == 0 && ad.rows >> m16 & 1) {
            float* h = a.h + ((size_t)split * a.T + row0 + m16) * a.rp + 4 * j;
#pragma unroll
            for (int k = 0; k < RT; k++) {
                if (16 * k < a.rp) *reinterpret_cast<v4f*>(h + 16 * k) = (acc[k] + s_acc[0][k][lane]) + (s_acc[1][k][lane] + s_acc[2][k][lane]);
            }
        }
    }
}

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

// A workgroup: 16 rows, a part of N, its slot's adapters; a wave 16 columns of N at a time. The rows' h, all parts of K together and
// times the adapter's scale, are the operands of every product
template <bool BF16, bool VEC, int RS>
__global__ __launch_bounds__(256) void k_lora_up(LoraArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m16 = lane & 15, j = lane >> 4;
    const int part = blockIdx.x % a.parts, slot = blockIdx.x / a.parts % a.slots, row0 = 16 * (blockIdx.x / (a.parts * a.slots));
    const int tiles = (a.N + 15) / 16, per = (tiles + a.parts - 1) / a.parts, t0 = part * per, t1 = ti_min(tiles, t0 + per);
    Adapters ad(a, row0);
    if (!ad.todo) return;
    const int row = ti_min(row0 + m16, a.T - 1), mine = __shfl(ad.own, m16);
    Pieces<BF16> hp[RS];
    float down;
    {
        float v[RS][8], mx = 0.0f;
        const float* h = a.h + (size_t)row * a.rp + 8 * j;
        const float sc = a.scale[ti_max(mine, 0)];
#pragma unroll
        for (int s = 0; s < RS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) v[s][e] = 0.0f;
        for (int k = 0; k < a.splits; k++) {
#pragma unroll
            for (int s = 0; s < RS; s++) {
                const float* p = h + (size_t)k * a.T * a.rp + ti_min(32 * s, a.rp - 8 - 8 * j);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const v4f q = *reinterpret_cast<const v4f*>(p + 4 * u);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[s][4 * u + e] += q[e];
                }
            }
        }
#pragma unroll
        for (int s = 0; s < RS; s++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                v[s][e] = 32 * s + 8 * j + e < a.r ? v[s][e] * sc : 0.0f;
                mx = fmaxf(mx, fabsf(v[s][e]));
            }
        const int ex = row_exponent<BF16>(mx);
        const float up = ldexpf(1.0f, ex);
        down = ldexpf(1.0f, -ex);
#pragma unroll
        for (int s = 0; s < RS; s++) hp[s].set(v[s], up);
    }
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    while (ad.next(a.slots, slot)) {
        const uint16_t* b = a.b + (size_t)ad.id * a.N * a.r;
        const bool in = ad.rows >> m16 & 1;
        for (int t = t0 + wave; t < t1; t += 4) {
            const uint16_t* br = b + (size_t)ti_min(16 * t + m16, a.N - 1) * a.r;
            v4f d = zero;
#pragma unroll
            for (int s = 0; s < RS; s++) d = hp[s].times(b_ranks<VEC>(br, 32 * s + 8 * j, a.r), d);
            if (!in) continue;
            float* y = a.y + (row0 + m16) * a.ldy + 16 * t + 4 * j;
            if (16 * t + 16 <= a.N) {
                v4f_u q = *reinterpret_cast<const v4f_u*>(y);
#pragma unroll
                for (int e = 0; e < 4; e++) q[e] = q[e] + d[e] * down;
                *reinterpret_cast<v4f_u*>(y) = q;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if (16 * t + 4 * j + e < a.N) y[e] = y[e] + d[e] * down;
            }
        }
    }
}

template <bool BF16, bool VEC>
void launch_up(ti_ctx* c, const LoraArgs& a, unsigned grid) {
    const int rs = (a.r + 31) / 32;
    if (rs == 1) k_lora_up<BF16, VEC, 1><<<grid, 256, 0, c->stream>>>(a);
    else if (rs == 2) k_lora_up<BF16, VEC, 2><<<grid, 256, 0, c->stream>>>(a);
    else k_lora_up<BF16, VEC, 4><<<grid, 256, 0, c->stream>>>(a);
}

template <bool BF16>
int launch(ti_ctx* c, const LoraArgs& a, unsigned down, unsigned up) {
    if (a.rp == 16) k_lora_down<BF16, 1><<<down, 256, 0, c->stream>>>(a);
    else if (a.rp == 32) k_lora_down<BF16, 2><<<down, 256, 0, c->stream>>>(a);
    else if (a.rp <= 64) k_lora_down<BF16, 4><<<down, 256, 0, c->stream>>>(a);
    else k_lora_down<BF16, 8><<<down, 256, 0, c->stream>>>(a);
    TI_LAUNCHED("k_lora_down");
    if (a.r % 8 == 0) launch_up<BF16, true>(c, a, up);
    else launch_up<BF16, false>(c, a, up);
    TI_LAUNCHED("k_lora_up");
    return TI_OK;
}

}  // namespace

extern "C" int ti_lora_add(ti_ctx* c, const float* x, const int32_t* idx, const uint16_t* a, const uint16_t* b, const float* scale, float* y,
                           int T, int K, int N, int r, int n, int ldx, int ldy, int bf16) {
    TI_CHECK_CTX(c);
    TI_REQUIRE(x && idx && a && b && scale && y, "ti_lora_add: null buffer");
    TI_REQUIRE(T > 0 && K > 0 && K % 32 == 0 && N > 0 && n > 0, "ti_lora_add: bad shape (T=%d K=%d N=%d n=%d), K a multiple of 32", T, K, N, n);
    TI_REQUIRE(r > 0 && r <= RANK_MAX, "ti_lora_add: rank %d, at most %d", r, RANK_MAX);
    TI_REQUIRE(bf16 == 0 || bf16 == 1, "ti_lora_add: bf16 is 0 or 1 (%d)", bf16);
    LoraArgs g = {x, idx, a, b, scale, y, c->attn_po, ldx ? ldx : K, ldy ? ldy : N, T, K, N, r, n, (r + 15) / 16 * 16, 1, 1, 1};
    TI_REQUIRE(g.ldx >= K && g.ldx % 4 == 0 && g.ldy >= N, "ti_lora_add: rows of %ld and %ld floats, of K = %d and N = %d; x's in multiples of 4", g.ldx, g.ldy, K, N);
    TI_REQUIRE(ti_al16(x) && ti_al16(a) && ti_al16(b), "ti_lora_add: x, a and b must be 16-byte aligned");
    TI_REQUIRE((long)T * g.rp <= H_WORDS && (long)T <= 1 << 20, "ti_lora_add: %d rows of rank %d in one call", T, r);
    const uintptr_t x0 = (uintptr_t)x, y0 = (uintptr_t)y, x1 = x0 + 4 * ((T - 1) * (size_t)g.ldx + K), y1 = y0 + 4 * ((T - 1) * (size_t)g.ldy + N);
    TI_REQUIRE(x1 <= y0 || y1 <= x0, "ti_lora_add: x and y overlap");
    const long tiles = (T + 15) / 16;
    // a tile's adapters apart where there are few tiles; K and N in parts until four workgroups a CU are there
    g.slots = (int)ti_min((long)ti_min(16, T), ti_max(1L, c->cus / tiles));
    const long want = ti_max(1L, (4L * c->cus + tiles - 1) / tiles);
    g.splits = (int)ti_max(1L, ti_min(ti_min(want, (long)(K / 32 + 4 * CS - 1) / (4 * CS)), ti_min((long)SPLITS_MAX, H_WORDS / ((long)T * g.rp))));
    g.parts = (int)ti_max(1L, ti_min(want, ((long)N + 63) / 64));
    const unsigned down = (unsigned)(tiles * g.slots * g.splits), up = (unsigned)(tiles * g.slots * g.parts);
    return bf16 ? launch<true>(c, g, down, up) : launch<false>(c, g, down, up);
}
