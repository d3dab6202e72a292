// k_window_attn.hip — causal attention of a prompt's tokens over the int8 KV cache under a sliding window with sinks,
// both products on the matrix cores at f32 accuracy; and the columns' sums of its weights.
//
// Workgroup (4 waves): one KV head, 64 RW query rows (row = token x query head of the KV head), 16 RW a wave, and the keys
// that any of them sees, or a range of these. Blocks of 64 keys, at multiples of 64, are staged in LDS as MFMA operands
// (K codes f16, V codes bf16, exact), the next block's loads in flight meanwhile; a wave passes over the 32 keys that none of its
// rows sees and masks only where an edge of the window cuts them.
//   - S^T = K Q^T (v_mfma_f32_16x16x32_f16 per 32-dim group, q half and 16 keys; the row scaled by a power of two, q =
//     hi + lo to 2^-22 of each element or 2^-28 of the row's largest, see k_token_attn.hip), each group's sum times its key's
//     scale in f32.
//   - O^T = V^T P^T with P times the V scale of (key, group) in f32 as three bf16, exactly; a lane's scores are the
//     operand as they stand.
// Bound by VALU work, most of it the weights': 4096 tokens of 16 heads of 128 dims under a window of 1024 in 137 us (220
// TFLOP/s), VALU instructions issuing 59% of the SIMDs' cycles, the matrix cores busy 26%. A weight is multiplied and split once for
// each 32-dim group, four times at 128 dims, since every group has a V scale of its own. 32 rows a wave at 128 dims take all 256 registers
// and spill 13 (two of them read again a block, the others around the loops). Chunks are split into
// ranges of keys until two workgroups a CU are there: 250 tokens of 32 heads of 64 dims under a window of 2000 in 29 + 5 us.
#include "ti_dev.h"
#include "ti_span.h"
#include "ti_window_attn.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_u __attribute__((ext_vector_type(4), aligned(4)));   // the caller's q and out need not be aligned

constexpr int KB = 64;                       // keys of a staged block
constexpr int VSTRIDE = 65;                  // 16-byte pieces of a V operand tile (1 of padding: writes of eight tiles would meet in one bank)
constexpr float FLOOR = -3.402823466e38f;    // below it only rows that see nothing: scores of -inf give NaN as the formula does
constexpr float VSCALE = 0x1p-24f;           // of every V scale: 127 x a V scale x thousands of keys stays in f32's range

struct WinArgs {
    TiWindowAttn p;
    float* po;                               // [row][nsplit][HD] partials, (m, l) of each; nsplit = 1: none
    float* pml;
    int G, nblk, nsplit;
    TiMassRows mr;
};

// The query row of this lane, its dims 32 g + 8 j..; as MFMA operands, and the factor that scales its scores to log2 units
template <int HD>
__device__ __forceinline__ void query_load(const float* q, v4f_u (&qv)[HD / 32][2]) {
#pragma unroll
    for (int g = 0; g < HD / 32; g++)
#pragma unroll
        for (int u = 0; u < 2; u++) qv[g][u] = *reinterpret_cast<const v4f_u*>(q + 32 * g + 4 * u);
}
template <int HD>
__device__ __forceinline__ float query_operand(const v4f_u (&qv)[HD / 32][2], ti_h8 (&qh)[HD / 32], ti_h8 (&ql)[HD / 32]) {
    constexpr int NG = HD / 32;
    float mx = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(qv[g][e / 4][e % 4]));
    mx = fmaxf(mx, ti_xor(mx, 16));
    mx = fmaxf(mx, ti_xor(mx, 32));
    int ex = 4;
    if (mx > 0.0f && mx < INFINITY) (void)frexpf(mx, &ex);
    const int k = ti_min(4 - ex, 100);
    const float up = ldexpf(1.0f, k);
#pragma unroll
    for (int g = 0; g < NG; g++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float v = qv[g][e / 4][e % 4] * up;
            const _Float16 hi = (_Float16)v;
            qh[g][e] = hi;
            ql[g][e] = (_Float16)(v - (float)hi);
        }
    return 1.44269504088896341f / (127.0f * sqrtf((float)HD)) * ldexpf(1.0f, -k);
}

// what became of row gr of KV head hk, for the columns' sums
__device__ __forceinline__ void mass_row(const WinArgs& a, int hk, int gr, float m, float l) {
    float* rec = reinterpret_cast<float*>(a.mr.row + (size_t)hk * a.mr.tiles * 16 + gr);
    rec[1] = m;
    rec[2] = 1.0f / l;
}

// 4 x 4 bytes: in, w[r] = row r's four bytes; out, w[e] = byte e of rows 0..3
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

template <int HD>
struct WinLds {
    ti_h8 k[KB / 16][HD / 32][64];           // [16 keys][group][lane]: key lane % 16, dims 8 (lane / 16)..
    ti_b8 v[KB / 32][HD / 16][VSTRIDE];      // [32 keys][16 dims][lane]: dim lane % 16, keys 4 j.., 16 + 4 j..
    float ks[HD / 32][KB], vs[HD / 32][KB];
};

template <int HD, int RW>
__global__ __launch_bounds__(256, RW == 2 ? 2 : 3) void k_window_attn(WinArgs a) {
    constexpr int NG = HD / 32, PC = HD / 16;
    constexpr int KL = (KB * PC + 255) / 256, VL = (KB * HD / 16 + 255) / 256, SL = (KB * NG + 255) / 256;
    __shared__ WinLds<HD> L;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m16 = lane & 15, j = lane >> 4;
    const int hk = blockIdx.x % a.p.nKv, blk = (blockIdx.x / a.p.nKv) % a.nblk, split = blockIdx.x / (a.p.nKv * a.nblk);
    const int nrows = a.G * a.p.T, window = a.p.window, sinks = a.p.sinks, pos0 = a.p.pos0;
    const int wg0 = blk * 64 * RW, wg1 = ti_min(wg0 + 64 * RW, nrows) - 1;
    auto low_of = [&](int pos) { return window < 0 || window > pos ? 0 : pos + 1 - window; };

    // the blocks that hold keys which some row of the workgroup sees, this range's part of them
    const TiSpan sp = ti_span(pos0 + wg0 / a.G, window, sinks);
    const int end = pos0 + wg1 / a.G + 1;
    const int sb = (sp.first + KB - 1) / KB, skip = ti_max(sb, sp.low / KB) - sb;
    const int nb = ti_max(0, (int)(((long)end + KB - 1) / KB) - skip);
    const int per = (nb + a.nsplit - 1) / a.nsplit;
    const int c0 = split * per, c1 = ti_min(nb, c0 + per);
    auto block_key = [&](int i) { return (i < sb ? i : i + skip) * KB; };

    // a thread's loads of a block: K, 16 codes of a key; V, 4 dims of 4 keys; scales. Bytes from the block's first row on
    uint4 kr[KL];
    uint32_t vr[VL][4];
    float ksr[SL], vsr[SL];
    const uint32_t code_row = (uint32_t)a.p.nKv * HD, scale_row = (uint32_t)a.p.nKv * NG;
    auto k_at = [&](int u) { const int x = ti_min(tid + 256 * u, KB * PC - 1); return make_int2((x >> 4) / PC * 16 + (x & 15), 16 * ((x >> 4) % PC)); };
    auto v_at = [&](int u) { const int x = ti_min(tid + 256 * u, KB * HD / 16 - 1); return make_int2(4 * (x / (HD / 4)), 4 * (x % (HD / 4))); };
    auto s_at = [&](int u) { const int x = ti_min(tid + 256 * u, KB * NG - 1); return make_int2(x / NG, x % NG); };
    uint32_t ko[KL], vo[VL], so[SL];
#pragma unroll
    for (int u = 0; u < KL; u++) ko[u] = k_at(u).x * code_row + k_at(u).y;
#pragma unroll
    for (int u = 0; u < VL; u++) vo[u] = v_at(u).x * code_row + v_at(u).y;
#pragma unroll
    for (int u = 0; u < SL; u++) so[u] = s_at(u).x * scale_row + s_at(u).y;
    auto load = [&](int k0) {
        const size_t row = (size_t)k0 * a.p.nKv + hk;
        const uint8_t *kb = a.p.kq + row * HD, *vb = a.p.vq + row * HD;
        const float *ksb = a.p.ks + row * NG, *vsb = a.p.vs + row * NG;
        if (k0 + KB <= end) {
#pragma unroll
            for (int u = 0; u < KL; u++) kr[u] = *reinterpret_cast<const uint4*>(kb + ko[u]);
#pragma unroll
            for (int u = 0; u < VL; u++)
#pragma unroll
                for (int r = 0; r < 4; r++) vr[u][r] = *reinterpret_cast<const uint32_t*>(vb + (size_t)r * code_row + vo[u]);
#pragma unroll
            for (int u = 0; u < SL; u++) {
                ksr[u] = ksb[so[u]];
                vsr[u] = vsb[so[u]];
            }
            return;
        }
        const int top = end - 1 - k0;                      // the last row there is
#pragma unroll
        for (int u = 0; u < KL; u++) kr[u] = *reinterpret_cast<const uint4*>(kb + ti_min(k_at(u).x, top) * code_row + k_at(u).y);
#pragma unroll
        for (int u = 0; u < VL; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) vr[u][r] = *reinterpret_cast<const uint32_t*>(vb + ti_min(v_at(u).x + r, top) * code_row + v_at(u).y);
#pragma unroll
        for (int u = 0; u < SL; u++) {
            const uint32_t o = ti_min(s_at(u).x, top) * scale_row + s_at(u).y;
            ksr[u] = ksb[o];
            vsr[u] = vsb[o];
        }
    };
    auto stage = [&]() {
#pragma unroll
        for (int u = 0; u < KL; u++) {
            const int x = tid + 256 * u, t = (x >> 4) / PC, c = (x >> 4) % PC, m = x & 15;
            if (KB * PC % 256 == 0 || x < KB * PC) {
                L.k[t][c >> 1][(c & 1) * 32 + m] = ti_i8x8_h8(kr[u].x, kr[u].y);
                L.k[t][c >> 1][(c & 1) * 32 + 16 + m] = ti_i8x8_h8(kr[u].z, kr[u].w);
            }
        }
#pragma unroll
        for (int u = 0; u < VL; u++) {
            const int x = tid + 256 * u, db = x % (HD / 4), kb = x / (HD / 4), kk = kb & 7;
            if (KB * HD / 16 % 256 == 0 || x < KB * HD / 16) {
                transpose4(vr[u]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    ti_b8* p = &L.v[kb >> 3][db >> 2][(kk & 3) * 16 + 4 * (db & 3) + e];
                    reinterpret_cast<uint2*>(p)[kk >> 2] = ti_i8x4_b4(vr[u][e]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < SL; u++) {
            const int x = tid + 256 * u;
            if (KB * NG % 256 == 0 || x < KB * NG) {
                L.ks[x % NG][x / NG] = ksr[u];
                L.vs[x % NG][x / NG] = vsr[u] * VSCALE;
            }
        }
    };
    // 32 rows a wave leave no registers for a block ahead: their two workgroups a CU load and compute in turn
    constexpr bool AHEAD = RW == 1;
    constexpr int HN = RW == 1 ? 2 : 1;                    // 32-key parts whose scores are formed together
    if (AHEAD && c0 < c1) load(block_key(c0));

    // this lane's rows (past the last: that one again), and what all rows of the wave and any of them see
    const int row0 = wg0 + wave * 16 * RW;
    int pos[RW], low[RW];
    size_t orow[RW];
    ti_h8 qh[RW][NG], ql[RW][NG];
    float fr[RW];
#pragma unroll
    for (int r = 0; r < RW; r++) {
        const int gr = ti_min(row0 + 16 * r + m16, nrows - 1), t = gr / a.G;
        pos[r] = pos0 + t;
        low[r] = low_of(pos[r]);
        orow[r] = (size_t)t * a.p.nHq + hk * a.G + gr % a.G;
        v4f_u qv[NG][2];
        query_load<HD>(a.p.qr + orow[r] * HD + 8 * j, qv);
        fr[r] = query_operand<HD>(qv, qh[r], ql[r]);
        if (RW == 1 && a.mr.op && split == 0 && row0 < 16 * a.mr.tiles) {
            const size_t u = (size_t)hk * a.mr.tiles + row0 / 16;
            ti_h8* op = a.mr.op + u * 2 * NG * 64 + lane;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                op[g * 64] = qh[r][g];
                op[(NG + g) * 64] = ql[r][g];
            }
            const bool in = row0 + m16 < nrows;
            float* rec = reinterpret_cast<float*>(a.mr.row + u * 16 + m16);
            if (j == 0) {
                rec[0] = in ? fr[r] : 0.0f;
                rec[3] = __builtin_bit_cast(float, in ? pos[r] : -1);
                if (!in) rec[1] = rec[2] = 0.0f;           // the others': at the end, or in the merge
            }
        }
    }
    const int first_pos = pos0 + ti_min(row0, nrows - 1) / a.G, last_pos = pos0 + ti_min(row0 + 16 * RW - 1, nrows - 1) / a.G;
    const int any_low = low_of(first_pos), all_low = low_of(last_pos);

    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    v4f o[RW][HD / 16];
    float mx[RW], l[RW];
#pragma unroll
    for (int r = 0; r < RW; r++) {
        mx[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) o[r][d] = zero;
    }
    for (int i = c0; i < c1; i++) {
        const int t0 = block_key(i);
        if (!AHEAD) load(t0);
        __syncthreads();                                   // the last block is read
        stage();
        __syncthreads();
        if (AHEAD && i + 1 < c1) load(block_key(i + 1));
        TI_ISSUE_FENCE();
#pragma unroll 1
        for (int h = 0; h < KB / 32; h += HN) {            // 32 HN keys
            const int k0 = t0 + 32 * h, kn = k0 + 32 * HN;
            // wave-uniform: no row of the wave sees any of them
            if (row0 >= nrows || k0 > last_pos || (kn <= any_low && k0 >= sinks)) continue;
            const bool whole = kn - 1 <= first_pos && (k0 >= all_low || kn <= sinks);
            float s[RW][8 * HN];
#pragma unroll
            for (int b = 0; b < 2 * HN; b++) {
                v4f acc[RW];
#pragma unroll
                for (int r = 0; r < RW; r++) acc[r] = zero;
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const ti_h8 kk = L.k[2 * h + b][g][lane];
                    const v4f sc = *reinterpret_cast<const v4f*>(&L.ks[g][32 * h + 16 * b + 4 * j]);
#pragma unroll
                    for (int r = 0; r < RW; r++) {
                        v4f d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qh[r][g], zero, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, ql[r][g], d, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[r][e] = fmaf(d[e], sc[e], acc[r][e]);
                    }
                }
#pragma unroll
                for (int r = 0; r < RW; r++)
#pragma unroll
                    for (int e = 0; e < 4; e++) s[r][4 * b + e] = acc[r][e];
            }
            // the largest of the lane's scores of each row, in log2; what a row sees is never below the floor
            uint32_t seen[RW];
            float tm[RW];
            bool bump = false;
#pragma unroll
            for (int r = 0; r < RW; r++) {
                if (!whole) {
                    asm volatile("");                      // a branch: not computed where every key is seen
                    seen[r] = 0;
                    tm[r] = -INFINITY;
#pragma unroll
                    for (int e = 0; e < 8 * HN; e++) {
                        const int key = k0 + 16 * (e >> 2) + 4 * j + (e & 3);
                        const bool ok = (key <= pos[r]) & ((key >= low[r]) | (key < sinks));
                        seen[r] |= ok ? 1u << e : 0u;
                        tm[r] = fmaxf(tm[r], ok ? fmaxf(s[r][e], FLOOR) : -INFINITY);
                    }
                    tm[r] = tm[r] > -INFINITY ? fmaxf(tm[r] * fr[r], FLOOR) : -INFINITY;
                } else {
                    seen[r] = ~0u;
                    tm[r] = FLOOR;
#pragma unroll
                    for (int e = 0; e < 8 * HN; e++) tm[r] = fmaxf(tm[r], s[r][e]);
                    tm[r] = fmaxf(tm[r] * fr[r], FLOOR);
                }
                bump |= tm[r] > mx[r] + 6.0f;
            }
            // the reference maximum moves when it is exceeded by more than 2^6 (weights up to 64): o is rescaled rarely
            if (__any(bump)) {
#pragma unroll
                for (int r = 0; r < RW; r++) {
                    tm[r] = fmaxf(tm[r], ti_xor(tm[r], 16));
                    tm[r] = fmaxf(tm[r], ti_xor(tm[r], 32));
                    const bool up = tm[r] > mx[r] + 6.0f;
                    const float mn = up ? tm[r] : mx[r];
                    const float alpha = up ? __builtin_amdgcn_exp2f(mx[r] - mn) : 1.0f;
                    l[r] = l[r] * alpha;
#pragma unroll
                    for (int d = 0; d < HD / 16; d++) o[r][d] = o[r][d] * alpha;
                    mx[r] = mn;
                }
            }
#pragma unroll
            for (int r = 0; r < RW; r++) {
#pragma unroll
                for (int e = 0; e < 8 * HN; e++) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[r][e], fr[r], -mx[r]));
                    s[r][e] = whole || (seen[r] >> e & 1u) ? p : 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 8 * HN; e += 8)
                    l[r] += ((s[r][e] + s[r][e + 1]) + (s[r][e + 2] + s[r][e + 3])) + ((s[r][e + 4] + s[r][e + 5]) + (s[r][e + 6] + s[r][e + 7]));
            }
#pragma unroll
            for (int x = 0; x < HN * NG; x++) {
                const int hh = x / NG, g = x % NG;
                const v4f v0 = *reinterpret_cast<const v4f*>(&L.vs[g][32 * (h + hh) + 4 * j]);
                const v4f v1 = *reinterpret_cast<const v4f*>(&L.vs[g][32 * (h + hh) + 16 + 4 * j]);
                ti_b8 p[RW][3];
#pragma unroll
                for (int r = 0; r < RW; r++) {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        w[e] = s[r][8 * hh + e] * v0[e];
                        w[4 + e] = s[r][8 * hh + 4 + e] * v1[e];
                    }
                    if (!whole) {                          // the scale of a key that the row does not see may be NaN
#pragma unroll
                        for (int e = 0; e < 8; e++) w[e] = seen[r] >> (8 * hh + e) & 1u ? w[e] : 0.0f;
                    }
                    ti_bf16x3(w, p[r]);
                }
#pragma unroll
                for (int d = 2 * g; d < 2 * g + 2; d++) {
                    const ti_b8 vv = L.v[h + hh][d][lane];
#pragma unroll
                    for (int r = 0; r < RW; r++)
#pragma unroll
                        for (int e = 2; e >= 0; e--) o[r][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, p[r][e], o[r][d], 0, 0, 0);
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < RW; r++) {
        float lt = l[r] + ti_xor(l[r], 16);
        lt += ti_xor(lt, 32);
        if (row0 + 16 * r + m16 >= nrows) continue;
        const bool direct = a.nsplit == 1;
        const float inv = 1.0f / (127.0f * VSCALE * lt);
        const float f = !direct ? 1.0f : mx[r] == -INFINITY ? 0.0f : inv;
        float* dst = direct ? a.p.out + orow[r] * HD : a.po + (orow[r] * a.nsplit + split) * HD;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) *reinterpret_cast<v4f_u*>(dst + 16 * d + 4 * j) = o[r][d] * f;
        if (j == 0 && !direct) {
            float* ml = a.pml + 2 * (orow[r] * a.nsplit + split);
            ml[0] = mx[r];
            ml[1] = lt;
        }
        if (j == 0 && direct && a.mr.op) mass_row(a, hk, row0 + 16 * r + m16, mx[r], lt);
    }
}

// A wave a row: its ranges' partials (at most 64) into the output
template <int HD>
__global__ __launch_bounds__(256) void k_window_merge(WinArgs a, int rows) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;                               // wave-uniform
    const int n = a.nsplit;
    const float* ml = a.pml + 2 * (size_t)row * n;
    const float mi = lane < n ? ml[2 * lane] : -INFINITY, li = lane < n ? ml[2 * lane + 1] : 0.0f;
    const float M = ti_wave_max(mi);
    const float wi = mi == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mi - M);
    const float Lt = ti_wave_sum(wi * li);
    const int d = lane % (HD / 2);
    const float* po = a.po + (size_t)row * n * HD + 2 * d;
    float v0 = 0.0f, v1 = 0.0f;
    for (int i0 = 0; i0 < n; i0 += 8) {
        float2 x[8];
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = *reinterpret_cast<const float2*>(po + (size_t)ti_min(i0 + k, n - 1) * HD);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float f = i0 + k < n ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wi), i0 + k)) : 0.0f;
            v0 = fmaf(x[k].x, f, v0);
            v1 = fmaf(x[k].y, f, v1);
        }
    }
    if (lane < HD / 2) {
        const float div = 127.0f * VSCALE * Lt;
        float* out = a.p.out + (size_t)row * HD + 2 * d;
        out[0] = M == -INFINITY ? 0.0f : v0 / div;
        out[1] = M == -INFINITY ? 0.0f : v1 / div;
    }
    if (a.mr.op && lane == 0) {
        const int hq = row % a.p.nHq;
        mass_row(a, hq / a.G, row / a.p.nHq * a.G + hq % a.G, M, Lt);
    }
}

// ---- column sums of the weights --------------------------------------------------------------------------
constexpr int KT = 2;                        // 16-key tiles of a workgroup
constexpr int MASS_GRID = 4096;              // key parts a grid row: a grid's side holds less than 2^32 threads

// A workgroup 16 KT keys of a KV head, in each wave the same as A operands, and each wave every fourth row tile, the next
// one's loads in flight; a lane adds up what one row in 16 gives to four keys of each 16, in a fixed order. Bound by the
// operands' way out of L2 and by each wave's start, its keys' operands and scales (256 rows of 16 heads over 2048 keys of 8:
// 11.8 us; with 3 and 4 key tiles, too few workgroups, 14.7 and 17.0)
template <int HD>
__global__ __launch_bounds__(256, 2) void k_mass_columns(WinArgs a, float* __restrict__ mass) {
    constexpr int NG = HD / 32;
    __shared__ float s_sum[4][16 * KT];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m16 = lane & 15, j = lane >> 4;
    const int hk = blockIdx.x % a.p.nKv, tiles = a.mr.tiles;
    const long k0 = ((long)blockIdx.y * MASS_GRID + blockIdx.x / a.p.nKv) * 16 * KT, S = (long)a.p.pos0 + a.p.T;
    // row tiles before the one that holds the first query at or behind the first key see none of the keys
    const int start = (int)(ti_max(0L, k0 - a.p.pos0) * a.G / 16);
    const ti_h8* op = a.mr.op + (size_t)hk * tiles * 2 * NG * 64 + lane;
    const float4* rows = a.mr.row + (size_t)hk * tiles * 16 + m16;
    ti_h8 q[2 * NG], qn[2 * NG];
    float4 r, rn;
    auto load = [&](int t) {
#pragma unroll
        for (int x = 0; x < 2 * NG; x++) qn[x] = op[((size_t)t * 2 * NG + x) * 64];
        rn = rows[(size_t)t * 16];
    };
    int t = start + wave;
    if (t < tiles) load(t);
    ti_h8 kk[KT][NG];
    float sc[KT][NG][4];
#pragma unroll
    for (int b = 0; b < KT; b++) {
        const uint8_t* kr = a.p.kq + ((size_t)ti_min(k0 + 16 * b + m16, S - 1) * a.p.nKv + hk) * HD + 8 * j;
#pragma unroll
        for (int g = 0; g < NG; g++) {
            const uint2 w = *reinterpret_cast<const uint2*>(kr + 32 * g);
            kk[b][g] = ti_i8x8_h8(w.x, w.y);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float* sr = a.p.ks + ((size_t)ti_min(k0 + 16 * b + 4 * j + e, S - 1) * a.p.nKv + hk) * NG;
#pragma unroll
            for (int g = 0; g < NG; g++) sc[b][g][e] = sr[g];
        }
    }
    float sum[4 * KT] = {};
    for (; t < tiles; t += 4) {
#pragma unroll
        for (int x = 0; x < 2 * NG; x++) q[x] = qn[x];
        r = rn;
        if (t + 4 < tiles) load(t + 4);
        const long pos = __builtin_bit_cast(int, r.w);
#pragma unroll
        for (int b = 0; b < KT; b++) {
            const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
            v4f acc = zero;
#pragma unroll
            for (int g = 0; g < NG; g++) {
                v4f d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[b][g], q[g], zero, 0, 0, 0);
                d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk[b][g], q[NG + g], d, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[e] = fmaf(d[e], sc[b][g][e], acc[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float p = __builtin_amdgcn_exp2f(fmaf(acc[e], r.x, -r.y)) * r.z;
                sum[4 * b + e] += k0 + 16 * b + 4 * j + e <= pos ? p : 0.0f;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4 * KT; e++) {
        sum[e] += ti_xor(sum[e], 1);
        sum[e] += ti_xor(sum[e], 2);
        sum[e] += ti_xor(sum[e], 4);
        sum[e] += ti_xor(sum[e], 8);
        if (m16 == 0) s_sum[wave][16 * (e >> 2) + 4 * j + (e & 3)] = sum[e];
    }
    __syncthreads();
    const long key = k0 + tid;
    if (tid >= 16 * KT || key >= S) return;                // k0 too may lie behind the last key, in the last grid row
    const float all = (s_sum[0][tid] + s_sum[1][tid]) + (s_sum[2][tid] + s_sum[3][tid]);
    float* d = mass + (size_t)key * a.p.nKv + hk;
    *d = key < a.p.pos0 ? *d + all : all;
}

template <int HD>
int launch(ti_ctx* c, const TiWindowAttn& p, const TiMassRows& mr, long slots) {
    const int G = p.nHq / p.nKv, nrows = G * p.T;
    // keys that 64 rows see, at most, in blocks
    const int tokens = (63 + G) / G + 1;
    const long keys = p.window < 0 ? (long)p.pos0 + p.T : ti_min((long)p.pos0 + p.T, (long)p.window + p.sinks + tokens);
    const long kb = keys / KB + 3;
    // 32 rows a wave where that still gives every CU its workgroups (4096 tokens of 16 heads: 159 us, 16 rows 169); columns'
    // sums, of few rows, take 16
    const bool two = !mr.op && (long)p.nKv * ((nrows + 127) / 128) >= c->cus;
    const int rows = two ? 128 : 64, nblk = (nrows + rows - 1) / rows;
    const long wg = (long)p.nKv * nblk;
    long ns = (2L * c->cus + wg - 1) / wg;
    if (two) ns = 1;
    if (ns > kb / 2) ns = kb / 2;
    if (ns > 64) ns = 64;
    ns = ti_min(ns, slots / ((long)p.T * p.nHq));
    if (ns < 1) ns = 1;
    const WinArgs a = {p, c->attn_po, c->attn_ml, G, nblk, (int)ns, mr};
    const unsigned grid = (unsigned)(wg * ns);
    if (two) k_window_attn<HD, 2><<<grid, 256, 0, c->stream>>>(a);
    else k_window_attn<HD, 1><<<grid, 256, 0, c->stream>>>(a);
    TI_LAUNCHED("k_window_attn");
    if (ns > 1) {
        const int total = p.T * p.nHq;
        k_window_merge<HD><<<(unsigned)((total + 3) / 4), 256, 0, c->stream>>>(a, total);
        TI_LAUNCHED("k_window_merge");
    }
    return TI_OK;
}

// Attention that leaves the rows' operands behind, in the upper half of the partials' scratch, and the columns' sums
template <int HD>
int launch_mass(ti_ctx* c, const TiWindowAttn& p, float* mass) {
    // each row 4 HD bytes of operand and 16 of its own, padded to whole tiles a KV head
    static_assert((TI_ATTN_ROWS_MAX + 15 * TI_ATTN_HEADS_MAX) * (4L * TI_ATTN_HD_MAX + 16) <= 2L * TI_ATTN_ROWSPLITS * TI_ATTN_HD_MAX,
                  "the rows' operands fit half of the scratch");
    const int G = p.nHq / p.nKv, tiles = (G * p.T + 15) / 16;
    ti_h8* op = reinterpret_cast<ti_h8*>(c->attn_po + TI_ATTN_ROWSPLITS / 2 * (size_t)TI_ATTN_HD_MAX);
    const TiMassRows mr = {op, reinterpret_cast<float4*>(op + (size_t)p.nKv * tiles * 2 * (HD / 32) * 64), tiles};
    const int rc = launch<HD>(c, p, mr, TI_ATTN_ROWSPLITS / 2);
    if (rc) return rc;
    const WinArgs a = {p, nullptr, nullptr, G, 0, 0, mr};
    const long kb = ((long)p.pos0 + p.T + 16 * KT - 1) / (16 * KT);
    const dim3 grid((unsigned)(ti_min(kb, (long)MASS_GRID) * p.nKv), (unsigned)((kb + MASS_GRID - 1) / MASS_GRID));
    k_mass_columns<HD><<<grid, 256, 0, c->stream>>>(a, mass);
    TI_LAUNCHED("k_mass_columns");
    return TI_OK;
}

}  // namespace

int ti_window_attn_launch(ti_ctx* c, const TiWindowAttn& p, int hd) {
    const TiMassRows none = {nullptr, nullptr, 0};
    const long slots = TI_ATTN_ROWSPLITS;
    return hd == 128 ? launch<128>(c, p, none, slots) : hd == 96 ? launch<96>(c, p, none, slots)
         : hd == 64 ? launch<64>(c, p, none, slots) : launch<32>(c, p, none, slots);
}
int ti_mass_attn_launch(ti_ctx* c, const TiWindowAttn& p, int hd, float* mass) {
    return hd == 128 ? launch_mass<128>(c, p, mass) : hd == 96 ? launch_mass<96>(c, p, mass)
         : hd == 64 ? launch_mass<64>(c, p, mass) : launch_mass<32>(c, p, mass);
}
