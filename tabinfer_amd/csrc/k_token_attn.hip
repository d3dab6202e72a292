// k_token_attn.hip — attention of few query rows a KV head over a part of the int8 KV cache: a decode step under a
// sliding window with sinks, one token of each of B sequences over pages, and the scores that accumulated weights are
// made of. At most 16 rows a tile (row = token x query head of the KV head), both products on the matrix cores.
//
//  - The visible keys are cut into blocks of 32 at multiples of 32 (a page of 32 and more covers whole blocks). The
//    blocks of all sequences, one sequence's behind the other's, are dealt out in runs of `chunk` to the workgroups of a
//    KV head: each has the same work whatever the lengths, a run that ends one sequence begins the next, and its part of
//    a sequence is a partial in slot (workgroup + sequence). Every workgroup finds its run by a scan over the lengths;
//    nothing depends on them on the host.
//  - A wave takes a block at a time, on its own, loaded straight into LDS of its own; 12 waves a CU cover each other's
//    loads (16 have too few registers: 57 us for 32 ragged sequences against 49).
//    S^T = K Q^T, one v_mfma_f32_16x16x32_f16 per 32-dim group, 16 keys and q half (q = hi + lo in f16, the
//    row scaled by a power of two: an element is off by 2^-22 of itself or 2^-28 of the row's largest, which the f32 sum of
//    hd products loses anyway unless a key's scales make up for a group 2^10 below it; three bf16 would be exact for half as
//    many products again), each group's sum times its key's scale in f32. A
//    lane's scores are those of one row: they are the B operand of O^T = V^T P^T as they stand.
//    P times the V scale of (key, group) in f32, as three bf16, exactly; V through the transposing LDS read.
//  - The waves' (m, l, O) meet in LDS; the workgroups' partials in k_token_merge.
//  - Bound by the stream where the keys are many (32 ragged sequences of 8 heads of 128 dims, 211 MB: 49.6 + 4.8 us: 4.3
//    TB/s, 3.9 with the merge), else by its round trips (length, table, rows) and the second launch: 4100
//    keys 8.3 + 4.2 us, one sequence of 8191 over pages 11.6 + 4.4.
//  - A row that sees nothing has m = -inf; one that sees only scores of -inf has the finite floor, and gives NaN as the formula does.
#include "ti_dev.h"
#include "ti_span.h"
#include "ti_token_attn.h"
#include <type_traits>

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_u __attribute__((ext_vector_type(4), aligned(4)));   // the caller's q and out need not be aligned
typedef int v2i __attribute__((ext_vector_type(2)));

constexpr int BLK = 32;                      // keys of a wave's block
constexpr int WAVES = 4, THREADS = 64 * WAVES;
constexpr float FLOOR = -3.402823466e38f;
constexpr float PSCALE = 0x1p-24f;           // of every weight in P V: 127 x a V scale x thousands of keys stays in f32's range

struct TokArgs {
    TiTokenAttn p;
    float* po;                               // [slot][nKv][T G][HD] partials, (m, l) of each
    float* pml;
    int32_t* meta;                           // [B][2]: a sequence's first slot and their number
    int G, R, RT, wgs;                       // R = T G rows a KV head in RT tiles; wgs: workgroups of HW KV heads, at most
    int HW, BW;                              // a workgroup's waves: HW KV heads x BW blocks
};

// Blocks that hold the keys [0, first) and [low, end): [0, sb) and [wb, sb + ... )
struct Blocks {
    int sb, skip, n;                         // sink blocks; blocks between them and the window; all that are visited
    __device__ int at(int i) const { return i < sb ? i : i + skip; }
};
__host__ __device__ __forceinline__ Blocks blocks_of(const TiSpan& s) {
    Blocks b;
    b.sb = (s.first + BLK - 1) / BLK;
    const int w = ti_max(b.sb, s.low / BLK);
    b.skip = w - b.sb;
    b.n = ti_max(0, (int)(((long)s.end + BLK - 1) / BLK) - b.skip);
    return b;
}

template <bool PAGED>
__device__ __forceinline__ int seq_last(const TokArgs& a, int b) {      // position of the sequence's last query
    if (!PAGED) return a.p.pos0 + a.p.T - 1;
    return ti_last_pos(a.p.lens[b], (long)a.p.pg.width << a.p.pg.shift);
}
template <bool PAGED>
__device__ __forceinline__ TiSpan seq_span(const TokArgs& a, int last) {   // the keys that any of its queries sees
    TiSpan s = ti_span(last - (a.p.T - 1), a.p.window, a.p.sinks);
    s.end = last + 1;
    return s;
}
// blocks of a sequence; one (of nothing) where no key is visible, so that every sequence has a slot
template <bool PAGED>
__device__ __forceinline__ int seq_blocks(const TokArgs& a, int b) {
    const int last = seq_last<PAGED>(a, b);
    return last < 0 ? 1 : ti_max(1, blocks_of(seq_span<PAGED>(a, last)).n);
}

// sum of the threads before this one, and of all of the workgroup
__device__ __forceinline__ long wg_scan(long v, long* s4, long& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    long x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long y = __shfl_up(x, o);
        x += lane >= o ? y : 0;
    }
    if (lane == 63) s4[wave] = x;
    __syncthreads();
    long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) {
        const long t = s4[w];
        before += w < wave ? t : 0;
        all += t;
    }
    total = all;
    return before + x - v;
}

// a value that all lanes hold, in scalar registers
__device__ __forceinline__ long uniform(long v) {
    const int lo = __builtin_amdgcn_readfirstlane((int)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return (long)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}

// The run of blocks of a workgroup, in sequence b from its block `block` (at block `start` of all) on
struct Run {
    long chunk, left;                        // blocks of every workgroup's run; of this one, still to do
    long start;
    int b, block;
};
// blocks of a run: an equal share, but a block for each of the BW waves of a head where the sequences have as many
__host__ __device__ __forceinline__ long run_chunk(long total, int B, int wgs, int BW) {
    return ti_max((total + wgs - 1) / wgs, ti_min((long)BW, (total + B - 1) / B));
}
template <bool PAGED>
__device__ bool find_run(const TokArgs& a, int w, Run& r, long* s4, long* s_at, int* s_b) {
    const int B = a.p.B, tid = threadIdx.x;
    if (B == 1) {
        const long n = seq_blocks<PAGED>(a, 0);
        r.chunk = run_chunk(n, 1, a.wgs, a.BW);
        r.b = 0;
        r.start = 0;
        r.block = (int)ti_min(w * r.chunk, n);
        r.left = ti_min(r.chunk, n - r.block);
        return r.left > 0;
    }
    // a thread: the sequences [tid per, tid per + per)
    const int per = (B + THREADS - 1) / THREADS, b0 = ti_min(B, tid * per), b1 = ti_min(B, b0 + per);
    long mine = 0, total;
    for (int b = b0; b < b1; b++) mine += seq_blocks<PAGED>(a, b);
    long at = wg_scan(mine, s4, total);
    total = uniform(total);
    r.chunk = run_chunk(total, B, a.wgs, a.BW);
    const long g0 = w * r.chunk;
    if (g0 >= at && g0 < at + mine) {
        for (int b = b0; b < b1; b++) {
            const int n = seq_blocks<PAGED>(a, b);
            if (g0 < at + n) {
                *s_b = b;
                *s_at = at;
                break;
            }
            at += n;
        }
    }
    __syncthreads();
    if (g0 >= total) return false;
    r.left = ti_min(r.chunk, total - g0);
    r.b = __builtin_amdgcn_readfirstlane(*s_b);
    r.start = uniform(*s_at);
    r.block = (int)(g0 - r.start);
    return true;
}

// Query rows in a tile's 16 columns. COLS: a row has a column for each of its 32-dim groups (four for three groups), which
// scales one group's dots and weights, so that a lane splits 8 weights a block instead of 8 for every group; taken where one
// tile holds the rows so (32 ragged sequences 49.6 us, a column a row 63.6; 4096 keys 7.5 / 8.8). Else a column a row.
constexpr int tile_slots(int hd, bool cols) { return !cols || hd == 32 ? 1 : hd == 64 ? 2 : 4; }
constexpr int tile_rows(int hd, bool cols) { return 16 / tile_slots(hd, cols); }

template <int HD, bool COLS>
struct TokLds {
    static constexpr int NG = HD / 32;
    // a block as its loads write it: rows of HD bytes one behind the other, their 16-byte pieces permuted (piece_slot)
    struct Wave {
        uint8_t k[BLK * HD], v[BLK * HD];
        float ks[(NG * BLK + 63) / 64 * 64], vs[(NG * BLK + 63) / 64 * 64];       // [group][key]
    };
    union {
        Wave w[WAVES];
        float o[WAVES][tile_rows(HD, COLS)][HD];
    };
    float m[WAVES][16], l[WAVES][16];
    long s4[WAVES], at;
    int b;
};

// Where piece c of a key's row lies: both operand reads, 16 keys' piece and 8 keys' 16 bytes, without bank conflicts (rows of
// 32 and 96 bytes are so as they are)
template <int HD>
__device__ __forceinline__ int piece_slot(int key, int c) {
    return HD == 128 ? c ^ ((key >> 1) & 7) : HD == 64 ? c ^ ((key >> 2) & 3) : c;
}

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef const __attribute__((address_space(1))) void* glb_ptr;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const void* base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, 0x00020000);
}
// a lane's 16 bytes (streamed) or 4 (scales: neighbouring heads share their cache lines) to LDS, lane after lane
__device__ __forceinline__ void run_to_lds16(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t lane_off, int off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)lds, 16, lane_off, off, 0, 2);
}
__device__ __forceinline__ void run_to_lds4(__amdgpu_buffer_rsrc_t r, void* lds, uint32_t lane_off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)lds, 4, lane_off, 0, 0, 0);
}
__device__ __forceinline__ void to_lds16(const void* p, void* lds) { __builtin_amdgcn_global_load_lds((glb_ptr)p, (lds_ptr)lds, 16, 0, 2); }
__device__ __forceinline__ void to_lds4(const void* p, void* lds) { __builtin_amdgcn_global_load_lds((glb_ptr)p, (lds_ptr)lds, 4, 0, 0); }

// v of the 16 / SLOTS columns of one row, added up in each of them
template <int SLOTS>
__device__ __forceinline__ float slot_sum(float v) {
    auto ror = [](float x, auto c) {
        const int i = __builtin_bit_cast(int, x);
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, i, decltype(c)::value, 0xF, 0xF, true));
    };
    if constexpr (SLOTS >= 2) v += ror(v, std::integral_constant<int, 0x128>{});   // row_ror:8
    if constexpr (SLOTS == 4) v += ror(v, std::integral_constant<int, 0x124>{});   // row_ror:4
    return v;
}

template <int HD, bool PAGED, bool COLS>
__global__ __launch_bounds__(THREADS, COLS ? 3 : 2) void k_token_attn(TokArgs a) {
    constexpr int NG = HD / 32, PC = HD / 16, NL = HD / 32;            // 16-byte pieces a row; loads a lane a block
    constexpr int SL = (BLK * NG + 63) / 64;                           // scale loads a lane
    constexpr int SLOTS = tile_slots(HD, COLS), ROWS = tile_rows(HD, COLS);
    constexpr int NQ = COLS ? 2 : NG, NU = HD > 64 ? 2 : 1;            // Q operands; COLS: of NU x 64 dims, a column's own
    __shared__ __align__(16) TokLds<HD, COLS> L;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the waves of a workgroup read HW heads of the same positions together: rows of a position lie side by side
    const int groups = a.p.nKv / a.HW, hr = blockIdx.x % (groups * a.RT), w = blockIdx.x / (groups * a.RT);
    const int hs = wave % a.HW, bw = wave / a.HW, hk0 = hr % groups * a.HW, hk = hk0 + hs, rt = hr / groups;
    Run run;
    if (!find_run<PAGED>(a, w, run, L.s4, &L.at, &L.b)) return;        // workgroup-uniform
    const int r16 = lane & 15, j = lane >> 4;

    const int slot = r16 / ROWS, grp = ti_min(slot, NG - 1), tr = r16 % ROWS;   // this lane's column: row of the tile, group
    const int rg = ti_min(rt * ROWS + tr, a.R - 1), t = rg / a.G, h = rg % a.G;
    const v4f zero = {0.0f, 0.0f, 0.0f, 0.0f};
    // the transposing read's rows: lanes 2 rr, 2 rr + 1 of 16 address key 4 j + rr (rr < 4) or 16 + 4 j + rr - 4
    const int rr = r16 >> 1, vrow = rr < 4 ? 4 * j + rr : 12 + 4 * j + rr;
    // a lane's loads of a block: row and byte in it
    // (of 64 and 128 dims the loads p and p + PF are a fixed distance apart)
    constexpr int PF = HD == 96 ? NL : HD == 128 ? 2 : 1;
    uint32_t po[PF];
    auto l_key = [&](int p) { return (lane + 64 * p) / PC; };
    auto l_byte = [&](int p) { return 16 * piece_slot<HD>(l_key(p), (lane + 64 * p) % PC); };
    const int s_key = lane % BLK;
    auto s_grp = [&](int p) { return ti_min(2 * p + lane / BLK, NG - 1); };
#pragma unroll
    for (int p = 0; p < PF; p++) po[p] = (uint32_t)(l_key(p) * a.p.nKv) * HD + l_byte(p);
    const uint32_t so = 4 * ((uint32_t)(s_key * a.p.nKv) * NG + s_grp(0));
    const int far = 64 / PC * PF * a.p.nKv * HD;

    for (;;) {
        // ---- this workgroup's part of sequence run.b: blocks [c0, c1)
        const int last = seq_last<PAGED>(a, run.b);
        const TiSpan span = seq_span<PAGED>(a, last);
        Blocks bl = blocks_of(span);
        if (last < 0) bl.n = 0;
        const int nb = ti_max(1, bl.n);
        const int c0 = run.block, part = (int)ti_min((long)(nb - c0), run.left), c1 = ti_min(bl.n, c0 + part);
        const int pos = last - (a.p.T - 1) + t;
        const int low = a.p.window < 0 || a.p.window > pos ? 0 : pos + 1 - a.p.window;
        // what every row of the tile sees: [full_low, full_end)
        const int full_low = a.p.window < 0 || a.p.window > last ? 0 : last + 1 - a.p.window, full_end = last - (a.p.T - 1) + 1;
        // the query's loads before the keys': they come back first
        v4f_u qv[NQ][2];
        const int qc = j + 4 * (slot / 2);                     // COLS: the lane's 16 dims of the 64 that its column's group is in
        auto q_dim = [&](int x) { return COLS ? 16 * ti_min(qc, PC - 1) + 8 * x : 32 * x + 8 * j; };
        {
            const float* q = a.p.qr + ((size_t)(run.b * a.p.T + t) * a.p.nHq + hk * a.G + h) * HD;
#pragma unroll
            for (int x = 0; x < NQ; x++)
#pragma unroll
                for (int u = 0; u < 2; u++) qv[x][u] = *reinterpret_cast<const v4f_u*>(q + q_dim(x) + 4 * u);
        }

        // ---- a block's loads, straight to the wave's LDS
        // the table's entry for key k0 + lane % 32 of block i; and, once it is there, the page of that key: -1 where no row sees
        // the key or there is no such page. Apart, so that nothing waits where the entry is asked for
        auto fetch_page = [&](int i) -> int {
            if constexpr (!PAGED) return 0;
            const int k = ti_min((bl.at(i) * BLK + (lane & 31)) >> a.p.pg.shift, a.p.pg.width - 1);
            return a.p.pg.table[(size_t)run.b * a.p.pg.width + k];
        };
        auto check_page = [&](int i, int id) -> int {
            const int key = bl.at(i) * BLK + (lane & 31);
            const bool in = key < span.end && (key >= span.low || key < span.first);
            if constexpr (!PAGED) return in ? 0 : -1;
            return in && (key >> a.p.pg.shift) < a.p.pg.width && id >= 0 && id < a.p.pg.pages ? id : -1;
        };
        // rows of one page, or of the contiguous cache, follow each other: one base and the lanes' fixed offsets
        const bool runs = !PAGED || a.p.pg.shift >= 5;
        // the first row of block i
        auto base_row = [&](int i, int page) -> size_t {
            const int k0 = bl.at(i) * BLK;
            if constexpr (!PAGED) return (size_t)k0;
            // the id of any of the block's keys that is seen (the others carry -1); page 0 where there is none
            const uint64_t some = __ballot(page >= 0);
            const int id = some ? __builtin_amdgcn_readlane(page, __builtin_ctzll(some)) : 0;
            return ((size_t)(uint32_t)id << a.p.pg.shift) + (k0 & ((1 << a.p.pg.shift) - 1));
        };
        auto in_run = [&](int i) { return runs && (PAGED || bl.at(i) * BLK + BLK <= span.end); };
        auto row_of = [&](int k0, int kl, int page) -> size_t {            // a row that exists where the key does not
            if constexpr (!PAGED) return (size_t)ti_min(k0 + kl, span.end - 1);
            const int id = ti_max(__shfl(page, kl), 0);
            return ((size_t)id << a.p.pg.shift) + ((k0 + kl) & ((1 << a.p.pg.shift) - 1));
        };
        auto& W = L.w[wave];
        auto load = [&](int i, int page) {
            const int k0 = bl.at(i) * BLK;
            if (in_run(i)) {
                // scalar bases and the lanes' 32-bit offsets
                const size_t row = base_row(i, page) * a.p.nKv + hk;
                const int codes = BLK * a.p.nKv * HD, scales = BLK * a.p.nKv * NG * 4;
                const __amdgpu_buffer_rsrc_t rk = resource(a.p.kq + row * HD, codes), rv = resource(a.p.vq + row * HD, codes);
                const __amdgpu_buffer_rsrc_t rks = resource(a.p.ks + row * NG, scales), rvs = resource(a.p.vs + row * NG, scales);
#pragma unroll
                for (int p = 0; p < NL; p++) {
                    run_to_lds16(rk, &W.k[1024 * p], po[p % PF], p / PF * far);
                    run_to_lds16(rv, &W.v[1024 * p], po[p % PF], p / PF * far);
                }
#pragma unroll
                for (int p = 0; p < SL; p++) {
                    const uint32_t o = so + 4 * (s_grp(p) - s_grp(0));
                    run_to_lds4(rks, &W.ks[64 * p], o);
                    run_to_lds4(rvs, &W.vs[64 * p], o);
                }
                return;
            }
#pragma unroll
            for (int p = 0; p < NL; p++) {
                const size_t off = (row_of(k0, l_key(p), page) * a.p.nKv + hk) * HD + l_byte(p);
                to_lds16(a.p.kq + off, &W.k[1024 * p]);
                to_lds16(a.p.vq + off, &W.v[1024 * p]);
            }
#pragma unroll
            for (int p = 0; p < SL; p++) {
                const size_t off = (row_of(k0, s_key, page) * a.p.nKv + hk) * NG + s_grp(p);
                to_lds4(a.p.ks + off, &W.ks[64 * p]);
                to_lds4(a.p.vs + off, &W.vs[64 * p]);
            }
        };

        int i = c0 + bw;
        int page = -1, entry = 0;
        if (i < c1) {
            page = check_page(i, fetch_page(i));
            if (i + a.BW < c1) entry = fetch_page(i + a.BW);
            load(i, page);
        }
        TI_ISSUE_FENCE();

        // ---- Q operand: the lane's row, dims 32 g + 8 j.. (COLS: dims 16 j.. of 64, those of other groups than the column's
        // as zeros), scaled by 2^k so that the row's largest element is below 16
        ti_h8 qh[NQ], ql[NQ];
        float fr = 1.44269504088896341f / (127.0f * sqrtf((float)HD));
        {
            float mx = 0.0f;
#pragma unroll
            for (int x = 0; x < NQ; x++)
#pragma unroll
                for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(qv[x][e / 4][e % 4]));
            mx = fmaxf(mx, ti_xor(mx, 16));
            mx = fmaxf(mx, ti_xor(mx, 32));
            if (COLS && NU == 2) mx = fmaxf(mx, ti_xor(mx, 8));            // the row's other 64 dims
            int ex = 4;
            if (mx > 0.0f && mx < INFINITY) (void)frexpf(mx, &ex);
            const int k = ti_min(4 - ex, 100);
            const float up = ldexpf(1.0f, k);
            fr = fr * ldexpf(1.0f, -k);
#pragma unroll
            for (int x = 0; x < NQ; x++) {
                const bool mine = !COLS || (qc < PC && qc / 2 == slot);
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float v = mine ? qv[x][e / 4][e % 4] * up : 0.0f;
                    const _Float16 hi = (_Float16)v;
                    qh[x][e] = hi;
                    ql[x][e] = (_Float16)(v - (float)hi);
                }
            }
        }

        v4f o[HD / 16];
#pragma unroll
        for (int d = 0; d < HD / 16; d++) o[d] = zero;
        float m = -INFINITY, l = 0.0f;

        for (; i < c1; i += a.BW) {
            __builtin_amdgcn_s_waitcnt(0x0F70);                // vmcnt(0): the block is there
            ti_wave_lds_fence();
            const int k0 = bl.at(i) * BLK;
            const uint32_t there = (uint32_t)__ballot(page >= 0);

            float s[8];
#pragma unroll
            for (int b = 0; b < 2; b++) {
                v4f acc = zero;
                if constexpr (COLS) {
#pragma unroll
                    for (int u = 0; u < NU; u++) {
                        const int key = 16 * b + r16;
                        const uint4 kw = *reinterpret_cast<const uint4*>(&W.k[key * HD + 16 * piece_slot<HD>(key, ti_min(j + 4 * u, PC - 1))]);
                        const ti_h8 k0f = ti_i8x8_h8(kw.x, kw.y), k1f = ti_i8x8_h8(kw.z, kw.w);
                        v4f d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0f, qh[0], zero, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0f, ql[0], d, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1f, qh[1], d, 0, 0, 0);
                        d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1f, ql[1], d, 0, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; e++) acc[e] = u == 0 || slot / 2 == u ? d[e] : acc[e];
                    }
                    const v4f sc = *reinterpret_cast<const v4f*>(&W.ks[BLK * grp + 16 * b + 4 * j]);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[e] = slot_sum<SLOTS>(acc[e] * sc[e]);
                } else
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const int key = 16 * b + r16;
                    const uint2 kw = *reinterpret_cast<const uint2*>(&W.k[key * HD + 16 * piece_slot<HD>(key, 2 * g + j / 2) + 8 * (j & 1)]);
                    const ti_h8 kf = ti_i8x8_h8(kw.x, kw.y);
                    const v4f sc = *reinterpret_cast<const v4f*>(&W.ks[BLK * g + 16 * b + 4 * j]);
                    v4f d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qh[g], zero, 0, 0, 0);
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, ql[g], d, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[e] = fmaf(d[e], sc[e], acc[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; e++) s[4 * b + e] = acc[e];
            }
            // which of the lane's keys its row sees
            uint32_t seen = 0xffu;
            const bool whole = there == 0xffffffffu && k0 + BLK <= full_end && (k0 >= full_low || k0 + BLK <= a.p.sinks);
            if (!whole) {                                      // wave-uniform
                asm volatile("");                              // a branch: not computed where every key is seen
                seen = 0;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int kl = 16 * (e >> 2) + 4 * j + (e & 3), key = k0 + kl;
                    const bool ok = ((there >> kl) & 1u) & (key <= pos) & ((key >= low) | (key < a.p.sinks));
                    seen |= ok ? 1u << e : 0u;
                }
            }
            if (a.p.mass && slot == 0 && rt * ROWS + tr < a.R) {
                float* sp = a.p.scores + (size_t)(hk * a.G + rg) * a.p.sstride + k0 + 4 * j;
                *reinterpret_cast<v4f*>(sp) = v4f{s[0], s[1], s[2], s[3]} * fr;
                *reinterpret_cast<v4f*>(sp + 16) = v4f{s[4], s[5], s[6], s[7]} * fr;
            }
            // the largest of the lane's scores, in log2; what a row sees is never below the floor
            float tm = FLOOR;
            if (!whole) {
                tm = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; e++) tm = fmaxf(tm, seen >> e & 1u ? fmaxf(s[e], FLOOR) : -INFINITY);
                tm = tm > -INFINITY ? fmaxf(tm * fr, FLOOR) : -INFINITY;
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) tm = fmaxf(tm, s[e]);
                tm = fmaxf(tm * fr, FLOOR);
            }
            // the reference maximum moves when it is exceeded by more than 2^6 (weights up to 64): o is rescaled rarely
            if (__any(tm > m + 6.0f)) {
                tm = fmaxf(tm, ti_xor(tm, 16));
                tm = fmaxf(tm, ti_xor(tm, 32));
                const bool bump = tm > m + 6.0f;
                const float mn = bump ? tm : m;
                const float alpha = bump ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
                l = l * alpha;
#pragma unroll
                for (int d = 0; d < HD / 16; d++) o[d] = o[d] * alpha;
                m = mn;
            }
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                float p = __builtin_amdgcn_exp2f(fmaf(s[e], fr, -m));
                if (!whole) p = seen >> e & 1u ? p : 0.0f;
                sum += p;
                s[e] = p * PSCALE;
            }
            l += sum;
            ti_b8 pb[3];
#pragma unroll
            for (int g = 0; g < NG; g++) {
                if constexpr (COLS) TI_ISSUE_FENCE();          // a group's operands at a time: registers for three waves a SIMD
                if (!COLS || g == 0) {
                    const v4f v0 = *reinterpret_cast<const v4f*>(&W.vs[BLK * (COLS ? grp : g) + 4 * j]);
                    const v4f v1 = *reinterpret_cast<const v4f*>(&W.vs[BLK * (COLS ? grp : g) + 16 + 4 * j]);
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        x[e] = s[e] * v0[e];
                        x[4 + e] = s[4 + e] * v1[e];
                    }
                    if (!whole) {                              // the scale of a key that the row does not see may be NaN
#pragma unroll
                        for (int e = 0; e < 8; e++) x[e] = seen >> e & 1u ? x[e] : 0.0f;
                    }
                    ti_bf16x3(x, pb);
                }
#pragma unroll
                for (int d = 2 * g; d < 2 * g + 2; d++) {      // COLS: of these 16 dims, the columns of group g hold the output
                    const v2i vb = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                        (__attribute__((address_space(3))) v2i*)&W.v[vrow * HD + 16 * piece_slot<HD>(vrow, d) + 8 * (r16 & 1)]);
                    const uint2 lo = ti_i8x4_b4((uint32_t)vb.x), hi = ti_i8x4_b4((uint32_t)vb.y);
                    const ti_b8 vv = __builtin_bit_cast(ti_b8, make_uint4(lo.x, lo.y, hi.x, hi.y));
#pragma unroll
                    for (int e = 2; e >= 0; e--) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vv, pb[e], o[d], 0, 0, 0);
                }
            }
            // the next block into the place of this one, which has been read
            if (i + a.BW < c1) {
                ti_wave_lds_fence();
                __builtin_amdgcn_s_waitcnt(0xC07F);            // lgkmcnt(0)
                page = check_page(i + a.BW, entry);
                if (i + 2 * a.BW < c1) entry = fetch_page(i + 2 * a.BW);
                load(i + a.BW, page);
            }
        }

        // ---- the waves' parts into the workgroup's partial
        l += ti_xor(l, 16);
        l += ti_xor(l, 32);
        __syncthreads();                                       // the tiles are read
        if (j == 0 && slot == 0) {
            L.m[wave][tr] = m;
            L.l[wave][tr] = l;
        }
#pragma unroll
        for (int d = 0; d < HD / 16; d++)
            if (!COLS || slot == d / 2) *reinterpret_cast<v4f*>(&L.o[wave][tr][16 * d + 4 * j]) = o[d];
        __syncthreads();
        const int nr = ti_min(ROWS, a.R - rt * ROWS);
        for (int e = tid; e < a.HW * nr * (HD / 4); e += THREADS) {
            const int q = e / (HD / 4), d = e % (HD / 4), hh = q / nr, r = q % nr;
            float M = L.m[hh][r];
            for (int k = hh + a.HW; k < WAVES; k += a.HW) M = fmaxf(M, L.m[k][r]);
            v4f x = zero;
            float y = 0.0f;
            for (int k = hh; k < WAVES; k += a.HW) {
                const float mk = L.m[k][r], f = mk == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mk - M);
                const v4f ok = *reinterpret_cast<const v4f*>(&L.o[k][r][4 * d]);
#pragma unroll
                for (int c = 0; c < 4; c++) x[c] = fmaf(ok[c], f, x[c]);
                y = fmaf(L.l[k][r], f, y);
            }
            const size_t at = ((size_t)(w + run.b) * a.p.nKv + hk0 + hh) * a.R + rt * ROWS + r;
            *reinterpret_cast<v4f*>(a.po + at * HD + 4 * d) = x;
            if (d == 0) {
                a.pml[2 * at] = M;
                a.pml[2 * at + 1] = y;
            }
        }
        if (PAGED && c0 == 0 && hr == 0 && tid == 0) {          // the sequence's slots, for the merge
            a.meta[2 * run.b] = w + run.b;
            a.meta[2 * run.b + 1] = (int)((run.start + nb - 1) / run.chunk) - w + 1;
        }
        run.left -= part;
        if (run.left <= 0) return;
        run.b++;
        run.start += nb;
        run.block = 0;
        __syncthreads();                                   // the parts are read
    }
}

// The weights that each key received, by the merge's workgroups behind the rows' own (part of parts): every head's (max, sum)
// from the slots', then a thread a (key, KV head). In the merge's launch and not behind it: 4096 slots of 8 heads
// 4.9 us for both, apart 4.7 + 2.9
__device__ __forceinline__ void token_mass(const TokArgs& a, int ns, int part, int parts) {
    __shared__ float2 s_ml[TI_ATTN_HEADS_MAX];
    const int lane = threadIdx.x & 63, heads = a.p.nHq, G = a.G;
    for (int h = threadIdx.x >> 6; h < heads; h += 4) {
        float m = -INFINITY, l = 0.0f;
        for (int s = lane; s < ns; s += 64) {
            const float2 x = *reinterpret_cast<const float2*>(a.pml + 2 * ((size_t)s * heads + h));
            const float mn = fmaxf(m, x.x);
            if (mn == -INFINITY) continue;
            l = fmaf(l, __builtin_amdgcn_exp2f(m - mn), x.y * __builtin_amdgcn_exp2f(x.x - mn));
            m = mn;
        }
        const float M = ti_wave_max(m);
        const float L = ti_wave_sum(m == -INFINITY ? 0.0f : l * __builtin_amdgcn_exp2f(m - M));
        if (lane == 0) s_ml[h] = make_float2(M, L);
    }
    __syncthreads();
    const long n = (a.p.pos0 + 1L) * a.p.nKv;
    for (long i = (long)part * 256 + threadIdx.x; i < n; i += (long)parts * 256) {
        const long j = i / a.p.nKv;
        const int hk = (int)(i % a.p.nKv);
        float sum = 0.0f;
        for (int h = hk * G; h < (hk + 1) * G; h++)
            sum += __builtin_amdgcn_exp2f(a.p.scores[h * a.p.sstride + j] - s_ml[h].x) / s_ml[h].y;
        a.p.mass[i] = j < a.p.pos0 ? a.p.mass[i] + sum : sum;
    }
}

// A workgroup a (sequence, token, head) and DW of its dims: the slots' partials into the output row, each group of threads
// those of its own slots with every load in flight at once. DW = 32 where whole rows leave CUs idle (16 rows of 128
// dims: 4.1 us, whole rows 5.4)
template <int HD, int DW>
__global__ __launch_bounds__(256) void k_token_merge(TokArgs a, int ns1) {
    constexpr int D4 = DW / 4, SG = 256 / D4, UN = 8;
    __shared__ float s_m[SG], s_l[SG];
    __shared__ __align__(16) float s_o[SG][4 * D4];
    const int tid = threadIdx.x, sg = tid / D4, d = tid % D4;
    const int rows = a.p.B * a.p.T * a.p.nHq, row = blockIdx.x, d0 = DW * blockIdx.y;
    if (row >= rows) return token_mass(a, ns1, (row - rows) * gridDim.y + blockIdx.y, (gridDim.x - rows) * gridDim.y);
    const int hq = row % a.p.nHq, t = (row / a.p.nHq) % a.p.T, b = row / (a.p.nHq * a.p.T);
    const int hk = hq / a.G, r = t * a.G + hq % a.G;
    const int s0 = ns1 ? 0 : a.meta[2 * b], ns = ns1 ? ns1 : a.meta[2 * b + 1];
    const size_t step = (size_t)a.p.nKv * a.R, base = (size_t)s0 * step + (size_t)hk * a.R + r;
    float m = -INFINITY, l = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i0 = sg; i0 < ns && (256 % D4 == 0 || sg < SG); i0 += UN * SG) {
        v4f x[UN];
        float mi[UN], li[UN];
#pragma unroll
        for (int k = 0; k < UN; k++) {
            const size_t at = base + (size_t)ti_min(i0 + k * SG, ns - 1) * step;
            mi[k] = a.pml[2 * at];
            li[k] = a.pml[2 * at + 1];
            x[k] = *reinterpret_cast<const v4f*>(a.po + at * HD + d0 + 4 * d);
        }
        float mn = m;
#pragma unroll
        for (int k = 0; k < UN; k++) mn = fmaxf(mn, mi[k]);
        if (mn == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(m - mn);
        l *= f;
        o = o * f;
        m = mn;
#pragma unroll
        for (int k = 0; k < UN; k++) {
            const float e = i0 + k * SG < ns && mi[k] != -INFINITY ? __builtin_amdgcn_exp2f(mi[k] - m) : 0.0f;
            l = fmaf(li[k], e, l);
#pragma unroll
            for (int c = 0; c < 4; c++) o[c] = fmaf(x[k][c], e, o[c]);
        }
    }
    if (256 % D4 == 0 || sg < SG) {
        *reinterpret_cast<v4f*>(&s_o[sg][4 * d]) = o;
        if (d == 0) {
            s_m[sg] = m;
            s_l[sg] = l;
        }
    }
    __syncthreads();
    if (tid >= DW) return;
    const int n = ti_min(SG, ns);
    float M = -INFINITY, Lt = 0.0f, v = 0.0f;
    for (int g = 0; g < n; g++) M = fmaxf(M, s_m[g]);
    for (int g = 0; g < n; g++) {
        const float e = s_m[g] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[g] - M);
        Lt = fmaf(s_l[g], e, Lt);
        v = fmaf(s_o[g][tid], e, v);
    }
    a.p.out[(size_t)row * HD + d0 + tid] = M == -INFINITY ? 0.0f : v / (127.0f * PSCALE * Lt);
}

template <int HD, bool PAGED>
void launch(ti_ctx* c, const TokArgs& a, long wgs, int ns1) {
    const unsigned grid = (unsigned)(wgs * a.RT * (a.p.nKv / a.HW));
    if (HD == 32 || a.R <= tile_rows(HD, true)) k_token_attn<HD, PAGED, true><<<grid, THREADS, 0, c->stream>>>(a);
    else if constexpr (HD > 32) k_token_attn<HD, PAGED, false><<<grid, THREADS, 0, c->stream>>>(a);
    const int rows = a.p.B * a.p.T * a.p.nHq;
    // the weights' workgroups: two a CU at most, since each forms every head's sum
    const long n = a.p.mass ? ti_min(((a.p.pos0 + 1L) * a.p.nKv + 255) / 256, 2L * c->cus) : 0;
    if (HD == 32 || rows >= c->cus) k_token_merge<HD, HD><<<rows + n, 256, 0, c->stream>>>(a, ns1);
    else if constexpr (HD > 32) k_token_merge<HD, 32><<<dim3(rows + (n + HD / 32 - 1) / (HD / 32), HD / 32), 256, 0, c->stream>>>(a, ns1);
}

}  // namespace

int ti_token_attn_launch(ti_ctx* c, const TiTokenAttn& p, int hd) {
    TokArgs a;
    a.p = p;
    a.po = c->attn_po;
    a.pml = c->attn_ml;
    a.meta = reinterpret_cast<int32_t*>(c->tg_part);
    a.G = p.nHq / p.nKv;
    a.R = p.T * a.G;
    const int rows = tile_rows(hd, true) >= a.R ? tile_rows(hd, true) : 16;
    a.RT = (a.R + rows - 1) / rows;
    static_assert(TI_TG_SPLIT_BLOCKS * 2 * 256 >= 2 * TI_TOKEN_SEQS, "the sequences' slots fit the scratch");
    // four heads of a position together where their number allows it: more of each 1 KB row at a time, though one head a workgroup
    // would join four blocks in LDS. Kernel + merge of 8 heads of 128 dims, a head a wave of 1 / 4: 32 ragged sequences (211 MB) 71.2 + 4.8 /
    // 50.0 + 4.9 us, one token of 4100 keys 9.5 + 4.0 / 8.8 + 4.0, of 8191 in pages of 16 13.3 + 3.9 / 12.2 + 4.2, with the weights added up
    // 8.2 + 4.5 / 7.4 + 5.2; 8 windowed sequences of 64 dims 18.3 + 3.9 / 13.7 + 3.9
    a.HW = p.nKv % 4 == 0 ? 4 : p.nKv % 2 == 0 ? 2 : 1;
    a.BW = WAVES / a.HW;
    // the workgroups that the CUs hold at once (three; two of those with a column a row); as many as there are sequences,
    // if that is more; as far as the partials' slots (one for each workgroup and one for each sequence) fit: half of the
    // scratch where the other half holds scores
    const int groups = p.nKv / a.HW * a.RT, held = a.R <= tile_rows(hd, true) ? 3 : 2;
    long wgs = ti_max(((long)held * c->cus + groups - 1) / groups, (long)p.B);
    wgs = ti_max(1L, ti_min(wgs, (p.mass ? TI_ATTN_ROWSPLITS / 2L : (long)TI_ATTN_ROWSPLITS) / (p.T * p.nHq) - p.B));
    a.wgs = (int)wgs;
    const bool paged = p.lens != nullptr;
    int ns1 = 0;
    if (!paged) {                                          // one sequence of known length: its blocks, and slots
        const int last = p.pos0 + p.T - 1;
        TiSpan s = ti_span(p.pos0, p.window, p.sinks);
        s.end = last + 1;
        const long n = ti_max(1, blocks_of(s).n), chunk = run_chunk(n, 1, a.wgs, a.BW);
        wgs = (n + chunk - 1) / chunk;
        ns1 = (int)wgs;
    } else {
        const long most = p.max_keys / BLK + 3;            // blocks of a sequence, at most (three ragged ends)
        wgs = ti_min(wgs, p.B * most);
    }
#define TOK(HD_) if (hd == HD_) { if (paged) launch<HD_, true>(c, a, wgs, ns1); else launch<HD_, false>(c, a, wgs, ns1); }
    TOK(128) TOK(96) TOK(64) TOK(32)
#undef TOK
    TI_LAUNCHED("k_token_attn");
    return TI_OK;
}
