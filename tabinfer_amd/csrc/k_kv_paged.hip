// k_kv_paged.hip — rows of K and V into and out of an int8 KV cache in pages: the paged counterpart of the contiguous
// kvQuantWrite (models/qwen3.js:2180-2216), with the same codes and scales bit for bit, and its inverse.
//
// Row t goes to position pos[t] of sequence seq[t]; a page holds its positions as the contiguous cache does (position,
// then head, then dim), so the contiguous cache is the case of no table. A row whose place does not exist (a negative
// position, past the table's width, an unknown sequence, a page id outside the pool) is not written, and reads as zeros.
#include "ti_dev.h"
#include "ti_span.h"

namespace {

struct PlaceArgs {
    TiPages pg;
    const int32_t* seq;     // nullptr: row t is sequence t
    const int32_t* pos;
    int T, B, rowg;         // rowg: 32-groups of a cached position (KV heads x head_dim / 32)
};

__device__ __forceinline__ long place_row(const PlaceArgs& a, int t) {
    const int s = a.seq ? a.seq[t] : t;
    if (a.pg.table && (s < 0 || s >= a.B)) return -1;
    return a.pg.row(s, a.pos[t]);
}

// thread = one 32-group of K, then of V
__global__ __launch_bounds__(256) void k_kv_write_paged(PlaceArgs a, const float* __restrict__ k, const float* __restrict__ v,
                                                        uint32_t* __restrict__ kq, float* __restrict__ ks,
                                                        uint32_t* __restrict__ vq, float* __restrict__ vs) {
    const long nG = (long)a.T * a.rowg;
    const long idx = (long)blockIdx.x * 256 + threadIdx.x;
    if (idx >= 2 * nG) return;
    const bool isv = idx >= nG;
    const long g = isv ? idx - nG : idx;
    const long row = place_row(a, (int)(g / a.rowg));
    if (row < 0) return;
    float x[32];
    load32((isv ? v : k) + g * 32, x);
    float mx = 1e-12f;
#pragma unroll
    for (int j = 0; j < 32; j++) mx = fmaxf(mx, fabsf(x[j]));
    const long at = row * a.rowg + g % a.rowg;
    (isv ? vs : ks)[at] = mx;
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; j++)
        w[j] = snorm_code(x[4 * j], mx) | (snorm_code(x[4 * j + 1], mx) << 8) | (snorm_code(x[4 * j + 2], mx) << 16) |
               (snorm_code(x[4 * j + 3], mx) << 24);
    uint4* o = reinterpret_cast<uint4*>(isv ? vq : kq) + at * 2;
    o[0] = make_uint4(w[0], w[1], w[2], w[3]);
    o[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

__global__ __launch_bounds__(256) void k_kv_read_paged(PlaceArgs a, const uint32_t* __restrict__ kq, const float* __restrict__ ks,
                                                       const uint32_t* __restrict__ vq, const float* __restrict__ vs,
                                                       float* __restrict__ k, float* __restrict__ v) {
    const long nG = (long)a.T * a.rowg;
    const long idx = (long)blockIdx.x * 256 + threadIdx.x;
    if (idx >= 2 * nG) return;
    const bool isv = idx >= nG;
    const long g = isv ? idx - nG : idx;
    const long row = place_row(a, (int)(g / a.rowg));
    float* out = (isv ? v : k) + g * 32;
    const long at = row * a.rowg + g % a.rowg;
    const float s = row < 0 ? 0.0f : (isv ? vs : ks)[at] / 127.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t w = row < 0 ? 0u : (isv ? vq : kq)[at * 8 + j];
#pragma unroll
        for (int e = 0; e < 4; e++) out[4 * j + e] = (float)(int8_t)(w >> (8 * e)) * s;
    }
}

int place_args(PlaceArgs& a, const char* fn, const int32_t* table, const int32_t* seq, const int32_t* pos, int T, int B,
               int nKv, int hd, int page, int pages, int width) {
    TI_REQUIRE(T > 0 && B > 0 && nKv > 0 && hd > 0 && hd % 32 == 0 && hd <= TI_ATTN_HD_MAX, "%s: bad shape (T=%d B=%d nKv=%d hd=%d)", fn,
               T, B, nKv, hd);
    TI_REQUIRE(ti_pow2(page) && pages > 0, "%s: the page length must be a power of two (%d), the pool not empty (%d)", fn, page, pages);
    TI_REQUIRE(table == nullptr || width > 0, "%s: a table of width %d", fn, width);
    TI_REQUIRE((long)page * (table ? width : pages) <= 0x7fffffffL, "%s: %d pages of %d hold more than 2^31 - 1 positions", fn,
               table ? width : pages, page);
    TI_REQUIRE(seq || table == nullptr || T <= B, "%s: %d rows without sequence numbers, %d sequences", fn, T, B);
    TI_REQUIRE((long)T * nKv * (hd / 32) <= 0x3fffffffL, "%s: %d rows of %d heads in one call", fn, T, nKv);
    a.pg = TiPages{table, ti_log2(page), pages, width};
    a.seq = seq;
    a.pos = pos;
    a.T = T;
    a.B = B;
    a.rowg = nKv * hd / 32;
    return TI_OK;
}

}  // namespace

extern "C" int ti_kv_write_paged_q8(ti_ctx* c, const float* kr, const float* v, uint32_t* kq, float* ks, uint32_t* vq, float* vs,
                                    const int32_t* table, const int32_t* seq, const int32_t* pos, int T, int B, int nKv, int hd,
                                    int page, int pages, int width) {
    TI_CHECK_CTX(c);
    TI_REQUIRE(kr && v && kq && ks && vq && vs && pos, "ti_kv_write_paged_q8: null buffer");
    TI_REQUIRE(ti_al16(kr) && ti_al16(v) && ti_al16(kq) && ti_al16(vq), "ti_kv_write_paged_q8: kr, v, kq and vq must be 16-byte aligned");
    PlaceArgs a;
    const int rc = place_args(a, "ti_kv_write_paged_q8", table, seq, pos, T, B, nKv, hd, page, pages, width);
    if (rc) return rc;
    const long threads = 2L * T * a.rowg;
    k_kv_write_paged<<<(unsigned)((threads + 255) / 256), 256, 0, c->stream>>>(a, kr, v, kq, ks, vq, vs);
    TI_LAUNCHED("k_kv_write_paged");
    return TI_OK;
}

extern "C" int ti_kv_read_paged_q8(ti_ctx* c, const uint32_t* kq, const float* ks, const uint32_t* vq, const float* vs,
                                   const int32_t* table, const int32_t* seq, const int32_t* pos, float* k, float* v, int T, int B,
                                   int nKv, int hd, int page, int pages, int width) {
    TI_CHECK_CTX(c);
    TI_REQUIRE(kq && ks && vq && vs && pos && k && v, "ti_kv_read_paged_q8: null buffer");
    TI_REQUIRE(ti_al16(kq) && ti_al16(vq) && ti_al16(k) && ti_al16(v), "ti_kv_read_paged_q8: kq, vq, k and v must be 16-byte aligned");
    PlaceArgs a;
    const int rc = place_args(a, "ti_kv_read_paged_q8", table, seq, pos, T, B, nKv, hd, page, pages, width);
    if (rc) return rc;
    const long threads = 2L * T * a.rowg;
    k_kv_read_paged<<<(unsigned)((threads + 255) / 256), 256, 0, c->stream>>>(a, kq, ks, vq, vs, k, v);
    TI_LAUNCHED("k_kv_read_paged");
    return TI_OK;
}
