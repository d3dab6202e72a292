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

// A thread takes four elements (a word of codes) at a time, a workgroup WORDS words of K or V, row behind row, so that both
// sides are read and written in whole lines; eight neighbouring lanes share a 32-group. Bound by the launch below a few
// hundred rows (256 rows of 8 heads of 128 dims written in 5.3 us, read in 4.7), by the floats' traffic above (4096 rows, 42
// MB, read in 10 us: 4.2 TB/s).
constexpr int WORDS = 1024;

// word x of the workgroup -> row t and word of it; false: behind the last
struct WordAt {
    int t, w;
    __device__ WordAt(const PlaceArgs& a, int x) {
        const int rw = a.rowg * 8;
        const long base = (long)blockIdx.x * WORDS;
        const long t0 = base / rw;                         // workgroup-uniform
        const unsigned l = (unsigned)(base - t0 * rw) + x;
        t = (int)(t0 + l / (unsigned)rw);
        w = (int)(l % (unsigned)rw);
    }
};

__global__ __launch_bounds__(256) void k_kv_write_paged(PlaceArgs a, const float* __restrict__ k, const float* __restrict__ v,
                                                        uint32_t* __restrict__ kq, float* __restrict__ ks,
                                                        uint32_t* __restrict__ vq, float* __restrict__ vs) {
    const bool isv = blockIdx.y;
    const float4* src = reinterpret_cast<const float4*>(isv ? v : k);
    float4 x[WORDS / 256];
    long row[WORDS / 256];
    int w[WORDS / 256];
#pragma unroll
    for (int u = 0; u < WORDS / 256; u++) {
        const WordAt at(a, threadIdx.x + 256 * u);
        const bool in = at.t < a.T;
        x[u] = in ? src[(size_t)at.t * a.rowg * 8 + at.w] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        row[u] = in ? place_row(a, at.t) : -1;
        w[u] = at.w;
    }
#pragma unroll
    for (int u = 0; u < WORDS / 256; u++) {
        const float4 f = x[u];
        const float mx = fmaxf(group_max_contig<4>(fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w)))), 1e-12f);
        if (row[u] < 0) continue;
        const size_t at = (size_t)row[u] * a.rowg * 8 + w[u];
        (isv ? vq : kq)[at] = snorm_code(f.x, mx) | (snorm_code(f.y, mx) << 8) | (snorm_code(f.z, mx) << 16) | (snorm_code(f.w, mx) << 24);
        if ((w[u] & 7) == 0) (isv ? vs : ks)[at / 8] = mx;
    }
}

__global__ __launch_bounds__(256) void k_kv_read_paged(PlaceArgs a, const uint32_t* __restrict__ kq, const float* __restrict__ ks,
                                                       const uint32_t* __restrict__ vq, const float* __restrict__ vs,
                                                       float* __restrict__ k, float* __restrict__ v) {
    const bool isv = blockIdx.y;
    const uint32_t* codes = isv ? vq : kq;
    const float* scales = isv ? vs : ks;
    float4* out = reinterpret_cast<float4*>(isv ? v : k);
    uint32_t c[WORDS / 256];
    float s[WORDS / 256];
    long dst[WORDS / 256];
#pragma unroll
    for (int u = 0; u < WORDS / 256; u++) {
        const WordAt at(a, threadIdx.x + 256 * u);
        const bool in = at.t < a.T;
        const long row = in ? place_row(a, at.t) : -1;
        const size_t g = (size_t)(row < 0 ? 0 : row) * a.rowg * 8 + at.w;
        c[u] = row < 0 ? 0u : codes[g];
        s[u] = row < 0 ? 0.0f : scales[g / 8];
        dst[u] = in ? (long)at.t * a.rowg * 8 + at.w : -1;
    }
#pragma unroll
    for (int u = 0; u < WORDS / 256; u++) {
        if (dst[u] < 0) continue;
        const float f = s[u] / 127.0f;
        out[dst[u]] = make_float4((float)(int8_t)c[u] * f, (float)(int8_t)(c[u] >> 8) * f, (float)(int8_t)(c[u] >> 16) * f,
                                  (float)(int8_t)(c[u] >> 24) * f);
    }
}

dim3 word_grid(const PlaceArgs& a) { return dim3((unsigned)(((long)a.T * a.rowg * 8 + WORDS - 1) / WORDS), 2); }

int place_args(PlaceArgs& a, const char* fn, const int32_t* table, const int32_t* seq, const int32_t* pos, int T, int B,
               int nKv, int hd, int page, int pages, int width) {
    TI_REQUIRE(T > 0 && (B > 0 || table == nullptr) && nKv > 0 && nKv <= TI_ATTN_HEADS_MAX && hd > 0 && hd % 32 == 0 && hd <= TI_ATTN_HD_MAX,
               "%s: bad shape (T=%d B=%d nKv=%d hd=%d)", fn, T, B, nKv, hd);
    TI_REQUIRE(ti_pow2(page) && pages > 0, "%s: the page length must be a power of two (%d), the pool not empty (%d)", fn, page, pages);
    TI_REQUIRE(table == nullptr || width > 0, "%s: a table of width %d", fn, width);
    TI_REQUIRE((long)page * (table ? width : pages) <= 0x7fffffffL, "%s: %d pages of %d hold more than 2^31 - 1 positions", fn,
               table ? width : pages, page);
    TI_REQUIRE(seq || table == nullptr || T <= B, "%s: %d rows without sequence numbers, %d sequences", fn, T, B);
    TI_REQUIRE((long)T * nKv * (hd / 32) <= 0x3fffffffL, "%s: %d rows of %d heads in one call", fn, T, nKv);
    a.pg = TiPages{table, ti_log2(page), pages, width};
    a.seq = table ? seq : nullptr;
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
    k_kv_write_paged<<<word_grid(a), 256, 0, c->stream>>>(a, kr, v, kq, ks, vq, vs);
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
    k_kv_read_paged<<<word_grid(a), 256, 0, c->stream>>>(a, kq, ks, vq, vs, k, v);
    TI_LAUNCHED("k_kv_read_paged");
    return TI_OK;
}
