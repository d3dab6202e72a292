// k_kv_paged.hip — rows of K and V into and out of an int8 KV cache in pages: the paged counterpart of the contiguous
// kvQuantWrite (models/qwen3.js:2180-2216), with the same codes and scales bit for bit, and its inverse.
//
// Row t goes to position pos[t] of sequence seq[t]; a page holds its positions as the contiguous cache does (position,
// then head, then dim), so the contiguous cache is the case of no table. A row whose place does not exist (a negative
// position, past the table's width, an unknown sequence, a page id outside the pool) is not written, and reads as zeros.
#include "ti_dev.h"
#include "ti_span.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

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

// A thread takes four elements (a word of codes) of K or V, row behind row, so that both sides are read and written in whole
// lines; eight neighbouring lanes share a 32-group. Bound by the launch below a few hundred rows (256 rows of 8 heads of 128
// dims written in 3.3 us, read in 3.0; two and four words a thread 3.7 and 5.2, 3.6 and 4.5), by the floats' traffic above (4096
// rows, 42 MB, read in 8.8 us: 4.8 TB/s; with stores that stay in the caches 10.2).
struct WordAt {
    int t;
    unsigned w;                                            // word x of all: row t, word w of it
    __device__ explicit WordAt(const PlaceArgs& a) {
        const unsigned x = blockIdx.x * 256 + threadIdx.x, rw = a.rowg * 8;
        t = (int)(x / rw);
        w = x % rw;
    }
};

__global__ __launch_bounds__(256) void k_kv_write_paged(PlaceArgs a, const float* __restrict__ k, const float* __restrict__ v,
                                                        uint32_t* __restrict__ kq, float* __restrict__ ks,
                                                        uint32_t* __restrict__ vq, float* __restrict__ vs) {
    const bool isv = blockIdx.y;
    const WordAt at(a);
    if (at.t >= a.T) return;                               // whole groups of eight lanes
    const float4 f = reinterpret_cast<const float4*>(isv ? v : k)[(size_t)at.t * a.rowg * 8 + at.w];
    const long row = place_row(a, at.t);
    const float mx = fmaxf(group_max_contig<4>(fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w)))), 1e-12f);
    if (row < 0) return;
    const size_t to = (size_t)row * a.rowg * 8 + at.w;
    (isv ? vq : kq)[to] = snorm_code(f.x, mx) | (snorm_code(f.y, mx) << 8) | (snorm_code(f.z, mx) << 16) | (snorm_code(f.w, mx) << 24);
    if ((at.w & 7) == 0) (isv ? vs : ks)[to / 8] = mx;
}

__global__ __launch_bounds__(256) void k_kv_read_paged(PlaceArgs a, const uint32_t* __restrict__ kq, const float* __restrict__ ks,
                                                       const uint32_t* __restrict__ vq, const float* __restrict__ vs,
                                                       float* __restrict__ k, float* __restrict__ v) {
    const bool isv = blockIdx.y;
    const WordAt at(a);
    if (at.t >= a.T) return;
    const long row = place_row(a, at.t);
    v4f x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (row >= 0) {
        const size_t from = (size_t)row * a.rowg * 8 + at.w;
        const uint32_t c = (isv ? vq : kq)[from];
        const float f = (isv ? vs : ks)[from / 8] / 127.0f;
        x = v4f{(float)(int8_t)c * f, (float)(int8_t)(c >> 8) * f, (float)(int8_t)(c >> 16) * f, (float)(int8_t)(c >> 24) * f};
    }
    __builtin_nontemporal_store(x, reinterpret_cast<v4f*>(isv ? v : k) + (size_t)at.t * a.rowg * 8 + at.w);
}

dim3 word_grid(const PlaceArgs& a) { return dim3((unsigned)(((long)a.T * a.rowg * 8 + 255) / 256), 2); }

int place_args(PlaceArgs& a, const char* fn, const int32_t* table, const int32_t* seq, const int32_t* pos, int T, int B,
               int nKv, int hd, int page, int pages, int width) {
    TI_REQUIRE(T > 0 && (B > 0 || table == nullptr) && nKv > 0 && nKv <= TI_ATTN_HEADS_MAX && hd > 0 && hd % 32 == 0 && hd <= TI_ATTN_HD_MAX,
               "%s: bad shape (T=%d B=%d nKv=%d hd=%d)", fn, T, B, nKv, hd);
    TI_REQUIRE(ti_pow2(page) && pages > 0, "%s: the page length must be a power of two (%d), the pool not empty (%d)", fn, page, pages);
    TI_REQUIRE(table == nullptr || width > 0, "%s: a table of width %d", fn, width);
    TI_REQUIRE((long)page * (table ? width : pages) <= 0x7fffffffL, "%s: %d pages of %d hold more than 2^31 - 1 positions", fn,
               table ? width : pages, page);
    TI_REQUIRE(seq || table == nullptr || T <= B, "%s: %d rows without sequence numbers, %d sequences", fn, T, B);
    TI_REQUIRE((long)T * nKv * (hd / 32) <= 0x0fffffffL, "%s: %d rows of %d heads in one call", fn, T, nKv);
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
    TI_REQUIRE_DENSE("ti_kv_write_paged_q8", kq);
    TI_REQUIRE_DENSE("ti_kv_write_paged_q8", vq);
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
    TI_REQUIRE_DENSE("ti_kv_read_paged_q8", kq);
    TI_REQUIRE_DENSE("ti_kv_read_paged_q8", vq);
    PlaceArgs a;
    const int rc = place_args(a, "ti_kv_read_paged_q8", table, seq, pos, T, B, nKv, hd, page, pages, width);
    if (rc) return rc;
    k_kv_read_paged<<<word_grid(a), 256, 0, c->stream>>>(a, kq, ks, vq, vs, k, v);
    TI_LAUNCHED("k_kv_read_paged");
    return TI_OK;
}
