// k_kv_paged.hip — rows of K and V into and out of an int8 KV cache in pages: the paged counterparts of the contiguous
// kvQuantWrite (models/qwen3.js:2180-2216), with the same codes and scales bit for bit, and of attnPrepQ8 (:2297-2308), the same but for the last
// bits of an angle's f64; and the inverse.
//
// Row t goes to position pos[t] of sequence seq[t]; a page holds its positions as the contiguous cache does (position,
// then head, then dim), so the contiguous cache is the case of no table. A row whose place does not exist (a negative
// position, past the table's width, an unknown sequence, a page id outside the pool) is not written, and reads as zeros.
#include "ti_dev.h"
#include "ti_span.h"
#include <math.h>

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

// ---- rows of Q, K and V at once: norm, rotation, and K and V into their places ------------------------------------
// attnPrepQ8 (models/qwen3.js:2297-2308) for rows of any sequences, with ti_attn_prep_q8's operations in its order: the squares' sum is the
// tree of halves of 128, the angle pos * theta^(-2i/hd) is a double, its cosine and sine are rounded to f32.
struct PrepArgs {
    PlaceArgs at;
    const int32_t* rot;     // positions of the rotation; nullptr: those of the places
    const float *q, *k, *v;
    const uint16_t *qw, *kw;
    float* qr;
    uint32_t *kq, *vq;
    float *ks, *vs;
    long ldq, ldkv;
    int nHq, nKv;
    float eps;
    double freq[TI_ATTN_HD_MAX / 2];
};

// Sine and cosine of x, |x| < 2^32: x - n pi/2 with pi/2 in two doubles (the first difference is exact), then the series to r^17 and
// r^16, whose next terms are below 2^-63 and 2^-58 at pi/4: off by an ulp of f64 or so. ti_attn_prep_q8 takes the device library's power, cosine and
// sine: a frequency's last bit grows with the position and may turn an f32's rounding. Of 1.15 million rotated values, a dozen layouts', none differs
// at positions below 10^4, 2 from there to 10^5, 23 to 10^6, 301 to 10^7: by a step of the rotation's terms or few.
__device__ __forceinline__ void sin_cos(double x, double& sn, double& cs) {
    const double n = rint(x * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489661923, x);
    r = fma(-n, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double s = 1.0 / 355687428096000.0, c = 1.0 / 20922789888000.0;
    s = fma(s, z, -1.0 / 1307674368000.0);
    s = fma(s, z, 1.0 / 6227020800.0);
    s = fma(s, z, -1.0 / 39916800.0);
    s = fma(s, z, 1.0 / 362880.0);
    s = fma(s, z, -1.0 / 5040.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, -1.0 / 6.0);
    s = fma(s * z, r, r);
    c = fma(c, z, -1.0 / 87178291200.0);
    c = fma(c, z, 1.0 / 479001600.0);
    c = fma(c, z, -1.0 / 3628800.0);
    c = fma(c, z, 1.0 / 40320.0);
    c = fma(c, z, -1.0 / 720.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const int k = (int)(long)n & 3;
    const double a = k & 1 ? c : s, b = k & 1 ? s : c;
    sn = k & 2 ? -a : a;
    cs = (k + 1) & 2 ? -b : b;
}

// A workgroup a row's 256 / LPH heads of Q, then K, then V; a lane four elements, LPH lanes a head, so that the tree's halves are lanes
// 16, 8, 4, 2 and 1 apart and the rotation's partner is in another lane's registers. The row's angles are formed once a workgroup.
// Bound by the launch and its round trips below some hundred rows (one row of 16 and 8 heads of 128 dims 3.7 us, 64 rows 4.0), then by the floats: 2000 rows
// of 32 and 8 heads of 64 dims (43 MB) 14.2 us, 3.0 TB/s.
template <int HD>
__global__ __launch_bounds__(256) void k_attn_prep_paged(PrepArgs a) {
    constexpr int LPH = HD > 64 ? 32 : HD / 4, HALF = HD / 2;
    __shared__ __align__(16) float s_cs[HALF], s_sn[HALF];
    const int heads = a.nHq + 2 * a.nKv, parts = (heads + 256 / LPH - 1) / (256 / LPH);
    const int tid = threadIdx.x, m = tid % LPH, t = blockIdx.x / parts, first = (blockIdx.x % parts) * (256 / LPH), head = first + tid / LPH;
    const bool isq = head < a.nHq, isv = head >= a.nHq + a.nKv, live = head < heads && 4 * m < HD;
    const int h = isq ? head : isv ? ti_min(head, heads - 1) - a.nHq - a.nKv : head - a.nHq;
    const float* src = isq ? a.q + t * a.ldq : (isv ? a.v : a.k) + t * a.ldkv;
    const int e0 = ti_min(4 * m, HD - 4);
    const v4f x = *reinterpret_cast<const v4f*>(src + h * HD + e0);
    const int pos = a.at.pos[t], turn = a.rot ? a.rot[t] : pos;
    const uint16_t* nw = isq ? a.qw : a.kw;
    const bool norm = !isv && nw;
    uint2 w2 = make_uint2(0, 0);
    if (norm) w2 = *reinterpret_cast<const uint2*>(nw + e0);
    const bool turns = first < a.nHq + a.nKv;              // workgroup-uniform: any but V heads
    if (turns && tid < HALF) {
        double sn, cs;
        sin_cos((double)turn * a.freq[tid], sn, cs);
        s_cs[tid] = (float)cs;
        s_sn[tid] = (float)sn;
    }
    const long row = isq ? 0 : place_row(a.at, t);
    __syncthreads();
    v4f y = x;
    if (norm) {
        v4f s;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float v = 4 * m < HD ? x[e] * x[e] : 0.0f;
            if constexpr (LPH == 32) v += ti_xor(v, 16);
            if constexpr (LPH >= 16) v += ti_xor(v, 8);
            v += ti_xor(v, 4);
            v += ti_xor(v, 2);
            s[e] = v + ti_xor(v, 1);
        }
        const float sum = (s[0] + s[2]) + (s[1] + s[3]);
        float mean = sum / (float)HD;
        mean = mean + a.eps;
        const float inv = 1.0f / sqrtf(mean);
        const uint16_t w[4] = {(uint16_t)w2.x, (uint16_t)(w2.x >> 16), (uint16_t)w2.y, (uint16_t)(w2.y >> 16)};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float p = x[e] * inv;
            y[e] = p * ti_h2f(w[e]);
        }
    }
    if (turns) {
        const int i0 = e0 % HALF;
        const v4f c = *reinterpret_cast<const v4f*>(&s_cs[i0]), s = *reinterpret_cast<const v4f*>(&s_sn[i0]);
        const bool lo = e0 < HALF;
        v4f z;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float o;
            if constexpr (HD == 96) o = __shfl(y[e], ((tid & 63) & 32) + (lo ? m + HALF / 4 : m - HALF / 4));
            else o = ti_xor(y[e], HALF / 4);
            const float p = y[e] * c[e], r = (lo ? -o : o) * s[e];
            z[e] = p + r;
        }
        if (!isv) y = z;
    }
    if (!live) return;                                     // whole groups of eight lanes
    if (isq) {
        __builtin_nontemporal_store(y, reinterpret_cast<v4f*>(a.qr + ((size_t)t * a.nHq + h) * HD + e0));
        return;
    }
    const float mx = fmaxf(group_max_contig<4>(fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3])))), 1e-12f);
    if (row < 0) return;
    const size_t to = ((size_t)row * a.nKv + h) * (HD / 4) + m;
    (isv ? a.vq : a.kq)[to] = snorm_code(y[0], mx) | (snorm_code(y[1], mx) << 8) | (snorm_code(y[2], mx) << 16) | (snorm_code(y[3], mx) << 24);
    if ((m & 7) == 0) (isv ? a.vs : a.ks)[to / 8] = mx;
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

extern "C" int ti_attn_prep_paged_q8(ti_ctx* c, const float* q, const float* k, const float* v, const uint16_t* qn_w, const uint16_t* kn_w,
                                     float* qr, uint32_t* kq, float* ks, uint32_t* vq, float* vs, const int32_t* table,
                                     const int32_t* seq, const int32_t* pos, const int32_t* rot, int T, int B, int nHq, int nKv, int hd,
                                     int page, int pages, int width, int ldq, int ldkv, float theta, float eps) {
    TI_CHECK_CTX(c);
    const char* fn = "ti_attn_prep_paged_q8";
    TI_REQUIRE(k && v && kq && ks && vq && vs && pos, "%s: null buffer", fn);
    TI_REQUIRE(nHq >= 0 && nHq <= TI_ATTN_HEADS_MAX && (nHq == 0 || (q && qr)), "%s: %d query heads need q and qr, and are at most %d", fn, nHq, TI_ATTN_HEADS_MAX);
    PrepArgs a;
    const int rc = place_args(a.at, fn, table, seq, pos, T, B, nKv, hd, page, pages, width);
    if (rc) return rc;
    const int per = 256 / (hd > 64 ? 32 : hd / 4);
    const long grid = (long)T * ((nHq + 2 * nKv + per - 1) / per);
    TI_REQUIRE(grid <= 0xffffff, "%s: %d rows of %d heads in one call", fn, T, nHq + 2 * nKv);
    TI_REQUIRE(theta >= 1.0f && theta < INFINITY, "%s: theta must be finite and at least 1", fn);
    a.ldq = ldq ? ldq : nHq * hd;
    a.ldkv = ldkv ? ldkv : nKv * hd;
    TI_REQUIRE((nHq == 0 || a.ldq >= nHq * hd) && a.ldkv >= nKv * hd && a.ldq % 4 == 0 && a.ldkv % 4 == 0,
               "%s: rows of %ld and %ld floats: at least a row's heads, and multiples of 4", fn, a.ldq, a.ldkv);
    TI_REQUIRE(ti_al16(k) && ti_al16(v) && ti_al16(kq) && ti_al16(vq) && (nHq == 0 || (ti_al16(q) && ti_al16(qr))),
               "%s: q, k, v, qr, kq and vq must be 16-byte aligned", fn);
    TI_REQUIRE((((uintptr_t)qn_w | (uintptr_t)kn_w) & 7u) == 0, "%s: norm weights must be 8-byte aligned", fn);
    if (nHq) {
        const uintptr_t q0 = (uintptr_t)q, r0 = (uintptr_t)qr, q1 = q0 + 4 * ((T - 1) * (size_t)a.ldq + nHq * hd), r1 = r0 + 4 * (size_t)T * nHq * hd;
        TI_REQUIRE((q0 == r0 && a.ldq == nHq * hd) || q1 <= r0 || r1 <= q0, "%s: qr is q itself, with dense rows, or does not overlap it", fn);
        const size_t kv = 4 * ((T - 1) * (size_t)a.ldkv + nKv * hd);
        for (const float* p : {k, v}) TI_REQUIRE((uintptr_t)p + kv <= r0 || r1 <= (uintptr_t)p, "%s: qr overlaps k or v", fn);
    }
    TI_REQUIRE_DENSE(fn, kq);
    TI_REQUIRE_DENSE(fn, vq);
    a.rot = rot;
    a.q = q; a.k = k; a.v = v;
    a.qw = qn_w; a.kw = kn_w;
    a.qr = qr;
    a.kq = kq; a.vq = vq; a.ks = ks; a.vs = vs;
    a.nHq = nHq;
    a.nKv = nKv;
    a.eps = eps;
    // theta^(-2i/hd) by products of 64 bits' mantissas: within half an ulp of f64 and 2^-57, and one power a call
    const long double step = powl((long double)theta, -2.0L / hd), ln = logl((long double)theta);
    long double f = 1.0L;
    for (int i = 0; i < hd / 2; i++, f *= step) {
        // the exponent is a double there, which rounds it where hd is no power of two
        const long double off = ti_pow2(hd) ? 0.0L : (long double)(-2.0 * i / hd) - -2.0L * i / hd;
        a.freq[i] = (double)(f + f * off * ln);
    }
#define PREP(HD_) if (hd == HD_) k_attn_prep_paged<HD_><<<(unsigned)grid, 256, 0, c->stream>>>(a);
    PREP(128) PREP(96) PREP(64) PREP(32)
#undef PREP
    TI_LAUNCHED("k_attn_prep_paged");
    return TI_OK;
}
