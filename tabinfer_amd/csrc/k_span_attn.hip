// k_span_attn.hip — attention over a part of the int8 KV cache: under a sliding window with sinks, over pages, and with
// the weight that each key receives added up. See ti_span.h for the visible keys and their rows.
//
// One workgroup a (query, head), over the visible keys in tiles of 256: a thread's dot product, the tile's maximum and sum
// in the running softmax, then P V with a thread a dim and half of the tile's keys.
#include "ti_dev.h"
#include "ti_span.h"
#include "ti_token_attn.h"

namespace {

constexpr int TILE = 256;
constexpr float PSCALE = 0x1p-24f;       // of every weight: 127 x a V scale x thousands of keys stays in f32's range
constexpr long MASS_SCORES = 1L << 24;   // (query head, slot) scores of a one-token call

struct SpanArgs {
    const float* qr;
    const uint8_t* kq;
    const float* ks;
    const uint8_t* vq;
    const float* vs;
    float* out;
    float* ml;               // (max, sum) of each row, or nullptr
    TiPages pg;
    const int32_t* lens;     // paged: keys of each sequence; else query t is at pos0 + t
    int pos0, nHq, nKv, hd, window, sinks;
};

__device__ __forceinline__ int span_pos(const SpanArgs& a, int t) {
    if (!a.lens) return a.pos0 + t;
    const long most = (long)a.pg.width << a.pg.shift;
    const int n = a.lens[t];
    return (int)(n < most ? n : most) - 1;
}

__device__ __forceinline__ float key_score(const SpanArgs& a, const float* q, long row, int hk) {
    const uint8_t* k = a.kq + ((size_t)row * a.nKv + hk) * a.hd;
    const float* ks = a.ks + ((size_t)row * a.nKv + hk) * (a.hd / 32);
    float s = 0.0f;
    for (int g = 0; g < a.hd / 32; g++) {
        const uint4* w4 = reinterpret_cast<const uint4*>(k + 32 * g);
        float d = 0.0f;
        for (int u = 0; u < 2; u++) {
            const uint4 w = w4[u];
            const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
            for (int i = 0; i < 16; i++) d = fmaf(q[32 * g + 16 * u + i], (float)(int8_t)(ww[i >> 2] >> (8 * (i & 3))), d);
        }
        s = fmaf(d, ks[g], s);
    }
    return s * (1.0f / (127.0f * sqrtf((float)a.hd)));
}

__global__ __launch_bounds__(256) void k_span_attn(SpanArgs a) {
    __shared__ float q[TI_ATTN_HD_MAX], p[TILE], red[4], o2[2][TI_ATTN_HD_MAX];
    __shared__ long rows[TILE];
    const int tid = threadIdx.x;
    const int t = blockIdx.x / a.nHq, hq = blockIdx.x % a.nHq, hk = hq / (a.nHq / a.nKv);
    const int pos = span_pos(a, t);
    const TiSpan sp = ti_span(pos, a.window, a.sinks);
    const int n = pos < 0 ? 0 : sp.count();
    const size_t orow = (size_t)t * a.nHq + hq;
    if (tid < a.hd) q[tid] = a.qr[orow * a.hd + tid];
    float m = -INFINITY, l = 0.0f, acc = 0.0f;
    const int d = tid & 127, half = tid >> 7;
    for (int i0 = 0; i0 < n; i0 += TILE) {
        __syncthreads();
        const long row = i0 + tid < n ? a.pg.row(t, sp.at(i0 + tid)) : -1;
        const bool ok = row >= 0;
        const float s = ok ? key_score(a, q, row, hk) : -INFINITY;
        rows[tid] = row;
        // the finite floor: a row that sees only scores of -inf is not an empty one
        float mt = ti_wave_max(ok ? fmaxf(s, -3.402823466e38f) : -INFINITY);
        if ((tid & 63) == 0) red[tid >> 6] = mt;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
        const float pe = ok ? expf(s - mn) * PSCALE : 0.0f;
        p[tid] = pe;
        __syncthreads();
        const float sum = ti_wave_sum(pe);
        if ((tid & 63) == 0) red[tid >> 6] = sum;
        const float corr = m == mn ? 1.0f : expf(m - mn);
        m = mn;
        acc *= corr;
        if (d < a.hd)
            for (int j = half * (TILE / 2); j < (half + 1) * (TILE / 2); j++) {
                if (rows[j] < 0) continue;
                const size_t r = (size_t)rows[j] * a.nKv + hk;
                const float w = p[j] * a.vs[r * (a.hd / 32) + d / 32];
                acc = fmaf(w, (float)(int8_t)a.vq[r * a.hd + d], acc);
            }
        __syncthreads();
        l = l * corr + ((red[0] + red[1]) + (red[2] + red[3]));
    }
    o2[half][d] = acc;
    __syncthreads();
    if (tid < a.hd) a.out[orow * a.hd + tid] = m == -INFINITY ? 0.0f : (o2[0][tid] + o2[1][tid]) / (127.0f * l);
    if (a.ml && tid == 0) {
        a.ml[2 * orow] = m;
        a.ml[2 * orow + 1] = l;
    }
}

// thread = one (key, KV head): the weights that the T queries of its G heads gave it
__global__ __launch_bounds__(256) void k_span_mass(SpanArgs a, float* __restrict__ mass, int T) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= ((long)a.pos0 + T) * a.nKv) return;
    const int j = (int)(i / a.nKv), hk = (int)(i % a.nKv), G = a.nHq / a.nKv;
    float sum = 0.0f;
    for (int t = j > a.pos0 ? j - a.pos0 : 0; t < T; t++)
        for (int h = 0; h < G; h++) {
            const size_t row = (size_t)t * a.nHq + hk * G + h;
            sum += expf(key_score(a, a.qr + row * a.hd, j, hk) - a.ml[2 * row]) * PSCALE / a.ml[2 * row + 1];
        }
    mass[i] = j < a.pos0 ? mass[i] + sum : sum;
}

// thread = one (slot, KV head) of a one-token call: the weights that its G heads gave the slot, from their scores
__global__ __launch_bounds__(256) void k_token_mass(const float* __restrict__ scores, long sstride, const float* __restrict__ ml,
                                                    float* __restrict__ mass, int pos0, int nHq, int nKv) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (pos0 + 1L) * nKv) return;
    const int j = (int)(i / nKv), hk = (int)(i % nKv), G = nHq / nKv;
    float sum = 0.0f;
    for (int h = hk * G; h < (hk + 1) * G; h++) sum += __builtin_amdgcn_exp2f(scores[h * sstride + j] - ml[2 * h]) / ml[2 * h + 1];
    mass[i] = j < pos0 ? mass[i] + sum : sum;
}

int check_attn(const char* fn, const void* qr, const void* kq, const void* ks, const void* vq, const void* vs, const void* out,
               int n, int nHq, int nKv, int hd) {
    TI_REQUIRE(qr && kq && ks && vq && vs && out, "%s: null buffer", fn);
    TI_REQUIRE(qr != out, "%s: out must not be the queries", fn);
    TI_REQUIRE(n > 0 && nKv > 0 && nHq > 0 && nHq % nKv == 0 && nHq <= TI_ATTN_HEADS_MAX, "%s: bad rows/heads (%d rows, nHq=%d nKv=%d)",
               fn, n, nHq, nKv);
    TI_REQUIRE(hd > 0 && hd % 32 == 0 && hd <= TI_ATTN_HD_MAX, "%s: hd must be a multiple of 32 and <= %d", fn, TI_ATTN_HD_MAX);
    TI_REQUIRE(ti_al16(kq) && ti_al16(vq), "%s: kq/vq must be 16-byte aligned", fn);
    return TI_OK;
}

}  // namespace

extern "C" int ti_attn_window_q8(ti_ctx* c, const float* qr, const uint32_t* kq, const float* ks, const uint32_t* vq, const float* vs,
                                 float* out, int T, int pos0, int nHq, int nKv, int hd, int window, int sinks) {
    TI_CHECK_CTX(c);
    const int rc = check_attn("ti_attn_window_q8", qr, kq, ks, vq, vs, out, T, nHq, nKv, hd);
    if (rc) return rc;
    TI_REQUIRE(pos0 >= 0 && pos0 <= 0x7fffffff - T && sinks >= 0, "ti_attn_window_q8: bad positions (T=%d pos0=%d sinks=%d)", T, pos0, sinks);
    TI_REQUIRE((long)T * nHq <= 0x7fffffffL / 256, "ti_attn_window_q8: %d x %d query rows in one call", T, nHq);
    if (T == 1 || T * (nHq / nKv) <= 16) {
        const long keys = window < 0 ? (long)pos0 + T : min((long)pos0 + T, (long)window + sinks + T);
        const TiTokenAttn p = {qr, reinterpret_cast<const uint8_t*>(kq), ks, reinterpret_cast<const uint8_t*>(vq), vs, out,
                               TiPages{nullptr, 0, 0, 0}, nullptr, 1, T, pos0, nHq, nKv, window, sinks, keys, nullptr, 0, nullptr};
        return ti_token_attn_launch(c, p, hd);
    }
    SpanArgs a = {qr, reinterpret_cast<const uint8_t*>(kq), ks, reinterpret_cast<const uint8_t*>(vq), vs, out, nullptr,
                  TiPages{nullptr, 0, 0x7fffffff, 0}, nullptr, pos0, nHq, nKv, hd, window, sinks};
    k_span_attn<<<(unsigned)(T * nHq), 256, 0, c->stream>>>(a);
    TI_LAUNCHED("k_span_attn");
    return TI_OK;
}

extern "C" int ti_attn_paged_q8(ti_ctx* c, const float* qr, const uint32_t* kq, const float* ks, const uint32_t* vq, const float* vs,
                                const int32_t* table, const int32_t* lens, float* out, int B, int nHq, int nKv, int hd, int page,
                                int pages, int width, int window, int sinks) {
    TI_CHECK_CTX(c);
    const int rc = check_attn("ti_attn_paged_q8", qr, kq, ks, vq, vs, out, B, nHq, nKv, hd);
    if (rc) return rc;
    TI_REQUIRE(table && lens, "ti_attn_paged_q8: null table or lengths");
    TI_REQUIRE(B <= 4096, "ti_attn_paged_q8: %d sequences > 4096", B);
    TI_REQUIRE(ti_pow2(page) && pages > 0 && width > 0 && (long)page * width <= 0x7fffffffL,
               "ti_attn_paged_q8: bad pages (length %d, a power of two; %d of them; table width %d)", page, pages, width);
    TI_REQUIRE(sinks >= 0, "ti_attn_paged_q8: sinks = %d", sinks);
    const long all = (long)page * width, keys = window < 0 ? all : min(all, (long)window + sinks + 1);
    const TiTokenAttn p = {qr, reinterpret_cast<const uint8_t*>(kq), ks, reinterpret_cast<const uint8_t*>(vq), vs, out,
                           TiPages{table, ti_log2(page), pages, width}, lens, B, 1, 0, nHq, nKv, window, sinks, keys, nullptr, 0, nullptr};
    return ti_token_attn_launch(c, p, hd);
}

extern "C" int ti_attn_mass_q8(ti_ctx* c, const float* qr, const uint32_t* kq, const float* ks, const uint32_t* vq, const float* vs,
                               float* out, float* mass, int T, int pos0, int nHq, int nKv, int hd) {
    TI_CHECK_CTX(c);
    const int rc = check_attn("ti_attn_mass_q8", qr, kq, ks, vq, vs, out, T, nHq, nKv, hd);
    if (rc) return rc;
    TI_REQUIRE(mass, "ti_attn_mass_q8: null mass");
    TI_REQUIRE(pos0 >= 0 && pos0 <= 0x7fffffff - T, "ti_attn_mass_q8: bad positions (T=%d pos0=%d)", T, pos0);
    TI_REQUIRE((long)T * nHq <= TI_ATTN_ROWS_MAX, "ti_attn_mass_q8: T*nHq = %ld > %d", (long)T * nHq, TI_ATTN_ROWS_MAX);
    TI_REQUIRE(T > 1 || (long)nHq * ((pos0 + 32L) / 32 * 32) <= MASS_SCORES, "ti_attn_mass_q8: %d heads over %d slots exceed the scratch (%ld scores)",
               nHq, pos0 + 1, MASS_SCORES);
    if (T == 1) {
        // the upper half of the partials' scratch holds the scores (2048 slots of 64 heads fill the lower one), the
        // argmax scratch each head's (max, sum)
        const TiTokenAttn p = {qr, reinterpret_cast<const uint8_t*>(kq), ks, reinterpret_cast<const uint8_t*>(vq), vs, out,
                               TiPages{nullptr, 0, 0, 0}, nullptr, 1, 1, pos0, nHq, nKv, -1, 0, pos0 + 1L, c->attn_po + MASS_SCORES,
                               (pos0 + 32L) / 32 * 32, c->amax_v};
        const int rt = ti_token_attn_launch(c, p, hd);
        if (rt) return rt;
        const long n = (pos0 + 1L) * nKv;
        k_token_mass<<<(unsigned)((n + 255) / 256), 256, 0, c->stream>>>(p.scores, p.sstride, p.ml, mass, pos0, nHq, nKv);
        TI_LAUNCHED("k_token_mass");
        return TI_OK;
    }
    SpanArgs a = {qr, reinterpret_cast<const uint8_t*>(kq), ks, reinterpret_cast<const uint8_t*>(vq), vs, out, c->attn_ml,
                  TiPages{nullptr, 0, 0x7fffffff, 0}, nullptr, pos0, nHq, nKv, hd, -1, 0};
    k_span_attn<<<(unsigned)(T * nHq), 256, 0, c->stream>>>(a);
    TI_LAUNCHED("k_span_attn");
    const long keys = ((long)pos0 + T) * nKv;
    k_span_mass<<<(unsigned)((keys + 255) / 256), 256, 0, c->stream>>>(a, mass, T);
    TI_LAUNCHED("k_span_mass");
    return TI_OK;
}
