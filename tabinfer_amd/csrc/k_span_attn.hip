// k_span_attn.hip — the entry points of the attention over a part of the int8 KV cache: under a sliding window with sinks, over
// pages, and with the weight that each key receives added up. See ti_span.h for the visible keys and their rows.
#include "ti_dev.h"
#include "ti_span.h"
#include "ti_token_attn.h"
#include "ti_window_attn.h"

namespace {

constexpr long MASS_SCORES = 1L << 24;       // (query head, slot) scores of a one-token call: half of the partials' scratch
static_assert(2 * MASS_SCORES <= (long)TI_ATTN_ROWSPLITS * TI_ATTN_HD_MAX, "the scores fit");

// Single tokens and up to 8 query rows a KV head take k_token_attn.hip, more k_window_attn.hip. Tokens x query heads of 16
// and 8 KV heads of 128 dims over 2000 keys, the two kernels with their merges: 4 tokens (8 rows) 13.9 / 15.6 us, 8 tokens
// (16 rows) 16.5 / 15.9, over 16000 keys 30.9 / 27.4
bool few_rows(int T, int G) { return T == 1 || T * G <= 8; }

int check_attn(const char* fn, const void* qr, const void* kq, const void* ks, const void* vq, const void* vs, const void* out,
               int n, int nHq, int nKv, int hd) {
    TI_REQUIRE(qr && kq && ks && vq && vs && out, "%s: null buffer", fn);
    TI_REQUIRE(qr != out, "%s: out must not be the queries", fn);
    TI_REQUIRE(n > 0 && nKv > 0 && nHq > 0 && nHq % nKv == 0 && nHq <= TI_ATTN_HEADS_MAX, "%s: bad rows/heads (%d rows, nHq=%d nKv=%d)",
               fn, n, nHq, nKv);
    TI_REQUIRE(hd > 0 && hd % 32 == 0 && hd <= TI_ATTN_HD_MAX, "%s: hd must be a multiple of 32 and <= %d", fn, TI_ATTN_HD_MAX);
    TI_REQUIRE(ti_al16(kq) && ti_al16(vq), "%s: kq/vq must be 16-byte aligned", fn);
    TI_REQUIRE_DENSE(fn, kq);
    TI_REQUIRE_DENSE(fn, vq);
    return TI_OK;
}

}  // namespace

extern "C" int ti_attn_window_q8(ti_ctx* c, const float* qr, const uint32_t* kq, const float* ks, const uint32_t* vq, const float* vs,
                                 float* out, int T, int pos0, int nHq, int nKv, int hd, int window, int sinks) {
    TI_CHECK_CTX(c);
    const int rc = check_attn("ti_attn_window_q8", qr, kq, ks, vq, vs, out, T, nHq, nKv, hd);
    if (rc) return rc;
    TI_REQUIRE(pos0 >= 0 && pos0 <= TI_POS_END - T && sinks >= 0, "ti_attn_window_q8: bad positions (T=%d pos0=%d sinks=%d)", T, pos0, sinks);
    TI_REQUIRE((long)T * nHq <= 0x7fffffffL / 256, "ti_attn_window_q8: %d x %d query rows in one call", T, nHq);
    if (few_rows(T, nHq / nKv)) {
        const TiTokenAttn p = {qr, reinterpret_cast<const uint8_t*>(kq), ks, reinterpret_cast<const uint8_t*>(vq), vs, out,
                               TiPages{nullptr, 0, 0, 0}, nullptr, 1, T, pos0, nHq, nKv, window, sinks, 0, nullptr, nullptr, 0};
        return ti_token_attn_launch(c, p, hd);
    }
    const TiWindowAttn p = {qr, reinterpret_cast<const uint8_t*>(kq), ks, reinterpret_cast<const uint8_t*>(vq), vs, out,
                            T, pos0, nHq, nKv, window, sinks};
    return ti_window_attn_launch(c, p, hd);
}

extern "C" int ti_attn_paged_q8(ti_ctx* c, const float* qr, const uint32_t* kq, const float* ks, const uint32_t* vq, const float* vs,
                                const int32_t* table, const int32_t* lens, float* out, int B, int nHq, int nKv, int hd, int page,
                                int pages, int width, int window, int sinks) {
    TI_CHECK_CTX(c);
    const int rc = check_attn("ti_attn_paged_q8", qr, kq, ks, vq, vs, out, B, nHq, nKv, hd);
    if (rc) return rc;
    TI_REQUIRE(table && lens, "ti_attn_paged_q8: null table or lengths");
    TI_REQUIRE(B <= TI_TOKEN_SEQS, "ti_attn_paged_q8: %d sequences > %d", B, TI_TOKEN_SEQS);
    TI_REQUIRE(ti_pow2(page) && pages > 0 && width > 0 && (long)page * width <= TI_POS_END,
               "ti_attn_paged_q8: bad pages (length %d, a power of two; %d of them; table width %d)", page, pages, width);
    TI_REQUIRE(sinks >= 0, "ti_attn_paged_q8: sinks = %d", sinks);
    const long all = (long)page * width, keys = window < 0 ? all : ti_min(all, (long)window + sinks + 1);
    const TiTokenAttn p = {qr, reinterpret_cast<const uint8_t*>(kq), ks, reinterpret_cast<const uint8_t*>(vq), vs, out,
                           TiPages{table, ti_log2(page), pages, width}, lens, B, 1, 0, nHq, nKv, window, sinks, keys, nullptr, nullptr, 0};
    return ti_token_attn_launch(c, p, hd);
}

extern "C" int ti_attn_mass_q8(ti_ctx* c, const float* qr, const uint32_t* kq, const float* ks, const uint32_t* vq, const float* vs,
                               float* out, float* mass, int T, int pos0, int nHq, int nKv, int hd) {
    TI_CHECK_CTX(c);
    const int rc = check_attn("ti_attn_mass_q8", qr, kq, ks, vq, vs, out, T, nHq, nKv, hd);
    if (rc) return rc;
    TI_REQUIRE(mass, "ti_attn_mass_q8: null mass");
    TI_REQUIRE(pos0 >= 0 && pos0 <= TI_POS_END - T, "ti_attn_mass_q8: bad positions (T=%d pos0=%d)", T, pos0);
    TI_REQUIRE((long)T * nHq <= TI_ATTN_ROWS_MAX, "ti_attn_mass_q8: T*nHq = %ld > %d", (long)T * nHq, TI_ATTN_ROWS_MAX);
    TI_REQUIRE(T > 1 || (long)nHq * ((pos0 + 32L) / 32 * 32) <= MASS_SCORES, "ti_attn_mass_q8: %d heads over %d slots exceed the scratch (%ld scores)",
               nHq, pos0 + 1, MASS_SCORES);
    const uint8_t *k8 = reinterpret_cast<const uint8_t*>(kq), *v8 = reinterpret_cast<const uint8_t*>(vq);
    if (T > 1) return ti_mass_attn_launch(c, TiWindowAttn{qr, k8, ks, v8, vs, out, T, pos0, nHq, nKv, -1, 0}, hd, mass);
    // the scores go to the upper half of the partials' scratch
    const TiTokenAttn t = {qr, k8, ks, v8, vs, out, TiPages{nullptr, 0, 0, 0}, nullptr, 1, 1, pos0, nHq, nKv, -1, 0, 0, mass,
                           c->attn_po + MASS_SCORES, (pos0 + 32L) / 32 * 32};
    return ti_token_attn_launch(c, t, hd);
}
