// ti_window_attn.h — the launches of k_window_attn.hip, used by the entry points of k_span_attn.hip.
#pragma once
#include "ti_internal.h"

// What the columns' sums of a call's weights need of its query rows, in tiles of 16 rows of a KV head: the MFMA operands
// [KV head][tile][hi, lo][group][lane] and of each row its score factor, maximum in log2, 1 / sum and position (rows behind
// the last: weights of 0). op = nullptr: not kept
struct TiMassRows {
    ti_h8* op;
    float4* row;
    int tiles;
};
struct TiWindowAttn {
    const float* qr;                         // [T][nHq][hd], query t at position pos0 + t
    const uint8_t* kq;
    const float* ks;
    const uint8_t* vq;
    const float* vs;
    float* out;
    int T, pos0, nHq, nKv, window, sinks;
};
int ti_window_attn_launch(ti_ctx* c, const TiWindowAttn& p, int hd);
// causal attention, and mass[j nKv + h] (+)= the weights of key j over the rows; T nHq <= TI_ATTN_ROWS_MAX
int ti_mass_attn_launch(ti_ctx* c, const TiWindowAttn& p, int hd, float* mass);
