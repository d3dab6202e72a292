// ti_window_attn.h — the launches of k_window_attn.hip, used by the entry points of k_span_attn.hip.
#pragma once
#include "ti_internal.h"

struct TiWindowAttn {
    const float* qr;                         // [T][nHq][hd], query t at position pos0 + t
    const uint8_t* kq;
    const float* ks;
    const uint8_t* vq;
    const float* vs;
    float* out;
    int T, pos0, nHq, nKv, window, sinks;
    float* ml;                               // [T nHq][2] (max in log2, sum) of each row, or nullptr
};
int ti_window_attn_launch(ti_ctx* c, const TiWindowAttn& p, int hd);
// mass[j nKv + h] (+)= the weights of key j over the rows, given each row's (max, sum) in p.ml; causal
int ti_mass_columns_launch(ti_ctx* c, const TiWindowAttn& p, int hd, float* mass);
