// ti_token_attn.h — the launch of k_token_attn.hip, used by the entry points of k_span_attn.hip.
#pragma once
#include "ti_internal.h"
#include "ti_span.h"

constexpr int TI_TOKEN_SEQS = 2048;          // sequences of one call, at most: of 64 heads, half of the partials' slots

struct TiTokenAttn {
    const float* qr;                         // [B][T][nHq][hd]
    const uint8_t* kq;
    const float* ks;
    const uint8_t* vq;
    const float* vs;
    float* out;
    TiPages pg;
    const int32_t* lens;                     // keys of each sequence (pages); else the one sequence's queries are at pos0 ..
    int B, T, pos0, nHq, nKv, window, sinks;
    long max_keys;                           // of a sequence over pages: keys that its query can see, at most
    float* mass;                             // of one token of one sequence: mass[j nKv + h] (+)= the weights of key j, or nullptr
    float* scores;                           // [nHq][sstride] room for its scores in log2
    long sstride;
};
int ti_token_attn_launch(ti_ctx* c, const TiTokenAttn& p, int hd);
