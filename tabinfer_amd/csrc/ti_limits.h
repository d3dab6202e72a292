// ti_limits.h — capacities of the attention's scratch (ti_ctx), which other calls borrow. Plain C++.
#pragma once

#define TI_ATTN_HEADS_MAX 64
#define TI_ATTN_ROWS_MAX 4096     // T * nHq of one attention call (a 256-token prefill of 16 heads)
#define TI_ATTN_SPLITS_MAX 512
#define TI_ATTN_ROWSPLITS (512 * 512)   // (T * nHq) x splits of one call: the partials' capacity
#define TI_ATTN_HD_MAX 128
