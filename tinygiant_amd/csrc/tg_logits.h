/*
 * tg_logits.h -- adjustments of logits before a token is chosen (internal
 * launch interface).
 */
#ifndef TG_LOGITS_H
#define TG_LOGITS_H
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#define LOGITS_MAX_ROWS 65535   /* a row is a grid's y */
#define LOGITS_MAX_VOCAB (1 << 24)

namespace tg {

struct LogitsArgs {
    const float *logits;      /* [k][nrows] */
    float *out;               /* may be logits, may be null */
    int k, nrows;
    const int32_t *hist;      /* [k][hist_stride] */
    int hist_stride;
    const int32_t *hist_len, *gen_start;
    const float *pen;         /* [k][3] repetition, frequency, presence */
    const int32_t *bias_tok;  /* [k][bias_stride] */
    const float *bias_val;
    int bias_stride;
    const int32_t *bias_len;
    const uint32_t *allow;    /* [k][allow_stride] bits; stride 0: one row for all */
    int allow_stride;
    int32_t *argmax;
    float *maxval;
};
size_t logits_scratch(int k, int nrows);
void launch_logits_adjust(const LogitsArgs &a, void *scratch, hipStream_t st);

}  // namespace tg
#endif
