/*
 * tg_prompt.h -- packed rows of several sequences: cache append and
 * attention (internal launch interface).
 */
#ifndef TG_PROMPT_H
#define TG_PROMPT_H
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

enum { TG_KV_F32 = 0, TG_KV_F16 = 1 };   /* element type of a KV cache */

#define PROMPT_MAX_HEAD_DIM 128   /* head_dim: a multiple of 8, at most this */
#define PROMPT_MAX_GQA 64         /* query heads per KV head, at most this */
#define PROMPT_MAX_KV (1 << 20)   /* kv_max, prefix_max: offsets in one head's rows stay below 2^30 bytes */
#define PROMPT_MAX_ROWS (1 << 22)
#define PROMPT_MAX_STRIDE (1 << 21)   /* floats from row to row: a tile's rows within 2^31 bytes */
#define PROMPT_MAX_SEQS (1 << 16)
/* What a grid holds: 2^32 work-items, of which a row and head take 64 in the
 * combine, a sequence and KV head 256 (one tile of its own). */
#define PROMPT_MAX_ROW_HEADS (1 << 25)
#define PROMPT_MAX_SEQ_HEADS (1 << 20)

namespace tg {

/* Packed rows and where their sequences' caches are.  Rows cu[s] .. cu[s + 1]
 * - 1 belong to sequence s, row cu[s] + i at place len[s] + i of its slot. */
struct PackedSeqs {
    const int32_t *cu;      /* [n + 1] */
    const int32_t *len;     /* [n] rows cached before these; null: 0 */
    const int32_t *slot;    /* [n] cache slot; null: s */
    int n, rows;
    int n_slots, kv_max;
};

struct AppendArgs {
    const float *q, *k, *v;
    int q_stride, kv_stride;
    const float *q_norm, *k_norm;
    float eps;
    const float *rope_cos, *rope_sin;
    int rope_len, base_pos;
    PackedSeqs s;
    void *kv_k, *kv_v;
    int n_heads, n_kv, head_dim;
    float *q_out;
    int q_out_stride;
};
void launch_kv_append(const AppendArgs &a, bool half, hipStream_t st);

struct PromptArgs {
    const float *q;
    int q_stride;
    const void *kv_k, *kv_v;         /* [n_slots][n_kv][kv_max][head_dim] */
    const void *pre_k, *pre_v;       /* [n_kv][pre_max][head_dim] */
    int pre_len, pre_max;            /* positions in front of every sequence */
    PackedSeqs s;
    int window;
    const float *sinks;
    int n_heads, n_kv, head_dim;
    float *out;
    int out_stride;
};
/* scratch: attention_rows_need(a, half) bytes, 16-byte aligned */
void launch_attention_rows(const PromptArgs &a, bool half, void *scratch, hipStream_t st);
size_t attention_rows_need(const PromptArgs &a, bool half);
/* enough for every call of at most these sizes, of any cache type and window */
size_t attention_rows_scratch(int n_rows, int n_seqs, int n_heads, int n_kv, int head_dim, int kv_max, int pre_len);

}  // namespace tg
#endif
