/*
 * tg_paged.h -- 8-bit caches in pages, and rotary positions (internal launch
 * interface).
 */
#ifndef TG_PAGED_H
#define TG_PAGED_H
#include "tg_prompt.h"

#define PAGE_BLOCK 16          /* positions of a head that share a power of two */
#define PAGE_MAX 1024          /* positions of a page: a power of two from 16 on */
#define PAGE_EXP_MIN (-42)     /* exponents of a block; held as a byte, + 127 */
#define PAGE_EXP_MAX 42
#define PAGE_EXP_NAN 255       /* a block that took in a value that is not finite */
#define ROPE_MAX_PAIRS 128

namespace tg {

/* Pages [n_pages][n_kv][size][head_dim] of signed bytes, bytes of exponents
 * [n_pages][n_kv][size / 16], and each sequence's pages in order
 * table[s * stride ..]; an entry that is no page stands for none. */
struct Pages {
    int8_t *k, *v;
    uint8_t *ek, *ev;
    const int32_t *table;
    int n_pages, stride;
    int shift;              /* size = 16 << shift */
};

struct Turn {
    const float *cos, *sin;   /* [len][dim / 2]; null: none */
    int len, dim;             /* the first dim values of a head are turned */
    bool inter;               /* pairs (2 i, 2 i + 1); else (i, i + dim / 2) */
};

struct PagedAppendArgs {
    const float *q, *k, *v;
    int q_stride, kv_stride;
    const float *q_norm, *k_norm;
    float eps;
    Turn turn;
    PackedSeqs s;
    Pages pages;
    int n_heads, n_kv, head_dim;
    float *q_out;
    int q_out_stride;
};
void launch_paged_append(const PagedAppendArgs &a, hipStream_t st);

struct PagedReadArgs {
    Pages pages;
    const int32_t *len, *slot;   /* [n] */
    int n, n_kv, head_dim;
    void *k, *v;                 /* [n_slots][n_kv][kv_max][head_dim] */
    int n_slots, kv_max;
    int most;                    /* positions that fit both a slot and a row of the table */
};
void launch_paged_read(const PagedReadArgs &a, bool half, hipStream_t st);

/* a.kv_k, a.kv_v and the prefix are not used; a.s.kv_max bounds the sequences'
 * positions.  scratch: attention_paged_need(a) bytes, 16-byte aligned */
void launch_attention_paged(const PromptArgs &a, const Pages &pages, void *scratch, hipStream_t st);
size_t attention_paged_need(const PromptArgs &a);
size_t attention_paged_scratch(int n_rows, int n_seqs, int n_heads, int n_kv, int head_dim, int kv_max);

struct RopeTablesArgs {
    float *cos, *sin;
    int len, first, pairs;
    float mscale;
    double turns[ROPE_MAX_PAIRS];   /* frequency / (2 pi): turns a position */
};
void launch_rope_tables(const RopeTablesArgs &a, hipStream_t st);

struct RopeArgs {
    const float *x;
    int x_stride;
    const int32_t *pos;
    Turn turn;
    int rows, heads, head_dim;
    float *out;
    int out_stride;
};
void launch_rope(const RopeArgs &a, hipStream_t st);

}  // namespace tg
#endif
