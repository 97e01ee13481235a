/*
 * voxtral_b200_serve.h - operators for servers of language models, on device memory of the caller:
 * a key/value cache held in 4 bits (append, attention, eviction by accumulated attention weight) and
 * log probabilities of tokens out of logits. No counterpart in mudler/voxtral-tts.c.
 *
 * Every call returns 0 on success and a negative value on failure, with the reason in
 * vb200_serve_error() (of the calling thread). A call that fails has queued nothing. Calls are queued on `stream` (a cudaStream_t, NULL:
 * the default stream) and return at once; they allocate nothing, wait for nothing and can be captured
 * into graphs. There is no CPU fallback.
 */
#ifndef VOXTRAL_B200_SERVE_H
#define VOXTRAL_B200_SERVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

const char *vb200_serve_error(void);

enum { VB200_F32 = 0, VB200_BF16 = 1, VB200_F16 = 2 };

/* Rows of heads in device memory: element (s, r, h, d) of [seqs][rows][heads][head_dim] lies at
 * data[s * seq + r * row + h * head + d]; strides count elements and may be anything that does not make written elements overlap.
 * data is aligned to its elements. */
typedef struct {
    void *data;
    int type;
    long long seq, row, head;
} vb200_rows_t;

/* ---- the cache ----
 * Keys and values of `seqs` sequences of up to `capacity` tokens. A row of a head is held in blocks of
 * 32 values (OCP microscaling format, MXFP4): a scale 2^e, e = max(floor(log2 largest magnitude) - 2, -126), and 32 codes of
 * 4 bits, each value / 2^e rounded to the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 with its sign (ties to the even code, larger
 * ones to 6). A block with a value that is not finite reads as NaN throughout. (head_dim + head_dim / 16) bytes a token
 * and head, keys and values together, where fp32 takes 8 head_dim.
 *
 * The handle owns the rows and a workspace (up to 30 MB) on the device that was current when it was opened, and is used with that
 * device current. Calls on one handle are made one after another: on one stream, or on streams that events put in order;
 * graphs that hold such calls likewise. Different handles are independent.
 *
 * How many tokens a sequence has is the caller's: lengths (device, [seqs]) counts the tokens in the cache INCLUDING those
 * that the call is about, which are the last ones; rows (device, [seqs], or NULL: max_rows of each) says how many of them are real where
 * sequences have unequal portions. Values of lengths outside [0, capacity] and of rows outside [0, max_rows] count as the nearest
 * in the range. Row r of sequence s, r < rows[s], is token lengths[s] - rows[s] + r; rows that would lie before token 0 are
 * not written by append and read, and see no key. Nothing is written for rows from rows[s] on, and what they hold
 * does not count. */
typedef struct vb200_kv4 vb200_kv4_t;

/* head_dim: 32, 64, 96, 128, 192 or 256; at most 65535 seqs, 16384 kv_heads, 2^30 tokens, 2^40 bytes of rows. */
vb200_kv4_t *vb200_kv4_open(int seqs, int kv_heads, int head_dim, int capacity);
void vb200_kv4_close(vb200_kv4_t *cache);
size_t vb200_kv4_bytes(const vb200_kv4_t *cache);      /* device memory it holds */
/* Waits for the device; 0, or the code of a bounded wait inside the attention kernels that ran out since the last time this was asked (results since
 * then are not to be relied on; later ones are sound again). */
int vb200_kv4_status(const vb200_kv4_t *cache);

typedef struct {
    const int *lengths, *rows;
    int max_rows;
    vb200_rows_t k, v;        /* [seqs][max_rows][kv_heads][head_dim], of one type */
} vb200_kv4_rows_t;

/* k, v into the cache. */
int vb200_kv4_append(vb200_kv4_t *cache, const vb200_kv4_rows_t *a, void *stream);
/* What the cache holds, out into k, v. */
int vb200_kv4_read(const vb200_kv4_t *cache, const vb200_kv4_rows_t *a, void *stream);

/* Causal softmax attention of the portion's rows (whose keys and values have been appended):
 *   out = sum_j softmax_j(scale q . k_j) v_j   over tokens j <= the row's own
 * heads is a multiple of kv_heads; query head h reads KV head h / (heads / kv_heads). A row that sees no key is zeros with
 * lse = -inf. Scores, weights and sums are fp32, keys and values exact: what a row does not see does not reach it, whatever its size. (Where the
 * scales of a head's blocks lie more than 2^36 apart, blocks of zeros aside, the call is exact on a path of its own that takes ten to a hundred times as long.) Queries and
 * weights go through the tensor cores as two FP16 terms each for fp32 (22 bits), queries exactly otherwise, and weights as two terms for fp16,
 * one (11 bits) for bf16: a query's values below 2^-39 (fp32) or 2^-29 of its largest, and weights below 2^-36 of a row's largest, round
 * to steps of about that. Keys of 2^100 and more may pass fp32 on the way to a score.
 * mass_out: the weight that each token of the cache was given, summed over the rows and over the query heads that read
 *   its KV head, added to mass_in (NULL: zeros; the portion's own tokens count as zero there); [seqs][kv_heads][capacity] fp32, may be
 *   mass_in itself; elements from a sequence's length on are left as they were. The same bits on every run. */
typedef struct {
    const int *lengths, *rows;
    int max_rows, heads;
    float scale;
    vb200_rows_t q, out;      /* [seqs][max_rows][heads][head_dim], of one type; they may not overlap */
    float *lse;               /* [seqs][max_rows][heads] natural logarithms of the softmax sums, or NULL; mass_out needs it */
    const float *mass_in;
    float *mass_out;          /* or NULL */
} vb200_kv4_attention_t;

int vb200_kv4_attention(vb200_kv4_t *cache, const vb200_kv4_attention_t *a, void *stream);

/* Sequences of more than `keep` tokens are cut to `keep`, each KV head for itself: the `first` first and the `recent` last
 * tokens stay, and those of the largest mass between them (the earlier one of two that tie; NaN counts as the smallest); their order
 * stays. Shorter sequences stay whole. The rows go into the first slots of `into`: another cache of the same seqs,
 * kv_heads and head_dim, or `cache` itself. What lies behind them there is left as it was. */
typedef struct {
    const int *lengths;
    int *new_lengths;         /* [seqs] min(length, keep); may be lengths itself */
    const float *mass;        /* [seqs][kv_heads][capacity of `cache`] */
    float *new_mass;          /* [seqs][kv_heads][new_mass_ld] of the rows that stayed, or NULL; may be mass itself where `into` is `cache` */
    long long new_mass_ld;    /* at least keep; capacity where new_mass is mass */
    int *kept;                /* [seqs][kv_heads][keep] the token that each row was */
    int keep, recent, first;  /* recent + first <= keep <= capacity of `into` */
} vb200_kv4_evict_t;

int vb200_kv4_evict(vb200_kv4_t *cache, vb200_kv4_t *into, const vb200_kv4_evict_t *a, void *stream);

/* ---- log probabilities ----
 * Of every row of logits [rows][vocab] (row_stride elements apart, aligned to its elements), with natural logarithms:
 *   logprobs[r]      = x[tokens[r]] - lse, lse = log sum exp x; NaN for a token outside [0, vocab)
 *   entropy[r]       = -sum p log p
 *   top_ids[r][i], top_logprobs[r][i]: the `top` largest, largest first, the lower index first where two tie
 * Logits of -inf are tokens of probability 0. A row with NaN or +inf has NaN for logprobs, entropy and top_logprobs (NaN ranks above
 * +inf); one of nothing but -inf has -inf, 0 and -inf. Sums are fp32. Outputs are dense; any of them may be NULL. */
typedef struct {
    const void *logits;
    int type;
    int rows, vocab;
    long long row_stride;
    const int *tokens;        /* device, [rows] */
    float *logprobs, *entropy;
    int top;                  /* 0 .. 32, at most vocab */
    int *top_ids;
    float *top_logprobs;
} vb200_logprobs_t;

int vb200_token_logprobs(const vb200_logprobs_t *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif
