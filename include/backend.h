/* backend.h — the 40-function compute-backend ABI, as exported by the MI355X
 * HIP backend (libct_hip.so).
 *
 * Every prototype below replaces the declaration at the cited line of the
 * reference's backends/backend.h; names, argument order and meaning are the
 * ABI and are kept identical so the unmodified host (transcribe.c, model.h,
 * tests/test_kernels.c) links against this backend.  Contract notes that the
 * reference leaves implicit are stated here.
 *
 * Conventions (all functions):
 *  - Activations are fp32 device pointers carved by the caller out of the
 *    arena returned by backend_arena_alloc.
 *  - Weight pointers are bf16 and point INTO THE HOST blob passed to
 *    backend_weights_upload_blob; the backend translates them by offset.
 *    A non-NULL weight pointer outside that blob is a fatal error.
 *  - Host arrays (tokens, S_dev, active, T_enc, argmax out) are host memory.
 *  - Compute calls are asynchronous on the calling thread's stream; htod,
 *    dtoh, arena_free and argmax_batch synchronise.
 *  - All mutable state is thread-local: each thread calls backend_init(dev)
 *    and, before exiting, backend_thread_cleanup().
 *  - Errors print a message to stderr and exit(1); nothing returns codes.
 */
#ifndef CT_BACKEND_H
#define CT_BACKEND_H

#include "model_types.h"
#include <stdint.h>
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- Lifecycle (backends/backend.h:20-30) ---- */
void  backend_init(int device_id);                        /* backend.h:20 */
void  backend_destroy(void);                              /* backend.h:21 */
int   backend_num_devices(void);                          /* backend.h:25 */
void  backend_thread_cleanup(void);                       /* backend.h:30 */

/* ---- Weights and memory (backends/backend.h:34-46) ---- */
void  backend_weights_upload_blob(const void *host_base, size_t bytes);  /* :34 */
void *backend_device_ptr(const void *host_ptr);           /* backend.h:38 */
float *backend_arena_alloc(size_t floats);                /* backend.h:41 */
void   backend_arena_free(float *arena);                  /* backend.h:42 */
void backend_htod(float *dev_dst, const float *host_src, size_t floats);  /* :45 */
void backend_dtoh(void *host_dst, const void *dev_src, size_t bytes);     /* :46 */

/* ---- Dense ops (backends/backend.h:52-67) ---- */
void backend_layernorm(float *dst, const float *src,
                       const uint16_t *w, const uint16_t *b, int T, int D);     /* :52 */
void backend_linear(float *y, const float *x,
                    const uint16_t *W, const uint16_t *b, int T, int in_d, int out_d); /* :56 */
void backend_linear_silu(float *y, const float *x,
                         const uint16_t *W, const uint16_t *b, int T, int in_d, int out_d); /* :58 */
void backend_linear_relu(float *y, const float *x,
                         const uint16_t *W, const uint16_t *b, int T, int in_d, int out_d); /* :60 */
/* acc[t] += scale * (W x[t] + b) */
void backend_linear_fmadd(float *acc, float scale, const float *x,
                          const uint16_t *W, const uint16_t *b, int T, int in_d, int out_d); /* :63 */
void backend_add_inplace(float *dst, const float *src, int n);                   /* :67 */

/* ---- Encoder (backends/backend.h:72-86) ---- */
/* mel is (N_MELS, T_mel) with row stride T_mel_stride; writes x_enc (T_enc, ENC_D). */
void backend_encoder_subsampling(const float *mel, int T_mel, int T_mel_stride,
                                 float *x_enc, int T_enc, float *work,
                                 const Weights *W);                               /* :72 */
/* (2T-1, ENC_D) sinusoid table, row p is relative position T-1-p. */
void backend_make_rel_pos_emb(float *pe, int T);                                 /* :77 */
/* x (T, ENC_D) in place: x <- MHSA_relpos(x). */
void backend_rel_pos_mhsa(float *x, const float *pos_emb,
                          int T, const ELayer *L, float *work);                  /* :81 */
/* x (T, ENC_D) in place: pw1 -> GLU -> depthwise(9) -> BN -> SiLU -> pw2. */
void backend_conformer_conv(float *x, int T, const ELayer *L, float *work);     /* :86 */

/* ---- Decoder, prefill / single (backends/backend.h:90-106) ---- */
void backend_sdp_attn(float *out, const float *q, const float *k, const float *v,
                      const float *mask, int T_q, int T_k, float *work);          /* :90 */
void backend_embed(float *h, const int *tokens, int S, int pos_start,
                   const uint16_t *etw, const uint16_t *epw,
                   const uint16_t *elnw, const uint16_t *elnb);                  /* :96 */
void backend_fill_causal_mask(float *mask, int S);                               /* :101 */
void backend_lm_head(float *logits_out, const float *last,
                     const uint16_t *etw, const uint16_t *hdb);                  /* :105 */

/* ---- Graph capture / replay (backends/backend.h:113-138) ---- */
#define GRAPH_TAG_ENCODER    0
#define GRAPH_TAG_PRECOMPUTE 1
#define GRAPH_TAG_DECODER    2
void backend_upload_tokens(const int *host_tokens, int S);                       /* :121 */
/* Replays the graph cached under (tag, T_enc, S, B, current arena); returns 1
 * if one ran, 0 if the caller must run and capture the region. */
int  backend_graph_replay(int tag, int T_enc, int S, int B);                     /* :128 */
void backend_graph_begin_capture(int tag);                                       /* :133 */
/* Instantiates, caches and launches the captured region once. */
void backend_graph_end_capture(int tag, int T_enc, int S, int B);               /* :138 */

/* ---- Device-side sequence counter, batch = 1 (backends/backend.h:147-175) ---- */
void backend_decode_set_S(int n);                                                /* :147 */
void backend_decode_inc_S(void);                                                 /* :152 */
/* cache[(*S - 1) * out_d + j] = (W x + b)[j] */
void backend_linear_to_kvcache(float *cache, const float *x,
                               const uint16_t *W, const uint16_t *b,
                               int in_d, int out_d);                             /* :159 */
/* T_q = 1, T_k = *S, no mask. */
void backend_sdp_attn_devS(float *out, const float *q,
                           const float *k, const float *v, float *work);         /* :166 */
/* Embeds the staged token at position *S - 1, then layer-norms. */
void backend_embed_decode(float *h,
                          const uint16_t *etw, const uint16_t *epw,
                          const uint16_t *elnw, const uint16_t *elnb);           /* :173 */

/* ---- Batched decode step (backends/backend.h:185-228) ---- */
/* Latches S_dev[0..B) as the per-item self-attention lengths used by
 * linear_to_kvcache_batch and sdp_attn_batch_decode_sa.  Rows of inactive
 * items are left unchanged. */
void backend_embed_decode_batch(float *h, const int *tokens,
                                const int *S_dev, const int *active, int B,
                                const uint16_t *etw, const uint16_t *epw,
                                const uint16_t *elnw, const uint16_t *elnb);     /* :185 */
void backend_lm_head_batch(float *logits, const float *h,
                           const uint16_t *etw, const uint16_t *hdb,
                           const int *active, int B);                            /* :192 */
/* First index of the maximum (ties -> lowest id) for each active row; out[b]
 * of inactive rows is left unchanged. */
void backend_argmax_batch(int *out, const float *logits,
                          const int *active, int B);                             /* :198 */
void backend_upload_T_enc(const int *T_enc, int B);                              /* :207 */
void backend_linear_to_kvcache_batch(float *cache, const float *x,
                                     const uint16_t *W, const uint16_t *b,
                                     int B, int cache_seq_stride,
                                     int in_d, int out_d);                       /* :214 */
void backend_sdp_attn_batch_decode_sa(float *out, const float *Q,
                                      const float *K, const float *V,
                                      int T_k_stride, int B, float *work);       /* :223 */
void backend_sdp_attn_batch_decode_ca(float *out, const float *Q,
                                      const float *K, const float *V,
                                      int T_k_stride, int B, float *work);       /* :226 */

/* ---- Beyond the reference ABI ------------------------------------------ */
/* backend_rel_pos_mhsa without the workspace argument, for callers that
 * cannot allocate device memory (code under graph capture, serving loops,
 * harnesses that forbid allocation).  It has no counterpart in the
 * reference.  Its scratch (Q, K, V, P, O: (6T - 1) x ENC_D floats) is a
 * static device array of 11.5 MB per device, held until the process ends,
 * so T must be at most 376 frames (a 30 s clip); larger T prints an error
 * and exits.  Allocates nothing.  Every call on one device uses the same
 * scratch: calls that overlap on one device (other threads, other streams)
 * race.  Same results, bit for bit, as backend_rel_pos_mhsa. */
void backend_rel_pos_mhsa_noalloc(float *x, const float *pos_emb, int T, const ELayer *L);

/* ---- Paged key/value cache in 8 bits ------------------------------------ *
 * The batched decode step above keeps K and V as fp32 rows of MAX_SEQ tokens
 * per item.  The calls below keep them as e4m3 codes (a quarter of the bytes)
 * in pages that sequences take as they grow, share and give back: long texts,
 * grouped heads, beams, streams with a window.  They have no counterpart in
 * the reference.
 *
 * A page holds page_tokens consecutive tokens of one sequence, in every
 * layer, K and V.  Its codes have one scale for each layer and kv head, a
 * power of two (also where a caller fills the arrays itself): value = code *
 * scale, and dividing by the scale is exact, so a value is rounded once.  The
 * cache holds finite values and NaN: what lies beyond 448 scales, infinities
 * included, is stored as +-448 scales.
 *
 * Conventions beside those at the head of this file:
 *  - Every pointer in the structs and every int array argument is DEVICE
 *    memory, and the calls read nothing back: they are asynchronous on the
 *    calling thread's stream, allocate nothing and can be captured in a graph
 *    (backend_kv8_status and the size functions apart).
 *  - Calls on one cache are ordered by the stream they run on; two threads
 *    that share a cache order their calls themselves, and graphs that were
 *    captured over one cache, or one work buffer, do not run at the same time.
 *  - Sizes and pointers that the host sees are checked (errors print and
 *    exit).  Contents of device arrays are checked by the kernels: page ids
 *    outside the pool, rows outside [0, n_rows) and sequence numbers outside
 *    the table are not followed, as each call says. */
typedef struct {
    int layers;          /* layers the pools hold, >= 1                       */
    int pages;           /* pages of each layer's pools, >= 1                 */
    int page_tokens;     /* tokens of a page: 16, 32, 64 or 128               */
    int kv_heads;        /* heads of K and V, 1..256                          */
    int head_dim;        /* 64 or 128                                         */
    int seqs;            /* sequences, rows of the table: 1..256              */
    int table_w;         /* page ids of a table row;
                            table_w * page_tokens <= 2^24                     */
    /* pools [layers][pages][kv_heads][page_tokens][head_dim] of codes
     * (16-byte aligned) and [layers][pages][kv_heads] of scales */
    uint8_t *k, *v;
    float   *kscale, *vscale;
    int *table;          /* [seqs][table_w] page ids; -1: none                */
    int *len;            /* [seqs] tokens held                                */
    int *refs;           /* [pages] table entries that hold the page; 0: free */
    int *rows;           /* [seqs + 1] rows of the step, written by
                            backend_kv8_reserve (may be NULL without it)      */
    int *plan;           /* scratch of the page calls and the status word:
                            backend_kv8_plan_ints ints, zeroed once           */
} BackendKv8;

/* Floats the cache's arrays take together; ints of its plan. */
size_t backend_kv8_floats(const BackendKv8 *c);
size_t backend_kv8_plan_ints(const BackendKv8 *c);
/* Points the arrays into mem (device memory of backend_kv8_floats floats,
 * 16-byte aligned, as backend_arena_alloc gives it) and empties the cache:
 * no pages taken, lengths 0, status 0. */
void backend_kv8_bind(BackendKv8 *c, float *mem);
/* Opens a step: sequence s gets add[s] (>= 0) more tokens.  Writes
 * rows[0..seqs], the prefix sums of add; takes the pages the new tokens need,
 * in the order of sequences, lowest free page first; adds add[s] to len[s].
 * If the pool or a table row has no room, an add[s] is negative or the step
 * has more than 2^24 rows, nothing is taken: rows become all 0, so that the appends and attention of the
 * step do nothing, and the status tells it (KV8_NO_PAGES, KV8_NO_ROOM,
 * KV8_BAD_ARG). */
void backend_kv8_reserve(const BackendKv8 *c, const int *add);
/* Rounds a layer's new K and V rows into their pages.  Sequence s has the
 * rows rows[s] .. rows[s + 1] - 1 (in all at most n_rows, n_rows * kv_heads
 * <= 2^26); they are the last
 * ones of its len[s] tokens.  A row is kv_heads * head_dim values (fp32, or
 * bf16 if bf16 != 0), ld values after the one before it.  The scale of a
 * page is the smallest 2^e >= 2^-100 that holds its largest finite value
 * within 448 scales.  Where a page held tokens already its scale never gets
 * smaller; where it has to grow, those tokens' codes are rounded again (exact
 * but for the smallest values).  Tokens behind the last one are left as they
 * are.  A row whose page is not in the pool, or shared (refs above 1), is
 * skipped; sequences whose rows lie outside [0, n_rows) are skipped. */
void backend_kv8_append(const BackendKv8 *c, int layer, const void *k, const void *v, long ld, int bf16,
                        const int *rows, int n_rows);
typedef struct {
    void *out;           /* [n_rows] rows of heads * head_dim, ld_out apart   */
    const void *q;       /* the same, ld_q apart                              */
    long ld_out, ld_q;   /* in values                                         */
    int bf16;            /* q and out: 0 fp32, 1 bf16                         */
    int heads;           /* query heads, a multiple of kv_heads: head h reads
                            kv head h / (heads / kv_heads)                    */
    float scale;         /* of the scores; 1 / sqrt(head_dim) for this model;
                            positive, at most 2e38                            */
    int causal;          /* 1: a sequence's rows are its last tokens and see
                            the tokens up to their own; 0: they see all       */
    int window;          /* causal only: a row at position p sees p - window
                            + 1 .. p; 0: no limit                             */
    int sinks;           /* with a window: tokens 0 .. sinks - 1 stay visible */
    const int *rows;     /* [seqs + 1] as in backend_kv8_append               */
    int n_rows;          /* rows of q and out; n_rows * heads <= 2^27         */
    int max_rows;        /* no sequence has more rows than this; the rows of
                            one that has more may be left as they are         */
    int max_len;         /* no sequence holds more tokens than this; those
                            past it are not seen; 0: table_w * page_tokens    */
    float *work;         /* backend_kv8_attn_work floats, 16-byte aligned     */
} BackendKv8Attn;
/* Floats of work (0: none, work may be NULL) that are enough for this call
 * and for any with the same cache, heads, window and sinks and no more n_rows,
 * max_rows and max_len, whichever type its rows have.  It depends on the sizes
 * alone, not on the pointers. */
size_t backend_kv8_attn_work(const BackendKv8 *c, const BackendKv8Attn *a);
/* Softmax attention of the rows over a layer's pages: o = sum_j p_j v_j,
 * p = softmax_j(scale * q . k_j) over the tokens the row sees.  A row that
 * sees none gets zeros; tokens on a page that is not in the pool are not
 * seen; what a masked token holds, NaN included, has no effect.  Rows of out
 * that belong to no sequence are left as they are.  Scores, softmax and sums
 * are fp32.  fp32 rows keep fp32 accuracy relative to the largest value that
 * the pages of the tokens a row sees can hold (448 of their scales, which are
 * powers of two from 2^-100 to 2^120), whatever other pages hold.  bf16 rows
 * enter the products as they are, and their weights rounded to f16: by at most
 * 2^-11 of themselves, or 2^-30 of the row's largest where they are smaller
 * than 2^-20 of it (a weight counted with its page's scale).  The sum of the
 * weights is of what they are in fp32. */
void backend_kv8_attn(const BackendKv8 *c, int layer, const BackendKv8Attn *a);
/* Sequences dst[i] become copies of src[i], all n (<= seqs) at once, from
 * what the cache held before the call (beam search: src = each beam's
 * parent).  Full pages are shared; a partly filled last page is copied, in
 * every layer, to the lowest free page, in the order of i.  dst[i]'s earlier
 * pages are given back.  A pair with dst == src changes nothing.  Pages given
 * back by this call are not taken by it, so it needs as many free pages as
 * there are partly filled pages to copy.  If there are fewer, or a sequence
 * number is out of range, or a dst appears twice, nothing changes and the
 * status tells it (KV8_NO_PAGES, KV8_BAD_ARG). */
void backend_kv8_fork(const BackendKv8 *c, const int *dst, const int *src, int n);
/* Gives back the pages of n (<= seqs) sequences and empties them.  Numbers
 * out of range change nothing and set KV8_BAD_ARG; one that appears twice is
 * freed once. */
void backend_kv8_free(const BackendKv8 *c, const int *seqs, int n);
/* Gives back the pages that a causal row with this window (>= 1) and sinks
 * at position len[s] or later does not see; their table entries become -1. */
void backend_kv8_trim(const BackendKv8 *c, int window, int sinks);
/* Moves the pages in use to the front: with m pages in use, those at m and
 * above go, in ascending order, to the free ones below m. */
void backend_kv8_compact(const BackendKv8 *c);
/* Waits for the stream; returns the flags since the last call and clears
 * them. */
#define KV8_NO_PAGES 1
#define KV8_NO_ROOM  2
#define KV8_BAD_ARG  4
int  backend_kv8_status(const BackendKv8 *c);
/* The calling thread's stream (hipStream_t), to order other work with. */
void *backend_stream(void);

#ifdef __cplusplus
}
#endif

#endif /* CT_BACKEND_H */
