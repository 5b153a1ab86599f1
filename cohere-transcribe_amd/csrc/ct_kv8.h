/* ct_kv8.h — launchers of the paged 8-bit key/value cache (k_kv8.hip,
 * k_kv8_attn.hip).  Arguments are checked by kv8.c; the kernels check what
 * only the device sees (lengths, page ids, rows). */
#ifndef CT_KV8_H
#define CT_KV8_H

#include "../../include/backend.h"
#include <hip/hip_runtime_api.h>

#define CT_KV8_SEQS 256        /* sequences of a cache                       */
#define CT_KV8_ROWS (1 << 24)  /* rows of a step                             */
#define CT_KV8_ROW_HEADS (1L << 26)  /* appended rows * kv heads, and        */
#define CT_KV8_HEAD_ROWS (1L << 27)  /* rows * query heads: with these the
                                  grids stay below 2^32 threads              */
#define CT_KV8_KEYS (1 << 24)  /* tokens a table row may hold                */

/* Places in BackendKv8.plan, in ints: a header, four ints for each pair of
 * a fork, its staged table rows, then the moved pages and their new places. */
enum {
    CT_KV8_STATUS = 0, /* sticky flags                                       */
    CT_KV8_COUNT = 1,  /* pages to copy                                      */
    CT_KV8_LIVE = 2,   /* pages in use                                       */
    CT_KV8_HEAD = 16
};

#ifdef __cplusplus
extern "C" {
#endif

void ctk_kv8_reset(const BackendKv8 *c, hipStream_t s);
void ctk_kv8_reserve(const BackendKv8 *c, const int *add, hipStream_t s);
void ctk_kv8_append(const BackendKv8 *c, int layer, const void *k, const void *v, long ld, int bf16,
                    const int *rows, int n_rows, hipStream_t s);
void ctk_kv8_fork(const BackendKv8 *c, const int *dst, const int *src, int n, hipStream_t s);
void ctk_kv8_free(const BackendKv8 *c, const int *seqs, int n, hipStream_t s);
void ctk_kv8_trim(const BackendKv8 *c, int window, int sinks, hipStream_t s);
void ctk_kv8_compact(const BackendKv8 *c, hipStream_t s);
size_t ctk_kv8_plan_ints(const BackendKv8 *c);
/* floats a call of these sizes writes; floats for it and any smaller one */
size_t ctk_kv8_attn_need(const BackendKv8 *c, const BackendKv8Attn *a);
size_t ctk_kv8_attn_work(const BackendKv8 *c, const BackendKv8Attn *a);
void ctk_kv8_attn(const BackendKv8 *c, int layer, const BackendKv8Attn *a, hipStream_t s);

#ifdef __cplusplus
}
#endif
#endif
