/* kv8.c — the backend_kv8_* calls of include/backend.h: argument checks and
 * the cache's memory; the kernels are in k_kv8.hip and k_kv8_attn.hip.
 * Checks come before any device work, so they fire without a GPU too. */
#include "../../include/backend.h"
#include "ct_abi_state.h"
#include "ct_kv8.h"

static void check_sizes(const BackendKv8 *c) {
    if (!c) CT_FATAL("kv8: no cache");
    if (c->layers < 1 || c->layers > 4096) CT_FATAL("kv8: layers outside [1, 4096]");
    if (c->pages < 1 || c->pages > 1 << 24) CT_FATAL("kv8: pages outside [1, 2^24]");
    if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
        CT_FATAL("kv8: page_tokens is not 16, 32, 64 or 128");
    if (c->head_dim != 64 && c->head_dim != 128) CT_FATAL("kv8: head_dim is not 64 or 128");
    if (c->kv_heads < 1 || c->kv_heads > 256) CT_FATAL("kv8: kv_heads outside [1, 256]");
    if (c->seqs < 1 || c->seqs > CT_KV8_SEQS) CT_FATAL("kv8: seqs outside [1, 256]");
    if (c->table_w < 1 || (long)c->table_w * c->page_tokens > CT_KV8_KEYS)
        CT_FATAL("kv8: table_w outside [1, 2^24 / page_tokens]");
}

static void check_cache(const BackendKv8 *c) {
    check_sizes(c);
    if (!c->k || !c->v || !c->kscale || !c->vscale || !c->table || !c->len || !c->refs || !c->plan)
        CT_FATAL("kv8: a pointer of the cache is NULL");
    if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) CT_FATAL("kv8: pools are not 16-byte aligned");
}

static void check_layer(const BackendKv8 *c, int layer) {
    if (layer < 0 || layer >= c->layers) CT_FATAL("kv8: layer outside the cache");
}

static void require_init(void) {
    if (ct_t.dev < 0) CT_FATAL("backend used on a thread that has not called backend_init");
}

void *backend_stream(void) {
    require_init();
    return (void *)ct_t.stream;
}

/* Floats of each array, in the order they are laid out (each rounded up to
 * 16 bytes). */
enum { A_K, A_V, A_KS, A_VS, A_TABLE, A_LEN, A_REFS, A_ROWS, A_PLAN, A_N };

static void arrays(const BackendKv8 *c, size_t n[A_N]) {
    const size_t heads = (size_t)c->layers * c->pages * c->kv_heads;
    n[A_K] = n[A_V] = heads * c->page_tokens * c->head_dim / 4;
    n[A_KS] = n[A_VS] = heads;
    n[A_TABLE] = (size_t)c->seqs * c->table_w;
    n[A_LEN] = (size_t)c->seqs;
    n[A_REFS] = (size_t)c->pages;
    n[A_ROWS] = (size_t)c->seqs + 1;
    n[A_PLAN] = ctk_kv8_plan_ints(c);
    for (int i = 0; i < A_N; i++) n[i] = (n[i] + 3) & ~(size_t)3;
}

size_t backend_kv8_plan_ints(const BackendKv8 *c) {
    check_sizes(c);
    return ctk_kv8_plan_ints(c);
}

size_t backend_kv8_floats(const BackendKv8 *c) {
    check_sizes(c);
    size_t n[A_N], sum = 0;
    arrays(c, n);
    for (int i = 0; i < A_N; i++) sum += n[i];
    return sum;
}

void backend_kv8_bind(BackendKv8 *c, float *mem) {
    check_sizes(c);
    if (!mem || ((uintptr_t)mem & 15)) CT_FATAL("kv8_bind: memory is NULL or not 16-byte aligned");
    require_init();
    size_t n[A_N];
    arrays(c, n);
    float *at[A_N];
    for (int i = 0; i < A_N; i++) {
        at[i] = mem;
        mem += n[i];
    }
    c->k = (uint8_t *)at[A_K];
    c->v = (uint8_t *)at[A_V];
    c->kscale = at[A_KS];
    c->vscale = at[A_VS];
    c->table = (int *)at[A_TABLE];
    c->len = (int *)at[A_LEN];
    c->refs = (int *)at[A_REFS];
    c->rows = (int *)at[A_ROWS];
    c->plan = (int *)at[A_PLAN];
    ctk_kv8_reset(c, ct_t.stream);
}

void backend_kv8_reserve(const BackendKv8 *c, const int *add) {
    check_cache(c);
    if (!add || !c->rows) CT_FATAL("kv8_reserve: add or the cache's rows are NULL");
    require_init();
    ctk_kv8_reserve(c, add, ct_t.stream);
}

static void check_rows(const int *rows, int n_rows) {
    if (!rows) CT_FATAL("kv8: rows are NULL");
    if (n_rows < 0 || n_rows > CT_KV8_ROWS) CT_FATAL("kv8: n_rows outside [0, 2^24]");
}

void backend_kv8_append(const BackendKv8 *c, int layer, const void *k, const void *v, long ld, int bf16,
                        const int *rows, int n_rows) {
    check_cache(c);
    check_layer(c, layer);
    check_rows(rows, n_rows);
    if ((long)n_rows * c->kv_heads > CT_KV8_ROW_HEADS) CT_FATAL("kv8_append: n_rows * kv_heads above 2^26");
    if (n_rows == 0) return;
    const uintptr_t al = bf16 ? 1 : 3;
    if (!k || !v || ((uintptr_t)k & al) || ((uintptr_t)v & al)) CT_FATAL("kv8_append: k or v is NULL or not aligned");
    if (ld < (long)c->kv_heads * c->head_dim) CT_FATAL("kv8_append: ld below kv_heads * head_dim");
    require_init();
    ctk_kv8_append(c, layer, k, v, ld, bf16 != 0, rows, n_rows, ct_t.stream);
}

static void check_attn(const BackendKv8 *c, const BackendKv8Attn *a) {
    if (!a) CT_FATAL("kv8_attn: no arguments");
    if (a->heads < 1 || a->heads > 1 << 16 || a->heads % c->kv_heads)
        CT_FATAL("kv8_attn: heads is not a multiple of kv_heads in [1, 2^16]");
    if (a->n_rows < 0 || a->n_rows > CT_KV8_ROWS || (long)a->n_rows * a->heads > CT_KV8_HEAD_ROWS)
        CT_FATAL("kv8_attn: n_rows outside [0, 2^24] or n_rows * heads above 2^27");
    if (a->max_rows < 1) CT_FATAL("kv8_attn: max_rows < 1");
    if (a->max_len < 0) CT_FATAL("kv8_attn: max_len < 0");
    if (a->window < 0 || a->sinks < 0) CT_FATAL("kv8_attn: window or sinks < 0");
    if (a->window > 0 && !a->causal) CT_FATAL("kv8_attn: a window needs causal rows");
    /* the kernels multiply it by log2(e), which must not overflow */
    if (!(a->scale > 0.0f && a->scale <= 2.0e38f)) CT_FATAL("kv8_attn: scale is not positive and at most 2e38");
}

size_t backend_kv8_attn_work(const BackendKv8 *c, const BackendKv8Attn *a) {
    check_sizes(c);
    check_attn(c, a);
    return ctk_kv8_attn_work(c, a);
}

void backend_kv8_attn(const BackendKv8 *c, int layer, const BackendKv8Attn *a) {
    check_cache(c);
    check_layer(c, layer);
    check_attn(c, a);
    check_rows(a->rows, a->n_rows);
    if (a->n_rows == 0) return;
    const uintptr_t al = a->bf16 ? 1 : 3;
    if (!a->q || !a->out || ((uintptr_t)a->q & al) || ((uintptr_t)a->out & al))
        CT_FATAL("kv8_attn: q or out is NULL or not aligned");
    const long row = (long)a->heads * c->head_dim;
    if (a->ld_q < row || a->ld_out < row) CT_FATAL("kv8_attn: ld_q or ld_out below heads * head_dim");
    if (ctk_kv8_attn_need(c, a) && (!a->work || ((uintptr_t)a->work & 15)))
        CT_FATAL("kv8_attn: work is NULL or not 16-byte aligned");
    require_init();
    ctk_kv8_attn(c, layer, a, ct_t.stream);
}

void backend_kv8_fork(const BackendKv8 *c, const int *dst, const int *src, int n) {
    check_cache(c);
    if (n < 0 || n > c->seqs) CT_FATAL("kv8_fork: n outside [0, seqs]");
    if (n == 0) return;
    if (!dst || !src) CT_FATAL("kv8_fork: dst or src is NULL");
    require_init();
    ctk_kv8_fork(c, dst, src, n, ct_t.stream);
}

void backend_kv8_free(const BackendKv8 *c, const int *seqs, int n) {
    check_cache(c);
    if (n < 0 || n > c->seqs) CT_FATAL("kv8_free: n outside [0, seqs]");
    if (n == 0) return;
    if (!seqs) CT_FATAL("kv8_free: seqs is NULL");
    require_init();
    ctk_kv8_free(c, seqs, n, ct_t.stream);
}

void backend_kv8_trim(const BackendKv8 *c, int window, int sinks) {
    check_cache(c);
    if (window < 1 || sinks < 0) CT_FATAL("kv8_trim: window < 1 or sinks < 0");
    require_init();
    ctk_kv8_trim(c, window, sinks, ct_t.stream);
}

void backend_kv8_compact(const BackendKv8 *c) {
    check_cache(c);
    require_init();
    ctk_kv8_compact(c, ct_t.stream);
}

int backend_kv8_status(const BackendKv8 *c) {
    check_cache(c);
    require_init();
    int flags = 0;
    const int none = 0;
    CHK(hipMemcpyAsync(&flags, c->plan + CT_KV8_STATUS, sizeof flags, hipMemcpyDeviceToHost, ct_t.stream));
    CHK(hipMemcpyAsync(c->plan + CT_KV8_STATUS, &none, sizeof none, hipMemcpyHostToDevice, ct_t.stream));
    CHK(hipStreamSynchronize(ct_t.stream));
    return flags;
}
