/* w4.c — the backend_w4_*, backend_linear_w4 and backend_logits* calls of
 * include/backend.h: argument checks and memory; the kernels are in k_w4.hip
 * and k_logits.hip.  Checks come before any device work, so they fire without
 * a GPU too. */
#include "../../include/backend.h"
#include "ct_abi_state.h"
#include "ct_w4.h"

static void require_init(void) {
    if (ct_t.dev < 0) CT_FATAL("backend used on a thread that has not called backend_init");
}

/* Whether any of `rows` pieces of wa bytes, lda bytes apart from a on, shares a
 * byte with one of wb bytes, ldb apart from b on (wa <= lda, wb <= ldb). */
int ct_rows_meet(const void *a, size_t lda, size_t wa, const void *b, size_t ldb, size_t wb, long rows) {
    const uintptr_t pa = (uintptr_t)a, pb = (uintptr_t)b;
    const size_t last = (size_t)rows - 1;
    if (pa + last * lda + wa <= pb || pb + last * ldb + wb <= pa) return 0;
    /* one within the other's pitch, as columns of one array are: all pairs of rows
     * at once, else row by row */
    const size_t n = lda == ldb ? 1 : (size_t)rows;
    for (size_t i = 0; i < n; i++) {
        const uintptr_t lo = pa + i * lda, hi = lo + wa;
        /* the first piece of b that ends past lo */
        size_t j = pb + wb > lo ? 0 : (lo - pb - wb) / ldb + 1;
        if (j <= last && pb + j * ldb < hi) return 1;
        if (lda != ldb) continue;
        /* and a's pieces over b's first */
        j = pa + wa > pb ? 0 : (pb - pa - wa) / lda + 1;
        if (j <= last && pa + j * lda < pb + wb) return 1;
    }
    return 0;
}

/* ---- Linear maps with 4-bit weights ---- */
static void check_sizes(const BackendW4 *w) {
    if (!w) CT_FATAL("w4: no weight");
    if (w->in_d < 1 || w->in_d > 1 << 20 || w->out_d < 1 || w->out_d > 1 << 20 ||
        (long)w->in_d * w->out_d > 1L << 31)
        CT_FATAL("w4: in_d or out_d outside [1, 2^20], or their product above 2^31");
    if (w->group != 32 && w->group != 64 && w->group != 128) CT_FATAL("w4: group is not 32, 64 or 128");
    if (w->scale_f16 != 0 && w->scale_f16 != 1) CT_FATAL("w4: scale_f16 is not 0 or 1");
}

static void check_weight(const BackendW4 *w) {
    check_sizes(w);
    if (!w->codes || !w->scales || (((uintptr_t)w->codes | (uintptr_t)w->scales) & 15))
        CT_FATAL("w4: codes or scales are NULL or not 16-byte aligned");
}

static size_t tiles(const BackendW4 *w) {
    return (size_t)((w->out_d + CT_W4_TILE_O - 1) / CT_W4_TILE_O) * ((w->in_d + CT_W4_TILE_I - 1) / CT_W4_TILE_I);
}

static size_t code_words(const BackendW4 *w) { return tiles(w) * (CT_W4_TILE_O * CT_W4_TILE_I / 8); }

size_t backend_w4_floats(const BackendW4 *w) {
    check_sizes(w);
    return code_words(w) + tiles(w) * (CT_W4_TILE_O * CT_W4_TILE_I / w->group);
}

void backend_w4_bind(BackendW4 *w, float *mem) {
    check_sizes(w);
    if (!mem || ((uintptr_t)mem & 15)) CT_FATAL("w4_bind: memory is NULL or not 16-byte aligned");
    w->codes = (uint32_t *)mem;
    w->scales = (uint32_t *)mem + code_words(w);
}

void backend_w4_load(const BackendW4 *w, const uint8_t *codes, const uint16_t *scales, const uint8_t *zeros) {
    check_weight(w);
    if (!codes || !scales || ((uintptr_t)scales & 1)) CT_FATAL("w4_load: codes or scales are NULL or not aligned");
    require_init();
    ctk_w4_load(w, codes, scales, zeros, ct_t.stream);
}

void backend_w4_quantize(const BackendW4 *w, const uint16_t *W) {
    check_weight(w);
    if (!W || ((uintptr_t)W & 1)) CT_FATAL("w4_quantize: the weight is NULL or not aligned");
    require_init();
    ctk_w4_quantize(w, W, ct_t.stream);
}

void backend_w4_unpack(const BackendW4 *w, float *values) {
    check_weight(w);
    if (!values || ((uintptr_t)values & 3)) CT_FATAL("w4_unpack: values are NULL or not aligned");
    require_init();
    ctk_w4_unpack(w, values, ct_t.stream);
}

void backend_linear_w4(const BackendW4 *w, const BackendW4Linear *a) {
    check_weight(w);
    if (!a) CT_FATAL("linear_w4: no arguments");
    if (a->rows < 0 || a->rows > 1 << 24) CT_FATAL("linear_w4: rows outside [0, 2^24]");
    if (a->act < W4_STORE || a->act > W4_ADD) CT_FATAL("linear_w4: unknown act");
    if (a->rows == 0) return;
    const uintptr_t al = a->bf16 ? 1 : 3;
    if (!a->x || !a->y || ((uintptr_t)a->x & al) || ((uintptr_t)a->y & al))
        CT_FATAL("linear_w4: x or y is NULL or not aligned");
    if (a->x == a->y) CT_FATAL("linear_w4: y is x");
    if (a->ld_x < w->in_d || a->ld_y < w->out_d) CT_FATAL("linear_w4: ld_x below in_d or ld_y below out_d");
    const size_t size = a->bf16 ? 2 : 4;
    if (ct_rows_meet(a->x, a->ld_x * size, w->in_d * size, a->y, a->ld_y * size, w->out_d * size, a->rows))
        CT_FATAL("linear_w4: y and x overlap");
    if ((uintptr_t)a->bias & 1) CT_FATAL("linear_w4: bias is not aligned");
    require_init();
    ctk_w4_linear(w, a, ct_t.stream);
}

/* ---- Penalties, biases and masks on logits ---- */
static void check_logits_sizes(const BackendLogits *a) {
    if (!a) CT_FATAL("logits: no arguments");
    if (a->rows < 0 || a->rows > 65535) CT_FATAL("logits: rows outside [0, 65535]");
    if (a->vocab < 1 || a->vocab > 1 << 24) CT_FATAL("logits: vocab outside [1, 2^24]");
}

size_t backend_logits_work(const BackendLogits *a) {
    check_logits_sizes(a);
    return ctk_logits_work(a);
}

static int off4(const void *p) { return ((uintptr_t)p & 3) != 0; }

void backend_logits(const BackendLogits *a) {
    check_logits_sizes(a);
    if (a->rows == 0) return;
    if (!a->logits || off4(a->logits) || off4(a->out) || off4(a->id) || off4(a->score))
        CT_FATAL("logits: logits are NULL or a pointer is not aligned");
    if (!a->out && !a->id && !a->score) CT_FATAL("logits: nothing to write");
    if (a->ld < a->vocab || (a->out && a->ld_out < a->vocab)) CT_FATAL("logits: ld or ld_out below vocab");
    if (a->out == a->logits && a->ld_out != a->ld) CT_FATAL("logits: in place with another ld_out");
    if (off4(a->hist) || off4(a->hist_len) || off4(a->prompt_len) || off4(a->repeat) || off4(a->frequency) ||
        off4(a->presence) || off4(a->ngram))
        CT_FATAL("logits: a pointer of the history or its penalties is not aligned");
    if (a->hist) {
        if (!a->hist_len) CT_FATAL("logits: a history without hist_len");
        if (a->ld_hist < 0 || a->ld_hist > 1 << 24) CT_FATAL("logits: ld_hist outside [0, 2^24]");
    } else if (a->repeat || a->frequency || a->presence || a->ngram) {
        CT_FATAL("logits: penalties without a history");
    }
    if (a->bias_start) {
        if (a->biases < 0) CT_FATAL("logits: biases < 0");
        if (a->biases > 0 && (!a->bias_id || !a->bias)) CT_FATAL("logits: bias_start without bias_id or bias");
        if (off4(a->bias_start) || off4(a->bias_id) || off4(a->bias)) CT_FATAL("logits: a bias pointer is not aligned");
    }
    if (a->mask) {
        if (off4(a->mask) || off4(a->mask_of)) CT_FATAL("logits: mask or mask_of is not aligned");
        if (a->masks < 1 || a->ld_mask < (a->vocab + 31) / 32) CT_FATAL("logits: masks < 1 or ld_mask below vocab / 32");
    }
    if (ctk_logits_work(a) && (!a->work || ((uintptr_t)a->work & 15)))
        CT_FATAL("logits: work is NULL or not 16-byte aligned");
    require_init();
    if (a->out && a->out != a->logits &&
        ct_rows_meet(a->logits, 4 * a->ld, 4 * (size_t)a->vocab, a->out, 4 * a->ld_out, 4 * (size_t)a->vocab, a->rows))
        CT_FATAL("logits: out overlaps the logits without being them");
    ctk_logits(a, ct_t.stream);
}
