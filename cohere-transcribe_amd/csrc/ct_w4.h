/* ct_w4.h — launchers of the linear maps with 4-bit weights (k_w4.hip) and of
 * the logits' penalties and masks (k_logits.hip).  Arguments are checked by
 * w4.c. */
#ifndef CT_W4_H
#define CT_W4_H

#include "../../include/backend.h"
#include <hip/hip_runtime_api.h>

#define CT_W4_TILE_O 16        /* outputs and                                */
#define CT_W4_TILE_I 128       /* inputs of a tile of codes: 1 KB            */

#ifdef __cplusplus
extern "C" {
#endif

void ctk_w4_load(const BackendW4 *w, const uint8_t *codes, const uint16_t *scales, const uint8_t *zeros,
                 hipStream_t s);
void ctk_w4_quantize(const BackendW4 *w, const uint16_t *W, hipStream_t s);
void ctk_w4_unpack(const BackendW4 *w, float *values, hipStream_t s);
void ctk_w4_linear(const BackendW4 *w, const BackendW4Linear *a, hipStream_t s);

int ct_rows_meet(const void *a, size_t lda, size_t wa, const void *b, size_t ldb, size_t wb, long rows);

size_t ctk_logits_work(const BackendLogits *a);
void ctk_logits(const BackendLogits *a, hipStream_t s);

#ifdef __cplusplus
}
#endif
#endif
