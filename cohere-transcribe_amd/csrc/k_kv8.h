// k_kv8.h — what the kernels of the 8-bit cache share.
#pragma once
#include "ct_dev.h"

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Exponent of the smallest scale a page may have (all-zero pages get it).
#define KV8_MIN_EXP (-100)
