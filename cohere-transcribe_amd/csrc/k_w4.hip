// k_w4.hip — linear maps whose weights are held in 4 bits.
//
//   y[t][o] = act(sum_i s (c - z) x[t][i] + b[o])
//
// with a scale s and a zero point z for each output and group of inputs.
// Layout.  A tile is 16 outputs x 128 inputs, 1 KB: 16 bytes a lane, dword j of
// lane (o, q) = (lane % 16, lane / 16) holds inputs 32 j + 8 q .. + 7 of output
// o, which is the B operand of one 16x16x32 product: value e of the eight in
// bits 4 (e / 2) + 16 (e % 2), so that a mask leaves a pair of them in the low
// bits of two f16.  Each (output, group) has one word: the scale's 16 bits above
// the f16 bits of -(1024 + z).
// Products.  c | 0x6400 is the f16 1024 + c, and adding -(1024 + z) gives c - z
// exactly: two instructions for a pair of weights.  Activations are brought, 128 inputs
// of a row at a time, to a largest value in [2^14, 2^15) by a power of two and
// split into two f16 (bf16 rows are one f16).  A group's products are summed by
// the matrix unit in fp32 and enter the row's sum times the scale.
#include "ct_dev.h"
#include "ct_w4.h"

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int TO = CT_W4_TILE_O, TI = CT_W4_TILE_I;
constexpr int SEGS = 8;          // runs of tiles that a row's inputs are summed in, then joined in order

struct Args {
    const uint32_t *codes, *scales;
    int in_d, out_d, itiles, otiles, per;    // per: tiles of a segment
    int scale_f16;
    void *y;
    const void *x;
    long ld_y, ld_x;
    int rows, act, vec;
    float scale;
    const uint16_t *bias;
};

__device__ __forceinline__ float scale_of(uint32_t word, int f16) {
    if (f16) return (float)__builtin_bit_cast(f16x2, word)[1];
    return __uint_as_float(word & 0xffff0000u);
}

// Eight codes less their zero point (both halves of `less`: -(1024 + z)).
__device__ __forceinline__ f16x8 weights8(uint32_t q, f16x2 less) {
    f16x8 w;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const f16x2 c = __builtin_bit_cast(f16x2, (q >> (4 * p) & 0x000f000fu) | 0x64006400u) + less;
        w[2 * p] = c[0];
        w[2 * p + 1] = c[1];
    }
    return w;
}

__device__ __forceinline__ f16x2 less_of(uint32_t word) {
    return __builtin_bit_cast(f16x2, (word & 0xffffu) | word << 16);
}

// Two values as f16 terms: rounded, and what the rounding left, rounded.
__device__ __forceinline__ void two_terms(float a, float b, f16x2 &hi, f16x2 &lo) {
    float minus = -1.0f;
    asm("" : "+s"(minus));       // a known -1 makes a conversion and a subtraction of the mixed fma
    hi = __builtin_convertvector((f32x2){a, b}, f16x2);
    lo = __builtin_convertvector((f32x2){__builtin_fmaf((float)hi[0], minus, a), __builtin_fmaf((float)hi[1], minus, b)}, f16x2);
}

// The largest of a row of 16 lanes, for each of them.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x122, 0xF, 0xF, false));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x121, 0xF, 0xF, false));
}

// Values k .. k + 7 of row t; zeros past in_d.
template <bool BF16>
__device__ __forceinline__ void fetch8(const Args &a, long t, int k, float (&v)[8]) {
    if constexpr (BF16) {
        const uint16_t *p = reinterpret_cast<const uint16_t *>(a.x) + t * a.ld_x + k;
        if (a.vec && k + 8 <= a.in_d) {
            const u16x8 u = *reinterpret_cast<const u16x8 *>(p);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = bf2f(u[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = k + i < a.in_d ? bf2f(p[i]) : 0.0f;
        }
    } else {
        const float *p = reinterpret_cast<const float *>(a.x) + t * a.ld_x + k;
        if (a.vec && k + 8 <= a.in_d) {
            const f32x4 u = *reinterpret_cast<const f32x4 *>(p), w = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = u[i]; v[4 + i] = w[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = k + i < a.in_d ? p[i] : 0.0f;
        }
    }
}

// A row's 128 inputs, eight in each of its 16 lanes, as f16 terms; returns the
// power of two that undoes theirs.
template <int NB>
__device__ __forceinline__ float split8(const float (&v)[8], f16x8 (&h)[NB]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    // exponent of the largest, at least 15 - 127 so that the factor is in range
    const int e = max((int)(max16(top) >> 23), 15);
    const float up = __uint_as_float((uint32_t)(127 + 14 - (e - 127)) << 23);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const float a = v[i] * up, b = v[i + 1] * up;
        f16x2 hi, lo;
        if (NB > 1) two_terms(a, b, hi, lo);
        else hi = __builtin_convertvector((f32x2){a, b}, f16x2);
#pragma unroll
        for (int n = 0; n < 2; n++) {
            h[0][i + n] = hi[n];
            if (NB > 1) h[NB - 1][i + n] = lo[n];
        }
    }
    return __uint_as_float((uint32_t)(127 - 14 + (e - 127)) << 23);
}

// Where a row's eight inputs 8 k8 .. + 7 lie among a tile's 256 pieces of 16
// bytes: piece k8 * 16 + row, rows changed so that neither the stores of a row
// nor the loads of a product meet in a bank.
__device__ __forceinline__ int piece(int k8, int row) { return k8 * 16 + (row ^ k8); }

// One tile of 16 outputs times 16 rows: the groups' products into the rows' sums.
// A operand x (row = lane % 16), B operand the weights (output = lane % 16);
// lane (o, q) gets rows 4 q + i of output o.
template <int NB, int GS>
__device__ __forceinline__ void tile_product(const u32x4 &code, const uint32_t (&word)[4 / GS], int scale_f16,
                                             const f16x8 (&xf)[NB][4], const f32x4 &undo, f32x4 &sum) {
#pragma unroll
    for (int g = 0; g < 4 / GS; g++) {
        const f16x2 less = less_of(word[g]);
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int j = g * GS; j < (g + 1) * GS; j++) {
            const f16x8 w = weights8(code[j], less);
#pragma unroll
            for (int n = 0; n < NB; n++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[n][j], w, acc, 0, 0, 0);
        }
        const float s = scale_of(word[g], scale_f16);
#pragma unroll
        for (int i = 0; i < 4; i++) sum[i] = __builtin_fmaf(mul_rn(acc[i], s), undo[i], sum[i]);
    }
}

template <int GS>
__device__ __forceinline__ void fetch_words(const uint32_t *p, uint32_t (&word)[4 / GS]) {
#pragma unroll
    for (int g = 0; g < 4 / GS; g++) word[g] = p[g];
}

template <bool BF16>
__device__ __forceinline__ void finish(const Args &a, long t, int o, float v) {
    if (a.bias) v += bf2f(a.bias[o]);
    if (a.act == W4_SILU) v = v * sigmoid_hw(v);
    else if (a.act == W4_RELU) v = v < 0.0f ? 0.0f : v;      // a NaN stays
    if constexpr (BF16) {
        uint16_t *p = reinterpret_cast<uint16_t *>(a.y) + t * a.ld_y + o;
        if (a.act == W4_ADD) v = __builtin_fmaf(a.scale, v, bf2f(*p));
        *p = f2bf(v);
    } else {
        float *p = reinterpret_cast<float *>(a.y) + t * a.ld_y + o;
        if (a.act == W4_ADD) v = __builtin_fmaf(a.scale, v, *p);
        *p = v;
    }
}

// NT tiles of outputs a workgroup, 16 rows at a time; its eight wavefronts each
// take one segment of the inputs and join their sums in LDS, in order.
template <bool BF16, int GS, int NT>
__global__ __launch_bounds__(SEGS * CT_WAVE) void linear_kernel(Args a) {
    constexpr int NB = BF16 ? 1 : 2;
    __shared__ __align__(16) union {
        f16x8 x[SEGS][NB][256];
        float sum[SEGS][NT][16][TO];
    } sh;
    __shared__ __align__(16) float sundo[SEGS][16];
    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE);
    const int c = lane & 15, q = lane >> 4;
    const int ot0 = blockIdx.x * NT;
    const int k0 = w * a.per, k1 = min(k0 + a.per, a.itiles);
    for (long r0 = 16L * blockIdx.y; r0 < a.rows; r0 += 16L * gridDim.y) {
        const int nr = (int)min(16L, a.rows - r0);
        f32x4 sum[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) sum[n] = (f32x4){0, 0, 0, 0};
        for (int kt = k0; kt < k1; kt++) {
            u32x4 code[NT];
            uint32_t word[NT][4 / GS];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const long tile = (long)min(ot0 + n, a.otiles - 1) * a.itiles + kt;
                code[n] = reinterpret_cast<const u32x4 *>(a.codes)[tile * CT_WAVE + lane];
                fetch_words<GS>(a.scales + (tile * 16 + c) * (4 / GS), word[n]);
            }
            for (int r = q; r < nr; r += 4) {
                float v[8];
                f16x8 h[NB];
                fetch8<BF16>(a, r0 + r, kt * TI + 8 * c, v);
                const float undo = split8<NB>(v, h);
#pragma unroll
                for (int n = 0; n < NB; n++) sh.x[w][n][piece(c, r)] = h[n];
                if (c == 0) sundo[w][r] = undo;
            }
            // the wavefront's own part of LDS: its accesses are in order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            f16x8 xf[NB][4];
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) xf[n][j] = sh.x[w][n][piece(4 * j + q, c)];
            const f32x4 undo = *reinterpret_cast<const f32x4 *>(&sundo[w][4 * q]);
#pragma unroll
            for (int n = 0; n < NT; n++) tile_product<NB, GS>(code[n], word[n], a.scale_f16, xf, undo, sum[n]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) sh.sum[w][n][4 * q + i][c] = sum[n][i];
        __syncthreads();
        for (int i = threadIdx.x; i < NT * 256; i += SEGS * CT_WAVE) {
            const int n = i >> 8, r = i >> 4 & 15, o = (ot0 + n) * TO + (i & 15);
            if (r < nr && o < a.out_d) {
                float v = sh.sum[0][n][r][i & 15];
#pragma unroll
                for (int s = 1; s < SEGS; s++) v += sh.sum[s][n][r][i & 15];
                finish<BF16>(a, r0 + r, o, v);
            }
        }
        __syncthreads();
    }
}

// ---- Laying out ----------------------------------------------------------

__device__ __forceinline__ uint32_t word_of(uint16_t scale, int zero) {
    return (uint32_t)scale << 16 | __builtin_bit_cast(uint16_t, (_Float16)(float)(-1024 - zero));
}

// Codes of one tile, a byte each [16][128] in LDS, as its 64 lanes' dwords.
__device__ __forceinline__ void put_tile(const uint8_t (&code)[TO][TI], uint32_t *to) {
    const int i = threadIdx.x;               // dword j of lane l: 4 l + j
    const int j = i & 3, o = (i >> 2) & 15, q = i >> 6;
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) v |= (uint32_t)(code[o][32 * j + 8 * q + e] & 15) << (4 * (e >> 1) + 16 * (e & 1));
    to[i] = v;
}

// A workgroup a tile, 256 threads.
__global__ __launch_bounds__(256) void load_kernel(BackendW4 w, const uint8_t *codes, const uint16_t *scales,
                                                   const uint8_t *zeros, int itiles, long ntiles) {
    __shared__ uint8_t code[TO][TI];
    const int groups = (w.in_d + w.group - 1) / w.group, per = TI / w.group;
    const long ld = (w.in_d + 1) / 2;
    for (long tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
        const int ot = (int)(tile / itiles), it = (int)(tile % itiles);
        for (int i = threadIdx.x; i < TO * TI; i += 256) {
            const int o = ot * TO + i / TI, k = it * TI + i % TI;
            const int b = o < w.out_d && k < w.in_d ? codes[o * ld + k / 2] : 0;
            code[i / TI][i % TI] = (uint8_t)(b >> (4 * (k & 1)));
        }
        if (threadIdx.x < TO * per) {
            const int o = ot * TO + threadIdx.x / per, g = it * per + threadIdx.x % per;
            const bool in = o < w.out_d && g < groups;
            const long at = (long)o * groups + g;
            w.scales[tile * TO * per + threadIdx.x] =
                word_of(in ? scales[at] : 0, in ? (zeros ? zeros[at] & 15 : 8) : 0);
        }
        __syncthreads();
        put_tile(code, w.codes + tile * 256);
        __syncthreads();
    }
}

// A workgroup a tile: 16 threads an output, 8 inputs a thread; a group's
// extremes over its threads.
__global__ __launch_bounds__(256) void quantize_kernel(BackendW4 w, const uint16_t *W, int itiles, long ntiles) {
    __shared__ uint8_t code[TO][TI];
    const int per = TI / w.group, each = 16 / per;       // groups of a tile; threads of a group
    const int t = threadIdx.x & 15, row = threadIdx.x >> 4;
    for (long tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
        const int o = (int)(tile / itiles) * TO + row, k = (int)(tile % itiles) * TI + 8 * t;
        float v[8], lo = 0.0f, hi = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            v[i] = o < w.out_d && k + i < w.in_d ? bf2f(W[(long)o * w.in_d + k + i]) : 0.0f;
            lo = fminf(lo, v[i]);
            hi = fmaxf(hi, v[i]);
        }
        for (int m = 1; m < each; m <<= 1) {
            lo = fminf(lo, __shfl_xor(lo, m, CT_WAVE));
            hi = fmaxf(hi, __shfl_xor(hi, m, CT_WAVE));
        }
        const float want = (hi - lo) / 15.0f;
        uint16_t bits;
        float s;
        if (w.scale_f16) {
            const _Float16 h = (_Float16)fminf(want, 65504.0f);
            bits = __builtin_bit_cast(uint16_t, h);
            s = (float)h;
        } else {
            bits = f2bf(fminf(want, 3.3895313892515355e38f));
            s = bf2f(bits);
        }
        const int z = s > 0.0f ? (int)fminf(fmaxf(rintf(-lo / s), 0.0f), 15.0f) : 0;
#pragma unroll
        for (int i = 0; i < 8; i++)
            code[row][8 * t + i] = s > 0.0f && k + i < w.in_d ? (uint8_t)fminf(fmaxf(rintf(v[i] / s) + (float)z, 0.0f), 15.0f) : 0;
        if (t % each == 0) w.scales[(tile * TO + row) * per + t / each] = word_of(bits, z);
        __syncthreads();
        put_tile(code, w.codes + tile * 256);
        __syncthreads();
    }
}

__global__ __launch_bounds__(256) void unpack_kernel(BackendW4 w, float *values, int itiles, long ntiles) {
    const int per = TI / w.group;
    for (long tile = blockIdx.x; tile < ntiles; tile += gridDim.x) {
        const int i = threadIdx.x, j = i & 3, row = (i >> 2) & 15, q = i >> 6;
        const int o = (int)(tile / itiles) * TO + row, k = (int)(tile % itiles) * TI + 32 * j + 8 * q;
        const uint32_t v = w.codes[tile * 256 + i], word = w.scales[(tile * TO + row) * per + (32 * j + 8 * q) / w.group];
        const float s = scale_of(word, w.scale_f16), less = (float)less_of(word)[0] + 1024.0f;
        if (o < w.out_d)
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (k + e < w.in_d)
                    values[(long)o * w.in_d + k + e] = s * ((float)(v >> (4 * (e >> 1) + 16 * (e & 1)) & 15) + less);
    }
}

int itiles_of(const BackendW4 *w) { return (w->in_d + TI - 1) / TI; }
int otiles_of(const BackendW4 *w) { return (w->out_d + TO - 1) / TO; }
unsigned blocks_of(long ntiles) { return (unsigned)(ntiles < 65536 ? ntiles : 65536); }

}  // namespace

extern "C" void ctk_w4_load(const BackendW4 *w, const uint8_t *codes, const uint16_t *scales, const uint8_t *zeros,
                            hipStream_t s) {
    const long n = (long)itiles_of(w) * otiles_of(w);
    hipLaunchKernelGGL(load_kernel, dim3(blocks_of(n)), dim3(256), 0, s, *w, codes, scales, zeros, itiles_of(w), n);
}

extern "C" void ctk_w4_quantize(const BackendW4 *w, const uint16_t *W, hipStream_t s) {
    const long n = (long)itiles_of(w) * otiles_of(w);
    hipLaunchKernelGGL(quantize_kernel, dim3(blocks_of(n)), dim3(256), 0, s, *w, W, itiles_of(w), n);
}

extern "C" void ctk_w4_unpack(const BackendW4 *w, float *values, hipStream_t s) {
    const long n = (long)itiles_of(w) * otiles_of(w);
    hipLaunchKernelGGL(unpack_kernel, dim3(blocks_of(n)), dim3(256), 0, s, *w, values, itiles_of(w), n);
}

extern "C" void ctk_w4_linear(const BackendW4 *w, const BackendW4Linear *p, hipStream_t s) {
    Args a;
    a.codes = w->codes; a.scales = w->scales;
    a.in_d = w->in_d; a.out_d = w->out_d;
    a.itiles = itiles_of(w); a.otiles = otiles_of(w);
    a.per = (a.itiles + SEGS - 1) / SEGS;
    a.scale_f16 = w->scale_f16;
    a.y = p->y; a.x = p->x; a.ld_y = p->ld_y; a.ld_x = p->ld_x;
    a.rows = p->rows; a.act = p->act; a.scale = p->scale; a.bias = p->bias;
    a.vec = ((uintptr_t)p->x & 15) == 0 && p->ld_x % (p->bf16 ? 8 : 4) == 0;
    const long rt = ((long)p->rows + 15) / 16;
    const dim3 grid((unsigned)a.otiles, (unsigned)(rt < 4096 ? rt : 4096));
#define LINEAR(B, GS) hipLaunchKernelGGL((linear_kernel<B, GS, 1>), grid, dim3(SEGS * CT_WAVE), 0, s, a)
    if (p->bf16) {
        if (w->group == 32) LINEAR(true, 1);
        else if (w->group == 64) LINEAR(true, 2);
        else LINEAR(true, 4);
    } else {
        if (w->group == 32) LINEAR(false, 1);
        else if (w->group == 64) LINEAR(false, 2);
        else LINEAR(false, 4);
    }
#undef LINEAR
}
