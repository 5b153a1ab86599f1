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
// the f16 bits of -(2^-1 + z 2^-11).
// Products.  c | 0x3800 is the f16 2^-1 + c 2^-11, and adding -(2^-1 + z 2^-11)
// gives (c - z) 2^-11 exactly: 9 instructions for 8 weights.  Activations are
// brought, 128 inputs of a row at a time, to a largest value in [2^14, 2^15) by a
// power of two and split into two f16 (bf16 rows are one f16): 22 bits of each
// fp32 input stay.  A group's products are summed by the matrix unit in fp32,
// brought back by the power of two and enter the row's sum times the scale, in
// that order: with the weights' 2^-11, 128 times 15 times the largest float is
// within fp32's range, so nothing is infinite before the result is, whatever the
// sizes of inputs and scales.  The sums are brought back from the 2^-11 at the end.
// A row's inputs are summed in SEGS runs of tiles that are joined in order, in
// every kernel here, so that a row's answer does not depend on how many rows the
// call has.
//
// What bounds them.  One row of a small map: the launch and one pass of loads
// (1024 -> 1024, 0.55 MB: 3.8 us, where a call of one workgroup takes 3.6).  Few rows
// of large maps: the codes' bytes (1 x 8192 -> 24576, 106 MB: 22.5 us, 4.7 TB/s).
// Many rows: vector instructions that prepare both operands and the products, which
// take turns (752 x 1280 -> 5120: 32 us, 308 Tflop/s of them, twice that of f16 terms;
// 48% and 29% of the SIMDs' time).
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
    uint32_t scale_f16;
    void *y;
    const void *x;
    long ld_y, ld_x;
    int rows, act;
    float scale;
    const uint16_t *bias;
};

// f16: all ones for f16 scales, 0 for bf16.  A choice, not a branch: branches
// among the products took twice the registers.
__device__ __forceinline__ float scale_of(uint32_t word, uint32_t f16) {
    const uint32_t h = __float_as_uint((float)__builtin_bit_cast(f16x2, word)[1]);
    return __uint_as_float((h & f16) | (word & 0xffff0000u & ~f16));
}

// A zero point as it is taken off: -(2^-1 + z 2^-11) and -(2^-5 + z 2^-11), in both halves.
struct Less {
    f16x2 low, high;
};
__device__ __forceinline__ Less less_of(uint32_t word) {
    const f16x2 low = __builtin_bit_cast(f16x2, (word & 0xffffu) | word << 16);
    return {low, low + (f16x2){0.46875, 0.46875}};
}

// Eight codes less their zero point, times 2^-11.  A code in the low four bits of a
// f16 2^-1 makes it 2^-1 + c 2^-11, in the next four of a 2^-5 2^-5 + c 2^-11: one
// shift and four masks a dword (a shift a pair took 15 instructions where this takes 9).
__device__ __forceinline__ f16x8 weights8(uint32_t q, const Less &less) {
    // constants in registers: one instruction takes a mask and a constant only so
    uint32_t m0 = 0x000f000fu, m1 = 0x00f000f0u, one = 0x38003800u, two = 0x28002800u;
    asm("" : "+s"(m0), "+s"(m1), "+v"(one), "+v"(two));
    u32x4 w;                     // whole registers: halves set one by one took twice as many
#pragma unroll
    for (int p = 0; p < 2; p++) {
        const uint32_t x = p ? q >> 8 : q;
        w[2 * p] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, (x & m0) | one) + less.low);
        w[2 * p + 1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, (x & m1) | two) + less.high);
    }
    return __builtin_bit_cast(f16x8, w);
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

// pieces of a row, which need not lie on 16 bytes
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t u16x8u __attribute__((ext_vector_type(8), aligned(2)));

// Input k of row t.
template <bool BF16>
__device__ __forceinline__ const char *input_at(const Args &a, long t, int k) {
    return reinterpret_cast<const char *>(a.x) + (t * a.ld_x + k) * (BF16 ? 2 : 4);
}

// Eight inputs from p on, of a tile that ends before in_d.
template <bool BF16>
__device__ __forceinline__ void fetch8(const char *x, float (&v)[8]) {
    if constexpr (BF16) {
        const u16x8u u = *reinterpret_cast<const u16x8u *>(x);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = bf2f(u[i]);
    } else {
        const float *p = reinterpret_cast<const float *>(x);
        const f32x4u u = *reinterpret_cast<const f32x4u *>(p), w = *reinterpret_cast<const f32x4u *>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; i++) { v[i] = u[i]; v[4 + i] = w[i]; }
    }
}

// The same of a row's last tile, zeros after the first `n`; those take the row's last
// input's place, so that all loads are in flight at once (64 x 1000 -> 4096: 6.8 us, one
// after another 8.9).
template <bool BF16>
__device__ __forceinline__ void fetch_last8(const char *x, int n, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int at = min(i, n - 1);
        if constexpr (BF16) v[i] = bf2f(reinterpret_cast<const uint16_t *>(x)[at]);
        else v[i] = reinterpret_cast<const float *>(x)[at];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = i < n ? v[i] : 0.0f;
}

// A row's 128 inputs, eight in each of its 16 lanes, as f16 terms; returns the
// power of two that undoes theirs.
template <int NB>
__device__ __forceinline__ float split8(const float (&v)[8], f16x8 (&h)[NB]) {
    // a NaN is no largest value: it stays one without
    float big = fmaxf(fabsf(v[0]), fabsf(v[1]));
#pragma unroll
    for (int i = 2; i < 8; i++) big = fmaxf(big, fabsf(v[i]));
    const uint32_t top = __float_as_uint(big);
    // exponent of the largest, at least 15 - 127 so that the factor is in range
    const int e = max((int)(max16(top) >> 23), 15);
    const float up = __uint_as_float((uint32_t)(127 + 14 - (e - 127)) << 23);
    u32x4 t[NB];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float a = v[2 * i] * up, b = v[2 * i + 1] * up;
        f16x2 hi, lo = {0, 0};
        if (NB > 1) two_terms(a, b, hi, lo);
        else hi = __builtin_convertvector((f32x2){a, b}, f16x2);
        t[0][i] = __builtin_bit_cast(uint32_t, hi);
        if (NB > 1) t[NB - 1][i] = __builtin_bit_cast(uint32_t, lo);
    }
#pragma unroll
    for (int n = 0; n < NB; n++) h[n] = __builtin_bit_cast(f16x8, t[n]);
    return __uint_as_float((uint32_t)(127 - 14 + (e - 127)) << 23);
}

// Where a row's eight inputs 8 k8 .. + 7 lie among a tile's pieces of 16 bytes:
// piece k8 * 16 + row, rows changed so that neither the stores of a row nor the
// loads of a product meet in a bank.
__device__ __forceinline__ int piece(int k8, int row) { return k8 * 16 + (row ^ k8); }

// One tile of 16 outputs times 16 rows: the groups' products into the rows' sums.
// A operand x (row = lane % 16), B operand the weights (output = lane % 16);
// lane (o, q) gets rows 4 q + i of output o.
template <int NB, int GS>
__device__ __forceinline__ void tile_product(const u32x4 &code, const uint32_t (&word)[4 / GS], uint32_t scale_f16,
                                             const f16x8 (&xf)[NB][4], const f32x4 &undo, f32x4 &sum) {
#pragma unroll
    for (int g = 0; g < 4 / GS; g++) {
        const Less less = less_of(word[g]);
        f32x4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int j = g * GS; j < (g + 1) * GS; j++) {
            const f16x8 w = weights8(code[j], less);
#pragma unroll
            for (int n = 0; n < NB; n++) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[n][j], w, acc, 0, 0, 0);
        }
        const float s = scale_of(word[g], scale_f16);
#pragma unroll
        for (int i = 0; i < 4; i++) sum[i] = __builtin_fmaf(acc[i] * undo[i], s, sum[i]);
    }
}

template <bool BF16>
__device__ __forceinline__ void finish(const Args &a, long t, int o, float v) {
    v *= 0x1p11f;                            // the weights' 2^-11
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

// Work of a round or few: NT tiles of outputs a workgroup, 16 rows at a time; its
// eight wavefronts each take one segment of the inputs, split them a tile at a time
// and join their sums in LDS, in order.  A wavefront has AHEAD tiles of codes and
// inputs in flight, or, of four tiles together, asks for each operand of the next
// one as this one leaves its registers (two whole sets spill).  64 x 1024 -> 4096:
// 6.1 us, bound by the chain of loads, split, products and join; 64 x 4096 -> 4096
// 13.6: vector instructions, most of which make operands of codes and inputs, take
// 55% of the SIMDs' time and products 13%, and wavefronts wait 41% of theirs.
template <bool BF16, int GS, int NT>
__global__ __launch_bounds__(SEGS * CT_WAVE, 2) void linear_kernel(Args a) {
    constexpr int NB = BF16 ? 1 : 2, RR = 16, RI = RR / 4, AHEAD = NT == 4 ? 1 : 2;
    __shared__ __align__(16) union {
        f16x8 x[SEGS][NB][16 * RR];
        float sum[SEGS][NT][RR][TO];
    } sh;
    __shared__ __align__(16) float sundo[SEGS][RR];
    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE);
    const int c = lane & 15, q = lane >> 4;
    const int k0 = w * a.per, k1 = min(k0 + a.per, a.itiles);
    struct Ahead {
        u32x4 code[NT];
        uint32_t word[NT][4 / GS];
        float v[RI][8];
    };
    for (long r0 = (long)RR * blockIdx.y; r0 < a.rows; r0 += (long)RR * gridDim.y) {
        const int nr = (int)min((long)RR, a.rows - r0);
        f32x4 sum[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) sum[n] = (f32x4){0, 0, 0, 0};
        Ahead t[AHEAD];
        auto fetch_w = [&](int kt, int n, Ahead &f) __attribute__((always_inline)) {
            const long tile = (long)min((int)blockIdx.x * NT + n, a.otiles - 1) * a.itiles + kt;
            f.code[n] = reinterpret_cast<const u32x4 *>(a.codes)[tile * CT_WAVE + lane];
#pragma unroll
            for (int g = 0; g < 4 / GS; g++) f.word[n][g] = a.scales[(tile * 16 + c) * (4 / GS) + g];
        };
        auto fetch_x = [&](int kt, Ahead &f) __attribute__((always_inline)) {
            if (kt * TI + TI <= a.in_d)
#pragma unroll
                for (int i = 0; i < RI; i++)
                    if (q + 4 * i < nr) fetch8<BF16>(input_at<BF16>(a, r0 + q + 4 * i, kt * TI + 8 * c), f.v[i]);
        };
        // what the tile leaves takes the one AHEAD of it at once (past the last one: that again)
        auto use = [&](int kt, Ahead &f) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < RI; i++) {
                const int r = q + 4 * i;
                if (r < nr) {
                    f16x8 h[NB];
                    if (kt * TI + TI > a.in_d)
                        fetch_last8<BF16>(input_at<BF16>(a, r0 + r, kt * TI + 8 * c), a.in_d - kt * TI - 8 * c, f.v[i]);
                    const float undo = split8<NB>(f.v[i], h);
#pragma unroll
                    for (int n = 0; n < NB; n++) sh.x[w][n][piece(c, r)] = h[n];
                    if (c == 0) sundo[w][r] = undo;
                }
            }
            const int next = min(kt + AHEAD, k1 - 1);
            fetch_x(next, f);
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
            for (int n = 0; n < NT; n++) {
                tile_product<NB, GS>(f.code[n], f.word[n], a.scale_f16, xf, undo, sum[n]);
                fetch_w(next, n, f);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (k0 + i < k1) {
                fetch_x(k0 + i, t[i]);
#pragma unroll
                for (int n = 0; n < NT; n++) fetch_w(k0 + i, n, t[i]);
            }
        for (int kt = k0; kt < k1; kt += AHEAD)
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
                if (kt + i < k1) use(kt + i, t[i]);
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) sh.sum[w][n][4 * q + i][c] = sum[n][i];
        __syncthreads();
        for (int i = threadIdx.x; i < NT * RR * TO; i += SEGS * CT_WAVE) {
            const int n = i / (RR * TO), r = i >> 4 & (RR - 1), o = (blockIdx.x * NT + n) * TO + c;
            if (r < nr && o < a.out_d) {
                float v = 0.0f;
#pragma unroll
                for (int s = 0; s < SEGS; s++) v += sh.sum[s][n][r][c];
                finish<BF16>(a, r0 + r, o, v);
            }
        }
        __syncthreads();
    }
}

// Few rows whose inputs fit LDS: a workgroup splits all of them once, RR rows (a
// power of two up to 16), and then goes from outputs to outputs, NT tiles at a
// time; its eight wavefronts each take one segment of the inputs and join
// their sums in LDS, in order.  A wavefront has AHEAD tiles of codes in flight,
// those of the next outputs among them, from before the inputs are split.
// Where linear_kernel would take many rounds, splitting inputs in each: 1 x 8192 -> 24576
// 22.5 us, there 36.
constexpr int FEW_LDS = 136 << 10;           // of inputs, beside 16 KB of sums, within a CU's 160

template <bool BF16, int GS, int NT>
__global__ __launch_bounds__(SEGS * CT_WAVE, 4) void linear_few_kernel(Args a, int lr, int groups) {
    constexpr int NB = BF16 ? 1 : 2, AHEAD = 4 / NT;
    extern __shared__ __align__(16) f16x8 sx[];          // [NB][itiles][16][RR], then undo [itiles][RR]
    __shared__ float ssum[2][SEGS][NT][16][TO];
    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE);
    const int c = lane & 15, q = lane >> 4, RR = 1 << lr;
    const int k0 = w * a.per, mine = max(min(a.per, a.itiles - k0), 0);
    const int pieces = (a.itiles * 16) << lr;
    float *sundo = reinterpret_cast<float *>(sx + NB * pieces);
    const long r0 = (long)RR * blockIdx.y;
    const int nr = (int)min((long)RR, a.rows - r0);

    u32x4 code[AHEAD][NT];
    uint32_t word[AHEAD][NT][4 / GS];
    auto fetch = [&](int grp, int t, u32x4 (&cd)[NT], uint32_t (&wd)[NT][4 / GS]) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const long tile = (long)min(grp * NT + n, a.otiles - 1) * a.itiles + k0 + t;
            cd[n] = reinterpret_cast<const u32x4 *>(a.codes)[tile * CT_WAVE + lane];
#pragma unroll
            for (int g = 0; g < 4 / GS; g++) wd[n][g] = a.scales[(tile * 16 + c) * (4 / GS) + g];
        }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; i++)
        if (i < mine) fetch(blockIdx.x, i, code[i], word[i]);

    // 16 lanes a row's tile
    auto at = [&](int kt, int k8, int row) { return ((kt * 16 + k8) << lr) + ((row ^ k8) & (RR - 1)); };
    for (int i = threadIdx.x >> 4; i < a.itiles * nr; i += SEGS * CT_WAVE / 16) {
        const int kt = nr == 1 ? i : i / nr, row = i - kt * nr;
        f16x8 h[NB];
        float v[8];
        f16x8 *hi = &sx[at(kt, c, row)], *lo = &sx[(NB - 1) * pieces + at(kt, c, row)];
        const char *x = input_at<BF16>(a, r0 + row, kt * TI + 8 * c);
        if (kt * TI + TI <= a.in_d) fetch8<BF16>(x, v);
        else fetch_last8<BF16>(x, a.in_d - kt * TI - 8 * c, v);
        const float undo = split8<NB>(v, h);
        *hi = h[0];
        if (NB > 1) *lo = h[NB - 1];
        if (c == 0) sundo[(kt << lr) + row] = undo;
    }
    __syncthreads();

    const int row = c & (RR - 1);
    int px[4];                               // this lane's pieces of a tile
#pragma unroll
    for (int j = 0; j < 4; j++) px[j] = at(k0, 4 * j + q, row);
    for (int grp = blockIdx.x, turn = 0; grp < groups; grp += gridDim.x, turn ^= 1) {
        f32x4 sum[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) sum[n] = (f32x4){0, 0, 0, 0};
        for (int t = 0; t < mine; t += AHEAD)
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                if (t + i >= mine) break;
                f16x8 xf[NB][4];
#pragma unroll
                for (int n = 0; n < NB; n++)
#pragma unroll
                    for (int j = 0; j < 4; j++) xf[n][j] = sx[n * pieces + px[j] + ((t + i) << (4 + lr))];
                // rows 4 q + i of the products; past RR they repeat and are not used
                f32x4 undo;
                const float *u = sundo + ((k0 + t + i) << lr);
                if (lr < 2) undo = (f32x4){u[0], u[RR - 1], u[0], u[0]};
                else undo = *reinterpret_cast<const f32x4 *>(u + (4 * q & (RR - 1)));
#pragma unroll
                for (int n = 0; n < NT; n++) tile_product<NB, GS>(code[i][n], word[i][n], a.scale_f16, xf, undo, sum[n]);
                if (t + i + AHEAD < mine) fetch(grp, t + i + AHEAD, code[i], word[i]);
                else if (grp + (int)gridDim.x < groups) fetch(grp + gridDim.x, i, code[i], word[i]);
            }
        // two buffers: the one written here was read before the last barrier
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (4 * q + i < RR) ssum[turn][w][n][4 * q + i][c] = sum[n][i];
        __syncthreads();
        for (int i = threadIdx.x; i < (NT * 16) << lr; i += SEGS * CT_WAVE) {
            const int n = i >> (4 + lr), r = i >> 4 & (RR - 1), o = (grp * NT + n) * TO + (i & 15);
            if (r < nr && o < a.out_d) {
                float v = 0.0f;
#pragma unroll
                for (int s = 0; s < SEGS; s++) v += ssum[turn][s][n][r][i & 15];
                finish<BF16>(a, r0 + r, o, v);
            }
        }
    }
}

// Many rows: a workgroup takes 64 rows and 32 outputs a wavefront.  Its inputs are
// split once and left in LDS as the products' A operands, in two buffers: while
// one tile is multiplied the next is split, between the products, and the one
// after it is asked for.  No branches among them: they cost registers for operands
// that are read a step ahead.  The sums are those of linear_few_kernel, segment by
// segment.  in_d >= 128.  W = 8 splits the inputs half as often for an output as
// W = 4: 752 x 1280 -> 5120 in 32 us instead of 38, 4000 x 4096 -> 4096 of bf16 in
// 212 instead of 263.
constexpr int BR = 64;

template <bool BF16, int GS, int W>
__global__ __launch_bounds__(W * CT_WAVE, 2) void linear_rows_kernel(Args a) {
    constexpr int NB = BF16 ? 1 : 2, MT = BR / 16, NT = 2, BO = W * 16 * NT, BT = W * CT_WAVE, SI = BR * 16 / BT, RS = BT / 16;
    __shared__ __align__(16) f16x8 sx[2][NB][BR / 16][256];
    __shared__ __align__(16) float sundo[2][BR];
    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE);
    const int c = lane & 15, q = lane >> 4;
    const int ot0 = (blockIdx.y * W + w) * NT;
    const int k8 = threadIdx.x & 15, sr = threadIdx.x >> 4;      // staged: rows sr + SR i, piece k8
    const u32x4 *codes[NT];
    // scale words: WT a tile, tile after tile; threads past the last repeat it
    constexpr int WT = 16 * (4 / GS), WORDS = BO / 16 * WT, SW = (WORDS + BT - 1) / BT;
    __shared__ uint32_t sword[2][SW * BT];
    uint32_t words[SW];
#pragma unroll
    for (int i = 0; i < SW; i++) {
        const int t = min((int)threadIdx.x + i * BT, WORDS - 1);
        words[i] = (min((int)blockIdx.y * (BO / 16) + t / WT, a.otiles - 1) * a.itiles * WT + t % WT) * 4u;
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        codes[n] = reinterpret_cast<const u32x4 *>(a.codes) + (long)min(ot0 + n, a.otiles - 1) * a.itiles * CT_WAVE;
    }
    const long r0 = (long)BR * blockIdx.x;
    const int nr = (int)min((long)BR, a.rows - r0);
    float total[MT][NT][4], sum[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) total[m][n][i] = sum[m][n][i] = 0.0f;
    // 32-bit offsets beside scalar bases, here and of the words: 64-bit addresses
    // do not fit the registers
    uint32_t xat[SI];
#pragma unroll
    for (int i = 0; i < SI; i++)                 // rows that are not there repeat the last one
        xat[i] = ((uint32_t)min(sr + RS * i, nr - 1) * (uint32_t)a.ld_x + 8 * k8) * (BF16 ? 2 : 4);
    const char *xbase = input_at<BF16>(a, r0, 0);
    float v[SI][8];
    const int whole = a.in_d / TI;               // tiles that end before in_d
    auto fetch_x = [&](int kt, int i) __attribute__((always_inline)) {
        fetch8<BF16>(xbase + min(kt, whole - 1) * (TI * (BF16 ? 2 : 4)) + xat[i], v[i]);
    };
    auto place_x = [&](int b, int i) __attribute__((always_inline)) {
        const int row = sr + RS * i, m = row >> 4, at = piece(k8, row & 15);
        f16x8 h[NB];
        const float undo = split8<NB>(v[i], h);
#pragma unroll
        for (int n = 0; n < NB; n++) sx[b][n][m][at] = h[n];
        sundo[b][row] = undo;                    // the same of all 16 lanes
    };
    auto last_x = [&](int kt) __attribute__((always_inline)) {           // a tile past the whole ones, into v
#pragma unroll
        for (int i = 0; i < SI; i++) {
            fetch_last8<BF16>(xbase + kt * (TI * (BF16 ? 2 : 4)) + xat[i], a.in_d - kt * TI - 8 * k8, v[i]);
        }
    };
    u32x4 code[NT];
    uint32_t word[SW];
    auto fetch_w = [&](int kt) __attribute__((always_inline)) {
        kt = min(kt, a.itiles - 1);
#pragma unroll
        for (int n = 0; n < NT; n++) code[n] = codes[n][kt * CT_WAVE + lane];
#pragma unroll
        for (int i = 0; i < SW; i++)
            word[i] = *reinterpret_cast<const uint32_t *>(reinterpret_cast<const char *>(a.scales) + (words[i] + kt * WT * 4u));
    };
    auto place_w = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < SW; i++) sword[b][threadIdx.x + i * BT] = word[i];
    };
#pragma unroll
    for (int i = 0; i < SI; i++) fetch_x(0, i);
    fetch_w(0);
#pragma unroll
    for (int i = 0; i < SI; i++) place_x(0, i);
    place_w(0);
#pragma unroll
    for (int i = 0; i < SI; i++) fetch_x(1, i);
    int left = a.per;                            // tiles of this segment
    for (int kt = 0; kt < a.itiles; kt++) {
        __syncthreads();
        const int b = kt & 1;
        // the buffer that the tile before last leaves is free
        if (kt + 1 == whole && whole < a.itiles) last_x(kt + 1);
        // operands are read a step (a term of 32 inputs) ahead of their products
        f16x8 wf[2][NT], xf[2][MT];
        auto read_x = [&](int step) __attribute__((always_inline)) {
#pragma unroll
            for (int m = 0; m < MT; m++) xf[step & 1][m] = sx[b][step % NB][m][piece(4 * (step / NB) + q, c)];
        };
        uint32_t nw[2][NT];
        auto read_w = [&](int j) __attribute__((always_inline)) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if (j % GS == 0) nw[j / GS & 1][n] = sword[b][(w * NT + n) * WT + c * (4 / GS) + j / GS];
                wf[j & 1][n] = weights8(code[n][j], less_of(nw[j / GS & 1][n]));
            }
        };
        f32x4 acc[MT][NT];
        read_x(0);
        read_w(0);
#pragma unroll
        for (int step = 0; step < 4 * NB; step++) {
            const int j = step / NB;
            if (step + 1 < 4 * NB) read_x(step + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (step % NB == 0 && j % GS == 0)
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int n = 0; n < NT; n++) acc[m][n] = (f32x4){0, 0, 0, 0};
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[step & 1][m], wf[j & 1][n], acc[m][n], 0, 0, 0);
            if (step % NB == NB - 1 && j < 3) read_w(j + 1);
            if (step % NB == NB - 1 && j == 2) fetch_w(kt + 1);
            // the next tile's inputs, and the one after it
            constexpr int EVERY = 4 * NB / SI ? 4 * NB / SI : 1, AT = SI > 4 * NB ? SI / (4 * NB) : 1;
            if (step % EVERY == 0)
#pragma unroll
                for (int i = step / EVERY * AT; i < (step / EVERY + 1) * AT; i++) {
                    place_x(b ^ 1, i);
                    fetch_x(kt + 2, i);
                }
            if (step == 4 * NB - 1) place_w(b ^ 1);
            if (step % NB == NB - 1 && j % GS == GS - 1) {
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    const f32x4 undo = *reinterpret_cast<const f32x4 *>(&sundo[b][16 * m + 4 * q]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const float s = scale_of(nw[j / GS & 1][n], a.scale_f16);
#pragma unroll
                        for (int i = 0; i < 4; i++) sum[m][n][i] = __builtin_fmaf(acc[m][n][i] * undo[i], s, sum[m][n][i]);
                        // a group's sums before the next one's products: side by side
                        // they do not fit the registers
                        if (GS < 4) asm volatile("" : "+v"(sum[m][n][0]), "+v"(sum[m][n][1]), "+v"(sum[m][n][2]), "+v"(sum[m][n][3]));
                    }
                }
            }
        }
        if (--left == 0 || kt + 1 == a.itiles) {
            left = a.per;
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        total[m][n][i] += sum[m][n][i];
                        sum[m][n][i] = 0.0f;
                    }
        }
    }
    __syncthreads();
    // through LDS, in as many turns as a part of each wavefront's [64][32] needs
    constexpr int TURN = BF16 ? 2 : 1, ROWS = BR / TURN;
    float *out = reinterpret_cast<float *>(sx) + w * (ROWS * 16 * NT);
    static_assert(sizeof(float) * W * ROWS * 16 * NT <= sizeof(sx), "the sums take the inputs' place");
    const int o = ot0 * TO + (lane & 31);
#pragma unroll
    for (int h = 0; h < TURN; h++) {
#pragma unroll
        for (int m = 0; m < MT / TURN; m++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) out[(16 * m + 4 * q + i) * (16 * NT) + 16 * n + c] = total[h * (MT / TURN) + m][n][i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll 2
        for (int r = lane >> 5; r < min(nr - ROWS * h, ROWS); r += 2)
            if (o < a.out_d) finish<BF16>(a, r0 + ROWS * h + r, o, out[r * (16 * NT) + (lane & 31)]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// ---- Laying out ----------------------------------------------------------

__device__ __forceinline__ uint32_t word_of(uint16_t scale, int zero) {
    return (uint32_t)scale << 16 | __builtin_bit_cast(uint16_t, (_Float16)(-0.5f - (float)zero * 0x1p-11f));
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
        const float s = scale_of(word, w.scale_f16 ? ~0u : 0u), less = ((float)less_of(word).low[0] + 0.5f) * 0x1p11f;
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
    a.scale_f16 = w->scale_f16 ? ~0u : 0u;
    a.y = p->y; a.x = p->x; a.ld_y = p->ld_y; a.ld_x = p->ld_x;
    a.rows = p->rows; a.act = p->act; a.scale = p->scale; a.bias = p->bias;
    const long rows = p->rows;
    const long rt64 = (rows + BR - 1) / BR;
    const int lr = rows == 1 ? 0 : rows <= 4 ? 2 : rows <= 8 ? 3 : 4;
    const size_t inputs = (size_t)a.itiles * ((256 * (p->bf16 ? 1 : 2) + 4) << lr);
    const long rt = (rows + (1 << lr) - 1) >> lr;
    const bool fits = inputs <= FEW_LDS && rt <= 65535;
    // linear_kernel's tiles of outputs together.  A CU holds one of its workgroups: as few
    // rounds of them as there can be.  Two cost 1.2 times one, four 1.4 (one / two / four in
    // us: 64 x 4096 -> 1024, 256 tiles 9.6 / 10.5 / 12.6; 64 x 5120 -> 1280, 320 tiles 19 /
    // 12.7 / 15.6; 64 x 4096 -> 4096, 1024 tiles 31 / 20.8 / 13.6; bf16 16 x 8192 -> 8192,
    // 512 tiles 34 / 23 / 26; 64 x 8192 -> 8192, 2048 tiles 129 / 85 / 49).
    const long rt16 = (rows + 15) / 16;
    auto rounds = [&](int n) { return ((a.otiles + n - 1) / n * rt16 + 255) / 256; };
    const int nt = rounds(4) * 14 < rounds(2) * 12 && rounds(4) * 14 < rounds(1) * 10 ? 4 : rounds(2) * 12 < rounds(1) * 10 ? 2 : 1;
    // It takes inputs that fit LDS too where it is done in one round, or in three for fp32
    // rows that fill its tiles (it / linear_few_kernel: 64 x 1024 -> 4096 6.2 / 7.0 us; 5 x
    // 1024 -> 16384 5.8 / 6.9; 3 x 8192 -> 8192 14.2 / 19.6; three rounds: 48 x 1024 -> 16384
    // 15.9 / 18.5; four: 64 x 1024 -> 16384 20.7 / 19.2; bf16, two: 1 x 8192 -> 24576 36 /
    // 22.5; four: 256 x 1024 -> 4096 19.3 / 12.7).
    const bool few = fits && rounds(nt) > (rows > 16 && !p->bf16 ? 3 : 1);
    // Many rows in tiles of 64 once these fill the card.  With the inputs in LDS in us, few /
    // rows, in 128 workgroups of 64 rows: 64 x 1024 -> 16384 19.3 / 24.1; in 160: 300 x 1024
    // -> 4096 23.6 / 24.5; in 176: 700 x 1024 -> 2048 28.8 / 24.8; in 256: 128 x 1024 ->
    // 16384 35 / 25.  Inputs that do not fit LDS, linear_kernel / rows: in 120: 752 x 5120
    // -> 1280 58 / 81; in 128: bf16 256 x 8192 -> 4096 95 / 108; in 150: 900 x 5120 -> 1280
    // 73 / 81, some 11 us for each of its rounds.
    if (rt64 * ((w->out_d + 127) / 128) >= (fits ? 176 : p->bf16 ? 144 : 200) && rows > 32 && w->in_d >= TI && p->ld_x < 1 << 24) {
        // 256 outputs a workgroup where that leaves enough of them: 752 x 5120 -> 1280, 60
        // of them, 104 us instead of 84; 752 x 1280 -> 5120, 240, 32 instead of 38
        const int wide = rt64 * ((w->out_d + 255) / 256) >= 200;
        const dim3 grid((unsigned)rt64, (unsigned)(wide ? (w->out_d + 255) / 256 : (w->out_d + 127) / 128));
#define ROWS(B, GS)                                                                                                 \
    do {                                                                                                            \
        if (wide) hipLaunchKernelGGL((linear_rows_kernel<B, GS, 8>), grid, dim3(8 * CT_WAVE), 0, s, a);             \
        else hipLaunchKernelGGL((linear_rows_kernel<B, GS, 4>), grid, dim3(4 * CT_WAVE), 0, s, a);                  \
    } while (0)
        if (p->bf16) {
            if (w->group == 32) ROWS(true, 1);
            else if (w->group == 64) ROWS(true, 2);
            else ROWS(true, 4);
        } else {
            if (w->group == 32) ROWS(false, 1);
            else if (w->group == 64) ROWS(false, 2);
            else ROWS(false, 4);
        }
#undef ROWS
        return;
    }
    if (few) {
        // two tiles of outputs at a time share the inputs' loads from LDS (256 x 1024 ->
        // 4096: 17.9 us, one at a time 24.2; 1 x 8192 -> 24576: 22.5, 24.8); words for
        // each 32 inputs do not fit the registers twice
        const int two = w->group > 32 && inputs <= 120 << 10;
        const int groups = (a.otiles + two) / (1 + two);
        // as many workgroups as the CUs hold at once: one more than that is a second round
        // for all (48 x 1024 -> 16384 in 513 of them 28 us, in 510 18.5)
        const long fit = inputs + (two ? 32768 : 16384) <= 80 << 10 ? 512 : 256;
        const dim3 grid((unsigned)(groups * rt <= fit ? groups : rt < fit ? fit / rt : 1), (unsigned)rt);
#define FEW(B, GS)                                                                                                              \
    do {                                                                                                                        \
        if (two) hipLaunchKernelGGL((linear_few_kernel<B, GS, (GS > 1 ? 2 : 1)>), grid, dim3(SEGS * CT_WAVE), inputs, s, a, lr, groups); \
        else hipLaunchKernelGGL((linear_few_kernel<B, GS, 1>), grid, dim3(SEGS * CT_WAVE), inputs, s, a, lr, groups);           \
    } while (0)
        if (p->bf16) {
            if (w->group == 32) FEW(true, 1);
            else if (w->group == 64) FEW(true, 2);
            else FEW(true, 4);
        } else {
            if (w->group == 32) FEW(false, 1);
            else if (w->group == 64) FEW(false, 2);
            else FEW(false, 4);
        }
#undef FEW
        return;
    }
    const dim3 grid((unsigned)((a.otiles + nt - 1) / nt), (unsigned)(rt16 < 4096 ? rt16 : 4096));
#define LINEAR(B, GS)                                                                                               \
    do {                                                                                                            \
        if (nt == 4) hipLaunchKernelGGL((linear_kernel<B, GS, 4>), grid, dim3(SEGS * CT_WAVE), 0, s, a);            \
        else if (nt == 2) hipLaunchKernelGGL((linear_kernel<B, GS, 2>), grid, dim3(SEGS * CT_WAVE), 0, s, a);       \
        else hipLaunchKernelGGL((linear_kernel<B, GS, 1>), grid, dim3(SEGS * CT_WAVE), 0, s, a);                    \
    } while (0)
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
