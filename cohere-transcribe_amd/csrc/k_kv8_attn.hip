// k_kv8_attn.hip — softmax attention over the paged 8-bit key/value cache.
//
// A wavefront holds a tile of 16 query rows (tokens x query heads of one kv
// head) and walks over the keys 32 at a time, all in registers:
//   S^T = K Q^T   MFMA 16x16x32 f16, two 16-key halves; lane (c, g), c = lane
//                 % 16, g = lane / 16, holds query c's scores of keys 4g..4g+3
//                 of each half;
//   P             online softmax in base 2; the four lanes of a query share
//                 one running maximum, which follows the scores only when
//                 they pass it by 2^8 (most steps then rescale nothing);
//   O^T += V^T P^T  the same lane's eight p are one B operand if the product's
//                 k index runs over keys {4g..4g+3, 16+4g..16+4g+3}, so P
//                 never leaves its lane; V's rows are loaded to match, 8 dims
//                 a lane, and byte pairs of two keys interleaved (v_perm) on
//                 the way to f16.
// e4m3 values are f16 values, so codes are converted exactly and the products
// are those of the codes.  Scales are powers of two and never touch a code:
// the key scale multiplies the score; the value scale 2^e is an offset of the
// softmax exponent.  What enters the second product is p' = 2^(s + e - z), z a
// whole number some 6 below the largest s + e among the keys that the row
// sees, so p' <= 2^14 and the largest is never small, whatever scales the pages
// of the other rows have; the denominator counts p' 2^-e, in fp32.  z is of the
// row alone: with a reference exponent that the rows of a wavefront shared,
// rows that saw none of the large values lost their own.  Query rows are
// brought to a largest value in [2^12, 2^13) by a power of two.  fp32 rows
// enter as the sum of two f16 (22 bits and more), and so do their p'; bf16 rows
// are one f16 each (exact down to 2^-26 of the row's largest), and so p'.
#include "ct_dev.h"
#include "ct_kv8.h"
#include "k_kv8.h"
#include <type_traits>

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int NT = 256, NW = NT / CT_WAVE;   // threads, wavefronts of a workgroup
constexpr float LOG2E = 1.4426950408889634f;
constexpr int P_EXP = 6;                     // p' is at most 2^(P_EXP + SLACK), within f16
constexpr int SLACK = 8;                     // how far s + e may pass the running maximum, in bits
constexpr float ONE_V = 1.0f / (1 << P_EXP); // what the sums of p' v have to be scaled by to count as l does
constexpr int FAR = 90;                      // value scales 2^FAR apart: see add_far
constexpr int MAX_EXP = 120;                 // exponent of the largest scale that an append gives

struct Args {
    const uint8_t *k, *v;        // the layer's pools
    const float *ks, *vs;
    const int *table, *len, *rows;
    int pages, lp, kv, seqs, table_w;
    const void *q;
    void *out;
    long ld_q, ld_out;
    int group, causal, window, sinks, n_rows, cap;   // cap: tokens looked at
    float scale2;                // scale * log2(e)
    int vec;                     // q rows are 16-byte aligned
    int one_tile;                // every sequence's rows fit one tile: tile = sequence
    int chunk, nchunk;           // 32-key steps of a chunk, chunks of the grid
    int tile_rows;               // packed rows of a tile: 16 or rows_of(bf16)
    int rpt;                     // rows of a tile kept in the partial results
    float *part;                 // partial O [tile][kv][chunk][rpt][D], then (m, l) pairs
    float2 *stat;
};

// The kernel's arguments read again, past this point: what only its end
// needs does not hold scalar registers through the loop.
__device__ __forceinline__ const Args &args_again() {
    auto p = (const __attribute__((address_space(4))) Args *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Args *)p;
}

// A tile's rows and the keys they see: 32-key steps 0 .. sink_steps - 1 hold
// the first tokens, the rest start at lo (a multiple of 32).
struct Tile {
    int seq, r0, n, row;         // sequence, its first row and rows; first packed row of the tile
    int len, pos0;               // tokens held; position of the sequence's first row
    int end, lo, sink_steps, steps;
    int full_lo, full_hi;        // steps at keys in [full_lo, full_hi) are seen whole by every row
};

// Inclusive prefix sum over the workgroup's W wavefronts.
template <int W>
__device__ __forceinline__ int block_sum(int v, int *part, int &total) {
    const int lane = threadIdx.x % CT_WAVE, w = threadIdx.x / CT_WAVE;
#pragma unroll
    for (int o = 1; o < CT_WAVE; o <<= 1) {
        const int u = __shfl_up(v, o, CT_WAVE);
        if (lane >= o) v += u;
    }
    if (lane == CT_WAVE - 1) part[w] = v;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < W; i++) {
        if (i < w) before += part[i];
        total += part[i];
    }
    __syncthreads();
    return v + before;
}

// Finds tile `id` (rows_per_tile packed rows each); false if there is none.
// Every thread of the workgroup calls it with the same id.
template <int W>
__device__ __forceinline__ bool find_tile(const Args &a, int id, int rows_per_tile, int *sh, Tile &t) {
    int tile = 0;
    if (a.one_tile) {
        t.seq = id;
        t.r0 = a.rows[id];
        t.n = a.rows[id + 1] - t.r0;
        t.len = a.len[id];
        if (t.r0 < 0 || t.n <= 0 || t.n > a.n_rows - t.r0) return false;
    } else {
        int n = 0, r0 = 0, rows = 0, len = 0;
        const int s = threadIdx.x;
        if (s < a.seqs) {
            r0 = a.rows[s];
            rows = a.rows[s + 1] - r0;
            len = a.len[s];
            if (r0 >= 0 && rows > 0 && rows <= a.n_rows - r0) n = (rows * a.group + rows_per_tile - 1) / rows_per_tile;
        }
        int total;
        const int upto = block_sum<W>(n, sh, total);
        if (id >= total) return false;
        if (id >= upto - n && id < upto) {
            sh[W] = s; sh[W + 1] = id - (upto - n); sh[W + 2] = r0; sh[W + 3] = rows; sh[W + 4] = len;
        }
        __syncthreads();
        t.seq = __builtin_amdgcn_readfirstlane(sh[W]);
        tile = __builtin_amdgcn_readfirstlane(sh[W + 1]);
        t.r0 = __builtin_amdgcn_readfirstlane(sh[W + 2]);
        t.n = __builtin_amdgcn_readfirstlane(sh[W + 3]);
        t.len = __builtin_amdgcn_readfirstlane(sh[W + 4]);
    }
    t.row = tile * rows_per_tile;
    // one tile: the joined sums have room for rpt rows, so a sequence with more
    // rows than max_rows is left out
    if (t.row >= t.n * a.group || (a.one_tile && t.n * a.group > a.rpt)) return false;
    t.len = max(t.len, 0);
    t.pos0 = t.len - t.n;
    // divisions only where they are needed: each is 0.1 us of a short call
    int first = t.row, last = min(t.row + rows_per_tile, t.n * a.group) - 1;
    if (a.group > 1) {
        first = a.one_tile ? 0 : first / a.group;
        last = a.one_tile ? t.n - 1 : last / a.group;
    }
    const int p0 = t.pos0 + first, p1 = t.pos0 + last;             // first and last row's positions
    t.end = max(min(a.causal ? p1 + 1 : t.len, a.cap), 0);
    t.lo = a.window ? max(p0 - a.window + 1, 0) & ~31 : 0;
    t.sink_steps = a.window ? (min(a.sinks, t.lo) + 31) >> 5 : 0;
    t.sink_steps = min(t.sink_steps, (t.end + 31) >> 5);
    t.steps = t.sink_steps + (t.end > t.lo ? (t.end - t.lo + 31) >> 5 : 0);
    t.full_lo = a.window ? p1 - a.window + 1 : 0;
    t.full_hi = min(a.causal ? p0 + 1 : t.len, a.cap);
    return true;
}

__device__ __forceinline__ int step_key(const Tile &t, int step) {
    return step < t.sink_steps ? step << 5 : t.lo + ((step - t.sink_steps) << 5);
}

__device__ __forceinline__ float fmax_q(float v) {      // over the four lanes of a query
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_q(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Two values as f16 terms: rounded, and what the rounding left, rounded; two
// at a time, by one conversion and one mixed fma each (fp32 prompts of 2500
// tokens 125 -> 120 us).
__device__ __forceinline__ void two_terms(float a, float b, f16x2 &hi, f16x2 &lo) {
    float minus = -1.0f;
    asm("" : "+s"(minus));       // a known -1 makes a conversion and a subtraction of the mixed fma
    hi = __builtin_convertvector((f32x2){a, b}, f16x2);
    lo = __builtin_convertvector((f32x2){__builtin_fmaf((float)hi[0], minus, a), __builtin_fmaf((float)hi[1], minus, b)}, f16x2);
}

__device__ __forceinline__ f16x2 cvt2(uint32_t w, bool hi) {
    return hi ? __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))
              : __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
}
__device__ __forceinline__ f16x8 cvt8(uint32_t a, uint32_t b) {
    const f16x2 x = cvt2(a, false), y = cvt2(a, true), z = cvt2(b, false), w = cvt2(b, true);
    return (f16x8){x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}

__device__ __forceinline__ f32x4 mfma_f16(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float pow2i(int e) {          // 2^e, e in [-126, 127]
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Bytes that are a NaN code (0x7f, 0xff) as 0x80 in their place.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

template <bool NONTEMPORAL, class T>
__device__ __forceinline__ T ask(const T *p) {
    if constexpr (NONTEMPORAL) return __builtin_nontemporal_load(p);
    else return *p;
}

// The raw codes of one 32-key step: K as 16-byte pieces (half, 64-dim group),
// V as D / 16 dims of keys 4g + j (j < 4) and 16 + 4g + j - 4.
template <int D>
struct Raw {
    u32x4 k[2][D / 64];
    uint32_t v[8][D / 64];
};

// The query row at element `off`: this lane's dims of each B operand, as
// they lie in memory.
template <bool BF16>
struct QPiece;
template <>
struct QPiece<true> {
    u16x8 v;
    __device__ __forceinline__ float at(int j) const { return bf2f(v[j]); }
};
template <>
struct QPiece<false> {
    f32x4 v[2];
    __device__ __forceinline__ float at(int j) const { return v[j >> 2][j & 3]; }
};

template <int D>
__device__ __forceinline__ void fetch_query(const Args &a, long off, int g, QPiece<true> (&x)[D / 32]) {
    const uint16_t *q = reinterpret_cast<const uint16_t *>(a.q) + off + 16 * g;
    if (a.vec) {
#pragma unroll
        for (int i = 0; i < D / 32; i++) x[i].v = *reinterpret_cast<const u16x8 *>(q + 64 * (i >> 1) + 8 * (i & 1));
    } else {
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) x[i].v[j] = q[64 * (i >> 1) + 8 * (i & 1) + j];
    }
}
template <int D>
__device__ __forceinline__ void fetch_query(const Args &a, long off, int g, QPiece<false> (&x)[D / 32]) {
    const float *q = reinterpret_cast<const float *>(a.q) + off + 16 * g;
    if (a.vec) {
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
                x[i].v[j] = *reinterpret_cast<const f32x4 *>(q + 64 * (i >> 1) + 8 * (i & 1) + 4 * j);
    } else {
#pragma unroll
        for (int i = 0; i < D / 32; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) x[i].v[j >> 2][j & 3] = q[64 * (i >> 1) + 8 * (i & 1) + j];
    }
}

// Brings the row to a largest value in [2^12, 2^13) and splits it into f16
// terms; returns the factor of its scores: what the power of two and the
// softmax scale leave.  A row with a value that is not finite is all NaN.
template <int D, bool BF16>
__device__ __forceinline__ float split_query(const Args &a, bool have, const QPiece<BF16> (&x)[D / 32],
                                             f16x8 (&qf)[BF16 ? 1 : 2][D / 32]) {
    constexpr int KS = D / 32, NB = BF16 ? 1 : 2;
    // the largest magnitude as an integer: infinities and NaN are the largest
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < KS; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(x[i].at(j)) & 0x7fffffffu);
    if (!have) top = 0;
    auto r = __builtin_amdgcn_permlane32_swap(top, top, false, false);
    top = max(r[0], r[1]);
    r = __builtin_amdgcn_permlane16_swap(top, top, false, false);
    top = max(r[0], r[1]);
    const bool fine = top < 0x7f800000u;
    // exponent of the row's largest value (zero and subnormal rows: 2^-126)
    const int e = fine ? max((int)(top >> 23), 1) - 127 : 0;
    const int up = 12 - e;                   // in [-115, 138]
    if constexpr (BF16) {
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const f16x2 y = __builtin_convertvector((f32x2){__builtin_amdgcn_ldexpf(x[i].at(j), up),
                                                                __builtin_amdgcn_ldexpf(x[i].at(j + 1), up)}, f16x2);
                qf[0][i][j] = y[0];
                qf[0][i][j + 1] = y[1];
            }
        // lanes without a row, and rows that are not finite
        if (__builtin_expect(__any(!have || !fine), 0)) {
            const bool keep = have && fine;
            const _Float16 other = have ? (_Float16)__builtin_nanf("") : (_Float16)0.0f;
#pragma unroll
            for (int i = 0; i < KS; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) qf[0][i][j] = keep ? qf[0][i][j] : other;
        }
    } else {
        // two factors, and every value chosen as it is split: the form above took
        // calls of 12 fp32 rows from 15.5 to 15.9 us
        const float f0 = pow2i(up >> 1), f1 = pow2i(up - (up >> 1));
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                float y[2];
#pragma unroll
                for (int n = 0; n < 2; n++) y[n] = !have ? 0.0f : fine ? x[i].at(j + n) * f0 * f1 : __uint_as_float(0x7fc00000u);
                f16x2 hi, lo;
                two_terms(y[0], y[1], hi, lo);
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    qf[0][i][j + n] = hi[n];
                    qf[NB - 1][i][j + n] = lo[n];
                }
            }
    }
    return a.scale2 * pow2i((-up) >> 1) * pow2i(-up - ((-up) >> 1));
}

// Exponent of a value page's scale.
__device__ __forceinline__ int exp_of(float scale) {
    return min(max((int)(__float_as_uint(scale) >> 23 & 255) - 127, KV8_MIN_EXP), MAX_EXP);
}

// What the queries of a step's U 16-key halves share: the key scales, the
// value scales' exponents and what makes a weight's share of l of p' (l counts
// in units of 2^P_EXP, which keeps undo in fp32's range).  least: the smallest
// factor of a score where some are masked, 0 elsewhere: -inf * 0 is NaN, and
// scores that small are 0 to the softmax.
template <int U>
struct Halves {
    float ks[U], ev[U], undo[U], least;
    __device__ __forceinline__ void set(int u, int e) {
        ev[u] = (float)e;
        undo[u] = pow2i(-e - P_EXP);
    }
};

// By how much the exponents of sums change (ldexp) whose maximum rises: x is the
// old one less the new, whole; NaN (none yet on either side) counts as
// -infinity.  No factor 2^x: it may be 0 where l, up to 2^100 over pages of
// zeros, still counts.
__device__ __forceinline__ int down(float x) { return (int)fmaxf(x, -400.0f); }

// p' of one query over U halves, 2^(s qs ks + ev - m), as B operands, and
// their sums.  The softmax is online, but its maximum is found only when it
// has to be: p' are computed with the one so far, and again (settle) if that
// was too_low for a lane of the wavefront.
template <int U, int NB>
__device__ __forceinline__ void powers(const f32x4 (&s)[U], float qs, const Halves<U> &hv, float m,
                                       float (&sum)[U], f16x8 (&pf)[U / 2][NB]) {
    const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const float ms = mu - hv.ev[u], f = fmaxf(qs * hv.ks[u], hv.least);
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; j++) p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j], f, -ms));
        if (NB > 1) {
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                f16x2 hi, lo;
                two_terms(p[j], p[j + 1], hi, lo);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    pf[u >> 1][0][4 * (u & 1) + j + i] = hi[i];
                    pf[u >> 1][NB - 1][4 * (u & 1) + j + i] = lo[i];
                }
            }
        } else {
            // the matrix instruction takes 16 bits: 11 of f16 are 8 times finer than
            // the bf16 that the output is rounded to, and a second term would
            // double the products
            const f16x2 a = __builtin_convertvector((f32x2){p[0], p[1]}, f16x2), b = __builtin_convertvector((f32x2){p[2], p[3]}, f16x2);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                pf[u >> 1][0][4 * (u & 1) + i] = a[i];
                pf[u >> 1][0][4 * (u & 1) + 2 + i] = b[i];
            }
        }
        // of the fp32 weights, not of those the product takes: where a half's
        // values are far smaller than others, f16 has none of its p' left, but
        // its keys keep their share of the softmax
        sum[u] = (p[0] + p[1]) + (p[2] + p[3]);
    }
}

// Whether a lane's p' of one query were computed with a maximum that is too
// low: none yet, or four of them pass 2^(P_EXP + SLACK) together.
template <int U>
__device__ __forceinline__ bool too_low(float m, const float (&sum)[U]) {
    float top = sum[0];
#pragma unroll
    for (int u = 1; u < U; u++) top = fmaxf(top, sum[u]);
    return m == -INFINITY || top > (float)(1 << (P_EXP + SLACK));    // a NaN needs no maximum
}

// Moves a query's maximum to that of its scores s (-inf: not seen) and
// computes its p' again; returns the factor of the sums so far.  A whole number:
// factors are then exact, and so is m - ev.
template <int U, int NB>
__device__ __forceinline__ float settle(const f32x4 (&s)[U], float qs, const Halves<U> &hv, float &m, float &l,
                                        float (&sum)[U], f16x8 (&pf)[U / 2][NB]) {
    float mt = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; u++)
        mt = fmaxf(mt, __builtin_fmaf(fmaxf(qs * hv.ks[u], hv.least), fmaxf(fmaxf(s[u][0], s[u][1]), fmaxf(s[u][2], s[u][3])), hv.ev[u]));
    const float mn = fmaxf(m, __builtin_ceilf(fmax_q(mt)) - P_EXP);
    const int by = down(m - mn);
    m = mn;
    l = __builtin_amdgcn_ldexpf(l, by);
    powers<U, NB>(s, qs, hv, m, sum, pf);
    return __builtin_amdgcn_ldexpf(1.0f, by);
}

// The weights' share of l of halves `far` (bits): those whose values are 2^-FAR
// of the largest that the wavefront met and less, pages of zeros among them.
// Their p' may be below fp32's range where the weights are not, so these come
// without the value scale, straight from the scores.  Elsewhere p' of the row's
// largest weight is 2^(5 - FAR) at least, so what fp32 loses is 2^-40 of it.
template <int U>
__device__ __forceinline__ void add_far(const f32x4 (&s)[U], float qs, const Halves<U> &hv, uint32_t far, float m,
                                        float (&sum)[U], float &l) {
    const float mu = (m == -INFINITY ? 0.0f : m) + P_EXP;
#pragma unroll
    for (int u = 0; u < U; u++)
        if (far >> u & 1) {
            const float f = fmaxf(qs * hv.ks[u], hv.least);
#pragma unroll
            for (int j = 0; j < 4; j++) l += __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j], f, -mu));
            sum[u] = 0.0f;
        }
}

// The score where the mask is all ones, -inf where it is 0.
__device__ __forceinline__ float masked(uint32_t m, float s) {
    return __uint_as_float((__float_as_uint(s) & m) | (0xff800000u & ~m));
}

// The keys the row at position pos of a sequence of len tokens sees: [0,
// first) and [lo, lo + n).
struct Sight {
    int first, n, lo;
    __device__ __forceinline__ Sight(const Args &a, int len, int pos) {
        const int end = max(min(a.causal ? pos + 1 : len, a.cap), 0);
        lo = a.window ? pos - a.window + 1 : 0;
        first = a.window ? min(a.sinks, end) : end;
        n = a.window ? max(end - lo, 0) : 0;
    }
    // all ones if the query sees the key, else 0: no comparison, whose results
    // for many keys at once would not fit the scalar registers
    __device__ __forceinline__ uint32_t sees(bool window, int key) const {
        const int before = (key - first) >> 31;
        if (!window) return before;
        return before | ~(((key - lo) | (lo + n - 1 - key)) >> 31);
    }
    // scores of keys key, key + 1, ...: -inf where they are not seen
    __device__ __forceinline__ void mask(bool window, int key, f32x4 &s) const {
#pragma unroll
        for (int j = 0; j < 4; j++) s[j] = masked(sees(window, key + j), s[j]);
    }
};
constexpr int NO_KEY = 1 << 30;                  // past every row's keys

// V's A operands of four dims, code(j) their codes of the lane's key j: pairs
// of keys side by side.
template <int D, class Code>
__device__ __forceinline__ void operand_v(Code code, f16x8 (&vf)[4]) {
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int y = 0; y < 4; y++) {
        lo[y] = __builtin_amdgcn_perm(code(2 * y + 1), code(2 * y), 0x05010400u);
        hi[y] = __builtin_amdgcn_perm(code(2 * y + 1), code(2 * y), 0x07030602u);
    }
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
        for (int y = 0; y < 4; y++) {
            const f16x2 z = cvt2(b < 2 ? lo[y] : hi[y], b & 1);
            vf[b][2 * y] = z[0];
            vf[b][2 * y + 1] = z[1];
        }
}

// The NaN codes among a step's values, which the products took as zeros: they
// reach the rows that see their token, and they alone (0 * NaN is NaN, so a
// product over a masked one would spread it).  Rare, so it is done after all
// steps, from the codes read again: in the loop it cost 40 registers.
template <int D, int NQ>
__device__ __forceinline__ void spread_nan(const Args &a, const Tile &t, int h, int key, int c, int g,
                                           const int (&pos)[NQ], f32x4 (&o)[NQ][D / 16]) {
    f16x8 one[NQ];
    uint32_t nan[8][D / 64];
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int kk = key + 16 * (j >> 2) + 4 * g + (j & 3);
        const bool held = kk < min(t.len, a.cap);
        const int p = a.table[(long)t.seq * a.table_w + (held ? kk >> a.lp : 0)];
        const bool in = held && (unsigned)p < (unsigned)a.pages;
        const long base = ((((long)(in ? p : 0) * a.kv + h) << a.lp) + (in ? kk & ((1 << a.lp) - 1) : 0)) * D + c * (D / 16);
#pragma unroll
        for (int x = 0; x < D / 64; x++)
            nan[j][x] = in ? nan_bytes(*reinterpret_cast<const uint32_t *>(a.v + base + 4 * x)) : 0;
#pragma unroll
        for (int n = 0; n < NQ; n++)
            one[n][j] = in && Sight(a, t.len, pos[n]).sees(a.window, kk) ? (_Float16)1.0f : (_Float16)0.0f;
    }
#pragma unroll
    for (int i = 0; i < D / 16; i++) {
        f16x8 hit;
#pragma unroll
        for (int j = 0; j < 8; j++) hit[j] = (nan[j][i >> 2] >> (8 * (i & 3) + 7)) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            const f32x4 x = mfma_f16(hit, one[n], (f32x4){0, 0, 0, 0});
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (x[j] > 0.0f) o[n][i][j] = __uint_as_float(0x7fc00000u);
        }
    }
}

// w with its NaN codes as zeros.
__device__ __forceinline__ uint32_t without_nan(uint32_t w) {
    const uint32_t b = nan_bytes(w);
    return w & ~(b | (b - (b >> 7)));
}

// Few rows of a sequence: W wavefronts share a tile's keys, step by step in
// turn, each with two steps of codes in flight, and join their sums in LDS.
// Bound by memory: 32 sequences of up to 30000 tokens, 32 heads over 8 of 128,
// bf16 (1.35 GB of codes) take 238 us, 5.7 TB/s where a plain read reaches 6.3
// to 7.1 and a copy 4.8; 64 of up to 1000 tokens, 8 heads, fp32 (88 MB) 21.1 us;
// one of 376 tokens 6.7 us, of which 4.7 are an empty call's.  fp32
// rows take two terms each, so twice the products.
// ONCE: a sequence's rows are one tile, so its codes are read once.
template <int D, bool BF16, int W, bool ONCE>
__global__ __launch_bounds__(W * CT_WAVE, BF16 ? 3 : 2) void attn_kernel(Args a) {
    constexpr int KS = D / 32;            // k steps of the score product
    constexpr int DI = D / 16;            // 16-dim tiles of O; dims of V a lane loads
    constexpr int NB = BF16 ? 1 : 2;      // f16 terms of a query value and of p
    // the wavefronts' sums [W][rpt][D], maxima and l [W][16]: of the rows a tile
    // has, mostly one
    extern __shared__ float so[];
    __shared__ int sh[W + 5];
    __shared__ float sm[W][16], sl[W][16];

    // heads vary fastest: workgroup i runs on XCD i % 8, so with 8 kv heads the
    // tiles of one head share an L2
    const int id = blockIdx.x / a.kv, h = blockIdx.x - id * a.kv, ch = blockIdx.y;
    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE), c = lane & 15, g = lane >> 4;
    // this wavefront's steps: first, first + W, ...; lane i keeps the page and
    // the scales of 16-key half i (-1: not in the pool).  Where a step's keys do
    // not depend on the lengths, its page is read along with them.
    const int first = ch * a.chunk + w;
    const bool ahead = a.one_tile && !a.window;
    int key_i = 32 * (first + W * (lane >> 1)) + 16 * (lane & 1), pg = -1;
    if (ahead && (lane >> 1) * W < a.chunk && key_i < a.cap) pg = a.table[(long)id * a.table_w + (key_i >> a.lp)];
    Tile t;
    if (!find_tile<W>(a, id, 16, sh, t)) return;
    const int chunks = a.nchunk > 1 ? (t.steps + a.chunk - 1) / a.chunk : 1;
    if (ch >= max(chunks, 1)) return;
    const int last = min(t.steps, (ch + 1) * a.chunk);

    // this lane's query row: asked for first, used after the keys are asked for
    const int R = t.row + c;
    const bool have = R < t.n * a.group;
    const int qi = have ? (a.group > 1 ? R / a.group : R) : 0, qh = have ? R - qi * a.group : 0;
    {
        const int st = first + W * (lane >> 1);
        key_i = step_key(t, st) + 16 * (lane & 1);
        const bool mine = st < last && key_i < t.end;
        if (!ahead && mine) pg = a.table[(long)t.seq * a.table_w + (key_i >> a.lp)];
        if (!mine || (unsigned)pg >= (unsigned)a.pages) pg = -1;
    }
    QPiece<BF16> x[KS];
    fetch_query<D>(a, (long)(t.r0 + qi) * a.ld_q + (long)(h * a.group + qh) * D, g, x);

    const int P = 1 << a.lp;
    const unsigned koff = c * D + 16 * g, voff = 4 * g * D + c * DI;
    auto load = [&](int st, int i, Raw<D> &r) {          // step st, this wavefront's i-th
        unsigned ka = koff, va = voff;
        asm volatile("" : "+v"(ka), "+v"(va));   // 32-bit offsets beside a scalar base, not a 64-bit sum a load
        const int key = step_key(t, st);
        long base[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int p = max(__builtin_amdgcn_readlane(pg, 2 * i + u), 0);   // any page if there is none
            base[u] = ((((long)p * a.kv + h) << a.lp) + ((key + 16 * u) & (P - 1))) * D;
        }
        // non-temporal where codes are read once (7.1 against 6.3 TB/s in a
        // plain read of 4 GiB); tiles of one sequence share them in L2.  K
        // first, as it is used first (32 x 30000 tokens 244 -> 240 us)
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int y = 0; y < D / 64; y++)
                r.k[u][y] = ask<ONCE>(reinterpret_cast<const u32x4 *>(a.k + base[u] + ka + 64 * y));
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint8_t *vp = a.v + base[u] + va + j * D;
                if (D == 128) {
                    const u32x2 y = ask<ONCE>(reinterpret_cast<const u32x2 *>(vp));
                    r.v[4 * u + j][0] = y[0];
                    r.v[4 * u + j][D / 64 - 1] = y[1];
                } else {
                    r.v[4 * u + j][0] = ask<ONCE>(reinterpret_cast<const uint32_t *>(vp));
                }
            }
    };
    float pks = 0.0f, pvs = 0.0f;
    if (pg >= 0) {
        pks = a.ks[(long)pg * a.kv + h];
        pvs = a.vs[(long)pg * a.kv + h];
    }
    Raw<D> ra, rb;
    if (first < last) load(first, 0, ra);
    f16x8 qf[NB][KS];
    const float qs = split_query<D, BF16>(a, have, x, qf);
    const int pos[1] = {t.pos0 + qi};
    const int hard = min(t.len, a.cap);      // tokens at and past it hold anything

    f32x4 o[1][DI];
#pragma unroll
    for (int i = 0; i < DI; i++) o[0][i] = (f32x4){0, 0, 0, 0};
    float m = have ? -INFINITY : INFINITY, l = 0.0f;     // lanes without a row: no weights, and never a new maximum
    int emax = KV8_MIN_EXP;
    bool dirty = false;

    auto use = [&](int st, int i, Raw<D> &r) {
        const int key = step_key(t, st);
        f32x4 s[2];
        Halves<2> hv;
        int ev[2];
        bool in[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            in[u] = __builtin_amdgcn_readlane(pg, 2 * i + u) >= 0;
            hv.ks[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pks), 2 * i + u));
            ev[u] = exp_of(__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pvs), 2 * i + u)));
        }
        // a chain of products per half and query term, next to each other
        f32x4 sb[NB][2];
#pragma unroll
        for (int b = 0; b < NB; b++) sb[b][0] = sb[b][1] = (f32x4){0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < KS; x++) {
            f16x8 kf[2];
#pragma unroll
            for (int u = 0; u < 2; u++) kf[u] = cvt8(r.k[u][x >> 1][2 * (x & 1)], r.k[u][x >> 1][2 * (x & 1) + 1]);
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int u = 0; u < 2; u++) sb[b][u] = mfma_f16(kf[u], qf[b][x], sb[b][u]);
        }
#pragma unroll
        for (int u = 0; u < 2; u++) s[u] = NB > 1 ? sb[0][u] + sb[NB - 1][u] : sb[0][u];
        const bool whole = key >= t.full_lo && key + 32 <= t.full_hi && in[0] && in[1];   // sink steps lie below full_lo
        if (__builtin_expect(!whole, 0)) {
            uint32_t bad = 0;
            const Sight see(a, t.len, pos[0]);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int k4 = (in[u] ? key + 16 * u : NO_KEY) + 4 * g;
                if (a.window) see.mask(true, k4, s[u]);
                else see.mask(false, k4, s[u]);
            }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int kk = key + 16 * u + 4 * g + j;
                    // a token nobody sees may hold anything: 0 * NaN is NaN
                    const bool any = in[u] && kk < hard;
#pragma unroll
                    for (int y = 0; y < D / 64; y++) {
                        if (!any) r.v[4 * u + j][y] = 0;
                        bad |= nan_bytes(r.v[4 * u + j][y]);
                    }
                }
            if (__builtin_expect(__any(bad != 0), 0)) {
                dirty = true;
#pragma unroll
                for (int j = 0; j < 8; j++)
#pragma unroll
                    for (int y = 0; y < D / 64; y++) r.v[j][y] = without_nan(r.v[j][y]);
            }
        }
        emax = max(emax, max(ev[0], ev[1]));     // pages that are not there have the least
        uint32_t far = 0;
        if (__builtin_expect(min(ev[0], ev[1]) < emax - FAR, 0))
#pragma unroll
            for (int u = 0; u < 2; u++) far |= (uint32_t)(in[u] && ev[u] < emax - FAR) << u;
        hv.least = whole ? 0.0f : 0x1p-100f;
        hv.set(0, ev[0]);
        hv.set(1, ev[1]);
        f16x8 pf[1][NB];
        float sum[2];
        powers<2, NB>(s, qs, hv, m, sum, pf);
        if (__builtin_expect(__any(too_low(m, sum)), 0)) {
            const float al = settle<2, NB>(s, qs, hv, m, l, sum, pf);
#pragma unroll
            for (int y = 0; y < DI; y++) o[0][y] *= al;
        }
        if (__builtin_expect(far, 0)) add_far<2>(s, qs, hv, far, m, sum, l);
#pragma unroll
        for (int u = 0; u < 2; u++) l = __builtin_fmaf(sum[u], hv.undo[u], l);
#pragma unroll
        for (int y = 0; y < D / 64; y++) {
            f16x8 vf[4];
            operand_v<D>([&](int j) { return r.v[j][y]; }, vf);
#pragma unroll
            for (int n = 0; n < NB; n++)
#pragma unroll
                for (int b = 0; b < 4; b++) o[0][4 * y + b] = mfma_f16(vf[b], pf[0][n], o[0][4 * y + b]);
        }
    };

    // the scales are here before the loop: a wait for them inside it would be
    // one for every load, the next step's too
    asm volatile("" : "+v"(pks), "+v"(pvs));
    // two steps in flight
    for (int st = first, i = 0; st < last; st += 2 * W, i += 2) {
        if (st + W < last) load(st + W, i + 1, rb);
        use(st, i, ra);
        if (st + W >= last) break;
        if (st + 2 * W < last) load(st + 2 * W, i + 2, ra);
        use(st + W, i + 1, rb);
    }
    if (__builtin_expect(dirty, 0))
        for (int st = first; st < last; st += W) spread_nan<D, 1>(a, t, h, step_key(t, st), c, g, pos, o);

    // the wavefronts' sums joined, in their order
    l = sum_q(l);
    if (have) {
        if (g == 0) { sm[w][c] = m; sl[w][c] = l; }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < DI; i++) so[(w * a.rpt + c) * D + (4 * g + j) * DI + i] = o[0][i][j];
    }
    __syncthreads();
    const int nr = min(16, t.n * a.group - t.row);
    for (int x = threadIdx.x; x < nr * D; x += W * CT_WAVE) {
        const int r = x / D, d = x % D;
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < W; i++) M = fmaxf(M, sm[i][r]);
        const float Mu = M == -INFINITY ? 0.0f : M;
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int i = 0; i < W; i++) {
            const int by = down(sm[i][r] - Mu);
            num += __builtin_amdgcn_ldexpf(so[(i * a.rpt + r) * D + d], by);
            den += __builtin_amdgcn_ldexpf(sl[i][r], by);
        }
        if (chunks <= 1) {
            const int R2 = t.row + r, i = a.group > 1 ? R2 / a.group : R2;
            const float y = den == 0.0f ? 0.0f : num * ONE_V / den;
            const long off = (long)(t.r0 + i) * a.ld_out + (long)(h * a.group + R2 - i * a.group) * D + d;
            if (BF16) reinterpret_cast<uint16_t *>(a.out)[off] = f2bf(y);
            else reinterpret_cast<float *>(a.out)[off] = y;
        } else {
            const long at = (((long)id * a.kv + h) * a.nchunk + ch) * a.rpt + r;
            a.part[at * D + d] = num;
            if (d == 0) a.stat[at] = make_float2(M, den);
        }
    }
}

// Many rows of a sequence: a workgroup holds 128 packed rows, 32 a wavefront
// (fp32: 64 and 16, whose two f16 terms make as many products of each operand
// read from LDS), and takes 64 keys at a time.  Each wavefront fetches and
// converts a quarter of them (K or V of one 32-key step) and leaves them in
// LDS as the products' A operands, lane by lane, so that every LDS access is
// a run of 1 KB; all four then read the whole 64 keys.  Two LDS buffers: the
// next keys' codes are in flight while this step's products run, and one
// barrier a step keeps them apart.
// Bound by instructions: 6 prompts of up to 2500 tokens, 32 heads over 8 of
// 128, bf16 (163 GFLOP) take 218 us, 749 TFLOP/s; the matrix units are busy
// 34% of the time, and vector instructions issue in 57% of it, with the two
// wavefronts a SIMD that the registers allow.  Measured slower, when this form
// took 259 us: 8 wavefronts with 128 keys an iteration (273), the two 32-key
// halves a stage apart so that weights and products interleave (266).
constexpr int rows_of(bool bf16) { return bf16 ? 128 : 64; }

template <int D, bool BF16>
__global__ __launch_bounds__(NT, 2) void rows_kernel(Args a) {
    constexpr int KS = D / 32, DI = D / 16, NB = BF16 ? 1 : 2;
    constexpr int ROWS = rows_of(BF16), WR = ROWS / NW, NQ = WR / 16;
    constexpr int UNIT = D * 32;               // halves of a 32-key step's K or V
    static_assert(2 * KS == DI, "K and V take the same number of operands");
    __shared__ int sh[NW + 5];
    __shared__ __align__(16) _Float16 lds[2][4][UNIT];   // buffer; K, K, V, V of the two steps
    // key scales and value scales' exponents (GONE: not in the pool) of each
    // iteration's four 16-key halves; two batches of 32 iterations in turn
    __shared__ __align__(16) float sscale[2][32][4];
    __shared__ __align__(16) int sexp[2][32][4];
    constexpr int GONE = KV8_MIN_EXP - 1;
    __shared__ int spos[ROWS];                 // the rows' positions, for the steps that not all see
    __shared__ int snan;                       // the V of some step holds a NaN

    const int h = blockIdx.x % a.kv, id = gridDim.x / a.kv - 1 - blockIdx.x / a.kv, ch = blockIdx.y;
    Tile t;
    if (!find_tile<NW>(a, id, ROWS, sh, t)) return;
    const int chunks = a.nchunk > 1 ? (t.steps + a.chunk - 1) / a.chunk : 1;
    if (ch >= max(chunks, 1)) return;
    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE), c = lane & 15, g = lane >> 4;
    const int all = t.n * a.group, hard = min(t.len, a.cap);

    const int wr0 = min(t.row + WR * w, all - 1), wr1 = min(t.row + WR * w + WR, all) - 1;
    const bool idle = t.row + WR * w >= all;
    const int p0 = t.pos0 + wr0 / a.group, p1 = t.pos0 + wr1 / a.group;
    const int full_lo = a.window ? p1 - a.window + 1 : 0, full_hi = min(a.causal ? p0 + 1 : t.len, a.cap);
    const int wend = idle ? 0 : min(a.causal ? p1 + 1 : t.len, a.cap);

    // the unit this wavefront fetches: K (isv 0) or V of step 2 it + kb; lane i
    // keeps the page and place of half i & 1 of the step of iteration base + i / 2
    const int kb = w & 1, isv = w >> 1;
    const int s0 = ch * a.chunk, s1 = min(t.steps, s0 + a.chunk), iters = (s1 - s0 + 1) >> 1;
    const int P = 1 << a.lp;
    auto key_of = [&](int it0) {                 // first key of this lane's half
        return step_key(t, min(s0 + 2 * (it0 + (lane >> 1)) + kb, s1 - 1)) + 16 * (lane & 1);
    };
    auto fetch_page = [&](int it0) {
        const int st = s0 + 2 * (it0 + (lane >> 1)) + kb, key = key_of(it0);
        int p = -1;
        if (st < s1 && key < t.end) p = a.table[(long)t.seq * a.table_w + (key >> a.lp)];
        return (unsigned)p < (unsigned)a.pages ? p : -1;
    };
    // where the half's codes start; page 0 for one that is not there
    auto place_of = [&](int p, int it0) { return ((((long)max(p, 0) * a.kv + h) << a.lp) + (key_of(it0) & (P - 1))) * D; };
    auto fetch_scale = [&](int p) { return p >= 0 ? (isv ? a.vs : a.ks)[(long)p * a.kv + h] : 0.0f; };
    // asked for together: the first pages, the query rows; then what they lead to
    int pg = fetch_page(0), pg2 = fetch_page(32);
    QPiece<BF16> x[NQ][KS];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int R = min(t.row + WR * w + 16 * n + c, all - 1);
        fetch_query<D>(a, (long)(t.r0 + R / a.group) * a.ld_q + (long)(h * a.group + R % a.group) * D, g, x[n]);
    }
    float psc = fetch_scale(pg);
    long at64 = place_of(pg, 0);
    const uint8_t *pool = isv ? a.v : a.k;
    // the scales of the batch that starts at iteration it0, into LDS
    auto put_scales = [&](int it0) {
        const int bt = it0 >> 5 & 1, i = lane >> 1, half = 2 * kb + (lane & 1);
        if (!isv) sscale[bt][i][half] = psc;
        else sexp[bt][i][half] = pg < 0 ? GONE : exp_of(psc);
    };
    const unsigned off = isv ? 4 * g * D + c * DI : c * D + 16 * g;

    // the codes of a unit, asked for AHEAD iterations before they are converted,
    // with their pages and scales; bf16 has no registers for a second one
    constexpr int AHEAD = BF16 ? 1 : 2;
    struct Unit {
        uint32_t raw[D / 8];
        int p0, p1;
    };
    auto fetch = [&](int it, Unit &r, auto is_v) __attribute__((always_inline)) {
        constexpr bool V = decltype(is_v)::value;
        unsigned at = off;
        asm volatile("" : "+v"(at));            // a 32-bit offset beside a scalar base, not a 64-bit sum a load
        const int i = 2 * (it & 31);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int page = __builtin_amdgcn_readlane(pg, i + u);
            if (u) r.p1 = page;
            else r.p0 = page;
            const uint32_t lo = __builtin_amdgcn_readlane((int)at64, i + u), hi = __builtin_amdgcn_readlane((int)(at64 >> 32), i + u);
            const uint8_t *p = pool + ((uint64_t)hi << 32 | lo);
            uint32_t *to = r.raw + u * (D / 16);
            if constexpr (!V) {
#pragma unroll
                for (int x = 0; x < D / 64; x++) {
                    const u32x4 y = *reinterpret_cast<const u32x4 *>(p + at + 64 * x);
#pragma unroll
                    for (int i2 = 0; i2 < 4; i2++) to[4 * x + i2] = y[i2];
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (D == 128) {
                        const u32x2 y = *reinterpret_cast<const u32x2 *>(p + at + j * D);
                        to[2 * j] = y[0];
                        to[2 * j + 1] = y[1];
                    } else {
                        to[j] = *reinterpret_cast<const uint32_t *>(p + at + j * D);
                    }
                }
            }
        }
        // pages and scales of the next 32 iterations, well before they are used
        if ((it & 31) == 15) psc = fetch_scale(pg2);
        if ((it & 31) == 31) {
            pg = pg2;
            at64 = place_of(pg, it + 1);
            put_scales(it + 1);
            pg2 = fetch_page(it + 33);
        }
    };
    bool dirty = false;
    auto place = [&](int it, Unit &r, auto is_v) __attribute__((always_inline)) {       // a fetched unit into buffer it & 1
        constexpr bool V = decltype(is_v)::value;
        const int b = it & 1;
        f16x8 *to = reinterpret_cast<f16x8 *>(lds[b][2 * V + kb]) + lane;
        if constexpr (!V) {
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int x = 0; x < D / 64; x++) {
                    const uint32_t *y = r.raw + u * (D / 16) + 4 * x;
                    to[(u * KS + 2 * x) * CT_WAVE] = cvt8(y[0], y[1]);
                    to[(u * KS + 2 * x + 1) * CT_WAVE] = cvt8(y[2], y[3]);
                }
        } else {
        // a step that every row of the tile sees whole may spread its NaN; one
        // that some row does not: tokens that are not there hold anything, and
        // a NaN must not meet a masked row's zero
        const int key = step_key(t, min(s0 + 2 * it + kb, s1 - 1));
        if (__builtin_expect(!(r.p0 >= 0 && r.p1 >= 0 && key >= t.full_lo && key + 32 <= t.full_hi), 0)) {
            uint32_t bad = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                // all ones where the token is there
                const uint32_t in = (j < 4 ? r.p0 : r.p1) < 0 ? 0 : (key + 4 * g + 16 * (j >> 2) + (j & 3) - hard) >> 31;
#pragma unroll
                for (int x = 0; x < D / 64; x++) {
                    uint32_t &y = r.raw[j * (D / 64) + x];
                    y &= in;
                    bad |= nan_bytes(y);
                }
            }
            if (__builtin_expect(__any(bad != 0), 0)) {
                dirty = true;
#pragma unroll
                for (int x = 0; x < D / 8; x++) r.raw[x] = without_nan(r.raw[x]);
            }
        }
#pragma unroll
        for (int x = 0; x < D / 64; x++) {
            f16x8 vf[4];
            operand_v<D>([&](int j) { return r.raw[j * (D / 64) + x]; }, vf);
#pragma unroll
            for (int i = 0; i < 4; i++) to[(4 * x + i) * CT_WAVE] = vf[i];
        }
        }
    };


    // this wavefront's rows
    f16x8 qf[NQ][NB][KS];
    float qs[NQ];
    auto split = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int R = t.row + WR * w + 16 * n + c;
        const bool have = R < all;
        qs[n] = split_query<D, BF16>(a, have, x[n], qf[n]);
        if (g == 0) spos[WR * w + 16 * n + c] = t.pos0 + (have ? R / a.group : 0);
    }
    };

    f32x4 o[NQ][DI];
    float m[NQ], l[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        m[n] = t.row + WR * w + 16 * n + c < all ? -INFINITY : INFINITY;     // lanes without a row
        l[n] = 0.0f;
#pragma unroll
        for (int i = 0; i < DI; i++) o[n][i] = (f32x4){0, 0, 0, 0};
    }
    int emax = KV8_MIN_EXP;

    // iteration `it`: the unit asked for AHEAD iterations ago into the other
    // buffer, the next one asked for, and this one's products.  One barrier:
    // before it every wavefront has filled its part of this buffer and is done
    // with the other.
    auto step = [&](int it, Unit &r, auto is_v) __attribute__((always_inline)) {
        __syncthreads();
        if (it + 1 < iters) place(it + 1, r, is_v);
        if (it + 1 + AHEAD < iters) fetch(it + 1 + AHEAD, r, is_v);
        const int b = it & 1, k0 = step_key(t, s0 + 2 * it), k1 = step_key(t, min(s0 + 2 * it + 1, s1 - 1));
        if (k0 < wend) {
            const f16x8 *kl = reinterpret_cast<const f16x8 *>(lds[b][0]) + lane;
            const f16x8 *vl = reinterpret_cast<const f16x8 *>(lds[b][2]) + lane;
            // operands are read a group of KG ahead of the products they feed: of
            // one 32-dim step, KG of the four halves
            constexpr int KG = NQ == 2 ? 2 : 4;
            f32x4 s[NQ][4];
            f16x8 kf[2][KG];
            auto read_k = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                for (int v = 0; v < KG; v++) {
                    const int x = i / (4 / KG), u = i % (4 / KG) * KG + v;
                    kf[i & 1][v] = kl[((u >> 1) * DI + (u & 1) * KS + x) * CT_WAVE];
                }
            };
            read_k(0);
#pragma unroll
            for (int n = 0; n < NQ; n++)
#pragma unroll
                for (int u = 0; u < 4; u++) s[n][u] = (f32x4){0, 0, 0, 0};
            int ev[4];
            Halves<4> hv;
            const f32x4 ks = *reinterpret_cast<const f32x4 *>(sscale[it >> 5 & 1][it & 31]);
            const i32x4 ex = *reinterpret_cast<const i32x4 *>(sexp[it >> 5 & 1][it & 31]);
#pragma unroll
            for (int u = 0; u < 4; u++) {
                hv.ks[u] = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(ks[u])));
                ev[u] = __builtin_amdgcn_readfirstlane(ex[u]);
            }
            f16x8 vf[2][4];
#pragma unroll
            for (int i = 0; i < KS * 4 / KG; i++) {
                if (i + 1 < KS * 4 / KG) read_k(i + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < NB; y++)
#pragma unroll
                    for (int v = 0; v < KG; v++)
#pragma unroll
                        for (int n = 0; n < NQ; n++) {
                            f32x4 &to = s[n][i % (4 / KG) * KG + v];
                            to = mfma_f16(kf[i & 1][v], qf[n][y][i / (4 / KG)], to);
                        }
            }
            const int least = min(min(ev[0], ev[1]), min(ev[2], ev[3]));
            const bool whole = least > GONE && k0 >= full_lo && k0 + 32 <= full_hi && k1 >= full_lo && k1 + 32 <= full_hi;
            if (__builtin_expect(!whole, 0)) {
#pragma unroll
                for (int n = 0; n < NQ; n++) {
                    const Sight see(a, t.len, spos[WR * w + 16 * n + c]);
                    // one form for both kinds of mask: two took fp32 prompts from 120 to 124 us
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int kk = (u < 2 ? k0 : k1) + 16 * (u & 1) + 4 * g + j;
                            s[n][u][j] = ev[u] == GONE ? -INFINITY : masked(see.sees(a.window, kk), s[n][u][j]);
                        }
                }
            }
            emax = max(emax, max(max(ev[0], ev[1]), max(ev[2], ev[3])));
            uint32_t far = 0;
            if (__builtin_expect(least < emax - FAR, 0))
#pragma unroll
                for (int u = 0; u < 4; u++) far |= (uint32_t)(ev[u] > GONE && ev[u] < emax - FAR) << u;
            hv.least = whole ? 0.0f : 0x1p-100f;
#pragma unroll
            for (int u = 0; u < 4; u++) hv.set(u, ev[u]);
            f16x8 pf[NQ][2][NB];
            float sum[NQ][4];
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                powers<4, NB>(s[n], qs[n], hv, m[n], sum[n], pf[n]);
                if (__builtin_expect(__any(too_low(m[n], sum[n])), 0)) {
                    const float al = settle<4, NB>(s[n], qs[n], hv, m[n], l[n], sum[n], pf[n]);
#pragma unroll
                    for (int i = 0; i < DI; i++) o[n][i] *= al;
                }
                if (__builtin_expect(far, 0)) add_far<4>(s[n], qs[n], hv, far, m[n], sum[n], l[n]);
#pragma unroll
                for (int u = 0; u < 4; u++) l[n] = __builtin_fmaf(sum[n][u], hv.undo[u], l[n]);
            }
            // group y of the V operands: four dim tiles of step y / (DI / 4); a
            // second step that is not there has p' = 0 and holds finite values
            constexpr int VG = DI / 2;
#pragma unroll
            for (int i = 0; i < 4; i++) vf[0][i] = vl[i * CT_WAVE];
#pragma unroll
            for (int y = 0; y < VG; y++) {
                if (y + 1 < VG)
#pragma unroll
                    for (int i = 0; i < 4; i++) vf[(y + 1) & 1][i] = vl[(4 * (y + 1) + i) * CT_WAVE];
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int z = 0; z < NB; z++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int n = 0; n < NQ; n++) {
                            f32x4 &to = o[n][(4 * y + i) % DI];
                            to = mfma_f16(vf[y & 1][i], pf[n][y / (DI / 4)][z], to);
                        }
            }
        }
    };
    // the loop twice: what a wavefront fetches and converts stays in registers
    // of its own, whether K or V
    auto walk = [&](auto is_v) __attribute__((always_inline)) {
        Unit r[AHEAD];
        if (iters > 0) fetch(0, r[0], is_v);
        split();
        put_scales(0);
        if (iters > 0) place(0, r[0], is_v);
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (i + 1 < iters) fetch(i + 1, r[i], is_v);
        for (int it = 0; it < iters; it += AHEAD)
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
                if (it + i < iters) step(it + i, r[i], is_v);
    };
    if (threadIdx.x == 0) snan = 0;              // the first step's barrier comes before the flag is set
    if (isv) walk(std::true_type());
    else walk(std::false_type());
    if (dirty && lane == 0) snan = 1;
    __syncthreads();
    const Args &z = args_again();
    int pos[NQ];
#pragma unroll
    for (int n = 0; n < NQ; n++) pos[n] = spos[WR * w + 16 * n + c];
    if (__builtin_expect(snan, 0))
        for (int st = s0; st < s1; st++) spread_nan<D, NQ>(z, t, h, step_key(t, st), c, g, pos, o);

#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const float den = sum_q(l[n]);
        const int r = WR * w + 16 * n + c, R = t.row + r;
        if (R >= all) continue;
        if (chunks <= 1) {
            const float f = den == 0.0f ? 0.0f : 1.0f / den;
            const long off = (long)(t.r0 + R / z.group) * z.ld_out + (long)(h * z.group + R % z.group) * D;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < DI; i++) {
                    const float y = den == 0.0f ? 0.0f : o[n][i][j] * ONE_V * f;
                    if (BF16) reinterpret_cast<uint16_t *>(z.out)[off + (4 * g + j) * DI + i] = f2bf(y);
                    else reinterpret_cast<float *>(z.out)[off + (4 * g + j) * DI + i] = y;
                }
        } else {
            const long at = (((long)id * z.kv + h) * z.nchunk + ch) * z.rpt + r;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < DI; i++) z.part[at * D + (4 * g + j) * DI + i] = o[n][i][j];
            if (g == 0) z.stat[at] = make_float2(m[n], den);
        }
    }
}

// Joins a tile's chunks, in an order that the lengths alone give (32 x 4 heads
// over 8 chunks: 4 us): WPR wavefronts a row (chunks w, w + WPR, ...), each
// with four chunks' loads in flight, then their sums in order.
template <int D, bool BF16, int WPR>
__global__ __launch_bounds__(NT) void join_kernel(Args a) {
    constexpr int DL = D / CT_WAVE, RPB = NW / WPR;       // dims of a lane, rows of a workgroup
    __shared__ int sh[NW + 5];
    __shared__ float so[NW][D], sl[NW];
    const int h = blockIdx.x % a.kv, id = blockIdx.x / a.kv;
    Tile t;
    if (!find_tile<NW>(a, id, a.tile_rows, sh, t)) return;
    const int chunks = (t.steps + a.chunk - 1) / a.chunk;
    if (chunks <= 1) return;
    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE), part = w % WPR;
    const int r = blockIdx.y * RPB + w / WPR, nr = min(a.tile_rows, t.n * a.group - t.row);
    const bool have = r < nr;
    const long at = ((long)id * a.kv + h) * a.nchunk * a.rpt + (have ? r : 0);
    float M = -INFINITY;
    for (int k = lane; k < chunks; k += CT_WAVE) M = fmaxf(M, a.stat[at + (long)k * a.rpt].x);
    M = wave_max(M);
    const float Mu = M == -INFINITY ? 0.0f : M;
    float num[DL] = {}, den = 0.0f;
    for (int k0 = part; k0 < chunks; k0 += 4 * WPR) {
        float2 st[4];
        float x[4][DL];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int k = min(k0 + u * WPR, chunks - 1);
            st[u] = a.stat[at + (long)k * a.rpt];
#pragma unroll
            for (int j = 0; j < DL; j++) x[u][j] = a.part[(at + (long)k * a.rpt) * D + lane * DL + j];
        }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            if (k0 + u * WPR >= chunks) break;
            const int by = down(st[u].x - Mu);
            den += __builtin_amdgcn_ldexpf(st[u].y, by);
#pragma unroll
            for (int j = 0; j < DL; j++) num[j] += __builtin_amdgcn_ldexpf(x[u][j], by);
        }
    }
    if (WPR > 1) {
#pragma unroll
        for (int j = 0; j < DL; j++) so[w][lane * DL + j] = num[j];
        if (lane == 0) sl[w] = den;
        __syncthreads();
        if (part) return;
#pragma unroll
        for (int i = 1; i < WPR; i++) {
            den += sl[w + i];
#pragma unroll
            for (int j = 0; j < DL; j++) num[j] += so[w + i][lane * DL + j];
        }
    }
    if (!have) return;
    const int R = t.row + r;
    const long off = (long)(t.r0 + R / a.group) * a.ld_out + (long)(h * a.group + R % a.group) * D + lane * DL;
#pragma unroll
    for (int j = 0; j < DL; j++) {
        const float y = den == 0.0f ? 0.0f : num[j] * ONE_V / den;
        if (BF16) reinterpret_cast<uint16_t *>(a.out)[off + j] = f2bf(y);
        else reinterpret_cast<float *>(a.out)[off + j] = y;
    }
}

// The launch's shape, from the sizes alone.  Both sides of each rule below were
// measured when it was set; the kernels have become up to 15% faster since.
struct Shape {
    int tile_rows, one_tile, tiles, waves, chunk, nchunk, rpt;
};

constexpr int SMALL_UNITS = 640;    // tiles of 16 rows * kv heads up to which they are taken

// The longest walk of a tile of `tile_rows` rows, in steps.
long walk_of(const BackendKv8 *c, const BackendKv8Attn *a, int tile_rows) {
    long keys = (long)c->table_w * c->page_tokens;
    if (a->max_len > 0 && a->max_len < keys) keys = a->max_len;
    long steps = (keys + 31) / 32;
    if (a->window > 0) {
        const long span = ((long)a->window + tile_rows + 62) / 32 + ((long)a->sinks + 31) / 32;
        if (span < steps) steps = span;
    }
    return steps;
}

Shape shape_of(const BackendKv8 *c, const BackendKv8Attn *a) {
    Shape s;
    const int group = a->heads / c->kv_heads;
    const long rows = (long)(a->max_rows < a->n_rows ? a->max_rows : a->n_rows) * group;   // of a sequence
    // Tiles of 16 rows while they leave CUs free, then the rows kernel's
    // (bf16 1 x 500 rows, 256 units of 16: 12.7 us against 24.2; 32 x 32, 600
    // units: 18.3 against 21.7; 4 x 500, 700 units: 27.3 against 24.5; fp32
    // 8 x 300, 860 units: 30.5 against 16.2).
    const long tiles16 = (long)a->n_rows * group / 16 + c->seqs;
    s.tile_rows = rows > 16 && tiles16 * c->kv_heads > SMALL_UNITS ? rows_of(a->bf16) : 16;
    s.one_tile = rows <= s.tile_rows;
    s.tiles = s.one_tile ? c->seqs : (int)((long)a->n_rows * group / s.tile_rows + c->seqs);
    s.rpt = rows < s.tile_rows ? (int)rows : s.tile_rows;
    const long steps = walk_of(c, a, s.tile_rows);
    const long units = (long)s.tiles * c->kv_heads;
    s.waves = NW;
    if (s.tile_rows == 16) {
        // A CU reads some 30 GB/s, so a few units have to be spread over many
        // CUs, which costs a join (3.5 us).  One chunk up to 24 steps (8 units
        // of 12 steps: 7.0 us, in two chunks 10.1), or up to 64 where there is
        // a unit for every other CU (192 units of 36 steps: 9.2 us, in chunks
        // of 16 13.2); else 512 chunks in all, of 8 to 128 steps (8 units of
        // 125 steps: 10.6 us at 8, 24.8 at 64; 256 units of 938 steps: 325 us
        // at 8, 245 at 64 and 128).  seqs counts whether they have rows or not,
        // so with a tile a sequence (max_rows * group up to 16) a row's bits do
        // not depend on the others.
        s.chunk = (int)steps;
        if (steps > 24 && (steps > 64 || units < 128)) {
            const long each = (units * steps + 511) / 512;
            s.chunk = each < 8 ? 8 : each > 128 ? 128 : (int)each;
        }
        // 8 wavefronts a unit while that fills no CU twice (192 units of 36
        // steps: 9.2 us against 12.4; 512 of 10: 13.4 against 10.2)
        if (s.chunk >= steps && units <= 256) s.waves = 8;
        if (!s.one_tile) {
            // rows of one sequence share its codes in L2: fewer, longer chunks
            // (fp32 3 x 201 rows, 248 units of 219 steps: 55 us in chunks of
            // 128, 85 of 32; 4 x 100 rows over 63 steps: 23 us whole, 28 of 16)
            const long each = (units * steps + 255) / 256;
            s.waves = NW;
            s.chunk = each < 64 ? 64 : each > 128 ? 128 : (int)each;
        }
    } else {
        // a workgroup for each CU, of at least 512 keys (1 x 2000 rows, 32
        // heads over 8, 504 units: 71 us whole, 100 in two chunks)
        const long want = (256 + units - 1) / units;
        s.chunk = (int)((steps + want - 1) / want);
        s.chunk = s.chunk < 16 ? 16 : (s.chunk + 1) & ~1;
    }
    if (s.chunk < 1) s.chunk = 1;
    s.nchunk = (int)((steps + s.chunk - 1) / s.chunk);
    if (s.nchunk < 1) s.nchunk = 1;
    return s;
}

// Floats of the partial results of a shape: none for one chunk.
size_t partials_of(const BackendKv8 *c, const Shape &s) {
    if (s.nchunk == 1) return 0;
    return (size_t)s.tiles * c->kv_heads * s.nchunk * s.rpt * (c->head_dim + 2);
}

}  // namespace

extern "C" size_t ctk_kv8_attn_need(const BackendKv8 *c, const BackendKv8Attn *a) {
    return partials_of(c, shape_of(c, a));
}

// An upper bound of ctk_kv8_attn_need over all calls with at most these rows
// and tokens, of rows whose larger tiles hold `most_rows`: the chunks of all
// units are at most the number aimed at, or one for every 128 steps where that is
// more, and one a unit for rounding up.
static size_t work_of(const BackendKv8 *c, const BackendKv8Attn *a, int most_rows) {
    const long group = a->heads / c->kv_heads, kv = c->kv_heads;
    const long rows = (long)(a->max_rows < a->n_rows ? a->max_rows : a->n_rows) * group;
    const long steps = walk_of(c, a, most_rows), row = c->head_dim + 2;
    const long all16 = (long)a->n_rows * group / 16 + c->seqs;
    auto chunks = [&](long units, long aim) {
        const long by128 = units * steps / 128;
        return (by128 > aim ? by128 : aim) + units;
    };
    // a sequence's rows in one tile of 16
    long most = chunks(c->seqs * kv, 512) * (rows < 16 ? rows : 16);
    if (rows > 16) {
        // in several, while there are few; then tiles of most_rows, split while
        // there are fewer than 256
        const long few = all16 * kv < SMALL_UNITS ? all16 * kv : SMALL_UNITS;
        const long some = chunks(few, 256) * 16;
        const long wide = ((long)a->n_rows * group / most_rows + c->seqs) * kv;
        const long whole = all16 * kv > SMALL_UNITS ? (256 + 2 * (wide < 256 ? wide : 256)) * most_rows : 0;
        most = some > most ? some : most;
        most = whole > most ? whole : most;
    }
    // nothing is split where no tile walks further than one chunk's least
    return steps <= 8 ? 0 : (size_t)(most * row);
}

// Either type of rows: their tiles, and with them the split, differ.
extern "C" size_t ctk_kv8_attn_work(const BackendKv8 *c, const BackendKv8Attn *a) {
    const size_t f32 = work_of(c, a, rows_of(false)), bf16 = work_of(c, a, rows_of(true));
    return f32 > bf16 ? f32 : bf16;
}

extern "C" void ctk_kv8_attn(const BackendKv8 *c, int layer, const BackendKv8Attn *p, hipStream_t s) {
    const Shape sh = shape_of(c, p);
    const long heads = (long)layer * c->pages * c->kv_heads;
    Args a;
    a.lp = 31 - __builtin_clz((unsigned)c->page_tokens);
    a.k = c->k + (heads << a.lp) * c->head_dim;
    a.v = c->v + (heads << a.lp) * c->head_dim;
    a.ks = c->kscale + heads;
    a.vs = c->vscale + heads;
    a.table = c->table; a.len = c->len; a.rows = p->rows;
    a.pages = c->pages; a.kv = c->kv_heads; a.seqs = c->seqs; a.table_w = c->table_w;
    a.q = p->q; a.out = p->out; a.ld_q = p->ld_q; a.ld_out = p->ld_out;
    a.group = p->heads / c->kv_heads;
    a.causal = p->causal != 0; a.n_rows = p->n_rows;
    a.window = p->window < CT_KV8_KEYS ? p->window : CT_KV8_KEYS;      // wider ones hide nothing more
    a.sinks = p->sinks < CT_KV8_KEYS ? p->sinks : CT_KV8_KEYS;
    const long cap = (long)c->table_w * c->page_tokens;
    a.cap = (int)(p->max_len > 0 && p->max_len < cap ? p->max_len : cap);
    a.scale2 = p->scale * LOG2E;
    a.vec = ((uintptr_t)p->q & 15) == 0 && p->ld_q % (p->bf16 ? 8 : 4) == 0;
    a.tile_rows = sh.tile_rows; a.one_tile = sh.one_tile; a.chunk = sh.chunk; a.nchunk = sh.nchunk; a.rpt = sh.rpt;
    const size_t n = (size_t)sh.tiles * c->kv_heads * sh.nchunk * sh.rpt;
    a.part = p->work;
    a.stat = sh.nchunk > 1 ? reinterpret_cast<float2 *>(p->work + n * c->head_dim) : nullptr;
    const int wpr = sh.nchunk > 4 ? NW : 1;      // wavefronts that join a row
    const size_t lds = (size_t)sh.waves * sh.rpt * c->head_dim * sizeof(float);
    const dim3 grid((unsigned)(c->kv_heads * sh.tiles), sh.nchunk);
    const dim3 join(grid.x, (unsigned)((sh.rpt * wpr + NW - 1) / NW));
#define ATTN(D, B)                                                            \
    do {                                                                      \
        if (sh.tile_rows > 16)                                                \
            hipLaunchKernelGGL((rows_kernel<D, B>), grid, dim3(NT), 0, s, a); \
        else if (!sh.one_tile)                                                \
            hipLaunchKernelGGL((attn_kernel<D, B, 4, false>), grid, dim3(4 * CT_WAVE), lds, s, a); \
        else if (sh.waves == 4)                                               \
            hipLaunchKernelGGL((attn_kernel<D, B, 4, true>), grid, dim3(4 * CT_WAVE), lds, s, a); \
        else                                                                  \
            hipLaunchKernelGGL((attn_kernel<D, B, 8, true>), grid, dim3(8 * CT_WAVE), lds, s, a); \
        if (sh.nchunk > 1) {                                                  \
            if (wpr == 1) hipLaunchKernelGGL((join_kernel<D, B, 1>), join, dim3(NT), 0, s, a);  \
            else hipLaunchKernelGGL((join_kernel<D, B, NW>), join, dim3(NT), 0, s, a);          \
        }                                                                     \
    } while (0)
    if (c->head_dim == 64) { if (p->bf16) ATTN(64, true); else ATTN(64, false); }
    else { if (p->bf16) ATTN(128, true); else ATTN(128, false); }
#undef ATTN
}
