// k_kv8_attn.hip — softmax attention over the paged 8-bit key/value cache.
//
// A wavefront holds a tile of 16 query rows (tokens x query heads of one kv
// head) and walks over the keys 32 at a time, all in registers:
//   S^T = K Q^T   MFMA 16x16x32 f16, two 16-key halves; lane (c, g), c = lane
//                 % 16, g = lane / 16, holds query c's scores of keys 4g..4g+3
//                 of each half;
//   P             online softmax in base 2; the four lanes of a query share
//                 one running maximum;
//   O^T += V^T P^T  the same lane's eight p are one B operand if the product's
//                 k index runs over keys {4g..4g+3, 16+4g..16+4g+3}, so P
//                 never leaves its lane; V's rows are loaded to match, 8 dims
//                 a lane, and byte pairs of two keys interleaved (v_perm) on
//                 the way to f16.
// e4m3 values are f16 values, so codes are converted exactly and the products
// are those of the codes.  Scales are powers of two and never touch a code:
// the key scale multiplies the score; the value scale is an offset of the
// softmax exponent, relative to a running reference exponent (eref) of the
// sums: p' = 2^(s - m + 14 + e - eref) enters the product, O counts in units
// of 2^(eref - 14).  Query rows are brought to a largest value in [2^12, 2^13)
// by a power of two.  fp32 rows enter as the sum of two f16 (22 bits and
// more), and so do their p; bf16 rows are one f16 each, exactly, and so p.
#include "ct_dev.h"
#include "ct_kv8.h"
#include "k_kv8.h"

namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int NT = 256, NW = NT / CT_WAVE;   // threads, wavefronts of a workgroup
constexpr float LOG2E = 1.4426950408889634f;
constexpr int P_EXP = 14;                    // p' is at most 2^14

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
    int one_tile;                // every sequence's rows fit one tile: tile = sequence
    int chunk, nchunk;           // 32-key steps of a chunk, chunks of the grid
    int rpt;                     // rows of a tile kept in the partial results
    float *part;                 // partial O [tile][kv][chunk][rpt][D], then (m, l) pairs
    float2 *stat;
};

// A tile's rows and the keys they see: 32-key steps 0 .. sink_steps - 1 hold
// the first tokens, the rest start at lo (a multiple of 32).
struct Tile {
    int seq, r0, n, row;         // sequence, its first row and rows; first packed row of the tile
    int len, pos0;               // tokens held; position of the sequence's first row
    int end, lo, sink_steps, steps;
    int full_lo, full_hi;        // steps at keys in [full_lo, full_hi) are seen whole by every row
};

// Inclusive prefix sum over the workgroup.
__device__ __forceinline__ int scan256(int v, int *part, int &total) {
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
    for (int i = 0; i < NW; i++) {
        if (i < w) before += part[i];
        total += part[i];
    }
    __syncthreads();
    return v + before;
}

// Finds tile `id` (rows_per_tile packed rows each); false if there is none.
// Every thread of the workgroup calls it with the same id.
__device__ __forceinline__ bool find_tile(const Args &a, int id, int rows_per_tile, int *sh, Tile &t) {
    int tile = 0;
    if (a.one_tile) {
        t.seq = id;
    } else {
        int n = 0;
        const int s = threadIdx.x;
        if (s < a.seqs) {
            const int r0 = a.rows[s], r1 = a.rows[s + 1];
            if (r0 >= 0 && r1 > r0 && r1 <= a.n_rows)
                n = ((r1 - r0) * a.group + rows_per_tile - 1) / rows_per_tile;
        }
        int total;
        const int upto = scan256(n, sh, total);
        if (id >= total) return false;
        if (id >= upto - n && id < upto) { sh[NW] = s; sh[NW + 1] = id - (upto - n); }
        __syncthreads();
        t.seq = sh[NW];
        tile = sh[NW + 1];
    }
    t.r0 = a.rows[t.seq];
    t.n = a.rows[t.seq + 1] - t.r0;
    if (t.r0 < 0 || t.n <= 0 || t.r0 + t.n > a.n_rows) return false;
    t.row = tile * rows_per_tile;
    if (t.row >= t.n * a.group || (a.one_tile && t.n * a.group > rows_per_tile)) return false;
    t.len = max(a.len[t.seq], 0);
    t.pos0 = t.len - t.n;
    const int last = (min(t.row + rows_per_tile, t.n * a.group) - 1) / a.group;
    const int p0 = t.pos0 + t.row / a.group, p1 = t.pos0 + last;   // first and last row's positions
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

// The raw codes of one 32-key step: K as 16-byte pieces (half, 64-dim group),
// V as D / 16 dims of keys 4g + j (j < 4) and 16 + 4g + j - 4.
template <int D>
struct Raw {
    uint4 k[2][D / 64];
    uint32_t v[8][D / 64];
};

template <int D, bool BF16>
__global__ __launch_bounds__(NT) void attn_kernel(Args a) {
    constexpr int KS = D / 32;            // k steps of the score product
    constexpr int DI = D / 16;            // 16-dim tiles of O; dims of V a lane loads
    constexpr int NB = BF16 ? 1 : 2;      // f16 terms of a query value and of p
    __shared__ int sh[NW + 2];
    __shared__ float so[NW][16][D];
    __shared__ float sm[NW][16], sl[NW][16];

    // heads vary fastest: workgroup i runs on XCD i % 8, so with 8 kv heads the
    // tiles of one head share an L2
    const int h = blockIdx.x % a.kv, id = blockIdx.x / a.kv, ch = blockIdx.y;
    Tile t;
    if (!find_tile(a, id, 16, sh, t)) return;
    const int chunks = (t.steps + a.chunk - 1) / a.chunk;
    if (ch >= max(chunks, 1)) return;
    const int lane = threadIdx.x % CT_WAVE, w = threadIdx.x / CT_WAVE, c = lane & 15, g = lane >> 4;

    // this lane's query row, normalised and split
    const int R = t.row + c;
    const bool have = R < t.n * a.group;
    const int qi = have ? R / a.group : 0, qh = have ? R % a.group : 0;
    const int pos = t.pos0 + qi;
    f16x8 qf[NB][KS];
    float qs;
    {
        const long off = (long)(t.r0 + qi) * a.ld_q + (long)(h * a.group + qh) * D;
        float x[KS][8];
        float amax = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const long d = off + 64 * (i >> 1) + 16 * g + 8 * (i & 1) + j;
                const float u = BF16 ? bf2f(reinterpret_cast<const uint16_t *>(a.q)[d])
                                     : reinterpret_cast<const float *>(a.q)[d];
                x[i][j] = have ? u : 0.0f;
                amax = fmaxf(amax, fabsf(x[i][j]));
                bad |= !(fabsf(x[i][j]) < INFINITY);
            }
        amax = fmax_q(bad ? INFINITY : amax);
        // exponent of the row's largest value (zero and subnormal rows: 2^-126)
        const int e = amax < INFINITY ? max((int)(__float_as_uint(amax) >> 23), 1) - 127 : 0;
        // a row that is not finite has no scores
        qs = amax < INFINITY ? 1.0f : __uint_as_float(0x7fc00000u);
        const int up = 12 - e;               // in [-115, 138]: two factors
        const float f0 = pow2i(up >> 1), f1 = pow2i(up - (up >> 1));
        qs = qs * a.scale2 * pow2i((-up) >> 1) * pow2i(-up - ((-up) >> 1));
#pragma unroll
        for (int i = 0; i < KS; i++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = x[i][j] * f0 * f1;
                qf[0][i][j] = (_Float16)y;
                if (NB > 1) qf[NB - 1][i][j] = (_Float16)(y - (float)qf[0][i][j]);
            }
    }
    // keys this lane's query sees: [wlo, kend) and [0, sink_end)
    const int kend = have ? min(a.causal ? pos + 1 : t.len, a.cap) : 0;
    const int wlo = a.window ? pos - a.window + 1 : 0;
    const int hard = min(t.len, a.cap);      // tokens at and past it hold anything

    // this wavefront's steps: first, first + NW, ...; lane i keeps the page and
    // the scales of 16-key half i (-1: not in the pool)
    const int first = ch * a.chunk + w, last = min(t.steps, (ch + 1) * a.chunk);
    int pg = -1;
    float pks = 0.0f, pvs = 0.0f;
    {
        const int st = first + NW * (lane >> 1);
        if (st < last) {
            const int key = step_key(t, st) + 16 * (lane & 1);
            if (key < t.end) pg = a.table[(long)t.seq * a.table_w + (key >> a.lp)];
            if ((unsigned)pg >= (unsigned)a.pages) pg = -1;
            if (pg >= 0) {
                pks = a.ks[(long)pg * a.kv + h];
                pvs = a.vs[(long)pg * a.kv + h];
            }
        }
    }
    const int P = 1 << a.lp;
    auto load = [&](int st, int i, Raw<D> &r) {          // step st, this wavefront's i-th
        const int key = step_key(t, st);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int p = max(__builtin_amdgcn_readlane(pg, 2 * i + u), 0);   // any page if there is none
            const long base = ((((long)p * a.kv + h) << a.lp) + ((key + 16 * u) & (P - 1))) * D;
            const uint8_t *kp = a.k + base + c * D + 16 * g, *vp = a.v + base + 4 * g * D + c * DI;
#pragma unroll
            for (int x = 0; x < D / 64; x++) r.k[u][x] = *reinterpret_cast<const uint4 *>(kp + 64 * x);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (D == 128) {
                    const uint2 y = *reinterpret_cast<const uint2 *>(vp + j * D);
                    r.v[4 * u + j][0] = y.x;
                    r.v[4 * u + j][D / 64 - 1] = y.y;
                } else {
                    r.v[4 * u + j][0] = *reinterpret_cast<const uint32_t *>(vp + j * D);
                }
            }
        }
    };

    f32x4 o[DI];
#pragma unroll
    for (int i = 0; i < DI; i++) o[i] = (f32x4){0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    int eref = KV8_MIN_EXP, emax = KV8_MIN_EXP;

    auto use = [&](int st, int i, Raw<D> &r) {
        const int key = step_key(t, st);
        float s[2][4];
        int ev[2];
        bool in[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            in[u] = __builtin_amdgcn_readlane(pg, 2 * i + u) >= 0;
            const float ks = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(pks), 2 * i + u));
            ev[u] = max((int)(__builtin_amdgcn_readlane(__float_as_uint(pvs), 2 * i + u) >> 23 & 255) - 127, KV8_MIN_EXP);
            f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < D / 64; x++) {
                const f16x8 k0 = cvt8(r.k[u][x].x, r.k[u][x].y), k1 = cvt8(r.k[u][x].z, r.k[u][x].w);
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    acc = mfma_f16(k0, qf[b][2 * x], acc);
                    acc = mfma_f16(k1, qf[b][2 * x + 1], acc);
                }
            }
            const float f = qs * ks;
#pragma unroll
            for (int j = 0; j < 4; j++) s[u][j] = acc[j] * f;
        }
        const bool whole = key >= t.full_lo && key + 32 <= t.full_hi && in[0] && in[1];   // sink steps lie below full_lo
        uint32_t bad = 0;
        uint32_t vis = 0xff;                 // bit 4u + j: this lane's query sees key 16u + 4g + j
        if (!whole) {
            vis = 0;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int kk = key + 16 * u + 4 * g + j;
                    const bool see = in[u] && kk < kend && (kk >= wlo || kk < a.sinks);
                    if (see) vis |= 1u << (4 * u + j);
                    else s[u][j] = -INFINITY;
                    // a token nobody sees may hold anything: 0 * NaN is NaN
                    const bool any = in[u] && kk < hard;
#pragma unroll
                    for (int x = 0; x < D / 64; x++) {
                        if (!any) r.v[4 * u + j][x] = 0;
                        bad |= nan_bytes(r.v[4 * u + j][x]);
                    }
                }
        }
        float mt = s[0][0];
#pragma unroll
        for (int j = 1; j < 8; j++) mt = fmaxf(mt, s[j >> 2][j & 3]);
        mt = fmax_q(mt);
        // reference exponent of the sums: follows the value scales, but not
        // more than 60 below the largest one met
        const int e1 = max(in[0] ? ev[0] : KV8_MIN_EXP, in[1] ? ev[1] : KV8_MIN_EXP);
        emax = max(emax, e1);
        if (e1 > eref || e1 < eref - 8) {
            const int to = max(e1, emax - 60);
            const int by = max(min(eref - to, 126), -126);
            eref = to;
            const float f = pow2i(by);
#pragma unroll
            for (int i2 = 0; i2 < DI; i2++) o[i2] *= f;
        }
        if (__any(mt > m)) {
            const float mn = fmaxf(m, mt);
            const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int i2 = 0; i2 < DI; i2++) o[i2] *= al;
        }
        const float mu = m == -INFINITY ? 0.0f : m;
        f16x8 pf[NB];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int adj = max(in[u] ? P_EXP + ev[u] - eref : P_EXP, -40);
            const float ms = mu - (float)adj;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float p = __builtin_amdgcn_exp2f(s[u][j] - ms);
                sum += p;
                pf[0][4 * u + j] = (_Float16)p;
                if (NB > 1) pf[NB - 1][4 * u + j] = (_Float16)(p - (float)pf[0][4 * u + j]);
            }
            l += sum * pow2i(-adj);
        }
        if (__any(bad)) {
            // a NaN among values that some row sees and another does not: it
            // reaches the rows that see it, and they alone
            f16x8 one;
#pragma unroll
            for (int j = 0; j < 8; j++) one[j] = (vis >> j) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
            for (int x = 0; x < D / 64; x++)
#pragma unroll
                for (int b = 0; b < 4; b++) {
                    f16x8 hit;
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        hit[j] = (nan_bytes(r.v[j][x]) >> (8 * b + 7)) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
                    const f32x4 n = mfma_f16(hit, one, (f32x4){0, 0, 0, 0});
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (n[j] > 0.0f) o[4 * x + b][j] = __uint_as_float(0x7fc00000u);
                }
#pragma unroll
            for (int j = 0; j < 8; j++)
#pragma unroll
                for (int x = 0; x < D / 64; x++) {
                    const uint32_t z = nan_bytes(r.v[j][x]);
                    r.v[j][x] &= ~((z >> 7) * 0xffu);
                }
        }
#pragma unroll
        for (int x = 0; x < D / 64; x++) {
            // pairs of keys side by side: byte b of keys 2y, 2y + 1
            uint32_t lo[4], hi[4];
#pragma unroll
            for (int y = 0; y < 4; y++) {
                lo[y] = __builtin_amdgcn_perm(r.v[2 * y + 1][x], r.v[2 * y][x], 0x05010400u);
                hi[y] = __builtin_amdgcn_perm(r.v[2 * y + 1][x], r.v[2 * y][x], 0x07030602u);
            }
#pragma unroll
            for (int b = 0; b < 4; b++) {
                f16x8 vf;
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const f16x2 z = cvt2(b < 2 ? lo[y] : hi[y], b & 1);
                    vf[2 * y] = z[0];
                    vf[2 * y + 1] = z[1];
                }
#pragma unroll
                for (int n = 0; n < NB; n++) o[4 * x + b] = mfma_f16(vf, pf[n], o[4 * x + b]);
            }
        }
    };

    // two steps in flight
    Raw<D> ra, rb;
    if (first < last) load(first, 0, ra);
    for (int st = first, i = 0; st < last; st += 2 * NW, i += 2) {
        if (st + NW < last) load(st + NW, i + 1, rb);
        use(st, i, ra);
        if (st + NW >= last) break;
        if (st + 2 * NW < last) load(st + 2 * NW, i + 2, ra);
        use(st + NW, i + 1, rb);
    }

    // the wavefronts' sums joined, in their order
    l = sum_q(l);
    const float unit = pow2i(eref - P_EXP);
    if (have) {
        if (g == 0) { sm[w][c] = m; sl[w][c] = l; }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < DI; i++) so[w][c][(4 * g + j) * DI + i] = o[i][j] * unit;
    }
    __syncthreads();
    const int nr = min(16, t.n * a.group - t.row);
    for (int x = threadIdx.x; x < nr * D; x += NT) {
        const int r = x / D, d = x % D;
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < NW; i++) M = fmaxf(M, sm[i][r]);
        const float Mu = M == -INFINITY ? 0.0f : M;
        float num = 0.0f, den = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            const float f = __builtin_amdgcn_exp2f(sm[i][r] - Mu);
            num += f * so[i][r][d];
            den += f * sl[i][r];
        }
        if (chunks <= 1) {
            const int R2 = t.row + r;
            const float y = den == 0.0f ? 0.0f : num / den;
            const long off = (long)(t.r0 + R2 / a.group) * a.ld_out + (long)(h * a.group + R2 % a.group) * D + d;
            if (BF16) reinterpret_cast<uint16_t *>(a.out)[off] = f2bf(y);
            else reinterpret_cast<float *>(a.out)[off] = y;
        } else {
            const long at = (((long)id * a.kv + h) * a.nchunk + ch) * a.rpt + r;
            a.part[at * D + d] = num;
            if (d == 0) a.stat[at] = make_float2(M, den);
        }
    }
}

// Joins a tile's chunks, in their order: a wavefront a row.
template <int D, bool BF16>
__global__ __launch_bounds__(NT) void join_kernel(Args a) {
    __shared__ int sh[NW + 2];
    const int h = blockIdx.x % a.kv, id = blockIdx.x / a.kv;
    Tile t;
    if (!find_tile(a, id, 16, sh, t)) return;
    const int chunks = (t.steps + a.chunk - 1) / a.chunk;
    if (chunks <= 1) return;
    const int lane = threadIdx.x % CT_WAVE, nr = min(16, t.n * a.group - t.row);
    constexpr int DL = D / CT_WAVE;
    for (int r = threadIdx.x / CT_WAVE; r < nr; r += NW) {
        const long at = ((long)id * a.kv + h) * a.nchunk * a.rpt + r;
        float M = -INFINITY;
        for (int k = lane; k < chunks; k += CT_WAVE) M = fmaxf(M, a.stat[at + (long)k * a.rpt].x);
        M = wave_max(M);
        const float Mu = M == -INFINITY ? 0.0f : M;
        float num[DL] = {}, den = 0.0f;
        for (int k = 0; k < chunks; k++) {
            const float2 st = a.stat[at + (long)k * a.rpt];
            const float f = __builtin_amdgcn_exp2f(st.x - Mu);
            den += f * st.y;
#pragma unroll
            for (int j = 0; j < DL; j++) num[j] += f * a.part[(at + (long)k * a.rpt) * D + lane * DL + j];
        }
        const int R = t.row + r;
        const long off = (long)(t.r0 + R / a.group) * a.ld_out + (long)(h * a.group + R % a.group) * D + lane * DL;
#pragma unroll
        for (int j = 0; j < DL; j++) {
            const float y = den == 0.0f ? 0.0f : num[j] / den;
            if (BF16) reinterpret_cast<uint16_t *>(a.out)[off + j] = f2bf(y);
            else reinterpret_cast<float *>(a.out)[off + j] = y;
        }
    }
}

// The launch's shape, from the sizes alone.
struct Shape {
    int one_tile, tiles, chunk, nchunk, rpt;
};

Shape shape_of(const BackendKv8 *c, const BackendKv8Attn *a) {
    Shape s;
    const int group = a->heads / c->kv_heads;
    const long rows = (long)(a->max_rows < a->n_rows ? a->max_rows : a->n_rows) * group;   // of a sequence
    s.one_tile = rows <= 16;
    s.tiles = s.one_tile ? c->seqs : (int)((long)a->n_rows * group / 16 + c->seqs);
    s.rpt = rows < 16 ? (int)rows : 16;
    long keys = (long)c->table_w * c->page_tokens;
    if (a->max_len > 0 && a->max_len < keys) keys = a->max_len;
    // the longest walk of a tile, in steps
    long steps = (keys + 31) / 32;
    if (a->window > 0) {
        const long span = ((long)a->window + 16 + 62) / 32 + ((long)a->sinks + 31) / 32;
        if (span < steps) steps = span;
    }
    s.chunk = (long)s.tiles * c->kv_heads >= 1024 ? 128 : 16;
    s.nchunk = (int)((steps + s.chunk - 1) / s.chunk);
    if (s.nchunk < 1) s.nchunk = 1;
    return s;
}

}  // namespace

extern "C" size_t ctk_kv8_attn_work(const BackendKv8 *c, const BackendKv8Attn *a) {
    const Shape s = shape_of(c, a);
    if (s.nchunk == 1) return 0;
    return (size_t)s.tiles * c->kv_heads * s.nchunk * s.rpt * (c->head_dim + 2);
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
    a.one_tile = sh.one_tile; a.chunk = sh.chunk; a.nchunk = sh.nchunk; a.rpt = sh.rpt;
    const size_t n = (size_t)sh.tiles * c->kv_heads * sh.nchunk * sh.rpt;
    a.part = p->work;
    a.stat = sh.nchunk > 1 ? reinterpret_cast<float2 *>(p->work + n * c->head_dim) : nullptr;
    const dim3 grid((unsigned)(c->kv_heads * sh.tiles), sh.nchunk), join((unsigned)(c->kv_heads * sh.tiles));
#define ATTN(D, B)                                                            \
    do {                                                                      \
        hipLaunchKernelGGL((attn_kernel<D, B>), grid, dim3(NT), 0, s, a);     \
        if (sh.nchunk > 1)                                                    \
            hipLaunchKernelGGL((join_kernel<D, B>), join, dim3(NT), 0, s, a); \
    } while (0)
    if (c->head_dim == 64) { if (p->bf16) ATTN(64, true); else ATTN(64, false); }
    else { if (p->bf16) ATTN(128, true); else ATTN(128, false); }
#undef ATTN
}
