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
#include <limits.h>
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
    // sequences with common tokens; partial results are [item][kv][row of the
    // item's tile] there, first those of the items of common tokens, tile_rows each
    const int *share;
    int most;                    // rows of a sequence
    int pitems, oitems;          // items of common and of own tokens in the grid
    int want[2], least[2];       // chunks aimed at, least steps of one
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
    int base;                    // keys below it are another tile's (shared launches)
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

// Inclusive prefix sum over a wavefront, without LDS: shifts by 1, 2, 4 and 8
// within rows of 16 lanes, then lane 15 into row 1 (and 47 into 3), lane 31 into
// rows 2 and 3.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}
// The same over the workgroup's W wavefronts.
template <int W>
__device__ __forceinline__ int group_sum(int v, int *part, int &total) {
    const int w = threadIdx.x / CT_WAVE;
    v = wave_scan(v);
    if (threadIdx.x % CT_WAVE == CT_WAVE - 1) part[w] = v;
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

// Sequences with common tokens.  A group's are E tokens: those that the caller
// names, as far as every row of the group sees them (no row masks any of them),
// if two sequences or more have rows.  All workgroups of the launches work
// out the same groups and the same chunks: a part's steps (of tiles, over all
// groups or sequences) are dealt in equal chunks to as many workgroups as are
// meant for it, since only the device knows how many tokens are common.
struct Groups {
    int lead[CT_KV8_SEQS];                                             // as given
    int least[CT_KV8_SEQS], rows[CT_KV8_SEQS], members[CT_KV8_SEQS];   // by leader
    int part[8], info[8], steps[2];
    __device__ __forceinline__ int common(int l) const { return members[l] > 1 ? least[l] : 0; }
};
struct Member {                  // thread s: sequence s, and what it leads
    int r0, n, len, lead, base;  // base: its group's common tokens
    int tiles[2], steps[2];      // tiles and steps of each: [0] over the common tokens of s's group, [1] over s's own
    int chunk[2];                // of all
    __device__ __forceinline__ int each(int part) const { return (steps[part] + chunk[part] - 1) / chunk[part]; }
};

// Every thread of a workgroup of at least CT_KV8_SEQS calls it.  What it reads
// is asked for at once: three rounds of loads, as the leaders lead to them, took
// 1.5 us more.
__device__ __forceinline__ Member read_groups(const Args &a, Groups &g) {
    const int s = threadIdx.x;
    Member m = {0, 0, 0, s, 0, {0, 0}, {0, 0}, {0, 0}};
    int l = -1;
    if (s < a.seqs) {
        m.r0 = a.rows[s];
        const int end = a.rows[s + 1], len = a.len[s], want = a.share[a.seqs + s];
        l = a.share[s];
        m.n = end - m.r0;
        m.len = max(len, 0);
        if (m.r0 < 0 || m.n <= 0 || m.n > a.n_rows - m.r0 || m.n > a.most) m.n = 0;
        g.least[s] = l == s ? max(want, 0) : 0;
        g.lead[s] = l;
        g.rows[s] = g.members[s] = 0;
    }
    if (s < 2) g.steps[s] = 0;
    __syncthreads();
    if ((unsigned)l < (unsigned)a.seqs && g.lead[l] == l) m.lead = l;
    if (m.n > 0) {
        const int sees = min(a.causal ? m.len - m.n + 1 : m.len, a.cap);
        atomicMin(&g.least[m.lead], max(sees, 0));
        atomicAdd(&g.rows[m.lead], m.n);
        atomicAdd(&g.members[m.lead], 1);
    }
    __syncthreads();
    if (s < a.seqs) {
        m.steps[0] = (g.common(s) + 31) >> 5;
        m.tiles[0] = m.steps[0] ? (g.rows[s] * a.group + a.tile_rows - 1) / a.tile_rows : 0;
        m.base = g.common(m.lead);
        m.tiles[1] = (m.n * a.group + 15) >> 4;
        m.steps[1] = max(min(m.len, a.cap) - (m.base & ~31) + 31, 0) >> 5;
        if (min(m.len, a.cap) <= m.base) m.tiles[1] = m.steps[1] = 0;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int all = wave_scan(m.tiles[i] * m.steps[i]);
        if ((s & (CT_WAVE - 1)) == CT_WAVE - 1) atomicAdd(&g.steps[i], all);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) m.chunk[i] = max((g.steps[i] + a.want[i] - 1) / a.want[i], a.least[i]);
    m.chunk[0] += m.chunk[0] & 1;            // the rows kernel takes two steps at a time
    return m;
}

// The keys that tile `tile` of a sequence's n rows has to itself: those past base.
__device__ __forceinline__ void own_keys(const Args &a, int tile, Tile &t) {
    t.row = tile * 16;
    t.pos0 = t.len - t.n;
    const int first = t.row / a.group, last = (min(t.row + 16, t.n * a.group) - 1) / a.group;
    t.end = max(min(a.causal ? t.pos0 + last + 1 : t.len, a.cap), 0);
    t.lo = t.base & ~31;
    t.sink_steps = 0;
    t.steps = t.end > t.base ? (t.end - t.lo + 31) >> 5 : 0;
    t.full_lo = t.base;
    t.full_hi = min(a.causal ? t.pos0 + first + 1 : t.len, a.cap);
}

// Where the sums of item `id` of the grid begin, of those with 16 rows at most a tile.
__device__ __forceinline__ long own_at(const Args &a, int id, int h, int rows) {
    if (id < a.pitems) return ((long)id * a.kv + h) * rows;
    return (long)a.pitems * a.kv * a.tile_rows + ((long)(id - a.pitems) * a.kv + h) * rows;
}

// Finds item `id`, a chunk of a tile, of part 0 or 1 (then row[i] becomes the
// i-th row of a tile of common tokens); returns its chunk, -1 if there is none.
template <int W>
__device__ __forceinline__ int find_item(const Args &a, int part, int id, Groups &g, int *row, Tile &t, int &chunk) {
    const Member m = read_groups(a, g);
    const int s = threadIdx.x;
    chunk = part ? m.chunk[1] : m.chunk[0];
    const int each = part ? m.each(1) : m.each(0), n = (part ? m.tiles[1] : m.tiles[0]) * each;
    int total;
    const int upto = group_sum<W>(n, g.part, total);
    if (id >= total) return -1;
    if (id >= upto - n && id < upto) {
        g.info[0] = s; g.info[1] = (id - (upto - n)) / each; g.info[2] = (id - (upto - n)) % each;
        if (part) {
            g.info[3] = m.n; g.info[4] = m.len; g.info[5] = m.r0; g.info[6] = m.base;
        } else {
            g.info[3] = g.rows[s]; g.info[4] = g.common(s);
        }
    }
    __syncthreads();
    t.seq = __builtin_amdgcn_readfirstlane(g.info[0]);
    const int tile = __builtin_amdgcn_readfirstlane(g.info[1]), ch = __builtin_amdgcn_readfirstlane(g.info[2]);
    t.n = __builtin_amdgcn_readfirstlane(g.info[3]);
    t.len = __builtin_amdgcn_readfirstlane(g.info[4]);
    if (part) {
        t.r0 = __builtin_amdgcn_readfirstlane(g.info[5]);
        t.base = __builtin_amdgcn_readfirstlane(g.info[6]);
        own_keys(a, tile, t);
        return ch;
    }
    t.row = tile * a.tile_rows;
    t.end = t.full_hi = t.len;
    t.r0 = t.pos0 = t.lo = t.sink_steps = t.full_lo = t.base = 0;
    t.steps = (t.end + 31) >> 5;
    const int mine = m.lead == t.seq ? m.n : 0, to = group_sum<W>(mine, g.part, total), from = to - mine;
    const int first = t.row / a.group, last = (min(t.row + a.tile_rows, t.n * a.group) - 1) / a.group;
    for (int i = max(from, first); i < min(to, last + 1); i++) row[i - first] = m.r0 + i - from;
    __syncthreads();
    return ch;
}

// Sequence `id`'s tile where no row masks a token: if all tokens of all its group
// are common and the group's rows fit one tile, they are the tile of its first
// sequence that has rows (then row[i] is the i-th), and there is none for the
// others; else the sequence's own rows, as find_tile finds them.
template <int W>
__device__ __forceinline__ bool find_group(const Args &a, int id, int *sh, int *row, Tile &t, bool &common) {
    const int s = threadIdx.x;
    int r0 = 0, n = 0, len = 0, l = -1;
    if (s < a.seqs) {
        r0 = a.rows[s];
        n = a.rows[s + 1] - r0;
        len = a.len[s];
        l = a.share[s];
        if (r0 < 0 || n <= 0 || n > a.n_rows - r0 || n > a.most) n = 0;
    }
    t.r0 = a.rows[id];
    t.n = a.rows[id + 1] - t.r0;
    t.len = max(a.len[id], 0);
    if (t.r0 < 0 || t.n <= 0 || t.n > a.n_rows - t.r0 || t.n > a.most) return false;
    t.end = min(t.len, a.cap);
    const int lead = a.share[id];
    const bool led = (unsigned)lead < (unsigned)a.seqs && a.share[lead] == lead && a.share[a.seqs + lead] >= t.end;
    // a sequence that holds other tokens, or too many rows, counts as 4096
    const int mine = led && l == lead ? (min(max(len, 0), a.cap) == t.end ? min(n, 4096) : n ? 4096 : 0) : 0;
    int total;
    const int to = group_sum<W>(mine, sh, total), from = to - mine;
    common = total > t.n && total * a.group <= 16;
    t.seq = id;
    if (common) {
        if (s == id) sh[W] = from;
        for (int i = from; i < to; i++) row[i] = r0 + i - from;
        __syncthreads();
        if (__builtin_amdgcn_readfirstlane(sh[W]) != 0) return false;
        t.seq = lead;
        t.n = total;
    }
    t.row = t.lo = t.sink_steps = t.full_lo = t.base = 0;
    t.pos0 = t.len - t.n;
    t.steps = (t.end + 31) >> 5;
    t.full_hi = t.end;
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
    // base: keys below it are another tile's
    __device__ __forceinline__ Sight(const Args &a, int len, int pos, int base) {
        first = 0;
        lo = base;
        n = max(min(a.causal ? pos + 1 : len, a.cap) - base, 0);
    }
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
template <int D, int NQ, bool SHARED>
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
            one[n][j] = in && (SHARED ? Sight(a, t.len, pos[n], t.base).sees(true, kk)
                                      : Sight(a, t.len, pos[n]).sees(a.window, kk)) ? (_Float16)1.0f : (_Float16)0.0f;
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
// HOW: ALONE, a sequence's rows.  APART, a workgroup takes either rows of a group
// over its common tokens (the first pitems items) or a sequence's rows over the
// others, and leaves its sums.  GROUPS, rows of a group that has all tokens in
// common, or else a sequence's.
enum How { ALONE, APART, GROUPS };
template <int D, bool BF16, int W, bool ONCE, How HOW>
__device__ __forceinline__ void attn_body(const Args &a, const int id, const int h, float *so) {
    constexpr int KS = D / 32;            // k steps of the score product
    constexpr int DI = D / 16;            // 16-dim tiles of O; dims of V a lane loads
    constexpr int NB = BF16 ? 1 : 2;      // f16 terms of a query value and of p
    constexpr bool SHARED = HOW == APART;
    // the wavefronts' sums so [W][rpt][D], maxima and l [W][16]: of the rows a tile
    // has, mostly one
    __shared__ int sh[W + 5];
    __shared__ float sm[W][16], sl[W][16];
    __shared__ std::conditional_t<SHARED, Groups, int> gr;
    __shared__ int grow[HOW != ALONE ? 16 : 1];  // rows of a tile of common tokens

    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE), c = lane & 15, g = lane >> 4;
    // this wavefront's steps: first, first + W, ...; lane i keeps the page and
    // the scales of 16-key half i (-1: not in the pool).  Where a step's keys do
    // not depend on the lengths, its page is read along with them.
    bool common = SHARED && id < a.pitems;
    int ch = blockIdx.y, chunk = a.chunk;
    Tile t;
    if constexpr (SHARED) ch = find_item<W>(a, !common, common ? id : id - a.pitems, gr, grow, t, chunk);
    const int first = ch * chunk + w;
    const bool ahead = HOW == ALONE && a.one_tile && !a.window;
    int key_i = 32 * (first + W * (lane >> 1)) + 16 * (lane & 1), pg = -1;
    if (ahead && (lane >> 1) * W < chunk && key_i < a.cap) pg = a.table[(long)id * a.table_w + (key_i >> a.lp)];
    if constexpr (HOW == ALONE)
        if (!find_tile<W>(a, id, 16, sh, t)) return;
    if constexpr (HOW == GROUPS)
        if (!find_group<W>(a, id, sh, grow, t, common)) return;
    const int chunks = !SHARED && a.nchunk > 1 ? (t.steps + chunk - 1) / chunk : 1;
    // a tile of own tokens may end before the last of its sequence's chunks
    if (SHARED ? ch < 0 || ch * chunk >= t.steps : ch >= max(chunks, 1)) return;
    const int last = min(t.steps, (ch + 1) * chunk);

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
    const int qrow = common ? grow[have ? qi - t.row / a.group : 0] : t.r0 + qi;
    fetch_query<D>(a, (long)qrow * a.ld_q + (long)(h * a.group + qh) * D, g, x);

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
    const int pos[1] = {common ? t.end - 1 : t.pos0 + qi};      // all rows see all common tokens
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
            const Sight see = SHARED ? Sight(a, t.len, pos[0], t.base) : Sight(a, t.len, pos[0]);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int k4 = (in[u] ? key + 16 * u : NO_KEY) + 4 * g;
                if (SHARED || a.window) see.mask(true, k4, s[u]);
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
        const bool more = st + 2 * W < last, out = SHARED && i + 2 == CT_WAVE / 2;
        if (more && !out) load(st + 2 * W, i + 2, ra);
        use(st + W, i + 1, rb);
        if constexpr (SHARED) {
            // Only the device knows how long the chunks of common and own tokens are:
            // after each 32 steps the lanes take the pages of the next ones.
            if (more && out) {
                const Args &z = args_again();
                const int mine = st + W * (2 + (lane >> 1)), key = step_key(t, mine) + 16 * (lane & 1);
                pg = mine < last && key < t.end ? z.table[(long)t.seq * z.table_w + (key >> z.lp)] : -1;
                if ((unsigned)pg >= (unsigned)z.pages) pg = -1;
                pks = pvs = 0.0f;
                if (pg >= 0) {
                    pks = z.ks[(long)pg * z.kv + h];
                    pvs = z.vs[(long)pg * z.kv + h];
                }
                load(st + 2 * W, 0, ra);
                // all loads (vmcnt 0): left pending they would make every step wait for the
                // next one's (64 rows, 8000 common tokens and up to 1000 more: 44.2 -> 46.6 us)
                __builtin_amdgcn_s_waitcnt(0x0f70);
                i = -2;
            }
        }
    }
    if (__builtin_expect(dirty, 0))
        for (int st = first; st < last; st += W) spread_nan<D, 1, SHARED>(a, t, h, step_key(t, st), c, g, pos, o);

    // the wavefronts' sums joined, in their order
    const int so_rows = HOW != ALONE ? 16 : a.rpt;
    l = sum_q(l);
    if (have) {
        if (g == 0) { sm[w][c] = m; sl[w][c] = l; }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < DI; i++) so[(w * so_rows + c) * D + (4 * g + j) * DI + i] = o[0][i][j];
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
            num += __builtin_amdgcn_ldexpf(so[(i * so_rows + r) * D + d], by);
            den += __builtin_amdgcn_ldexpf(sl[i][r], by);
        }
        if constexpr (SHARED) {
            const long at = own_at(a, id, h, common ? 16 : a.rpt) + r;
            a.part[at * D + d] = num;
            if (d == 0) a.stat[at] = make_float2(M, den);
        } else if (chunks <= 1) {
            const int R2 = t.row + r, i = a.group > 1 ? R2 / a.group : R2;
            const float y = den == 0.0f ? 0.0f : num * ONE_V / den;
            const long off = (long)(common ? grow[i] : t.r0 + i) * a.ld_out + (long)(h * a.group + R2 - i * a.group) * D + d;
            if (BF16) reinterpret_cast<uint16_t *>(a.out)[off] = f2bf(y);
            else reinterpret_cast<float *>(a.out)[off] = y;
        } else {
            const long at = (((long)id * a.kv + h) * a.nchunk + ch) * a.rpt + r;
            a.part[at * D + d] = num;
            if (d == 0) a.stat[at] = make_float2(M, den);
        }
    }
}

template <int D, bool BF16, int W, bool ONCE>
__global__ __launch_bounds__(W * CT_WAVE, BF16 ? 3 : 2) void attn_kernel(Args a) {
    extern __shared__ float so[];
    // heads vary fastest: workgroup i runs on XCD i % 8, so with 8 kv heads the
    // tiles of one head share an L2
    const int id = blockIdx.x / a.kv, h = blockIdx.x - id * a.kv;
    attn_body<D, BF16, W, ONCE, ALONE>(a, id, h, so);
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

// SHARED: the rows are a group's, the keys its common tokens; the sums are left.
template <int D>
using Operands = _Float16[2][4][D * 32];         // buffer; K, K, V, V of two 32-key steps

template <int D, bool BF16, bool SHARED>
__device__ __forceinline__ void rows_body(const Args &a, Operands<D> &lds) {
    constexpr int KS = D / 32, DI = D / 16, NB = BF16 ? 1 : 2;
    constexpr int ROWS = rows_of(BF16), WR = ROWS / NW, NQ = WR / 16;
    static_assert(2 * KS == DI, "K and V take the same number of operands");
    __shared__ int sh[NW + 5];
    // key scales and value scales' exponents (GONE: not in the pool) of each
    // iteration's four 16-key halves; two batches of 32 iterations in turn
    __shared__ __align__(16) float sscale[2][32][4];
    __shared__ __align__(16) int sexp[2][32][4];
    constexpr int GONE = KV8_MIN_EXP - 1;
    __shared__ int spos[ROWS];                 // the rows' positions, for the steps that not all see
    __shared__ int snan;                       // the V of some step holds a NaN

    const int h = blockIdx.x % a.kv, id = gridDim.x / a.kv - 1 - blockIdx.x / a.kv;
    __shared__ std::conditional_t<SHARED, Groups, int> gr;
    __shared__ int grow[SHARED ? ROWS : 1];
    int ch = blockIdx.y, chunk = a.chunk;
    Tile t;
    if constexpr (SHARED) {
        ch = find_item<NW>(a, 0, blockIdx.x / a.kv, gr, grow, t, chunk);
        if (ch < 0) return;
    } else {
        if (!find_tile<NW>(a, id, ROWS, sh, t)) return;
    }
    const int chunks = !SHARED && a.nchunk > 1 ? (t.steps + chunk - 1) / chunk : 1;
    if (!SHARED && ch >= max(chunks, 1)) return;
    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE), c = lane & 15, g = lane >> 4;
    const int all = t.n * a.group, hard = min(t.len, a.cap);

    const int wr0 = min(t.row + WR * w, all - 1), wr1 = min(t.row + WR * w + WR, all) - 1;
    const bool idle = t.row + WR * w >= all;
    const int p0 = t.pos0 + wr0 / a.group, p1 = t.pos0 + wr1 / a.group;
    const int full_lo = !SHARED && a.window ? p1 - a.window + 1 : 0;
    const int full_hi = SHARED ? t.full_hi : min(a.causal ? p0 + 1 : t.len, a.cap);
    const int wend = idle ? 0 : SHARED ? t.end : min(a.causal ? p1 + 1 : t.len, a.cap);

    // the unit this wavefront fetches: K (isv 0) or V of step 2 it + kb; lane i
    // keeps the page and place of half i & 1 of the step of iteration base + i / 2
    const int kb = w & 1, isv = w >> 1;
    const int s0 = ch * chunk, s1 = min(t.steps, s0 + chunk), iters = (s1 - s0 + 1) >> 1;
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
        const int row = SHARED ? grow[R / a.group - t.row / a.group] : t.r0 + R / a.group;
        fetch_query<D>(a, (long)row * a.ld_q + (long)(h * a.group + R % a.group) * D, g, x[n]);
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
        if (g == 0) spos[WR * w + 16 * n + c] = SHARED ? t.end - 1 : t.pos0 + (have ? R / a.group : 0);
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
                    const int pos = spos[WR * w + 16 * n + c];
                    const Sight see = SHARED ? Sight(a, t.len, pos, 0) : Sight(a, t.len, pos);
                    // one form for both kinds of mask: two took fp32 prompts from 120 to 124 us
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int j = 0; j < 4; j++) {
                            const int kk = (u < 2 ? k0 : k1) + 16 * (u & 1) + 4 * g + j;
                            s[n][u][j] = ev[u] == GONE ? -INFINITY : masked(see.sees(SHARED || a.window, kk), s[n][u][j]);
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
        for (int st = s0; st < s1; st++) spread_nan<D, NQ, SHARED>(z, t, h, step_key(t, st), c, g, pos, o);

#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const float den = sum_q(l[n]);
        const int r = WR * w + 16 * n + c, R = t.row + r;
        if (R >= all) continue;
        if constexpr (SHARED) {
            const long at = ((long)(blockIdx.x / z.kv) * z.kv + h) * ROWS + r;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < DI; i++) z.part[at * D + (4 * g + j) * DI + i] = o[n][i][j];
            if (g == 0) z.stat[at] = make_float2(m[n], den);
        } else if (chunks <= 1) {
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

template <int D, bool BF16>
__global__ __launch_bounds__(NT, 2) void rows_kernel(Args a) {
    __shared__ __align__(16) Operands<D> lds;
    rows_body<D, BF16, false>(a, lds);
}

// Common and own tokens in one launch: the first pitems items' workgroups wait for
// the matrix unit, the others for memory.  WIDE: common tokens in tiles of many
// rows.  64 rows, 32 heads over 8, 8000 common tokens and up to 1000 more, bf16 (105
// MB): 37 us and a join of 7, each sequence by itself 116; in a launch each 62 in all.
// An item of common tokens is 16 iterations of 64 keys, 27 us, one wavefront a SIMD;
// one of own tokens 12 us, of which finding the groups is 2 and the keys 5.
template <int D, bool BF16, bool WIDE>
__global__ __launch_bounds__(NT, WIDE || !BF16 ? 2 : 3) void shared_kernel(Args a) {
    constexpr int SUMS = NW * 16 * D * sizeof(float), OPS = sizeof(Operands<D>);
    __shared__ __align__(16) char mem[WIDE && OPS > SUMS ? OPS : SUMS];
    const int id = blockIdx.x / a.kv, h = blockIdx.x - id * a.kv;
    if (WIDE && id < a.pitems) rows_body<D, BF16, true>(a, reinterpret_cast<Operands<D> &>(mem));
    else attn_body<D, BF16, NW, true, APART>(a, id, h, reinterpret_cast<float *>(mem));
}

// Sequences whose tokens are all common, as a clip's hypotheses have them, in one
// launch: a workgroup for each of them, of which those that do not begin a group
// leave.  24 clips of up to 376 tokens, 5 hypotheses each, 8 heads, fp32 (13.6
// MB): 12.9 us, where a call of one workgroup takes 3.6; finding the group is some 2.
template <int D, bool BF16>
__global__ __launch_bounds__(NT, 2) void groups_kernel(Args a) {
    __shared__ __align__(16) float so[NW * 16 * D];
    const int id = blockIdx.x / a.kv, h = blockIdx.x - id * a.kv;
    attn_body<D, BF16, NW, true, GROUPS>(a, id, h, so);
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

// Joins the chunks of common tokens and of a sequence's own, a wavefront a packed
// row of a kv head, in that order.  A kv head's workgroups run on the XCD that
// wrote its sums.
template <int D, bool BF16>
__global__ __launch_bounds__(NT) void join_shared_kernel(Args a) {
    constexpr int DL = D / CT_WAVE;
    __shared__ Groups g;
    __shared__ int sr0[CT_KV8_SEQS], sn[CT_KV8_SEQS], slen[CT_KV8_SEQS], slead[CT_KV8_SEQS], sitem[2][CT_KV8_SEQS];
    const int h = blockIdx.x % a.kv, s = threadIdx.x;
    const Member m = read_groups(a, g);
    static_assert(NT == CT_KV8_SEQS, "a thread a sequence");
    sr0[s] = m.r0; sn[s] = m.n; slen[s] = m.len; slead[s] = m.lead;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        int total;
        const int n = m.tiles[i] * m.each(i);
        sitem[i][s] = group_sum<NW>(n, g.part, total) - n;       // ends with a barrier
    }
    __syncthreads();
    const int lane = threadIdx.x % CT_WAVE, w = __builtin_amdgcn_readfirstlane(threadIdx.x / CT_WAVE);
    const long packed = (long)(blockIdx.x / a.kv) * NW + w;
    const int r = (int)(packed / a.group), gq = (int)(packed % a.group), head = h * a.group + gq;
    if (r >= a.n_rows) return;
    int seq = -1;
#pragma unroll
    for (int i = 0; i < CT_KV8_SEQS / CT_WAVE; i++) {
        const int q = i * CT_WAVE + lane;
        const unsigned long long here = __ballot(sn[q] > 0 && r >= sr0[q] && r - sr0[q] < sn[q]);
        if (seq < 0 && here) seq = i * CT_WAVE + __builtin_ctzll(here);
    }
    if (seq < 0) return;                     // no sequence's row
    const int lead = __builtin_amdgcn_readfirstlane(slead[seq]);
    Tile t;
    t.n = sn[seq]; t.r0 = sr0[seq]; t.len = slen[seq];
    t.base = g.common(lead);
    const int row = (r - t.r0) * a.group + gq;
    own_keys(a, row / 16, t);
    // the row's place in its group
    int before = 0;
#pragma unroll
    for (int i = 0; i < CT_KV8_SEQS / CT_WAVE; i++) {
        const int q = i * CT_WAVE + lane;
        before += q < seq && slead[q] == lead ? sn[q] : 0;
    }
    before = __builtin_amdgcn_readlane(wave_scan(before), CT_WAVE - 1);
    const int grow = before * a.group + row;
    const int first = (((t.base + 31) >> 5) + m.chunk[0] - 1) / m.chunk[0];
    const int slots = __builtin_amdgcn_readfirstlane(first + (t.steps + m.chunk[1] - 1) / m.chunk[1]);
    const int each = (max(min(t.len, a.cap) - (t.base & ~31) + 31, 0) / 32 + m.chunk[1] - 1) / m.chunk[1];
    // sequences that name the same rows may have more items than the grid: no sums of them
    const int item0 = sitem[0][lead] + grow / a.tile_rows * first, item1 = sitem[1][seq] + row / 16 * each;
    if (item0 + first > a.pitems || item1 + slots - first > a.oitems) return;
    const long common = ((long)item0 * a.kv + h) * a.tile_rows + grow % a.tile_rows;
    const long own = own_at(a, a.pitems + item1, h, a.rpt) + row % 16;
    float M = -INFINITY, num[DL] = {}, den = 0.0f;
    constexpr int AT = 8;                    // slots in flight
    for (int k0 = 0; k0 < slots; k0 += AT) {
        float2 st[AT];
        float x[AT][DL];
#pragma unroll
        for (int u = 0; u < AT; u++) {
            const int k = k0 + u;
            st[u] = make_float2(-INFINITY, 0.0f);
            if (k < slots) {
                const long at = k < first ? common + (long)k * a.kv * a.tile_rows : own + (long)(k - first) * a.kv * a.rpt;
                st[u] = a.stat[at];
#pragma unroll
                for (int j = 0; j < DL; j++) x[u][j] = a.part[at * D + lane * DL + j];
            } else {
#pragma unroll
                for (int j = 0; j < DL; j++) x[u][j] = 0.0f;
            }
        }
        float mn = M;
#pragma unroll
        for (int u = 0; u < AT; u++) mn = fmaxf(mn, st[u].x);
        const int was = down(M - mn);
        M = mn;
        const float Mu = M == -INFINITY ? 0.0f : M;
        den = __builtin_amdgcn_ldexpf(den, was);
#pragma unroll
        for (int j = 0; j < DL; j++) num[j] = __builtin_amdgcn_ldexpf(num[j], was);
#pragma unroll
        for (int u = 0; u < AT; u++) {
            const int by = down(st[u].x - Mu);
            den += __builtin_amdgcn_ldexpf(st[u].y, by);
#pragma unroll
            for (int j = 0; j < DL; j++) num[j] += __builtin_amdgcn_ldexpf(x[u][j], by);
        }
    }
    const long off = (long)r * a.ld_out + (long)head * D + lane * DL;
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

// The arguments that a launch's shape does not change.
static Args args_of(const BackendKv8 *c, int layer, const BackendKv8Attn *p) {
    const long heads = (long)layer * c->pages * c->kv_heads;
    Args a = {};
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
    return a;
}

extern "C" void ctk_kv8_attn(const BackendKv8 *c, int layer, const BackendKv8Attn *p, hipStream_t s) {
    const Shape sh = shape_of(c, p);
    Args a = args_of(c, layer, p);
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

// ---- Sequences with common tokens ----

namespace {

constexpr int ITEMS = 512, WIDE_ITEMS = 128;     // items aimed at
constexpr double APART_BYTES = 192.0 * (1 << 20);
constexpr long JOIN_ROWS = 1L << 25;             // rows * query heads of a call
constexpr int OWN_ROWS = 64;     // packed rows of a sequence up to which common tokens are taken apart

struct SharedShape {
    int apart;                   // 0: every sequence through its own table
    int wide;                    // common tokens by the rows kernel
    int tile_rows, rpt, one_tile, want[2], least[2], items[2];
};

SharedShape shared_shape_of(const BackendKv8 *c, const BackendKv8Attn *a) {
    SharedShape s = {};
    const int group = a->heads / c->kv_heads, kv = c->kv_heads;
    const long each = (long)(a->max_rows < a->n_rows ? a->max_rows : a->n_rows) * group;
    const long all = (long)a->n_rows * group, steps = walk_of(c, a, 16);
    // Two launches and what finding the groups takes are 13 us at least, and codes
    // that several sequences read come from the caches: every sequence by itself
    // up to 192 MB of codes in all (120 sequences of up to 376 tokens, 92 MB:
    // 17.4 us against 19.0; 64 of 1100, 144 MB: 18.6, 22.1; 240 of up to 376,
    // 184 MB: 28.9, 27.2; 64 of 2200, four heads a group, 288 MB: 31.2, 28.6;
    // 64 of 9000, 1.2 GB: 116, 43.5).
    const double codes = (double)(c->seqs < a->n_rows ? c->seqs : a->n_rows) * steps * 32 * kv * 2 * c->head_dim;
    // The join has a wavefront for each row and head, whether a sequence has the row
    // or not: up to 2^25 of them, so that its grid stays below 2^32 threads too.
    s.apart = each <= OWN_ROWS && c->seqs > 1 && codes > APART_BYTES && (long)a->n_rows * a->heads <= JOIN_ROWS;
    if (!s.apart) return s;
    s.wide = all > 64;
    s.tile_rows = s.wide ? rows_of(a->bf16) : 16;
    s.one_tile = each <= 16;
    s.want[0] = ((s.wide ? WIDE_ITEMS : ITEMS) + kv - 1) / kv;
    s.want[1] = (ITEMS + kv - 1) / kv;
    s.least[0] = s.wide ? 16 : 8;
    s.least[1] = 8;
    // chunks of equal steps: those aimed at, and one a tile for rounding up
    s.items[0] = s.want[0] + (int)(all / s.tile_rows) + c->seqs / 2;
    s.items[1] = s.want[1] + (int)(all / 16) + c->seqs;
    s.rpt = each < 16 ? (int)each : 16;
    return s;
}

// Rows of partial results.
size_t rows_apart(const BackendKv8 *c, const SharedShape &s) {
    return ((size_t)s.items[0] * s.tile_rows + (size_t)s.items[1] * s.rpt) * c->kv_heads;
}

}  // namespace

extern "C" size_t ctk_kv8_attn_shared_need(const BackendKv8 *c, const BackendKv8Attn *a) {
    const SharedShape s = shared_shape_of(c, a);
    if (!s.apart) return ctk_kv8_attn_need(c, a);
    return rows_apart(c, s) * (c->head_dim + 2);
}

// Whatever a smaller call's shape: more rows or heads make no part of any smaller.
extern "C" size_t ctk_kv8_attn_shared_work(const BackendKv8 *c, const BackendKv8Attn *a) {
    size_t most = ctk_kv8_attn_work(c, a);
    const long kv = c->kv_heads, all = (long)a->n_rows * (a->heads / kv);
    const int rows[3] = {16, rows_of(false), rows_of(true)};
    for (int i = 0; i < 3; i++) {
        SharedShape s = {};
        s.tile_rows = rows[i];
        s.rpt = 16;
        s.items[0] = (int)(((i ? WIDE_ITEMS : ITEMS) + kv - 1) / kv + all / rows[i] + c->seqs / 2);
        s.items[1] = (int)((ITEMS + kv - 1) / kv + all / 16 + c->seqs);
        const size_t n = rows_apart(c, s) * (c->head_dim + 2);
        most = n > most ? n : most;
    }
    return most;
}

extern "C" void ctk_kv8_attn_shared(const BackendKv8 *c, int layer, const BackendKv8Attn *p, const int *share, hipStream_t s) {
    const SharedShape sh = shared_shape_of(c, p);
    const Shape plain = shape_of(c, p);
    // A group's rows in one workgroup, where all tokens may be common and there
    // are so many sequences that those that leave free CUs for it (fp32, 376
    // tokens, 8 heads, groups of sequences; us by groups / each alone: 13 of 5, 520
    // units 9.5 / 12.5; 24 of 5 13.1 / 17.3; 48 of 5 17.7 / 29.2; 40 of 3 with 60
    // tokens 9.0 / 11.2; but 1 of 64, 512 units 10.6 / 9.7; 24 of 2 11.4 / 10.4; bf16 8
    // of 8 with 700 tokens 16.9 / 12.4).  8 wavefronts each: 24 of 5 16.1.
    const bool groups = !sh.apart && !p->causal && plain.one_tile && plain.tile_rows == 16 && plain.nchunk == 1 &&
                        plain.tiles * c->kv_heads > 512;
    if (!sh.apart && !groups) {
        ctk_kv8_attn(c, layer, p, s);
        return;
    }
    Args a = args_of(c, layer, p);
    a.share = share;
    if (groups) {
        a.most = p->max_rows < p->n_rows ? p->max_rows : p->n_rows;
        a.one_tile = 1; a.chunk = plain.chunk; a.nchunk = 1;
        const dim3 grid((unsigned)(c->kv_heads * plain.tiles));
#define GROUPS(D, B) hipLaunchKernelGGL((groups_kernel<D, B>), grid, dim3(NT), 0, s, a)
        if (c->head_dim == 64) { if (p->bf16) GROUPS(64, true); else GROUPS(64, false); }
        else { if (p->bf16) GROUPS(128, true); else GROUPS(128, false); }
#undef GROUPS
        return;
    }
    a.most = p->max_rows < p->n_rows ? p->max_rows : p->n_rows;
    a.tile_rows = sh.tile_rows; a.one_tile = sh.one_tile; a.rpt = sh.rpt;
    for (int i = 0; i < 2; i++) { a.want[i] = sh.want[i]; a.least[i] = sh.least[i]; }
    a.pitems = sh.items[0];
    a.oitems = sh.items[1];
    a.part = p->work;
    a.stat = reinterpret_cast<float2 *>(p->work + rows_apart(c, sh) * c->head_dim);
    const dim3 grid((unsigned)(c->kv_heads * (sh.items[0] + sh.items[1])));
    const dim3 join((unsigned)(c->kv_heads * (((long)p->n_rows * a.group + NW - 1) / NW)));
#define SHARED(D, B)                                                                              \
    do {                                                                                          \
        if (sh.wide) hipLaunchKernelGGL((shared_kernel<D, B, true>), grid, dim3(NT), 0, s, a);    \
        else hipLaunchKernelGGL((shared_kernel<D, B, false>), grid, dim3(NT), 0, s, a);           \
        hipLaunchKernelGGL((join_shared_kernel<D, B>), join, dim3(NT), 0, s, a);                  \
    } while (0)
    if (c->head_dim == 64) { if (p->bf16) SHARED(64, true); else SHARED(64, false); }
    else { if (p->bf16) SHARED(128, true); else SHARED(128, false); }
#undef SHARED
}
