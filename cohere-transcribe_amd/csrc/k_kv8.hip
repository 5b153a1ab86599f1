// k_kv8.hip — the paged 8-bit key/value cache: rows rounded into pages, and
// the page book-keeping (reserve, fork, free, trim, compact).
//
// Codes are e4m3 with one power-of-two scale s = 2^e per (page, kv head):
// value = code * s.  e is the smallest with amax <= 448 * 2^e, read off amax's
// exponent and fraction, so x / s is exact and each value is rounded once, by
// the conversion instruction (to nearest, ties to even).  A float format does
// not gain from a finer scale: its relative step is the same in every binade.
#include "ct_dev.h"
#include "ct_kv8.h"
#include "k_kv8.h"

namespace {

constexpr int NT = 256;     // threads of an append or copy workgroup
constexpr int PNT = 1024;   // threads of a planning workgroup

// Inclusive prefix sum over the workgroup's threads; `total` gets the sum.
// part: one int per wavefront.  Ends with a barrier, so part may be reused.
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, int *part, int &total) {
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
    for (int i = 0; i < THREADS / CT_WAVE; i++) {
        const int p = part[i];
        if (i < w) before += p;
        total += p;
    }
    __syncthreads();
    return v + before;
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------

// 8 values of a row, as they lie in memory.
template <bool BF16>
struct Piece;
template <>
struct Piece<true> {
    u16x8 v;
    __device__ __forceinline__ void load(const void *p, long off, bool vec) {
        const uint16_t *q = reinterpret_cast<const uint16_t *>(p) + off;
        if (vec) v = *reinterpret_cast<const u16x8 *>(q);
        else
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = q[i];
    }
    __device__ __forceinline__ float at(int i) const { return bf2f(v[i]); }
};
template <>
struct Piece<false> {
    f32x4 v[2];
    __device__ __forceinline__ void load(const void *p, long off, bool vec) {
        const float *q = reinterpret_cast<const float *>(p) + off;
        if (vec) {
#pragma unroll
            for (int i = 0; i < 2; i++) v[i] = reinterpret_cast<const f32x4 *>(q)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i >> 2][i & 3] = q[i];
        }
    }
    __device__ __forceinline__ float at(int i) const { return v[i >> 2][i & 3]; }
};

// Exponent of the smallest 2^e >= 2^-100 with amax <= 448 * 2^e; amax finite,
// >= 0.  448 = 1.75 * 2^8.
__device__ __forceinline__ int need_exp(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffff) > 0x600000);
    return max(e, KV8_MIN_EXP);   // also zero and subnormals (exponent field 0)
}

// x * inv (a power of two) held within +-448; NaN stays NaN.
__device__ __forceinline__ float clamp448(float x) {
    x = x > 448.0f ? 448.0f : x;
    return x < -448.0f ? -448.0f : x;
}

template <bool BF16>
__device__ __forceinline__ uint2 codes8(const Piece<BF16> &x, float inv) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = clamp448(x.at(i) * inv);
    uint2 r;
    int a = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    r.x = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], a, true);
    a = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    r.y = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], a, true);
    return r;
}

// Codes of a smaller scale rounded again for one that is 1 / ratio times as
// large (ratio < 1, a power of two).
__device__ __forceinline__ uint32_t recode4(uint32_t c, float ratio) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
    const int r = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * ratio, a[1] * ratio, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(b[0] * ratio, b[1] * ratio, r, true);
}

// One workgroup per (page a sequence's new rows touch, kv head, K or V).  The
// rows' values stay in registers between the search for their largest and
// their rounding: each is read once and its code written once.
// Pieces (pages touched) are numbered sequence by sequence; a workgroup finds
// its own by a prefix sum over the sequences, so the grid follows n_rows and
// not the longest sequence: at most n_rows, and n_rows / page_tokens + 2 *
// seqs.  Heads vary fastest, then K and V: the workgroups of a piece, which
// read parts of the same rows, run together.
// Bound by memory where there are many rows: 66439 bf16 rows of 8 x 128 (408
// MB) take 87 us, 4.7 TB/s of the 4.8 a copy reaches; 6156 fp32 rows (63 MB)
// 17 us.  64 single rows take 5 us, launch and chain of dependent loads (rows
// -> table -> scale and refs).  The 6156 rows took 20.5 us with rows loaded
// non-temporally: a step's keys and values come from a product just before.
template <int D, bool BF16>
__global__ __launch_bounds__(NT) void append_kernel(BackendKv8 c, int layer, const void *xk, const void *xv,
                                                    long ld, int vec, const int *rows, int n_rows, int lp) {
    constexpr int TPR = D / 8;            // threads of a row
    constexpr int RPP = NT / TPR;         // rows of a pass
    constexpr int MAXP = 128 / RPP;       // passes of the largest page
    __shared__ int part[NT / CT_WAVE];
    __shared__ int own[4];                // first row, first position, end, sequence of the piece
    __shared__ float wmax[NT / CT_WAVE];
    const int P = 1 << lp, t = threadIdx.x;
    const long cap = (long)c.table_w << lp;

    int r0 = 0, a = 0, e = 0, n = 0;      // this thread's sequence: rows, positions [a, e), pieces
    if (t < c.seqs) {
        r0 = rows[t];
        const int r1 = rows[t + 1], len = c.len[t];
        if (r0 >= 0 && r1 > r0 && r1 <= n_rows && len > 0) {
            const int first = len - (r1 - r0);
            e = (int)min((long)len, cap);
            a = max(first, 0);
            r0 += a - first;
            if (e > a) n = ((e - 1) >> lp) - (a >> lp) + 1;
        }
    }
    int total;
    const int upto = block_scan<NT>(n, part, total);
    const int piece = blockIdx.x / (2 * c.kv_heads);
    if (piece >= total) return;           // the same for every thread
    if (piece >= upto - n && piece < upto) {
        const int p0 = ((a >> lp) + piece - (upto - n)) << lp;   // first token of the page
        const int b = max(a, p0);
        own[0] = r0 + (b - a);
        own[1] = b;
        own[2] = min(e, p0 + P);
        own[3] = t;
    }
    __syncthreads();
    const int row0 = own[0], pos0 = own[1], m = own[2] - pos0, tok0 = pos0 & (P - 1);
    const bool isv = blockIdx.x / c.kv_heads & 1;
    const int h = blockIdx.x % c.kv_heads;
    const void *x = isv ? xv : xk;
    // the rows and the page are asked for together
    const int tr = t / TPR, col = t % TPR * 8;
    Piece<BF16> val[MAXP];
#pragma unroll
    for (int i = 0; i < MAXP; i++) {
        const int r = i * RPP + tr;
        if (r < m) val[i].load(x, (row0 + r) * ld + h * D + col, vec);
    }
    const int page = c.table[(long)own[3] * c.table_w + (pos0 >> lp)];
    if ((unsigned)page >= (unsigned)c.pages) return;
    const long at = ((long)layer * c.pages + page) * c.kv_heads + h;
    uint8_t *codes = (isv ? c.v : c.k) + (at << lp) * D;
    float *scale = (isv ? c.vscale : c.kscale) + at;
    const float was = tok0 ? *scale : 0.0f;      // read before any thread writes it
    if (c.refs[page] > 1) return;                // the same for every thread

    float amax = 0.0f;
#pragma unroll
    for (int i = 0; i < MAXP; i++) {
        const int r = i * RPP + tr;
        if (r < m) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float u = fabsf(val[i].at(j));
                amax = u < INFINITY ? fmaxf(amax, u) : amax;     // finite values only
            }
        }
    }
    amax = wave_max(amax);
    if (t % CT_WAVE == 0) wmax[t / CT_WAVE] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / CT_WAVE; i++) amax = fmaxf(amax, wmax[i]);
    const int ne = need_exp(amax);
    float now = __uint_as_float((uint32_t)(ne + 127) << 23);
    if (tok0 && !(was < now)) now = was;
    else if (tok0) {
        // the page's scale grows: round what it holds again
        const float ratio = was / now;
        for (int q = t; q < tok0 * (D / 16); q += NT) {
            uint4 w = reinterpret_cast<uint4 *>(codes)[q];
            w.x = recode4(w.x, ratio); w.y = recode4(w.y, ratio);
            w.z = recode4(w.z, ratio); w.w = recode4(w.w, ratio);
            reinterpret_cast<uint4 *>(codes)[q] = w;
        }
    }
    const float inv = 1.0f / now;
    if (t == 0) *scale = now;
#pragma unroll
    for (int i = 0; i < MAXP; i++) {
        const int r = i * RPP + tr;
        if (r < m) *reinterpret_cast<uint2 *>(codes + (long)(tok0 + r) * D + col) = codes8(val[i], inv);
    }
}

// ---------------------------------------------------------------------------
// Pages
// ---------------------------------------------------------------------------

__device__ __forceinline__ void flag(const BackendKv8 &c, int bit) { atomicOr(c.plan + CT_KV8_STATUS, bit); }

// Places of the plan past its header.
__device__ __forceinline__ int *plan_pairs(const BackendKv8 &c) { return c.plan + CT_KV8_HEAD; }
__device__ __forceinline__ int *plan_table(const BackendKv8 &c) { return plan_pairs(c) + 4 * c.seqs; }
__device__ __forceinline__ int *plan_from(const BackendKv8 &c) {
    return plan_table(c) + (long)c.seqs * c.table_w;
}
__device__ __forceinline__ int *plan_to(const BackendKv8 &c) { return plan_from(c) + max(c.pages, c.seqs); }

// A planning thread's run of pages and which of the first 64 of them are
// free, asked for before the rest of the plan needs them.
// One workgroup reads the whole pool's counts, so a reserve of 64 or 256
// sequences takes 3.8 us with 2000 pages, 10.7 with 16000 and 90 with 200000.
struct FreeRun {
    int p0, p1, n;
    uint64_t mask;
    __device__ __forceinline__ FreeRun(const BackendKv8 &c) {
        const int per = (c.pages + PNT - 1) / PNT;
        p0 = min((int)threadIdx.x * per, c.pages);
        p1 = min(p0 + per, c.pages);
        n = 0;
        mask = 0;
        for (int p = p0; p < p1; p++) {
            const bool f = c.refs[p] == 0;
            n += f;
            if (p - p0 < 64) mask |= (uint64_t)f << (p - p0);
        }
    }
    // Calls take(rank, page) for the lowest `want` free pages, in ascending
    // order of page; returns the number of free pages.  Nothing is taken if
    // there are fewer.  All of the workgroup's threads call it.
    template <class Take>
    __device__ __forceinline__ int take(const BackendKv8 &c, int want, int *part, Take take) const {
        int total;
        int r = block_scan<PNT>(n, part, total) - n;
        if (total >= want)
            for (int p = p0; p < p1 && r < want; p++)
                if (p - p0 < 64 ? mask >> (p - p0) & 1 : c.refs[p] == 0) take(r++, p);
        return total;
    }
};

__global__ __launch_bounds__(PNT) void reserve_kernel(BackendKv8 c, const int *add, int lp) {
    __shared__ int part[PNT / CT_WAVE];
    __shared__ int off[CT_KV8_SEQS + 1], col[CT_KV8_SEQS];
    __shared__ int bad;
    const int t = threadIdx.x, P = 1 << lp;
    const long cap = (long)c.table_w << lp;
    const FreeRun run(c);
    if (t == 0) bad = 0;
    __syncthreads();
    int n = 0, a = 0, len = 0, first = 0;
    if (t < c.seqs) {
        a = add[t];
        len = c.len[t];
        if (a < 0 || len < 0) atomicOr(&bad, KV8_BAD_ARG);
        else if ((long)len + a > cap) atomicOr(&bad, KV8_NO_ROOM);
        else {
            first = (len + P - 1) >> lp;
            n = ((len + a + P - 1) >> lp) - first;
        }
        if (a < 0 || a > cap) a = 0;               // refused; keeps the sums in range
    }
    int rows, want;
    const int upto = block_scan<PNT>(n, part, want);
    if (t < c.seqs) { off[t] = upto - n; col[t] = first; }
    // rows: at most 256 * 2^24, summed as counts of 2^8 and rest to stay in 32 bits
    int hi, rest;
    const int uhi = block_scan<PNT>(a >> 8, part, hi), ulo = block_scan<PNT>(a & 255, part, rest);
    const long all = ((long)hi << 8) + rest;
    if (all > CT_KV8_ROWS && t == 0) bad |= KV8_BAD_ARG;
    __syncthreads();
    int refuse = bad;
    rows = (int)min(((long)uhi << 8) + ulo, (long)CT_KV8_ROWS);
    if (!refuse && want > 0) {
        const int have = run.take(c, want, part, [&](int r, int p) {
            int lo = 0, up = c.seqs - 1;           // the last sequence with off <= r
            while (lo < up) {
                const int mid = (lo + up + 1) >> 1;
                if (off[mid] <= r) lo = mid;
                else up = mid - 1;
            }
            c.table[(long)lo * c.table_w + col[lo] + (r - off[lo])] = p;
            c.refs[p] = 1;
        });
        if (have < want) refuse = KV8_NO_PAGES;
    }
    if (refuse) {
        if (t <= c.seqs) c.rows[t] = 0;
        if (t == 0) flag(c, refuse);
        return;
    }
    if (t == 0) c.rows[0] = 0;
    if (t < c.seqs) {
        c.rows[t + 1] = rows;
        c.len[t] = len + a;
    }
}

// Fork, first of two launches (a fork of 128 beams, 193 MB of copied pages,
// takes 41 us, one of 5 beams 8 us; with a third launch, and ordinary stores in
// the copies, 54 and 14).  The workgroups past the first set the sources' table
// rows aside.  The first checks the pairs and picks the pages
// that partly filled last pages are copied to: for pair i the plan gets the
// source sequence (-1: nothing to do), the table column of the copied page
// (-1: none), its new page and the source's length; and the pages to copy.
__global__ __launch_bounds__(PNT) void fork_plan_kernel(BackendKv8 c, const int *dst, const int *src, int n, int cols,
                                                        int lp) {
    if (blockIdx.x > 0) {
        const int i = (blockIdx.x - 1) / cols, j = (blockIdx.x - 1) % cols * PNT + threadIdx.x;
        const int s = src[i];
        if ((unsigned)s < (unsigned)c.seqs && j < c.table_w)
            plan_table(c)[(long)i * c.table_w + j] = c.table[(long)s * c.table_w + j];
        return;
    }
    __shared__ int part[PNT / CT_WAVE];
    __shared__ int seen[CT_KV8_SEQS], who[CT_KV8_SEQS], from[CT_KV8_SEQS];
    __shared__ int bad;
    const int t = threadIdx.x, P = 1 << lp;
    const FreeRun run(c);
    if (t == 0) bad = 0;
    if (t < CT_KV8_SEQS) seen[t] = 0;
    __syncthreads();
    int s = -1, col = -1, len = 0, old = -1;
    if (t < n) {
        const int d = dst[t];
        s = src[t];
        if ((unsigned)d >= (unsigned)c.seqs || (unsigned)s >= (unsigned)c.seqs) atomicOr(&bad, 1);
        else {
            if (atomicAdd(&seen[d], 1)) atomicOr(&bad, 1);
            len = c.len[s];
            if (len < 0 || len > (long)c.table_w << lp) atomicOr(&bad, 1);
            else if (d == s) s = -1;
            else if (len & (P - 1)) {
                old = c.table[(long)s * c.table_w + (len >> lp)];
                if ((unsigned)old < (unsigned)c.pages) col = len >> lp;
            }
        }
    }
    int want;
    const int r = block_scan<PNT>(col >= 0, part, want) - 1;     // ends with a barrier: bad is whole
    if (col >= 0) { who[r] = t; from[r] = old; }
    __syncthreads();
    int refuse = bad ? KV8_BAD_ARG : 0;
    int *pairs = plan_pairs(c);
    if (!refuse && want > 0) {
        const int have = run.take(c, want, part, [&](int i, int p) {
            pairs[4 * who[i] + 2] = p;
            c.refs[p] = 1;
            plan_from(c)[i] = from[i];
            plan_to(c)[i] = p;
        });
        if (have < want) refuse = KV8_NO_PAGES;
    }
    if (t < n) {
        pairs[4 * t] = refuse ? -1 : s;
        pairs[4 * t + 1] = col;
        pairs[4 * t + 3] = len;
    }
    if (t == 0) {
        c.plan[CT_KV8_COUNT] = refuse ? 0 : want;
        if (refuse) flag(c, refuse);
    }
}

// Bound by memory: 893 pages of 32 tokens in 8 layers (577 MB read and
// written) move in 108 us, 5.3 TB/s; non-temporal, as neither side is used
// soon (129 against 118 us for the whole call).
// Copies page `from` to page `to` in every layer: unit u of a page is one
// layer's K or V, `bytes` of codes and kv_heads scales; a workgroup takes
// 16 KB parts of units, all over the grid.
__device__ __forceinline__ void copy_pages(const BackendKv8 &c, int lp, int first, int step) {
    const int count = c.plan[CT_KV8_COUNT];
    const long bytes = (long)c.kv_heads * c.head_dim << lp;
    const int parts = (int)((bytes + 16383) >> 14);
    const int *from = plan_from(c), *to = plan_to(c);
    const long items = (long)count * c.layers * 2 * parts;
    for (long i = first; i < items; i += step) {
        const int part = (int)(i % parts);
        const long u = i / parts;
        const int isv = (int)(u & 1);
        const long pl = u >> 1;
        const int lay = (int)(pl % c.layers), r = (int)(pl / c.layers);
        const long a = (long)lay * c.pages + from[r], b = (long)lay * c.pages + to[r];
        uint8_t *pool = isv ? c.v : c.k;
        const u32x4 *p = reinterpret_cast<const u32x4 *>(pool + a * bytes);
        u32x4 *q = reinterpret_cast<u32x4 *>(pool + b * bytes);
        const int w0 = part << 10, w1 = (int)min((long)w0 + 1024, bytes >> 4);
        u32x4 x[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int w = w0 + j * NT + threadIdx.x;
            if (w < w1) x[j] = __builtin_nontemporal_load(p + w);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int w = w0 + j * NT + threadIdx.x;
            if (w < w1) __builtin_nontemporal_store(x[j], q + w);
        }
        if (part == 0 && (int)threadIdx.x < c.kv_heads) {
            float *sc = isv ? c.vscale : c.kscale;
            sc[b * c.kv_heads + threadIdx.x] = sc[a * c.kv_heads + threadIdx.x];
        }
    }
}

// Fork, second launch: the rows set aside, with the copied pages in their
// places, replace the old ones; pages gain and lose a holder.  The workgroups
// behind copy the partly filled pages.
__global__ __launch_bounds__(NT) void fork_swap_kernel(BackendKv8 c, const int *dst, int n, int cols, int lp) {
    const int books = n * cols;
    if ((int)blockIdx.x >= books) {
        copy_pages(c, lp, blockIdx.x - books, gridDim.x - books);
        return;
    }
    const int i = blockIdx.x / cols, j = blockIdx.x % cols * NT + threadIdx.x;
    const int *pair = plan_pairs(c) + 4 * i;
    if (pair[0] < 0) return;
    const int d = dst[i], used = (pair[3] + (1 << lp) - 1) >> lp;
    if (j == 0) c.len[d] = pair[3];
    if (j >= c.table_w) return;
    int *e = c.table + (long)d * c.table_w + j;
    const int old = *e;
    int p = -1;
    if (j < used) {
        if (j == pair[1]) p = pair[2];             // counted when it was taken
        else {
            p = plan_table(c)[(long)i * c.table_w + j];
            if ((unsigned)p < (unsigned)c.pages) atomicAdd(c.refs + p, 1);
        }
    }
    *e = p;
    if ((unsigned)old < (unsigned)c.pages) atomicSub(c.refs + old, 1);
}

// Table entries [lo, hi) of a sequence given back: each entry is taken out
// once, whoever else frees it.
__device__ __forceinline__ void give_back(const BackendKv8 &c, int s, int j) {
    const int old = atomicExch(c.table + (long)s * c.table_w + j, -1);
    if ((unsigned)old < (unsigned)c.pages) atomicSub(c.refs + old, 1);
}

__global__ __launch_bounds__(NT) void free_kernel(BackendKv8 c, const int *seqs, int n, int cols) {
    __shared__ int bad;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    if ((int)threadIdx.x < n && (unsigned)seqs[threadIdx.x] >= (unsigned)c.seqs) atomicOr(&bad, 1);
    __syncthreads();
    if (bad) {
        if (blockIdx.x == 0 && threadIdx.x == 0) flag(c, KV8_BAD_ARG);
        return;
    }
    const int s = seqs[blockIdx.x / cols], j = blockIdx.x % cols * NT + threadIdx.x;
    if (j == 0) c.len[s] = 0;
    if (j < c.table_w) give_back(c, s, j);
}

__global__ __launch_bounds__(NT) void trim_kernel(BackendKv8 c, int window, int sinks, int cols, int lp) {
    const int s = blockIdx.x / cols, j = blockIdx.x % cols * NT + threadIdx.x;
    // the next row, at position len, sees tokens from len - window + 1
    const long seen = (long)c.len[s] - window + 1;
    const long lo = ((long)sinks + (1 << lp) - 1) >> lp, hi = seen < 0 ? 0 : min(seen >> lp, (long)c.table_w);
    if (j >= lo && j < hi) give_back(c, s, j);
}

// Compact, first of two launches: pages in use at m and above (m pages are in
// use) are paired, in ascending order, with the free ones below m.
__global__ __launch_bounds__(PNT) void compact_plan_kernel(BackendKv8 c) {
    __shared__ int part[PNT / CT_WAVE];
    const int per = (c.pages + PNT - 1) / PNT, p0 = min((int)threadIdx.x * per, c.pages), p1 = min(p0 + per, c.pages);
    int n = 0, live, moves, holes;
    for (int p = p0; p < p1; p++) n += c.refs[p] != 0;
    block_scan<PNT>(n, part, live);
    int mv = 0, ho = 0;
    for (int p = p0; p < p1; p++) {
        const bool used = c.refs[p] != 0;
        mv += used && p >= live;
        ho += !used && p < live;
    }
    int r = block_scan<PNT>(mv, part, moves) - mv, q = block_scan<PNT>(ho, part, holes) - ho;
    int *from = plan_from(c), *to = plan_to(c);
    for (int p = p0; p < p1; p++) {
        const bool used = c.refs[p] != 0;
        if (used && p >= live) from[r++] = p;
        if (!used && p < live) to[q++] = p;
    }
    __threadfence_block();
    __syncthreads();
    // the lists are in ascending order, so a page's new place is found by
    // bisection when the tables are rewritten
    for (int i = threadIdx.x; i < moves; i += PNT) {
        c.refs[to[i]] = c.refs[from[i]];
        c.refs[from[i]] = 0;
    }
    if (threadIdx.x == 0) {
        c.plan[CT_KV8_COUNT] = moves;
        c.plan[CT_KV8_LIVE] = live;
    }
}

__global__ __launch_bounds__(NT) void compact_move_kernel(BackendKv8 c, int books, int lp) {
    if ((int)blockIdx.x >= books) {
        copy_pages(c, lp, blockIdx.x - books, gridDim.x - books);
        return;
    }
    const long j = (long)blockIdx.x * NT + threadIdx.x;
    if (j >= (long)c.seqs * c.table_w) return;
    const int p = c.table[j];
    if (p < c.plan[CT_KV8_LIVE] || p >= c.pages) return;
    const int *from = plan_from(c);
    int lo = 0, up = c.plan[CT_KV8_COUNT];
    while (lo < up) {
        const int mid = (lo + up) >> 1;
        if (from[mid] < p) lo = mid + 1;
        else up = mid;
    }
    if (lo < c.plan[CT_KV8_COUNT] && from[lo] == p) c.table[j] = plan_to(c)[lo];
}

__global__ __launch_bounds__(NT) void reset_kernel(BackendKv8 c) {
    const long i = (long)blockIdx.x * NT + threadIdx.x;
    if (i < (long)c.seqs * c.table_w) c.table[i] = -1;
    if (i < c.pages) c.refs[i] = 0;
    if (i < c.seqs) c.len[i] = 0;
    if (i <= c.seqs) c.rows[i] = 0;
    if (i < CT_KV8_HEAD) c.plan[i] = 0;
}

int log2_of(int p) { return 31 - __builtin_clz((unsigned)p); }

// Workgroups of a copy launch: every 16 KB part of `pages` pages its own, at
// most 8192 (each then takes several).
int copy_grid(const BackendKv8 *c, long pages) {
    const long bytes = (long)c->kv_heads * c->head_dim * c->page_tokens;
    const long items = pages * c->layers * 2 * ((bytes + 16383) >> 14);
    return (int)(items < 8192 ? items : 8192);
}

}  // namespace

extern "C" size_t ctk_kv8_plan_ints(const BackendKv8 *c) {
    const size_t most = c->pages > c->seqs ? c->pages : c->seqs;
    return CT_KV8_HEAD + 4 * (size_t)c->seqs + (size_t)c->seqs * c->table_w + 2 * most;
}

extern "C" void ctk_kv8_reset(const BackendKv8 *c, hipStream_t s) {
    long n = (long)c->seqs * c->table_w;
    if (n < c->pages) n = c->pages;
    if (n < c->seqs + 1) n = c->seqs + 1;
    if (n < CT_KV8_HEAD) n = CT_KV8_HEAD;
    hipLaunchKernelGGL(reset_kernel, dim3((unsigned)((n + NT - 1) / NT)), dim3(NT), 0, s, *c);
}

extern "C" void ctk_kv8_reserve(const BackendKv8 *c, const int *add, hipStream_t s) {
    hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(PNT), 0, s, *c, add, log2_of(c->page_tokens));
}

extern "C" void ctk_kv8_append(const BackendKv8 *c, int layer, const void *k, const void *v, long ld, int bf16,
                               const int *rows, int n_rows, hipStream_t s) {
    const int lp = log2_of(c->page_tokens);
    const int vec = ((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ld % (bf16 ? 8 : 4) == 0);
    const int most = (n_rows >> lp) + 2 * c->seqs, pieces = most < n_rows ? most : n_rows;
    const dim3 grid((unsigned)pieces * 2 * c->kv_heads);
#define APPEND(D, B) \
    hipLaunchKernelGGL((append_kernel<D, B>), grid, dim3(NT), 0, s, *c, layer, k, v, ld, vec, rows, n_rows, lp)
    if (c->head_dim == 64) { if (bf16) APPEND(64, true); else APPEND(64, false); }
    else { if (bf16) APPEND(128, true); else APPEND(128, false); }
#undef APPEND
}

extern "C" void ctk_kv8_fork(const BackendKv8 *c, const int *dst, const int *src, int n, hipStream_t s) {
    const int lp = log2_of(c->page_tokens), cols = (c->table_w + NT - 1) / NT;
    const int wide = (c->table_w + PNT - 1) / PNT;
    hipLaunchKernelGGL(fork_plan_kernel, dim3((unsigned)(1 + n * wide)), dim3(PNT), 0, s, *c, dst, src, n, wide, lp);
    hipLaunchKernelGGL(fork_swap_kernel, dim3((unsigned)(n * cols + copy_grid(c, n))), dim3(NT), 0, s, *c, dst, n, cols,
                       lp);
}

extern "C" void ctk_kv8_free(const BackendKv8 *c, const int *seqs, int n, hipStream_t s) {
    const int cols = (c->table_w + NT - 1) / NT;
    hipLaunchKernelGGL(free_kernel, dim3((unsigned)(n * cols)), dim3(NT), 0, s, *c, seqs, n, cols);
}

extern "C" void ctk_kv8_trim(const BackendKv8 *c, int window, int sinks, hipStream_t s) {
    const int cols = (c->table_w + NT - 1) / NT;
    hipLaunchKernelGGL(trim_kernel, dim3((unsigned)(c->seqs * cols)), dim3(NT), 0, s, *c, window, sinks, cols,
                       log2_of(c->page_tokens));
}

extern "C" void ctk_kv8_compact(const BackendKv8 *c, hipStream_t s) {
    const long entries = (long)c->seqs * c->table_w;
    const int books = (int)((entries + NT - 1) / NT);
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(PNT), 0, s, *c);
    hipLaunchKernelGGL(compact_move_kernel, dim3((unsigned)(books + copy_grid(c, (c->pages + 1) / 2))), dim3(NT), 0, s,
                       *c, books, log2_of(c->page_tokens));
}
