// k_logits.hip — penalties for tokens that were said, biases, n-gram bans and
// grammar masks on a step's logits, and the largest logit that is left.
//
// A thread holds 16 of a row's logits, a workgroup 16 x NT of them, asked for
// first and the first of the history and bias list behind them; the four words of
// the mask are each waited for, and all that was asked for before with them.  The
// workgroup then goes through the row's history and counts in LDS how often each
// of its tokens was said and whether it is banned (whole numbers, so the order of
// the atomics changes nothing); then through the bias list, which leaves each
// token's last entry in the same word.  4 bytes a logit are read and, where wanted,
// 4 written: bound by memory where there are many (200 x 100003, 165 MB: 48.4 us, of
// which a copy of as much takes 34.5), else by the chain arguments, logits and masks,
// history, LDS, largest (5 x 16384: 7.6 us, 64 x 16384 with histories of 1000: 8.7; a
// call of one workgroup is 3.6).  A row's
// workgroups meet in one 64-bit maximum of (value, lowest id) in memory; the
// last of them writes the token and leaves the memory as it was.
#include "ct_dev.h"
#include "ct_w4.h"
#include <limits.h>

namespace {

constexpr int EACH = 16;                                 // logits of a thread
constexpr int SMALL = 256, LARGE = 512;                 // threads of a workgroup
// a token's word: a count in the low bits (a history holds at most 2^24), or
// ENTRY and the number of its last bias entry
constexpr uint32_t BAN = 1u << 29, SEEN = 1u << 30, ENTRY = 1u << 31;

struct Row {                     // of work: zero between calls
    unsigned long long best;     // order_key(value) << 32 | ~id; 0: none
    uint32_t done, unused;       // workgroups that have added theirs
};

// Larger for larger floats; 0 is below all of them.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_key(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ float sub_rn(float a, float b) {
#pragma clang fp contract(off)
    return a - b;
}

// four floats that need not lie on 16 bytes
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float max_dpp(float v) {      // over a wavefront, in lane 63
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x111, 0xF, 0xF, false)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x112, 0xF, 0xF, false)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x114, 0xF, 0xF, false)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x118, 0xF, 0xF, false)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x142, 0xA, 0xF, false)));
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x143, 0xC, 0xF, false)));
}
__device__ __forceinline__ int min_dpp(int v) {
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xF, 0xF, false));
    v = min(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));
    return min(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xC, 0xF, false));
}
// The largest of a wavefront's values and the lowest place of it, for all lanes.
__device__ __forceinline__ void wave_best(float &v, int &at) {
    const float top = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(max_dpp(v)), CT_WAVE - 1));
    at = __builtin_amdgcn_readlane(min_dpp(v == top ? at : INT_MAX), CT_WAVE - 1);
    v = top;
}

template <int NT>
__global__ __launch_bounds__(NT, 6) void logits_kernel(BackendLogits a) {
    constexpr int CHUNK = EACH * NT, STEP = 4 * NT;
    __shared__ __align__(16) uint32_t state[CHUNK];
    __shared__ float stop[NT / CT_WAVE];
    __shared__ int splace[NT / CT_WAVE], slast;
    const int r = blockIdx.y, v0 = blockIdx.x * CHUNK, n = min(CHUNK, a.vocab - v0), tid = threadIdx.x;

    // asked for first: the logits
    const float *x = a.logits + (long)r * a.ld + v0;
    float l[EACH];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = j * STEP + 4 * tid;
        f32x4u y = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i + 4 <= n) {
            y = *reinterpret_cast<const f32x4u *>(x + i);
        } else {
            if (i < n) y[0] = x[i];
            if (i + 1 < n) y[1] = x[i + 1];
            if (i + 2 < n) y[2] = x[i + 2];
        }
#pragma unroll
        for (int e = 0; e < 4; e++) l[4 * j + e] = y[e];
    }
    const int *h = a.hist ? a.hist + (long)r * a.ld_hist : nullptr;
    // no more than the row's tokens: behind the last row's there need be no memory
    const int len = h ? (int)min((long)max(a.hist_len[r], 0), a.ld_hist) : 0;
    int said[4], prev[4];                    // the token at i and the one before it
#pragma unroll
    for (int u = 0; u < 4; u++) {
        const int i = u * NT + tid;
        said[u] = i < len ? h[i] : -1;
        prev[u] = a.ngram && i > 0 && i - 1 < len ? h[i - 1] : -1;
    }

    // the row's entries: nb from b0 on.  Counted from there: a start near 2^31 plus a
    // thread's number would be below any end
    int b0 = 0;
    uint32_t nb = 0;
    if (a.bias_start) {
        const int start = a.bias_start[r], end = a.bias_start[r + 1];
        if (start >= 0 && end <= a.biases && start < end) {
            b0 = start;
            nb = (uint32_t)(end - start);
        }
    }
    const int *bias_id = a.bias_id + b0;
    const float *bias = a.bias + b0;
    const int from = a.prompt_len ? a.prompt_len[r] : 0, k = a.ngram ? a.ngram[r] : 0;
    // the first of the bias list; its values are near when they are looked up
    int biased = -1;
    if ((uint32_t)tid < nb) {
        biased = bias_id[tid];
        __builtin_prefetch(bias + tid);
    }
    const float repeat = a.repeat ? a.repeat[r] : 1.0f, frequency = a.frequency ? a.frequency[r] : 0.0f,
                presence = a.presence ? a.presence[r] : 0.0f;
    const int which = !a.mask ? -1 : a.mask_of ? a.mask_of[r] : r;
    uint32_t allowed[4];                     // bits 0..3: this thread's tokens of group j
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int v = v0 + j * STEP + 4 * tid;
        allowed[j] = 15;
        if (which >= a.masks && a.mask) allowed[j] = 0;      // a mask that is not there allows nothing
        else if (which >= 0 && v < a.vocab) allowed[j] = a.mask[(long)which * a.ld_mask + (v >> 5)] >> (v & 31) & 15;
    }

    if (len > 0 || nb) {
        u32x4 *mine = reinterpret_cast<u32x4 *>(state) + tid;
#pragma unroll
        for (int j = 0; j < 4; j++) mine[j * NT] = (u32x4){0, 0, 0, 0};
        if (len <= 4 * NT) {
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (u * NT + tid == len - 1) slast = said[u];
        } else if (tid == 0) {
            slast = h[len - 1];
        }
        __syncthreads();
    }
    uint32_t banned = 0;                     // a bit for each of the 16
    if (len > 0) {
        for (int i0 = 0;;) {
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * NT + tid;
                const unsigned t = (unsigned)said[u] - (unsigned)v0;
                if (i < len && t < (unsigned)n) {
                    if (i >= from) atomicAdd(&state[t], 1u);
                    else atomicOr(&state[t], SEEN);
                }
            }
            // the token at i is banned if the k - 1 before it are the last ones
            if (k >= 1 && k <= len) {
                const int last = slast;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int i = i0 + u * NT + tid;
                    const unsigned t = (unsigned)said[u] - (unsigned)v0;
                    if (i >= k - 1 && i < len && t < (unsigned)n) {
                        bool same = k == 1 || prev[u] == last;
                        for (int j = 2; same && j < k; j++) same = h[i - j] == h[len - j];
                        if (same) atomicOr(&state[t], BAN);
                    }
                }
            }
            i0 += 4 * NT;
            if (i0 >= len) break;
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int i = i0 + u * NT + tid;
                said[u] = i < len ? h[i] : -1;
                prev[u] = a.ngram && i - 1 < len ? h[i - 1] : -1;
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const u32x4 st = reinterpret_cast<const u32x4 *>(state)[j * NT + tid];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t w = st[e], times = w & (BAN - 1);
                banned |= (w & BAN ? 1u : 0u) << (4 * j + e);
                if (w) {
                    float y = l[4 * j + e];
                    if (a.repeat && (w & ~BAN)) y = y > 0.0f ? y / repeat : mul_rn(y, repeat);
                    const float less = a.frequency ? sub_rn(y, mul_rn(frequency, (float)times)) : y;
                    l[4 * j + e] = times ? (a.presence ? sub_rn(less, presence) : less) : y;
                }
            }
        }
    }
    if (nb) {
        // over the counts, which all have read
        __syncthreads();
        for (uint32_t i = tid; i < nb; i += NT) {
            const unsigned t = (unsigned)biased - (unsigned)v0;
            if (t < (unsigned)n) atomicMax(&state[t], ENTRY | i);
            if (i + NT < nb) biased = bias_id[i + NT];
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const u32x4 st = reinterpret_cast<const u32x4 *>(state)[j * NT + tid];
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (st[e] & ENTRY) l[4 * j + e] += bias[st[e] & ~ENTRY];
        }
    }

    float top = -INFINITY;
    int at = INT_MAX;
    float *y = a.out ? a.out + (long)r * a.ld_out + v0 : nullptr;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = j * STEP + 4 * tid;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float &z = l[4 * j + e];
            z = (banned >> (4 * j + e) & 1) || !(allowed[j] >> e & 1) ? -INFINITY : z;
            at = z > top ? v0 + i + e : at;
            top = z > top ? z : top;
        }
        if (y && i + 4 <= n) {
            *reinterpret_cast<f32x4u *>(y + i) = (f32x4u){l[4 * j], l[4 * j + 1], l[4 * j + 2], l[4 * j + 3]};
        } else if (y) {
            if (i < n) y[i] = l[4 * j];
            if (i + 1 < n) y[i + 1] = l[4 * j + 1];
            if (i + 2 < n) y[i + 2] = l[4 * j + 2];
        }
    }
    if (!a.id && !a.score) return;

    wave_best(top, at);
    if ((tid & (CT_WAVE - 1)) == 0) { stop[tid / CT_WAVE] = top; splace[tid / CT_WAVE] = at; }
    __syncthreads();
    if (tid >= CT_WAVE) return;
    top = tid < NT / CT_WAVE ? stop[tid] : -INFINITY;
    at = tid < NT / CT_WAVE ? splace[tid] : INT_MAX;
    wave_best(top, at);
    if (tid) return;
    if (gridDim.x > 1) {
        // + 0: a negative zero counts as zero
        unsigned long long best = top == -INFINITY ? 0 : (unsigned long long)order_key(top + 0.0f) << 32 | (uint32_t)~at;
        Row *row = reinterpret_cast<Row *>(a.work) + r;
        // Only these words pass between workgroups, and device-wide atomics meet in
        // one place, so the maximum has to be done before the count and nothing
        // else has to be visible: a wait.  A fence writes the XCD's whole L2 back,
        // once a workgroup (200 x 100003 logits: 142 us with it).
        if (best) atomicMax(&row->best, best);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (atomicAdd(&row->done, 1u) != gridDim.x - 1) return;
        best = atomicExch(&row->best, 0ull);
        atomicExch(&row->done, 0u);
        top = best ? from_key((uint32_t)(best >> 32)) : -INFINITY;
        at = (int)~(uint32_t)best;
    }
    if (a.id) a.id[r] = top == -INFINITY ? -1 : at;
    if (a.score) a.score[r] = top;
}

// 512 threads go through a row's history half as often as 256 (200 x 100003 on one card:
// 46 us, with 1024 48); a row that 256 hold has no use for more (300 x 4000: 8.2 us, 512
// 8.8; 1 x 4000: 6.2, 6.7).
int threads_of(const BackendLogits *a) { return a->vocab > EACH * SMALL ? LARGE : SMALL; }

}  // namespace

extern "C" size_t ctk_logits_work(const BackendLogits *a) {
    return a->vocab > EACH * LARGE ? (size_t)a->rows * (sizeof(Row) / sizeof(float)) : 0;
}

extern "C" void ctk_logits(const BackendLogits *a, hipStream_t s) {
    const int nt = threads_of(a);
    const dim3 grid((unsigned)((a->vocab + EACH * nt - 1) / (EACH * nt)), (unsigned)a->rows);
    if (nt == SMALL) hipLaunchKernelGGL((logits_kernel<SMALL>), grid, dim3(SMALL), 0, s, *a);
    else hipLaunchKernelGGL((logits_kernel<LARGE>), grid, dim3(LARGE), 0, s, *a);
}
