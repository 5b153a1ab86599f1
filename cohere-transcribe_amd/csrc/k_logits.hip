// k_logits.hip — penalties for tokens that were said, biases, n-gram bans and
// grammar masks on a step's logits, and the largest logit that is left.
//
// A workgroup holds CHUNK tokens of one row: it reads the row's history and bias
// list once, leaves in LDS for each of its tokens how often it was said, whether
// it is banned and which bias it has (whole numbers, so the order of the atomics
// changes nothing), and then passes over its logits once: 4 bytes read and, where
// wanted, 4 written.  The row's workgroups meet in one 64-bit maximum of (value,
// lowest id) in memory; the last of them writes the token and leaves the
// memory as it was.
#include "ct_dev.h"
#include "ct_w4.h"

namespace {

constexpr int CHUNK = 4096, NT = 256;
constexpr uint32_t SEEN = 1u << 30, BAN = 1u << 31;     // above the counts: a history holds at most 2^24

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

__global__ __launch_bounds__(NT) void logits_kernel(BackendLogits a) {
    __shared__ uint32_t state[CHUNK];
    __shared__ int entry[CHUNK];             // the token's last bias entry, from 1
    __shared__ unsigned long long part[NT / CT_WAVE];
    const int r = blockIdx.y, v0 = blockIdx.x * CHUNK, n = min(CHUNK, a.vocab - v0);
    const int tid = threadIdx.x;

    const int len = a.hist ? (int)min((long)max(a.hist_len[r], 0), a.ld_hist) : 0;
    int b0 = 0, b1 = 0;
    if (a.bias_start) {
        b0 = a.bias_start[r];
        b1 = a.bias_start[r + 1];
        if (b0 < 0 || b1 > a.biases) b1 = b0;
    }
    const bool listed = len > 0 || b1 > b0;
    if (listed) {
        for (int i = tid; i < CHUNK; i += NT) {
            state[i] = 0;
            entry[i] = 0;
        }
        __syncthreads();
        const int *h = a.hist + (long)r * a.ld_hist;
        const int from = a.prompt_len ? a.prompt_len[r] : 0;
        for (int i = tid; i < len; i += NT) {
            const unsigned t = (unsigned)h[i] - (unsigned)v0;
            if (t < (unsigned)n) {
                if (i >= from) atomicAdd(&state[t], 1u);
                else atomicOr(&state[t], SEEN);
            }
        }
        const int k = a.ngram ? a.ngram[r] : 0;
        if (k >= 1 && k <= len) {
            const int *end = h + len - (k - 1);
            for (int i = tid; i <= len - k; i += NT) {
                const unsigned t = (unsigned)h[i + k - 1] - (unsigned)v0;
                if (t >= (unsigned)n) continue;
                int j = 0;
                while (j < k - 1 && h[i + j] == end[j]) j++;
                if (j == k - 1) atomicOr(&state[t], BAN);
            }
        }
        for (int i = b0 + tid; i < b1; i += NT) {
            const unsigned t = (unsigned)a.bias_id[i] - (unsigned)v0;
            if (t < (unsigned)n) atomicMax(&entry[t], i - b0 + 1);
        }
        __syncthreads();
    }

    const float repeat = a.repeat ? a.repeat[r] : 1.0f, frequency = a.frequency ? a.frequency[r] : 0.0f,
                presence = a.presence ? a.presence[r] : 0.0f;
    const int which = !a.mask ? -1 : a.mask_of ? a.mask_of[r] : r;
    const uint32_t *mask = which >= 0 && which < a.masks ? a.mask + (long)which * a.ld_mask : nullptr;
    const bool none = which >= a.masks && a.mask;           // a mask that is not there allows nothing
    const float *x = a.logits + (long)r * a.ld + v0;
    float *y = a.out ? a.out + (long)r * a.ld_out + v0 : nullptr;

    float top = -INFINITY;
    int at = 0;
    for (int i = tid; i < n; i += NT) {
        float l = x[i];
        if (listed) {
            const uint32_t st = state[i];
            if (st) {
                const uint32_t said = st & (SEEN - 1);
                if (a.repeat && (st & ~BAN)) l = l > 0.0f ? l / repeat : mul_rn(l, repeat);
                if (said) {
                    if (a.frequency) l = sub_rn(l, mul_rn(frequency, (float)said));
                    if (a.presence) l = sub_rn(l, presence);
                }
            }
            if (entry[i]) l += a.bias[b0 + entry[i] - 1];
            if (st & BAN) l = -INFINITY;
        }
        if (none || (mask && !(mask[(v0 + i) >> 5] >> ((v0 + i) & 31) & 1))) l = -INFINITY;
        if (y) y[i] = l;
        if (l > top) { top = l; at = i; }
    }
    if (!a.id && !a.score) return;

    // + 0: a negative zero counts as zero
    unsigned long long best = top == -INFINITY ? 0 : (unsigned long long)order_key(top + 0.0f) << 32 | (uint32_t)~(v0 + at);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor(best, o, CT_WAVE);
        best = other > best ? other : best;
    }
    if ((tid & (CT_WAVE - 1)) == 0) part[tid / CT_WAVE] = best;
    __syncthreads();
    if (tid) return;
#pragma unroll
    for (int i = 1; i < NT / CT_WAVE; i++) best = part[i] > best ? part[i] : best;
    if (gridDim.x > 1) {
        Row *row = reinterpret_cast<Row *>(a.work) + r;
        if (best) atomicMax(&row->best, best);
        __threadfence();
        if (atomicAdd(&row->done, 1u) != gridDim.x - 1) return;
        __threadfence();
        best = atomicExch(&row->best, 0ull);
        atomicExch(&row->done, 0u);
    }
    if (a.id) a.id[r] = best ? (int)~(uint32_t)best : -1;
    if (a.score) a.score[r] = best ? from_key((uint32_t)(best >> 32)) : -INFINITY;
}

}  // namespace

extern "C" size_t ctk_logits_work(const BackendLogits *a) {
    return a->vocab > CHUNK ? (size_t)a->rows * (sizeof(Row) / sizeof(float)) : 0;
}

extern "C" void ctk_logits(const BackendLogits *a, hipStream_t s) {
    const dim3 grid((unsigned)((a->vocab + CHUNK - 1) / CHUNK), (unsigned)a->rows);
    hipLaunchKernelGGL(logits_kernel, grid, dim3(NT), 0, s, *a);
}
