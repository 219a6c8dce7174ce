// Log probabilities of given tokens, the entropy of their distributions and the
// most likely alternatives, over rows of logits x (gfx950):
//   m = max x, S = sum e^(x - m), log p(i) = x_i - m - log S,
//   entropy = log S - sum e^(x - m) (x - m) / S,
// the alternatives in the order of x, equal ones by the lower index.  A logit
// of -Inf is a token that cannot come (p = 0, no part in the entropy); a row of
// nothing else has log probabilities of -Inf and entropy 0.  NaN or +Inf in a
// row makes its log probabilities and entropy NaN; its alternatives are ordered
// with NaN as the lowest value.  An id outside the vocabulary gives NaN.
#include <math.h>

#include "pixhip_device.h"
#include "pixhip_internal.h"

namespace pixhip {

namespace {

constexpr int kLPThreads = 1024;

// Orders logits as unsigned numbers: -0 as 0, NaN the lowest.
__device__ __forceinline__ uint32_t lp_key(float x)
{
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u >> 31? ~u : u | 0x80000000u;
}

// Largest of v over the workgroup.
__device__ __forceinline__ uint64_t group_max(uint64_t v, uint64_t* waves)
{
    for (int e = 1; e < 64; e <<= 1) {
        const uint64_t u = (uint64_t)__shfl_xor((unsigned long long)v,e);
        v = u > v? u : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = waves[0];
    for (int w = 1; w < kLPThreads / 64; w++) v = waves[w] > v? waves[w] : v;
    return v;
}

__device__ __forceinline__ float group_sum(float v, float* waves)
{
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
    __syncthreads();
    v = waves[0];
    for (int w = 1; w < kLPThreads / 64; w++) v += waves[w];
    return v;
}

// One workgroup per row.  An alternative is the largest of (key, ~index) below
// the one before it.
__global__ __launch_bounds__(kLPThreads) void log_probs_kernel(LogProbs a)
{
    __shared__ uint64_t best[kLPThreads / 64];
    __shared__ float sums[kLPThreads / 64];
    const size_t row = blockIdx.x;
    const float* x = a.x + row * a.ld;
    uint64_t v = 0;
    for (size_t i = threadIdx.x; i < a.vocab; i += kLPThreads) {
        const uint64_t k = (uint64_t)lp_key(x[i]) << 32 | (uint32_t)~(uint32_t)i;
        v = k > v? k : v;
    }
    v = group_max(v,best);
    float m = x[(uint32_t)~(uint32_t)v];
    float sum = 0.0f, mean = 0.0f;
    const float shift = m == -INFINITY? 0.0f : m;
    for (size_t i = threadIdx.x; i < a.vocab; i += kLPThreads) {
        const float d = x[i] - shift, e = expf(d);
        sum += e;
        mean += e == 0.0f? 0.0f : e * d;
    }
    sum = group_sum(sum,sums);
    mean = group_sum(mean,sums);
    const float norm = sum == 0.0f? 0.0f : logf(sum);
    if (threadIdx.x == 0) {
        if (a.log_probs) {
            const int32_t id = a.ids[row];
            a.log_probs[row] = id < 0 || (size_t)id >= a.vocab? NAN : x[id] - shift - norm;
        }
        if (a.entropy) a.entropy[row] = sum == 0.0f? 0.0f : norm - mean / sum;
    }
    for (int k = 0; k < a.top; k++) {
        if (threadIdx.x == 0) {
            const uint32_t i = ~(uint32_t)v;
            a.top_ids[row * a.top + k] = (int32_t)i;
            a.top_log_probs[row * a.top + k] = x[i] - shift - norm;
        }
        uint64_t next = 0;
        for (size_t i = threadIdx.x; i < a.vocab; i += kLPThreads) {
            const uint64_t c = (uint64_t)lp_key(x[i]) << 32 | (uint32_t)~(uint32_t)i;
            next = c < v && c > next? c : next;
        }
        v = group_max(next,best);
    }
}

}  // namespace

size_t log_probs_workspace_bytes(size_t rows, size_t vocab, int top)
{
    (void)rows;
    (void)vocab;
    (void)top;
    return 0;
}

hipError_t launch_log_probs(const LogProbs& a, void* workspace, hipStream_t s)
{
    (void)workspace;
    if (a.rows > (size_t)INT32_MAX) return hipErrorInvalidValue;
    log_probs_kernel<<<dim3((unsigned)a.rows),dim3(kLPThreads),0,s>>>(a);
    return hipGetLastError();
}

}  // namespace pixhip
