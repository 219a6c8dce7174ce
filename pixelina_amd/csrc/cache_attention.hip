// Attention over the 8-bit key/value cache (cache.hip), gfx950.
//
// Query row r of a call of `rows` rows sees the tokens j < n (all of them, or
// with `causal` those up to its own, j <= n - rows + r: the rows are the last
// ones of the sequence).  With the codes K, V and their block scales k, v
//   s_j = q . K_j * k / sqrt(dim),  p_j = exp(s_j - max s) / sum,  out = sum_j p_j V_j v
// and, where the weights are counted, w_j = decay * w_j + the sum of p_j over
// the rows and the heads of the kv head.
#include <math.h>

#include "pixhip_device.h"
#include "pixhip_internal.h"

namespace pixhip {

namespace {

constexpr int kCAThreads = 256;
constexpr float kCLog2e = 1.44269504088896340736f;

struct CAArgs {
    CacheLayer c;
    const float* q;
    float* out;
    float2* stats;  // [kv_heads][rows * group]: maximum (log2 units) and sum of each query
    size_t ld;
    int rows, group, n, causal;
    float scale;  // log2(e) / sqrt(dim)
    float decay;
};

__device__ __forceinline__ int ca_limit(const CAArgs& a, int row)
{
    return a.causal? a.n - a.rows + row + 1 : a.n;
}

// The score of token t of a block against the query in `q` (D values), in log2
// units.
template <int D> __device__ __forceinline__ float ca_score(const int8_t* block, float ks, int t, const float* q, float scale)
{
    float s = 0.0f;
    for (int d = 0; d < D; d += 16) {
        const v4i w = *reinterpret_cast<const v4i*>(block + cache_k_offset(t,d,D));
#pragma unroll
        for (int j = 0; j < 16; j++) s = __builtin_fmaf((float)(int8_t)(w[j >> 2] >> (8 * (j & 3))),q[d + j],s);
    }
    return s * (ks * scale);
}

// One workgroup per query row and head: 256 tokens' scores, then their part of
// the output, D threads a dim each.
template <int D>
__global__ __launch_bounds__(kCAThreads) void cache_attn_kernel(CAArgs a)
{
    __shared__ float q[D], p[kCAThreads], red[kCAThreads / 64];
    const int tid = (int)threadIdx.x;
    const int heads = a.c.kv_heads * a.group, head = (int)blockIdx.x % heads, row = (int)blockIdx.x / heads;
    const int h = head / a.group, limit = ca_limit(a,row);
    const int32_t* table = a.c.table + (size_t)h * a.c.blocks;
    if (tid < D) q[tid] = tid < a.c.dim? a.q[(size_t)row * a.ld + (size_t)head * a.c.dim + tid] : 0.0f;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (int j0 = 0; j0 < limit; j0 += kCAThreads) {
        const int j = j0 + tid;
        float s = -INFINITY;
        if (j < limit) {
            const size_t at = (size_t)h * a.c.blocks + (size_t)table[j / kCacheBlock];
            s = ca_score<D>(a.c.k + at * (kCacheBlock * D),a.c.ks[at],j % kCacheBlock,q,a.scale);
        }
        float x = s;
        for (int e = 1; e < 64; e <<= 1) x = fmaxf(x,__shfl_xor(x,e));
        if ((tid & 63) == 0) red[tid >> 6] = x;
        __syncthreads();
        const float m_new = fmaxf(m,fmaxf(fmaxf(red[0],red[1]),fmaxf(red[2],red[3])));
        const float alpha = exp2f(m - m_new);
        p[tid] = j < limit? exp2f(s - m_new) : 0.0f;
        __syncthreads();
        m = m_new;
        l *= alpha;
        o *= alpha;
        const int count = min(kCAThreads,limit - j0);
        for (int t = 0; t < count; t++) l += p[t];
        if (tid < D) {
            for (int t = 0; t < count; t += kCacheBlock) {
                const size_t at = (size_t)h * a.c.blocks + (size_t)table[(j0 + t) / kCacheBlock];
                const float vs = a.c.vs[at];
                const int8_t* v = a.c.v + at * (kCacheBlock * D) + cache_v_offset(0,tid);
                float part = 0.0f;
                for (int e = 0; e < min(kCacheBlock,count - t); e++) part = __builtin_fmaf(p[t + e],(float)v[e],part);
                o = __builtin_fmaf(part,vs,o);
            }
        }
        __syncthreads();
    }
    if (tid < a.c.dim) a.out[((size_t)row * heads + head) * a.c.dim + tid] = o / l;
    if (a.stats && tid == 0) a.stats[((size_t)h * a.rows + row) * a.group + head % a.group] = make_float2(m,l);
}

// One thread per token and kv head: its probabilities again, from each query's
// maximum and sum.
template <int D>
__global__ __launch_bounds__(kCAThreads) void cache_weights_kernel(CAArgs a, int groups)
{
    const int h = (int)blockIdx.x / groups, j = (int)blockIdx.x % groups * kCAThreads + (int)threadIdx.x;
    if (j >= a.n) return;
    const size_t at = (size_t)h * a.c.blocks + (size_t)a.c.table[(size_t)h * a.c.blocks + j / kCacheBlock];
    const int8_t* block = a.c.k + at * (kCacheBlock * D);
    const float ks = a.c.ks[at];
    float w = 0.0f;
    for (int row = 0; row < a.rows; row++) {
        if (j >= ca_limit(a,row)) continue;
        for (int g = 0; g < a.group; g++) {
            const float* q = a.q + (size_t)row * a.ld + (size_t)(h * a.group + g) * a.c.dim;
            float s = 0.0f;
            for (int d = 0; d < a.c.dim; d++)
                s = __builtin_fmaf((float)block[cache_k_offset(j % kCacheBlock,d,D)],q[d],s);
            const float2 st = a.stats[((size_t)h * a.rows + row) * a.group + g];
            w += exp2f(s * (ks * a.scale) - st.x) / st.y;
        }
    }
    float* to = a.c.weights + at * kCacheBlock + j % kCacheBlock;
    *to = a.decay == 0.0f? w : __builtin_fmaf(a.decay,*to,w);
}

}  // namespace

size_t cache_attention_workspace_bytes(size_t kv_heads, size_t blocks, int D)
{
    (void)blocks;
    (void)D;
    return kv_heads * 65536 * sizeof(float2);
}

hipError_t launch_cache_attention(const CacheLayer& c, const CacheAttention& a, void* workspace, size_t workspace_bytes, hipStream_t s)
{
    CAArgs k = {};
    k.c = c;
    k.q = a.q;
    k.out = a.out;
    k.ld = a.ld;
    k.rows = (int)a.rows;
    k.group = (int)(a.heads / c.kv_heads);
    k.n = (int)a.length;
    k.causal = a.causal? 1 : 0;
    k.scale = kCLog2e / sqrtf((float)c.dim);
    k.decay = a.decay;
    if (a.weigh) {
        k.stats = static_cast<float2*>(workspace);
        if (a.rows * a.heads * sizeof(float2) > workspace_bytes) return hipErrorInvalidValue;
    }
    if (a.rows * a.heads > (size_t)INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(a.rows * a.heads));
    if (c.D == 128) cache_attn_kernel<128><<<grid,dim3(kCAThreads),0,s>>>(k);
    else cache_attn_kernel<64><<<grid,dim3(kCAThreads),0,s>>>(k);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.weigh) return e;
    const int groups = (k.n + kCAThreads - 1) / kCAThreads;
    const dim3 tokens((unsigned)(groups * c.kv_heads));
    if (c.D == 128) cache_weights_kernel<128><<<tokens,dim3(kCAThreads),0,s>>>(k,groups);
    else cache_weights_kernel<64><<<tokens,dim3(kCAThreads),0,s>>>(k,groups);
    return hipGetLastError();
}

}  // namespace pixhip
