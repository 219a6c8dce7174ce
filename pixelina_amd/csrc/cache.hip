// The 8-bit key/value cache: append, read, copy and eviction (gfx950).  The
// attention that reads it is in cache_attention.hip.
//
// One layer of a cache holds, per kv head, blocks of 32 tokens: 32 * D codes of
// the keys and 32 * D of the values (D: the head size rounded up to 64 or 128,
// zero codes beyond it), one scale each, and the 32 tokens' accumulated
// attention weights.  With x the rows of a block and kv head,
//   s = max |x| / 127 over the finite x (fp32, 0 below 2^-100),
//   code = round to nearest even of x / s (NaN: 0, +-Inf: +-127),
// so a code stands for code * s.  The block that the last append ended in also
// keeps its rows in fp32 (a tail), and an append that goes on in it quantizes all
// its rows again from them: what a block holds depends on its rows alone, not on
// the calls that brought them.  A second tail has the last other block that an
// append ended in, for sequences that are cut back into it.  A table per kv head
// maps the blocks of the sequence to those of the memory; eviction permutes it
// and moves no codes.
//
// Code layouts inside a block (what the matrix instructions of the attention
// take without a rearrangement, cache_attention.hip):
//   keys    16-byte pieces of 16 dims of one token at cache_k_offset
//   values  [dim][32 tokens]
#include "pixhip_device.h"
#include "pixhip_internal.h"

namespace pixhip {

namespace {

constexpr float kSmallestScale = 7.888609052210118e-31f;  // 2^-100

// round(x / s) to the nearest even whole number for |x| <= 127 s (1 + 2^-24),
// `inverse` = 1 / s, 0 for a scale of 0: x * inverse is within 127.5 * 2^-23 <
// 2^-15 of the quotient, which settles the code unless that lies as near to a
// half (`tie`); there cache_code_exact takes the quotient in fp64, where only a
// true tie is one.
__device__ __forceinline__ int cache_code(float x, float inverse, bool& tie)
{
    float y = x * inverse;
    y = y == y? __builtin_amdgcn_fmed3f(y,-127.0f,127.0f) : 0.0f;
    const float r = __builtin_rintf(y);
    tie |= fabsf(y - r) > 0.5f - 0x1p-15f;
    return (int)r;
}

__device__ __forceinline__ int cache_code_exact(float x, float s)
{
    if (!(s > 0.0f) || x != x) return 0;
    if (fabsf(x) == INFINITY) return x > 0.0f? 127 : -127;
    return (int)__builtin_rint((double)x / (double)s);
}

// One workgroup per (block, kv head, keys or values) that the call touches, 2
// * D threads: thread (half, d) holds dim d of the tokens 16 half .. 16 half +
// 15, so that rows are read along d.  Bound by HBM: 4 bytes in and 1 out per
// value.
template <int D>
__global__ __launch_bounds__(2 * D) void cache_append_kernel(CacheLayer c, CacheAppend a)
{
    constexpr int T = 2 * D, P = D / 16;
    __shared__ float wave_max[T / 64];
    __shared__ __attribute__((aligned(16))) int8_t codes[kCacheBlock * (D + 16)];
    const int which = (int)blockIdx.x & 1;  // 0 keys, 1 values
    const int h = (int)(blockIdx.x >> 1) % c.kv_heads;
    const size_t b = (size_t)a.start / kCacheBlock + (blockIdx.x >> 1) / (unsigned)c.kv_heads;
    const int tid = (int)threadIdx.x, half = tid / D, d = tid % D;
    const size_t total = a.start + a.rows, slot = (size_t)h * c.blocks + (size_t)c.table[(size_t)h * c.blocks + b];
    const float* in = which? a.v : a.k;
    const float* tail = c.tail + ((((size_t)a.old_slot * c.kv_heads + h) * 2 + which) * kCacheBlock) * D;
    float x[16];
    float m = 0.0f;
    if (b * kCacheBlock >= a.start && (b + 1) * kCacheBlock <= total) {  // a block of new rows alone
        const float* row = in + (b * kCacheBlock - a.start + 16 * half) * a.ld + (size_t)h * c.dim + d;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            x[j] = d < c.dim? *row : 0.0f;
            row += a.ld;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int t = 16 * half + j;
            const size_t i = b * kCacheBlock + t;
            x[j] = 0.0f;
            if (i < a.start) x[j] = tail[t * D + d];
            else if (i < total && d < c.dim) x[j] = in[(i - a.start) * a.ld + (size_t)h * c.dim + d];
        }
    }
#pragma unroll
    for (int j = 0; j < 16; j++) {
        const float v = fabsf(x[j]);
        m = fmaxf(m,v < INFINITY? v : 0.0f);
    }
    m = fmaxf(m,dpp_f32<kDppXor1>(m));
    m = fmaxf(m,dpp_f32<kDppXor2>(m));
    m = fmaxf(m,dpp_f32<kDppHalfMirror>(m));
    m = fmaxf(m,dpp_f32<kDppMirror>(m));
    m = fmaxf(fmaxf(lane_f32(m,0),lane_f32(m,16)),fmaxf(lane_f32(m,32),lane_f32(m,48)));
    if ((tid & 63) == 0) wave_max[tid >> 6] = m;
    __syncthreads();
    m = wave_max[0];
#pragma unroll
    for (int w = 1; w < T / 64; w++) m = fmaxf(m,wave_max[w]);
    float s = __fdiv_rn(m,127.0f);
    if (s < kSmallestScale) s = 0.0f;

    const float inverse = s > 0.0f? __fdiv_rn(1.0f,s) : 0.0f;
    int q[16];
    bool tie = false;
#pragma unroll
    for (int j = 0; j < 16; j++) q[j] = cache_code(x[j],inverse,tie);
    if (tie) {  // (about one wave of 16)
#pragma unroll
        for (int j = 0; j < 16; j++) q[j] = cache_code_exact(x[j],s);
    }
    // The codes go through LDS, so that each wave stores 1 KB in a row.
    if (which) {
        v4i w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (int)pack_bytes(q[4 * j],q[4 * j + 1],q[4 * j + 2],q[4 * j + 3]);
        *reinterpret_cast<v4i*>(codes + cache_v_offset(16 * half,d)) = w;
        __syncthreads();
        reinterpret_cast<v4i*>(c.v + slot * (kCacheBlock * D))[tid] = reinterpret_cast<const v4i*>(codes)[tid];
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) codes[(16 * half + j) * (D + 16) + d] = (int8_t)q[j];
        __syncthreads();
        // piece `tid` of the block holds 16 dims of one token (cache_k_offset)
        const int g = tid / 8, t = 16 * (tid % 8 / 4) + 4 * (g / P) + tid % 4, p = g % P;
        reinterpret_cast<v4i*>(c.k + slot * (kCacheBlock * D))[tid] = *reinterpret_cast<const v4i*>(codes + t * (D + 16) + 16 * p);
        if (tid < kCacheBlock) {
            const size_t i = b * kCacheBlock + tid;
            if (i >= a.start && i < total)
                c.weights[slot * kCacheBlock + tid] = a.weights? a.weights[(i - a.start) * c.kv_heads + h] : 0.0f;
        }
    }
    if (tid == 0) (which? c.vs : c.ks)[slot] = s;
    // the block that the rows end in, and the open one that they went on from
    if ((b + 1) * kCacheBlock >= total || b * kCacheBlock < a.start) {
        const int slot_to = (b + 1) * kCacheBlock >= total? a.new_slot : a.old_slot;
        float* to = c.tail + ((((size_t)slot_to * c.kv_heads + h) * 2 + which) * kCacheBlock) * D;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const int t = 16 * half + j;
            const size_t i = b * kCacheBlock + t;
            if (i >= a.start && i < total) to[t * D + d] = x[j];
        }
    }
}

// The tail of a block whose rows are no longer held in fp32 (a sequence cut
// back into a full block): the values that its codes stand for.
template <int D>
__global__ __launch_bounds__(2 * D) void cache_refill_kernel(CacheLayer c, size_t b, int slot)
{
    const int which = (int)blockIdx.x & 1, h = (int)(blockIdx.x >> 1);
    const size_t at = (size_t)h * c.blocks + (size_t)c.table[(size_t)h * c.blocks + b];
    const float s = (which? c.vs : c.ks)[at];
    const int8_t* codes = (which? c.v : c.k) + at * (kCacheBlock * D);
    float* to = c.tail + ((((size_t)slot * c.kv_heads + h) * 2 + which) * kCacheBlock) * D;
    for (int e = (int)threadIdx.x; e < kCacheBlock * D; e += 2 * D) {
        const int t = e / D, d = e % D;
        to[e] = (float)codes[which? cache_v_offset(t,d) : cache_k_offset(t,d,D)] * s;
    }
}

// Rows first .. first + rows - 1 as the values that their codes stand for: one
// workgroup per (block, kv head, keys or values), and (after those) 256 rows'
// weights of one kv head each.  Bound by HBM: 1 byte in and 4 out per value.
template <int D>
__global__ __launch_bounds__(2 * D) void cache_read_kernel(CacheLayer c, CacheRead a)
{
    const int tid = (int)threadIdx.x;
    const size_t end = a.first + a.rows, b0 = a.first / kCacheBlock;
    const size_t nb = (end - 1) / kCacheBlock - b0 + 1;
    const size_t values = (a.k || a.v)? nb * c.kv_heads * 2 : 0;
    if (blockIdx.x >= values) {
        const size_t e = (blockIdx.x - values) * (2 * D) + tid;
        if (e >= a.rows * c.kv_heads) return;
        const size_t i = a.first + e / c.kv_heads;
        const int h = (int)(e % c.kv_heads);
        const size_t at = (size_t)h * c.blocks + (size_t)c.table[(size_t)h * c.blocks + i / kCacheBlock];
        a.weights[e] = c.weights[at * kCacheBlock + i % kCacheBlock];
        return;
    }
    const int which = (int)blockIdx.x & 1, h = (int)(blockIdx.x >> 1) % c.kv_heads;
    float* out = which? a.v : a.k;
    if (!out) return;
    const size_t b = b0 + (blockIdx.x >> 1) / (unsigned)c.kv_heads;
    const size_t at = (size_t)h * c.blocks + (size_t)c.table[(size_t)h * c.blocks + b];
    const size_t stride = (size_t)c.kv_heads * c.dim;
    if (which) {
        const int half = tid / D, d = tid % D;
        const float s = c.vs[at];
        const v4i w = *reinterpret_cast<const v4i*>(c.v + at * (kCacheBlock * D) + cache_v_offset(16 * half,d));
        if (d >= c.dim) return;
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const size_t i = b * kCacheBlock + 16 * half + j;
            if (i >= a.first && i < end) out[(i - a.first) * stride + (size_t)h * c.dim + d] = (float)(int8_t)(w[j >> 2] >> (8 * (j & 3))) * s;
        }
        return;
    }
    // 4 dims of a token per thread and turn, so that a wave's stores are contiguous
    constexpr int QUADS = D / 4, TURNS = kCacheBlock * QUADS / (2 * D);
    const float s = c.ks[at];
    int w[TURNS];
#pragma unroll
    for (int j = 0; j < TURNS; j++) {
        const int e = tid + 2 * D * j, d = 4 * (e % QUADS);
        w[j] = *reinterpret_cast<const int*>(c.k + at * (kCacheBlock * D) + cache_k_offset(e / QUADS,d,D));
    }
#pragma unroll
    for (int j = 0; j < TURNS; j++) {
        const int e = tid + 2 * D * j, d = 4 * (e % QUADS);
        const size_t i = b * kCacheBlock + e / QUADS;
        if (i < a.first || i >= end) continue;
        float* to = out + (i - a.first) * stride + (size_t)h * c.dim + d;
        const float4 x = make_float4((float)(int8_t)w[j] * s,(float)(int8_t)(w[j] >> 8) * s,(float)(int8_t)(w[j] >> 16) * s,
                                     (float)(int8_t)(w[j] >> 24) * s);
        if (a.vec) {  // dim a multiple of 4, 16-byte aligned outputs
            if (d < c.dim) *reinterpret_cast<float4*>(to) = x;
        } else {
            const float xs[4] = {x.x,x.y,x.z,x.w};
#pragma unroll
            for (int n = 0; n < 4; n++)
                if (d + n < c.dim) to[n] = xs[n];
        }
    }
}

// One layer's blocks in use, copied to another cache in the order of the
// sequence, and its tails; the destination's table becomes the identity.
template <int D>
__global__ __launch_bounds__(4 * D) void cache_copy_kernel(CacheLayer from, CacheLayer to, size_t nb, bool tails)
{
    const int tid = (int)threadIdx.x;
    const size_t heads = (size_t)from.kv_heads;
    size_t id = blockIdx.x;
    if (id < nb * heads) {  // D / 16 * 32 16-byte pieces of the keys, then of the values
        const size_t h = id % heads, b = id / heads;
        const size_t src = h * from.blocks + (size_t)from.table[h * from.blocks + b], dst = h * to.blocks + b;
        const bool value = tid >= 2 * D;
        const int p = tid % (2 * D);
        const int8_t* s = (value? from.v : from.k) + src * (kCacheBlock * D);
        int8_t* d = (value? to.v : to.k) + dst * (kCacheBlock * D);
        reinterpret_cast<v4i*>(d)[p] = reinterpret_cast<const v4i*>(s)[p];
        if (tid < kCacheBlock) to.weights[dst * kCacheBlock + tid] = from.weights[src * kCacheBlock + tid];
        if (tid == 64) to.ks[dst] = from.ks[src];
        if (tid == 65) to.vs[dst] = from.vs[src];
        return;
    }
    id -= nb * heads;
    const size_t tail_groups = tails? heads * 2 * 2 : 0;  // both slots, keys and values
    if (id < tail_groups) {
        const v4f* s = reinterpret_cast<const v4f*>(from.tail + id * kCacheBlock * D);
        v4f* d = reinterpret_cast<v4f*>(to.tail + id * kCacheBlock * D);
        for (int e = tid; e < kCacheBlock * D / 4; e += 4 * D) d[e] = s[e];
        return;
    }
    id -= tail_groups;
    const size_t e = id * (4 * D) + tid;
    if (e < heads * to.blocks) to.table[e] = (int32_t)(e % to.blocks);
}

__global__ __launch_bounds__(256) void cache_table_kernel(int32_t* table, size_t count, size_t blocks)
{
    const size_t e = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (e < count) table[e] = (int32_t)(e % blocks);
}

// ---------------------------------------------------------------- eviction

constexpr int kEvictThreads = 1024;

// Orders a block's weight as a 64-bit number: larger weights give larger
// numbers, NaN the smallest.
__device__ __forceinline__ uint64_t evict_key(double w)
{
    if (w != w) return 0;
    w += 0.0;  // -0 as 0
    const uint64_t u = (uint64_t)__double_as_longlong(w);
    return u >> 63? ~u : u | (1ull << 63);
}

// How many threads of the workgroup before this one (`before`), and of all, have
// `v` set; `waves` holds a count per wave.
__device__ __forceinline__ int group_count(bool v, int* waves, int& before)
{
    const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
    const uint64_t set = __builtin_amdgcn_ballot_w64(v);
    __syncthreads();
    if (lane == 0) waves[wave] = __builtin_popcountll(set);
    __syncthreads();
    int all = 0;
    before = __builtin_popcountll(set & ((1ull << lane) - 1));
#pragma unroll
    for (int w = 0; w < kEvictThreads / 64; w++) {
        const int n = waves[w];
        before += w < wave? n : 0;
        all += n;
    }
    return all;
}

// One workgroup per kv head: the fp64 sum of each block's weights as a key, the
// `pick` largest of the candidates, then the table: kept blocks in order, behind
// them the dropped ones.  The keys' 12 leading bits are counted in 4096 bins,
// then the next 12 of those in the bin where the count reaches `pick`, and so on
// until that bin is taken whole or no bits are left; of equal keys the first
// blocks in order stay.  Keys and the old table lie in LDS, or for more than
// kEvictLds blocks in workspace [kv_heads][nb].  Bound by latency: with bins of
// 8 bits that one thread searched 75 us at 512 blocks.
constexpr int kEvictBits = 12, kEvictBins = 1 << kEvictBits, kEvictLds = 4096;
// Candidates that are ranked against one another instead: a copy, an eviction and a
// read 16.5 us instead of 18.2 at 81 blocks, 17.6 / 19.1 at 129, 25.3 / 24.0 at 257.
constexpr int kEvictRanked = 128;
template <bool LDS>
__global__ __launch_bounds__(kEvictThreads) void cache_evict_kernel(CacheLayer c, int nb, int keep, int recent, size_t length,
                                                                    uint64_t* far_keys, int32_t* far_old, int32_t* kept)
{
    __shared__ uint64_t lds_keys[LDS? kEvictLds : 1];
    __shared__ int32_t lds_old[LDS? kEvictLds : 1];
    __shared__ int hist[kEvictBins];
    __shared__ int waves[kEvictThreads / 64];
    __shared__ int found[3];  // the bin, how many of it stay, how many it has
    const int h = (int)blockIdx.x, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int32_t* table = c.table + (size_t)h * c.blocks;
    uint64_t* keys = LDS? lds_keys : far_keys + (size_t)h * nb;
    int32_t* old = LDS? lds_old : far_old + (size_t)h * nb;
    const int candidates = nb - recent;
    // 8 lanes per block, 4 weights each; four blocks' loads at a time
    constexpr int G = kEvictThreads / 8;
    for (int b0 = 0; b0 < nb; b0 += 4 * G) {
        int at[4];
        float4 x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) at[i] = table[min(b0 + G * i + tid / 8,nb - 1)];
#pragma unroll
        for (int i = 0; i < 4; i++)
            x[i] = *reinterpret_cast<const float4*>(c.weights + ((size_t)h * c.blocks + (size_t)at[i]) * kCacheBlock + 4 * (lane & 7));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int b = b0 + G * i + tid / 8;
            const size_t t = (size_t)b * kCacheBlock + 4 * (lane & 7);
            double w = (t < length? (double)x[i].x : 0.0) + (t + 1 < length? (double)x[i].y : 0.0);
            w += (t + 2 < length? (double)x[i].z : 0.0) + (t + 3 < length? (double)x[i].w : 0.0);
            w += dpp_f64<kDppXor1>(w);
            w += dpp_f64<kDppXor2>(w);
            w += dpp_f64<kDppHalfMirror>(w);
            if (b < nb && (lane & 7) == 0) {
                keys[b] = evict_key(w);
                old[b] = at[i];
            }
        }
    }
    uint64_t prefix = 0;
    int shift = 64, pick = keep - recent, equals = candidates;
    // few: 8 lanes count the candidates before theirs in the order of the keys
    const bool ranked = candidates <= kEvictRanked;
    if (ranked) {
        __syncthreads();
        for (int b0 = 0; b0 < candidates; b0 += G) {
            const int b = b0 + tid / 8;
            const uint64_t k = keys[min(b,candidates - 1)];
            int before = 0;
            for (int j = lane & 7; j < candidates; j += 8) {
                const uint64_t other = keys[j];
                before += other > k || (other == k && j < b)? 1 : 0;
            }
            before += dpp_i32<kDppXor1>(before);
            before += dpp_i32<kDppXor2>(before);
            before += dpp_i32<kDppHalfMirror>(before);
            if ((lane & 7) == 0 && b < candidates) hist[b] = before < pick;
        }
        equals = pick;  // (found)
    }
    // stay: candidates whose key >> shift is above `prefix`, and `pick` of those equal to it
    while (pick > 0 && pick < equals && shift > 0) {
        const int bits = min(kEvictBits,shift);
        const int above = shift;  // (64 at first: every candidate)
        shift -= bits;
        for (int e = tid; e < kEvictBins; e += kEvictThreads) hist[e] = 0;
        __syncthreads();
        for (int b = tid; b < candidates; b += kEvictThreads) {
            const uint64_t k = keys[b];
            if (above == 64 || k >> above == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)],1);
        }
        __syncthreads();
        // thread t has bins 4 t' .. 4 t' + 3 from the top down
        constexpr int E = kEvictBins / kEvictThreads;
        int n[E], mine = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            n[e] = hist[kEvictBins - 1 - (E * tid + e)];
            mine += n[e];
        }
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(upto,o);
            if (lane >= o) upto += u;
        }
        if (lane == 63) waves[wave] = upto;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kEvictThreads / 64; w++) upto += w < wave? waves[w] : 0;
        int before = upto - mine;
        if (before < pick && upto >= pick) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                if (before < pick && before + n[e] >= pick) {
                    found[0] = kEvictBins - 1 - (E * tid + e);
                    found[1] = pick - before;
                    found[2] = n[e];
                }
                before += n[e];
            }
        }
        __syncthreads();
        prefix = prefix << bits | (uint64_t)found[0];
        pick = found[1];
        equals = found[2];
    }
    __syncthreads();
    const bool cut = pick > 0 && pick < equals;  // equal keys: the first `pick` in order
    int equal = 0, stay = 0;
    for (int b0 = 0; b0 < nb; b0 += kEvictThreads) {
        const int b = b0 + tid;
        bool keeps = b >= candidates && b < nb, tie = false;
        if (ranked && b < candidates) {
            keeps = hist[b];
        } else if (b < candidates) {
            const uint64_t k = shift == 64? 0 : keys[b] >> shift;
            tie = pick > 0 && k == prefix;
            keeps = shift != 64 && k > prefix;
        }
        if (cut) {
            int before;
            const int ties = group_count(tie,waves,before);
            tie = tie && equal + before < pick;
            equal += ties;
        }
        keeps = keeps || tie;
        int before;
        const int n = group_count(keeps,waves,before);
        if (keeps) {
            table[stay + before] = old[b];
            if (kept) kept[(size_t)h * keep + stay + before] = b;
        } else if (b < nb) {
            table[keep + b - stay - before] = old[b];
        }
        stay += n;
    }
}

unsigned blocks_of(size_t threads, size_t per)
{
    return (unsigned)((threads + per - 1) / per);
}

}  // namespace

hipError_t launch_cache_table(int32_t* table, size_t count, size_t blocks, hipStream_t s)
{
    cache_table_kernel<<<dim3(blocks_of(count,256)),dim3(256),0,s>>>(table,count,blocks);
    return hipGetLastError();
}

hipError_t launch_cache_append(const CacheLayer& c, const CacheAppend& a, hipStream_t s)
{
    const size_t nb = (a.start + a.rows - 1) / kCacheBlock - a.start / kCacheBlock + 1, groups = nb * c.kv_heads * 2;
    if (groups > (size_t)INT32_MAX) return hipErrorInvalidValue;
    if (c.D == 128) cache_append_kernel<128><<<dim3((unsigned)groups),dim3(256),0,s>>>(c,a);
    else cache_append_kernel<64><<<dim3((unsigned)groups),dim3(128),0,s>>>(c,a);
    return hipGetLastError();
}

hipError_t launch_cache_refill(const CacheLayer& c, size_t block, int slot, hipStream_t s)
{
    if (c.D == 128) cache_refill_kernel<128><<<dim3(2u * c.kv_heads),dim3(256),0,s>>>(c,block,slot);
    else cache_refill_kernel<64><<<dim3(2u * c.kv_heads),dim3(128),0,s>>>(c,block,slot);
    return hipGetLastError();
}

hipError_t launch_cache_read(const CacheLayer& c, const CacheRead& a, hipStream_t s)
{
    const size_t nb = (a.first + a.rows - 1) / kCacheBlock - a.first / kCacheBlock + 1;
    const size_t groups = ((a.k || a.v)? nb * c.kv_heads * 2 : 0) + (a.weights? (a.rows * c.kv_heads + 2 * c.D - 1) / (2 * c.D) : 0);
    if (!groups) return hipSuccess;
    if (groups > (size_t)INT32_MAX) return hipErrorInvalidValue;
    if (c.D == 128) cache_read_kernel<128><<<dim3((unsigned)groups),dim3(256),0,s>>>(c,a);
    else cache_read_kernel<64><<<dim3((unsigned)groups),dim3(128),0,s>>>(c,a);
    return hipGetLastError();
}

hipError_t launch_cache_copy(const CacheLayer& from, const CacheLayer& to, size_t length, bool tails, hipStream_t s)
{
    const size_t nb = (length + kCacheBlock - 1) / kCacheBlock, threads = 4 * (size_t)from.D;
    const size_t groups = nb * from.kv_heads + (tails? (size_t)from.kv_heads * 4 : 0) + (from.kv_heads * to.blocks + threads - 1) / threads;
    if (groups > (size_t)INT32_MAX) return hipErrorInvalidValue;
    if (from.D == 128) cache_copy_kernel<128><<<dim3((unsigned)groups),dim3(512),0,s>>>(from,to,nb,tails);
    else cache_copy_kernel<64><<<dim3((unsigned)groups),dim3(256),0,s>>>(from,to,nb,tails);
    return hipGetLastError();
}

size_t cache_evict_workspace_bytes(size_t kv_heads, size_t blocks)
{
    return kv_heads * blocks * (sizeof(uint64_t) + sizeof(int32_t));
}

hipError_t launch_cache_evict(const CacheLayer& c, size_t length, size_t keep, size_t recent, int32_t* kept, void* workspace, hipStream_t s)
{
    const size_t nb = (length + kCacheBlock - 1) / kCacheBlock;
    uint64_t* keys = static_cast<uint64_t*>(workspace);
    int32_t* old = reinterpret_cast<int32_t*>(keys + (size_t)c.kv_heads * nb);
    const dim3 grid((unsigned)c.kv_heads), block(kEvictThreads);
    if (nb <= kEvictLds) cache_evict_kernel<true><<<grid,block,0,s>>>(c,(int)nb,(int)keep,(int)recent,length,keys,old,kept);
    else cache_evict_kernel<false><<<grid,block,0,s>>>(c,(int)nb,(int)keep,(int)recent,length,keys,old,kept);
    return hipGetLastError();
}

}  // namespace pixhip
