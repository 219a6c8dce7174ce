// Attention over the 8-bit key/value cache (cache.hip), gfx950.
//
// Query row r of a call of `rows` rows sees the tokens j < n (all of them, or
// with `causal` those up to its own, j <= n - rows + r: the rows are the last
// ones of the sequence).  With the codes K, V and their block scales k, v
//   s_j = q . K_j * k / sqrt(dim),  p_j = exp(s_j - max s) / sum,  out = sum_j p_j V_j v
// and, where the weights are counted, w_j = decay * w_j + the sum of p_j over
// the rows and the heads of the kv head.
#include <math.h>

#include <algorithm>

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

// ---------------------------------------------------------------- few queries
//
// A decode step: the codes are the traffic, and each is used by the few queries
// of its kv head.  Both products run on the int8 matrix instruction with the
// codes as they lie in memory, exactly: the fp32 operand is written in digits
// that take the columns which so few queries leave idle.  The 16 columns of
// v_mfma_i32_16x16x64_i8 are 4 queries x 4 digits.
//   scores  q / step, a whole number of 24 bits (step = the row's largest |q| /
//           8355708, so half a step is 2^-24 of it), in three balanced digits
//           of 8 bits; the column sums are exact in 32 bits and meet in fp32.
//   output  p v with p = 2^(score - largest score) and v the value scale of the
//           token's block, relative to the largest such term of the 64 tokens,
//           in four digits of 7 bits (half a step is 2^-27 of that term); the
//           sums over 64 tokens are exact and meet the running ones in fp32.
// A query has two running maxima, of its scores for the sum of its
// probabilities and of score + log2 v for the output: blocks whose values are
// of very different sizes leave each other's sums whole.
// Row i of a score tile t is the token 16 (i / 4) + 4 t + i % 4 of 64, so that
// the scores a lane gets are 16 tokens in a row: its operand of the second
// product, whose other operand is 16 bytes of a dim's row of the value codes.
//
// A wave takes 64 tokens at a time, alone; the next keys are requested as soon
// as the present ones are in the products, the next values likewise.  Waves of
// a workgroup interleave over its piece of the tokens and merge through LDS;
// pieces are merged by cache_combine_kernel.
constexpr int kFewWaves = 4, kFewTile = 64;  // waves per workgroup, tokens per wave and step
constexpr int kFewPieces = 128;              // pieces of a query's tokens, at most
constexpr int kFewUnits = 512;               // workgroups a launch is cut into, about
constexpr int kFewScores = 8;                // queries per kv head whose scores are kept for the weights
// The largest whole number that q becomes: three below the largest that balanced
// digits reach (0x7F7F7F), as the two roundings of the quotient may add one.
constexpr float kFewSteps = 8355708.0f;

struct FewArgs {
    CacheLayer c;
    const float* q;
    float* out;
    float* part;    // [kv_heads][nq][pieces][D]
    float4* stats;  // [kv_heads][nq][pieces]: FewStats
    float* scores;  // [kv_heads][nq][n_pad] in log2 units, or null
    size_t ld;
    int rows, row0, all_rows, group, nq, n, n_pad, causal;  // rows row0 .. row0 + rows - 1 of the call's all_rows
    int qgroups, pieces, chunk;                             // steps (64 tokens) per piece
    float scale;                                            // log2(e) / sqrt(dim)
    float decay;
};

// What a query knows of some of its tokens: the largest score s (log2 units) and
// the sum of 2^(score - s), and the largest score + exponent of the value scale,
// which its output is relative to.
struct FewStats {
    float s, l, o;
};
__device__ __forceinline__ float from_max(float m, float ref)
{
    return m == -INFINITY? 0.0f : __builtin_amdgcn_exp2f(m - ref);
}

__device__ __forceinline__ float quad_sum(float v)
{
    v += dpp_f32<kDppXor1>(v);
    v += dpp_f32<kDppXor2>(v);
    return v;
}
// Over the lanes of equal lane % 16.
__device__ __forceinline__ float rows_max(float v)
{
    v = fmaxf(v,__shfl_xor(v,16));
    return fmaxf(v,__shfl_xor(v,32));
}
__device__ __forceinline__ float rows_sum(float v)
{
    v += __shfl_xor(v,16);
    return v + __shfl_xor(v,32);
}

template <int D, int NT>
__global__ __launch_bounds__(64 * kFewWaves,NT <= 2? 2 : 1) void cache_few_kernel(FewArgs a)
{
    constexpr int U = D / 64, T = D / 16, NQ = 4 * NT;
    __shared__ float so[kFewWaves][NQ][D];
    __shared__ FewStats st[kFewWaves][NQ];
    const int piece = (int)blockIdx.x % a.pieces, unit = (int)blockIdx.x / a.pieces;
    const int h = unit / a.qgroups, q0 = unit % a.qgroups * NQ;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int lane = (int)(threadIdx.x & 63), g = lane >> 4, col = lane & 15, digit = col & 3;
    const int32_t* table = a.c.table + (size_t)h * a.c.blocks;
    const int nb = (a.n + kCacheBlock - 1) / kCacheBlock;
    const size_t head_block = (size_t)h * a.c.blocks;

    // the queries' digits (operand of the scores: column = (query, digit), dims 64 u + 16 g .. + 15)
    v4i qd[NT][U];
    float cq[NT];
    int limit[NT], last = 0;
    const float wd = digit == 0? 65536.0f : digit == 1? 256.0f : digit == 2? 1.0f : 0.0f;
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const int qi = min(q0 + 4 * j + (col >> 2),a.nq - 1), row = a.row0 + qi / a.group;
        const float* p = a.q + (size_t)row * a.ld + (size_t)(h * a.group + qi % a.group) * a.c.dim;
        float x[U][16];
        float top = 0.0f;
        bool finite = true;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int d = 64 * u + 16 * g + i;
                x[u][i] = d < a.c.dim? p[d] : 0.0f;
                top = fmaxf(top,fabsf(x[u][i]));
                finite = finite && fabsf(x[u][i]) < INFINITY;
            }
        top = rows_max(top);
        const float bad = rows_max(finite? 0.0f : 1.0f);
        // (queries below 2^-64 are brought up first, so that the step's inverse is finite)
        const float up = top < 5.421010862427522e-20f? 18446744073709551616.0f : 1.0f;
        const float inverse = top > 0.0f && bad == 0.0f? __fdiv_rn(kFewSteps,top * up) : 0.0f;
        cq[j] = bad != 0.0f? NAN : __fdiv_rn(top * up,kFewSteps) * a.scale / up;
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int w = 0; w < 4; w++) {
                int b[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // balanced digits: those of v + 0x808080, less 128 each
                    const int v = (int)__builtin_rintf(x[u][4 * w + i] * up * inverse) + 0x808080;
                    b[i] = digit == 3? 0 : ((v >> (16 - 8 * digit)) & 255) ^ 128;
                }
                qd[j][u][w] = (int)pack_bytes(b[0],b[1],b[2],b[3]);
            }
        }
        limit[j] = a.causal? a.n - a.all_rows + row + 1 : a.n;
        last = max(last,limit[j]);
    }
    last = max(last,__shfl_xor(last,4));
    last = __builtin_amdgcn_readfirstlane(max(last,__shfl_xor(last,8)));

    v4i k[4][U], v[T];
    float ks, vs;  // this lane's scores' block
    auto load_keys = [&](int step) {
        const int b = min(2 * step + (col >> 3),nb - 1);
        const int8_t* at = a.c.k + (head_block + (size_t)table[b]) * (kCacheBlock * D) + g * 128 + (col & 7) * 16;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int u = 0; u < U; u++) k[t][u] = *reinterpret_cast<const v4i*>(at + (t * U + u) * 512);
    };
    auto load_values = [&](int step) {
        const size_t slot = head_block + (size_t)table[min(2 * step + (g >> 1),nb - 1)];
        const int8_t* at = a.c.v + slot * (kCacheBlock * D) + col * kCacheBlock + 16 * (g & 1);
        ks = a.c.ks[slot];
        vs = a.c.vs[slot];
#pragma unroll
        for (int t = 0; t < T; t++) v[t] = *reinterpret_cast<const v4i*>(at + t * 16 * kCacheBlock);
    };

    float m[NT], mo[NT], l[NT];
    v4f o[NT][T];
#pragma unroll
    for (int j = 0; j < NT; j++) {
        m[j] = mo[j] = -INFINITY;
        l[j] = 0.0f;
#pragma unroll
        for (int t = 0; t < T; t++) o[j][t] = v4f{0.0f,0.0f,0.0f,0.0f};
    }
    // (kept scores are written for every token)
    const int end = min(((a.scores? a.n : last) + kFewTile - 1) / kFewTile,(piece + 1) * a.chunk);
    int step = piece * a.chunk + wave;
    if (step < end) {
        load_keys(step);
        load_values(step);
    }
    for (; step < end; step += kFewWaves) {
        const bool more = step + kFewWaves < end;
        const v4i zero = {0,0,0,0};
        v4i sc[NT][4];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                sc[j][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][0],qd[j][0],zero,0,0,0);
                if constexpr (U == 2) sc[j][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][1],qd[j][1],sc[j][t],0,0,0);
            }
        if (more) load_keys(step + kFewWaves);
        // v = f 2^e (0: a block of zeros, or of values below 2^-93)
        const uint32_t bits = __float_as_uint(vs);
        const float e = bits? (float)((int)(bits >> 23) - 127) : -INFINITY;
        const float f = __uint_as_float((bits & 0x007FFFFFu) | 0x3F800000u) * 0x1p26f;
        const int token = kFewTile * step + 16 * g;
        v4i pd[NT];
        float beta[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const float c = cq[j] * ks;
            float s[16], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = quad_sum((float)sc[j][i >> 2][i & 3] * wd);
            if (kFewTile * (step + 1) > last || a.causal) {
#pragma unroll
                for (int i = 0; i < 16; i++) s[i] = token + i < limit[j]? s[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top,s[i]);
            // (a query of zeros has c = 0: hidden tokens are told by their score, not by the product)
            const float lane_top = top == -INFINITY? -INFINITY : top * c;
            const float ms = rows_max(lane_top), mt = rows_max(lane_top + e);
            const float ref = ms == -INFINITY? 0.0f : ms, ref_o = mt == -INFINITY? 0.0f : mt;
            // (below 2^-99 a probability's term is cut, not scaled up past fp32)
            const float factor = e == -INFINITY? 0.0f : f * __builtin_amdgcn_exp2f(fminf(e + ref - ref_o,99.0f));
            float sum = 0.0f;
            uint32_t word[4] = {0,0,0,0};
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float p = s[i] == -INFINITY? 0.0f : __builtin_amdgcn_exp2f(__builtin_fmaf(s[i],c,-ref));
                sum += p;
                const uint32_t n = (uint32_t)__builtin_rintf(p * factor);
                word[i >> 2] |= ((n >> (21 - 7 * digit)) & 127u) << (8 * (i & 3));
            }
            pd[j] = v4i{(int)word[0],(int)word[1],(int)word[2],(int)word[3]};
            if (a.scores) {
                // the four lanes of a query hold the same 16 scores: each writes four of them
                const int qi = q0 + 4 * j + (col >> 2);
                float4 w;
                float* ws = &w.x;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float x = digit == 0? s[r] : digit == 1? s[4 + r] : digit == 2? s[8 + r] : s[12 + r];
                    ws[r] = x == -INFINITY? x : x * c;
                }
                if (qi < a.nq) *reinterpret_cast<float4*>(a.scores + ((size_t)h * a.nq + qi) * a.n_pad + token + 4 * digit) = w;
            }
            const float m_new = fmaxf(m[j],ms), mr = m_new == -INFINITY? 0.0f : m_new;
            l[j] = __builtin_fmaf(l[j],from_max(m[j],mr),sum * __builtin_amdgcn_exp2f(ref - mr));
            m[j] = m_new;
            const float o_new = fmaxf(mo[j],mt);
            beta[j] = from_max(mt,o_new);
            if (__builtin_amdgcn_ballot_w64(o_new != mo[j])) {
                const float alpha = from_max(mo[j],o_new);
#pragma unroll
                for (int t = 0; t < T; t++) o[j][t] *= alpha;
            }
            mo[j] = o_new;
        }
#pragma unroll
        for (int t = 0; t < T; t++)
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const v4i x = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[t],pd[j],zero,0,0,0);
#pragma unroll
                for (int r = 0; r < 4; r++) o[j][t][r] = __builtin_fmaf((float)x[r],beta[j],o[j][t][r]);
            }
        if (more) load_values(step + kFewWaves);
    }

    // digits, then waves in order
    const float place = digit == 0? 0x1p-5f : digit == 1? 0x1p-12f : digit == 2? 0x1p-19f : 0x1p-26f;
#pragma unroll
    for (int j = 0; j < NT; j++) {
        const float lt = rows_sum(l[j]);
        const int i = 4 * j + (col >> 2);
#pragma unroll
        for (int t = 0; t < T; t++) {
            v4f x;
#pragma unroll
            for (int r = 0; r < 4; r++) x[r] = quad_sum(o[j][t][r] * place);
            if (digit == 0) *reinterpret_cast<v4f*>(&so[wave][i][16 * t + 4 * g]) = x;
        }
        if (digit == 0 && g == 0) st[wave][i] = FewStats{m[j],lt,mo[j]};
    }
    __syncthreads();
    for (int e = (int)threadIdx.x; e < NQ * D; e += 64 * kFewWaves) {
        const int i = e / D, d = e % D, qi = q0 + i;
        if (qi >= a.nq) continue;
        FewStats all = st[0][i];
#pragma unroll
        for (int w = 1; w < kFewWaves; w++) {
            all.s = fmaxf(all.s,st[w][i].s);
            all.o = fmaxf(all.o,st[w][i].o);
        }
        float acc = 0.0f;
        all.l = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWaves; w++) {
            acc = __builtin_fmaf(from_max(st[w][i].o,all.o),so[w][i][d],acc);
            all.l = __builtin_fmaf(from_max(st[w][i].s,all.s),st[w][i].l,all.l);
        }
        const size_t query = (size_t)h * a.nq + qi;
        if (a.pieces > 1) a.part[(query * a.pieces + piece) * D + d] = acc;
        else if (d < a.c.dim)
            a.out[(size_t)(a.row0 + qi / a.group) * a.c.kv_heads * a.group * a.c.dim + (size_t)(h * a.group + qi % a.group) * a.c.dim + d] =
                acc * from_max(all.o,all.s) / all.l;
        if (d == 0 && (a.pieces > 1 || a.scores)) a.stats[query * a.pieces + piece] = make_float4(all.s,all.l,all.o,0.0f);
    }
}

// A query's FewStats over its pieces, in every lane of the wave (at most
// kFewPieces = 128 of them).
__device__ __forceinline__ FewStats merged_stats(const float4* stats, int pieces)
{
    const int lane = (int)(threadIdx.x & 63);
    const float4 a = stats[min(lane,pieces - 1)], b = stats[min(lane + 64,pieces - 1)];
    FewStats all = {fmaxf(a.x,b.x),0.0f,fmaxf(a.z,b.z)};
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        all.s = fmaxf(all.s,__shfl_xor(all.s,o));
        all.o = fmaxf(all.o,__shfl_xor(all.o,o));
    }
    float l = lane < pieces? a.y * from_max(a.x,all.s) : 0.0f;
    l += lane + 64 < pieces? b.y * from_max(b.x,all.s) : 0.0f;
    all.l = wave_sum(l);
    return all;
}

// Merges the pieces of one query per workgroup (those after the first
// kv_heads * nq: 1024 tokens of one kv head each, whose weights get the
// probabilities that the kept scores and the queries' merged sums give).
template <int D>
__global__ __launch_bounds__(256) void cache_combine_kernel(FewArgs a, int outputs)
{
    constexpr int G = 256 / D;
    __shared__ float so[G][D];
    __shared__ float2 sq[kFewScores];
    const int tid = (int)threadIdx.x;
    if ((int)blockIdx.x < outputs) {
        const int h = (int)blockIdx.x / a.nq, qi = (int)blockIdx.x % a.nq, d = tid % D, first = tid / D;
        const size_t query = (size_t)h * a.nq + qi;
        const float4* stats = a.stats + query * a.pieces;
        const float* part = a.part + query * a.pieces * D + d;
        const FewStats all = merged_stats(stats,a.pieces);
        float acc = 0.0f;
        for (int p = first; p < a.pieces; p += G) acc = __builtin_fmaf(from_max(stats[p].z,all.o),part[(size_t)p * D],acc);
        so[first][d] = acc;
        __syncthreads();
        if (first || d >= a.c.dim) return;
#pragma unroll
        for (int i = 1; i < G; i++) acc += so[i][d];
        a.out[(size_t)(a.row0 + qi / a.group) * a.c.kv_heads * a.group * a.c.dim + (size_t)(h * a.group + qi % a.group) * a.c.dim + d] =
            acc * from_max(all.o,all.s) / all.l;
        return;
    }
    const int groups = (a.n + 1023) / 1024, id = (int)blockIdx.x - outputs, h = id / groups;
    for (int q = tid >> 6; q < a.nq; q += 4) {
        const FewStats all = merged_stats(a.stats + ((size_t)h * a.nq + q) * a.pieces,a.pieces);
        if ((tid & 63) == 0) sq[q] = make_float2(all.s,1.0f / all.l);
    }
    __syncthreads();
    const int j = id % groups * 1024 + 4 * tid;
    if (j >= a.n) return;
    float4 w = {0.0f,0.0f,0.0f,0.0f};
    for (int q = 0; q < a.nq; q++) {
        const float4 s = *reinterpret_cast<const float4*>(a.scores + ((size_t)h * a.nq + q) * a.n_pad + j);
        w.x = __builtin_fmaf(__builtin_amdgcn_exp2f(s.x - sq[q].x),sq[q].y,w.x);
        w.y = __builtin_fmaf(__builtin_amdgcn_exp2f(s.y - sq[q].x),sq[q].y,w.y);
        w.z = __builtin_fmaf(__builtin_amdgcn_exp2f(s.z - sq[q].x),sq[q].y,w.z);
        w.w = __builtin_fmaf(__builtin_amdgcn_exp2f(s.w - sq[q].x),sq[q].y,w.w);
    }
    float4* to = reinterpret_cast<float4*>(a.c.weights + ((size_t)h * a.c.blocks + (size_t)a.c.table[(size_t)h * a.c.blocks + j / kCacheBlock]) * kCacheBlock +
                                           j % kCacheBlock);
    if (a.decay != 0.0f) {
        const float4 old = *to;
        w.x = __builtin_fmaf(a.decay,old.x,w.x);
        w.y = __builtin_fmaf(a.decay,old.y,w.y);
        w.z = __builtin_fmaf(a.decay,old.z,w.z);
        w.w = __builtin_fmaf(a.decay,old.w,w.w);
    }
    *to = w;
}

}  // namespace

// Parts of the workspace: records of D values and statistics of a query's
// pieces, and the few-query kernel's scores.
static size_t ca_records(size_t kv_heads, size_t blocks)
{
    return std::min<size_t>(65536,kv_heads * blocks * 64);
}

size_t cache_attention_workspace_bytes(size_t kv_heads, size_t blocks, int D)
{
    return ca_records(kv_heads,blocks) * (D * sizeof(float) + sizeof(float4)) + kv_heads * kFewScores * (blocks + 1) * kCacheBlock * sizeof(float);
}

static hipError_t launch_few(FewArgs a, hipStream_t s)
{
    const int width = a.nq <= 4? 1 : a.nq <= 8? 2 : 4;
    a.qgroups = (a.nq + 4 * width - 1) / (4 * width);
    const size_t units = (size_t)a.c.kv_heads * a.qgroups, steps = ((size_t)a.n + kFewTile - 1) / kFewTile;
    const size_t fit = ca_records(a.c.kv_heads,a.c.blocks) / ((size_t)a.c.kv_heads * a.nq);
    size_t want = std::min({(steps + kFewWaves - 1) / kFewWaves,(size_t)kFewPieces,fit,kFewUnits / units});
    if (!want) want = 1;
    a.chunk = (int)((steps + want - 1) / want);
    a.pieces = (int)((steps + a.chunk - 1) / a.chunk);
    if (units * a.pieces > (size_t)INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(units * a.pieces)), block(64 * kFewWaves);
    if (a.c.D == 128) {
        if (width == 4) cache_few_kernel<128,4><<<grid,block,0,s>>>(a);
        else if (width == 2) cache_few_kernel<128,2><<<grid,block,0,s>>>(a);
        else cache_few_kernel<128,1><<<grid,block,0,s>>>(a);
    } else {
        if (width == 4) cache_few_kernel<64,4><<<grid,block,0,s>>>(a);
        else if (width == 2) cache_few_kernel<64,2><<<grid,block,0,s>>>(a);
        else cache_few_kernel<64,1><<<grid,block,0,s>>>(a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || (a.pieces == 1 && !a.scores)) return e;
    const int outputs = a.pieces > 1? a.c.kv_heads * a.nq : 0;
    const size_t groups = outputs + (a.scores? (size_t)a.c.kv_heads * ((a.n + 1023) / 1024) : 0);
    if (groups > (size_t)INT32_MAX) return hipErrorInvalidValue;
    if (a.c.D == 128) cache_combine_kernel<128><<<dim3((unsigned)groups),dim3(256),0,s>>>(a,outputs);
    else cache_combine_kernel<64><<<dim3((unsigned)groups),dim3(256),0,s>>>(a,outputs);
    return hipGetLastError();
}

hipError_t launch_cache_attention(const CacheLayer& c, const CacheAttention& a, void* workspace, size_t workspace_bytes, hipStream_t s)
{
    const size_t nq = a.rows * (a.heads / c.kv_heads);
    if (nq <= (a.weigh? (size_t)kFewScores : 64)) {
        FewArgs f = {};
        f.c = c;
        f.q = a.q;
        f.out = a.out;
        f.part = static_cast<float*>(workspace);
        f.stats = reinterpret_cast<float4*>(f.part + ca_records(c.kv_heads,c.blocks) * c.D);
        f.scores = a.weigh? reinterpret_cast<float*>(f.stats + ca_records(c.kv_heads,c.blocks)) : nullptr;
        f.ld = a.ld;
        f.rows = f.all_rows = (int)a.rows;
        f.group = (int)(a.heads / c.kv_heads);
        f.nq = (int)nq;
        f.n = (int)a.length;
        f.n_pad = (f.n + kFewTile - 1) / kFewTile * kFewTile;
        f.causal = a.causal? 1 : 0;
        f.scale = kCLog2e / sqrtf((float)c.dim);
        f.decay = a.decay;
        return launch_few(f,s);
    }
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
