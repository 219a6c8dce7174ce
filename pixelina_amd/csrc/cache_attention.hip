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
#include <type_traits>

#include "pixhip_device.h"
#include "pixhip_internal.h"

namespace pixhip {

namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr float kCLog2e = 1.44269504088896340736f;

struct CAArgs {
    CacheLayer c;
    const float* q;
    float* out;
    // A kv head's queries are a list, its group of heads of one row after the
    // other; this launch takes entries first .. first + nq - 1.
    float* part;     // few queries: [kv_heads][nq][pieces][D]; many: cache_tile_kernel
    float4* stats;   // and the QueryStats of each
    float* scores;   // few queries: [kv_heads][nq][n_pad] in log2 units, or null
    float2* merged;  // many queries: [kv_heads][nq] maximum and inverse sum, or null
    v8h* planes;     // many queries: fp16 halves of the queries for the weights, or null
    float* steps;    // and the value of a unit of theirs (a power of two), [kv_heads][nq_pad]
    size_t ld;
    int first, nq, nq_pad, group, rows, n, n_pad, causal;
    int qvec, ovec;              // q may be read, out written 16 bytes at a time
    int tiles_q, pieces, chunk;  // groups of queries, pieces of the tokens, 64-token steps per piece
    float scale;                 // log2(e) / sqrt(dim)
    float decay;
};

// What a query knows of some of its tokens: the largest score s (log2 units), the
// sum l of 2^(score - s), and o, the largest score - s + exponent of the value
// scale: its output is relative to 2^(s + o).  (o is kept relative to s, as s + o
// would lose o's bits where s is large.)
struct QueryStats {
    float s, l, o;
};
__device__ __forceinline__ float from_max(float m, float ref)
{
    return m == -INFINITY? 0.0f : __builtin_amdgcn_exp2f(m - ref);
}
// x's o relative to another largest score.
__device__ __forceinline__ float moved_o(QueryStats x, float s)
{
    return x.o == -INFINITY? x.o : x.o + (x.s - s);
}
// From this largest score on, scores are rounded products before it is taken from
// them, as the largest itself was: fused, the product's own rounding would be left in
// every probability.  Below it that is at most a quarter (log2 units), and so is what
// score + exponent loses: the few-query kernel's digits and the other one's halves
// have room for both.
constexpr float kLargeScore = 0x1p22f;

// Entry i of a kv head's list of queries: its row, and its place in q and out.
__device__ __forceinline__ int query_row(const CAArgs& a, int i)
{
    return (a.first + i) / a.group;
}
__device__ __forceinline__ const float* query_at(const CAArgs& a, int h, int i)
{
    return a.q + (size_t)query_row(a,i) * a.ld + (size_t)(h * a.group + (a.first + i) % a.group) * a.c.dim;
}
__device__ __forceinline__ float* output_at(const CAArgs& a, int h, int i)
{
    return a.out + ((size_t)query_row(a,i) * a.c.kv_heads * a.group + (size_t)(h * a.group + (a.first + i) % a.group)) * a.c.dim;
}
// Tokens that a row sees.
__device__ __forceinline__ int row_limit(const CAArgs& a, int row)
{
    return a.causal? a.n - a.rows + row + 1 : a.n;
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
constexpr int kFewWide = 8;                  // waves per workgroup that takes all tokens
constexpr int kFewPieces = 128;              // pieces of a query's tokens, at most
constexpr int kFewUnits = 512;               // workgroups a launch is cut into, about
constexpr int kFewQ = 4;                     // queries per workgroup
// Queries per kv head, at most; few / many, us, 8 kv heads of 128: 32 queries at
// 2501 tokens 13.1 / 18.0, at 16001 27.2 / 33.4, at 131072 145 / 150; 64 queries
// 16.3 / 18.2, 42.3 / 33.7, 263 / 154.
constexpr int kFewMax = 32;
// And up to 256 queries where queries x tokens x kv heads are few: 128 queries at
// 1000 tokens 14.2 / 16.3, at 2501 20.7 / 18.9; 256 queries 15.2 / 19.5, 27.3 /
// 22.3; of 2 kv heads 64 queries at 16001 18.6 / 25.7, 256 at 6000 22.7 / 20.1.
constexpr int kFewMaxShort = 256;
constexpr size_t kFewPairs = (size_t)1 << 21;
// Where the weights are counted the scores are kept for them: there is room for
// those of 8 queries per kv head in any case, and up to kFewMax where they are no
// more than 16 MB.  Few / many, us, 8 kv heads of 128: 16 queries at 1281 tokens
// 11.5 / 23.0, at 16001 21.1 / 39.4; 32 queries 14.8 / 22.8, 30.5 / 39.4.
constexpr int kFewScores = 8;
constexpr size_t kFewScoreBytes = 16 << 20;
// The largest whole number that q becomes: three below the largest that balanced
// digits reach (0x7F7F7F), as the two roundings of the quotient may add one.
constexpr float kFewSteps = 8355708.0f;

// What a unit of a block's score is worth, from the query's and the block's part:
// above 0, so that a hidden token's -Inf stays -Inf and its probability 0 without a
// test; where it is 0 (a query or a block of zeros) the scores themselves are 0.
// The two are multiplied first: with a score's whole number a large block scale
// alone would leave fp32's range.
__device__ __forceinline__ float score_unit(float query, float block)
{
    const float c = query * block;
    return c == 0.0f? 1e-37f : c;
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
    v = fmaxf(v,xor_lane<16>(v));
    return fmaxf(v,xor_lane<32>(v));
}
__device__ __forceinline__ float rows_sum(float v)
{
    v += xor_lane<16>(v);
    return v + xor_lane<32>(v);
}
// Read by scalar loads (nothing in a launch that reads them writes them).
template <typename T> using constant = const __attribute__((address_space(4))) T;
template <typename T> __device__ __forceinline__ constant<T>* as_constant(const T* p)
{
    return (constant<T>*)(uintptr_t)p;
}

// Four queries of one kv head per workgroup: more are more workgroups over the
// same tokens (8 and 16 queries per workgroup ran slower at every length: 8
// queries per kv head at 2501 tokens 10.2 us, as one group of 8 14.7; at 131072
// tokens 57.7 and 82.2).  SCORES: the scores are kept for the weights.
template <int D, bool SCORES, int WAVES>
__global__ __launch_bounds__(64 * WAVES,2) void cache_few_kernel(CAArgs a)
{
    constexpr int U = D / 64, T = D / 16;
    __shared__ float so[WAVES][kFewQ][D];
    __shared__ QueryStats st[WAVES][kFewQ];
    const int piece = (int)blockIdx.x % a.pieces, unit = (int)blockIdx.x / a.pieces;
    const int h = unit / a.tiles_q, q0 = unit % a.tiles_q * kFewQ;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int lane = (int)(threadIdx.x & 63), g = lane >> 4, col = lane & 15, digit = col & 3, qi = q0 + (col >> 2);
    constant<int32_t>* const table = as_constant(a.c.table) + (size_t)h * a.c.blocks;
    const int nb = (a.n + kCacheBlock - 1) / kCacheBlock;
    const size_t head_block = (size_t)h * a.c.blocks;

    // this lane's query, as it is: dims 64 u + 16 g .. + 15
    float x[U][16];
    const int qc = min(qi,a.nq - 1), limit = row_limit(a,query_row(a,qc));
    const float* const q = query_at(a,h,qc);
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = 64 * u + 16 * g + i;
            if (a.qvec) {  // dim a multiple of 4, 16-byte aligned rows
                const v4f w = *reinterpret_cast<const v4f*>(q + min(d,a.c.dim - 4));
#pragma unroll
                for (int e = 0; e < 4; e++) x[u][i + e] = d < a.c.dim? w[e] : 0.0f;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float w = q[min(d + e,a.c.dim - 1)];
                    x[u][i + e] = d + e < a.c.dim? w : 0.0f;
                }
            }
        }
    // the tokens that any of the workgroup's queries sees
    int last = max(limit,(int)xor_lane<4>((uint32_t)limit));
    last = __builtin_amdgcn_readfirstlane(max(last,(int)xor_lane<8>((uint32_t)last)));

    v4i k[4][U], v[T];
    float ks, vs;  // this lane's scores' block
    auto load_keys = [&](int step) {
        const int t0 = table[min(2 * step,nb - 1)], t1 = table[min(2 * step + 1,nb - 1)];
        const int8_t* at = a.c.k + (head_block + (size_t)(col >> 3? t1 : t0)) * (kCacheBlock * D) + g * 128 + (col & 7) * 16;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int u = 0; u < U; u++) k[t][u] = *reinterpret_cast<const v4i*>(at + (t * U + u) * 512);
    };
    auto load_values = [&](int step) {
        const int t0 = table[min(2 * step,nb - 1)], t1 = table[min(2 * step + 1,nb - 1)];
        const size_t s0 = head_block + (size_t)t0, s1 = head_block + (size_t)t1;
        const float k0 = as_constant(a.c.ks)[s0], k1 = as_constant(a.c.ks)[s1], v0 = as_constant(a.c.vs)[s0], v1 = as_constant(a.c.vs)[s1];
        ks = g >> 1? k1 : k0;
        vs = g >> 1? v1 : v0;
        const int8_t* at = a.c.v + (g >> 1? s1 : s0) * (kCacheBlock * D) + col * kCacheBlock + 16 * (g & 1);
#pragma unroll
        for (int t = 0; t < T; t++) v[t] = *reinterpret_cast<const v4i*>(at + t * 16 * kCacheBlock);
    };
    // (kept scores are written for every token)
    const int end = min(((SCORES? a.n : last) + kFewTile - 1) / kFewTile,(piece + 1) * a.chunk);
    int step = piece * a.chunk + wave;
    if (step < end) {
        load_keys(step);
        load_values(step);
    }

    // its digits: operand of the scores, column = (query, digit)
    uint32_t bits = 0;
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) bits = max(bits,__float_as_uint(x[u][i]) & 0x7FFFFFFFu);  // (NaN above infinity above the rest)
    bits = max(bits,xor_lane<16>(bits));
    bits = max(bits,xor_lane<32>(bits));
    const float largest = __uint_as_float(bits);
    const bool finite = bits < 0x7F800000u;
    // (queries below 2^-64 are brought up first, so that the step and its inverse stay
    // normal numbers; the block scale takes it back)
    const float up = largest < 0x1p-64f? 0x1p64f : 1.0f, down = largest < 0x1p-64f? 0x1p-64f : 1.0f;
    if (__builtin_amdgcn_ballot_w64(largest < 0x1p-64f)) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) x[u][i] *= up;
    }
    const float inverse = finite && bits? __fdiv_rn(kFewSteps,largest * up) : 0.0f;
    const float cq = finite? __fdiv_rn(largest * up,kFewSteps) * a.scale : NAN;
    const float wd = digit == 0? 65536.0f : digit == 1? 256.0f : digit == 2? 1.0f : 0.0f;
    v4i qd[U];
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int w = 0; w < 4; w++) {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; i++)  // balanced digits: those of v + 0x808080, less 128 each
                b[i] = (uint32_t)((int)__builtin_rintf(x[u][4 * w + i] * inverse) + 0x808080) >> (16 - 8 * (digit < 3? digit : 2));
            const uint32_t packed = __builtin_amdgcn_perm(b[1],b[0],0x0c0c0400u) | __builtin_amdgcn_perm(b[3],b[2],0x04000c0cu);
            qd[u][w] = digit == 3? 0 : (int)(packed ^ 0x80808080u);
        }

    float m = -INFINITY, mo = -INFINITY, l = 0.0f;
    v4f o[T];
#pragma unroll
    for (int t = 0; t < T; t++) o[t] = v4f{0.0f,0.0f,0.0f,0.0f};
    for (; step < end; step += WAVES) {
        const bool more = step + WAVES < end;
        const v4i zero = {0,0,0,0};
        v4i sc[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            sc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][0],qd[0],zero,0,0,0);
            if constexpr (U == 2) sc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[t][1],qd[1],sc[t],0,0,0);
        }
        if (more) load_keys(step + WAVES);
        // v = f 2^e (0: a block of zeros, or of values below 2^-93)
        const uint32_t vbits = __float_as_uint(vs);
        const float e = vbits? (float)((int)(vbits >> 23) - 127) : -INFINITY;
        const float f = __uint_as_float((vbits & 0x007FFFFFu) | 0x3F800000u) * 0x1p26f;
        const int token = kFewTile * step + 16 * g;
        const float c = score_unit(cq,ks * down);
        float s[16], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = quad_sum((float)sc[i >> 2][i & 3] * wd);
        if (kFewTile * (step + 1) > last || a.causal) {
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] = token + i < limit? s[i] : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) top = fmaxf(top,s[i]);
        const float lane_top = top * c, ms = rows_max(lane_top);
        const float ref = ms == -INFINITY? 0.0f : ms;
        float mt = rows_max(lane_top + e) - ref, each = c;
        const bool large = __builtin_amdgcn_ballot_w64(fabsf(ref) >= kLargeScore);
        if (large) mt = rows_max((lane_top - ref) + e);
        if (SCORES || large) {  // (kept scores are rounded products too)
#pragma unroll
            for (int i = 0; i < 16; i++) s[i] *= c;
            each = 1.0f;
        }
        const float ref_o = mt == -INFINITY? 0.0f : mt;
        // (below 2^-99 a probability's term is cut, not scaled up past fp32)
        const float factor = e == -INFINITY? 0.0f : f * __builtin_amdgcn_exp2f(fminf(e - ref_o,99.0f));
        float sum = 0.0f;
        uint32_t word[4] = {0,0,0,0};
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i],each,-ref));
            sum += p;
            const uint32_t n = (uint32_t)__builtin_rintf(p * factor);
            word[i >> 2] |= ((n >> (21 - 7 * digit)) & 127u) << (8 * (i & 3));
        }
        const v4i pd = {(int)word[0],(int)word[1],(int)word[2],(int)word[3]};
        if constexpr (SCORES) {
            // the four lanes of a query hold the same 16 scores: each writes four of them
            // (a query that is not finite: -Inf; its weights are NaN by its sum)
            v4f w;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float s0 = s[r], s1 = s[4 + r], s2 = s[8 + r], s3 = s[12 + r];
                const float even = digit & 2? s2 : s0, odd = digit & 2? s3 : s1;
                w[r] = fmaxf(digit & 1? odd : even,-INFINITY);
            }
            if (qi < a.nq) *reinterpret_cast<v4f*>(a.scores + ((size_t)h * a.nq + qi) * a.n_pad + token + 4 * digit) = w;
        }
        // (ms is -Inf in a step that the query sees nothing of)
        const float m_new = fmaxf(m,ms), mr = m_new == -INFINITY? 0.0f : m_new;
        l = __builtin_fmaf(l,from_max(m,mr),sum * from_max(ms,mr));
        const float mo_old = mo + (m - mr), mo_step = mt + (ms - mr);  // both relative to the new maximum
        m = m_new;
        const float o_new = fmaxf(mo_old,mo_step), beta = from_max(mo_step,o_new);
        if (__builtin_amdgcn_ballot_w64(o_new != mo_old)) {
            const float alpha = from_max(mo_old,o_new);
#pragma unroll
            for (int t = 0; t < T; t++) o[t] *= alpha;
        }
        mo = o_new;
#pragma unroll
        for (int t = 0; t < T; t++) {
            const v4i y = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[t],pd,zero,0,0,0);
#pragma unroll
            for (int r = 0; r < 4; r++) o[t][r] = __builtin_fmaf((float)y[r],beta,o[t][r]);
        }
        if (more) load_values(step + WAVES);
    }

    // digits, then waves in order
    const float place = digit == 0? 0x1p-5f : digit == 1? 0x1p-12f : digit == 2? 0x1p-19f : 0x1p-26f;
    const float lt = rows_sum(l);
#pragma unroll
    for (int t = 0; t < T; t++) {
        v4f y;
#pragma unroll
        for (int r = 0; r < 4; r++) y[r] = quad_sum(o[t][r] * place);
        if (digit == 0) *reinterpret_cast<v4f*>(&so[wave][col >> 2][16 * t + 4 * g]) = y;
    }
    if (digit == 0 && g == 0) st[wave][col >> 2] = QueryStats{m,lt,mo};
    __syncthreads();
    for (int i = (int)threadIdx.x; i < kFewQ * D; i += 64 * WAVES) {
        const int j = i / D, d = i % D;
        if (q0 + j >= a.nq) continue;
        QueryStats all = {-INFINITY,0.0f,-INFINITY};
#pragma unroll
        for (int w = 0; w < WAVES; w++) all.s = fmaxf(all.s,st[w][j].s);
        float other[WAVES], acc = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            other[w] = moved_o(st[w][j],all.s);
            all.o = fmaxf(all.o,other[w]);
        }
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            acc = __builtin_fmaf(from_max(other[w],all.o),so[w][j][d],acc);
            all.l = __builtin_fmaf(from_max(st[w][j].s,all.s),st[w][j].l,all.l);
        }
        const size_t query = (size_t)h * a.nq + q0 + j;
        if (a.pieces > 1) a.part[(query * a.pieces + piece) * D + d] = acc;
        else if (d < a.c.dim) output_at(a,h,q0 + j)[d] = acc / all.l * from_max(all.o,0.0f);  // (the sum itself may pass fp32's range)
        if (d == 0 && (a.pieces > 1 || SCORES)) a.stats[query * a.pieces + piece] = make_float4(all.s,all.l,all.o,0.0f);
    }
}

__device__ __forceinline__ float wave_max(float v)
{
    v = fmaxf(v,xor_lane<1>(v));
    v = fmaxf(v,xor_lane<2>(v));
    v = fmaxf(v,xor_lane<4>(v));
    v = fmaxf(v,xor_lane<8>(v));
    return rows_max(v);
}

// A query's QueryStats over its pieces, in every lane of the wave (at most
// kFewPieces = 128 of them); `own` are the factors of the output records of the
// pieces lane and lane + 64.
__device__ __forceinline__ QueryStats merged_stats(const float4* stats, int pieces, float (&own)[2])
{
    const int lane = (int)(threadIdx.x & 63);
    const float4 none = {-INFINITY,0.0f,-INFINITY,0.0f};
    const float4 a = lane < pieces? stats[lane] : none, b = lane + 64 < pieces? stats[lane + 64] : none;
    QueryStats all = {wave_max(fmaxf(a.x,b.x)),0.0f,-INFINITY};
    const float oa = moved_o({a.x,a.y,a.z},all.s), ob = moved_o({b.x,b.y,b.z},all.s);
    all.o = wave_max(fmaxf(oa,ob));
    all.l = wave_sum(a.y * from_max(a.x,all.s) + b.y * from_max(b.x,all.s));
    own[0] = from_max(oa,all.o);
    own[1] = from_max(ob,all.o);
    return all;
}

// One wave merges the pieces of a query: half a wave (a quarter at D = 64) a
// record, 16 bytes a lane, eight loads at a time; `lds` holds the factors and is
// the wave's own (128 floats).
template <int D>
__device__ __forceinline__ void merge_query(const CAArgs& a, int h, int qi, float* lds)
{
    constexpr int T = D / 4, G = 64 / T, N = 8;
    const int lane = (int)(threadIdx.x & 63), d = 4 * (lane % T), first = lane / T;
    const size_t query = (size_t)h * a.nq + qi;
    float own[2];
    const QueryStats all = merged_stats(a.stats + query * a.pieces,a.pieces,own);
    lds[lane] = own[0];
    lds[lane + 64] = own[1];
    const float* part = a.part + query * a.pieces * D + d;
    float4 acc = {0.0f,0.0f,0.0f,0.0f};
    for (int p = first; p < a.pieces; p += G * N) {
        float4 x[N];
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = *reinterpret_cast<const float4*>(part + (size_t)min(p + G * i,a.pieces - 1) * D);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float f = p + G * i < a.pieces? lds[p + G * i] : 0.0f;
            acc.x = __builtin_fmaf(f,x[i].x,acc.x);
            acc.y = __builtin_fmaf(f,x[i].y,acc.y);
            acc.z = __builtin_fmaf(f,x[i].z,acc.z);
            acc.w = __builtin_fmaf(f,x[i].w,acc.w);
        }
    }
    if constexpr (G == 4) {
        acc.x += xor_lane<16>(acc.x);
        acc.y += xor_lane<16>(acc.y);
        acc.z += xor_lane<16>(acc.z);
        acc.w += xor_lane<16>(acc.w);
    }
    acc.x += xor_lane<32>(acc.x);
    acc.y += xor_lane<32>(acc.y);
    acc.z += xor_lane<32>(acc.z);
    acc.w += xor_lane<32>(acc.w);
    if (first || d >= a.c.dim) return;
    const float scale = from_max(all.o,0.0f) / all.l;
    float* to = output_at(a,h,qi) + d;
    const float out[4] = {acc.x * scale,acc.y * scale,acc.z * scale,acc.w * scale};
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (d + e < a.c.dim) to[e] = out[e];
}

// Merges the pieces of the queries, a wave each, in the first `outputs` workgroups;
// those behind add up the weights of a few queries: 1024 tokens of one kv head
// get the probabilities that the kept scores and the queries' merged sums give.
// (The last workgroup of a query's pieces merging them, after a ticket, made
// this launch unnecessary, but the fences that takes cross the XCDs' caches: a
// step over 131072 tokens, 512 workgroups, 59 -> 71 us.  Shorter caches were not tried.)
template <int D>
__global__ __launch_bounds__(256) void cache_combine_kernel(CAArgs a, int outputs)
{
    __shared__ float lds[4][128];
    __shared__ float2 sq[kFewMax];
    __shared__ int spoiled[kFewMax];  // tokens that a query which is not finite sees, or 0
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if ((int)blockIdx.x < outputs) {
        const int i = (int)blockIdx.x * 4 + wave;
        if (i < a.c.kv_heads * a.nq) merge_query<D>(a,i / a.nq,i % a.nq,lds[wave]);
        return;
    }
    const int groups = (a.n + 1023) / 1024, id = (int)blockIdx.x - outputs, h = id / groups, j = id % groups * 1024 + 4 * tid;
    static_assert(kFewMax == 32,"8 threads per query");
    if (const int q = tid / 8; q < a.nq) {
        const float4* stats = a.stats + ((size_t)h * a.nq + q) * a.pieces;
        float m = -INFINITY, l = 0.0f;
        auto add = [&](float s, float sum) {
            const float top = fmaxf(m,s);
            l = __builtin_fmaf(from_max(s,top),sum,l * from_max(m,top));
            m = top;
        };
#pragma unroll 4
        for (int p = tid % 8; p < a.pieces; p += 8) {
            const float4 x = stats[p];
            add(x.x,x.y);
        }
        add(xor_lane<1>(m),xor_lane<1>(l));
        add(xor_lane<2>(m),xor_lane<2>(l));
        add(xor_lane<4>(m),xor_lane<4>(l));
        if (tid % 8 == 0) {
            sq[q] = l == l? make_float2(m,1.0f / l) : make_float2(0.0f,0.0f);
            spoiled[q] = l == l? 0 : row_limit(a,query_row(a,q));
        }
    }
    __syncthreads();
    const int lane = tid & 63;
    uint32_t seen = lane < a.nq? (uint32_t)spoiled[lane] : 0;
    seen = max(seen,xor_lane<1>(seen));
    seen = max(seen,xor_lane<2>(seen));
    seen = max(seen,xor_lane<4>(seen));
    seen = max(seen,xor_lane<8>(seen));
    seen = max(seen,xor_lane<16>(seen));
    const int bad = __builtin_amdgcn_readfirstlane((int)seen);  // (of 32 lanes: kFewMax)
    if (j >= a.n) return;
    float4 w = {0.0f,0.0f,0.0f,0.0f};
#pragma unroll 4
    for (int q = 0; q < a.nq; q++) {
        const float4 s = *reinterpret_cast<const float4*>(a.scores + ((size_t)h * a.nq + q) * a.n_pad + j);
        w.x = __builtin_fmaf(__builtin_amdgcn_exp2f(s.x - sq[q].x),sq[q].y,w.x);
        w.y = __builtin_fmaf(__builtin_amdgcn_exp2f(s.y - sq[q].x),sq[q].y,w.y);
        w.z = __builtin_fmaf(__builtin_amdgcn_exp2f(s.z - sq[q].x),sq[q].y,w.z);
        w.w = __builtin_fmaf(__builtin_amdgcn_exp2f(s.w - sq[q].x),sq[q].y,w.w);
    }
    if (j < bad) w.x = NAN;
    if (j + 1 < bad) w.y = NAN;
    if (j + 2 < bad) w.z = NAN;
    if (j + 3 < bad) w.w = NAN;
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

// ---------------------------------------------------------------- many queries
//
// A chunk of rows: bound by the matrix cores.  8-bit codes are exact in fp16, so
// only q and p are split, x = hi + lo in fp16 (22 bits), and each product is two
// v_mfma_f32_32x32x16_f16 with fp32 accumulation (three for fp32 keys and
// values, attention.hip).  A workgroup of 4 waves owns 128 entries of a kv head's
// list of queries (32 per wave, Q in registers) and streams steps of 64 tokens
// through two LDS stages: codes wait in registers and are turned into fp16 on
// their way to LDS, once for all four waves.  Per 32-token block a wave computes
// S^T = K Q^T (a lane owns one query and 16 of the tokens), then O^T += V^T P^T
// with the lane's own S^T results as the P^T operand; V^T rows hold each 16
// tokens' words in the order 0, 2, 1, 3, which is the order S^T comes out in.
// The running maxima (QueryStats) are raised only when a step exceeds one by more
// than 2^8.
//
// One wave per SIMD, all its registers: in order, a wave waits at a matrix
// instruction while the matrix core is taken, so the vector ALU's work goes
// between them, a step apart: S^T of the next step runs with the probabilities of
// this one, O^T of this one with the conversion of the codes to come and the
// maxima of S^T.  What bounds it is that mix: on random operands a SIMD of this
// chip takes 21.3 ns for such a product by itself (1.57 PFLOP/s), 29 to 30 ns with
// 8 vector instructions beside it, however many waves share it; a step is 64 of
// them with 480, and takes 2.0 us.  128 rows of 32 heads over 16401 tokens: 76 us,
// of them 66 in the steps.
constexpr int kTileQ = 128, kTileThreads = 256;
constexpr float kUnset = -3.4028235e38f, kSlack = 8.0f;  // (no score is below the first)
// p's unit in fp16: with the slack and a scale's fraction it stays below 2^15,
// and the smallest half (2^-24, subnormal) is 2^-30 of a row's largest term.
constexpr float kPUnit = 64.0f, kPUnitLog2 = 6.0f;

// Four codes in a word as fp16: the byte plus 128 behind the exponent of 1024,
// less 1152 (exact).
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& a, uint32_t& b)
{
    w ^= 0x80808080u;
    const v2h bias = {(_Float16)1152.0f,(_Float16)1152.0f};
    a = __builtin_bit_cast(uint32_t,__builtin_bit_cast(v2h,__builtin_amdgcn_perm(0x64646464u,w,0x04010400u)) - bias);
    b = __builtin_bit_cast(uint32_t,__builtin_bit_cast(v2h,__builtin_amdgcn_perm(0x64646464u,w,0x04030402u)) - bias);
}

// Rows in LDS are 16 bytes longer than their 2 D bytes of keys or 128 of values:
// 16 rows' reads at one piece spread over all banks, and every address is the
// lane's own plus a constant.
template <int D> constexpr int kTileKeyRow = 2 * D + 16;
constexpr int kTileValueRow = 2 * kFewTile + 16;
template <int D> constexpr int kTileKeys = kFewTile * kTileKeyRow<D>;
template <int D> constexpr int kTileStage = kTileKeys<D> + D * kTileValueRow;

// A query's dims 16 k + 8 (lane / 32) .. + 7 as fp16 halves of q 2^s with the
// largest in [2^14, 2^15); returns the value 2^-s of a unit (NaN where a value is
// not finite).
template <int KS>
__device__ __forceinline__ float split_query(const float* p, int dim, bool vec, v8h (&hi)[KS], v8h (&lo)[KS])
{
    const int hh = (int)(threadIdx.x & 63) >> 5;
    float x[KS][8];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < KS; k++) {
        const int d = 16 * k + 8 * hh;
        if (vec) {  // dim a multiple of 4, 16-byte aligned rows
            const v4f a = *reinterpret_cast<const v4f*>(p + min(d,dim - 4)), b = *reinterpret_cast<const v4f*>(p + min(d + 4,dim - 4));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                x[k][i] = d < dim? a[i] : 0.0f;
                x[k][4 + i] = d + 4 < dim? b[i] : 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float w = p[min(d + i,dim - 1)];
                x[k][i] = d + i < dim? w : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) top = max(top,__float_as_uint(x[k][i]) & 0x7FFFFFFFu);  // (NaN above infinity above the rest)
    }
    top = max(top,xor_lane<32>(top));
    const bool finite = top < 0x7F800000u;
    const int s = finite && top? 15 - __builtin_amdgcn_frexp_expf(__uint_as_float(top)) : 0;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float v = finite? __builtin_ldexpf(x[k][i],s) : 0.0f;
            hi[k][i] = (_Float16)v;
            lo[k][i] = (_Float16)(v - (float)hi[k][i]);
        }
    return finite? __builtin_ldexpf(1.0f,-s) : NAN;
}

template <int D>
__global__ __launch_bounds__(kTileThreads,1) void cache_tile_kernel(CAArgs a)
{
    constexpr int KS = D / 16, TD = D / 32, U = D / 64;
    constexpr int PRODUCTS = 2 * KS;  // pairs of matrix instructions of S^T, and of O^T
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kTileStage<D>];
    // workgroups of one kv head next to each other in steps of kv_heads: with 8
    // kv heads those of one head share an XCD's cache
    const int h = (int)blockIdx.x % a.c.kv_heads, rest = (int)blockIdx.x / a.c.kv_heads;
    const int qt = rest % a.tiles_q, piece = rest / a.tiles_q;
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, lr = lane & 31, hh = lane >> 5;
    const int qi = qt * kTileQ + wave * 32 + lr, qc = min(qi,a.nq - 1);
    const int limit = row_limit(a,query_row(a,qc));
    const int wg_limit = row_limit(a,query_row(a,min((qt + 1) * kTileQ,a.nq) - 1));
    const int wave_limit = row_limit(a,query_row(a,min(qt * kTileQ + wave * 32,a.nq - 1)));  // the smallest of the wave
    const int steps = (wg_limit + kFewTile - 1) / kFewTile;
    const int t0 = piece * a.chunk, t1 = min(steps,t0 + a.chunk);
    const int nb = (a.n + kCacheBlock - 1) / kCacheBlock;
    const int32_t* table = a.c.table + (size_t)h * a.c.blocks;
    const size_t head_block = (size_t)h * a.c.blocks;

    // This thread's 16-byte pieces of a step's codes: piece tid + 256 u of the two
    // blocks' 2 D each, keys and values alike.  All of the loop's loads are vector
    // loads, which come back in order: behind scalar ones the waits for LDS would
    // wait for those too.  A step's places in memory are read ahead of its codes.
    v4i kc[U], vc[U];
    struct Pair {
        float k[2], v[2];
    };
    struct Places {
        int b[2];
    };
    int per_lane;  // 0, for all that the compiler knows another one in each lane
    asm("v_mov_b32 %0, 0" : "=v"(per_lane));
    int32_t place[2];
    auto load_places = [&](int t, int32_t (&to)[2]) {
        t = max(t0,min(t,t1 - 1));
#pragma unroll
        for (int i = 0; i < 2; i++) to[i] = table[min(2 * t + i,nb - 1) + per_lane];
    };
    auto places = [&](const int32_t (&of)[2]) { return Places{__builtin_amdgcn_readfirstlane(of[0]),__builtin_amdgcn_readfirstlane(of[1])}; };
    auto load_scales = [&](Places b) {
        Pair sc;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const size_t at = head_block + (size_t)b.b[i] + per_lane;
            sc.k[i] = a.c.ks[at];
            sc.v[i] = a.c.vs[at];
        }
        return sc;
    };
    auto load_codes = [&](const int8_t* codes, Places b, v4i (&to)[U]) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int block = U == 2? u : wave >> 1, p = (tid + kTileThreads * u) % (2 * D);
            to[u] = *reinterpret_cast<const v4i*>(codes + (head_block + (size_t)b.b[block]) * (kCacheBlock * D) + 16 * p);
        }
    };
    Places next = {}, after = {};  // of the next step and the one behind it
    Pair scales = {};
    v4i kc1[U];  // keys of the second step
    if (t0 < t1) {
        int32_t place0[2], place1[2];
        load_places(t0,place0);
        load_places(t0 + 1,place1);
        load_places(t0 + 2,place);
        const Places first = places(place0);
        next = places(place1);
        load_codes(a.c.k,first,kc);
        load_codes(a.c.v,first,vc);
        load_codes(a.c.k,next,kc1);
        scales = load_scales(first);
    }

    v8h qh[KS], ql[KS];
    const float unit = split_query<KS>(query_at(a,h,qc),a.c.dim,a.qvec != 0,qh,ql);
    if (a.planes && piece == 0) {
        v8h* to = a.planes + (((size_t)h * (a.nq_pad / 32) + qt * 4 + wave) * 2 * KS) * 64 + lane;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            to[(2 * k) * 64] = qh[k];
            to[(2 * k + 1) * 64] = ql[k];
        }
        if (!hh) a.steps[(size_t)h * a.nq_pad + qt * kTileQ + wave * 32 + lr] = unit;
    }

    // One of the 4 U code words of this thread's keys (or values) turned into fp16,
    // and the 16 bytes of LDS that every second one fills: keys take words 0 1 and
    // 2 3, values (in the order of S^T) 0 2 and 1 3.
    uint32_t half[4];
    auto stage_word = [&](uint8_t* to, bool value, int i) {
        const int u = i / 4, j = i % 4;
        const int at = tid + kTileThreads * u, block = at / (2 * D), p = at % (2 * D);
        const int word = value? 2 * (j & 1) + (j >> 1) : j;
        codes_to_half((uint32_t)(value? vc[u][word] : kc[u][word]),half[2 * (j & 1)],half[2 * (j & 1) + 1]);
        if (!(j & 1)) return;
        const v4i w = {(int)half[0],(int)half[1],(int)half[2],(int)half[3]};
        if (value) {
            *reinterpret_cast<v4i*>(to + kTileKeys<D> + (p >> 1) * kTileValueRow + 16 * (4 * block + 2 * (p & 1) + (j >> 1))) = w;
        } else {
            const int tt = (p >> 5) / U, token = kCacheBlock * block + 16 * ((p & 7) >> 2) + 4 * tt + (p & 3);
            *reinterpret_cast<v4i*>(to + token * kTileKeyRow<D> + 16 * (2 * (4 * ((p >> 5) % U) + ((p >> 3) & 3)) + (j >> 1))) = w;
        }
    };

    // mo: relative to ms.  dl 2^dl_over: kPUnit 2^-mo, dl 0 while mo is unset; -mo has no
    // bound: a block of zero values raises ms alone.
    float ms = kUnset, mo = kUnset, l = 0.0f, dl = 0.0f;
    int dl_over = 0;
    // A step above these raises the maxima.  `rare`: a lane has kLargeScore, or
    // dl_over, and every step goes there.
    float ms_test = kUnset, mo_test = kUnset;
    bool rare = false;
    v16f o[TD], sa[2], sb[2];  // sa, sb: S^T of this step and the next one, in turn
#pragma unroll
    for (int t = 0; t < TD; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[t][r] = 0.0f;

    // product i of a step's S^T: 16 dims of one of its blocks
    auto key_at = [&](const uint8_t* buf, int i) {
        return *reinterpret_cast<const v8h*>(buf + (32 * (i & 1) + lr) * kTileKeyRow<D> + 16 * (2 * (i >> 1) + hh));
    };
    auto score_high = [&](v16f (&s)[2], v8h f, int i) {
        const v16f zero = {0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f,0.0f};
        s[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f,qh[i >> 1],i < 2? zero : s[i & 1],0,0,0);
    };
    auto score_low = [&](v16f (&s)[2], v8h f, int i) { s[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f,ql[i >> 1],s[i & 1],0,0,0); };
    // Two of a lane's 32 results of step t: hides what its query does not see if
    // the step may hold such tokens, and takes them into each block's largest.
    float top[2];
    auto max_part = [&](v16f (&s)[2], int i, int t, bool some_hidden) {
        const int b = i >> 3, r = 2 * (i & 7);
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {  // register r: token 8 (r / 4) + 4 hh + r % 4
            // out of the matrix cores' registers, and here, between the products
            // (that it must be in one makes the wait for the product the compiler's)
            asm volatile("" : : "a"(s[b][r + e]));
            x[e] = s[b][r + e];
            asm volatile("" : "+v"(x[e]));
            if (some_hidden) x[e] = 8 * (r >> 2) + (r & 3) + e < limit - 4 * hh - (kFewTile * t + 32 * b)? x[e] : -INFINITY;
            s[b][r + e] = x[e];
        }
        // (written out: fmaxf first takes each operand's maximum with itself)
        if (r == 0) asm("v_max_f32 %0, %1, %2" : "=v"(top[b]) : "v"(x[0]), "v"(x[1]));
        else asm("v_max3_f32 %0, %1, %2, %0" : "+v"(top[b]) : "v"(x[0]), "v"(x[1]));
    };

    if (t0 < t1) {
#pragma unroll
        for (int i = 0; i < 4 * U; i++) stage_word(lds,false,i);
#pragma unroll
        for (int i = 0; i < 4 * U; i++) stage_word(lds,true,i);
#pragma unroll
        for (int u = 0; u < U; u++) kc[u] = kc1[u];
#pragma unroll
        for (int i = 0; i < 4 * U; i++) stage_word(lds + kTileStage<D>,false,i);
        after = places(place);
        load_codes(a.c.v,next,vc);
        load_codes(a.c.k,after,kc);
        load_places(t0 + 3,place);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PRODUCTS; i++) {
            const v8h f = key_at(lds,i);
            score_high(sa,f,i);
            score_low(sa,f,i);
        }
#pragma unroll
        for (int i = 0; i < 16; i++) max_part(sa,i,t0,true);
        __syncthreads();  // (its keys make room for those of step t0 + 2)
    }
    // Step t, whose values (and whose successor's keys) lie in LDS and whose S^T is
    // `s`; `n` gets the next step's.  `odd`: in the second LDS stage.
    auto run = [&](int t, v16f (&s)[2], v16f (&n)[2], auto odd, auto some_hidden, auto last) {
        uint8_t* const buf = lds + (odd.value? kTileStage<D> : 0);
        uint8_t* const other = lds + (odd.value? 0 : kTileStage<D>);
        Pair incoming = {};
        if constexpr (!last.value) incoming = load_scales(next);
        float c[2], e[2], v[2] = {scales.v[0],scales.v[1]};  // e: exponent of the block's value scale
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const uint32_t bits = __float_as_uint(scales.v[b]);
            c[b] = score_unit(unit,scales.k[b] * a.scale);
            top[b] = fmaxf(top[b],xor_lane<32>(top[b])) * c[b];
            e[b] = bits? (float)((int)(bits >> 23) - 127) : -INFINITY;
        }
        const float top2 = fmaxf(top[0],top[1]), over2 = fmaxf(top[0] + e[0],top[1] + e[1]);
        if (__builtin_amdgcn_ballot_w64(top2 > ms_test || over2 > mo_test)) {
            const float s_new = fmaxf(ms,top2), mo_old = mo + (ms - s_new);
            const float o_new = fmaxf(fmaxf(mo_old,kUnset),fmaxf((top[0] - s_new) + e[0],(top[1] - s_new) + e[1]));
            l *= __builtin_amdgcn_exp2f(ms - s_new);
            const float alpha = __builtin_amdgcn_exp2f(mo_old - o_new);
#pragma unroll
            for (int d = 0; d < TD; d++) o[d] *= alpha;
            ms = s_new;
            mo = o_new;
            const float gap = mo == kUnset? 0.0f : -mo;
            dl_over = (int)__builtin_ceilf(fminf(fmaxf(gap - 100.0f,0.0f),400.0f));
            dl = mo == kUnset? 0.0f : kPUnit * __builtin_amdgcn_exp2f(fminf(gap - (float)dl_over,100.0f));
            rare = __builtin_amdgcn_ballot_w64((dl_over != 0) | ((ms != kUnset) & (fabsf(ms) >= kLargeScore)));
            ms_test = rare? -INFINITY : ms + kSlack;
            mo_test = ms + mo + kSlack;
            if (__builtin_expect(rare,0)) {
#pragma unroll
                for (int b = 0; b < 2; b++) {
#pragma unroll
                    for (int r = 0; r < 16; r++) s[b][r] *= c[b];
                    c[b] = 1.0f;
                    v[b] = __builtin_ldexpf(v[b],dl_over);
                }
            }
        }
        // (a term whose probability is below 2^-111 is cut, not scaled up past fp32; a
        // block of zero values has the factor 0 whatever dl is)
        const float factor[2] = {fminf(dl * v[0],0x1p126f),fminf(dl * v[1],0x1p126f)};
        v8h ph[2][2], pl[2][2];
        float sum = 0.0f;
        // Probabilities 2 i, 2 i + 1 of the step, in the scale's unit.  The high
        // halves by the instruction that cuts, the low ones as what the product
        // itself leaves (written as two conversions of the rounded product, the
        // compiler folds it into one of them, and the two round apart at a tie).
        float p[2];
        auto take = [&](int i) {
#pragma unroll
            for (int e = 0; e < 2; e++) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i >> 3][2 * (i & 7) + e],c[i >> 3],-ms));
        };
        auto split = [&](int i) {
            const int b = i >> 3, r = 2 * (i & 7);
            sum += p[0] + p[1];
            const v2h hi = __builtin_bit_cast(v2h,__builtin_amdgcn_cvt_pkrtz(p[0] * factor[b],p[1] * factor[b]));
#pragma unroll
            for (int e = 0; e < 2; e++) {
                ph[b][r >> 3][(r & 7) + e] = hi[e];
                pl[b][r >> 3][(r & 7) + e] = (_Float16)__builtin_fmaf(p[e],factor[b],-(float)hi[e]);
            }
        };
        constexpr int EACH = 16 / PRODUCTS;
        v8h kf[2] = {};
        if constexpr (!last.value) {
            kf[0] = key_at(other,0);
            kf[1] = key_at(other,1);
        }
#pragma unroll
        for (int i = 0; i < PRODUCTS; i++) {
            const v8h f = kf[i & 1];
            if (!last.value && i + 2 < PRODUCTS) kf[i & 1] = key_at(other,i + 2);
            if constexpr (!last.value) score_high(n,f,i);
#pragma unroll
            for (int e = 0; e < EACH; e++) {
                take(EACH * i + e);
                if (e + 1 < EACH) split(EACH * i + e);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!last.value) score_low(n,f,i);
            split(EACH * (i + 1) - 1);
            asm volatile("" : "+v"(sum));  // (the sum here, not later from all of them)
            __builtin_amdgcn_sched_barrier(0);
        }
        l += sum;
        // O^T, and the codes of the keys two steps on and of the next values
        auto value_at = [&](int i) {  // product of (block, 16 tokens, 32 dims)
            return *reinterpret_cast<const v8h*>(buf + kTileKeys<D> + (32 * (i % TD) + lr) * kTileValueRow + 16 * (2 * (i / TD) + hh));
        };
        v8h vf[2] = {value_at(0),value_at(1)};
#pragma unroll
        for (int i = 0; i < PRODUCTS; i++) {
            const int d = i % TD, b = i / (2 * TD), k = i / TD % 2;
            const v8h f = vf[i & 1];
            if (i + 2 < PRODUCTS) vf[i & 1] = value_at(i + 2);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f,ph[b][k],o[d],0,0,0);
            if constexpr (!last.value) {
                if (i < 4 * U) stage_word(buf,false,i);
                else stage_word(other,true,i - 4 * U);
            }
            __builtin_amdgcn_sched_barrier(0);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f,pl[b][k],o[d],0,0,0);
            if constexpr (!last.value) {
#pragma unroll
                for (int e = 0; e < EACH; e++) max_part(n,EACH * i + e,t + 1,some_hidden.value);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (last.value) return;
        scales = incoming;
        next = after;
        after = places(place);
        load_codes(a.c.v,next,vc);
        load_codes(a.c.k,after,kc);
        load_places(t + 4,place);
        __syncthreads();
    };
    static_assert(PRODUCTS == 8 * U && PRODUCTS == 4 * TD && 16 % PRODUCTS == 0,"one code word per product");
    const std::false_type no{};
    const std::true_type yes{};
    const int open = min(t1,wave_limit / kFewTile) - 1;  // up to here the next step is whole and seen by every query
    int t = t0;
    for (; t + 1 < open; t += 2) {
        run(t,sa,sb,no,no,no);
        run(t + 1,sb,sa,yes,no,no);
    }
    for (; t + 2 < t1; t += 2) {
        run(t,sa,sb,no,yes,no);
        run(t + 1,sb,sa,yes,yes,no);
    }
    if (t + 1 < t1) {
        run(t,sa,sb,no,yes,no);
        run(t + 1,sb,sa,yes,yes,yes);
    } else if (t < t1) {
        run(t,sa,sb,no,yes,yes);
    }

    l += xor_lane<32>(l);
    const float es = ms == kUnset? -INFINITY : ms, eo = mo == kUnset? -INFINITY : mo - kPUnitLog2;
    if (a.pieces > 1) {
        // a record per wave, in the order its lanes hold it
        const size_t record = ((size_t)(h * a.tiles_q + qt) * a.pieces + piece) * 4 + wave;
        v4f* to = reinterpret_cast<v4f*>(a.part) + record * (4 * TD) * 64 + lane;
#pragma unroll
        for (int d = 0; d < TD; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) to[(4 * d + g) * 64] = v4f{o[d][4 * g],o[d][4 * g + 1],o[d][4 * g + 2],o[d][4 * g + 3]};
        if (!hh) a.stats[record * 32 + lr] = make_float4(es,l,eo,0.0f);
        return;
    }
    if (qi >= a.nq) return;
    if (a.merged && !hh) a.merged[(size_t)h * a.nq + qi] = make_float2(es,1.0f / l);
    const float scale = from_max(eo,0.0f) / l;
    float* to = output_at(a,h,qi) + 4 * hh;
#pragma unroll
    for (int d = 0; d < TD; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (32 * d + 8 * g + 4 * hh + r < a.c.dim) to[32 * d + 8 * g + r] = o[d][4 * g + r] * scale;
}

// Merges the pieces of 32 queries, 8 dims of them (4 of its lane's query) per
// workgroup, as the records' lanes hold them: its waves take every fourth piece
// and meet in LDS.
template <int D>
__global__ __launch_bounds__(256) void cache_tile_combine_kernel(CAArgs a)
{
    constexpr int SLOTS = D / 8, N = 4;
    __shared__ v4f lds_o[4][64];
    __shared__ QueryStats lds_s[4][64];
    const int lane = (int)threadIdx.x & 63, lr = lane & 31, hh = lane >> 5, wave = (int)threadIdx.x >> 6;
    const int slot = (int)blockIdx.x % SLOTS, group = (int)blockIdx.x / SLOTS, unit = group >> 2;  // unit, and its 32 queries
    const int h = unit / a.tiles_q, qi = unit % a.tiles_q * kTileQ + (group & 3) * 32 + lr;
    const size_t first = (size_t)unit * a.pieces * 4 + (group & 3);
    const float4* stats = a.stats + first * 32 + lr;
    const v4f* part = reinterpret_cast<const v4f*>(a.part) + (first * SLOTS + slot) * 64 + lane;
    QueryStats all = {-INFINITY,0.0f,-INFINITY};
    v4f acc = {0.0f,0.0f,0.0f,0.0f};
    auto add = [&](QueryStats x, v4f y) {
        const float s = fmaxf(all.s,x.s), had = moved_o(all,s), got = moved_o(x,s), o = fmaxf(had,got);
        const float down = from_max(had,o), f = from_max(got,o);
        all.l = __builtin_fmaf(from_max(x.s,s),x.l,all.l * from_max(all.s,s));
#pragma unroll
        for (int r = 0; r < 4; r++) acc[r] = __builtin_fmaf(f,y[r],acc[r] * down);
        all.s = s;
        all.o = o;
    };
    for (int p = wave; p < a.pieces; p += 4 * N) {
        float4 x[N];
        v4f y[N];
#pragma unroll
        for (int i = 0; i < N; i++) {
            const size_t at = (size_t)min(p + 4 * i,a.pieces - 1);
            x[i] = stats[at * 128];
            y[i] = part[at * (4 * SLOTS * 64)];
        }
#pragma unroll
        for (int i = 0; i < N; i++)
            if (p + 4 * i < a.pieces) add({x[i].x,x[i].y,x[i].z},y[i]);
    }
    lds_s[wave][lane] = all;
    lds_o[wave][lane] = acc;
    __syncthreads();
    if (wave || qi >= a.nq) return;
#pragma unroll
    for (int w = 1; w < 4; w++) add(lds_s[w][lane],lds_o[w][lane]);
    if (a.merged && !hh && !slot) a.merged[(size_t)h * a.nq + qi] = make_float2(all.s,1.0f / all.l);
    const float scale = from_max(all.o,0.0f) / all.l;
    const int at = 8 * slot + 4 * hh;
    float* to = output_at(a,h,qi) + at;
    if (a.ovec) {  // dim a multiple of 4, 16-byte aligned outputs
        if (at < a.c.dim) *reinterpret_cast<v4f*>(to) = acc * scale;
    } else {
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (at + r < a.c.dim) to[r] = acc[r] * scale;
    }
}

// The weights of a launch's queries: the probabilities again, from the split
// queries that cache_tile_kernel left and their merged maxima and sums.  A wave
// owns 64 tokens, whose keys stay in registers as fp16, and runs over queries of
// the kv head, 32 at a time: S = Q K^T, a lane owns one token and 16 of the
// queries, so that the sum over the queries stays in the lane.
template <int D> struct WeightTokens {
    static constexpr int KS = D / 16;
    v8h kf[2][KS];
    float ks[2], w[2];  // the block's part of a score's unit, and the sum
    size_t slot[2];
    int b0;

    __device__ __forceinline__ void load(const CAArgs& a, int h, int first_block, int nb)
    {
        const int lane = (int)threadIdx.x & 63, lr = lane & 31, hh = lane >> 5;
        b0 = first_block;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            slot[b] = (size_t)h * a.c.blocks + (size_t)a.c.table[(size_t)h * a.c.blocks + min(b0 + b,nb - 1)];
            ks[b] = a.c.ks[slot[b]] * a.scale;
            w[b] = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; k++) {  // dims 16 k + 8 hh .. + 7 of token lr
                const uint2 c = *reinterpret_cast<const uint2*>(a.c.k + slot[b] * (kCacheBlock * D) + cache_k_offset(lr,16 * k + 8 * hh,D));
                uint32_t x[4];
                codes_to_half(c.x,x[0],x[1]);
                codes_to_half(c.y,x[2],x[3]);
                kf[b][k] = __builtin_bit_cast(v8h,v4i{(int)x[0],(int)x[1],(int)x[2],(int)x[3]});
            }
        }
    }
    // Adds 32 queries' probabilities over the first B blocks.  `piece` gives fragment
    // i of their planes for this lane, `done` is told when the two of a 16-dim part
    // are used; `stats`: unit, maximum, inverse sum and limit of each query; HIDDEN:
    // not every query may see all of the tokens; `large`: kLargeScore in one of them.
    // It is compiled for the usual scores (USUAL), the large ones, or both.
    template <int B, bool HIDDEN, bool USUAL, bool LARGE, class Piece, class Done>
    __device__ __forceinline__ void add(Piece piece, Done done, const float4* stats, bool large)
    {
        const int lane = (int)threadIdx.x & 63, lr = lane & 31, hh = lane >> 5;
        v16f sc[B];
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
            for (int r = 0; r < 16; r++) sc[b][r] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            const v8h qh = piece(2 * k), ql = piece(2 * k + 1);
#pragma unroll
            for (int b = 0; b < B; b++) {
                sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(qh,kf[b][k],sc[b],0,0,0);
                sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ql,kf[b][k],sc[b],0,0,0);
            }
            done(k);
        }
        auto sum_up = [&](auto rounded) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float4 st = stats[8 * (r >> 2) + 4 * hh + (r & 3)];
#pragma unroll
                for (int b = 0; b < B; b++) {
                    // (the first pass left no score above its maximum by more than the slack)
                    const float c = st.x * ks[b], x = rounded.value? fminf(sc[b][r] * c - st.y,kSlack) : __builtin_fmaf(sc[b][r],c,-st.y);
                    const float sum = __builtin_fmaf(__builtin_amdgcn_exp2f(x),st.z,w[b]);
                    w[b] = !HIDDEN || kCacheBlock * (b0 + b) + lr < __float_as_int(st.w)? sum : w[b];
                }
            }
        };
        const float before[2] = {w[0],w[1]};
        if constexpr (USUAL) sum_up(std::false_type{});
        if (LARGE && (!USUAL || __builtin_expect(large,0))) {  // (again: the usual form follows its products without a branch)
            w[0] = before[0];
            w[1] = before[1];
            sum_up(std::true_type{});
        }
    }
    // Queries 32 t .. of the launch (the first one sees the fewest tokens).
    template <class Piece, class Done>
    __device__ __forceinline__ void add_tile(const CAArgs& a, int t, int nb, bool large, Piece piece, Done done, const float4* stats)
    {
        if (__builtin_expect(large,0)) add<2,true,false,true>(piece,done,stats,large);
        else if (32 * (t + 1) <= a.nq && kCacheBlock * (b0 + 2) <= row_limit(a,query_row(a,32 * t))) add<2,false,true,false>(piece,done,stats,large);
        else if (b0 + 1 < nb) add<2,true,true,false>(piece,done,stats,large);
        else if (b0 < nb) add<1,true,true,false>(piece,done,stats,large);
    }
    __device__ __forceinline__ void store(const CAArgs& a, int b, float sum) const
    {
        const int lane = (int)threadIdx.x & 63, lr = lane & 31;
        if (lane >= 32 || kCacheBlock * (b0 + b) + lr >= a.n) return;
        float* to = a.c.weights + slot[b] * kCacheBlock + lr;
        *to = a.decay == 0.0f? sum : __builtin_fmaf(a.decay,*to,sum);
    }
};

// Query 32 t + i of a launch for WeightTokens::add; one behind the last sees nothing.
__device__ __forceinline__ float4 weight_stats(const CAArgs& a, int h, int t, int i)
{
    const int q = min(32 * t + i,a.nq - 1);
    const float2 st = a.merged[(size_t)h * a.nq + q];
    const int limit = 32 * t + i < a.nq? row_limit(a,query_row(a,q)) : 0;
    return make_float4(a.steps[(size_t)h * a.nq_pad + q],st.x,st.y,__int_as_float(limit));
}

// Long caches: four waves of 64 tokens each take all queries, whose planes pass
// through LDS once for the four.  Where every query of a tile sees all of the
// wave's tokens (all but a chunk's own) nothing is compared: of 51 us for 128 rows
// of 32 heads over 16401 tokens that saves 6.  The products by themselves would
// take 22 us; with the next tile's products between the probabilities it came to
// 49, two waves of each SIMD fill the gaps of one another as well.
template <int D>
__global__ __launch_bounds__(kTileThreads,2) void cache_tile_weights_kernel(CAArgs a)
{
    constexpr int KS = D / 16, PIECES = 2 * KS * 64;  // 16-byte pieces of 32 queries' planes
    __shared__ __attribute__((aligned(16))) v8h lds[2][PIECES];
    __shared__ __attribute__((aligned(16))) float4 lq[2][32];
    const int h = (int)blockIdx.x % a.c.kv_heads, group = (int)blockIdx.x / a.c.kv_heads;
    const int tid = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int nb = (a.n + kCacheBlock - 1) / kCacheBlock;
    WeightTokens<D> tokens;
    tokens.load(a,h,(group * 4 + wave) * 2,nb);
    const int tiles = (a.nq + 31) / 32;
    const v8h* planes = a.planes + (size_t)h * (a.nq_pad / 32) * PIECES;
    v8h in[PIECES / kTileThreads];
    float4 inq = {};
    bool staged_large = false;  // (kLargeScore: every wave looks itself, rather than in LDS behind the barrier)
    auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < PIECES / kTileThreads; i++) in[i] = planes[(size_t)t * PIECES + kTileThreads * i + tid];
        if (tid < 32) inq = weight_stats(a,h,t,tid);
        else if (lane < 32) inq.y = a.merged[(size_t)h * a.nq + min(32 * t + lane,a.nq - 1)].x;
    };
    auto stage = [&](int i) {
#pragma unroll
        for (int e = 0; e < PIECES / kTileThreads; e++) lds[i][kTileThreads * e + tid] = in[e];
        if (tid < 32) lq[i][tid] = inq;
        staged_large = __builtin_amdgcn_ballot_w64(lane < 32 && fabsf(inq.y) >= kLargeScore);
    };
    load(0);
    stage(0);
    if (tiles > 1) load(1);
    __syncthreads();
    for (int t = 0; t < tiles; t++) {
        const v8h* buf = lds[t & 1] + lane;
        const bool large = staged_large;
        tokens.add_tile(a,t,nb,large,[&](int i) { return buf[64 * i]; },[](int) {},lq[t & 1]);
        if (t + 1 < tiles) {
            stage((t + 1) & 1);
            if (t + 2 < tiles) load(t + 2);
        }
        __syncthreads();
    }
#pragma unroll
    for (int b = 0; b < 2; b++) tokens.store(a,b,tokens.w[b] + xor_lane<32>(tokens.w[b]));
}

// Short caches: the waves of a workgroup share GROUPS times 64 tokens and take
// every eighth (or fourth) tile of queries, so that a launch of few tokens is not a
// few workgroups that run over all queries in a row.  The planes come from the L2
// cache into registers, each for the next tile as soon as it is used (read where
// they are used, a tile took 5 us instead of 2.5).
constexpr int kShareWaves = 8;
// Groups of 64 tokens, of all kv heads, that are taken one by one; up to twice as
// many are taken in twos.  A weighed call, us, one by one / in twos / by the kernel
// above: 512 queries of 2 kv heads at 4000 tokens (126 groups) 30.6 / 34.2 / 48.9, of 8
// at 2100 (264) 39.5 / 37.1 / 53.0, at 4000 (504) 45.4 / 43.6 / 58.4, at 8000 (1000)
// 71.7 / 67.8 / 74.4, at 16001 125 / 117 / 112; 64 queries of 8 at 2100 25.7 / 23.3 /
// 24.9.
constexpr int kShareGroups = 256;
template <int D, int GROUPS>
__global__ __launch_bounds__(64 * kShareWaves,2) void cache_tile_weights_share_kernel(CAArgs a)
{
    constexpr int PIECES = 2 * (D / 16) * 64, SPLIT = kShareWaves / GROUPS;  // waves of one group of tokens
    __shared__ __attribute__((aligned(16))) float4 lq[kShareWaves][32];
    __shared__ float sums[kShareWaves][2][32];
    const int h = (int)blockIdx.x % a.c.kv_heads, group = (int)blockIdx.x / a.c.kv_heads;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = (int)threadIdx.x & 63;
    const int nb = (a.n + kCacheBlock - 1) / kCacheBlock;
    WeightTokens<D> tokens;
    tokens.load(a,h,2 * (GROUPS * group + wave % GROUPS),nb);
    const int tiles = (a.nq + 31) / 32;
    const v8h* planes = a.planes + (size_t)h * (a.nq_pad / 32) * PIECES + lane;
    float4 st = {};
    const int from = wave / GROUPS;
    if (lane < 32 && from < tiles) st = weight_stats(a,h,from,lane);
    // a tile's planes in registers, each replaced by the next tile's once it is used
    v8h q[2 * (D / 16)];
#pragma unroll
    for (int i = 0; i < 2 * (D / 16); i++) q[i] = planes[(size_t)min(from,tiles - 1) * PIECES + 64 * i];
    for (int t = from; t < tiles; t += SPLIT) {
        const bool large = __builtin_amdgcn_ballot_w64(lane < 32 && fabsf(st.y) >= kLargeScore);
        if (lane < 32) {
            lq[wave][lane] = st;
            if (t + SPLIT < tiles) st = weight_stats(a,h,t + SPLIT,lane);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL,"wavefront");  // (the wave's own part of LDS)
        __builtin_amdgcn_wave_barrier();
        const v8h* next = planes + (size_t)min(t + SPLIT,tiles - 1) * PIECES;
        tokens.template add<2,true,true,true>([&](int i) { return q[i]; },
                                    [&](int k) {
                                        q[2 * k] = next[64 * (2 * k)];
                                        q[2 * k + 1] = next[64 * (2 * k + 1)];
                                    },lq[wave],large);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL,"wavefront");
        __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const float sum = tokens.w[b] + xor_lane<32>(tokens.w[b]);
        if (lane < 32) sums[wave][b][lane] = sum;
    }
    __syncthreads();
    if (wave >= GROUPS) return;
#pragma unroll
    for (int b = 0; b < 2; b++) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < SPLIT; i++) sum += sums[GROUPS * i + wave][b][lane & 31];
        tokens.store(a,b,sum);
    }
}

}  // namespace

// Parts of the workspace: records of D values and statistics of a query's
// pieces, and the few-query kernel's scores.
static size_t ca_records(size_t kv_heads, size_t blocks)
{
    return std::min<size_t>(65536,kv_heads * blocks * 512);
}

// Queries per kv head of one launch of the many-query kernels that counts weights.
static size_t ca_plane_queries(size_t kv_heads)
{
    return std::max<size_t>(kTileQ,16384 / kv_heads / kTileQ * kTileQ);
}

static size_t ca_few_bytes(size_t kv_heads, size_t blocks)
{
    const size_t one = kv_heads * (blocks + 1) * kCacheBlock * sizeof(float);
    return std::max(one * kFewScores,std::min(one * kFewMax,kFewScoreBytes));
}

size_t cache_attention_workspace_bytes(size_t kv_heads, size_t blocks, int D)
{
    const size_t planes = kv_heads * ca_plane_queries(kv_heads) * (2 * D * sizeof(_Float16) + sizeof(float2) + sizeof(float));
    return ca_records(kv_heads,blocks) * (D * sizeof(float) + sizeof(float4)) + std::max(planes,ca_few_bytes(kv_heads,blocks));
}

// Merges the pieces of every query, and (kept scores) adds up the weights.
static hipError_t launch_combine(const CAArgs& a, hipStream_t s)
{
    const size_t outputs = a.pieces > 1? ((size_t)a.c.kv_heads * a.nq + 3) / 4 : 0;
    const size_t groups = outputs + (a.scores? (size_t)a.c.kv_heads * ((a.n + 1023) / 1024) : 0);
    if (!groups) return hipSuccess;
    if (groups > (size_t)INT32_MAX) return hipErrorInvalidValue;
    if (a.c.D == 128) cache_combine_kernel<128><<<dim3((unsigned)groups),dim3(256),0,s>>>(a,(int)outputs);
    else cache_combine_kernel<64><<<dim3((unsigned)groups),dim3(256),0,s>>>(a,(int)outputs);
    return hipGetLastError();
}

// Cuts the tokens into at most `want` pieces, as far as their records fit.
static void cut_tokens(CAArgs& a, size_t want, size_t queries)
{
    const size_t steps = ((size_t)a.n + kFewTile - 1) / kFewTile;
    const size_t fit = ca_records(a.c.kv_heads,a.c.blocks) / ((size_t)a.c.kv_heads * queries);
    want = std::max<size_t>(1,std::min({want,steps,(size_t)kFewPieces,fit}));
    a.chunk = (int)((steps + want - 1) / want);
    a.pieces = (int)((steps + a.chunk - 1) / a.chunk);
}

static hipError_t launch_few(CAArgs a, hipStream_t s)
{
    a.tiles_q = (a.nq + kFewQ - 1) / kFewQ;
    const size_t units = (size_t)a.c.kv_heads * a.tiles_q, steps = ((size_t)a.n + kFewTile - 1) / kFewTile;
    // A step for each wave, but no pieces (and no launch that merges them) up to two
    // for each of eight waves, three where there are many groups of queries and so
    // few pieces: 4 queries of 8 kv heads (8 groups) at 500 tokens 7.4 us whole / 9.3
    // in pieces, at 700 8.1 / 9.4, at 1000 9.4 / 9.4, at 1250 9.9 / 9.5; 128 queries
    // (256 groups) at 1000 10.6 / 14.2, at 1530 13.0 / 16.7; more groups than
    // compute units take four waves (256 queries at 300 tokens 14.3 / 9.6).  (Kept
    // scores take that launch anyway.)
    const bool wide = !a.scores && steps > (size_t)kFewWaves && units <= (size_t)device_cus() && steps <= (size_t)kFewWide * (units >= 64? 3 : 2);
    cut_tokens(a,wide? 1 : std::min((steps + kFewWaves - 1) / kFewWaves,kFewUnits / units),(size_t)a.nq);
    if (units * a.pieces > (size_t)INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(units * a.pieces)), block(64 * (wide? kFewWide : kFewWaves));
    if (wide && a.c.D == 128) cache_few_kernel<128,false,kFewWide><<<grid,block,0,s>>>(a);
    else if (wide) cache_few_kernel<64,false,kFewWide><<<grid,block,0,s>>>(a);
    else if (a.scores && a.c.D == 128) cache_few_kernel<128,true,kFewWaves><<<grid,block,0,s>>>(a);
    else if (a.scores) cache_few_kernel<64,true,kFewWaves><<<grid,block,0,s>>>(a);
    else if (a.c.D == 128) cache_few_kernel<128,false,kFewWaves><<<grid,block,0,s>>>(a);
    else cache_few_kernel<64,false,kFewWaves><<<grid,block,0,s>>>(a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess? launch_combine(a,s) : e;
}

static hipError_t launch_tile(CAArgs a, bool weigh, hipStream_t s)
{
    a.tiles_q = (a.nq + kTileQ - 1) / kTileQ;
    a.nq_pad = a.tiles_q * kTileQ;
    const size_t units = (size_t)a.c.kv_heads * a.tiles_q;
    cut_tokens(a,(size_t)device_cus() / units,(size_t)a.nq_pad);
    if (units * a.pieces > (size_t)INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(units * a.pieces)), block(kTileThreads);
    if (a.c.D == 128) cache_tile_kernel<128><<<grid,block,0,s>>>(a);
    else cache_tile_kernel<64><<<grid,block,0,s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.pieces > 1) {
        const size_t groups = units * 4 * (a.c.D / 8);
        if (groups > (size_t)INT32_MAX) return hipErrorInvalidValue;
        const dim3 parts((unsigned)groups);
        if (a.c.D == 128) cache_tile_combine_kernel<128><<<parts,dim3(256),0,s>>>(a);
        else cache_tile_combine_kernel<64><<<parts,dim3(256),0,s>>>(a);
        e = hipGetLastError();
    }
    if (e != hipSuccess || !weigh) return e;
    const size_t groups = ((size_t)a.n + kFewTile - 1) / kFewTile * a.c.kv_heads;
    if (groups > (size_t)INT32_MAX) return hipErrorInvalidValue;
    if (groups <= 2 * (size_t)kShareGroups) {
        const bool one = groups <= (size_t)kShareGroups;
        const dim3 tokens((unsigned)(one? groups : ((size_t)a.n + 2 * kFewTile - 1) / (2 * kFewTile) * a.c.kv_heads)), threads(64 * kShareWaves);
        if (one && a.c.D == 128) cache_tile_weights_share_kernel<128,1><<<tokens,threads,0,s>>>(a);
        else if (one) cache_tile_weights_share_kernel<64,1><<<tokens,threads,0,s>>>(a);
        else if (a.c.D == 128) cache_tile_weights_share_kernel<128,2><<<tokens,threads,0,s>>>(a);
        else cache_tile_weights_share_kernel<64,2><<<tokens,threads,0,s>>>(a);
        return hipGetLastError();
    }
    const dim3 tokens((unsigned)(((size_t)a.n + 4 * kFewTile - 1) / (4 * kFewTile) * a.c.kv_heads));
    if (a.c.D == 128) cache_tile_weights_kernel<128><<<tokens,block,0,s>>>(a);
    else cache_tile_weights_kernel<64><<<tokens,block,0,s>>>(a);
    return hipGetLastError();
}

hipError_t launch_cache_attention(const CacheLayer& c, const CacheAttention& a, void* workspace, hipStream_t s)
{
    const size_t group = a.heads / c.kv_heads, nq = a.rows * group, records = ca_records(c.kv_heads,c.blocks);
    CAArgs k = {};
    k.c = c;
    k.q = a.q;
    k.out = a.out;
    k.part = static_cast<float*>(workspace);
    k.stats = reinterpret_cast<float4*>(k.part + records * c.D);
    void* const more = k.stats + records;
    k.ld = a.ld;
    k.group = (int)group;
    k.rows = (int)a.rows;
    k.n = (int)a.length;
    k.n_pad = (k.n + kFewTile - 1) / kFewTile * kFewTile;
    k.causal = a.causal? 1 : 0;
    k.qvec = c.dim % 4 == 0 && a.ld % 4 == 0 && reinterpret_cast<uintptr_t>(a.q) % 16 == 0;
    k.ovec = c.dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
    k.scale = kCLog2e / sqrtf((float)c.dim);
    k.decay = a.decay;
    const bool few = a.weigh? nq <= (size_t)kFewMax && nq * c.kv_heads * k.n_pad * sizeof(float) <= ca_few_bytes(c.kv_heads,c.blocks)
                            : nq <= (size_t)kFewMax || (nq <= (size_t)kFewMaxShort && nq * a.length <= kFewPairs / c.kv_heads);
    if (few) {
        k.nq = (int)nq;
        k.scores = a.weigh? static_cast<float*>(more) : nullptr;
        return launch_few(k,s);
    }
    // As many queries of each kv head as fit one launch's grid and, where the
    // weights are counted, its planes.
    const size_t most = a.weigh? ca_plane_queries(c.kv_heads) : (size_t)1 << 20;
    for (size_t first = 0; first < nq; first += most) {
        k.first = (int)first;
        k.nq = (int)std::min(most,nq - first);
        if (a.weigh) {
            k.planes = static_cast<v8h*>(more);
            k.merged = reinterpret_cast<float2*>(k.planes + c.kv_heads * most * c.D / 4);
            k.steps = reinterpret_cast<float*>(k.merged + c.kv_heads * most);
            k.decay = first? 1.0f : a.decay;
        }
        const hipError_t e = launch_tile(k,a.weigh,s);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace pixhip
