// Log probabilities of given tokens, the entropy of their distributions and the
// most likely alternatives, over rows of logits x (gfx950):
//   m = max x, S = sum e^(x - m), log p(i) = x_i - m - log S,
//   entropy = log S - sum e^(x - m) (x - m) / S,
// the alternatives in the order of x, equal ones by the lower index.  A logit
// of -Inf is a token that cannot come (p = 0, no part in the entropy); a row of
// nothing else has log probabilities of -Inf and entropy 0.  NaN or +Inf in a
// row makes its log probabilities and entropy NaN; its alternatives are ordered
// with NaN as the lowest value.  An id outside the vocabulary gives NaN.
//
// One pass over the logits, each read once: bound by HBM.  A wave takes 1024
// logits at a time and keeps, per lane, the running maximum with the sum of the
// others relative to it (S - 1, so that log S = log1p of it stays exact where one
// token takes nearly all), the entropy's sum, and across its lanes the 64 best
// logits so far in order.  The first 1024 give each lane's best, sorted over the
// lanes; after that only a logit above the last of the wanted ones is put in, and
// above the least of what every wave of the workgroup has as its k-th, of which they
// hold as many as are wanted between them (128 rows of 151936 with 20 alternatives
// 40.7 -> 31.1 us, with 64 84.8 -> 37.9).  Lists meet two at a time (the larger ones
// of one and of the other reversed hold the 64 best), through LDS for the waves of a
// workgroup.
// Few rows are cut into pieces, whose lists and sums a second launch merges.
#include <math.h>

#include <algorithm>

#include "pixhip_device.h"
#include "pixhip_internal.h"

namespace pixhip {

namespace {

constexpr int kLPWaves = 8, kLPThreads = 64 * kLPWaves;
constexpr int kLPEach = 16, kLPChunk = 64 * kLPEach;  // logits per lane and per wave at a time
constexpr int kLPUnits = 512;                         // workgroups a launch is cut into, about
constexpr float kLPLog2e = 1.44269504088896340736f;
constexpr float kLPLn2 = 0.69314718055994530942f;

// A logit and its place as one number: larger logits, then lower places, give
// larger numbers; NaN counts as the lowest, -0 as 0; 0 is no logit.
__device__ __forceinline__ uint32_t lp_key(float x)
{
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u >> 31? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t lp_entry(float x, uint32_t i)
{
    return (uint64_t)lp_key(x) << 32 | (uint32_t)~i;
}

// The larger of v and lane ^ STEP's to the lane of the two whose bit is clear
// (`down`), or the smaller one.
template <int STEP> __device__ __forceinline__ uint64_t exchange(uint64_t v, bool down)
{
    const uint64_t u = xor_lane<STEP>(v);
    const bool low = ((int)threadIdx.x & STEP) == 0;
    return (low == down) == (u > v)? u : v;
}
// Both halves of every 2 STEP lanes, one of which is ascending, into order.
template <int STEP> __device__ __forceinline__ uint64_t bitonic(uint64_t v, bool down)
{
    v = exchange<STEP>(v,down);
    if constexpr (STEP > 1) v = bitonic<STEP / 2>(v,down);
    return v;
}
// Puts the lanes' values into descending order.
__device__ __forceinline__ uint64_t sort_lanes(uint64_t v)
{
    const int lane = (int)(threadIdx.x & 63);
    v = bitonic<1>(v,(lane & 2) == 0);
    v = bitonic<2>(v,(lane & 4) == 0);
    v = bitonic<4>(v,(lane & 8) == 0);
    v = bitonic<8>(v,(lane & 16) == 0);
    v = bitonic<16>(v,(lane & 32) == 0);
    return bitonic<32>(v,true);
}
__device__ __forceinline__ uint64_t reverse_lanes(uint64_t v)
{
    const auto turn = [](uint32_t w) {
        return xor_lane<32>(xor_lane<16>((uint32_t)dpp_i32<kDppMirror>((int)w)));
    };
    return (uint64_t)turn((uint32_t)(v >> 32)) << 32 | turn((uint32_t)v);
}
// The 64 largest of two descending lists, descending.
__device__ __forceinline__ uint64_t merge_lists(uint64_t a, uint64_t b)
{
    const uint64_t r = reverse_lanes(b);
    return bitonic<32>(a > r? a : r,true);
}

// Puts `e` (the same in every lane, not in the list) into a descending list.
__device__ __forceinline__ uint64_t insert_entry(uint64_t list, uint64_t e)
{
    const int lane = (int)(threadIdx.x & 63);
    const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(list > e));
    const uint64_t before = (uint64_t)(uint32_t)dpp_i32<0x138>((int)(list >> 32)) << 32 | (uint32_t)dpp_i32<0x138>((int)list);  // wave_shr:1
    return lane < at? list : lane == at? e : before;
}

// Sums of some logits: m their maximum, `rest` the sum of e^(x - m) without one
// place of the maximum, whose term is `one` (1, or 0 in the lanes that do not
// have it), `mean` the sum of e^(x - m) (x - m) in log2 units.  NaN and +Inf make
// `rest` or `one` NaN.  No logit but -Inf: m = -Inf, one = 0.
struct LPSums {
    float m, one, rest, mean;
};
__device__ __forceinline__ LPSums join(LPSums a, LPSums b)
{
    const bool swap = b.m > a.m || (b.m == a.m && b.one > a.one);
    const LPSums hi = swap? b : a, lo = swap? a : b;
    const float d = (lo.m - hi.m) * kLPLog2e, f = lo.m == -INFINITY? 0.0f : __builtin_amdgcn_exp2f(d), all = lo.one + lo.rest;
    // (a part too far below counts nothing but its NaN)
    if (f == 0.0f) return {hi.m,hi.one,all == all? hi.rest : all,hi.mean};
    return {hi.m,hi.one,__builtin_fmaf(f,all,hi.rest),__builtin_fmaf(f,__builtin_fmaf(d,all,lo.mean),hi.mean)};
}
template <int MASK> __device__ __forceinline__ LPSums join_lane(LPSums a)
{
    return join(a,LPSums{xor_lane<MASK>(a.m),xor_lane<MASK>(a.one),xor_lane<MASK>(a.rest),xor_lane<MASK>(a.mean)});
}

// -Inf as a power of two that is 0 in fp32 but has a product with 0; NaN stays.
__device__ __forceinline__ float least_term(float y)
{
    return __builtin_elementwise_maximum(y,-200.0f);
}

struct LPArgs {
    LogProbs a;
    LPSums* sums;    // [rows][pieces]
    uint64_t* lists; // [rows][pieces][64]
    int pieces;
    size_t chunk;    // logits per piece, a multiple of kLPChunk
};

// What is known of a row's logits, by one wave.
__device__ __forceinline__ void write_row(const LogProbs& a, size_t row, LPSums s, uint64_t list)
{
    const int lane = (int)(threadIdx.x & 63);
    const float* x = a.x + row * a.ld;
    const bool none = s.m == -INFINITY && s.rest == s.rest;
    const float m = none? 0.0f : s.m, rest = none? 0.0f : s.rest + (s.one - 1.0f), norm = log1pf(rest);  // (one is 1, or NaN)
    if (lane == 0) {
        if (a.log_probs) {
            const int32_t id = a.ids[row];
            a.log_probs[row] = id < 0 || (size_t)id >= a.vocab? NAN : x[id] - m - norm;
        }
        if (a.entropy) a.entropy[row] = none? 0.0f : norm - s.mean * kLPLn2 / (1.0f + rest);
    }
    if (lane < a.top) {
        const uint32_t i = ~(uint32_t)list;
        a.top_ids[row * a.top + lane] = (int32_t)i;
        a.top_log_probs[row * a.top + lane] = x[i] - m - norm;
    }
}

// The waves' lists and sums, in a tree; wave 0 gets the whole.
template <int WAVES, bool TOP>
__device__ __forceinline__ void join_waves(LPSums& s, uint64_t& list)
{
    __shared__ uint64_t lists[TOP? WAVES / 2 : 1][64];
    __shared__ LPSums sums[WAVES];
    const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
    if (lane == 0) sums[wave] = s;
#pragma unroll
    for (int half = WAVES / 2; half > 0; half >>= 1) {
        if (TOP && wave >= half && wave < 2 * half) lists[wave - half][lane] = list;
        __syncthreads();
        if (TOP && wave < half) list = merge_lists(list,lists[wave][lane]);
        if (half > 1) __syncthreads();
    }
    if (wave) return;
    s = sums[lane % WAVES];
    s = join_lane<1>(s);
    s = join_lane<2>(s);
    s = join_lane<4>(s);
    static_assert(WAVES == 8,"three steps");
}

// One workgroup per piece of a row.  VEC: rows are 16-byte aligned.
template <bool TOP, bool VEC>
__global__ __launch_bounds__(kLPThreads,4) void log_probs_kernel(LPArgs p)
{
    __shared__ v4f held[TOP? kLPWaves : 1][TOP? kLPChunk / 4 : 1];
    const LogProbs& a = p.a;
    const int lane = (int)(threadIdx.x & 63), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const size_t row = blockIdx.x / (unsigned)p.pieces;
    const int piece = (int)(blockIdx.x % (unsigned)p.pieces);
    const float* x = a.x + row * a.ld;
    const size_t begin = piece * p.chunk, end = std::min(a.vocab,begin + p.chunk);
    // element e of a lane: 4 in a row per load, or one
    auto place = [&](size_t at, int e, int of) { return at + (VEC? 256 * (e >> 2) + 4 * of + (e & 3) : 64 * e + of); };
    auto load = [&](float (&v)[kLPEach], size_t at) {
        if (at + kLPChunk <= end) {
            if constexpr (VEC) {
#pragma unroll
                for (int j = 0; j < kLPEach / 4; j++) {
                    const v4f w = __builtin_nontemporal_load(reinterpret_cast<const v4f*>(x + at + 256 * j) + lane);
#pragma unroll
                    for (int c = 0; c < 4; c++) v[4 * j + c] = w[c];
                }
            } else {
#pragma unroll
                for (int e = 0; e < kLPEach; e++) v[e] = __builtin_nontemporal_load(x + at + 64 * e + lane);
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < kLPEach; e++) v[e] = place(at,e,lane) < end? x[place(at,e,lane)] : -INFINITY;
    };

    // the wave's maximum, and this lane's sums relative to it
    LPSums s = {-INFINITY,0.0f,0.0f,0.0f};
    uint64_t list = 0;
    // What an entry has to exceed to be wanted: the last wanted one of the list,
    // and (`shared`) the least of what each wave whose first step is whole has as
    // its k-th, of which they hold `a.top` between them.
    uint64_t bound = 0, shared = 0;
    float last = -INFINITY;  // its logit, while its key is not 0
    auto set_last = [&]() {
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(list >> 32),a.top - 1);
        const uint64_t own = (uint64_t)hi << 32 | (uint32_t)__builtin_amdgcn_readlane((int)list,a.top - 1);
        bound = own > shared? own : shared;
        const uint32_t key = (uint32_t)(bound >> 32);
        last = __uint_as_float(key >> 31? key & 0x7FFFFFFFu : ~key);
    };
    __shared__ uint64_t share[kLPWaves];
    const int whole = (int)std::min((end - begin) / kLPChunk,(size_t)kLPWaves);
    const int kth = whole? (a.top + whole - 1) / whole - 1 : 0;
    // (relaxed: a wave's entry only grows, and an earlier one bounds as well)
    auto publish = [&](uint64_t e) {
        if (lane == kth) __hip_atomic_store(&share[wave],e,__ATOMIC_RELAXED,__HIP_MEMORY_SCOPE_WORKGROUP);
    };
    auto set_shared = [&]() {
        uint64_t least = __hip_atomic_load(&share[lane % kLPWaves],__ATOMIC_RELAXED,__HIP_MEMORY_SCOPE_WORKGROUP);
        least = std::min(least,xor_lane<1>(least));
        least = std::min(least,xor_lane<2>(least));
        least = std::min(least,xor_lane<4>(least));
        static_assert(kLPWaves == 8,"three steps");
        if (whole) shared = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(least >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)least);
    };
    size_t at = begin + (size_t)wave * kLPChunk;
    float v[kLPEach];
    if (at < end) load(v,at);
    if constexpr (TOP) {
        if (wave >= whole) publish(~(uint64_t)0);
        if (at >= end) __syncthreads();  // (the others' first step)
    }
    for (bool first = true; at < end; at += kLPWaves * kLPChunk, first = false) {
        float x16[kLPEach];
#pragma unroll
        for (int e = 0; e < kLPEach; e++) x16[e] = v[e];
        if (at + kLPWaves * kLPChunk < end) load(v,at + kLPWaves * kLPChunk);
        float top = x16[0];
#pragma unroll
        for (int e = 1; e < kLPEach; e++) top = fmaxf(top,x16[e]);
        float all = fmaxf(top,xor_lane<1>(top));
        all = fmaxf(all,xor_lane<2>(all));
        all = fmaxf(all,xor_lane<4>(all));
        all = fmaxf(all,xor_lane<8>(all));
        all = fmaxf(all,xor_lane<16>(all));
        all = fmaxf(all,xor_lane<32>(all));
        if (all > s.m) {  // (wave-uniform) the old maximum's term joins the others
            const float d = (s.m - all) * kLPLog2e, f = s.m == -INFINITY? 0.0f : __builtin_amdgcn_exp2f(d);
            s.rest += s.one;
            s.mean = f == 0.0f? 0.0f : f * __builtin_fmaf(d,s.rest,s.mean);
            s.rest *= f;
            s.m = all;
            // one lane leaves the new one out of `rest`
            const uint64_t has = __builtin_amdgcn_ballot_w64(top == all);
            bool mine = has && lane == __builtin_ctzll(has);
            s.one = mine? (all < INFINITY? 1.0f : NAN) : 0.0f;
#pragma unroll
            for (int e = 0; e < kLPEach; e++) {
                const float y = least_term((x16[e] - all) * kLPLog2e);
                const bool it = mine && x16[e] == all;
                mine = mine && !it;
                const float w = it? 0.0f : __builtin_amdgcn_exp2f(y);
                s.rest += w;
                s.mean = __builtin_fmaf(w,y,s.mean);
            }
        } else {
            const float shift = s.m == -INFINITY? 0.0f : s.m;
#pragma unroll
            for (int e = 0; e < kLPEach; e++) {
                const float y = least_term((x16[e] - shift) * kLPLog2e);
                const float w = __builtin_amdgcn_exp2f(y);
                s.rest += w;
                s.mean = __builtin_fmaf(w,y,s.mean);
            }
        }
        if constexpr (TOP) {
            float reach = top;  // the lane's largest logit that is not in the list
            int which = -1;     // its element that is
            if (first) {
                which = 0;
                reach = -INFINITY;
#pragma unroll
                for (int e = kLPEach - 1; e >= 0; e--) which = x16[e] == top? e : which;
#pragma unroll
                for (int e = 0; e < kLPEach; e++) reach = e == which? reach : fmaxf(reach,x16[e]);
                const size_t i = place(at,which,lane);
                list = sort_lanes(i < end? lp_entry(top,(uint32_t)i) : 0);
                if (wave < whole) publish(list);
                __syncthreads();
                set_shared();
                set_last();
            }
            // lanes that reach the bound (after the first step few do; a place
            // behind the bound's does not with an equal logit): each one's 16
            // logits come over 16 lanes through LDS, the wave's own part
            auto reaching = [&]() {
                const bool key = bound >> 32, equal = at < ~(uint32_t)bound;
                return __builtin_amdgcn_ballot_w64(key? reach > last || (equal && reach == last) : true);
            };
            uint64_t lanes = reaching();
            if (lanes && !first) {  // (the others may have raised it)
                set_shared();
                set_last();
                lanes = reaching();
            }
            if (!lanes) continue;
            v4f* const mine = held[wave];
#pragma unroll
            for (int j = 0; j < kLPEach / 4; j++) mine[kLPEach / 4 * lane + j] = v4f{x16[4 * j],x16[4 * j + 1],x16[4 * j + 2],x16[4 * j + 3]};
            while (lanes) {
                const int from = __builtin_ctzll(lanes);
                lanes &= lanes - 1;
                const float y = reinterpret_cast<const float*>(mine)[kLPEach * from + (lane & (kLPEach - 1))];
                const size_t i = place(at,lane & (kLPEach - 1),from);
                const uint64_t c = lp_entry(y,(uint32_t)i);
                uint64_t hits = __builtin_amdgcn_ballot_w64(lane < kLPEach && i < end && lane != __builtin_amdgcn_readlane(which,from) && c > bound);
                if (!hits) continue;
                while (hits) {
                    const int l = __builtin_ctzll(hits);
                    hits &= hits - 1;
                    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(c >> 32),l);
                    list = insert_entry(list,(uint64_t)hi << 32 | (uint32_t)__builtin_amdgcn_readlane((int)c,l));
                }
                set_last();
            }
            if (wave < whole) publish(list);
        }
    }
    s = join_lane<1>(s);
    s = join_lane<2>(s);
    s = join_lane<4>(s);
    s = join_lane<8>(s);
    s = join_lane<16>(s);
    s = join_lane<32>(s);
    join_waves<kLPWaves,TOP>(s,list);
    if (wave) return;
    if (p.pieces == 1) {
        write_row(a,row,s,list);
        return;
    }
    if (TOP) p.lists[((size_t)blockIdx.x) * 64 + lane] = list;
    if (lane == 0) p.sums[blockIdx.x] = s;
}

// Merges a row's pieces, a workgroup per row.
template <bool TOP>
__global__ __launch_bounds__(kLPThreads) void log_probs_merge_kernel(LPArgs p)
{
    const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
    const size_t row = blockIdx.x;
    LPSums s = {-INFINITY,0.0f,0.0f,0.0f};
    uint64_t list = 0;
    constexpr int N = 4;  // pieces whose loads are under way together
    for (int i0 = wave; i0 < p.pieces; i0 += N * kLPWaves) {
        LPSums sums[N];
        uint64_t lists[N];
#pragma unroll
        for (int n = 0; n < N; n++) {
            const size_t i = row * p.pieces + (size_t)min(i0 + n * kLPWaves,p.pieces - 1);
            sums[n] = p.sums[i];
            if (TOP) lists[n] = p.lists[i * 64 + lane];
        }
#pragma unroll
        for (int n = 0; n < N; n++) {
            if (i0 + n * kLPWaves >= p.pieces) break;
            s = join(s,sums[n]);
            if (TOP) list = merge_lists(list,lists[n]);
        }
    }
    join_waves<kLPWaves,TOP>(s,list);
    if (wave == 0) write_row(p.a,row,s,list);
}

// Pieces of a row: enough to fill the device, each at least one step of its
// workgroup's waves.
int lp_pieces(size_t rows, size_t vocab)
{
    const size_t steps = (vocab + kLPWaves * kLPChunk - 1) / (kLPWaves * kLPChunk);
    return (int)std::max<size_t>(1,std::min(steps,kLPUnits / std::max<size_t>(rows,1)));
}

}  // namespace

size_t log_probs_workspace_bytes(size_t rows, size_t vocab)
{
    const size_t pieces = (size_t)lp_pieces(rows,vocab);
    return pieces > 1? rows * pieces * (64 * sizeof(uint64_t) + sizeof(LPSums)) : 0;
}

hipError_t launch_log_probs(const LogProbs& a, void* workspace, hipStream_t s)
{
    LPArgs p = {};
    p.a = a;
    p.pieces = workspace? lp_pieces(a.rows,a.vocab) : 1;
    const size_t steps = (a.vocab + kLPWaves * kLPChunk - 1) / (kLPWaves * kLPChunk);
    p.chunk = (steps + p.pieces - 1) / p.pieces * kLPWaves * kLPChunk;
    p.pieces = (int)((a.vocab + p.chunk - 1) / p.chunk);
    if (a.rows * p.pieces > (size_t)INT32_MAX) return hipErrorInvalidValue;
    p.lists = static_cast<uint64_t*>(workspace);
    if (workspace) p.sums = reinterpret_cast<LPSums*>(p.lists + a.rows * p.pieces * 64);
    const dim3 grid((unsigned)(a.rows * p.pieces)), block(kLPThreads);
    const bool vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && (a.ld % 4 == 0 || a.rows == 1);
    if (a.top) {
        if (vec) log_probs_kernel<true,true><<<grid,block,0,s>>>(p);
        else log_probs_kernel<true,false><<<grid,block,0,s>>>(p);
    } else {
        if (vec) log_probs_kernel<false,true><<<grid,block,0,s>>>(p);
        else log_probs_kernel<false,false><<<grid,block,0,s>>>(p);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.pieces == 1) return e;
    if (a.top) log_probs_merge_kernel<true><<<dim3((unsigned)a.rows),block,0,s>>>(p);
    else log_probs_merge_kernel<false><<<dim3((unsigned)a.rows),block,0,s>>>(p);
    return hipGetLastError();
}

}  // namespace pixhip
