// One attention head of one row, normalized and rotated by G lanes (16: heads of
// up to 128 values, 64: up to 512), 8 values a lane as four pairs (a, b):
//   n = (x - mean) * inverse * weight     tensor_norm (src/tensor.cpp:174-197), the
//                                         statistics in double
//   (a, b) -> (a*c - b*s, a*s + b*c)      tensor_rope (:429-452) over the leading
//                                         `rotary` values, the others as they are
// in fp32, operation by operation.  Both values of a pair are in one lane, so the
// rotation moves nothing between lanes.
#pragma once

#include "heads_index.h"
#include "pixhip_device.h"
#include "pixhip_internal.h"

namespace pixhip {

struct Pairs {
    float a[4], b[4];
};

// The lane's values of the head at `p`, zeros past it.  The loads are unconditional
// (clamped), so that none waits for another.
template <int G, int MODE>
__device__ __forceinline__ Pairs turn_load(const HeadTurn& t, const float* p, int lp)
{
    Pairs v;
    if constexpr (MODE == kTurnScalar) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            int ia, ib;
            turn_pair<G>(lp,j,t.rotary,t.interleaved,ia,ib);
            const float a = p[ia < t.dim? ia : 0], b = p[ib < t.dim? ib : 0];
            v.a[j] = ia < t.dim? a : 0.0f;
            v.b[j] = ib < t.dim? b : 0.0f;
        }
    } else {
        int o1, o2;
        turn_quads<MODE>(lp,t.rotary,o1,o2);
        float4 x = *reinterpret_cast<const float4*>(p + (o1 < t.dim? o1 : 0)), y = *reinterpret_cast<const float4*>(p + (o2 < t.dim? o2 : 0));
        const float4 zero = make_float4(0.f,0.f,0.f,0.f);
        if (o1 >= t.dim) x = zero;
        if (o2 >= t.dim) y = zero;
        if constexpr (MODE == kTurnAdjacent) v = {{x.x,x.z,y.x,y.z},{x.y,x.w,y.y,y.w}};
        else v = {{x.x,x.y,x.z,x.w},{y.x,y.y,y.z,y.w}};
    }
    return v;
}

template <int G, int MODE>
__device__ __forceinline__ void turn_store(const HeadTurn& t, float* p, int lp, const Pairs& v)
{
    if constexpr (MODE == kTurnScalar) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            int ia, ib;
            turn_pair<G>(lp,j,t.rotary,t.interleaved,ia,ib);
            if (ia < t.dim) p[ia] = v.a[j];
            if (ib < t.dim) p[ib] = v.b[j];
        }
    } else {
        int o1, o2;
        turn_quads<MODE>(lp,t.rotary,o1,o2);
        float4 x = make_float4(v.a[0],v.a[1],v.a[2],v.a[3]), y = make_float4(v.b[0],v.b[1],v.b[2],v.b[3]);
        if constexpr (MODE == kTurnAdjacent) {
            x = make_float4(v.a[0],v.b[0],v.a[1],v.b[1]);
            y = make_float4(v.a[2],v.b[2],v.a[3],v.b[3]);
        }
        if (o1 < t.dim) *reinterpret_cast<float4*>(p + o1) = x;
        if (o2 < t.dim) *reinterpret_cast<float4*>(p + o2) = y;
    }
}

// Cosines (a) and sines (b) of the lane's pairs in row `row`; 0 where a pair does not turn.
template <int G, int MODE>
__device__ __forceinline__ Pairs turn_tables(const HeadTurn& t, size_t row, int lp)
{
    Pairs v = {};
    const int half = t.rotary / 2;
    if (!half) return v;
    const float *c = t.cosine + row * half, *s = t.sine + row * half;
    if constexpr (MODE == kTurnScalar) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int p = lp + G * j;
            v.a[j] = c[p < half? p : 0];
            v.b[j] = s[p < half? p : 0];
        }
    } else {
        const int p = 4 * lp < half? 4 * lp : 0;
        const float4 x = *reinterpret_cast<const float4*>(c + p), y = *reinterpret_cast<const float4*>(s + p);
        v = {{x.x,x.y,x.z,x.w},{y.x,y.y,y.z,y.w}};
    }
    return v;
}

// Sum over the G lanes of a head (every lane of the wave active).
template <int G>
__device__ __forceinline__ double turn_sum(double v)
{
    static_assert(G == 16 || G == 64,"a row of lanes, or a wave");
    if constexpr (G == 64) return wave_sum_f64(v);
    v += dpp_f64<kDppXor1>(v);
    v += dpp_f64<kDppXor2>(v);
    v += dpp_f64<kDppHalfMirror>(v);
    v += dpp_f64<kDppMirror>(v);
    return v;
}

// Norm and rotation of a head's values in place; `w` its norm weight's values as
// turn_load gives them (1 where there is none), `cs` its row's tables.  Every lane
// of the wave must call it.
template <int G, int MODE>
__device__ __forceinline__ void turn_head(const HeadTurn& t, int lp, const Pairs& w, const Pairs& cs, Pairs& v)
{
    if (t.norm) {
        bool in_a[4], in_b[4];
        if constexpr (MODE == kTurnScalar) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                int ia, ib;
                turn_pair<G>(lp,j,t.rotary,t.interleaved,ia,ib);
                in_a[j] = ia < t.dim;
                in_b[j] = ib < t.dim;
            }
        } else {
            int o1, o2;
            turn_quads<MODE>(lp,t.rotary,o1,o2);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                in_a[j] = MODE == kTurnAdjacent? (j < 2? o1 : o2) < t.dim : o1 < t.dim;
                in_b[j] = MODE == kTurnAdjacent? in_a[j] : o2 < t.dim;
            }
        }
        double mean = 0.0;
        if (t.norm == kTurnNormLayer) {
            double s = 0.0;
#pragma unroll
            for (int j = 0; j < 4; j++) s += (double)v.a[j] + (double)v.b[j];  // (zeros past the head)
            mean = turn_sum<G>(s) / (double)t.dim;
        }
        double sq = 0.0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const double a = in_a[j]? (double)v.a[j] - mean : 0.0, b = in_b[j]? (double)v.b[j] - mean : 0.0;
            sq += a * a + b * b;
        }
        const float inverse = (float)(1.0 / sqrt(turn_sum<G>(sq) / (double)t.dim + (double)t.eps));
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float a = t.norm == kTurnNormLayer? (float)((double)v.a[j] - mean) : v.a[j];
            const float b = t.norm == kTurnNormLayer? (float)((double)v.b[j] - mean) : v.b[j];
            v.a[j] = __fmul_rn(__fmul_rn(a,inverse),w.a[j]);
            v.b[j] = __fmul_rn(__fmul_rn(b,inverse),w.b[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int p = MODE == kTurnScalar? lp + G * j : 4 * lp + j;
        if (p >= t.rotary / 2) continue;
        const float a = v.a[j], b = v.b[j], c = cs.a[j], s = cs.b[j];
        v.a[j] = __fsub_rn(__fmul_rn(a,c),__fmul_rn(b,s));
        v.b[j] = __fadd_rn(__fmul_rn(a,s),__fmul_rn(b,c));
    }
}

template <int G, int MODE>
__device__ __forceinline__ Pairs turn_weight(const HeadTurn& t, const float* w, int lp)
{
    if (t.norm && w) return turn_load<G,MODE>(t,w,lp);
    return {{1.f,1.f,1.f,1.f},{1.f,1.f,1.f,1.f}};
}

// Heads of `x` ([rows] of `heads` heads, `ld` values apart) to `out` [rows][heads *
// dim], the workgroup's G-lane groups taking items item, item + 1, .. of `per`
// consecutive heads of a row each (`per` at most kTurnHeads): their row's tables are
// read once.  `plain`: copied as they are.
constexpr int kTurnHeads = 4;
template <int G, int MODE>
__device__ __forceinline__ void turn_rows(const HeadTurn& t, const float* x, size_t ld, float* out, size_t rows, int heads, int per, const float* weight,
                                          bool plain, size_t item)
{
    const int lp = (int)(threadIdx.x % G), parts = (heads + per - 1) / per;
    const size_t row = item / (unsigned)parts, last = rows - 1;
    const bool live = row < rows;
    const size_t r = live? row : last;
    const int h0 = (int)(item % (unsigned)parts) * per;
    const float* src = x + r * ld;
    Pairs v[kTurnHeads];
#pragma unroll
    for (int j = 0; j < kTurnHeads; j++)
        if (j < per) v[j] = turn_load<G,MODE>(t,src + (size_t)(h0 + j < heads? h0 + j : heads - 1) * t.dim,lp);
    Pairs cs = {}, w = {};
    if (!plain) {
        cs = turn_tables<G,MODE>(t,r,lp);
        w = turn_weight<G,MODE>(t,weight,lp);
    }
#pragma unroll
    for (int j = 0; j < kTurnHeads; j++) {
        if (j >= per) continue;  // (the same in every lane)
        if (!plain) turn_head<G,MODE>(t,lp,w,cs,v[j]);
        if (live && h0 + j < heads) turn_store<G,MODE>(t,out + (row * heads + h0 + j) * t.dim,lp,v[j]);
    }
}

}  // namespace pixhip
