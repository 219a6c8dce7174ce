// Low-rank adapters of the requests of a batch beside the linear layer that they
// share (gfx950): for each row c that an adapter a serves
//   y[c] = base[c] + scale * U_a (D_a x[c])
// with D_a [rank][inner] and U_a [rows][rank] of 16 or 32 bits, all else in fp32.
//
// Products.  A value of 24 bits is the exact sum of three bf16 values, an F16 weight of two,
// a BF16 weight is one itself.  Each product of planes p and q with p + q <= 2 is one
// v_mfma_f32_16x16x32_bf16 with fp32 sums: 3, 5 or 6 instructions per 16 x 16 x 32 products.
// Left out of a BF16 weight's product is nothing, so that the rows' planes are cut off one
// after the other.  Of an F16 weight's it is the rows' third plane times the weight's second.
// A second plane is below 2^-7 of the leading bit's value where the first is cut off, at most
// 2^-8 where that is rounded to nearest; a third one is at most 2^-16 where the second alone
// is rounded, 2^-17 where both are.  So D's first plane and the rows' second are rounded, and
// of U's product the sums' first and second: 2^-24 of a product, of either sign.  (The sums
// are fewer than U's values: 64 rows of 9 adapters 3584 -> 18944, the ranges packed by each
// call, 19.4 us and, with U's first plane rounded instead, 20.1.)  Of an F32 weight's it is
// second times third, twice, and third times third: all are rounded, 2^-24 + 2^-34.  (All cut
// off, up to 1.8 and 3.9 times 2^-23, always toward zero.)  A row that holds NaN or an
// infinity gives NaN (an infinity's second or third plane is Inf - Inf).
//
// Layouts, as the matrix instruction's lanes take them, 16 bytes a lane (so a wave
// reads 1 KB in a row):
//   down  [inner / 32][rank / 16][plane][64 lanes][8]: lane l holds rank l % 16 and, of
//         the 32 inner values, 4 (l / 16) .. + 3 and 16 + 4 (l / 16) .. + 3
//   up    [rows / 32][rank / 32][half][64 lanes][8]: lane l holds row 16 half + l % 16 of
//         the 32, ranks 8 (l / 16) .. + 7
// padded with zeros; down as planes, up as the values themselves (32 bits: four, then the
// other four, of 64 lanes), whose planes take a wave few instructions for the rows that it
// multiplies by them (64 rows of 9 adapters, 3584 -> 18944, the ranges packed beforehand:
// F16 15.9 us, as planes 19.0, F32 19.7 and 22.3).
//
// Rows of x, base and y are read and written as eight rows of 128 bytes per instruction
// (pair_rows): as sixteen of 64, which is how the matrix instruction's lanes have them, a
// copy of 4608 rows of 10240 takes 93 us instead of 74.  Through buffer descriptors, whose
// offsets take no instructions per step and which read any size and alignment as it is
// (3840 -> 10240 with rank 64, 4608 rows: 117 us, with pointers and clamps 123; 3839 ->
// 10239: 144 and, value by value, 206, its rows' lines being written in two parts).
//
// Bound by HBM where rows are many: 3840 -> 10240 with rank 64 and 4608 rows takes 109 us
// for 450 MB, 4.1 TB/s, 24 us of them x in the first launch, 85 base and y in the second; by
// the start of two launches, or the loads of D in one, where they are few (1 row of 4096:
// 7 and 8 us).  Rounded planes take nothing that shows beside it, but for 16 rows of F32 with
// rank 128, 4096 -> 4096, 12.3 -> 12.8 us.
#include <algorithm>

#include "pixhip_device.h"
#include "pixhip_internal.h"

namespace pixhip {

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kTokens = 16;  // rows of a tile
constexpr int kWaves = 8, kDownWaves = 4;

// Two values rounded to bf16 (nearest even), `a` in the lower half.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b)
{
    typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
    const v2bf h = {(__bf16)a,(__bf16)b};
    return __builtin_bit_cast(uint32_t,h);
}

// The N leading bf16 planes of 8 values, the leading one first: those from the FROM-th on
// rounded to nearest, the ones before cut off; the last holds what is left.  BIG:
// values may round to more than the largest bf16; their first plane is that one (16 bits are
// left, which the other two hold), an infinity's too, whose second plane is then infinite and
// whose third is NaN.
template <int N, int FROM, bool BIG = true>
__device__ __forceinline__ void split_planes(const float (&x)[8], v8bf (&p)[N])
{
    const float most = __uint_as_float(0x7f7f0000u);
    v4u w[N];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int q = 0; q < N; q++) {
            if (q < FROM || q == N - 1) {
                w[q][i] = __builtin_amdgcn_perm(__float_as_uint(b),__float_as_uint(a),0x07060302u);  // both upper halves
                if (q == N - 1) continue;
                a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
                b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
            } else {
                const bool limit = BIG && q == 0;
                w[q][i] = pack_bf16(limit? __builtin_amdgcn_fmed3f(a,-most,most) : a,limit? __builtin_amdgcn_fmed3f(b,-most,most) : b);
                if (q == N - 1) continue;
                // (as bytes: where the compiler sees a half of a pair it converts that value again)
                a -= __uint_as_float(__builtin_amdgcn_perm(0u,w[q][i],0x01000c0cu));
                b -= __uint_as_float(__builtin_amdgcn_perm(0u,w[q][i],0x03020c0cu));
            }
        }
    }
#pragma unroll
    for (int q = 0; q < N; q++) p[q] = __builtin_bit_cast(v8bf,w[q]);
}

__device__ __forceinline__ float source_value(const void* src, uint32_t type, size_t i)
{
    if (type == PIX_F32) return static_cast<const float*>(src)[i];
    const uint16_t u = static_cast<const uint16_t*>(src)[i];
    return type == PIX_BF16? __uint_as_float((uint32_t)u << 16) : half_bits_to_float(u);
}

// One thread per 8 values of each layout: down's pieces first, then up's.
__global__ __launch_bounds__(256) void adapter_form_kernel(const void* down, const void* up, uint32_t type, int rank, size_t inner, size_t rows, int planes,
                                                           uint16_t* down_out, uint16_t* up_out, size_t down_pieces, size_t up_pieces)
{
    const size_t e = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= down_pieces + up_pieces) return;
    const int lane = (int)(e % 64), lo = lane % 16, hi = lane / 16;
    float x[8];
    if (e < down_pieces) {
        const int tiles = (rank + 15) / 16;
        const size_t g = e / 64, step = g / (unsigned)tiles;
        const int t = (int)(g % (unsigned)tiles), r = 16 * t + lo;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const size_t k = 32 * step + 16 * (j / 4) + 4 * hi + j % 4;
            x[j] = r < rank && k < inner? source_value(down,type,(size_t)r * inner + k) : 0.0f;
        }
        v8bf p[3];
        if (type == PIX_F32) split_planes<3,0>(x,p);
        else split_planes<3,0,false>(x,p);  // (one or two planes are all of it)
        for (int q = 0; q < planes; q++) *reinterpret_cast<v8bf*>(down_out + (g * planes + q) * 512 + lane * 8) = p[q];
    } else {
        const int steps = (rank + 31) / 32;
        const size_t g = (e - down_pieces) / 64, T = g / (unsigned)(2 * steps);
        const int s = (int)(g % (unsigned)(2 * steps)) / 2, half = (int)(g % 2);
        const size_t row = 32 * T + 16 * half + lo;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int r = 32 * s + 8 * hi + j;
            x[j] = row < rows && r < rank? source_value(up,type,row * rank + r) : 0.0f;
        }
        if (type == PIX_F32) {
            float* to = reinterpret_cast<float*>(up_out) + g * 512 + lane * 4;
            *reinterpret_cast<v4f*>(to) = v4f{x[0],x[1],x[2],x[3]};
            *reinterpret_cast<v4f*>(to + 256) = v4f{x[4],x[5],x[6],x[7]};
            return;
        }
        v4u w;
        for (int j = 0; j < 4; j++) {  // (exact: they were 16 bits)
            const uint32_t lo = type == PIX_BF16? __float_as_uint(x[2 * j]) >> 16 : __builtin_bit_cast(uint16_t,(_Float16)x[2 * j]);
            const uint32_t hi = type == PIX_BF16? __float_as_uint(x[2 * j + 1]) >> 16 : __builtin_bit_cast(uint16_t,(_Float16)x[2 * j + 1]);
            w[j] = lo | hi << 16;
        }
        *reinterpret_cast<v4u*>(up_out + g * 512 + lane * 8) = w;
    }
}

// Of 16 rows and 32 values: the matrix instruction has in lane l row l % 16, values
// 4 (l / 16) .. + 3 (u) and 16 + those (v); memory instructions take in lane l the values
// 4 (l / 16) + 16 (l % 16 / 8) .. + 3 of row l % 8 (u) and of row 8 + l % 8 (v).  This
// turns each into the other.
__device__ __forceinline__ void pair_rows(v4f& u, v4f& v)
{
    const bool low = !(threadIdx.x & 8);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float other = xor_lane<8>(low? v[j] : u[j]);
        u[j] = low? u[j] : other;
        v[j] = low? other : v[j];
    }
}

// The first value among 32 of those that a lane reads or writes.
__device__ __forceinline__ int lane_value()
{
    return 4 * ((int)(threadIdx.x & 63) / 16) + 16 * ((int)(threadIdx.x & 15) / 8);
}

// The planes of 32 values of 16 rows, of which `left` are the rows', for weights of NP planes.
template <int NP>
__device__ __forceinline__ void split_rows(v4f u, v4f v, int left, v8bf (&p)[3])
{
    if (left < 32)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            u[j] = lane_value() + j < left? u[j] : 0.0f;
            v[j] = lane_value() + j < left? v[j] : 0.0f;
        }
    pair_rows(u,v);
    const float x[8] = {u[0],u[1],u[2],u[3],v[0],v[1],v[2],v[3]};
    split_planes<3,3 - NP>(x,p);
}

// acc += the products of planes p of x and q of w with p + q <= 2, the smallest first.
template <int NP>
__device__ __forceinline__ v4f multiply(const v8bf (&w)[NP], const v8bf (&x)[3], v4f acc)
{
#pragma unroll
    for (int sum = 2; sum >= 0; sum--)
#pragma unroll
        for (int q = NP - 1; q >= 0; q--) {
            if (sum - q < 0) continue;
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[q],x[sum - q],acc,0,0,0);
        }
    return acc;
}

// The segment of tile `tile`: the last one that begins at or before it (one load per lane).
__device__ __forceinline__ int find_segment(const AdapterCall& a, unsigned tile, bool groups)
{
    if (a.segments == 1) return 0;
    const int lane = (int)(threadIdx.x & 63);
    const AdapterSegment& s = a.segment[lane < a.segments? lane : 0];
    const unsigned begins = groups? s.first_group : s.first_tile;
    return __builtin_amdgcn_readfirstlane(__builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < a.segments && begins <= tile)) - 1);
}

// Rows of x, base or y from the batch's or, listed, the list's row `from` of a segment on,
// `count` at most, as one buffer: four values are one load or store at any multiple of 4
// bytes, and past the last row's end loads give zeros.
__device__ __forceinline__ RowBuffer batch_buffer(const AdapterCall& a, const AdapterSegment& seg, const float* p, unsigned from, unsigned count,
                                                  size_t ld, int K)
{
    const unsigned left = seg.rows - from, n = a.listed? a.columns : left < count? left : count;
    return RowBuffer(p + (a.listed? 0 : (size_t)(seg.first + from) * ld),(uint32_t)(((n - 1) * ld + K) * sizeof(float)));
}

// A tile's two rows that a lane reads or writes: where the first of its values lies in
// the buffer of the rows from `from` on.  The tile begins at the segment's row `first`
// (past its last row that one again).
struct LaneRows {
    uint32_t at[2];
    bool live[2];
};
__device__ __forceinline__ LaneRows batch_rows(const AdapterCall& a, const AdapterSegment& seg, unsigned from, unsigned first, size_t ld)
{
    LaneRows r;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const unsigned at = first + 8 * i + (threadIdx.x & 7), row = at < seg.rows? at : seg.rows - 1;
        r.live[i] = at < seg.rows;
        r.at[i] = ((a.listed? a.list[seg.first + row] : row - from) * (uint32_t)ld + (uint32_t)lane_value()) * (uint32_t)sizeof(float);
    }
    return r;
}

// acc[n][t] += D's ranks 16 (t0 + t) .. + 15 times tile n's rows over the steps first,
// first + stride, .. below `end`, U of them loaded at a time; in lane l of row l % 16,
// ranks 4 (l / 16) .. + 3.
template <int NP, int RC, int TN, int U>
__device__ __forceinline__ void multiply_down(const AdapterCall& a, const AdapterSegment& seg, const RowBuffer& in, const LaneRows (&rows)[TN], int t0,
                                              int nt, int tiles, int first, int end, int stride, v4f (&acc)[TN][RC])
{
    const int lane = (int)(threadIdx.x & 63);
    for (int s0 = first; s0 < end; s0 += stride * U) {
        v4f x[U][TN][2];
        v8bf w[U][RC][NP];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int s = s0 + stride * u, sc = s < end? s : end - 1;  // (a step too many: loads of the last one)
#pragma unroll
            for (int n = 0; n < TN; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) x[u][n][i] = in.load<v4f>(rows[n].at[i],128 * (uint32_t)sc);
            const uint16_t* d = seg.down + ((size_t)sc * tiles + t0) * (NP * 512) + lane * 8;
#pragma unroll
            for (int t = 0; t < RC; t++)
                if (t < nt)
#pragma unroll
                    for (int q = 0; q < NP; q++) w[u][t][q] = *reinterpret_cast<const v8bf*>(d + (t * NP + q) * 512);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (s0 + stride * u >= end) continue;  // whole wave
#pragma unroll
            for (int n = 0; n < TN; n++) {
                v8bf p[3];
                split_rows<NP>(x[u][n][0],x[u][n][1],a.inner - 32 * (s0 + stride * u),p);
#pragma unroll
                for (int t = 0; t < RC; t++)
                    if (t < nt) acc[n][t] = multiply<NP>(w[u][t],p,acc[n][t]);
            }
        }
    }
}

// The same for more than 64 ranks, which take a wave many steps of much work each: the
// rows are loaded L steps ahead (past the end the last step again), D's tiles G at a
// time, one group ahead.  RC tiles are multiplied, of which those past `tiles` repeat
// the last one, into sums that nobody reads.
template <int NP, int RC, int TN, int L>
__device__ __forceinline__ void multiply_down_wide(const AdapterCall& a, const AdapterSegment& seg, const RowBuffer& in, const LaneRows (&rows)[TN],
                                                   int tiles, int first, int end, int stride, v4f (&acc)[TN][RC])
{
    constexpr int G = NP == 1? 4 : NP == 2? 2 : 1, kTurns = RC / G;
    const int lane = (int)(threadIdx.x & 63);
    if (first >= end) return;
    v4f x[L][TN][2];
    auto load_x = [&](int s, v4f (&to)[TN][2]) {
        const int sc = s < end? s : end - 1;
#pragma unroll
        for (int n = 0; n < TN; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) to[n][i] = in.load<v4f>(rows[n].at[i],128 * (uint32_t)sc);
    };
    v8bf w[2][G][NP];
    auto load_group = [&](int s, int g, v8bf (&to)[G][NP]) {
        const uint16_t* d = seg.down + ((size_t)(s < end? s : end - 1) * tiles) * (NP * 512) + lane * 8;
#pragma unroll
        for (int t = 0; t < G; t++)
#pragma unroll
            for (int q = 0; q < NP; q++) to[t][q] = *reinterpret_cast<const v8bf*>(d + ((G * g + t < tiles? G * g + t : tiles - 1) * NP + q) * 512);
    };
    load_group(first,0,w[0]);
#pragma unroll
    for (int l = 0; l < L; l++) load_x(first + l * stride,x[l]);
    // (unrolled so that the group after next, and the rows after L, keep their registers)
    constexpr int kUnroll = kTurns % 2 && L % 2? 2 * L : L;
    for (int s0 = first; s0 < end; s0 += stride * kUnroll) {
#pragma unroll
        for (int l = 0; l < kUnroll; l++) {
            const int s = s0 + l * stride;
            if (s >= end) break;  // whole wave
            v8bf p[TN][3];
#pragma unroll
            for (int n = 0; n < TN; n++) split_rows<NP>(x[l % L][n][0],x[l % L][n][1],a.inner - 32 * s,p[n]);
            load_x(s + L * stride,x[l % L]);
#pragma unroll
            for (int g = 0; g < kTurns; g++) {
                const int at = (l * kTurns + g) % 2;
                load_group(g + 1 < kTurns? s : s + stride,(g + 1) % kTurns,w[1 - at]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int n = 0; n < TN; n++)
#pragma unroll
                    for (int t = 0; t < G; t++) acc[n][G * g + t] = multiply<NP>(w[at][t],p[n],acc[n][G * g + t]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
}

// Four of a row's sums (ranks `to` .. + 3 of row n of a tile), scaled, as the planes
// that multiply_up reads: parts [rank / 32][plane][64 lanes][8].
template <int NP>
__device__ __forceinline__ void store_parts(uint16_t* parts, int n, int to, v4f sum, float scale)
{
    const float v[8] = {sum[0] * scale,sum[1] * scale,sum[2] * scale,sum[3] * scale,0.f,0.f,0.f,0.f};
    v8bf p[3];
    split_planes<3,NP == 1? 2 : 0>(v,p);
    uint16_t* o = parts + ((to / 32) * 3 * 64 + 16 * (to % 32 / 8) + n) * 8 + to % 8;
#pragma unroll
    for (int q = 0; q < 3; q++) *reinterpret_cast<uint2*>(o + q * 512) = make_uint2(__builtin_bit_cast(v4u,p[q])[0],__builtin_bit_cast(v4u,p[q])[1]);
}

// A lane's 8 values of U, and their planes.
template <int NP>
struct UpWeights {
    v4u raw[NP == 3? 2 : 1];
    __device__ __forceinline__ void planes(v8bf (&p)[NP]) const
    {
        if constexpr (NP == 1) {
            p[0] = __builtin_bit_cast(v8bf,raw[0]);
        } else {
            typedef _Float16 v8h __attribute__((ext_vector_type(8)));
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                if constexpr (NP == 2) x[i] = (float)__builtin_bit_cast(v8h,raw[0])[i];
                else x[i] = __uint_as_float(raw[i / 4][i % 4]);
            }
            split_planes<NP,3 - NP>(x,p);
        }
    }
};

// What a wave reads ahead for one turn of 32 outputs of TN tiles of rows: base, and U's
// first step where there are registers for the next one's while it is multiplied.
template <int NP, int TN>
struct UpTurn {
    static constexpr bool kAhead = NP < 3 || TN <= 2;
    v4f base[TN][2];
    UpWeights<NP> w[2];
};

template <int NP>
__device__ __forceinline__ void load_up(const AdapterSegment& seg, int steps, int T, int s, UpWeights<NP> (&w)[2])
{
    constexpr int kPieces = NP == 3? 2 : 1;
    const uint16_t* u = seg.up + ((size_t)T * steps + s) * (2 * kPieces * 512) + (threadIdx.x & 63) * 8;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int j = 0; j < kPieces; j++) w[h].raw[j] = *reinterpret_cast<const v4u*>(u + (h * kPieces + j) * 512);
}

template <int NP, int TN>
__device__ __forceinline__ void load_turn(const AdapterCall& a, const AdapterSegment& seg, const RowBuffer& base, const LaneRows (&rows)[TN], int nt, int T,
                                          UpTurn<NP,TN>& t)
{
    const int steps = (seg.rank + 31) / 32;
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
            t.base[n][i] = v4f{0.f,0.f,0.f,0.f};
            if (a.base && n < nt) t.base[n][i] = base.load<v4f>(rows[n].at[i],128 * (uint32_t)T);
        }
    if (UpTurn<NP,TN>::kAhead && steps) load_up<NP>(seg,steps,T,0,t.w);
}

// One turn: base plus U times the rows' parts (tile n's at parts + n * part_stride).
template <int NP, int TN>
__device__ __forceinline__ void multiply_up(const AdapterCall& a, const AdapterSegment& seg, const RowBuffer& y, const LaneRows (&rows)[TN], int nt,
                                            const uint16_t* parts, int part_stride, int T, UpTurn<NP,TN>& t)
{
    const int lane = (int)(threadIdx.x & 63), steps = (seg.rank + 31) / 32;
    v4f acc[TN][2];
#pragma unroll
    for (int n = 0; n < TN; n++) acc[n][0] = acc[n][1] = v4f{0.f,0.f,0.f,0.f};
    for (int s = 0; s < steps; s++) {
        if constexpr (!UpTurn<NP,TN>::kAhead) load_up<NP>(seg,steps,T,s,t.w);
        v8bf w[2][NP];
#pragma unroll
        for (int h = 0; h < 2; h++) t.w[h].planes(w[h]);
        if (UpTurn<NP,TN>::kAhead && s + 1 < steps) load_up<NP>(seg,steps,T,s + 1,t.w);
#pragma unroll
        for (int n = 0; n < TN; n++) {
            if (n >= nt) continue;
            v8bf p[3];
#pragma unroll
            for (int q = 0; q < 3; q++) p[q] = *reinterpret_cast<const v8bf*>(parts + n * part_stride + ((s * 3 + q) * 64 + lane) * 8);
#pragma unroll
            for (int h = 0; h < 2; h++) acc[n][h] = multiply<NP>(w[h],p,acc[n][h]);
        }
    }
#pragma unroll
    for (int n = 0; n < TN; n++) {
        pair_rows(acc[n][0],acc[n][1]);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (!rows[n].live[i]) continue;
            const v4f v = steps? t.base[n][i] + acc[n][i] : t.base[n][i];
            const int left = a.rows - 32 * T - lane_value();
            if (left >= 4) y.store(rows[n].at[i],v,128 * (uint32_t)T,a.past);
            else
#pragma unroll
                for (int j = 0; j < 3; j++)
                    if (j < left) y.store(rows[n].at[i] + 4 * j,v[j],128 * (uint32_t)T);
        }
    }
}

// One workgroup per (tile of 16 rows, slice of the outputs): D x over the whole inner
// size, shared by the waves in steps of 32, their sums joined in LDS; then U times
// that for the slice's rows of U, 32 to a wave at a time.  RC: 16-rank tiles that the
// inner loop takes at once; more ranks take more turns over x.  Needs no workspace, and
// takes D x once per slice: for captured calls without one, short inner sizes and single
// rows.
constexpr int kFewWaves = 16;
template <int NP, int RC>
__global__ __launch_bounds__(64 * kFewWaves) void adapters_kernel(AdapterCall a)
{
    constexpr int LD = 16 * RC + 4;
    constexpr int U = NP * RC <= 2? 4 : NP * RC <= 4? 2 : 1;
    __shared__ __attribute__((aligned(16))) float red[kFewWaves * kTokens * LD];
    extern __shared__ __attribute__((aligned(16))) uint16_t parts[];
    const int tid = (int)threadIdx.x, lane = tid & 63, lo = lane % 16, hi = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned tile = blockIdx.x / (unsigned)a.slices, slice = blockIdx.x % (unsigned)a.slices;
    const AdapterSegment& seg = a.segment[find_segment(a,tile,false)];
    const unsigned first = (tile - seg.first_tile) * kTokens;
    const LaneRows in[1] = {batch_rows(a,seg,first,first,a.ldx)}, rows[1] = {batch_rows(a,seg,first,first,a.ldy)};
    const RowBuffer x = batch_buffer(a,seg,a.x,first,kTokens,a.ldx,a.inner), base = batch_buffer(a,seg,a.base,first,kTokens,a.ldy,a.rows);
    const RowBuffer y = batch_buffer(a,seg,a.y,first,kTokens,a.ldy,a.rows);
    const int tiles = (seg.rank + 15) / 16, ks = (a.inner + 31) / 32, nT = (a.rows + 31) / 32;
    const int T1 = (int)((size_t)(slice + 1) * nT / (unsigned)a.slices);
    int T = (int)((size_t)slice * nT / (unsigned)a.slices) + wave;
    UpTurn<NP,1> turn;
    if (T < T1) load_turn<NP,1>(a,seg,base,rows,1,T,turn);
    if (seg.rank) {
        for (int t0 = 0; t0 < tiles; t0 += RC) {
            const int nt = tiles - t0 < RC? tiles - t0 : RC;
            v4f acc[1][RC];
#pragma unroll
            for (int t = 0; t < RC; t++) acc[0][t] = v4f{0.f,0.f,0.f,0.f};
            // (as many steps at a time as a wave has)
            if (U >= 4 && ks > 2 * kFewWaves) multiply_down<NP,RC,1,U>(a,seg,x,in,t0,nt,tiles,wave,ks,kFewWaves,acc);
            else if (U >= 2 && ks > kFewWaves) multiply_down<NP,RC,1,2>(a,seg,x,in,t0,nt,tiles,wave,ks,kFewWaves,acc);
            else multiply_down<NP,RC,1,1>(a,seg,x,in,t0,nt,tiles,wave,ks,kFewWaves,acc);
#pragma unroll
            for (int t = 0; t < RC; t++)
                if (t < nt) *reinterpret_cast<v4f*>(red + (wave * kTokens + lo) * LD + 16 * t + 4 * hi) = acc[0][t];
            __syncthreads();
            // the waves' sums in order; ranks past the last tile up to a multiple of 32 are zeros
            const int ranks = t0 + RC >= tiles? (tiles + 1) / 2 * 32 - 16 * t0 : 16 * RC;
            for (int e = tid; e < kTokens * ranks / 4; e += 64 * kFewWaves) {
                const int n = e % kTokens, r = 4 * (e / kTokens);
                v4f sum = {0.f,0.f,0.f,0.f};
                if (r < 16 * nt) {
                    sum = *reinterpret_cast<const v4f*>(red + n * LD + r);
#pragma unroll
                    for (int w = 1; w < kFewWaves; w++) sum += *reinterpret_cast<const v4f*>(red + (w * kTokens + n) * LD + r);
                }
                store_parts<NP>(parts,n,16 * t0 + r,sum,seg.scale);
            }
            __syncthreads();
        }
    }
    while (T < T1) {
        multiply_up<NP,1>(a,seg,y,rows,1,parts,0,T,turn);
        T += kFewWaves;
        if (T < T1) load_turn<NP,1>(a,seg,base,rows,1,T,turn);
    }
}

// The same in two launches, for calls whose D x is worth being taken once.  First: one
// workgroup per (TN tiles of 16 rows, part of the inner size), its sums to work
// [part][tile][16 rows][ranks].
template <int NP, int RC, int TN>
__global__ __launch_bounds__(64 * kDownWaves,RC > 4? 2 : 4) void adapters_down_kernel(AdapterCall a)
{
    constexpr int R4 = RC < 4? RC : 4, LD = 16 * R4 + 4;  // rank tiles that are joined at a time
    constexpr int U = NP * RC * TN <= 2 && TN == 1? 4 : NP * RC * TN <= 4? 2 : 1, L = RC * TN > 16? 2 : 4;
    __shared__ __attribute__((aligned(16))) float red[2][kDownWaves * kTokens * LD];
    const int tid = (int)threadIdx.x, lane = tid & 63, lo = lane % 16, hi = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned tile = blockIdx.x / (unsigned)a.parts * TN, part = blockIdx.x % (unsigned)a.parts;
    // (segments begin at multiples of TN tiles)
    const AdapterSegment& seg = a.segment[find_segment(a,tile,false)];
    if (!seg.rank) return;
    const unsigned first = (tile - seg.first_tile) * kTokens;
    LaneRows rows[TN];
#pragma unroll
    for (int n = 0; n < TN; n++) rows[n] = batch_rows(a,seg,first,first + n * kTokens,a.ldx);
    const RowBuffer x = batch_buffer(a,seg,a.x,first,TN * kTokens,a.ldx,a.inner);
    const int tiles = (seg.rank + 15) / 16, ks = (a.inner + 31) / 32;
    const int s0 = (int)((size_t)part * ks / (unsigned)a.parts), s1 = (int)((size_t)(part + 1) * ks / (unsigned)a.parts);
    v4f acc[TN][RC];  // (all of the ranks)
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
        for (int t = 0; t < RC; t++) acc[n][t] = v4f{0.f,0.f,0.f,0.f};
    if constexpr (RC > 4) multiply_down_wide<NP,RC,TN,L>(a,seg,x,rows,tiles,s0 + wave,s1,kDownWaves,acc);
    else multiply_down<NP,RC,TN,U>(a,seg,x,rows,0,tiles,tiles,s0 + wave,s1,kDownWaves,acc);
    int turn = 0;
#pragma unroll
    for (int n = 0; n < TN; n++)
#pragma unroll
        for (int t0 = 0; t0 < RC; t0 += R4) {
            if (t0 >= tiles) continue;  // (the whole workgroup)
            float* r = red[turn];
            turn ^= 1;
#pragma unroll
            for (int t = 0; t < R4; t++)
                if (t0 + t < tiles) *reinterpret_cast<v4f*>(r + (wave * kTokens + lo) * LD + 16 * t + 4 * hi) = acc[n][t0 + t];
            __syncthreads();
            float* out = a.work + (((size_t)part * a.tiles + tile + n) * kTokens) * a.work_ld + 16 * t0;
            const int quads = 4 * (tiles - t0 < R4? tiles - t0 : R4);
            const int left = (int)seg.rows - (int)first - n * kTokens, live = left < kTokens? left : kTokens;
            for (int e = tid; e < live * quads; e += 64 * kDownWaves) {
                const int q = 4 * (e % quads), m = e / quads;
                v4f sum = *reinterpret_cast<const v4f*>(r + m * LD + q);
#pragma unroll
                for (int w = 1; w < kDownWaves; w++) sum += *reinterpret_cast<const v4f*>(r + (w * kTokens + m) * LD + q);
                *reinterpret_cast<v4f*>(out + m * a.work_ld + q) = sum;
            }
        }
}

// Second: one workgroup per (kGroup tiles of 16 rows, slice of the outputs); each wave
// multiplies what it has read of U by all of the rows.
template <int NP, int kGroup>
__global__ __launch_bounds__(64 * kWaves,4) void adapters_up_kernel(AdapterCall a)
{
    extern __shared__ __attribute__((aligned(16))) uint16_t parts[];
    const int tid = (int)threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // A group's slices beside one another on an XCD, whose L2 then has its rows' sums (1024
    // rows to 4096 outputs with rank 64 25.0 -> 22.4 us, 4608 to 10240 117.5 -> 114.6); few
    // groups, of which one may have many more ranks, over all of them (10 of ranks 8 to 64,
    // F32, 18944 outputs: 19.8 us or 20.3).
    const unsigned whole = gridDim.x / 8, rest = gridDim.x % 8, xcd = blockIdx.x % 8;
    const bool near = gridDim.x >= 16 * (unsigned)a.slices;
    const unsigned at = near? xcd * whole + (xcd < rest? xcd : rest) + blockIdx.x / 8 : blockIdx.x;
    const unsigned group = at / (unsigned)a.slices, slice = at % (unsigned)a.slices;
    const AdapterSegment& seg = a.segment[find_segment(a,group,true)];
    const unsigned first = (group - seg.first_group) * kGroup * kTokens;  // of the segment's rows
    const int steps = (seg.rank + 31) / 32, ranks = (seg.rank + 15) / 16 * 16, stride = steps * 3 * 512;
    LaneRows rows[kGroup];
#pragma unroll
    for (int n = 0; n < kGroup; n++) rows[n] = batch_rows(a,seg,first,first + n * kTokens,a.ldy);
    const RowBuffer base = batch_buffer(a,seg,a.base,first,kGroup * kTokens,a.ldy,a.rows), y = batch_buffer(a,seg,a.y,first,kGroup * kTokens,a.ldy,a.rows);
    const int live = (int)(seg.rows - first < kGroup * kTokens? seg.rows - first : kGroup * kTokens), nt = (live + kTokens - 1) / kTokens;
    const int nT = (a.rows + 31) / 32, T1 = (int)((size_t)(slice + 1) * nT / (unsigned)a.slices);
    int T = (int)((size_t)slice * nT / (unsigned)a.slices) + wave;
    UpTurn<NP,kGroup> t;
    if (T < T1) load_turn<NP,kGroup>(a,seg,base,rows,nt,T,t);
    // the inner parts' sums in order, eight loads at a time (rows past the last: what lies
    // there, in columns that nobody reads)
    const float* from = a.work + ((size_t)seg.first_tile * kTokens + first) * a.work_ld;
    const size_t next = (size_t)a.tiles * kTokens * a.work_ld;
    for (int e = tid; e < live * 8 * steps; e += 64 * kWaves) {
        const int r = 4 * (e % (8 * steps)), m = e / (8 * steps);
        v4f sum = {0.f,0.f,0.f,0.f};
        if (r < ranks)
            for (int k0 = 0; k0 < a.parts; k0 += 8) {
                v4f v[8];
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = *reinterpret_cast<const v4f*>(from + (k0 + k < a.parts? k0 + k : k0) * next + (size_t)m * a.work_ld + r);
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (k0 + k < a.parts) sum += v[k];
            }
        store_parts<NP>(parts + m / kTokens * stride,m % kTokens,r,sum,seg.scale);
    }
    __syncthreads();
    while (T < T1) {
        multiply_up<NP,kGroup>(a,seg,y,rows,nt,parts,stride,T,t);
        T += kWaves;
        if (T < T1) load_turn<NP,kGroup>(a,seg,base,rows,nt,T,t);
    }
}

template <int NP>
hipError_t launch_one(const AdapterCall& a, int rank, unsigned grid, hipStream_t s)
{
    const size_t lds = (size_t)((rank + 31) / 32) * 3 * 1024;
    const dim3 block(64 * kFewWaves);
    if (rank <= 16) adapters_kernel<NP,1><<<dim3(grid),block,lds,s>>>(a);
    else if (rank <= 32) adapters_kernel<NP,2><<<dim3(grid),block,lds,s>>>(a);
    else adapters_kernel<NP,4><<<dim3(grid),block,lds,s>>>(a);
    return hipGetLastError();
}

template <int NP>
hipError_t launch_two(const AdapterCall& a, int rank, unsigned grid, int down_tiles, hipStream_t s)
{
    const size_t lds = (size_t)((rank + 31) / 32) * 3 * 1024;
    const dim3 block(64 * kWaves), first(64 * kDownWaves), down(a.tiles / (unsigned)down_tiles * (unsigned)a.parts);
    if (down_tiles == 1) {
        if (rank <= 16) adapters_down_kernel<NP,1,1><<<down,first,0,s>>>(a);
        else if (rank <= 32) adapters_down_kernel<NP,2,1><<<down,first,0,s>>>(a);
        else if (rank <= 64) adapters_down_kernel<NP,4,1><<<down,first,0,s>>>(a);
        else if (rank <= 128) adapters_down_kernel<NP,8,1><<<down,first,0,s>>>(a);
        else adapters_down_kernel<NP,16,1><<<down,first,0,s>>>(a);
    } else if (rank <= 16) adapters_down_kernel<NP,1,2><<<down,first,0,s>>>(a);
    else if (rank <= 32) adapters_down_kernel<NP,2,2><<<down,first,0,s>>>(a);
    else if (rank <= 64) adapters_down_kernel<NP,4,2><<<down,first,0,s>>>(a);
    else if (rank <= 128) adapters_down_kernel<NP,8,2><<<down,first,0,s>>>(a);
    else adapters_down_kernel<NP,16,2><<<down,first,0,s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.group == 4) adapters_up_kernel<NP,4><<<dim3(grid),block,4 * lds,s>>>(a);
    else adapters_up_kernel<NP,2><<<dim3(grid),block,2 * lds,s>>>(a);
    return hipGetLastError();
}

template <int NP>
hipError_t launch_planes(const AdapterCall& a, int rank, unsigned grid, int down_tiles, hipStream_t s)
{
    return a.work? launch_two<NP>(a,rank,grid,down_tiles,s) : launch_one<NP>(a,rank,grid,s);
}

// Pieces to cut `work` units of each of `tiles` tiles into, at most `most`: the fewest
// turns of a wave in all, where `held` workgroups run at once and a workgroup's start and
// end cost as much as `start` turns.
size_t cut_evenly(size_t tiles, size_t work, size_t most, size_t waves, size_t held, size_t start)
{
    size_t best = 1, least = SIZE_MAX;
    for (size_t p = 1; p <= most && (p == 1 || tiles * (p - 1) < 4 * held); p++) {
        const size_t cost = (tiles * p + held - 1) / held * (((work + p - 1) / p + waves - 1) / waves + start);
        if (cost < least) {
            least = cost;
            best = p;
        }
    }
    return best;
}

// How a call's rows are cut: one launch, or two with parts of the inner size.
struct AdapterPlan {
    bool two;
    int down_tiles, group, parts, rank;  // tiles of a workgroup: of the first launch, of the second
    unsigned tiles, groups;
    size_t work_ld, work_bytes;
};

constexpr size_t kMostParts = 24, kHeldDown = 4;  // parts of the inner size; workgroups of the first launch that a CU holds

AdapterPlan plan_adapters(const AdapterCall& a, int planes)
{
    AdapterPlan p = {};
    size_t rows = 0;
    for (int i = 0; i < a.segments; i++) {
        rows += a.segment[i].rows;
        p.rank = std::max(p.rank,a.segment[i].rank);
    }
    const size_t cus = (size_t)device_cus(), ks = (size_t)(a.inner + 31) / 32, step = (size_t)planes * ((p.rank + 15) / 16);
    p.down_tiles = rows < 16 * cus? 1 : 2;
    // (four tiles share what is read of U, two start sooner: 4608 rows to 10240 outputs
    // with rank 64 92 us or 100, 2048 rows to 4096 24 or 23, 4608 to 3840 with rank 256,
    // where four take 96 KB of LDS, 91 or 64)
    p.group = p.rank <= 128 && rows / 64 * ((size_t)(a.rows + 31) / 32) >= 64 * cus? 4 : 2;
    for (int i = 0; i < a.segments; i++) {
        const unsigned n = (a.segment[i].rows + kTokens - 1) / kTokens;
        p.tiles += (n + p.down_tiles - 1) / p.down_tiles * p.down_tiles;
        p.groups += (n + p.group - 1) / p.group;
    }
    // Parts of the inner size, in steps of 32: four of them for a wave, two where a step
    // is much work; no more than kMostParts, whose sums the second launch reads (one row: 8.4 and
    // 10.0 us with rank 16 and, of F16, 64; two and four steps 8.8 and 11.8).
    const size_t most = std::min<size_t>(kMostParts,std::max<size_t>(1,ks / (kDownWaves * (step > 2? 2 : 4))));
    // One launch where taking D x again in each slice costs less than a second launch (its
    // start and, on the host, 3 us): short inner sizes of up to 8 rows per CU (1024 -> 4096,
    // rank 32: 1 row 5.8 us, in two 3.2 + 4.2, 300 rows 8.2 and 10.2, 1500 rows 14.3 and 15.6;
    // rank 64, 4608 rows 43.9 and 35.0; F32 with rank 64, 300 rows 12.0 and 12.1, 1500 rows
    // 21.9 and 20.7), and single rows of longer ones (2048 -> 2048, rank 32: 1 row 6.4 and
    // 7.6, 16 rows of as many requests 7.6 and 8.6, of one request 9.6 and 8.3; 4096 -> 4096,
    // rank 8 8.2 and 7.8, rank 32 9.2 and 8.1).
    const bool once = ks <= 32 && ks * step <= 256 && rows <= 8 * cus, single = rows <= 2 * p.tiles && ks * step <= 128;
    p.two = p.rank > 0 && !once && !single;
    if (!p.two) return p;
    p.parts = (int)cut_evenly(p.tiles / p.down_tiles,ks,most,kDownWaves,(p.rank > 64? kHeldDown / 2 : kHeldDown) * cus,4);
    p.work_ld = (size_t)(p.rank + 15) / 16 * 16;
    p.work_bytes = (size_t)p.parts * p.tiles * kTokens * p.work_ld * sizeof(float);
    return p;
}

}  // namespace

int adapter_planes(uint32_t type)
{
    return type == PIX_BF16? 1 : type == PIX_F16? 2 : 3;
}

size_t adapter_down_bytes(uint32_t type, size_t rank, size_t inner)
{
    return (inner + 31) / 32 * ((rank + 15) / 16) * (size_t)adapter_planes(type) * 1024;
}

size_t adapter_up_bytes(uint32_t type, size_t rank, size_t rows)
{
    return (rows + 31) / 32 * ((rank + 31) / 32) * 2 * (type == PIX_F32? 2048 : 1024);
}

hipError_t launch_adapter_form(const void* down, const void* up, uint32_t type, size_t rank, size_t inner, size_t rows, uint16_t* down_out, uint16_t* up_out,
                               hipStream_t s)
{
    const int planes = adapter_planes(type);
    const size_t down_pieces = adapter_down_bytes(type,rank,inner) / 16 / planes, up_pieces = adapter_up_bytes(type,rank,rows) / (type == PIX_F32? 32 : 16);
    const size_t grid = (down_pieces + up_pieces + 255) / 256;
    if (grid * 256 > (size_t)UINT32_MAX) return hipErrorInvalidValue;
    adapter_form_kernel<<<dim3((unsigned)grid),dim3(256),0,s>>>(down,up,type,(int)rank,inner,rows,planes,down_out,up_out,down_pieces,up_pieces);
    return hipGetLastError();
}

size_t adapters_workspace_bytes(const AdapterCall& a, int planes)
{
    return plan_adapters(a,planes).work_bytes;
}

size_t adapters_workspace_most(size_t columns, size_t requests, size_t rank)
{
    // tiles: a part of one and one to an even number for each run of rows, with an adapter
    // or between two; cut_evenly stops where the workgroups, of up to two tiles, are more
    // than four times what the CUs hold
    const size_t tiles = (columns + kTokens - 1) / kTokens + 2 * (2 * requests + 1);
    const size_t cut = std::min(kMostParts * tiles,8 * kHeldDown * (size_t)device_cus() + tiles);
    return cut * kTokens * ((rank + 15) / 16 * 16) * sizeof(float);
}

hipError_t launch_adapters(AdapterCall& a, int planes, void* workspace, hipStream_t s)
{
    AdapterPlan p = plan_adapters(a,planes);
    if (!workspace) p.two = false;
    if (!p.two) p.down_tiles = 1;
    unsigned tiles = 0, groups = 0;
    for (int i = 0; i < a.segments; i++) {
        const unsigned n = (a.segment[i].rows + kTokens - 1) / kTokens;
        a.segment[i].first_tile = tiles;
        a.segment[i].first_group = groups;
        tiles += (n + p.down_tiles - 1) / p.down_tiles * p.down_tiles;
        groups += (n + p.group - 1) / p.group;
    }
    if (!tiles) return hipSuccess;
    a.work = p.two? static_cast<float*>(workspace) : nullptr;
    a.work_ld = (int)p.work_ld;
    a.parts = p.parts;
    a.group = p.group;
    a.tiles = tiles;
    // (whole lines alone: 3839 -> 10239 in parts of lines 143 us and, around the caches, 181)
    a.past = (size_t)a.columns * a.rows * sizeof(float) >= kPastCaches && a.ldy % 32 == 0 && reinterpret_cast<uintptr_t>(a.y) % 128 == 0;
    // slices of the outputs, 32 to a wave at a time
    const size_t nT = (size_t)(a.rows + 31) / 32, waves = p.two? kWaves : kFewWaves, cut = p.two? groups : tiles;
    a.slices = (int)cut_evenly(cut,nT,(nT + waves - 1) / waves,waves,(p.two? 2 : 1) * (size_t)device_cus(),2);
    // (a launch has fewer than 2^32 threads)
    if (cut * a.slices * 64 * waves > (size_t)UINT32_MAX || (size_t)tiles * p.parts * 64 * kDownWaves > (size_t)UINT32_MAX) return hipErrorInvalidValue;
    const unsigned grid = (unsigned)(cut * a.slices);
    if (planes == 1) return launch_planes<1>(a,p.rank,grid,p.down_tiles,s);
    if (planes == 2) return launch_planes<2>(a,p.rank,grid,p.down_tiles,s);
    return launch_planes<3>(a,p.rank,grid,p.down_tiles,s);
}

}  // namespace pixhip
