// Low-rank adapters of the requests of a batch beside the linear layer that they
// share (gfx950): for each row c that an adapter a serves
//   y[c] = base[c] + scale * U_a (D_a x[c])
// with D_a [rank][inner] and U_a [rows][rank] of 16 or 32 bits, all else in fp32.
//
// Products.  A value of 24 bits is the exact sum of three bf16 values, each the
// leading 8 bits of what the ones before it leave; an F16 weight is one of two, a
// BF16 weight is one itself.  Each product of planes p and q with p + q <= 2 is one
// v_mfma_f32_16x16x32_bf16 with fp32 sums, the ones left out are below 2^-24 of the
// whole: 3, 5 or 6 instructions per 16 x 16 x 32 products.  A row that holds NaN or an
// infinity gives NaN (an infinity's second plane is Inf - Inf).
//
// Layouts, as the matrix instruction's lanes take them, 16 bytes a lane (so a wave
// reads 1 KB in a row):
//   down  [inner / 32][rank / 16][plane][64 lanes][8]: lane l holds rank l % 16,
//         inner values 8 (l / 16) .. + 7
//   up    [rows / 32][rank / 32][half][plane][64 lanes][8]: lane l holds row
//         8 (l % 16 / 4) + 4 half + l % 4 of the 32, ranks 8 (l / 16) .. + 7, so that
//         after both halves a lane has 8 consecutive rows of one token
// padded with zeros.
#include <algorithm>

#include "pixhip_device.h"
#include "pixhip_internal.h"

namespace pixhip {

namespace {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr int kTokens = 16;  // rows of a tile
constexpr int kWaves = 8;

// The three bf16 planes of 8 values, the leading bits first.
__device__ __forceinline__ void split_planes(const float (&x)[8], v8bf (&p)[3])
{
    v4u w[3];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int q = 0; q < 3; q++) {
            const uint32_t ua = __float_as_uint(a) & 0xffff0000u, ub = __float_as_uint(b) & 0xffff0000u;
            w[q][i] = ua >> 16 | ub;
            a -= __uint_as_float(ua);
            b -= __uint_as_float(ub);
        }
    }
#pragma unroll
    for (int q = 0; q < 3; q++) p[q] = __builtin_bit_cast(v8bf,w[q]);
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
    uint16_t* to;
    if (e < down_pieces) {
        const int tiles = (rank + 15) / 16;
        const size_t g = e / 64, step = g / (unsigned)tiles;
        const int t = (int)(g % (unsigned)tiles), r = 16 * t + lo;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const size_t k = 32 * step + 8 * hi + j;
            x[j] = r < rank && k < inner? source_value(down,type,(size_t)r * inner + k) : 0.0f;
        }
        to = down_out + g * planes * 512 + lane * 8;
    } else {
        const int steps = (rank + 31) / 32;
        const size_t g = (e - down_pieces) / 64, T = g / (unsigned)(2 * steps);
        const int s = (int)(g % (unsigned)(2 * steps)) / 2, half = (int)(g % 2);
        const size_t row = 32 * T + 8 * (lo / 4) + 4 * half + lo % 4;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int r = 32 * s + 8 * hi + j;
            x[j] = row < rows && r < rank? source_value(up,type,row * rank + r) : 0.0f;
        }
        to = up_out + g * planes * 512 + lane * 8;
    }
    v8bf p[3];
    split_planes(x,p);
    for (int q = 0; q < planes; q++) *reinterpret_cast<v8bf*>(to + q * 512) = p[q];
}

// 8 values of a row of x from k on, zeros past the row's end.
template <bool VEC>
__device__ __forceinline__ void load8(const float* row, int K, int k, float (&x)[8])
{
    if constexpr (VEC) {  // K a multiple of 4
        const float4 a = *reinterpret_cast<const float4*>(row + (k < K? k : 0)), b = *reinterpret_cast<const float4*>(row + (k + 4 < K? k + 4 : 0));
        const bool ina = k < K, inb = k + 4 < K;
        x[0] = ina? a.x : 0.0f;
        x[1] = ina? a.y : 0.0f;
        x[2] = ina? a.z : 0.0f;
        x[3] = ina? a.w : 0.0f;
        x[4] = inb? b.x : 0.0f;
        x[5] = inb? b.y : 0.0f;
        x[6] = inb? b.z : 0.0f;
        x[7] = inb? b.w : 0.0f;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float v = row[k + j < K? k + j : 0];
            x[j] = k + j < K? v : 0.0f;
        }
    }
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

// One workgroup per (tile of 16 rows, slice of the outputs): D x over the whole inner
// size, shared by the waves in steps of 32, their sums joined in LDS; then U times
// that for the slice's rows of U, 32 to a wave at a time.  RC: 16-rank tiles that the
// inner loop takes at once; more ranks take more turns over x.
template <int NP, int RC, bool VEC>
__global__ __launch_bounds__(64 * kWaves) void adapters_kernel(AdapterCall a)
{
    constexpr int LD = 16 * RC + 4;
    constexpr int U = NP * RC <= 2? 4 : 2;  // steps in flight
    __shared__ __attribute__((aligned(16))) float red[kWaves * kTokens * LD];
    extern __shared__ __attribute__((aligned(16))) uint16_t parts[];  // [rank / 32][plane][64][8]: the sums' planes
    const int tid = (int)threadIdx.x, lane = tid & 63, lo = lane % 16, hi = lane / 16;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned tile = blockIdx.x / (unsigned)a.slices, slice = blockIdx.x % (unsigned)a.slices;
    // the segment of this tile: the last one that begins at or before it (one load per lane)
    const unsigned begins = a.segment[lane < a.segments? lane : 0].first_tile;
    const int si = __builtin_amdgcn_readfirstlane(__builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < a.segments && begins <= tile)) - 1);
    const AdapterSegment& seg = a.segment[si];
    const unsigned at = (tile - seg.first_tile) * kTokens + (unsigned)lo;
    const bool live = at < seg.rows;
    const unsigned place = seg.first + (live? at : seg.rows - 1);
    const size_t row = a.listed? a.list[place] : place;
    const int rank = seg.rank, tiles = (rank + 15) / 16, steps = (rank + 31) / 32;
    if (rank) {
        const float* x = a.x + row * a.ldx;
        const int ks = (a.inner + 31) / 32;
        for (int t0 = 0; t0 < tiles; t0 += RC) {
            const int nt = tiles - t0 < RC? tiles - t0 : RC;
            v4f acc[RC];
#pragma unroll
            for (int t = 0; t < RC; t++) acc[t] = v4f{0.f,0.f,0.f,0.f};
            for (int s0 = wave; s0 < ks; s0 += kWaves * U) {
                float xv[U][8];
                v8bf w[U][RC][NP];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int s = s0 + kWaves * u;
                    load8<VEC>(x,a.inner,32 * s + 8 * hi,xv[u]);
                    const uint16_t* d = seg.down + ((size_t)(s < ks? s : ks - 1) * tiles + t0) * (NP * 512) + lane * 8;
#pragma unroll
                    for (int t = 0; t < RC; t++)
                        if (t < nt)
#pragma unroll
                            for (int q = 0; q < NP; q++) w[u][t][q] = *reinterpret_cast<const v8bf*>(d + (t * NP + q) * 512);
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    if (s0 + kWaves * u >= ks) continue;  // whole wave
                    v8bf p[3];
                    split_planes(xv[u],p);
#pragma unroll
                    for (int t = 0; t < RC; t++)
                        if (t < nt) acc[t] = multiply<NP>(w[u][t],p,acc[t]);
                }
            }
#pragma unroll
            for (int t = 0; t < RC; t++)
                if (t < nt) *reinterpret_cast<v4f*>(red + (wave * kTokens + lo) * LD + 16 * t + 4 * hi) = acc[t];
            __syncthreads();
            // 4 ranks of a token per thread: the waves' sums in order, scaled, as planes
            for (int e = tid; e < kTokens * 4 * RC; e += 64 * kWaves) {
                const int n = e % kTokens, r = 4 * (e / kTokens), to = 16 * t0 + r;
                if (to >= 32 * steps) continue;
                v4f sum = {0.f,0.f,0.f,0.f};
                if (r < 16 * nt) {  // (an odd last tile's neighbour: zeros)
                    sum = *reinterpret_cast<const v4f*>(red + n * LD + r);
#pragma unroll
                    for (int w = 1; w < kWaves; w++) sum += *reinterpret_cast<const v4f*>(red + (w * kTokens + n) * LD + r);
                }
                float v[8] = {sum[0] * seg.scale,sum[1] * seg.scale,sum[2] * seg.scale,sum[3] * seg.scale,0.f,0.f,0.f,0.f};
                v8bf p[3];
                split_planes(v,p);
                uint16_t* o = parts + ((to / 32) * 3 * 64 + 16 * (to % 32 / 8) + n) * 8 + to % 8;
#pragma unroll
                for (int q = 0; q < 3; q++) *reinterpret_cast<uint2*>(o + q * 512) = make_uint2(__builtin_bit_cast(v4u,p[q])[0],__builtin_bit_cast(v4u,p[q])[1]);
            }
            __syncthreads();
        }
        // RC 1: the neighbour of an odd last tile has no turn of its own
        if (RC == 1 && tiles % 2) {
            if (tid < kTokens * 4) {
                const int n = tid % kTokens, to = 16 * tiles + 4 * (tid / kTokens);
                uint16_t* o = parts + ((to / 32) * 3 * 64 + 16 * (to % 32 / 8) + n) * 8 + to % 8;
#pragma unroll
                for (int q = 0; q < 3; q++) *reinterpret_cast<uint2*>(o + q * 512) = make_uint2(0,0);
            }
            __syncthreads();
        }
    }
    const int nT = (a.rows + 31) / 32;
    const int T1 = (int)((size_t)(slice + 1) * nT / (unsigned)a.slices);
    const float* base = a.base? a.base + row * a.ldy : nullptr;
    float* y = a.y + row * a.ldy;
    for (int T = (int)((size_t)slice * nT / (unsigned)a.slices) + wave; T < T1; T += kWaves) {
        const int f = 32 * T + 8 * hi;
        float b[8] = {0.f,0.f,0.f,0.f,0.f,0.f,0.f,0.f};
        if (base) load8<VEC>(base,a.rows,f,b);
        v4f acc[2] = {{0.f,0.f,0.f,0.f},{0.f,0.f,0.f,0.f}};
        const uint16_t* u = seg.up + (size_t)T * steps * (2 * NP * 512) + lane * 8;
        for (int s = 0; s < steps; s++) {
            v8bf w[2][NP], p[3];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int q = 0; q < NP; q++) w[h][q] = *reinterpret_cast<const v8bf*>(u + ((s * 2 + h) * NP + q) * 512);
#pragma unroll
            for (int q = 0; q < 3; q++) p[q] = *reinterpret_cast<const v8bf*>(parts + ((s * 3 + q) * 64 + lane) * 8);
#pragma unroll
            for (int h = 0; h < 2; h++) acc[h] = multiply<NP>(w[h],p,acc[h]);
        }
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; j++) o[j] = rank? b[j] + acc[j / 4][j % 4] : b[j];
        if (!live) continue;
        if constexpr (VEC) {
            if (f < a.rows) *reinterpret_cast<float4*>(y + f) = make_float4(o[0],o[1],o[2],o[3]);
            if (f + 4 < a.rows) *reinterpret_cast<float4*>(y + f + 4) = make_float4(o[4],o[5],o[6],o[7]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (f + j < a.rows) y[f + j] = o[j];
        }
    }
}

template <int NP, int RC>
hipError_t launch_rank(const AdapterCall& a, unsigned grid, size_t lds, bool vec, hipStream_t s)
{
    if (vec) adapters_kernel<NP,RC,true><<<dim3(grid),dim3(64 * kWaves),lds,s>>>(a);
    else adapters_kernel<NP,RC,false><<<dim3(grid),dim3(64 * kWaves),lds,s>>>(a);
    return hipGetLastError();
}

template <int NP>
hipError_t launch_planes(const AdapterCall& a, int rank, unsigned grid, bool vec, hipStream_t s)
{
    const size_t lds = (size_t)((rank + 31) / 32) * 3 * 1024;
    if (rank <= 16) return launch_rank<NP,1>(a,grid,lds,vec,s);
    if (rank <= 32) return launch_rank<NP,2>(a,grid,lds,vec,s);
    return launch_rank<NP,4>(a,grid,lds,vec,s);
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
    return (rows + 31) / 32 * ((rank + 31) / 32) * 2 * (size_t)adapter_planes(type) * 1024;
}

hipError_t launch_adapter_form(const void* down, const void* up, uint32_t type, size_t rank, size_t inner, size_t rows, uint16_t* down_out, uint16_t* up_out,
                               hipStream_t s)
{
    const int planes = adapter_planes(type);
    const size_t down_pieces = adapter_down_bytes(type,rank,inner) / 16 / planes, up_pieces = adapter_up_bytes(type,rank,rows) / 16 / planes;
    const size_t grid = (down_pieces + up_pieces + 255) / 256;
    if (grid > (size_t)INT32_MAX) return hipErrorInvalidValue;
    adapter_form_kernel<<<dim3((unsigned)grid),dim3(256),0,s>>>(down,up,type,(int)rank,inner,rows,planes,down_out,up_out,down_pieces,up_pieces);
    return hipGetLastError();
}

hipError_t launch_adapters(AdapterCall& a, int planes, hipStream_t s)
{
    unsigned tiles = 0;
    int rank = 0;
    for (int i = 0; i < a.segments; i++) {
        a.segment[i].first_tile = tiles;
        tiles += (a.segment[i].rows + kTokens - 1) / kTokens;
        rank = std::max(rank,a.segment[i].rank);
    }
    if (!tiles) return hipSuccess;
    // Slices of the outputs: as many workgroups as the CUs hold two of, each with
    // work for all its waves.
    const size_t nT = (size_t)(a.rows + 31) / 32, most = (nT + kWaves - 1) / kWaves, want = (2 * (size_t)device_cus() + tiles - 1) / tiles;
    a.slices = (int)std::max<size_t>(1,std::min(most,want));
    if ((size_t)tiles * a.slices > (size_t)INT32_MAX) return hipErrorInvalidValue;
    const unsigned grid = tiles * (unsigned)a.slices;
    const bool vec = a.vec;
    if (planes == 1) return launch_planes<1>(a,rank,grid,vec,s);
    if (planes == 2) return launch_planes<2>(a,rank,grid,vec,s);
    return launch_planes<3>(a,rank,grid,vec,s);
}

}  // namespace pixhip
