// q, k and v out of the rows of a fused projection, the heads of q and k normalized
// and rotated (z_block, src/inference.cpp:301-318; qwen_vl.cpp's and qwen_chat.cpp's
// attention): one pass over the rows instead of a copy, a norm and a rotation of each.
// Bound by HBM: every value is read and written once (4608 rows of 90 heads of 128 with
// norms and rotation 85 us for 427 MB, 5.0 TB/s).
#include "heads_device.h"

namespace pixhip {

namespace {

constexpr int kSplitThreads = 256;

// Workgroups: q's items, then k's, then v's.
template <int G, int MODE>
__global__ __launch_bounds__(kSplitThreads) void split_heads_kernel(HeadTurn t, SplitHeads a, unsigned q_groups, unsigned k_groups, int per_q, int per_kv)
{
    constexpr int kItems = kSplitThreads / G;
    const unsigned id = blockIdx.x, lane_group = threadIdx.x / G;
    if (id < q_groups)
        turn_rows<G,MODE>(t,a.q,a.ld_q,a.q_out,a.rows,(int)a.heads,per_q,t.q_weight,false,(size_t)id * kItems + lane_group);
    else if (id < q_groups + k_groups)
        turn_rows<G,MODE>(t,a.k,a.ld_kv,a.k_out,a.rows,(int)a.kv_heads,per_kv,t.k_weight,false,(size_t)(id - q_groups) * kItems + lane_group);
    else
        turn_rows<G,MODE>(t,a.v,a.ld_kv,a.v_out,a.rows,(int)a.kv_heads,per_kv,nullptr,true,(size_t)(id - q_groups - k_groups) * kItems + lane_group);
}

template <int G, int MODE>
hipError_t launch_split(const HeadTurn& t, const SplitHeads& a, hipStream_t s)
{
    constexpr size_t kItems = kSplitThreads / G;
    const int per_q = turn_heads_per_item(a.rows,a.heads,t.dim,G), per_kv = turn_heads_per_item(a.rows,a.kv_heads,t.dim,G);
    auto groups = [&](const float* out, size_t heads, int per) { return out? (a.rows * ((heads + per - 1) / per) + kItems - 1) / kItems : 0; };
    const size_t q = groups(a.q_out,a.heads,per_q), k = groups(a.k_out,a.kv_heads,per_kv), v = groups(a.v_out,a.kv_heads,per_kv);
    if ((q + k + v) * kSplitThreads > (size_t)UINT32_MAX) return hipErrorInvalidValue;  // (a launch has fewer than 2^32 threads)
    split_heads_kernel<G,MODE><<<dim3((unsigned)(q + k + v)),dim3(kSplitThreads),0,s>>>(t,a,(unsigned)q,(unsigned)k,per_q,per_kv);
    return hipGetLastError();
}

}  // namespace

// Heads of a row that one group of lanes takes, one after the other with its tables read
// once: two, and four where a head leaves lanes idle, if that leaves enough groups to fill
// the CUs; one where the call is short.  4608 rows with 1, 2 and 4: 90 heads of 128 84.2,
// 85.0 and 89.8 us; 30 of 80 17.6, 16.9 and 15.7; 48 of 90 48.0, 42.2 and 40.1; 24 of 256
// 56.0, 50.0 and 48.6.
int turn_heads_per_item(size_t rows, size_t heads, int dim, int lanes)
{
    const size_t fill = (size_t)device_cus() * 1024 / (size_t)lanes;  // groups of lanes in flight
    const int most = dim > 6 * lanes? 2 : 4;
    int per = 1;
    while (per < most && (size_t)per * 2 <= heads && rows * heads / (size_t)(2 * per) >= fill) per *= 2;
    return per;
}

hipError_t launch_split_heads(const HeadTurn& t, const SplitHeads& a, hipStream_t s)
{
    const bool wide = t.dim > 128;
    if (!t.vec) return wide? launch_split<64,kTurnScalar>(t,a,s) : launch_split<16,kTurnScalar>(t,a,s);
    if (t.interleaved) return wide? launch_split<64,kTurnAdjacent>(t,a,s) : launch_split<16,kTurnAdjacent>(t,a,s);
    return wide? launch_split<64,kTurnHalves>(t,a,s) : launch_split<16,kTurnHalves>(t,a,s);
}

}  // namespace pixhip
