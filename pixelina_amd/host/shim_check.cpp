// Drives the C++ shim (backend_hip.h) the way the reference's model code
// drives its Vulkan backend, for the GPU tests: a session made current on the
// thread (VulkanSession::initialize, src/backend_vulkan.cpp:1004-1011),
// activations in HipAllocator vectors (PixTensorVals, src/tensor.h:19-24),
// weights reached through a model-file / weight pair shaped like PixModelFile
// and PixWeight (src/model.h:33-56), and the calls tensor_linear and the DiT
// block's FFN make (src/tensor.cpp:156-172, src/inference.cpp:328-336).
//
//   shim_check <in> <out>
//
// <in> (little-endian): uint32 type, down_type; uint64 M, K, N, F (FFN width);
// then W1 [N][K] (type), W2 [N][K] (type), Wdown [K][F] (down_type) as GGUF
// block bytes, each preceded by its uint64 byte count; X [M][K], norm weight
// [K], modulation [K], G [M][F], U [M][F], cos, sin [M][32] and bias [N] as
// float32 (the vectors in pageable std::vector memory, as tensor_norm,
// tensor_rope and tensor_bias hold them).
// <out>: float32 Y = X W1^T [M][N] (hip_matmul); Y1, Y2 = norm(X) W1^T,
// norm(X) W2^T (hip_norm_multiply, with the weight and the modulation); the
// normalized X [M][K]; D = (silu(G) * U) Wdown^T [M][K] (hip_silu_gate_multiply);
// the gated product [M][F]; RoPE of X with K/64 heads of 64 (hip_rope, split
// halves) [M][K]; Y + bias (hip_pointwise BIAS) [M][N]; self-attention of X
// with K/64 heads of 64 (hip_attention), causal [M][K], then in the ranges form
// with rows [0, M/2) seeing every key and [M/2, M) causal [M][K]; tensor_l2norm
// of X with the norm weight (hip_l2norm, epsilon 1e-12) [M][K];
// tensor_groupnorm of X with the norm weight and the modulation as bias
// (hip_groupnorm) [M][K]; the rows of X in reverse order gathered from the
// std::vector<size_t> (hip_rows) [M][K].
//
//   shim_check cache <in> <out>
//
// A chat over the 8-bit key/value cache.  <in>: uint64 rows R, heads H, kv heads
// G, head size D, vocabulary V; then k, v [R][G D], q [R][H D], logits [R][V] as
// float32 and ids [R] as int32.  <out>, float32: attention of the first R - 1
// rows, appended in one call and weighed [R - 1][H D]; of the last row, appended
// to a copy that was then cut back to them [1][H D]; the lengths of both caches;
// the log probability and the entropy of each row [R], [R] and its two most
// likely tokens' [R][2]; as int32 the two blocks that eviction kept for each kv
// head [G][2] and the two most likely tokens [R][2].
//
//   shim_check block <in> <out>
//
// What lies between a block's linears, with the vectors in std::vector memory.
// <in>: uint64 rows R, hidden size C, heads H, kv heads G, head size D, rank A; then
// stream, branch [R][C], the two norms' weights, gate and modulation [C], a fused
// projection's rows P [R][(H + 2 G) D], the head norms' weights [D], cosines and sines
// [R][D / 2], an adapter's down [A][C] and up [(H + 2 G) D][A], all float32.  <out>,
// float32: the residual sum and its norm Y [R][C]; P plus the adapter of Y with scale
// 1.5 in the rows from R / 2 on; its q [R][H D], k and v [R][G D] (hip_split_heads); the
// same with k and v through the 8-bit cache, and causal attention over it [R][H D].
#include <cstdio>
#include <cstring>
#include <string>
#include <vector>

#include "backend_hip.h"

namespace {

struct ModelFile {  // the members of PixModelFile that hip_matmul reads
    std::string filename;
    const unsigned char* data = nullptr;
};

struct Weight {  // the members of PixWeight that hip_matmul reads
    std::string name;
    std::vector<uint64_t> shape;  // {inner, rows}
    uint32_t type = 0;
    uint64_t offset = 0, bytes = 0;
};

template <class T> using Vals = std::vector<T,HipAllocator<T>>;

bool read_all(FILE* f, void* p, size_t n) { return std::fread(p,1,n,f) == n; }

template <class V> bool read_floats(FILE* f, V& v, size_t n)
{
    v.resize(n);
    return read_all(f,v.data(),n * sizeof(float));
}

template <class V> bool write_floats(FILE* f, const V& v)
{
    return std::fwrite(v.data(),sizeof(float),v.size(),f) == v.size();
}

int fail(const char* what)
{
    std::fprintf(stderr,"shim_check: %s (%s)\n",what,pixhip_last_error());
    return 1;
}

int run_cache(const char* from, const char* to)
{
    FILE* in = std::fopen(from,"rb");
    if (!in) return fail("cannot open input");
    uint64_t dims[5];
    if (!read_all(in,dims,sizeof(dims))) return fail("short header");
    const uint64_t R = dims[0], H = dims[1], G = dims[2], D = dims[3], V = dims[4];
    HipSession session;
    if (!session.initialize()) return fail("HipSession::initialize");
    {
        Vals<float> k, v, q, logits, first((R - 1) * H * D), last(H * D), log_probs(R), entropy(R), top_log_probs(2 * R);
        Vals<int32_t> ids(R), kept(2 * G), top_ids(2 * R);
        if (!read_floats(in,k,R * G * D) || !read_floats(in,v,R * G * D) || !read_floats(in,q,R * H * D) || !read_floats(in,logits,R * V) ||
            !read_all(in,ids.data(),R * 4)) return fail("short input");
        std::fclose(in);
        pixhip_cache *chat = hip_cache(1,G,D,R), *fork = hip_cache(1,G,D,R);
        if (!chat || !fork) return fail("hip_cache");
        if (!hip_cache_append(chat,0,k.data(),v.data(),R - 1)) return fail("hip_cache_append");
        if (!hip_cache_attention(chat,0,q.data(),R - 1,H,0,true,true,0.0f,first.data())) return fail("hip_cache_attention");
        if (!hip_cache_copy(fork,chat)) return fail("hip_cache_copy");
        for (int turn = 0; turn < 2; turn++) {
            if (!hip_cache_truncate(fork,0,R - 1)) return fail("hip_cache_truncate");
            if (!hip_cache_append(fork,0,k.data() + (R - 1) * G * D,v.data() + (R - 1) * G * D,1)) return fail("hip_cache_append (step)");
        }
        if (!hip_cache_attention(fork,0,q.data() + (R - 1) * H * D,1,H,0,true,false,0.0f,last.data())) return fail("hip_cache_attention (step)");
        if (!hip_cache_evict(chat,0,2,1,kept.data())) return fail("hip_cache_evict");
        if (!hip_log_probs(logits.data(),R,V,0,ids.data(),log_probs.data(),entropy.data(),2,top_ids.data(),top_log_probs.data()))
            return fail("hip_log_probs");
        if (!hip_synchronize()) return fail("hip_synchronize");
        std::vector<float> lengths = {(float)hip_cache_length(chat,0),(float)hip_cache_length(fork,0)};
        hip_cache_free(fork);  // (the other one ends with the session)
        FILE* out = std::fopen(to,"wb");
        if (!out) return fail("cannot open output");
        const bool ok = write_floats(out,first) && write_floats(out,last) && write_floats(out,lengths) && write_floats(out,log_probs) &&
                        write_floats(out,entropy) && write_floats(out,top_log_probs) && write_floats(out,kept) && write_floats(out,top_ids);
        std::fclose(out);
        if (!ok) return fail("short write");
    }
    std::printf("shim_check ok\n");
    return 0;
}

int run_block(const char* from, const char* to)
{
    FILE* in = std::fopen(from,"rb");
    if (!in) return fail("cannot open input");
    uint64_t dims[6];
    if (!read_all(in,dims,sizeof(dims))) return fail("short header");
    const uint64_t R = dims[0], C = dims[1], H = dims[2], G = dims[3], D = dims[4], A = dims[5], W = (H + 2 * G) * D;
    HipSession session;
    if (!session.initialize()) return fail("HipSession::initialize");
    {
        Vals<float> x, branch, p;
        std::vector<float> post, pre, gate, modulation, qw, kw, cosine, sine, down, up;
        if (!read_floats(in,x,R * C) || !read_floats(in,branch,R * C) || !read_floats(in,post,C) || !read_floats(in,pre,C) ||
            !read_floats(in,gate,C) || !read_floats(in,modulation,C) || !read_floats(in,p,R * W) || !read_floats(in,qw,D) ||
            !read_floats(in,kw,D) || !read_floats(in,cosine,R * D / 2) || !read_floats(in,sine,R * D / 2) || !read_floats(in,down,A * C) ||
            !read_floats(in,up,W * A)) return fail("short input");
        std::fclose(in);
        Vals<float> y(R * C), q(R * H * D), k(R * G * D), v(R * G * D), cq(R * H * D), ck(R * G * D), cv(R * G * D), att(R * H * D);
        pixhip_residual_norm norms{};
        norms.post = norms.pre = PIXHIP_NORM_RMS;
        norms.post_weight = post.data();
        norms.pre_weight = pre.data();
        norms.post_epsilon = norms.pre_epsilon = 1e-5f;
        norms.scale = 1.0f;
        norms.gate = gate.data();
        norms.modulation = modulation.data();
        if (!hip_residual_norm_multiply(0,nullptr,nullptr,0,x.data(),branch.data(),R,C,norms,x.data(),y.data())) return fail("hip_residual_norm_multiply");
        const ModelFile file{"adapter",reinterpret_cast<const unsigned char*>(down.data())};
        const Weight wd{"down",{C,A},0,0,down.size() * 4};
        const Weight wu{"up",{A,W},0,(uint64_t)(reinterpret_cast<const unsigned char*>(up.data()) - file.data),up.size() * 4};
        pixhip_adapter* adapter = hip_adapter_of(file,wd,wu);
        if (!adapter) return fail("hip_adapter_of");
        const pixhip_adapter_range range = {R / 2,R,adapter,1.5f};
        if (!hip_adapters_reserve(R,1,1) || hip_adapters_reserve(0,1,1)) return fail("hip_adapters_reserve");
        if (!hip_adapters(&range,1,y.data(),R,0,p.data(),p.data(),W,0)) return fail("hip_adapters");
        hip_adapter_free(adapter);
        pixhip_rotation turn{};
        turn.norm = PIXHIP_NORM_RMS;
        turn.q_weight = qw.data();
        turn.k_weight = kw.data();
        turn.epsilon = 1e-6f;
        turn.cosine = cosine.data();
        turn.sine = sine.data();
        const float *pq = p.data(), *pk = pq + H * D, *pv = pk + G * D;
        if (!hip_split_heads(pq,pk,pv,R,W,H,G,D,turn,q.data(),k.data(),v.data())) return fail("hip_split_heads");
        pixhip_cache* cache = hip_cache(1,G,D,R);
        if (!cache || !hip_cache_append_rotated(cache,0,pq,pk,pv,R,W,H,turn,nullptr,cq.data())) return fail("hip_cache_append_rotated");
        if (!hip_cache_read(cache,0,0,R,ck.data(),cv.data(),nullptr)) return fail("hip_cache_read");
        if (!hip_cache_attention(cache,0,cq.data(),R,H,0,true,false,0.0f,att.data())) return fail("hip_cache_attention");
        if (!hip_synchronize()) return fail("hip_synchronize");
        FILE* out = std::fopen(to,"wb");
        if (!out) return fail("cannot open output");
        const bool ok = write_floats(out,x) && write_floats(out,y) && write_floats(out,p) && write_floats(out,q) && write_floats(out,k) &&
                        write_floats(out,v) && write_floats(out,cq) && write_floats(out,ck) && write_floats(out,cv) && write_floats(out,att);
        std::fclose(out);
        if (!ok) return fail("short write");
    }
    std::printf("shim_check ok\n");
    return 0;
}

}  // namespace

int main(int argc, char** argv)
{
    if (argc == 4 && !std::strcmp(argv[1],"cache")) return run_cache(argv[2],argv[3]);
    if (argc == 4 && !std::strcmp(argv[1],"block")) return run_block(argv[2],argv[3]);
    if (argc != 3) {
        std::fprintf(stderr,"usage: shim_check [cache | block] <in> <out>\n");
        return 2;
    }
    FILE* in = std::fopen(argv[1],"rb");
    if (!in) return fail("cannot open input");
    uint32_t types[2];
    uint64_t dims[4];
    if (!read_all(in,types,sizeof(types)) || !read_all(in,dims,sizeof(dims))) return fail("short header");
    const uint64_t M = dims[0], K = dims[1], N = dims[2], F = dims[3];

    // The "model file": the three weights back to back in one buffer.
    std::vector<unsigned char> blob;
    uint64_t sizes[3];
    for (int i = 0; i < 3; i++) {
        if (!read_all(in,&sizes[i],8)) return fail("short weight size");
        const size_t at = blob.size();
        blob.resize(at + sizes[i]);
        if (!read_all(in,blob.data() + at,sizes[i])) return fail("short weight bytes");
    }
    ModelFile file{"shim_check.gguf",blob.data()};
    Weight w1{"blk.0.ffn_gate.weight",{K,N},types[0],0,sizes[0]};
    Weight w2{"blk.0.ffn_up.weight",{K,N},types[0],sizes[0],sizes[1]};
    Weight wd{"blk.0.ffn_down.weight",{F,K},types[1],sizes[0] + sizes[1],sizes[2]};

    HipSession session;
    if (!session.initialize()) return fail("HipSession::initialize");
    {
        // HipAllocator vectors allocate through the active session (pinned host memory).
        Vals<float> x, gate, up;
        std::vector<float> norm_weight, modulation, cosine, sine, bias;
        if (!read_floats(in,x,M * K) || !read_floats(in,norm_weight,K) || !read_floats(in,modulation,K) ||
            !read_floats(in,gate,M * F) || !read_floats(in,up,M * F) || !read_floats(in,cosine,M * 32) ||
            !read_floats(in,sine,M * 32) || !read_floats(in,bias,N))
            return fail("short activations");
        std::fclose(in);

        Vals<float> y(M * N), y1(M * N), y2(M * N), normalized(M * K), d(M * K), gated(M * F);
        // tensor_linear -> cpu_matmul -> (backend) matmul
        if (!hip_matmul(file,w1,x.data(),M,y.data())) return fail("hip_matmul");
        // the FFN input: norm + modulation, quantized once for both linears
        pixhip_weight* ws[2] = {hip_weight_of(file,w1),hip_weight_of(file,w2)};
        float* outs[2] = {y1.data(),y2.data()};
        if (!ws[0] || !ws[1]) return fail("hip_weight_of");
        if (!hip_norm_multiply(w1.type,ws,outs,2,x.data(),M,K,norm_weight.data(),1e-5f,false,modulation.data(),normalized.data()))
            return fail("hip_norm_multiply");
        // the FFN down input: silu(gate) * up, then the down linear
        pixhip_weight* down = hip_weight_of(file,wd);
        if (!down || !hip_silu_gate_multiply(wd.type,down,gate.data(),up.data(),M,F,d.data(),gated.data()))
            return fail("hip_silu_gate_multiply");
        // tensor_rope / tensor_bias hand their std::vector tables straight in
        Vals<float> roped(x.begin(),x.end()), biased(M * N);
        if (!hip_synchronize()) return fail("hip_synchronize");
        for (size_t i = 0; i < biased.size(); i++) biased[i] = y[i];
        if (!hip_rope(roped.data(),M,K,K / 64,cosine.data(),sine.data(),false)) return fail("hip_rope");
        if (!hip_pointwise(PIXHIP_OP_BIAS,biased.data(),bias.data(),M,N)) return fail("hip_pointwise(BIAS)");
        // tensor_attention, both forms
        Vals<float> att(M * K), att2(M * K);
        if (!hip_attention(x.data(),M,x.data(),x.data(),M,K / 64,K / 64,K,true,att.data())) return fail("hip_attention");
        const pixhip_attention_range ranges[2] = {{0,M / 2,M,0},{M / 2,M,M,1}};
        if (!hip_attention(x.data(),M,x.data(),x.data(),M,K / 64,K / 64,K,ranges,2,0,att2.data())) return fail("hip_attention(ranges)");
        // tensor_l2norm / tensor_groupnorm / tensor_gather with the reference's vectors
        Vals<float> l2(M * K), gn(M * K), gathered(M * K);
        if (!hip_l2norm(x.data(),M,K,norm_weight.data(),1e-12f,l2.data())) return fail("hip_l2norm");
        if (!hip_groupnorm(x.data(),M,K,norm_weight.data(),modulation.data(),gn.data())) return fail("hip_groupnorm");
        std::vector<size_t> reversed(M);
        for (size_t i = 0; i < M; i++) reversed[i] = M - 1 - i;
        if (!hip_rows(x.data(),M,gathered.data(),M,K,reversed.data(),M,false)) return fail("hip_rows");
        if (!hip_synchronize()) return fail("hip_synchronize");

        FILE* out = std::fopen(argv[2],"wb");
        if (!out) return fail("cannot open output");
        const bool ok = write_floats(out,y) && write_floats(out,y1) && write_floats(out,y2) && write_floats(out,normalized) &&
                        write_floats(out,d) && write_floats(out,gated) && write_floats(out,roped) && write_floats(out,biased) &&
                        write_floats(out,att) && write_floats(out,att2) && write_floats(out,l2) && write_floats(out,gn) &&
                        write_floats(out,gathered);
        std::fclose(out);
        if (!ok) return fail("short write");
    }
    std::printf("shim_check ok\n");
    return 0;
}
