// dcn_token_attention.cu -- attention over a paged cache with a sliding window of frames and first
// frames that stay visible, on CUDA cores: every type, head_dim up to 256, any strides.
//
// One warp computes one row, 32 keys at a time (RowByWarp).  Each lane reads a key of its own element by element,
// no key is shared between rows, and nothing goes to the tensor cores: four clips of 7,680 tokens take 487 ms here.
// The shapes that matter take the tensor-core kernel.
#include "dcn_token_attention.cuh"

namespace dcn {
namespace {

constexpr int kWarps = 4;
constexpr int kMaxHeadDim = 256;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) attention_direct_kernel(const AttentionParams p) {
    __shared__ float query[kWarps][kMaxHeadDim];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
    const int64_t token = row / p.args.q_heads;
    const int head = static_cast<int>(row - token * p.args.q_heads);
    if (token >= p.args.tokens) return;
    const int b = find_stream(p.cache.starts, p.cache.streams, token);
    if (b >= p.cache.streams) return;  // no stream's
    const int d = p.cache.head_dim;
    const int kv_head = head / (p.args.q_heads / p.cache.heads);

    const T *q = static_cast<const T *>(p.q.data) + token * p.q.token_stride + head * p.q.head_stride;
    for (int e = lane; e < d; e += 32) query[warp][e] = to_float<T>(q[e]);
    __syncwarp();

    const int64_t length = p.cache.lengths[b];
    const Visible seen = visible_keys(length - p.cache.starts[b + 1] + token, length, p.args.window, p.args.sinks,
                                      p.args.frame);
    RowByWarp<T, kMaxHeadDim / 32> row_sum;
    row_sum.run(p.cache, b, kv_head, query[warp], p.args.scale * 1.4426950408889634f, seen, {0, seen.low}, {seen.first, seen.high},
                nullptr);
    const bool none = seen.first <= 0 && seen.high <= seen.low;
    T *out = static_cast<T *>(p.out.data) + token * p.out.token_stride + head * p.out.head_stride;
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i)
        if (i * 32 + lane < d) out[i * 32 + lane] = from_float<T>(none ? 0.0f : row_sum.acc[i] / row_sum.l);
}

template <typename T>
cudaError_t launch_typed(const AttentionParams &p, cudaStream_t stream) {
    const int64_t rows = p.args.tokens * p.args.q_heads;
    attention_direct_kernel<T><<<static_cast<unsigned>((rows + kWarps - 1) / kWarps), kWarps * 32, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_token_attention_direct(const AttentionParams &p, cudaStream_t stream) {
    switch (p.cache.dtype) {
    case DCN_DTYPE_F16: return launch_typed<__half>(p, stream);
    case DCN_DTYPE_BF16: return launch_typed<__nv_bfloat16>(p, stream);
    default: return launch_typed<float>(p, stream);
    }
}

}  // namespace dcn
