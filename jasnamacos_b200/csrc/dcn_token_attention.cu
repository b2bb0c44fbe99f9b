// dcn_token_attention.cu -- attention over a paged cache with a sliding window of frames and first
// frames that stay visible, on CUDA cores: every type, head_dim up to 256, any strides.
//
// One warp computes one row: out = sum_s exp(scale q.k_s - m) v_s / sum_s exp(scale q.k_s - m) over
// the row's visible keys, m the running maximum.  It takes 32 keys at a time, one key a lane for the
// products (the query row lies in shared memory), then the lanes turn to the value's elements.
// Hidden keys are never read, so what they hold cannot matter.  It reads each key once per row and
// feeds no tensor core, so it is bound by issue; the shapes that matter take the tensor-core kernel.
#include "dcn_token_attention.cuh"
#include "dcn_tokens.cuh"

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
    if (b >= p.cache.streams) return;  // padding past the last stream
    const int d = p.cache.head_dim;
    const int kv_head = head / (p.args.q_heads / p.cache.heads);

    const T *q = static_cast<const T *>(p.q.data) + token * p.q.token_stride + head * p.q.head_stride;
    for (int e = lane; e < d; e += 32) query[warp][e] = to_float<T>(q[e]) * p.args.scale;
    __syncwarp();

    const int64_t length = p.cache.lengths[b];
    const Visible seen = visible_keys(length - p.cache.starts[b + 1] + token, length, p.args.window, p.args.sinks,
                                      p.args.frame);
    float m = -INFINITY, sum = 0.0f;
    float acc[kMaxHeadDim / 32];
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i) acc[i] = 0.0f;

    const T *keys = static_cast<const T *>(p.cache.keys) + kv_head * p.cache.key_head_stride;
    const T *values = static_cast<const T *>(p.cache.values) + kv_head * p.cache.value_head_stride;
    for (int part = 0; part < 2; ++part) {
        const int64_t begin = part == 0 ? 0 : seen.low, end = part == 0 ? seen.first : seen.high;
        for (int64_t base = begin; base < end; base += 32) {
            const int64_t key = base + lane;
            float score = -INFINITY;
            int64_t value_at = -1;
            if (key < end) {
                const int64_t column = key / p.cache.page_size, slot = key - column * p.cache.page_size;
                const int page = column < p.cache.table_columns
                                     ? p.cache.table[b * p.cache.table_stride + column] : -1;
                score = 0.0f;
                if (page >= 0 && page < p.cache.pages) {
                    const T *k = keys + page * p.cache.key_page_stride + slot * p.cache.key_slot_stride;
                    value_at = page * p.cache.value_page_stride + slot * p.cache.value_slot_stride;
                    for (int e = 0; e < d; ++e) score = fmaf(query[warp][e], to_float<T>(k[e]), score);
                }
            }
            float top = score;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(m, top);
            // -inf so far (scores of -inf only): nothing has weight yet, and -inf - -inf is not 0.
            const float base_of_exp = top == -INFINITY ? 0.0f : top;
            const float shrink = expf(m - base_of_exp);
            const float w = expf(score - base_of_exp);
            m = top;
            float total = w;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            sum = fmaf(sum, shrink, total);
#pragma unroll
            for (int i = 0; i < kMaxHeadDim / 32; ++i) acc[i] *= shrink;
            const int count = static_cast<int>(min(end - base, int64_t{32}));
            for (int s = 0; s < count; ++s) {
                const float ws = __shfl_sync(0xffffffffu, w, s);
                const int64_t at = __shfl_sync(0xffffffffu, value_at, s);
                if (at < 0) continue;  // a key without a page: zeros
#pragma unroll
                for (int i = 0; i < kMaxHeadDim / 32; ++i)
                    if (i * 32 + lane < d) acc[i] = fmaf(ws, to_float<T>(values[at + i * 32 + lane]), acc[i]);
            }
        }
    }
    const bool none = seen.first <= 0 && seen.high <= seen.low;
    T *out = static_cast<T *>(p.out.data) + token * p.out.token_stride + head * p.out.head_stride;
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i)
        if (i * 32 + lane < d) out[i * 32 + lane] = from_float<T>(none ? 0.0f : acc[i] / sum);
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
