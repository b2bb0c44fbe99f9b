// dcn_token_norm.cu -- the norms before and after a block, with its gate, residual scale and
// modulation, in one pass over the row.
//
//   branch = post ? N(x) post_weight + post_bias : x
//   hidden = residual_scale residual + gate branch
//   out    = (N(hidden) weight + bias) (1 + scale) + shift
//
// What bounds it is memory: each row is read once and written once (4 rows of traffic with a
// residual, 2 without; the width-long vectors stay in L1/L2).  So a row lives in the registers of
// the NT threads that hold it, 16 bytes a load, and its statistics are two-pass there (the mean
// first, then the squares of the centred values), which costs no traffic and does not cancel.
#include "dcn_tokens.cuh"

namespace dcn {
namespace {

template <int NT>
__device__ __forceinline__ float row_sum(float v, float *scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (NT == 32) return v;
    // A row of more than one warp is a whole block: sum the warps' sums in a fixed order.
    const int warp = threadIdx.x >> 5;
    __syncthreads();  // the previous sum has been read
    if ((threadIdx.x & 31) == 0) scratch[warp] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) s += scratch[w];
    return s;
}

template <typename T, int VEC, int NT, int NV>
struct Row {
    float v[NV][VEC];

    // x <- N(x) over `width` elements.  Places past the width hold 0.
    __device__ __forceinline__ void normalise(int kind, int width, float epsilon, int lane, float *scratch) {
        const float inv = 1.0f / static_cast<float>(width);
        if (kind == DCN_NORM_LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) s += v[i][j];
            const float mean = row_sum<NT>(s, scratch) * inv;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if ((i * NT + lane) * VEC < width) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) v[i][j] -= mean;
                }
        }
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) s = fmaf(v[i][j], v[i][j], s);
        const float r = rsqrtf(fmaf(row_sum<NT>(s, scratch), inv, epsilon));
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] *= r;
    }
};

// NT threads hold a row, NV packs of VEC elements each: pack i of thread t covers elements
// [(i NT + t) VEC, ...).  NT == 32: blockDim.x / 32 rows a block; otherwise one row a block.
template <typename T, int VEC, int NT, int NV>
__global__ void __launch_bounds__(NT == 32 ? 128 : NT) token_norm_kernel(const dcn_token_norm_args a) {
    __shared__ float scratch[NT / 32];
    const int lane = NT == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t row = NT == 32 ? static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= a.rows) return;
    const int width = a.width;
    const int64_t g = row / a.group;

    auto at = [&](const void *base, int64_t offset) { return static_cast<const T *>(base) + offset; };
    Row<T, VEC, NT, NV> x;
    Pack<T, VEC> xp[NV], rp[NV];
    // Both tensors' loads go out before anything waits for either.
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * NT + lane) * VEC;
        if (c < width) {
            xp[i] = load_pack<T, VEC>(at(a.x, row * a.x_stride + c));
            if (a.residual) rp[i] = load_pack<T, VEC>(at(a.residual, row * a.residual_stride + c));
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * NT + lane) * VEC;
#pragma unroll
        for (int j = 0; j < VEC; ++j) x.v[i][j] = 0.0f;
        if (c < width) unpack<T, VEC>(xp[i], x.v[i]);
    }
    if (a.residual) {
        if (a.post) {
            x.normalise(a.kind, width, a.epsilon, lane, scratch);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * NT + lane) * VEC;
                if (c < width) {
                    float w[VEC], b[VEC];
                    if (a.post_weight) {
                        unpack<T, VEC>(load_pack<T, VEC>(at(a.post_weight, c)), w);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) x.v[i][j] *= w[j];
                    }
                    if (a.post_bias) {
                        unpack<T, VEC>(load_pack<T, VEC>(at(a.post_bias, c)), b);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) x.v[i][j] += b[j];
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * NT + lane) * VEC;
            if (c < width) {
                if (a.gate) {
                    float m[VEC];
                    unpack<T, VEC>(load_pack<T, VEC>(at(a.gate, g * a.gate_stride + c)), m);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) x.v[i][j] *= m[j];
                }
                float r[VEC];
                unpack<T, VEC>(rp[i], r);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(r[j], a.residual_scale, x.v[i][j]);
                if (a.hidden)
                    store_pack<T, VEC>(static_cast<T *>(a.hidden) + row * a.hidden_stride + c, pack<T, VEC>(x.v[i]));
            }
        }
    }
    if (a.out == nullptr) return;
    x.normalise(a.kind, width, a.epsilon, lane, scratch);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * NT + lane) * VEC;
        if (c < width) {
            float m[VEC];
            if (a.weight) {
                unpack<T, VEC>(load_pack<T, VEC>(at(a.weight, c)), m);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x.v[i][j] *= m[j];
            }
            if (a.bias) {
                unpack<T, VEC>(load_pack<T, VEC>(at(a.bias, c)), m);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x.v[i][j] += m[j];
            }
            if (a.scale) {
                unpack<T, VEC>(load_pack<T, VEC>(at(a.scale, g * a.scale_stride + c)), m);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(x.v[i][j], m[j], x.v[i][j]);
            }
            if (a.shift) {
                unpack<T, VEC>(load_pack<T, VEC>(at(a.shift, g * a.shift_stride + c)), m);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x.v[i][j] += m[j];
            }
            store_pack<T, VEC>(static_cast<T *>(a.out) + row * a.out_stride + c, pack<T, VEC>(x.v[i]));
        }
    }
}

template <typename T, int VEC, int NT, int NV>
cudaError_t launch(const dcn_token_norm_args &a, cudaStream_t stream) {
    const int rows_per_block = NT == 32 ? 4 : 1;
    const int64_t blocks = (a.rows + rows_per_block - 1) / rows_per_block;
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    token_norm_kernel<T, VEC, NT, NV><<<static_cast<unsigned>(blocks), NT == 32 ? 128 : NT, 0, stream>>>(a);
    return cudaGetLastError();
}

// Whether every row and vector may be read in 16-byte packs.
template <typename T>
bool vectorised(const dcn_token_norm_args &a) {
    constexpr int V = kVec<T>;
    if (a.width % V != 0) return false;
    const void *pointers[] = {a.x, a.residual, a.post_weight, a.post_bias, a.weight, a.bias,
                              a.gate, a.scale, a.shift, a.hidden, a.out};
    for (const void *p : pointers)
        if (reinterpret_cast<uintptr_t>(p) % 16 != 0) return false;
    const int64_t strides[] = {a.x_stride, a.residual_stride, a.hidden_stride, a.out_stride,
                               a.gate_stride, a.scale_stride, a.shift_stride};
    for (int64_t s : strides)
        if (s % V != 0) return false;
    return true;
}

template <typename T>
cudaError_t launch_typed(const dcn_token_norm_args &a, cudaStream_t stream) {
    constexpr int V = kVec<T>;
    if (vectorised<T>(a)) {
        const int packs = a.width / V;
        if (packs <= 32) return launch<T, V, 32, 1>(a, stream);
        if (packs <= 64) return launch<T, V, 32, 2>(a, stream);
        if (packs <= 128) return launch<T, V, 32, 4>(a, stream);
        if (packs <= 512) return launch<T, V, 128, 4>(a, stream);
        return launch<T, V, 512, 4>(a, stream);
    }
    if (a.width <= 256) return launch<T, 1, 32, 8>(a, stream);
    if (a.width <= 2048) return launch<T, 1, 128, 16>(a, stream);
    return launch<T, 1, 512, 16>(a, stream);
}

}  // namespace

cudaError_t launch_token_norm(const dcn_token_norm_args &a, cudaStream_t stream) {
    switch (a.dtype) {
    case DCN_DTYPE_F16: return launch_typed<__half>(a, stream);
    case DCN_DTYPE_BF16: return launch_typed<__nv_bfloat16>(a, stream);
    default: return launch_typed<float>(a, stream);
    }
}

}  // namespace dcn
