// dcn_tokens.cuh -- what the token operators share: element types and their vector loads, the
// parameters of their kernels, and the launchers that dcn_token_api.cu calls.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "dcn_b200.h"
#include "dcn_common.cuh"

namespace dcn {

// ---- launchers (arguments already validated) ---------------------------------------

cudaError_t launch_token_norm(const dcn_token_norm_args &a, cudaStream_t stream);

// One strided head tensor that the rotation kernel reads and writes.  With to_cache, the
// destination is the cache: dst its first page, dst_token_stride unused.
struct HeadCopy {
    const void *src;
    void *dst;
    int64_t src_token, src_head;  // strides in elements
    int64_t dst_token, dst_head;
    int64_t dst_page, dst_slot;
    int32_t heads;
    bool rotate, to_cache;
};

struct RotateParams {
    HeadCopy part[3];
    int32_t parts;
    int32_t head_dim;
    int64_t tokens;
    dcn_rotation rotation;
    // Where tokens go in the cache (streams == 0: no part goes to a cache).
    const int32_t *table, *starts, *lengths;
    int64_t table_stride;
    int32_t streams, table_columns, pages, page_size;
};

cudaError_t launch_token_rotate(dcn_dtype dtype, const RotateParams &p, cudaStream_t stream);

struct AttentionParams {
    dcn_paged_cache cache;
    dcn_token_attention_args args;
    dcn_heads q, out;
};

cudaError_t launch_token_attention_direct(const AttentionParams &p, cudaStream_t stream);

// The tensor-core kernel: whether it takes a cache and arguments, its scratch, its set-up (once per
// device and context), its launch.
bool token_attention_tensor(const dcn_paged_cache &c, const dcn_token_attention_args &a);
size_t token_attention_tensor_workspace(const dcn_paged_cache &c, const dcn_token_attention_args &a);
cudaError_t token_attention_prepare_device();
cudaError_t launch_token_attention_tensor(const AttentionParams &p, void *workspace, int sm_count, uint32_t *err,
                                          cudaStream_t stream);

#if defined(__CUDACC__)

// ---- elements ------------------------------------------------------------------------

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// VEC elements as one load or store: 16 bytes, or a single element.
template <typename T, int VEC>
struct alignas(VEC == 1 ? sizeof(T) : 16) Pack {
    static_assert(VEC == 1 || VEC * sizeof(T) == 16, "a pack is one element or 16 bytes");
    T e[VEC];
};

template <typename T>
constexpr int kVec = static_cast<int>(16 / sizeof(T));

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC> &p, float (&v)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = to_float<T>(p.e[i]);
}

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const float (&v)[VEC]) {
    Pack<T, VEC> p;
#pragma unroll
    for (int i = 0; i < VEC; ++i) p.e[i] = from_float<T>(v[i]);
    return p;
}

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T *p) {
    return *reinterpret_cast<const Pack<T, VEC> *>(p);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, VEC> &v) {
    *reinterpret_cast<Pack<T, VEC> *>(p) = v;
}

// ---- streams ---------------------------------------------------------------------------

// The stream that holds `token`: how many of starts[1..streams] are at or below it.  Called by a
// whole warp; returns `streams` for a token past the last stream's.  One 32-wide load per 32
// streams instead of a chain of dependent loads.
__device__ __forceinline__ int find_stream(const int32_t *starts, int streams, int64_t token) {
    const int lane = threadIdx.x & 31;
    int below = 0;
    for (int b = 0; b < streams; b += 32) {
        const bool at_or_below = b + lane < streams && starts[b + lane + 1] <= token;
        below += __popc(__ballot_sync(0xffffffffu, at_or_below));
    }
    return below;
}

#endif  // __CUDACC__

}  // namespace dcn
