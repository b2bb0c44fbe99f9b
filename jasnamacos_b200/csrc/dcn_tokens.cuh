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

cudaError_t token_norm_prepare_device();  // set-up, once per device and context
cudaError_t launch_token_norm(const dcn_token_norm_args &a, uint32_t *err, cudaStream_t stream);

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

cudaError_t launch_token_rotate(dcn_dtype dtype, const RotateParams &p, uint32_t *err, cudaStream_t stream);

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

// The register type of one load or store of 2 to 16 bytes.
template <int Bytes>
struct Word;
template <>
struct Word<2> { using type = uint16_t; };
template <>
struct Word<4> { using type = uint32_t; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<16> { using type = uint4; };

// VEC elements as one load or store.
template <typename T, int VEC>
struct Pack {
    using W = typename Word<VEC * static_cast<int>(sizeof(T))>::type;
    W w;
};

template <typename T>
constexpr int kVec = static_cast<int>(16 / sizeof(T));

template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC> &p, float (&v)[VEC]) {
    union {
        typename Pack<T, VEC>::W w;
        uint16_t h[VEC];
        float f[VEC];
    } u;
    u.w = p.w;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = u.f[i];
        else if constexpr (__is_same(T, __half)) v[i] = __half2float(__ushort_as_half(u.h[i]));
        else v[i] = __uint_as_float(static_cast<uint32_t>(u.h[i]) << 16);
    }
}

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> pack(const float (&v)[VEC]) {
    union {
        typename Pack<T, VEC>::W w;
        uint16_t h[VEC];
        uint32_t hh[(VEC + 1) / 2];
        float f[VEC];
    } u;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) u.f[i] = v[i];
    } else if constexpr (VEC == 1) {
        const T t = from_float<T>(v[0]);
        u.h[0] = *reinterpret_cast<const uint16_t *>(&t);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            if constexpr (__is_same(T, __half)) {
                const __half2 t = __floats2half2_rn(v[i], v[i + 1]);
                u.hh[i / 2] = *reinterpret_cast<const uint32_t *>(&t);
            } else {
                const __nv_bfloat162 t = __floats2bfloat162_rn(v[i], v[i + 1]);
                u.hh[i / 2] = *reinterpret_cast<const uint32_t *>(&t);
            }
        }
    }
    Pack<T, VEC> p;
    p.w = u.w;
    return p;
}

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T *p) {
    Pack<T, VEC> v;
    v.w = *reinterpret_cast<const typename Pack<T, VEC>::W *>(p);
    return v;
}

template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, VEC> &v) {
    *reinterpret_cast<typename Pack<T, VEC>::W *>(p) = v.w;
}

// ---- streams ---------------------------------------------------------------------------

// The stream that holds `token`: the last one whose start is at or below it.  Called by a whole warp;
// returns `streams` for a token that no stream holds, past the last one's or before the first one's.
// One 32-wide load per 32 starts instead of a chain of dependent loads.
__device__ __forceinline__ int find_stream(const int32_t *starts, int streams, int64_t token) {
    const int lane = threadIdx.x & 31;
    int begun = 0;  // how many of starts[0..streams] are at or below the token
    for (int b = 0; b <= streams; b += 32) {
        const bool at_or_below = b + lane <= streams && starts[b + lane] <= token;
        begun += __popc(__ballot_sync(0xffffffffu, at_or_below));
    }
    return begun > 0 ? begun - 1 : streams;
}

#endif  // __CUDACC__

}  // namespace dcn
