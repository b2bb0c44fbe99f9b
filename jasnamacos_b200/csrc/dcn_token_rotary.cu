// dcn_token_rotary.cu -- rotary positions over three axes, and the append of a step's keys and
// values to a paged cache with that rotation on the way.
//
// Pair j of token t turns by theta = positions[t][axis(j)] frequencies[j]:
//   (a, b) -> (a cos theta - b sin theta, a sin theta + b cos theta).
//
// What bounds it is memory: every element is read once and written once, with a handful of
// multiplications.  The angles do not depend on the head, so a block takes a few tokens, forms
// their cosines and sines once in shared memory and applies them to all heads of queries and keys;
// values ride along.  Angles are reduced in FP64 (a time position of some thousands times a
// frequency near one leaves FP32 only a few digits behind the point).
#include "dcn_tokens.cuh"

namespace dcn {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;   // head_dim <= 512
constexpr int kMaxTokens = 8;    // tokens a block

__device__ __forceinline__ float2 unit_of_angle(double theta) {
    constexpr double kTwoPi = 6.283185307179586476925286766559;
    constexpr double kTwoPiRest = 2.4492935982947064e-16;  // 2 pi - kTwoPi
    const double turns = rint(theta * (1.0 / kTwoPi));
    const double r = fma(-turns, kTwoPiRest, fma(-turns, kTwoPi, theta));
    float2 u;
    sincosf(static_cast<float>(r), &u.y, &u.x);
    return u;
}

struct Place {
    int32_t page, slot;  // page < 0: nowhere
};

// VEC > 1: a unit of work is a 16-byte pack of a head (interleaved pairs, unrotated elements) or
// two packs P elements apart (split pairs).  VEC == 1: a unit is a pair, or an unrotated element.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) rotate_kernel(const RotateParams p, int tokens_per_block) {
    extern __shared__ float2 turn[];  // [tokens_per_block][P]
    __shared__ Place place[kMaxTokens];
    const int pairs = p.rotation.pairs[0] + p.rotation.pairs[1] + p.rotation.pairs[2];
    const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens_per_block;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(tokens_per_block), p.tokens - first));

    if (p.streams > 0) {
        for (int t = threadIdx.x >> 5; t < tokens; t += kThreads / 32) {
            const int64_t token = first + t;
            const int b = find_stream(p.starts, p.streams, token);
            if ((threadIdx.x & 31) == 0) {
                Place where{-1, 0};
                if (b < p.streams) {
                    const int64_t position = static_cast<int64_t>(p.lengths[b]) - p.starts[b + 1] + token;
                    const int64_t column = position / p.page_size;
                    if (position >= 0 && column < p.table_columns) {
                        const int32_t page = p.table[b * p.table_stride + column];
                        if (page >= 0 && page < p.pages)
                            where = Place{page, static_cast<int32_t>(position - column * p.page_size)};
                    }
                }
                place[t] = where;
            }
        }
    }
    for (int i = threadIdx.x; i < tokens * pairs; i += kThreads) {
        const int t = i / pairs, j = i - t * pairs;
        const int axis = j < p.rotation.pairs[0] ? 0 : j < p.rotation.pairs[0] + p.rotation.pairs[1] ? 1 : 2;
        turn[i] = unit_of_angle(static_cast<double>(p.rotation.positions[(first + t) * 3 + axis]) *
                                p.rotation.frequencies[j]);
    }
    __syncthreads();

    const bool interleaved = p.rotation.interleaved != 0;
    const int rotated_units = VEC == 1      ? p.head_dim - pairs
                              : interleaved ? p.head_dim / VEC
                                            : p.head_dim / VEC - pairs / VEC;
    for (int part = 0; part < p.parts; ++part) {
        const HeadCopy &c = p.part[part];
        const bool rotate = c.rotate && pairs > 0;
        const int head_units = rotate ? rotated_units : p.head_dim / VEC;
        const int token_units = head_units * c.heads;
        for (int i = threadIdx.x; i < tokens * token_units; i += kThreads) {
            const int t = i / token_units, in_token = i - t * token_units;
            const int head = in_token / head_units, unit = in_token - head * head_units;
            const T *src = static_cast<const T *>(c.src) + (first + t) * c.src_token + head * c.src_head;
            T *dst = static_cast<T *>(c.dst) + head * c.dst_head;
            if (c.to_cache) {
                if (place[t].page < 0) continue;
                dst += place[t].page * c.dst_page + place[t].slot * c.dst_slot;
            } else {
                dst += (first + t) * c.dst_token;
            }
            const float2 *u = turn + t * pairs;
            if (!rotate) {
                store_pack<T, VEC>(dst + unit * VEC, load_pack<T, VEC>(src + unit * VEC));
            } else if (VEC > 1 && interleaved) {
                float v[VEC];
                const int e = unit * VEC;
                unpack<T, VEC>(load_pack<T, VEC>(src + e), v);
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
                    if ((e + j) / 2 < pairs) {
                        const float2 w = u[(e + j) / 2];
                        const float a = v[j], b = v[j + 1 < VEC ? j + 1 : 0];
                        v[j] = a * w.x - b * w.y;
                        v[j + 1 < VEC ? j + 1 : 0] = a * w.y + b * w.x;
                    }
                }
                store_pack<T, VEC>(dst + e, pack<T, VEC>(v));
            } else if (unit * VEC < pairs) {
                const int e = unit * VEC;
                const int ea = VEC == 1 && interleaved ? 2 * e : e, eb = VEC == 1 && interleaved ? 2 * e + 1 : e + pairs;
                float a[VEC], b[VEC];
                unpack<T, VEC>(load_pack<T, VEC>(src + ea), a);
                unpack<T, VEC>(load_pack<T, VEC>(src + eb), b);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float2 w = u[e + j];
                    const float x = a[j];
                    a[j] = x * w.x - b[j] * w.y;
                    b[j] = x * w.y + b[j] * w.x;
                }
                store_pack<T, VEC>(dst + ea, pack<T, VEC>(a));
                store_pack<T, VEC>(dst + eb, pack<T, VEC>(b));
            } else {
                const int e = unit * VEC + pairs;  // past both halves of the rotated elements
                store_pack<T, VEC>(dst + e, load_pack<T, VEC>(src + e));
            }
        }
    }
}

template <typename T>
bool vectorised(const RotateParams &p) {
    constexpr int V = kVec<T>;
    const int pairs = p.rotation.pairs[0] + p.rotation.pairs[1] + p.rotation.pairs[2];
    if (p.head_dim % V != 0 || (!p.rotation.interleaved && pairs % V != 0)) return false;
    for (int i = 0; i < p.parts; ++i) {
        const HeadCopy &c = p.part[i];
        if (reinterpret_cast<uintptr_t>(c.src) % 16 != 0 || reinterpret_cast<uintptr_t>(c.dst) % 16 != 0) return false;
        const int64_t strides[] = {c.src_token, c.src_head, c.dst_token, c.dst_head, c.dst_page, c.dst_slot};
        for (int64_t s : strides)
            if (s % V != 0) return false;
    }
    return true;
}

template <typename T>
cudaError_t launch_typed(const RotateParams &p, cudaStream_t stream) {
    const int pairs = p.rotation.pairs[0] + p.rotation.pairs[1] + p.rotation.pairs[2];
    // Enough tokens a block to give its threads a few packs each, but never so many that the SMs idle.
    int tokens = kMaxTokens;
    while (tokens > 1 && p.tokens < static_cast<int64_t>(tokens) * 2 * 148) tokens /= 2;
    const int64_t blocks = (p.tokens + tokens - 1) / tokens;
    const size_t smem = static_cast<size_t>(tokens) * pairs * sizeof(float2);
    if (vectorised<T>(p))
        rotate_kernel<T, kVec<T>><<<static_cast<unsigned>(blocks), kThreads, smem, stream>>>(p, tokens);
    else
        rotate_kernel<T, 1><<<static_cast<unsigned>(blocks), kThreads, smem, stream>>>(p, tokens);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_token_rotate(dcn_dtype dtype, const RotateParams &p, cudaStream_t stream) {
    switch (dtype) {
    case DCN_DTYPE_F16: return launch_typed<__half>(p, stream);
    case DCN_DTYPE_BF16: return launch_typed<__nv_bfloat16>(p, stream);
    default: return launch_typed<float>(p, stream);
    }
}

}  // namespace dcn
