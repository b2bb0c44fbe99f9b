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

// The sum of a team's values, in every thread of it: NT threads, one warp or NT / 32 whole warps
// with the named barrier `team + 1` and the scratch of their own.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float *scratch, int team) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (NT == 32) return v;
    const int warp = (threadIdx.x % NT) >> 5;
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(NT) : "memory");  // the previous sum has been read
    if ((threadIdx.x & 31) == 0) scratch[warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(NT) : "memory");
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) s += scratch[w];  // in a fixed order
    return s;
}

template <typename T, int VEC, int NT, int NV>
struct Row {
    float v[NV][VEC];

    // x <- N(x) over `width` elements.  Places past the width hold 0.
    __device__ __forceinline__ void normalise(int kind, int width, float epsilon, int lane, float *scratch,
                                              int team) {
        const float inv = 1.0f / static_cast<float>(width);
        if (kind == DCN_NORM_LAYER) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < VEC; ++j) s += v[i][j];
            const float mean = row_sum<NT>(s, scratch, team) * inv;
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
        const float r = rsqrtf(fmaf(row_sum<NT>(s, scratch, team), inv, epsilon));
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[i][j] *= r;
    }
};

// NT threads (a team) hold a row, NV packs of VEC elements each: pack i of thread t covers elements
// [(i NT + t) VEC, ...).  A block has kTeams teams and takes `block_rows` rows one after another.
//
// Shared: the vectors of a modulation group are folded once into FP32 vectors in shared memory --
//   gate, w (1 + scale), b (1 + scale) + shift, and the post norm's two -- and all of the block's rows of
// that group read them there.  A row then costs its own loads and stores, three 16-byte shared loads per
// four elements and some ten instructions an element; without it each row converts and combines up to
// seven vectors anew, and that, not memory, is what it takes its time on.
constexpr int kCoefficients = 5;
enum { kGate = 0, kScale, kShift, kPostWeight, kPostBias };

template <typename T, int VEC, int NT, int NV, int kTeams, bool Shared>
__global__ void __launch_bounds__(NT *kTeams) token_norm_kernel(const dcn_token_norm_args a, int block_rows) {
    extern __shared__ float folded[];  // [kCoefficients][width], where Shared
    __shared__ float scratch_of[kTeams][NT / 32];
    const int lane = threadIdx.x % NT, team = threadIdx.x / NT;
    float *scratch = scratch_of[team];
    const int width = a.width;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * block_rows;
    const int64_t end = min(first + block_rows, a.rows);

    auto at = [&](const void *base, int64_t offset) { return static_cast<const T *>(base) + offset; };
    auto vector = [&](const void *base, int64_t offset, float (&v)[VEC], float otherwise) {
        if (base) {
            unpack<T, VEC>(load_pack<T, VEC>(at(base, offset)), v);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = otherwise;
        }
    };
    const bool has_gate = a.gate, has_scale = a.weight || a.scale, has_shift = a.bias || a.shift;

    for (int64_t segment = first; segment < end;) {
        const int64_t g = segment / a.group;
        const int64_t segment_end = Shared ? min((g + 1) * a.group, end) : end;
        if (Shared) {
            __syncthreads();
            for (int c = threadIdx.x; c < width; c += NT * kTeams) {
                auto one = [&](const void *base, int64_t offset, float otherwise) {
                    return base ? to_float<T>(*at(base, offset + c)) : otherwise;
                };
                const float scale = 1.0f + one(a.scale, g * a.scale_stride, 0.0f);
                folded[kGate * width + c] = one(a.gate, g * a.gate_stride, 1.0f);
                folded[kScale * width + c] = one(a.weight, 0, 1.0f) * scale;
                folded[kShift * width + c] = one(a.bias, 0, 0.0f) * scale + one(a.shift, g * a.shift_stride, 0.0f);
                if (a.post) {
                    folded[kPostWeight * width + c] = one(a.post_weight, 0, 1.0f);
                    folded[kPostBias * width + c] = one(a.post_bias, 0, 0.0f);
                }
            }
            __syncthreads();
        }
        auto coefficient = [&](int which, int c, float (&v)[VEC]) {
            if (VEC % 4 == 0) {
#pragma unroll
                for (int j = 0; j < VEC; j += 4)
                    *reinterpret_cast<float4 *>(v + j) = *reinterpret_cast<const float4 *>(folded + which * width + c + j);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = folded[which * width + c + j];
            }
        };
        for (int64_t row = segment + team; row < segment_end; row += kTeams) {
            const int64_t group = Shared ? g : row / a.group;
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
                    x.normalise(a.kind, width, a.epsilon, lane, scratch, team);
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const int c = (i * NT + lane) * VEC;
                        if (c < width) {
                            float w[VEC], b[VEC];
                            if (Shared) {
                                coefficient(kPostWeight, c, w);
                                coefficient(kPostBias, c, b);
                            } else {
                                vector(a.post_weight, c, w, 1.0f);
                                vector(a.post_bias, c, b, 0.0f);
                            }
#pragma unroll
                            for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(x.v[i][j], w[j], b[j]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = (i * NT + lane) * VEC;
                    if (c < width) {
                        float m[VEC], r[VEC];
                        unpack<T, VEC>(rp[i], r);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) r[j] *= a.residual_scale;
                        if (has_gate) {
                            if (Shared) coefficient(kGate, c, m);
                            else vector(a.gate, group * a.gate_stride + c, m, 1.0f);
#pragma unroll
                            for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(x.v[i][j], m[j], r[j]);
                        } else {
#pragma unroll
                            for (int j = 0; j < VEC; ++j) x.v[i][j] += r[j];
                        }
                        if (a.hidden)
                            store_pack<T, VEC>(static_cast<T *>(a.hidden) + row * a.hidden_stride + c, pack<T, VEC>(x.v[i]));
                    }
                }
            }
            if (a.out == nullptr) continue;
            x.normalise(a.kind, width, a.epsilon, lane, scratch, team);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * NT + lane) * VEC;
                if (c < width) {
                    float w[VEC], b[VEC];
                    if (Shared) {
                        if (has_scale) {
                            coefficient(kScale, c, w);
#pragma unroll
                            for (int j = 0; j < VEC; ++j) x.v[i][j] *= w[j];
                        }
                        if (has_shift) {
                            coefficient(kShift, c, b);
#pragma unroll
                            for (int j = 0; j < VEC; ++j) x.v[i][j] += b[j];
                        }
                    } else {
                        vector(a.weight, c, w, 1.0f);
                        vector(a.bias, c, b, 0.0f);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(x.v[i][j], w[j], b[j]);
                        if (a.scale || a.shift) {
                            vector(a.scale, group * a.scale_stride + c, w, 0.0f);
                            vector(a.shift, group * a.shift_stride + c, b, 0.0f);
#pragma unroll
                            for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(x.v[i][j], w[j], x.v[i][j]) + b[j];
                        }
                    }
                    store_pack<T, VEC>(static_cast<T *>(a.out) + row * a.out_stride + c, pack<T, VEC>(x.v[i]));
                }
            }
        }
        segment = segment_end;
    }
}

constexpr int kSharedRows = 64;  // rows a block takes where it folds the vectors

template <typename T, int VEC, int NT, int NV, int kTeams>
cudaError_t launch(const dcn_token_norm_args &a, cudaStream_t stream) {
    // Folding pays where a block's rows are mostly of one group and there are enough rows for every SM
    // to have some blocks; it needs its vectors in the 48 KB every block may have.
    const size_t smem = static_cast<size_t>(kCoefficients) * a.width * sizeof(float);
    const bool folds = a.weight || a.bias || a.scale || a.shift || a.gate || a.post;
    if (folds && a.group >= kSharedRows / 2 && a.rows >= kSharedRows * 296 && smem <= 48 * 1024) {
        const unsigned blocks = static_cast<unsigned>((a.rows + kSharedRows - 1) / kSharedRows);
        token_norm_kernel<T, VEC, NT, NV, kTeams, true><<<blocks, NT * kTeams, smem, stream>>>(a, kSharedRows);
    } else {
        // One row a team.  Few rows: one team a block, so that they spread over the SMs.
        if (kTeams > 1 && a.rows < 148 * kTeams)
            token_norm_kernel<T, VEC, NT, NV, 1, false><<<static_cast<unsigned>(a.rows), NT, 0, stream>>>(a, 1);
        else
            token_norm_kernel<T, VEC, NT, NV, kTeams, false>
                <<<static_cast<unsigned>((a.rows + kTeams - 1) / kTeams), NT * kTeams, 0, stream>>>(a, kTeams);
    }
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
        if (packs <= 32) return launch<T, V, 32, 1, 8>(a, stream);
        if (packs <= 64) return launch<T, V, 32, 2, 8>(a, stream);
        if (packs <= 128) return launch<T, V, 32, 4, 8>(a, stream);
        if (packs <= 512) return launch<T, V, 128, 4, 2>(a, stream);
        return launch<T, V, 512, 4, 1>(a, stream);
    }
    if (a.width <= 256) return launch<T, 1, 32, 8, 8>(a, stream);
    if (a.width <= 2048) return launch<T, 1, 256, 8, 1>(a, stream);
    return launch<T, 1, 512, 16, 1>(a, stream);
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
