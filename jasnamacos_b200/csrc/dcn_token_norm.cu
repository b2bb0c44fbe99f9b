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
// with the named barrier `team + 1` and scratch of their own.  `scratch` has two halves that take turns: a
// thread that is at the next sum but one has passed the barrier after all threads read this one.
template <int NT>
__device__ __forceinline__ float row_sum(float v, float *&scratch, int team) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (NT == 32) return v;
    const int warp = (threadIdx.x % NT) >> 5;
    if ((threadIdx.x & 31) == 0) scratch[warp] = v;
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(NT) : "memory");
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) s += scratch[w];  // in a fixed order
    const uint32_t half = NT / 32 * sizeof(float);
    scratch = reinterpret_cast<float *>(reinterpret_cast<uintptr_t>(scratch) ^ half);
    return s;
}

template <typename T, int VEC, int NT, int NV>
struct Row {
    float v[NV][VEC];

    // x <- N(x) over `width` elements.  Places past the width hold 0.
    __device__ __forceinline__ void normalise(int kind, int width, float epsilon, int lane, float *&scratch,
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

// The kernel for any row.  NT threads (a team) hold it, NV packs of VEC elements each: pack i of thread t
// covers elements [(i NT + t) VEC, ...).  A block has kTeams teams, one row each.
template <typename T, int VEC, int NT, int NV, int kTeams>
__global__ void __launch_bounds__(NT *kTeams) token_norm_kernel(const __grid_constant__ dcn_token_norm_args a) {
    __shared__ __align__(2 * NT / 32 * sizeof(float)) float scratch_of[kTeams][2 * NT / 32];
    const int lane = threadIdx.x % NT, team = threadIdx.x / NT;
    float *scratch = scratch_of[team];
    const int width = a.width;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + team;
    if (row >= a.rows) return;
    const int64_t group = row / a.group;

    auto at = [&](const void *base, int64_t offset) { return static_cast<const T *>(base) + offset; };
    auto vector = [&](const void *base, int64_t offset, float (&v)[VEC], float otherwise) {
        if (base) {
            unpack<T, VEC>(load_pack<T, VEC>(at(base, offset)), v);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = otherwise;
        }
    };
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
                    vector(a.post_weight, c, w, 1.0f);
                    vector(a.post_bias, c, b, 0.0f);
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
                vector(a.gate, group * a.gate_stride + c, m, 1.0f);
                unpack<T, VEC>(rp[i], r);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(x.v[i][j], m[j], r[j] * a.residual_scale);
                if (a.hidden)
                    store_pack<T, VEC>(static_cast<T *>(a.hidden) + row * a.hidden_stride + c, pack<T, VEC>(x.v[i]));
            }
        }
    }
    if (a.out == nullptr) return;
    x.normalise(a.kind, width, a.epsilon, lane, scratch, team);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * NT + lane) * VEC;
        if (c < width) {
            float w[VEC], b[VEC];
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
            store_pack<T, VEC>(static_cast<T *>(a.out) + row * a.out_stride + c, pack<T, VEC>(x.v[i]));
        }
    }
}

// The kernel for many rows of up to 128 packs that share their modulation.  A warp holds a row.
//
// The vectors of a modulation group are folded once a block into FP32 vectors in shared memory -- gate,
// w (1 + scale), b (1 + scale) + shift, the post norm's two -- and all of the block's rows of the group read
// them there; converting and combining up to seven vectors anew for each row takes longer than the row's
// memory traffic.  A warp's next row lands in shared memory by bulk copies while it works on this one,
// which costs it no registers.
enum { kGate = 0, kScale, kShift, kPostWeight, kPostBias };

// Where folding pays: a group's rows are worth its fold, and the whole is long enough to hide the blocks' start.
// With a residual, FP16, folded and not (us): 61,440 rows of 1,024 in groups of 8 rows 148 and 154 (without a
// residual 101 and 90), of 16 118 and 148, of 256 86 and 141; rows of 256 in groups of 32 31 and 30, of 64 27 and
// 30.  Groups of 256: 4,096 rows of 1,024 11.4 and 17.1, of 512 6.9 and 6.4; 9,472 of 512 9.7 and 12.5.
constexpr int64_t kFoldedPacks = 512 * 1024;  // 16-byte packs of a tensor
constexpr int64_t kFoldedGroupPacks = 2048;   // and of a group
constexpr int kStages = 2;       // rows of a warp in shared memory
constexpr int kFoldedBytes = 112 * 1024;  // shared memory of a block: two an SM

// (Registers for two blocks of 12 warps an SM; blocks of 6 leave room for more by themselves.)
template <typename T, int NV, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps == 12 ? 2 : 0)
token_norm_folded_kernel(const __grid_constant__ dcn_token_norm_args a, int block_rows, uint32_t *err) {
    constexpr int VEC = kVec<T>;
    extern __shared__ float4 raw[];
    __shared__ uint64_t landed[kWarps][kStages];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int width = a.width, bytes = width * static_cast<int>(sizeof(T));
    const int coefficients = a.post ? 5 : 3, tensors = a.residual ? 2 : 1;
    float *folded = reinterpret_cast<float *>(raw);  // [coefficients][width]
    uint8_t *rows = reinterpret_cast<uint8_t *>(folded + coefficients * width) + warp * kStages * tensors * bytes;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * block_rows;
    const int64_t end = min(first + block_rows, a.rows);

    auto at = [&](const void *base, int64_t offset) { return static_cast<const T *>(base) + offset; };
    auto fetch = [&](int64_t row, int stage) {  // one lane's call
        uint8_t *to = rows + stage * tensors * bytes;
        mbar_arrive_expect_tx(&landed[warp][stage], tensors * bytes);
        bulk_copy_g2s(to, at(a.x, row * a.x_stride), bytes, &landed[warp][stage]);
        if (a.residual) bulk_copy_g2s(to + bytes, at(a.residual, row * a.residual_stride), bytes, &landed[warp][stage]);
    };
    int64_t row = first + warp;
    if (lane == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(&landed[warp][s], 1);
        fence_mbarrier_init();
        for (int s = 0; s < kStages; ++s)
            if (row + s * kWarps < end) fetch(row + s * kWarps, s);
    }
    __syncwarp();
    // Where element c of a folded vector lies.  A lane reads eight in a row as two float4: the first four of
    // every eight come before all the others, or the reads of a warp, 32 bytes apart, would meet in half
    // of the banks.
    auto place = [&](int c) { return VEC == 8 ? (c & 4) * (width / 8) + (c >> 3) * 4 + (c & 3) : c; };
    auto coefficient = [&](int which, int c, float (&v)[VEC]) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4)
            *reinterpret_cast<float4 *>(v + j) = *reinterpret_cast<const float4 *>(folded + which * width + place(c + j));
    };
    bool ok = true;
    float *scratch = nullptr;  // a row is one warp's
    int stage = 0;
    uint32_t parity = 0;
    for (int64_t segment = first; segment < end;) {
        const int64_t g = segment / a.group;
        const int64_t segment_end = min((g + 1) * a.group, end);
        __syncthreads();
        for (int c = threadIdx.x; c < width; c += 32 * kWarps) {
            auto one = [&](const void *base, int64_t offset, float otherwise) {
                return base ? to_float<T>(*at(base, offset + c)) : otherwise;
            };
            const float scale = 1.0f + one(a.scale, g * a.scale_stride, 0.0f);
            folded[kGate * width + place(c)] = one(a.gate, g * a.gate_stride, 1.0f);
            folded[kScale * width + place(c)] = one(a.weight, 0, 1.0f) * scale;
            folded[kShift * width + place(c)] = one(a.bias, 0, 0.0f) * scale + one(a.shift, g * a.shift_stride, 0.0f);
            if (a.post) {
                folded[kPostWeight * width + place(c)] = one(a.post_weight, 0, 1.0f);
                folded[kPostBias * width + place(c)] = one(a.post_bias, 0, 0.0f);
            }
        }
        __syncthreads();
        for (; row < segment_end; row += kWarps) {
            if (ok) ok = __all_sync(0xffffffffu, mbar_wait_bounded(&landed[warp][stage], parity, nullptr));
            if (!ok) {
                if (lane == 0) atomicOr(err, kErrWaitTimeout);
                continue;
            }
            const T *here = reinterpret_cast<const T *>(rows + stage * tensors * bytes);
            Row<T, VEC, 32, NV> x;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 32 + lane) * VEC;
#pragma unroll
                for (int j = 0; j < VEC; ++j) x.v[i][j] = 0.0f;
                if (c < width) unpack<T, VEC>(load_pack<T, VEC>(here + c), x.v[i]);
            }
            if (a.residual) {
                if (a.post) {
                    x.normalise(a.kind, width, a.epsilon, lane, scratch, 0);
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const int c = (i * 32 + lane) * VEC;
                        if (c < width) {
                            float w[VEC], b[VEC];
                            coefficient(kPostWeight, c, w);
                            coefficient(kPostBias, c, b);
#pragma unroll
                            for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(x.v[i][j], w[j], b[j]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int c = (i * 32 + lane) * VEC;
                    if (c < width) {
                        float m[VEC], r[VEC];
                        unpack<T, VEC>(load_pack<T, VEC>(here + width + c), r);
                        coefficient(kGate, c, m);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(x.v[i][j], m[j], r[j] * a.residual_scale);
                        if (a.hidden)
                            store_pack<T, VEC>(static_cast<T *>(a.hidden) + row * a.hidden_stride + c, pack<T, VEC>(x.v[i]));
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && row + kStages * kWarps < end) fetch(row + kStages * kWarps, stage);
            if (++stage == kStages) {
                stage = 0;
                parity ^= 1u;
            }
            if (a.out == nullptr) continue;
            x.normalise(a.kind, width, a.epsilon, lane, scratch, 0);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 32 + lane) * VEC;
                if (c < width) {
                    float w[VEC], b[VEC];
                    coefficient(kScale, c, w);
                    coefficient(kShift, c, b);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) x.v[i][j] = fmaf(x.v[i][j], w[j], b[j]);
                    store_pack<T, VEC>(static_cast<T *>(a.out) + row * a.out_stride + c, pack<T, VEC>(x.v[i]));
                }
            }
        }
        segment = segment_end;
    }
    if (!ok) {  // the rows under way may still land: not in another block's memory
        static_assert(kStages == 2, "the other stage and its parity");
        mbar_wait_bounded(&landed[warp][stage], parity, nullptr);
        mbar_wait_bounded(&landed[warp][stage ^ 1], parity ^ static_cast<uint32_t>(stage), nullptr);
    }
}

template <typename T, int VEC, int NT, int NV, int kTeams>
cudaError_t launch(const dcn_token_norm_args &a, cudaStream_t stream) {
    // Few rows: one team a block, so that they spread over the SMs.
    if (kTeams > 1 && a.rows < 148 * kTeams)
        token_norm_kernel<T, VEC, NT, NV, 1><<<static_cast<unsigned>(a.rows), NT, 0, stream>>>(a);
    else
        token_norm_kernel<T, VEC, NT, NV, kTeams>
            <<<static_cast<unsigned>((a.rows + kTeams - 1) / kTeams), NT * kTeams, 0, stream>>>(a);
    return cudaGetLastError();
}

// Shared memory of a block of the folded kernel.
size_t folded_bytes(const dcn_token_norm_args &a, size_t element, int warps) {
    return (a.post ? 5 : 3) * sizeof(float) * a.width + warps * kStages * (a.residual ? 2 : 1) * element * a.width;
}

template <typename T, int NV, int kWarps>
cudaError_t launch_folded(const dcn_token_norm_args &a, uint32_t *err, cudaStream_t stream) {
    // Even shares of the rows for the blocks that are on the GPU at once, two an SM, so that no round of blocks is left
    // half empty.  Long blocks pay their start once; of short ones, one folds while others stream.  61,440 rows of
    // 1,024 (us): with a residual 93.6 in one round of blocks, 90.0 in two, 85.6 in four; without 48.7, 48.6, 50.6;
    // with a post norm (blocks of 6 warps) 85.6, 95, 102.  Of 256, with a residual, 25.4 in one and 29.0 in four.
    const int64_t packs = kWarps != 12 ? 32768 : a.residual ? 8192 : 16384;  // a block
    const int64_t most = packs / (a.width / kVec<T>);
    const size_t smem = folded_bytes(a, sizeof(T), kWarps);
    const int64_t at_once = 148 * 2;
    const int64_t rounds = (a.rows + at_once * most - 1) / (at_once * most);
    const int64_t rows = (a.rows + at_once * rounds - 1) / (at_once * rounds);
    token_norm_folded_kernel<T, NV, kWarps><<<static_cast<unsigned>((a.rows + rows - 1) / rows), 32 * kWarps, smem, stream>>>(
        a, static_cast<int>(rows), err);
    return cudaGetLastError();
}

// Blocks of 12 warps where two fit an SM (blocks of 8 took 8 % longer for 61,440 rows of 1,024 FP16 elements with a
// residual), else of 6: with a post norm's vectors 12 leave room for one block.
template <typename T, int NV>
cudaError_t launch_folded(const dcn_token_norm_args &a, uint32_t *err, cudaStream_t stream) {
    return folded_bytes(a, sizeof(T), 12) <= kFoldedBytes ? launch_folded<T, NV, 12>(a, err, stream)
                                                         : launch_folded<T, NV, 6>(a, err, stream);
}

template <typename T, int NV>
cudaError_t prepare_folded() {
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void *>(token_norm_folded_kernel<T, NV, 12>),
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, kFoldedBytes);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(reinterpret_cast<const void *>(token_norm_folded_kernel<T, NV, 6>),
                                 cudaFuncAttributeMaxDynamicSharedMemorySize, kFoldedBytes);
    return e;
}

template <typename T>
cudaError_t prepare() {
    cudaError_t e = prepare_folded<T, 1>();
    if (e == cudaSuccess) e = prepare_folded<T, 2>();
    if (e == cudaSuccess) e = prepare_folded<T, 4>();
    return e;
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
cudaError_t launch_typed(const dcn_token_norm_args &a, uint32_t *err, cudaStream_t stream) {
    constexpr int V = kVec<T>;
    if (vectorised<T>(a)) {
        const int packs = a.width / V;
        if (packs <= 128 && a.group >= kFoldedGroupPacks / packs && a.rows * packs >= kFoldedPacks) {
            if (packs <= 32) return launch_folded<T, 1>(a, err, stream);
            if (packs <= 64) return launch_folded<T, 2>(a, err, stream);
            return launch_folded<T, 4>(a, err, stream);
        }
        if (packs <= 32) return launch<T, V, 32, 1, 8>(a, stream);
        // A row on four warps is the faster the fewer rows there are (2.0 against 3.0 us for 8 of 128 packs).
        if (packs <= 128 && a.rows < 148 * 8) return launch<T, V, 128, 1, 1>(a, stream);
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

cudaError_t token_norm_prepare_device() {
    cudaError_t e = prepare<float>();
    if (e == cudaSuccess) e = prepare<__half>();
    if (e == cudaSuccess) e = prepare<__nv_bfloat16>();
    return e;
}

cudaError_t launch_token_norm(const dcn_token_norm_args &a, uint32_t *err, cudaStream_t stream) {
    switch (a.dtype) {
    case DCN_DTYPE_F16: return launch_typed<__half>(a, err, stream);
    case DCN_DTYPE_BF16: return launch_typed<__nv_bfloat16>(a, err, stream);
    default: return launch_typed<float>(a, err, stream);
    }
}

}  // namespace dcn
