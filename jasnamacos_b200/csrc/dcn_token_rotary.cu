// dcn_token_rotary.cu -- rotary positions over three axes, and the append of a step's keys and
// values to a paged cache with that rotation on the way.
//
// Pair j of token t turns by theta = positions[t][axis(j)] frequencies[j]:
//   (a, b) -> (a cos theta - b sin theta, a sin theta + b cos theta).
//
// What bounds it is memory: every element is read once and written once, with a handful of
// multiplications.  The angles do not depend on the head, so a block takes a few tokens, forms their
// cosines and sines once in shared memory and applies them to all heads of queries and keys.  Angles
// are reduced in FP64 (a time position of some thousands times a frequency near one leaves FP32 only a
// few digits behind the point).
//
// Two kernels.  Many rows on 16 bytes go through shared memory whole, by bulk copies both ways
// (rotate_rows_kernel): no thread spends registers or instructions on what is in flight.  Few rows, and
// others, are read by the threads (rotate_kernel).  BF16 queries of 30,720 tokens (16 heads of 128, 60
// pairs, 252 MB read and written): 44 us, 5.7 TB/s, against 82 us by the threads.
#include "dcn_tokens.cuh"

namespace dcn {
namespace {

constexpr int kUnroll = 4;       // tokens a thread has in flight
constexpr int kMaxTokens = 16;   // tokens a block
constexpr int kMaxThreads = 384;

// Fast: the hardware's sine and cosine, 2^-21 off at |r| <= pi, for outputs of 8 or 11 bits.
template <bool Fast>
__device__ __forceinline__ float2 unit_of_angle(double theta) {
    constexpr double kTwoPi = 6.283185307179586476925286766559;
    constexpr double kTwoPiRest = 2.4492935982947064e-16;  // 2 pi - kTwoPi
    const double turns = rint(theta * (1.0 / kTwoPi));
    const float r = static_cast<float>(fma(-turns, kTwoPiRest, fma(-turns, kTwoPi, theta)));
    float2 u;
    if (Fast) __sincosf(r, &u.y, &u.x);
    else sincosf(r, &u.y, &u.x);
    return u;
}

// N (cos, sin) from shared memory, two at a time (w on 16 bytes where N > 1).
template <int N>
__device__ __forceinline__ void load_turns(const float2 *w, float (&u)[2 * N]) {
    if (N % 2 == 0) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            const float4 v = *reinterpret_cast<const float4 *>(w + j);
            u[2 * j] = v.x;
            u[2 * j + 1] = v.y;
            u[2 * j + 2] = v.z;
            u[2 * j + 3] = v.w;
        }
    } else {
        const float2 v = *w;
        u[0] = v.x;
        u[1] = v.y;
    }
}

// Where a token's keys and values go in the cache (offsets in elements, -1: nowhere); nothing without a
// cache.  A whole warp's call.
__device__ __forceinline__ void find_places(const RotateParams &p, int64_t token, int lane, int64_t *key, int64_t *value) {
    if (p.streams == 0) return;
    const int b = find_stream(p.starts, p.streams, token);
    if (lane >= 2) return;
    int64_t at = -1;
    if (b < p.streams) {
        const int64_t position = static_cast<int64_t>(p.lengths[b]) - p.starts[b + 1] + token;
        const int64_t column = position / p.page_size;
        if (position >= 0 && column < p.table_columns) {
            const int32_t page = p.table[b * p.table_stride + column];
            const HeadCopy &c = p.part[p.parts - 2 + lane];  // keys, values
            if (page >= 0 && page < p.pages) at = page * c.dst_page + (position - column * p.page_size) * c.dst_slot;
        }
    }
    *(lane == 0 ? key : value) = at;
}

// A token's cosines and sines.  A whole warp's call.
template <bool Fast>
__device__ __forceinline__ void form_angles(const RotateParams &p, int64_t token, int lane, float2 *turn) {
    const int32_t *position = p.rotation.positions + token * 3;
    const int end0 = p.rotation.pairs[0], end1 = end0 + p.rotation.pairs[1], end2 = end1 + p.rotation.pairs[2];
    for (int j = lane; j < end2; j += 32) {
        const int axis = j < end0 ? 0 : j < end1 ? 1 : 2;
        turn[j] = unit_of_angle<Fast>(static_cast<double>(position[axis]) * p.rotation.frequencies[j]);
    }
}

// Pairs (x[j], y[j]) by (u[2j], u[2j+1]).
template <int VEC>
__device__ __forceinline__ void turn_split(float (&x)[VEC], float (&y)[VEC], const float (&u)[2 * VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        const float v = x[j];
        x[j] = v * u[2 * j] - y[j] * u[2 * j + 1];
        y[j] = v * u[2 * j + 1] + y[j] * u[2 * j];
    }
}

// Pairs (v[j], v[j+1]) among the first `count` elements by (u[j], u[j+1]).
template <int VEC>
__device__ __forceinline__ void turn_packed(float (&v)[VEC], const float (&u)[VEC], int count) {
#pragma unroll
    for (int j = 0; j < VEC; j += 2) {
        if (j < count) {
            const float x = v[j];
            v[j] = x * u[j] - v[j + 1] * u[j + 1];
            v[j + 1] = x * u[j + 1] + v[j + 1] * u[j];
        }
    }
}

// VEC > 1: a unit of work is a pack of a head (interleaved pairs, unrotated elements) or two packs P
// elements apart (split pairs).  VEC == 1: a unit is a pair, or an unrotated element.  A block takes some
// tokens of `parts` of the queries, keys and values.  A thread keeps its unit's place in the token and
// goes through the tokens with it, kUnroll loads in flight; where a token has fewer units than the block
// threads, several tokens go side by side.  (Finding head and element anew for each unit took 218
// instructions a unit, and they, not memory, were the bound.)  The first loads go out before the angles
// are formed, so that the latencies of positions, table and data overlap.
template <typename T, int VEC>
__global__ void __launch_bounds__(kMaxThreads) rotate_kernel(const __grid_constant__ RotateParams p, int tokens_per_block,
                                                            int parts) {
    extern __shared__ float4 turn_pairs[];  // [tokens of the block][pitch] (cos, sin), pitch even
    __shared__ int64_t place[2][kMaxTokens];  // keys' and values' offsets in the cache, -1: nowhere
    float2 *turn = reinterpret_cast<float2 *>(turn_pairs);
    const bool interleaved = p.rotation.interleaved != 0;
    const bool packed = VEC > 1 && interleaved;  // both elements of a pair lie in one pack
    const int pairs = p.rotation.pairs[0] + p.rotation.pairs[1] + p.rotation.pairs[2];
    const int pitch = (pairs + 1) & ~1;
    // How far a split pair's second element is from its first.
    const int apart = VEC == 1 && interleaved ? 1 : pairs;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens_per_block;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(tokens_per_block), p.tokens - first));
    const int threads = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int part0 = blockIdx.y * parts, part1 = min(part0 + parts, p.parts);

    // This thread's unit of the current part: its element, which tokens it takes (every `stride`-th from
    // `begin_token`), and its pointers there.
    bool rotate, split, to_cache;
    int e, begin_token, stride, per_token;
    int64_t src_token, dst_token;
    const T *src;
    T *dst;
    const int64_t *places;
    auto take = [&](int part, int begin) {
        const HeadCopy &c = p.part[part];
        rotate = c.rotate;
        to_cache = c.to_cache;
        src_token = c.src_token;
        dst_token = c.dst_token;
        places = place[part - (p.parts - 2) > 0 ? 1 : 0];
        const int per_head = rotate && !packed ? p.head_dim / VEC - pairs / VEC : p.head_dim / VEC;
        per_token = per_head * c.heads;
        stride = max(threads / per_token, 1);
        begin_token = stride > 1 ? threadIdx.x / per_token : 0;
        const int in_token = stride > 1 ? threadIdx.x - begin_token * per_token : begin + threadIdx.x;
        if (in_token >= per_token || begin_token >= stride) begin_token = tokens;  // no unit: no tokens
        const int head = in_token / per_head;
        e = (in_token - head * per_head) * VEC;
        split = rotate && !packed && e < pairs;
        // Split pairs come first, then the elements past both of their halves.
        if (rotate && !packed) e = e >= pairs ? e + pairs : VEC == 1 && interleaved ? 2 * e : e;
        src = static_cast<const T *>(c.src) + first * c.src_token + head * c.src_head + e;
        dst = static_cast<T *>(c.dst) + (to_cache ? 0 : first * c.dst_token) + head * c.dst_head + e;
    };
    Pack<T, VEC> a[kUnroll], b[kUnroll];
    auto load = [&](int t0) {
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            const int t = t0 + i * stride;
            if (t < tokens) {
                const T *from = src + t * src_token;
                a[i] = load_pack<T, VEC>(from);
                if (split) b[i] = load_pack<T, VEC>(from + apart);
            }
        }
    };
    auto store = [&](int t0) {
        const float2 *cs = turn + (interleaved ? e / 2 : e);  // the pack's first pair
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            const int t = t0 + i * stride;
            if (t >= tokens) break;
            const int64_t at = to_cache ? places[t] : t * dst_token;
            if (at < 0) continue;
            T *to = dst + at;
            const float2 *w = cs + t * pitch;
            if (split) {
                float x[VEC], y[VEC], u[2 * VEC];
                unpack<T, VEC>(a[i], x);
                unpack<T, VEC>(b[i], y);
                load_turns<VEC>(w, u);
                turn_split<VEC>(x, y, u);
                store_pack<T, VEC>(to, pack<T, VEC>(x));
                store_pack<T, VEC>(to + apart, pack<T, VEC>(y));
                continue;
            }
            if constexpr (VEC > 1) {
                if (rotate && packed && e < 2 * pairs) {
                    float v[VEC], u[VEC];
                    unpack<T, VEC>(a[i], v);
                    load_turns<VEC / 2>(w, u);
                    turn_packed<VEC>(v, u, 2 * pairs - e);
                    a[i] = pack<T, VEC>(v);
                }
            }
            store_pack<T, VEC>(to, a[i]);
        }
    };

    take(part0, 0);
    load(begin_token);
    for (int t = warp; t < tokens; t += threads / 32) {
        find_places(p, first + t, lane, place[0] + t, place[1] + t);
        form_angles<sizeof(T) == 2>(p, first + t, lane, turn + t * pitch);
    }
    __syncthreads();
    store(begin_token);
    int done = begin_token + kUnroll * stride;
    for (int part = part0; part < part1; ++part) {
        for (int begin = 0;;) {
            for (int t0 = done; t0 < tokens; t0 += kUnroll * stride) {
                load(t0);
                store(t0);
            }
            begin += threads;
            if (begin >= per_token) break;
            take(part, begin);
            done = begin_token;
        }
        if (part + 1 < part1) {
            take(part + 1, 0);
            done = begin_token;
        }
    }
}

// ---- rows through shared memory ------------------------------------------------------------

constexpr int kRowThreads = 128;
constexpr int kRowBytes = 32 * 1024;    // the longest rows of a token that are copied whole
constexpr int kBlockBytes = 24 * 1024;  // rows and angles of a block's tokens, where a token is shorter

struct RowsPlan {
    int tokens;       // tokens a block
    int pitch_bytes;  // a token's parts in shared memory, one after another
    int offset[3];    // of each part in it
    int rotated;      // heads to rotate: those of the first parts
};

// A block copies its tokens' rows in, rotates them where they lie, and copies them out.  VEC here only
// sizes the shared-memory accesses: 16 bytes, or as far as split pairs with an odd P allow.
template <typename T, int VEC>
__global__ void __launch_bounds__(kRowThreads) rotate_rows_kernel(const __grid_constant__ RotateParams p,
                                                                 const __grid_constant__ RowsPlan plan, uint32_t *err) {
    extern __shared__ uint8_t raw[];
    __shared__ uint64_t landed;
    __shared__ int64_t place[2][kMaxTokens];  // keys' and values' offsets in the cache, -1: nowhere
    uint8_t *rows = raw + (-smem_addr(raw) & 127);
    const int pairs = p.rotation.pairs[0] + p.rotation.pairs[1] + p.rotation.pairs[2];
    const int pitch = (pairs + 1) & ~1;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * plan.tokens;
    const int tokens = static_cast<int>(min(static_cast<int64_t>(plan.tokens), p.tokens - first));
    float2 *turn = reinterpret_cast<float2 *>(rows + plan.tokens * plan.pitch_bytes);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int head_bytes = p.head_dim * static_cast<int>(sizeof(T));

    if (threadIdx.x == 0) {
        mbar_init(&landed, 1);
        fence_mbarrier_init();
        mbar_arrive_expect_tx(&landed, tokens * plan.pitch_bytes);
    }
    __syncthreads();
    // A part of a token is one copy where its heads follow each other, else one for each head.
    if (warp == 0) {
        for (int i = 0; i < p.parts; ++i) {
            const HeadCopy &c = p.part[i];
            const int copies = c.src_head == p.head_dim ? 1 : c.heads, bytes = head_bytes * c.heads / copies;
            for (int n = lane; n < tokens * copies; n += 32) {
                const int t = n / copies, h = n - t * copies;
                bulk_copy_g2s(rows + t * plan.pitch_bytes + plan.offset[i] + h * bytes,
                              static_cast<const T *>(c.src) + (first + t) * c.src_token + h * c.src_head, bytes, &landed);
            }
        }
        __syncwarp();
    }
    for (int t = warp; t < tokens; t += kRowThreads / 32) {
        find_places(p, first + t, lane, place[0] + t, place[1] + t);
        form_angles<sizeof(T) == 2>(p, first + t, lane, turn + t * pitch);
    }
    __syncthreads();
    if (!mbar_wait_bounded(&landed, 0, nullptr)) {
        atomicOr(err, kErrWaitTimeout);
        mbar_wait_bounded(&landed, 0, nullptr);  // the copies may still land: not in another block's memory
        return;
    }

    const bool packed = VEC > 1 && p.rotation.interleaved;  // both elements of a pair lie in one pack
    const int apart = VEC == 1 && p.rotation.interleaved ? 1 : pairs;
    // Units that hold pairs; what lies past them stays.
    const int per_head = packed ? (2 * pairs + VEC - 1) / VEC : pairs / VEC;
    if (per_head > 0) {
        const int side = kRowThreads / per_head;  // heads at a time; 0: a head in several rounds
        const int first_unit = side > 0 ? threadIdx.x % per_head : threadIdx.x;
        const int first_row = side > 0 ? threadIdx.x / per_head : 0;
        for (int unit = first_unit; unit < per_head && first_row < max(side, 1); unit += side > 0 ? per_head : kRowThreads) {
            const int e = VEC == 1 && p.rotation.interleaved ? 2 * unit : unit * VEC;
            int t = first_row / plan.rotated, h = first_row - t * plan.rotated;
            while (t < tokens) {
                T *at = reinterpret_cast<T *>(rows + t * plan.pitch_bytes + h * head_bytes) + e;
                const float2 *w = turn + t * pitch + (p.rotation.interleaved ? e / 2 : e);
                if (!packed) {
                    float x[VEC], y[VEC], u[2 * VEC];
                    unpack<T, VEC>(load_pack<T, VEC>(at), x);
                    unpack<T, VEC>(load_pack<T, VEC>(at + apart), y);
                    load_turns<VEC>(w, u);
                    turn_split<VEC>(x, y, u);
                    store_pack<T, VEC>(at, pack<T, VEC>(x));
                    store_pack<T, VEC>(at + apart, pack<T, VEC>(y));
                } else if constexpr (VEC > 1) {
                    float v[VEC], u[VEC];
                    unpack<T, VEC>(load_pack<T, VEC>(at), v);
                    load_turns<VEC / 2>(w, u);
                    turn_packed<VEC>(v, u, 2 * pairs - e);
                    store_pack<T, VEC>(at, pack<T, VEC>(v));
                }
                h += max(side, 1);
                while (h >= plan.rotated) {
                    h -= plan.rotated;
                    ++t;
                }
            }
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    if (warp == 0) {
        for (int i = 0; i < p.parts; ++i) {
            const HeadCopy &c = p.part[i];
            const int copies = c.dst_head == p.head_dim ? 1 : c.heads, bytes = head_bytes * c.heads / copies;
            for (int n = lane; n < tokens * copies; n += 32) {
                const int t = n / copies, h = n - t * copies;
                const int64_t at = c.to_cache ? place[i - (p.parts - 2)][t] : (first + t) * c.dst_token;
                if (at >= 0)
                    bulk_copy_s2g(static_cast<T *>(c.dst) + at + h * c.dst_head,
                                  rows + t * plan.pitch_bytes + plan.offset[i] + h * bytes, bytes);
            }
        }
        bulk_copy_s2g_wait_read();
    }
}

// The largest pack that divides every row, pointer and stride, and (split pairs) P: 16 bytes down to one
// element.
template <typename T>
int pack_elements(const RotateParams &p) {
    const int pairs = p.rotation.pairs[0] + p.rotation.pairs[1] + p.rotation.pairs[2];
    uint64_t bits = p.head_dim;
    if (!p.rotation.interleaved) bits |= pairs;
    for (int i = 0; i < p.parts; ++i) {
        const HeadCopy &c = p.part[i];
        bits |= c.src_token | c.src_head | c.dst_token | c.dst_head | c.dst_page | c.dst_slot;
        bits |= (reinterpret_cast<uintptr_t>(c.src) | reinterpret_cast<uintptr_t>(c.dst)) / sizeof(T);
    }
    int elements = kVec<T>;
    while (bits % elements != 0) elements /= 2;
    return elements;
}

template <typename T, int VEC>
cudaError_t launch(const RotateParams &p, cudaStream_t stream) {
    const int pairs = p.rotation.pairs[0] + p.rotation.pairs[1] + p.rotation.pairs[2];
    const bool packed = VEC > 1 && p.rotation.interleaved;
    auto units = [&](const HeadCopy &c) {
        return c.heads * (c.rotate && !packed ? p.head_dim / VEC - pairs / VEC : p.head_dim / VEC);
    };
    // Threads a block: the size that its parts' units fill best, the smallest of equals.
    int threads = 128;
    double best = 0.0;
    for (int n = 128; n <= kMaxThreads; n += 32) {
        double wanted = 0.0, spent = 0.0;
        for (int i = 0; i < p.parts; ++i) {
            const int u = units(p.part[i]);
            wanted += u;
            spent += u <= n ? static_cast<double>(n) / (n / u) : static_cast<double>((u + n - 1) / n) * n;
        }
        if (wanted / spent > best + 0.01) {
            best = wanted / spent;
            threads = n;
        }
    }
    // Many tokens: a block takes all parts of some tokens and forms their angles once.  Few: a block for
    // each part of each token or two, so that more SMs share the latency.
    int tokens = kMaxTokens, parts = p.parts;
    while (tokens > 1 && p.tokens < static_cast<int64_t>(tokens) * 148 * 2) --tokens;
    if (tokens == 1) parts = 1;
    const dim3 grid(static_cast<unsigned>((p.tokens + tokens - 1) / tokens), (p.parts + parts - 1) / parts);
    // A last pack may begin before P and end past it: it reads, and does not use, what follows.
    const size_t smem = (static_cast<size_t>(tokens) * ((pairs + 1) & ~1) + VEC) * sizeof(float2);
    rotate_kernel<T, VEC><<<grid, threads, smem, stream>>>(p, tokens, parts);
    return cudaGetLastError();
}

// Whether every row may be copied whole, by 16 bytes; then fills the plan.
template <typename T>
bool plan_rows(const RotateParams &p, RowsPlan *plan) {
    constexpr int64_t V = kVec<T>;
    if (p.head_dim % V != 0) return false;
    *plan = RowsPlan{};
    for (int i = 0; i < p.parts; ++i) {
        const HeadCopy &c = p.part[i];
        if ((reinterpret_cast<uintptr_t>(c.src) | reinterpret_cast<uintptr_t>(c.dst)) % 16 != 0) return false;
        if ((c.src_token | c.src_head | c.dst_token | c.dst_head | c.dst_page | c.dst_slot) % V != 0) return false;
        plan->offset[i] = plan->pitch_bytes;
        const int64_t bytes = static_cast<int64_t>(c.heads) * p.head_dim * static_cast<int64_t>(sizeof(T));
        if (bytes > kRowBytes) return false;
        plan->pitch_bytes += static_cast<int>(bytes);
        if (c.rotate) plan->rotated += c.heads;
    }
    return plan->pitch_bytes <= kRowBytes;
}

template <typename T, int VEC>
cudaError_t launch_rows(const RotateParams &p, const RowsPlan &plan, uint32_t *err, cudaStream_t stream) {
    const int pairs = p.rotation.pairs[0] + p.rotation.pairs[1] + p.rotation.pairs[2];
    const size_t smem = static_cast<size_t>(plan.tokens) * plan.pitch_bytes + 128 +
                        (static_cast<size_t>(plan.tokens) * ((pairs + 1) & ~1) + VEC) * sizeof(float2);
    rotate_rows_kernel<T, VEC><<<static_cast<unsigned>((p.tokens + plan.tokens - 1) / plan.tokens), kRowThreads, smem, stream>>>(
        p, plan, err);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_typed(const RotateParams &p, uint32_t *err, cudaStream_t stream) {
    RowsPlan rows;
    const int elements = pack_elements<T>(p);
    // Staging a row costs two more steps, and pays from some 768 Ki packs on: with 16-byte packs 3.6 us
    // against 2.8 for 256 tokens of 16 heads of 128 (65,536 packs), 10.5 against 11.2 for 4,096.
    if (plan_rows<T>(p, &rows) && p.tokens * (rows.pitch_bytes / (elements * static_cast<int64_t>(sizeof(T)))) >= 786432) {
        const int pairs = p.rotation.pairs[0] + p.rotation.pairs[1] + p.rotation.pairs[2];
        // Blocks of this size, several an SM, hold more in flight than memory's latency needs; fewer tokens a
        // block where there are few.
        rows.tokens = kBlockBytes / (rows.pitch_bytes + (pairs + 1) * static_cast<int>(sizeof(float2)));
        if (rows.tokens < 1) rows.tokens = 1;
        if (rows.tokens > kMaxTokens) rows.tokens = kMaxTokens;
        while (rows.tokens > 1 && p.tokens < static_cast<int64_t>(rows.tokens) * 148 * 2) --rows.tokens;
        int in_rows = kVec<T>;
        while (!p.rotation.interleaved && pairs % in_rows != 0) in_rows /= 2;
        switch (in_rows) {
        case 8: return launch_rows<T, kVec<T>>(p, rows, err, stream);  // 16-bit types only
        case 4: return launch_rows<T, 4>(p, rows, err, stream);
        case 2: return launch_rows<T, 2>(p, rows, err, stream);
        default: return launch_rows<T, 1>(p, rows, err, stream);
        }
    }
    switch (elements) {
    case 8: return launch<T, kVec<T>>(p, stream);  // 16-bit types only
    case 4: return launch<T, 4>(p, stream);
    case 2: return launch<T, 2>(p, stream);
    default: return launch<T, 1>(p, stream);
    }
}

}  // namespace

cudaError_t launch_token_rotate(dcn_dtype dtype, const RotateParams &p, uint32_t *err, cudaStream_t stream) {
    switch (dtype) {
    case DCN_DTYPE_F16: return launch_typed<__half>(p, err, stream);
    case DCN_DTYPE_BF16: return launch_typed<__nv_bfloat16>(p, err, stream);
    default: return launch_typed<float>(p, err, stream);
    }
}

}  // namespace dcn
