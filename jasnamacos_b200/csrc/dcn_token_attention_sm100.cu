// dcn_token_attention_sm100.cu -- attention over a paged cache on the tensor cores (FP16, BF16;
// head_dim 64 and 128).
//
// For a row i of queries, over its visible keys s, in one pass with a running maximum m and sum l:
//   S = Q K^T            tcgen05.mma, Q and K tiles in shared memory, S in tensor memory
//   P = exp2(c S - c m + kRaise)  c = scale log2 e; a thread owns a row, so maximum and sum need no exchange
//   O += P V             tcgen05.mma, P (rounded to the element type) in tensor memory
//   out = O / l
//
// A tile is 128 rows by 128 keys.  A key head's q_heads / heads query heads read the same keys, so
// a tile's rows are (token, query head of that key head): 128 / ratio tokens.  A block runs two
// streams of tiles, each with its softmax warpgroup, and one warp that issues the products of both,
// so that one stream's exponentials run under the other's products:
//   shared: two row tiles against the same key tiles (steps of more than 128 rows);
//   split:  one row tile, each stream with its own range of key tiles (a few tokens).
// Keys are split further over blocks where rows alone do not fill the GPU; a second, dependent
// launch joins the parts.  Key tiles come by TMA, a box a page (or a power-of-two part of one), into a
// ring that is filled ahead across row blocks.
//
// Rounding P to the element type (as its values are the second product's operand) costs a weight a
// relative 2^-11 (FP16) or 2^-8 (BF16) at most, of the size of the result's own rounding; l sums the
// unrounded weights in FP32.  The maximum that P is taken against may lag the true one by up to
// 2^8 before O is rescaled, which spares almost every rescaling.  FP16 weights are taken 2^7 larger than
// that, up to 2^15 of its 65504: below 2^-21 of the maximum in use they are subnormal, to an absolute 2^-32 of
// it.  (Without, to 2^-25: of 262,143 weights of 2^-25.1 nothing was left in O, while l counted them.)
// The tensor core adds the products to O in FP32, each cut at 2^-25 of the sum it is added to: measured, beside one
// weight and value of 1 it keeps 97 % of FP16 weights of 2^-21.6, 73 % of 2^-24.5 and none of 2^-25.1; BF16 the same
// within its result's rounding.
//
// What bounds it, measured on one B200, a short burst of calls in a graph (in brackets one call of many back to
// back, where the 1 kW limit lowers the clock):
// - Four clips of 7,680 tokens (FP16, 16 query and 8 key heads of 128, a window of 8 frames of 256 and one that
//   stays): 490 to 497 us, 1,010 to 1,026 TFLOP/s (573 us, 877).  A pair of tiles takes some 3,600 cycles.  Its products
//   are 2,048 of them (512 for 128x128x128, measured alike with both operands in shared memory and with one in
//   tensor memory) and its exponentials 2,048 as well: neither unit is full, the two streams overlap in part.
// - Eight streams' frames of 256 tokens, head_dim 64: 50 us (51); 3,280 cycles a pair of tiles, 2,048 of them
//   exponentials, 1,024 products; the rest is the softmax warps' latency in this layout of two a scheduler.
// - 64 streams of one token over 4,160 keys (BF16, 32 and 8 heads of 128): 172 us, 5.98 TB/s (197, 5.2), memory.
// - Four streams of one token over up to 260 keys: 13.1 us, a chain of steps whose code each runs once.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <cfloat>
#include <mutex>

#include "dcn_token_attention.cuh"

namespace dcn {
namespace {

constexpr int kRows = 128;          // rows of a tile
constexpr int kKeys = 128;          // keys of a tile
constexpr int kSoftmaxWarps = 8;    // two warpgroups
constexpr int kThreads = 384;       // 2 softmax warpgroups, then a product, a scan and 2 load warps
constexpr int kTmemCols = 512;      // S0, S1 (128 each), O0, O1 (head_dim each), P0, P1
constexpr uint32_t kTmemO = 256;
constexpr uint32_t kTmemP = 384;    // P0, P1 of head_dim 64; of 128, where there is no room, P lies over S
constexpr float kLag = 8.0f;        // log2 of how far the maximum in use may lag
template <typename T>
constexpr float kRaise = __is_same(T, __half) ? 7.0f : 0.0f;  // log2 of what weights are larger by (BF16 has FP32's range)
constexpr int kSmCount = 148;
constexpr int64_t kMaxItems = int64_t{1} << 20;  // of a launch, where one stream's row blocks are what makes them many

template <int D, bool Shared>
struct Layout {
    static constexpr int kRings = Shared ? 1 : 2;
    static constexpr int kSlots = (Shared ? 5 : 3) * (D == 64 ? 2 : 1);  // tiles of a ring
    static constexpr int kTileBytes = kKeys * D * 2;
    static constexpr int kQTiles = Shared ? 2 : 1;
    // P in columns of its own: the next tile's scores are made as soon as this tile's have been read, while
    // their exponentials run, and no longer wait for the second product.
    static constexpr bool kApart = D == 64;
};

struct KernelParams {
    AttentionParams a;
    float *part_o;       // [parts][tokens][q_heads][head_dim] unnormalised O; null: write the result
    float2 *part_ml;     // [parts][tokens][q_heads] (c m - kRaise, l)
    uint32_t *err;
    int ratio;           // query heads of a key head
    int per_ratio;       // 2^16 / ratio, rounded up: r * per_ratio >> 16 is r / ratio for a tile's rows
    int tile_tokens;     // tokens of a row tile
    int row_blocks;      // row blocks of the longest step
    int splits;          // blocks that share one row block's keys
    int box_rows;        // keys of one TMA box
    int items;
    float c;             // |scale| log2 e
    int negate;          // scale < 0: scores change sign
};

// The keys that rows at positions p0 .. p1 (0 <= p0 <= p1) see: some row sees [0, pinned) and
// [low, high), cut to below high; every row sees [0, pinned) and [low_all, high_all), below high_all.
struct Span {
    int pinned, low, high, low_all, high_all;

    __device__ __forceinline__ void set(int p0, int p1, int length, const dcn_token_attention_args &a) {
        const uint32_t frame = a.frame;
        const int64_t f0 = static_cast<uint32_t>(p0) / frame, f1 = static_cast<uint32_t>(p1) / frame;
        const int64_t high0 = (f0 + 1) * a.frame, high1 = (f1 + 1) * a.frame;
        const int64_t low0 = (f0 - a.window + 1) * a.frame, low1 = (f1 - a.window + 1) * a.frame;
        high = static_cast<int>(min(high1, static_cast<int64_t>(length)));
        high_all = static_cast<int>(min(high0, static_cast<int64_t>(length)));
        low = static_cast<int>(max(low0, int64_t{0}));
        low_all = static_cast<int>(max(low1, int64_t{0}));
        pinned = static_cast<int>(min(static_cast<int64_t>(a.sinks) * a.frame, static_cast<int64_t>(length)));
    }
    __device__ __forceinline__ bool some(int key) const { return key < high && (key >= low || key < pinned); }
    __device__ __forceinline__ bool all(int key) const { return key < high_all && (key >= low_all || key < pinned); }
    __device__ __forceinline__ bool tile_some(int base) const {
        return base < high && (base + kKeys > low || base < pinned);
    }
    __device__ __forceinline__ bool tile_all(int base) const {
        return base + kKeys <= high_all && (base >= low_all || base + kKeys <= pinned);
    }
};

// One block's work for one of its two streams of tiles: the rows of a tile against a range of key
// tiles.  Every role walks the same sequence of items by itself.
struct Item {
    int stream, kv_head, start, steps, length;  // steps: the stream's tokens of this step
    int token0, token1;             // the tile's tokens in the step
    int first, last;                // range of the list of key tiles
    int both_last;                  // and the end of both streams' ranges
    int pinned_tiles, window_tile;  // the list: tiles [0, pinned_tiles), then from window_tile
    int part;

    __device__ __forceinline__ int key_tile(int i) const {
        return i < pinned_tiles ? i : window_tile + (i - pinned_tiles);
    }
    __device__ __forceinline__ int position(int token) const { return length - steps + token; }
    __device__ __forceinline__ bool rows() const { return token1 > token0; }
    // Whether some row of the tile has a position in the stream, and what such rows see.
    __device__ __forceinline__ bool keys() const { return rows() && length > 0 && position(token1 - 1) >= 0; }
    // Bit j: whether the tile's rows see some key of tile i + j of the block's range, and (cuts) whether some
    // of them do not see all of it.  A whole warp's call.
    __device__ __forceinline__ void look(int i, int lane, const dcn_token_attention_args &a, uint32_t *takes,
                                         uint32_t *cuts) const {
        const int at = first + i + lane;
        const bool in = keys() && at < last;
        const Span seen = span(a);
        const int base = key_tile(at) * kKeys;
        *takes = __ballot_sync(0xffffffffu, in && seen.tile_some(base));
        *cuts = __ballot_sync(0xffffffffu, in && seen.tile_some(base) && !seen.tile_all(base));
    }
    __device__ __forceinline__ Span span(const dcn_token_attention_args &a) const {
        Span out;
        out.set(max(position(token0), 0), position(token1 - 1), length, a);
        return out;
    }
};

template <bool Shared>
struct Walk {
    int w, block;  // item, and its row block (-1: take the item's first)
    int s;         // stream of tiles
    Span both;     // of the rows of both of the block's streams

    __device__ __forceinline__ explicit Walk(int stream_of_tiles) : w(blockIdx.x), block(-1), s(stream_of_tiles) {}
    __device__ __forceinline__ bool next(const KernelParams &p, Item &it) {
        const int block_tokens = p.tile_tokens * (Shared ? 2 : 1);
        while (w < p.items) {
            uint32_t rest = w;
            const uint32_t splits = p.splits, row_blocks = p.row_blocks, heads = p.a.cache.heads;
            const int split = rest % splits;
            rest /= splits;
            // Later row blocks first: under a causal mask they have the most keys.
            const int first_block = row_blocks - 1 - rest % row_blocks;
            rest /= row_blocks;
            it.kv_head = rest % heads;
            it.stream = rest / heads;
            it.start = p.a.cache.starts[it.stream];
            it.steps = p.a.cache.starts[it.stream + 1] - it.start;
            it.length = p.a.cache.lengths[it.stream];
            // No row outside the token tensors, whatever `starts` holds.
            const int64_t end_token = min(static_cast<int64_t>(it.steps), p.a.args.tokens - it.start);
            const int rows_end = it.start < 0 || end_token < 0 ? 0 : static_cast<int>(end_token);
            // Steps longer than max_q said: every row_blocks-th block is this item's too.
            block = block < 0 ? first_block : block + p.row_blocks;
            if (static_cast<int64_t>(block) * block_tokens >= rows_end) {
                block = -1;
                w += gridDim.x;
                continue;
            }
            const int t0 = block * block_tokens, end = min(t0 + block_tokens, rows_end);
            it.token0 = Shared ? t0 + s * p.tile_tokens : t0;
            it.token1 = min(it.token0 + p.tile_tokens, rows_end);
            int tiles = 0;
            it.pinned_tiles = it.window_tile = 0;
            if (it.length > 0 && it.position(end - 1) >= 0) {
                both.set(max(it.position(t0), 0), it.position(end - 1), it.length, p.a.args);
                it.pinned_tiles = (min(both.pinned, both.high) + kKeys - 1) / kKeys;
                it.window_tile = max(both.low / kKeys, it.pinned_tiles);
                tiles = it.pinned_tiles + max(0, (both.high + kKeys - 1) / kKeys - it.window_tile);
            }
            const uint32_t parts = Shared ? splits : 2 * splits;
            const int each = (static_cast<uint32_t>(tiles) + parts - 1) / parts;
            it.part = Shared ? split : 2 * split + s;
            it.first = min(it.part * each, tiles);
            it.last = min(it.first + each, tiles);
            it.both_last = Shared ? it.last : min((2 * split + 2) * each, tiles);
            return true;
        }
        return false;
    }
};

template <int D, bool Shared>
struct alignas(1024) Smem {
    using L = Layout<D, Shared>;
    uint8_t q[L::kQTiles][L::kTileBytes];
    uint8_t kv[L::kRings][L::kSlots][L::kTileBytes];
    uint64_t full[L::kRings][L::kSlots], empty[L::kRings][L::kSlots];
    uint64_t q_full[2], q_free, s_full[2], p_full[2][2], s_read[2], pv_done[2], o_full[2], scan_go, scanned, merge_ready, merge_read, drain;
    // The current item of each softmax warp and of the product warp's two streams, kept here: the 128
    // scores of a row need the registers.
    Item item[kSoftmaxWarps + 2];
    float2 other_ml[kRows];  // stream 1's (c m - kRaise, l), where stream 0 merges the two
    int other_dirty;         // and whether its rows are to be done alone
    int dirty[2][2];         // by the parity of an item's number: the last item whose rows are to be done alone
    int abort_flag;
    int beat;                // counts on while rows are done alone, which may take longer than a wait's limit
    uint32_t tmem_base;
};

// Position in a ring of tiles: the slot, and the parity of its current use.
template <int Slots>
struct RingAt {
    int slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void advance() {
        if (++slot == Slots) {
            slot = 0;
            parity ^= 1u;
        }
    }
};

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The lowest n bits of a word; none for n <= 0, all for n >= 32.
__device__ __forceinline__ uint32_t bits_below(int n) {
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// Two FP32 values in one register pair, and the instructions that take two at a time.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ float low_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float high_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Bit 15 or 31 is set where the lower or upper value of a pair is not finite: one more in the exponent's
// last place carries out of an exponent of ones, and of no other.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t pair) {
    constexpr uint32_t kExponents = __is_same(T, __half) ? 0x7c007c00u : 0x7f807f80u;
    constexpr uint32_t kOnes = __is_same(T, __half) ? 0x04000400u : 0x00800080u;
    return (pair & kExponents) + kOnes;
}

// Looks through one key's row of a tile of values for what is not finite.  Where it finds something and no
// row of the block sees the key (hidden), the row becomes zeros; true where some row does.
template <typename T, int D>
__device__ __forceinline__ bool scan_values(uint8_t *tile, int row, bool hidden) {
    uint8_t *v_row = tile + row * 128;
    auto pack_at = [&](int e) {
        return reinterpret_cast<uint4 *>(v_row + (e / 8) * (kKeys * 128) + (((e % 8) ^ (row % 8)) * 16));
    };
    uint32_t found = 0;
#pragma unroll 8
    for (int e = 0; e < D / 8; ++e) {
        const uint4 v = *pack_at(e);
        found |= not_finite<T>(v.x) | not_finite<T>(v.y) | not_finite<T>(v.z) | not_finite<T>(v.w);
    }
    if ((found & 0x80008000u) == 0) return false;
    if (!hidden) return true;
    for (int e = 0; e < D / 8; ++e) *pack_at(e) = make_uint4(0, 0, 0, 0);
    return false;
}

// One of the failure path's records: some wait ran out.
template <typename S>
__device__ __forceinline__ void give_up(S &s, uint32_t *err) {
    if (*reinterpret_cast<volatile int *>(&s.abort_flag) == 0) atomicOr(err, kErrWaitTimeout);
    *reinterpret_cast<volatile int *>(&s.abort_flag) = 1;
}

// A wait of bounded length, begun again for as long as some warp gets on with rows alone (whose work is finite).
template <typename S>
__device__ __forceinline__ bool wait_bounded(S &s, uint64_t *bar, uint32_t parity) {
    while (true) {
        const int beat = *reinterpret_cast<volatile int *>(&s.beat);
        if (mbar_wait_bounded(bar, parity, &s.abort_flag)) return true;
        if (*reinterpret_cast<volatile int *>(&s.abort_flag) || *reinterpret_cast<volatile int *>(&s.beat) == beat) return false;
    }
}

// The rows of a warp (token and head: this lane's, where valid), one after another, from their visible keys in the
// item's key tiles: for rows of a tile that holds a non-finite value which only some of its rows see (0 x inf in
// the product would reach the others).  Slow and rare.
template <typename T, int D>
__device__ __noinline__ void rows_alone(const KernelParams &p, const Item it, bool valid, int token, int head,
                                        const Visible seen, int64_t part_row, int *beat) {
    const int lane = threadIdx.x & 31;
    // The range of the list of tiles, as keys.
    const int64_t begin[2] = {static_cast<int64_t>(it.first) * kKeys,
                              (it.window_tile + max(it.first - it.pinned_tiles, 0)) * static_cast<int64_t>(kKeys)};
    const int64_t end[2] = {static_cast<int64_t>(min(it.last, it.pinned_tiles)) * kKeys,
                            it.last > it.pinned_tiles ? (it.window_tile + it.last - it.pinned_tiles) * static_cast<int64_t>(kKeys) : 0};
    for (uint32_t left = __ballot_sync(0xffffffffu, valid); left != 0; left &= left - 1) {
        const int from = __ffs(left) - 1;
        const int row_token = __shfl_sync(0xffffffffu, token, from), row_head = __shfl_sync(0xffffffffu, head, from);
        const Visible row_seen{__shfl_sync(0xffffffffu, seen.first, from), __shfl_sync(0xffffffffu, seen.low, from),
                               __shfl_sync(0xffffffffu, seen.high, from)};
        const int64_t row_part = __shfl_sync(0xffffffffu, part_row, from);
        const T *q = static_cast<const T *>(p.a.q.data) + (it.start + row_token) * p.a.q.token_stride + row_head * p.a.q.head_stride;
        RowByWarp<T, D / 32> row;
        row.run(p.a.cache, it.stream, it.kv_head, q, p.negate ? -p.c : p.c, row_seen, begin, end, beat);
        const bool none = row_seen.first <= 0 && row_seen.high <= row_seen.low;
        T *out = static_cast<T *>(p.a.out.data) + (it.start + row_token) * p.a.out.token_stride + row_head * p.a.out.head_stride;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            if (p.part_o) p.part_o[row_part * D + i * 32 + lane] = row.acc[i];
            else out[i * 32 + lane] = from_float<T>(none ? 0.0f : row.acc[i] / row.l);
        }
        if (p.part_o && lane == 0) p.part_ml[row_part] = make_float2(row.m, row.l);
    }
}

template <typename T, int D, bool Shared>
__global__ void __launch_bounds__(kThreads, 1)
attention_kernel(const __grid_constant__ KernelParams p, const __grid_constant__ CUtensorMap k_map,
                 const __grid_constant__ CUtensorMap v_map) {
    using L = Layout<D, Shared>;
    static_assert(sizeof(Smem<D, Shared>) + 1024 <= 227 * 1024, "a block's shared memory");
    extern __shared__ uint8_t raw[];
    Smem<D, Shared> &sm = *reinterpret_cast<Smem<D, Shared> *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t{1023});
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int r = 0; r < L::kRings; ++r)
            for (int i = 0; i < L::kSlots; ++i) {
                mbar_init(&sm.full[r][i], 1);
                mbar_init(&sm.empty[r][i], 1);
            }
        mbar_init(&sm.scan_go, 1);
        mbar_init(&sm.scanned, 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&sm.q_full[s], kRows);
            mbar_init(&sm.s_full[s], 1);
            mbar_init(&sm.p_full[s][0], 4);
            mbar_init(&sm.p_full[s][1], 4);
            mbar_init(&sm.s_read[s], 4);
            mbar_init(&sm.pv_done[s], 1);
            mbar_init(&sm.o_full[s], 2);
            sm.dirty[s][0] = sm.dirty[s][1] = -1;
        }
        mbar_init(&sm.q_free, 1);
        mbar_init(&sm.drain, 1);
        mbar_init(&sm.merge_ready, 4);
        mbar_init(&sm.merge_read, 4);
        sm.abort_flag = 0;
        sm.beat = 0;
        fence_mbarrier_init();
        prefetch_tensor_map(&k_map);
        prefetch_tensor_map(&v_map);
    }
    if (warp == kSoftmaxWarps) {
        tmem_alloc(&sm.tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;
    if (p.part_o) allow_dependent_launch();

    if (warp >= kSoftmaxWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == kSoftmaxWarps) {
            // -------------------------------------------------------------------- products
            // One warp issues for both streams, stream 0's second product and next scores before
            // stream 1's: that keeps the streams half a tile apart, so that one's exponentials run while the
            // other's products do.  (With a thread a stream both ran in step, each waiting for the tensor
            // core and then for the exponentials at the same time: 714 us where this took 651.)  All lanes run
            // through it and one issues: under a lane == 0 branch each product moved its operands into uniform
            // registers anew (651 us where this took 545).
            constexpr bool kBf16 = __is_same(T, __nv_bfloat16);
            constexpr uint32_t kTypes = kBf16 ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t kIdescS = make_idesc_f16_f32(kRows, kKeys) | kTypes;
            constexpr uint32_t kIdescO = make_idesc_f16_f32(kRows, D) | kTypes | (1u << 16);  // B: N contiguous
            constexpr int kLastRing = L::kRings - 1;
            RingAt<L::kSlots> at[L::kRings];
            uint32_t scan_phase = 0;
            uint32_t q_phase[2] = {0, 0}, p_phase[2] = {0, 0}, read_phase[2] = {0, 0};
            const uint32_t issue = elect_one();
            uint64_t q_desc[2], k_desc[L::kRings], v_desc[L::kRings];
#pragma unroll
            for (int s = 0; s < 2; ++s) q_desc[s] = make_sw128_kmajor_desc(smem_addr(sm.q[Shared ? s : 0]));
#pragma unroll
            for (int r = 0; r < L::kRings; ++r) {
                k_desc[r] = make_sw128_kmajor_desc(smem_addr(sm.kv[r][0]));
                v_desc[r] = make_sw128_mnmajor_desc(smem_addr(sm.kv[r][0]), kKeys * 128);
            }
            bool ok = true;
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
                ok = __all_sync(0xffffffffu, wait_bounded(sm, bar, parity));
                if (!ok && lane == 0) give_up(sm, p.err);
                return ok;
            };
            // Shared: tiles of values that some row does not see all of are looked through before their
            // product, by a warp of its own: asked for with the tile's scores, waited for before its product.
            auto scanned = [&]() {
                if (!wait(&sm.scanned, scan_phase)) return false;
                scan_phase ^= 1u;
                return true;
            };
            auto second = [&](int s, int r, int slot, uint32_t &more) {  // O += P V, half a tile's keys at a time
                const uint64_t desc = v_desc[r] + static_cast<uint32_t>(slot * (L::kTileBytes >> 4));
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (!wait(&sm.p_full[s][h], p_phase[s])) return false;
                    tc_fence_after();
#pragma unroll
                    for (int k = h * kKeys / 2; k < (h + 1) * kKeys / 2; k += 16) {
                        umma_f16_ts_if(issue, tmem + kTmemO + s * D,
                                       tmem + (L::kApart ? kTmemP + s * (kKeys / 2) : s * kKeys) + k / 2,
                                       desc + (k * 128 >> 4), kIdescO, more);
                        more = 1;
                    }
                }
                p_phase[s] ^= 1u;
                if (L::kApart) umma_commit_if(issue, &sm.pv_done[s]);
                return true;
            };
            auto scores_read = [&](int s) {
                if (!wait(&sm.s_read[s], read_phase[s])) return false;
                read_phase[s] ^= 1u;
                tc_fence_after();
                return true;
            };
            auto scores = [&](int s, int r, int slot) {  // S = Q K^T
                const uint64_t desc = k_desc[r] + static_cast<uint32_t>(slot * (L::kTileBytes >> 4));
#pragma unroll
                for (int d = 0; d < D; d += 16) {
                    const uint32_t off = ((d / 64) * (kKeys * 128) + (d % 64) * 2) >> 4;
                    umma_f16_ss_if(issue, tmem + s * kKeys, q_desc[s] + off, desc + off, kIdescS, d != 0);
                }
                umma_commit_if(issue, &sm.s_full[s]);
            };
            Walk<Shared> walk0(0), walk1(1);
            const Item *item = sm.item + kSoftmaxWarps;
            // Whether stream 1 may still be at the item before the last: it is not waited for over an item without rows
            // of its own.  An item's first tile is then asked to be looked through when it has begun that item too, as
            // the mark goes where the item before the last had its own, which stream 1 has yet to read.
            bool behind = false;
            for (; ok; behind = !item[1].rows()) {
                {
                    Item next[2];
                    if (!walk0.next(p, next[0]) || !walk1.next(p, next[1])) break;
                    __syncwarp();
                    if (lane == 0) {
                        sm.item[kSoftmaxWarps] = next[0];
                        sm.item[kSoftmaxWarps + 1] = next[1];
                    }
                    __syncwarp();
                }
                const int count[2] = {item[0].last - item[0].first, item[1].last - item[1].first};
                const int steps = max(count[0], count[1]);
                uint32_t more[2] = {0, 0}, takes[2] = {0, 0}, took[2] = {0, 0};
                uint32_t cuts = 0, scan = 0;  // Shared: tiles to be looked through, and whether the last is one
                // Step i: the second product of tile i, then the scores of tile i + 1.
                for (int i = -1; ok && i < steps; ++i) {
                    if (((i + 1) & 31) == 0) {  // bit j: whether a stream takes tile i + 1 + j of its list
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            uint32_t cut;
                            item[s].look(i + 1, lane, p.a.args, &takes[s], &cut);
                            cuts = Shared ? s == 0 ? cut : cuts | cut : 0;
                        }
                    }
                    // The step in the middle of a run of tiles that both streams take, without the general step's
                    // questions: this warp's instructions between two products are on every tile's path.
                    while (took[0] & took[1] & takes[0] & takes[1] & (((i + 1) & 31) != 31)) {
                        if (scan && !scanned()) break;
                        if (L::kApart) {
#pragma unroll
                            for (int s = 0; s < 2; ++s) {
                                const int r = s < kLastRing ? s : kLastRing;
                                RingAt<L::kSlots> here = at[r];
                                here.advance();
                                if ((!Shared || s == 0) && !wait(&sm.full[r][here.slot], here.parity)) break;
                                if (!scores_read(s)) break;
                                scores(s, r, here.slot);
                                if ((cuts & 1u) && s == 0 && lane == 0) mbar_arrive(&sm.scan_go);
                                if (!Shared || s == 1) umma_commit_if(issue, &sm.empty[r][here.slot]);
                            }
                            if (!ok) break;
                        }
#pragma unroll
                        for (int s = 0; s < 2; ++s) {
                            const int r = s < kLastRing ? s : kLastRing;
                            RingAt<L::kSlots> here = at[r];
                            if ((!Shared || s == 0) && !wait(&sm.full[r][here.slot], here.parity)) break;
                            if (!second(s, r, here.slot, more[s])) break;
                            if (!Shared || s == 1) umma_commit_if(issue, &sm.empty[r][here.slot]);
                            here.advance();
                            if (!L::kApart) {
                                if ((!Shared || s == 0) && !wait(&sm.full[r][here.slot], here.parity)) break;
                                scores(s, r, here.slot);
                                if ((cuts & 1u) && s == 0 && lane == 0) mbar_arrive(&sm.scan_go);
                                if (!Shared || s == 1) umma_commit_if(issue, &sm.empty[r][here.slot]);
                            }
                            if (!Shared || s == 1) {
                                here.advance();
                                at[r] = here;
                            }
                        }
                        if (!ok) break;
                        ++i;
                        takes[0] >>= 1;
                        takes[1] >>= 1;
                        scan = cuts & 1u;
                        cuts >>= 1;
                    }
                    if (!ok) break;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        const int r = s < kLastRing ? s : kLastRing;
                        const bool release = !Shared || s == 1;  // the last to read the tile
                        const bool take = takes[s] & 1u;
                        RingAt<L::kSlots> here = at[r];
                        if (i < 0 && item[s].rows()) {
                            if (!wait(&sm.q_full[s], q_phase[s])) break;
                            q_phase[s] ^= 1u;
                        }
                        if (i >= 0 && i < count[s]) {
                            if (!wait(&sm.full[r][here.slot], here.parity)) break;
                            if (scan && s == 0 && !scanned()) break;
                            if (took[s]) {
                                if (L::kApart && !scores_read(s)) break;
                                if (!second(s, r, here.slot, more[s])) break;
                            }
                            if (release) umma_commit_if(issue, &sm.empty[r][here.slot]);
                            here.advance();
                        }
                        if (i + 1 < count[s]) {
                            if (!wait(&sm.full[r][here.slot], here.parity)) break;
                            if (take) {
                                tc_fence_after();
                                scores(s, r, here.slot);
                            }
                            if ((cuts & 1u) && s == (i < 0 && behind ? 1 : 0) && lane == 0) mbar_arrive(&sm.scan_go);
                            if (release) umma_commit_if(issue, &sm.empty[r][here.slot]);
                            here.advance();
                        }
                        if (i + 1 == count[s] && item[s].rows()) {
                            // Once an item, with or without products: the softmax warpgroup moves on only after
                            // it, so no barrier of the item runs a phase ahead of this warp.
                            // The second arrival passes on what was written where values were looked through.
                            umma_commit_if(issue, &sm.o_full[s]);
                            if (lane == 0) mbar_arrive(&sm.o_full[s]);
                            if (!Shared && s == 1) umma_commit_if(issue, &sm.q_free);
                        }
                        took[s] = take;
                        takes[s] >>= 1;
                        if (release) at[r] = here;
                    }
                    scan = cuts & 1u;
                    cuts >>= 1;
                }
            }
            // Every product issued has ended before the block lets go of its memory.
            umma_commit_if(issue, &sm.drain);
            mbar_wait_bounded(&sm.drain, 0, nullptr);
            __syncwarp();
        } else if (Shared && warp == kSoftmaxWarps + 1) {
            // ------------------------------------------------------------------------ scan
            // A row's weights are 0 for the keys that it does not see, and 0 x non-finite is not 0.  So in each
            // tile of values that some row does not see all of, a key that no row of the block sees becomes
            // zeros, and where a key that only some see is not finite, those rows' tile is marked, and its rows
            // are done alone at the end.  (With one row tile a block, where memory is the bound, the softmax
            // warps do it while they wait for the scores.)
            RingAt<L::kSlots> at;
            uint32_t go_phase = 0;
            int number = 0;  // items with tiles so far
            bool ok = true;
            Walk<Shared> walk0(0), walk1(1);
            while (ok) {
                Item item0, item1;
                if (!walk0.next(p, item0) || !walk1.next(p, item1)) break;
                const Span span0 = item0.span(p.a.args), span1 = item1.span(p.a.args);
                const int count = item0.last - item0.first;
                uint32_t takes, cuts0 = 0, cuts1 = 0;
                for (int i = 0; ok && i < count; ++i, cuts0 >>= 1, cuts1 >>= 1) {
                    if ((i & 31) == 0) {
                        item0.look(i, lane, p.a.args, &takes, &cuts0);
                        item1.look(i, lane, p.a.args, &takes, &cuts1);
                    }
                    at.advance();  // from the keys' slot to the values'
                    const bool cut0 = cuts0 & 1u, cut1 = cuts1 & 1u;
                    if (cut0 || cut1) {
                        // The slot's earlier tiles have been used when this one is asked for, and it stays until it
                        // has been looked through: its barrier's next phase is this tile's.
                        ok = __all_sync(0xffffffffu, wait_bounded(sm, &sm.scan_go, go_phase) &&
                                                         wait_bounded(sm, &sm.full[0][at.slot], at.parity));
                        if (!ok) {
                            if (lane == 0) give_up(sm, p.err);
                            break;
                        }
                        go_phase ^= 1u;
                        const int base = item0.key_tile(item0.first + i) * kKeys;
                        for (int row = lane; row < kKeys; row += 32) {
                            const int key = base + row;
                            const bool some0 = cut0 && !span0.all(key), some1 = cut1 && !span1.all(key);
                            if (!some0 && !some1) continue;
                            if (scan_values<T, D>(sm.kv[0][at.slot], row, !walk0.both.some(key))) {
                                if (some0) *static_cast<volatile int *>(&sm.dirty[0][number & 1]) = number;
                                if (some1) *static_cast<volatile int *>(&sm.dirty[1][number & 1]) = number;
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.scanned);
                    }
                    at.advance();
                }
                number += count > 0;
            }
        } else if (warp >= kSoftmaxWarps + 2 && warp < kSoftmaxWarps + 2 + L::kRings) {
            const int s = warp - (kSoftmaxWarps + 2);
            // -------------------------------------------------------------------- loads of ring s
            RingAt<L::kSlots> at;
            uint32_t loaded = 0;
            const int groups = kKeys / p.box_rows, boxes = groups * (D / 64);
            bool ok = true;
            Walk<Shared> walk(s);
            Item it;
            while (ok && walk.next(p, it)) {
                for (int i = it.first; ok && i < it.last; ++i) {
                    // Box b of a tile: keys [group * box_rows, ...) and 64 elements.
                    const int group = lane % groups, half = lane / groups;
                    const int key = it.key_tile(i) * kKeys + group * p.box_rows;
                    const int column = key / p.a.cache.page_size;
                    int page = -1;  // outside the cache: the copy fills with zeros
                    if (lane < boxes && key < it.length && column < p.a.cache.table_columns) {
                        page = p.a.cache.table[it.stream * p.a.cache.table_stride + column];
                        if (page < 0 || page >= p.a.cache.pages) page = -1;
                    }
                    const int slot = key - column * p.a.cache.page_size;
#pragma unroll 1
                    for (int v = 0; v < 2; ++v) {
                        ok = wait_bounded(sm, &sm.empty[s][at.slot], at.parity ^ 1u);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) {
                            if (lane == 0) give_up(sm, p.err);
                            break;
                        }
                        if (lane == 0) mbar_arrive_expect_tx(&sm.full[s][at.slot], L::kTileBytes);
                        __syncwarp();
                        if (lane < boxes)
                            tma_load_4d(sm.kv[s][at.slot] + half * (kKeys * 128) + group * p.box_rows * 128,
                                        v == 0 ? &k_map : &v_map, &sm.full[s][at.slot], half * 64, slot, it.kv_head, page);
                        at.advance();
                        ++loaded;
                    }
                }
            }
            // Every copy issued has landed before the block lets go of its memory.
            for (uint32_t k = 0; k < L::kSlots && k < loaded; ++k) {
                const uint32_t last = loaded - 1 - k;
                mbar_wait_bounded(&sm.full[s][last % L::kSlots], (last / L::kSlots) & 1u, nullptr);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---------------------------------------------------------------------- softmax of stream s
        const int s = warp >> 2;
        const int row = threadIdx.x & (kRows - 1);
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_tmem = tmem + lanes + s * kKeys, o_tmem = tmem + lanes + kTmemO + s * D;
        const uint32_t p_tmem = L::kApart ? tmem + lanes + kTmemP + s * (kKeys / 2) : s_tmem;
        const int row_token = row * p.per_ratio >> 16, row_head = row - row_token * p.ratio;
        const bool row_used = row_token < p.tile_tokens;
        uint32_t s_phase = 0, item_phase = 0, free_phase = 0, merge_phase = 0;
        int tile_items = 0;  // items with tiles so far
        RingAt<L::kSlots> at;
        bool ok = true, q_loaded = false, tiles_done = false;
        auto wait = [&](uint64_t *bar, uint32_t parity) {  // the whole warp gives up together
            ok = __all_sync(0xffffffffu, wait_bounded(sm, bar, parity));
            if (!ok && lane == 0) give_up(sm, p.err);
            return ok;
        };
        Walk<Shared> walk(s);
        const Item &it = sm.item[warp];
        for (;;) {
            {
                Item next;
                if (!ok || !walk.next(p, next)) break;
                __syncwarp();
                if (lane == 0) sm.item[warp] = next;
                __syncwarp();
            }
            const bool rows = it.rows();
            const int token = it.token0 + row_token;
            const int head = it.kv_head * p.ratio + row_head;
            const bool valid = row_used && token < it.token1;
            if (rows && (Shared || s == 0)) {
                if (!Shared && q_loaded) {  // the other stream's products have read the last tile
                    if (!wait(&sm.q_free, free_phase)) break;
                    free_phase ^= 1u;
                }
                q_loaded = true;
                // 16 bytes a load, a row's packs on neighbouring threads.
                constexpr int kPacks = D / 8;
                const T *q = static_cast<const T *>(p.a.q.data);
                uint4 v[kPacks];
#pragma unroll
                for (int i = 0; i < kPacks; ++i) {
                    const int r = (i * kRows + row) / kPacks, e = (row % kPacks) * 8;
                    const int rt = r * p.per_ratio >> 16, rh = r - rt * p.ratio;
                    v[i] = make_uint4(0, 0, 0, 0);
                    if (rt < p.tile_tokens && it.token0 + rt < it.token1)
                        v[i] = *reinterpret_cast<const uint4 *>(q + (it.start + it.token0 + rt) * p.a.q.token_stride +
                                                                (it.kv_head * p.ratio + rh) * p.a.q.head_stride + e);
                }
#pragma unroll
                for (int i = 0; i < kPacks; ++i) {
                    const int r = (i * kRows + row) / kPacks, e = row % kPacks;
                    if (p.negate) {
                        v[i].x ^= 0x80008000u;
                        v[i].y ^= 0x80008000u;
                        v[i].z ^= 0x80008000u;
                        v[i].w ^= 0x80008000u;
                    }
                    // 128-byte swizzle: pack e of a row goes to place e ^ (row mod 8) of its 8.
                    uint8_t *dst = sm.q[Shared ? s : 0] + (e / 8) * (kRows * 128) + r * 128 + (((e % 8) ^ (r % 8)) * 16);
                    *reinterpret_cast<uint4 *>(dst) = v[i];
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                mbar_arrive(&sm.q_full[s]);
            } else if (rows) {
                mbar_arrive(&sm.q_full[s]);  // stream 0 loads the tile; this stream is ready for the item
            }
            int seen_first, seen_low, seen_high;
            {
                const Visible seen = visible_keys(it.position(token), it.length, p.a.args.window, p.a.args.sinks, p.a.args.frame);
                seen_first = static_cast<int>(seen.first);
                seen_low = static_cast<int>(seen.low);
                seen_high = static_cast<int>(seen.high);
            }
            const bool warp_used = __any_sync(0xffffffffu, valid);
            float m = -INFINITY, l = 0.0f;
            bool any = false;
            uint32_t takes = 0, cuts = 0;
            for (int i = 0, count = it.last - it.first; i < count; ++i, takes >>= 1, cuts >>= 1) {
                if ((i & 31) == 0) it.look(i, lane, p.a.args, &takes, &cuts);
                if (!Shared) at.advance();  // from the keys' slot to the values'
                if (!(takes & 1u)) {
                    if (!Shared) at.advance();
                    continue;
                }
                const bool cut = cuts & 1u;
                if (!Shared) {
                    if (cut) {
                        if (!wait(&sm.full[s][at.slot], at.parity)) break;
                        const Span span = it.span(p.a.args);
                        const int key = it.key_tile(it.first + i) * kKeys + row;
                        // (Both streams have the same rows.)
                        if (!span.all(key) && scan_values<T, D>(sm.kv[s][at.slot], row, !span.some(key)))
                            *static_cast<volatile int *>(&sm.dirty[s][tile_items & 1]) = tile_items;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                    at.advance();
                }
                if (!wait(&sm.s_full[s], s_phase)) break;
                s_phase ^= 1u;
                if (warp_used) {
                    tc_fence_after();
                    if (cut) {
                        // Hidden keys' scores become -inf where they lie, 32 columns at a time, which keeps the
                        // selects out of the code that every tile runs through.
                        const int base = it.key_tile(it.first + i) * kKeys;
                        // Bit k: key base + w + k is seen; rows of no query keep theirs.
                        const int first = valid ? seen_first - base : kKeys, low = seen_low - base, high = seen_high - base;
#pragma unroll 1
                        for (int w = 0; w < kKeys; w += 32) {
                            const uint32_t mask = bits_below(first - w) | (bits_below(high - w) & ~bits_below(low - w));
                            if (__all_sync(0xffffffffu, mask == 0xffffffffu)) continue;
                            uint32_t y[32];
                            tmem_ld_32x32b_x32(s_tmem + w, y);
                            tmem_wait_ld_x32(y);
#pragma unroll
                            for (int k = 0; k < 32; ++k)
                                if (!(mask >> k & 1u)) y[k] = 0xff800000u;
                            tmem_st_32x32b_x32_wait(s_tmem + w, y);
                        }
                    }
                    uint32_t x[kKeys];
#pragma unroll
                    for (int k = 0; k < kKeys; k += 32) tmem_ld_32x32b_x32(s_tmem + k, x + k);
#pragma unroll
                    for (int k = 0; k < kKeys; k += 32) tmem_wait_ld_x32(x + k);
                    if (L::kApart) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.s_read[s]);
                    }
                    float top[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) top[j] = __uint_as_float(x[j]);
#pragma unroll
                    for (int k = 4; k + 8 <= kKeys; k += 8)
#pragma unroll
                        for (int j = 0; j < 4; ++j) top[j] = max3(top[j], __uint_as_float(x[k + j]), __uint_as_float(x[k + 4 + j]));
#pragma unroll
                    for (int j = 0; j < 4; ++j) top[j] = fmaxf(top[j], __uint_as_float(x[kKeys - 4 + j]));
                    const float t = fmaxf(max3(top[0], top[1], top[2]), top[3]);
                    // The last tile's second product has ended: O may be scaled, P written again.  (Where P lies over S
                    // this tile's scores were issued after it.)
                    if (L::kApart && tiles_done) {
                        if (!wait(&sm.pv_done[s], s_phase)) break;
                        tc_fence_after();
                    }
                    if (!any) {
                        m = t;
                    } else if (__any_sync(0xffffffffu, (t - m) * p.c > kLag)) {
                        // Products up to the last tile's have ended: S of this tile was issued after them.
                        const float to = fmaxf(m, t);
                        const float shrink = to == -INFINITY ? 1.0f : exp2_approx((m - to) * p.c);
                        m = to;
                        l *= shrink;
#pragma unroll 1
                        for (int d = 0; d < D; d += 16) {  // 16 columns: the scores hold 128 registers
                            uint32_t o[16];
                            tmem_ld_32x32b_x16(o_tmem + d, o);
                            tmem_wait_ld_x16(o);
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * shrink);
                            tmem_st_32x32b_x16_wait(o_tmem + d, o);
                        }
                    }
                    const float mc = m == -INFINITY ? 0.0f : m * p.c - kRaise<T>;
                    const uint64_t c2 = pair_of(p.c, p.c), mc2 = pair_of(-mc, -mc);
                    uint64_t sum[2] = {0, 0};  // two FP32 zeros each
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // the second product starts on the first half's weights
#pragma unroll
                        for (int k = h * kKeys / 2; k < (h + 1) * kKeys / 2; k += 2) {
                            const uint64_t y = fma_pair(pair_of(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), c2, mc2);
                            const float a = exp2_approx(low_of(y)), b = exp2_approx(high_of(y));
                            sum[k / 2 % 2] = add_pair(sum[k / 2 % 2], pair_of(a, b));
                            x[k / 2] = pack_pair<T>(a, b);
                        }
                        tmem_st_32x32b_x32_wait(p_tmem + h * 32, x + h * 32);
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.p_full[s][h]);
                    }
                    const uint64_t sums = add_pair(sum[0], sum[1]);
                    l += low_of(sums) + high_of(sums);
                } else {  // no row of the step: keeps pace with the other warps, a phase at a time
                    if (L::kApart && lane == 0) mbar_arrive(&sm.s_read[s]);
                    if (L::kApart && tiles_done && !wait(&sm.pv_done[s], s_phase)) break;
                    if (lane == 0) {
                        mbar_arrive(&sm.p_full[s][0]);
                        mbar_arrive(&sm.p_full[s][1]);
                    }
                }
                any = tiles_done = true;
            }
            if (!ok) break;
            const bool has_tiles = it.last > it.first;
            const int tile_item = tile_items;  // this item's number among those with tiles, as the scan counts them
            tile_items += has_tiles;
            if (!rows) continue;
            if (!wait(&sm.o_full[s], item_phase)) break;
            item_phase ^= 1u;
            tc_fence_after();
            bool alone = has_tiles && *reinterpret_cast<volatile int *>(&sm.dirty[s][tile_item & 1]) == tile_item;
            const int64_t at_row = static_cast<int64_t>(it.start + token) * p.a.args.q_heads + head;
            const int64_t part_row = static_cast<int64_t>(it.part) * p.a.args.tokens * p.a.args.q_heads + at_row;
            T *out = static_cast<T *>(p.a.out.data) + (it.start + token) * p.a.out.token_stride + head * p.a.out.head_stride;
            // Unsplit, the block has all of its rows' keys: stream 0 merges stream 1's sums, and its O from
            // tensor memory, whose lanes both warpgroups reach.
            const bool merge = !Shared && p.part_o == nullptr;
            float2 other = make_float2(-INFINITY, 0.0f);
            const float mc = m * p.c - kRaise<T>;
            if (merge && s == 1) {
                sm.other_ml[row] = any ? make_float2(mc, l) : other;
                if (row == 0) sm.other_dirty = alone;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.merge_ready);
                if (!wait(&sm.merge_read, merge_phase)) break;  // its O may be written again
                merge_phase ^= 1u;
                continue;
            }
            if (merge) {
                if (!wait(&sm.merge_ready, merge_phase)) break;
                merge_phase ^= 1u;
                tc_fence_after();
                other = sm.other_ml[row];
                alone |= sm.other_dirty != 0;
            }
            if (alone) {
                Item all = it;
                if (merge) all.last = it.both_last;
                rows_alone<T, D>(p, all, valid, token, head, Visible{seen_first, seen_low, seen_high}, part_row, &sm.beat);
                __syncwarp();
            } else if (warp_used) {
                const bool none = seen_first <= 0 && seen_high <= seen_low;
                if (p.part_o && valid) p.part_ml[part_row] = any ? make_float2(mc, l) : make_float2(-INFINITY, 0.0f);
                if (any || !p.part_o) {  // a part without weight is not read
                    // Factors of the two streams' O; a stream without weight has none.
                    const bool two = merge && __any_sync(0xffffffffu, other.x != -INFINITY || other.y != 0.0f);
                    float mine = 1.0f, theirs = 0.0f;
                    if (two) {
                        const float to = fmaxf(any ? mc : -INFINITY, other.x);
                        const float base = to == -INFINITY ? 0.0f : to;
                        mine = any ? exp2_approx(mc - base) : 0.0f;
                        theirs = exp2_approx(other.x - base);
                        l = l * mine + other.y * theirs;
                    }
                    if (!p.part_o) {
                        const float inv = 1.0f / l;
                        mine *= inv;
                        theirs *= inv;
                    }
#pragma unroll 1
                    for (int d = 0; d < D; d += 32) {
                        uint32_t o[32];
#pragma unroll
                        for (int j = 0; j < 32; ++j) o[j] = 0u;
                        if (any) {
                            tmem_ld_32x32b_x32(o_tmem + d, o);
                            tmem_wait_ld_x32(o);
#pragma unroll
                            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * mine);
                        }
                        if (two) {
                            uint32_t b[32];
                            tmem_ld_32x32b_x32(o_tmem + D + d, b);
                            tmem_wait_ld_x32(b);
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                o[j] = __float_as_uint(fmaf(__uint_as_float(b[j]), theirs, __uint_as_float(o[j])));
                        }
                        if (valid && p.part_o) {
                            float4 *dst = reinterpret_cast<float4 *>(p.part_o + part_row * D + d);
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                dst[j] = make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]),
                                                     __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3]));
                        } else if (valid) {
                            uint4 *dst = reinterpret_cast<uint4 *>(out + d);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t w[4];
#pragma unroll
                                for (int n = 0; n < 4; ++n)
                                    w[n] = none ? 0u : pack_pair<T>(__uint_as_float(o[8 * j + 2 * n]),
                                                                    __uint_as_float(o[8 * j + 2 * n + 1]));
                                dst[j] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        }
                        __syncwarp();
                    }
                }
            }
            if (merge) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.merge_read);
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kSoftmaxWarps) tmem_dealloc(tmem, kTmemCols);
}

// Joins the parts of a row: out = sum_j 2^(M_j - M) O_j / sum_j 2^(M_j - M) l_j, M_j what the part's weights were
// taken against (in log2), M the largest of them.  One warp a row; parts in their order, so the result does not
// depend on which block was first.
template <typename T, int D>
__global__ void __launch_bounds__(128) attention_join_kernel(const __grid_constant__ KernelParams p, int parts) {
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    const int64_t rows = p.a.args.tokens * p.a.args.q_heads;
    const int64_t token = row / p.a.args.q_heads;
    const int head = static_cast<int>(row - token * p.a.args.q_heads);
    const int b = row < rows ? find_stream(p.a.cache.starts, p.a.cache.streams, token) : p.a.cache.streams;
    grid_dependency_wait();
    if (b >= p.a.cache.streams) return;  // no stream's
    const int64_t length = p.a.cache.lengths[b];
    const Visible seen = visible_keys(length - p.a.cache.starts[b + 1] + token, length, p.a.args.window, p.a.args.sinks,
                                      p.a.args.frame);
    float top = -INFINITY;
    for (int j = lane; j < parts; j += 32) top = fmaxf(top, p.part_ml[j * rows + row].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.0f : top;
    constexpr int kPer = D / 32;
    float acc[kPer], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = 0.0f;
    for (int j = 0; j < parts; ++j) {
        const float2 ml = p.part_ml[j * rows + row];
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;  // nothing visible in this part
        const float w = exp2_approx(ml.x - base);
        sum = fmaf(w, ml.y, sum);
        const float *o = p.part_o + (j * rows + row) * D + lane * kPer;
#pragma unroll
        for (int e = 0; e < kPer; ++e) acc[e] = fmaf(w, o[e], acc[e]);
    }
    const bool none = seen.first <= 0 && seen.high <= seen.low;
    T *out = static_cast<T *>(p.a.out.data) + token * p.a.out.token_stride + head * p.a.out.head_stride + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e) out[e] = from_float<T>(none ? 0.0f : acc[e] / sum);
}

// ---- host side -------------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// Keys of one TMA box: the largest power of two that divides the page, at most a tile.
int box_rows(int page_size) {
    int rows = 8;
    while (rows < kKeys && page_size % (rows * 2) == 0) rows *= 2;
    return rows;
}

bool page_map(CUtensorMap *map, const dcn_paged_cache &c, void *base, int64_t slot, int64_t head, int64_t page) {
    auto fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(c.page_size),
                                static_cast<cuuint64_t>(c.heads), static_cast<cuuint64_t>(c.pages)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(slot) * 2, static_cast<cuuint64_t>(head) * 2,
                                   static_cast<cuuint64_t>(page) * 2};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows(c.page_size)), 1, 1};
    const cuuint32_t step[4] = {1, 1, 1, 1};
    return fn(map, c.dtype == DCN_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base,
              dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
    bool shared;
    int ratio, tile_tokens, row_blocks, splits, parts;  // parts == 0: no join
    int64_t items;
};

Plan make_plan(const dcn_paged_cache &c, const dcn_token_attention_args &a) {
    Plan plan{};
    plan.ratio = a.q_heads / c.heads;
    plan.tile_tokens = kRows / plan.ratio;
    // The limits are hints and may be loose: no step is longer than all tokens, no stream than its row of pages.
    const int32_t max_q = static_cast<int32_t>(a.max_q < a.tokens ? a.max_q : a.tokens);
    const int64_t room = static_cast<int64_t>(c.table_columns) * c.page_size;
    const int32_t max_kv = static_cast<int32_t>(a.max_kv < room ? a.max_kv : room);
    plan.shared = max_q > plan.tile_tokens;
    const int block_tokens = plan.tile_tokens * (plan.shared ? 2 : 1);
    plan.row_blocks = max_q > 0 ? (max_q - 1) / block_tokens + 1 : 1;
    // One long step among many streams: an item takes several row blocks (Walk) rather than have millions of empty items.
    const int64_t most = kMaxItems / (static_cast<int64_t>(c.heads) * c.streams + 1) + 1;
    if (plan.row_blocks > most) plan.row_blocks = static_cast<int>(most);
    const int64_t blocks = static_cast<int64_t>(plan.row_blocks) * c.heads * c.streams;
    // Key tiles of a row block, at most.
    auto keys_of = [&](int32_t frames) {
        return frames > max_kv / a.frame ? int64_t{max_kv} : static_cast<int64_t>(frames) * a.frame;
    };
    const int64_t span = keys_of(a.window) + keys_of(a.sinks) + block_tokens;
    const int64_t tiles = (span < max_kv ? span : max_kv) / kKeys + 1;
    // Split the keys of a row block over as many blocks as make the whole shortest: rounds of the
    // GPU's blocks, each as long as its tiles plus a fixed part (start, queries, result), plus the join.  Both parts are
    // three tiles' time: with a join for nothing, 1,944 tokens of 2 heads over 29 of their keys were split and took 25.0 us
    // where unsplit they take 20.8.  Neither figure is a sharp one.
    const int streams = plan.shared ? 1 : 2;
    int64_t best = INT64_MAX;
    plan.splits = 1;
    for (int s = 1; s <= 64 && (s == 1 || s * streams <= tiles); ++s) {
        const int64_t rounds = (blocks * s + kSmCount - 1) / kSmCount;
        const int64_t cost = rounds * ((tiles + s * streams - 1) / (s * streams) + 3) + (s > 1 ? 3 : 0);
        if (cost < best) {
            best = cost;
            plan.splits = s;
        }
    }
    plan.parts = plan.splits == 1 ? 0 : plan.splits * streams;
    plan.items = blocks * plan.splits;
    return plan;
}

int64_t part_rows(const Plan &plan, const dcn_token_attention_args &a) {
    return static_cast<int64_t>(plan.parts) * a.tokens * a.q_heads;
}

template <typename T, int D, bool Shared>
cudaError_t launch(const KernelParams &k, const Plan &plan, const CUtensorMap &k_map, const CUtensorMap &v_map, int sm_count,
                   cudaStream_t stream) {
    const int grid = static_cast<int>(k.items < sm_count ? k.items : sm_count);
    attention_kernel<T, D, Shared><<<grid, kThreads, sizeof(Smem<D, Shared>) + 1024, stream>>>(k, k_map, v_map);
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || plan.parts == 0) return e;
    const int64_t rows = k.a.args.tokens * k.a.args.q_heads;
    return launch_dependent(attention_join_kernel<T, D>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(128), 0, stream, k,
                            plan.parts);
}

template <typename T>
cudaError_t launch_typed(const KernelParams &k, const Plan &plan, const CUtensorMap &k_map, const CUtensorMap &v_map,
                         int sm_count, cudaStream_t stream) {
    if (k.a.cache.head_dim == 64)
        return plan.shared ? launch<T, 64, true>(k, plan, k_map, v_map, sm_count, stream)
                           : launch<T, 64, false>(k, plan, k_map, v_map, sm_count, stream);
    return plan.shared ? launch<T, 128, true>(k, plan, k_map, v_map, sm_count, stream)
                       : launch<T, 128, false>(k, plan, k_map, v_map, sm_count, stream);
}

template <typename T, int D, bool Shared>
cudaError_t prepare() {
    const void *fn = reinterpret_cast<const void *>(attention_kernel<T, D, Shared>);
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(sizeof(Smem<D, Shared>) + 1024));
    if (e != cudaSuccess) return e;
    cudaFuncAttributes attr;
    e = cudaFuncGetAttributes(&attr, fn);
    if (e != cudaSuccess) return e;
    // The softmax warps grow to 216 registers out of what the block starts with (8 x 216 + 4 x 72 = 12 x 168).
    if (attr.maxThreadsPerBlock < kThreads || attr.numRegs < 168) return cudaErrorInvalidConfiguration;
    return cudaSuccess;
}

}  // namespace

bool token_attention_tensor(const dcn_paged_cache &c, const dcn_token_attention_args &a) {
    if (c.dtype != DCN_DTYPE_F16 && c.dtype != DCN_DTYPE_BF16) return false;
    if ((c.head_dim != 64 && c.head_dim != 128) || a.q_heads / c.heads > kRows || c.page_size % 8 != 0) return false;
    if (reinterpret_cast<uintptr_t>(c.keys) % 16 != 0 || reinterpret_cast<uintptr_t>(c.values) % 16 != 0) return false;
    const int64_t strides[] = {c.key_page_stride,   c.key_slot_stride,   c.key_head_stride,
                               c.value_page_stride, c.value_slot_stride, c.value_head_stride};
    for (int64_t s : strides)
        if (s <= 0 || s % 8 != 0 || s >= (int64_t{1} << 39)) return false;
    return true;
}

size_t token_attention_tensor_workspace(const dcn_paged_cache &c, const dcn_token_attention_args &a) {
    const int64_t rows = part_rows(make_plan(c, a), a);
    return static_cast<size_t>(rows) * (c.head_dim * sizeof(float) + sizeof(float2));
}

cudaError_t token_attention_prepare_device() {
    cudaError_t e = prepare<__half, 64, true>();
    if (e == cudaSuccess) e = prepare<__half, 64, false>();
    if (e == cudaSuccess) e = prepare<__half, 128, true>();
    if (e == cudaSuccess) e = prepare<__half, 128, false>();
    if (e == cudaSuccess) e = prepare<__nv_bfloat16, 64, true>();
    if (e == cudaSuccess) e = prepare<__nv_bfloat16, 64, false>();
    if (e == cudaSuccess) e = prepare<__nv_bfloat16, 128, true>();
    if (e == cudaSuccess) e = prepare<__nv_bfloat16, 128, false>();
    return e;
}

cudaError_t launch_token_attention_tensor(const AttentionParams &a, void *workspace, int sm_count, uint32_t *err,
                                          cudaStream_t stream) {
    const Plan plan = make_plan(a.cache, a.args);
    if (plan.items >= (int64_t{1} << 30)) return cudaErrorInvalidConfiguration;
    KernelParams k{};
    k.a = a;
    if (plan.parts > 0) {
        k.part_o = static_cast<float *>(workspace);
        k.part_ml = reinterpret_cast<float2 *>(k.part_o + part_rows(plan, a.args) * a.cache.head_dim);
    }
    k.err = err;
    k.ratio = plan.ratio;
    k.per_ratio = (65536 + plan.ratio - 1) / plan.ratio;
    k.tile_tokens = plan.tile_tokens;
    k.row_blocks = plan.row_blocks;
    k.splits = plan.splits;
    k.box_rows = box_rows(a.cache.page_size);
    k.items = static_cast<int>(plan.items);
    // Above zero, so that a hidden key's score of -inf stays -inf.  The smallest normal makes every weight 1 as 0 would,
    // to 2^-6 for products of 2^120 and to FP32's rounding below 2^102.
    const float c = fabsf(a.args.scale) * 1.4426950408889634f;
    k.c = c > FLT_MIN ? c : FLT_MIN;
    k.negate = a.args.scale < 0.0f;
    CUtensorMap k_map, v_map;
    const dcn_paged_cache &cache = a.cache;
    if (!page_map(&k_map, cache, cache.keys, cache.key_slot_stride, cache.key_head_stride, cache.key_page_stride) ||
        !page_map(&v_map, cache, cache.values, cache.value_slot_stride, cache.value_head_stride, cache.value_page_stride))
        return cudaErrorInvalidValue;
    return a.cache.dtype == DCN_DTYPE_F16 ? launch_typed<__half>(k, plan, k_map, v_map, sm_count, stream)
                                          : launch_typed<__nv_bfloat16>(k, plan, k_map, v_map, sm_count, stream);
}

}  // namespace dcn
