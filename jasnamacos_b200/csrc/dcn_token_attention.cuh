// dcn_token_attention.cuh -- which keys a query sees, and one row of attention by one warp, for both
// attention kernels.
#pragma once

#include <stdint.h>

#include "dcn_tokens.cuh"

namespace dcn {

// The keys visible to one query: [0, first) and [low, high), with first <= low (so the two do not
// overlap); empty when the row sees nothing.
struct Visible {
    int64_t first, low, high;
};

// The query at `position` of a stream of `length` tokens: frames up to its own, the last `window`
// of them and the first `sinks`.
__host__ __device__ inline Visible visible_keys(int64_t position, int64_t length, int window, int sinks, int frame) {
    Visible v{0, 0, 0};
    if (position < 0 || length <= 0) return v;
    // Positions are below 2^31: a 32-bit division (a 64-bit one is a routine of a hundred instructions).
    const int64_t own = static_cast<uint32_t>(position) / static_cast<uint32_t>(frame);
    const int64_t end = (own + 1) * frame;
    v.high = end < length ? end : length;
    const int64_t start = (own - window + 1) * frame;
    v.low = start > 0 ? start : 0;
    const int64_t pinned = static_cast<int64_t>(sinks) * frame;
    v.first = pinned < v.low ? pinned : v.low;
    // Pinned frames that reach into the window: [first, low) is empty of hidden keys.
    if (pinned >= v.low) {
        v.first = 0;
        v.low = 0;
    }
    if (v.low > v.high) v.low = v.high;
    return v;
}

#if defined(__CUDACC__)

// One row: acc = sum_s exp2(c q.k_s - m) v_s and l = sum_s exp2(c q.k_s - m) over the keys of `parts` ranges
// that the row sees, m the largest c q.k_s.  A whole warp's call: 32 keys at a time, one a lane for the products,
// then the lanes hold the value's elements (lane + 32 i).  Hidden keys are never read, so what they hold
// cannot matter.  `q` is read by every lane (one address at a time).  `beat` (nullable) counts on while it works,
// for waits that would take a long row for a dead one.
template <typename T, int kElements>
struct RowByWarp {
    float acc[kElements], m, l;

    template <typename Q>
    __device__ __forceinline__ void run(const dcn_paged_cache &cache, int stream, int kv_head, const Q *q, float c,
                                        const Visible &seen, const int64_t (&begin)[2], const int64_t (&end)[2], int *beat) {
        const int lane = threadIdx.x & 31, d = cache.head_dim;
        const T *keys = static_cast<const T *>(cache.keys) + kv_head * cache.key_head_stride;
        const T *values = static_cast<const T *>(cache.values) + kv_head * cache.value_head_stride;
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < kElements; ++i) acc[i] = 0.0f;
        for (int part = 0; part < 2; ++part) {
            for (int64_t base = begin[part]; base < end[part]; base += 32) {
                if (beat != nullptr && lane == 0) atomicAdd(beat, 1);
                const int64_t key = base + lane;
                float score = -INFINITY;
                int64_t value_at = -1;
                if (key < end[part] && (key < seen.first || (key >= seen.low && key < seen.high))) {
                    const uint32_t column = static_cast<uint32_t>(key) / static_cast<uint32_t>(cache.page_size);
                    const int64_t slot = key - static_cast<int64_t>(column) * cache.page_size;
                    const int page = column < static_cast<uint32_t>(cache.table_columns)
                                         ? cache.table[stream * cache.table_stride + column] : -1;
                    score = 0.0f;
                    if (page >= 0 && page < cache.pages) {
                        const T *k = keys + page * cache.key_page_stride + slot * cache.key_slot_stride;
                        value_at = page * cache.value_page_stride + slot * cache.value_slot_stride;
                        for (int e = 0; e < d; ++e) score = fmaf(to_float<Q>(q[e]), to_float<T>(k[e]), score);
                    }
                    score *= c;
                }
                float top = score;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                top = fmaxf(m, top);
                // -inf so far (scores of -inf only): nothing has weight yet, and -inf - -inf is not 0.
                const float from = top == -INFINITY ? 0.0f : top;
                const float shrink = exp2f(m - from);
                const float w = exp2f(score - from);
                m = top;
                float total = w;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
                l = fmaf(l, shrink, total);
#pragma unroll
                for (int i = 0; i < kElements; ++i) acc[i] *= shrink;
                for (int s = 0; s < 32; ++s) {
                    const float ws = __shfl_sync(0xffffffffu, w, s);
                    const int64_t at = __shfl_sync(0xffffffffu, value_at, s);
                    if (at < 0) continue;  // hidden, or without a page: zeros
#pragma unroll
                    for (int i = 0; i < kElements; ++i)
                        if (i * 32 + lane < d) acc[i] = fmaf(ws, to_float<T>(values[at + i * 32 + lane]), acc[i]);
                }
            }
        }
    }
};

#endif  // __CUDACC__

}  // namespace dcn
