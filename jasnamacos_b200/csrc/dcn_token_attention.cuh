// dcn_token_attention.cuh -- which keys a query sees, for both attention kernels.
#pragma once

#include <stdint.h>

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

}  // namespace dcn
