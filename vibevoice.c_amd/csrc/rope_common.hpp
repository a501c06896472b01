// What the rotary kernels share: the frequency table that a launch carries in its arguments.
#pragma once

#include <math.h>

#include "row_math.hpp"

namespace vv {

constexpr int kMaxPairs = 128;      // head_dim <= 256

struct FreqTable {
    float f[kMaxPairs];
};

// The table depends only on (theta, head_dim); each host thread remembers the
// last one it built (thread-local, so concurrent callers never share state).
inline const FreqTable& host_freqs(float theta, int head_dim) {
    thread_local FreqTable table;
    thread_local float cached_theta = 0.0f;
    thread_local int cached_dim = 0;
    if (cached_dim != head_dim || cached_theta != theta) {
        const int half = head_dim / 2;
        for (int i = 0; i < kMaxPairs; ++i)
            table.f[i] = i < half ? powf(theta, -2.0f * (float)i / (float)head_dim) : 0.0f;
        cached_theta = theta;
        cached_dim = head_dim;
    }
    return table;
}

}  // namespace vv
