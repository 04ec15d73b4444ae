// Shared by the losses whose row terms come back in pinned memory.
#pragma once

#include "mmh_internal.h"

namespace mmh {

// A call that fails after its first launch still waits for its kernels: they use
// the pinned memory that the next call writes.
struct Drain {
    Context &cx;
    bool done = false;
    ~Drain() {
        if (!done) (void)hipStreamSynchronize(cx.stream);
    }
};

// Waits for the call's kernels. The n row terms lie in pinned memory, and their sum over
// the `count` rows that count is taken here, in f64 and in eight sums of a fixed order: a launch of its own
// would take longer than the sum of a few thousand.
inline float mean_loss(Drain &drain, const float *rows, int64_t n, int64_t count) {
    drain.done = true;
    check_hip(hipStreamSynchronize(drain.cx.stream), "loss sync");
    double sum[8] = {};
    for (int64_t i = 0; i < n; ++i) sum[i & 7] += (double)rows[i];
    const double total = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
    return (float)(total / (double)count);
}

}  // namespace mmh
