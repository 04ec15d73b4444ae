// Ids that a call takes from the host and its kernels read once.
#pragma once

#include <algorithm>

#include "mmh_internal.h"

namespace mmh {

// n ids: in the launch's own arguments up to kHere (no copy goes before the kernel: calls
// on 64 rows of 256 logits, one after another, 11.7 -> 8.9 us each), else in memory.
struct HostIds {
    static constexpr int kHere = 256;
    const int32_t *ids = nullptr;
    int32_t given = 0, from = 0;
    int32_t here[kHere] = {};
    __device__ __forceinline__ int32_t at(int64_t i) const { return ids ? ids[i] : here[from + (int)i]; }
    // Those of index `first` on.
    void skip(int64_t first) {
        if (ids) ids += first;
        else from += (int32_t)first;
    }
};
// null: none are given. Copied into `which` of the context's id buffers where they are many.
inline HostIds host_ids(Context &cx, const int32_t *host, int64_t n, int which) {
    HostIds h;
    if (!host) return h;
    h.given = 1;
    if (n <= HostIds::kHere) std::copy(host, host + n, h.here);
    else h.ids = cx.stage_ids(host, n, which);
    return h;
}

}  // namespace mmh
