// Argument checks shared by the entry points of the C ABI.
#pragma once

#include <cstdint>
#include <initializer_list>
#include <string>

#include "mmh_error.h"

namespace mmh {

inline void need(const void *p, const char *what) {
    if (!p) fail(MMH_ERR_ARGUMENT, std::string(what) + " is a null pointer");
}
inline void positive(int64_t v, const char *what) {
    if (v <= 0) fail(MMH_ERR_SHAPE, std::string(what) + " must be at least 1, got " + std::to_string(v));
}
// A size whose tile counts the kernels hold in 32 bits.
inline void bounded(int64_t v, const char *what) {
    positive(v, what);
    if (v > INT32_MAX)
        fail(MMH_ERR_SHAPE, std::string(what) + " must be below 2^31, got " + std::to_string(v));
}
// rows * cols, at most 2^46 values (no device holds more; their byte offsets fit 64 bits).
inline int64_t extent(int64_t rows, int64_t cols, const char *what) {
    if (rows > (int64_t(1) << 46) / cols)
        fail(MMH_ERR_SHAPE, std::string(what) + " of " + std::to_string(rows) + " x " +
                                std::to_string(cols) + " values is too large");
    return rows * cols;
}

// One buffer of a call: a null pointer is a buffer that is not there.
struct Span {
    const void *ptr;
    int64_t floats;
    const char *what;
    bool meets(const Span &o) const {
        const uintptr_t a = reinterpret_cast<uintptr_t>(ptr), b = reinterpret_cast<uintptr_t>(o.ptr);
        return ptr && o.ptr && a < b + (uintptr_t)o.floats * 4 && b < a + (uintptr_t)floats * 4;
    }
};
// An output that meets one of these buffers would be overwritten while it is read (or written twice).
inline void apart(const Span &out, std::initializer_list<Span> others) {
    for (const Span &o : others)
        if (out.meets(o))
            fail(MMH_ERR_ARGUMENT, std::string(out.what) + " overlaps " + o.what);
}
// The same for an element-wise output, which may be the buffer itself.
inline void apart_or_same(const Span &out, std::initializer_list<Span> others) {
    for (const Span &o : others)
        if (o.ptr != out.ptr) apart(out, {o});
}

}  // namespace mmh
