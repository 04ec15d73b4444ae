// Per-value device functions of the linear layer's epilogue and of dropout:
// activations with their derivatives, and the counter-based generator.
#pragma once

#include "mmh_internal.h"

namespace mmh {

// ---- activations ------------------------------------------------------------
// Written so that no digits cancel: gelu through erfc(-x / sqrt 2) instead of
// 1 + erf(x / sqrt 2), 1 - sigmoid as the other side's sigmoid.
constexpr float kRoot1_2 = 0.70710678118654752f, kInvRoot2Pi = 0.39894228040143268f;
constexpr float kTanhC0 = 0.79788456080286536f, kTanhC1 = 0.044715f;

// sigmoid(y) and sigmoid(-y): the exponential's argument is never positive.
__device__ __forceinline__ void sigmoid_pair(float y, float &s, float &r) {
    const float a = expf(-fabsf(y)), p = __fdiv_rn(1.0f, 1.0f + a), q = a * p;
    s = y < 0.0f ? q : p;
    r = y < 0.0f ? p : q;
}
// gelu's tanh form 0.5 x (1 + tanh(u)) is x sigmoid(2 u), u = C0 (x + C1 x^3).
__device__ __forceinline__ float tanh_arg2(float x) {
    return 2.0f * kTanhC0 * x * (1.0f + kTanhC1 * x * x);
}

__device__ __forceinline__ float activate(int act, float x) {
    switch (act) {
        case MMH_ACT_RELU: return x < 0.0f ? 0.0f : x;
        case MMH_ACT_GELU: return 0.5f * x * erfcf(-kRoot1_2 * x);
        case MMH_ACT_GELU_TANH: return __fdiv_rn(x, 1.0f + expf(-tanh_arg2(x)));
        case MMH_ACT_SILU: return __fdiv_rn(x, 1.0f + expf(-x));
        default: return x;
    }
}

// dh * act'(x). The terms x * (something that has reached 0) are 0 for any x,
// infinities too.
__device__ __forceinline__ float activate_grad(int act, float x, float dh) {
    switch (act) {
        case MMH_ACT_RELU: return x > 0.0f ? dh : 0.0f;
        case MMH_ACT_GELU: {
            const float phi = kInvRoot2Pi * expf(-0.5f * x * x);
            const float t = phi == 0.0f ? 0.0f : x * phi;
            return dh * (0.5f * erfcf(-kRoot1_2 * x) + t);
        }
        case MMH_ACT_GELU_TANH: {
            float s, r;
            sigmoid_pair(tanh_arg2(x), s, r);
            const float sr = s * r;
            const float t = sr == 0.0f ? 0.0f : 2.0f * kTanhC0 * x * (1.0f + 3.0f * kTanhC1 * x * x) * sr;
            return dh * (s + t);
        }
        case MMH_ACT_SILU: {
            float s, r;
            sigmoid_pair(x, s, r);
            const float sr = s * r;
            return dh * (s + (sr == 0.0f ? 0.0f : x * sr));
        }
        default: return dh;
    }
}

// ---- dropout ----------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy
// as 1, 2, 3, SC 2011): block j is the bijection of the counter (j, 0) under
// the key, four words. Value i of a tensor takes word i % 4 of block offset + i / 4.
struct Drop {
    int on = 0;         // 0: nothing is dropped
    uint32_t last = 0;  // words up to this one are dropped
    float scale = 1.0f; // 1 / (1 - p)
    uint32_t k0 = 0, k1 = 0;
    uint64_t offset = 0;
};
// p as the probability 2^-32 floor(p 2^32); p = 1 drops everything.
Drop make_drop(float p, uint64_t seed, uint64_t offset);

__device__ __forceinline__ uint4 philox(uint64_t block, uint32_t k0, uint32_t k1) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = 0, c3 = 0;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return make_uint4(c0, c1, c2, c3);
}
__device__ __forceinline__ float drop_word(const Drop &d, uint32_t word, float x) {
    return word <= d.last ? 0.0f : x * d.scale;
}
// Value i alone (a block for one of its four words).
__device__ __forceinline__ float drop_value(const Drop &d, int64_t i, float x) {
    const uint4 w = philox(d.offset + ((uint64_t)i >> 2), d.k0, d.k1);
    const int j = (int)(i & 3);
    return drop_word(d, j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : w.w, x);
}

}  // namespace mmh
