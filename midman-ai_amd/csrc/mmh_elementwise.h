// Per-value device functions of the linear layer's epilogue and of dropout:
// activations with their derivatives, and the counter-based generator.
#pragma once

#include "mmh_internal.h"

namespace mmh {

// ---- activations ------------------------------------------------------------
// The VALU's time adds to the matrix core's, so these stay short, and yet no
// digits are lost: the hardware's exp2 and reciprocal, with the rounding errors of
// their arguments carried along, and no form that cancels (1 - sigmoid is the other
// side's sigmoid, gelu's far side a tail). Over [-13, 13] gelu is off by at most 8,
// silu 4 and gelu_tanh 40 times 2^-24 of its value (the last in the far tail, whose
// exponent's rounding grows with it), the slopes by 4 times 2^-24; values below
// 2^-126 |x| may be 0.
constexpr float kTanhC0 = 0.79788456080286536f, kTanhC1 = 0.044715f;  // sqrt(2 / pi), gelu_tanh's cubic

__device__ __forceinline__ float reciprocal(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
}
// exp(x), x <= 0: 2^(x log2 e), the low part of the exponent applied as 1 + low ln 2.
__device__ __forceinline__ float exp_neg(float x) {
    constexpr float kHi = 1.44269502f, kLo = 1.92596303e-8f, kLn2 = 0.69314718f;
    x = x < -104.0f ? -104.0f : x;  // (e^-104 is below the smallest f32; a NaN stays)
    const float t = x * kHi;
    const float low = __builtin_fmaf(x, kLo, __builtin_fmaf(x, kHi, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return __builtin_fmaf(e, low * kLn2, e);
}
// sigmoid(y) and sigmoid(-y).
__device__ __forceinline__ void sigmoid_pair(float y, float &s, float &r) {
    const float a = exp_neg(-fabsf(y)), p = reciprocal(1.0f + a), q = a * p;
    s = y < 0.0f ? q : p;
    r = y < 0.0f ? p : q;
}
// gelu's tanh form 0.5 x (1 + tanh(u)) is x sigmoid(2 u), u = C0 (x + C1 x^3).
__device__ __forceinline__ float tanh_arg2(float x) {
    return 2.0f * kTanhC0 * x * __builtin_fmaf(kTanhC1 * x, x, 1.0f);
}
// e = exp(-x^2 / 2) and the normal tail Phi(-|x|) = e erfcx(|x| / sqrt 2) / 2.
// erfcx is a polynomial in t = 1 / (1 + 0.35 |x| / sqrt 2), fitted here to the
// least largest relative error over |x| <= 13.15, where its f32 coefficients are
// within 5.7e-8 (beyond, e is 0 in f32).
__device__ __forceinline__ float normal_tail(float x, float &e) {
    const float ax = fabsf(x) > 15.0f ? 15.0f : fabsf(x), sq = ax * ax;  // (a NaN stays)
    e = exp_neg(-0.5f * sq);
    e = __builtin_fmaf(e, -0.5f * __builtin_fmaf(ax, ax, -sq), e);
    const float t = reciprocal(__builtin_fmaf(0.247487373f, ax, 1.0f));
    float q = 0.06764230132102966f;
    q = __builtin_fmaf(q, t, -0.40613067150115967f);
    q = __builtin_fmaf(q, t, 0.8532063364982605f);
    q = __builtin_fmaf(q, t, -0.757356584072113f);
    q = __builtin_fmaf(q, t, 0.6861104369163513f);
    q = __builtin_fmaf(q, t, -0.08201061189174652f);
    q = __builtin_fmaf(q, t, 0.2549700140953064f);
    q = __builtin_fmaf(q, t, 0.18484941124916077f);
    q = __builtin_fmaf(q, t, 0.1987789422273636f);
    q = __builtin_fmaf(q, t, -5.9628724557114765e-05f);
    return 0.5f * e * q;
}

__device__ __forceinline__ float gelu_f(float x) {
    float e;
    const float tail = normal_tail(x, e);
    return x * (x < 0.0f ? tail : 1.0f - tail);
}
__device__ __forceinline__ float gelu_tanh_f(float x) {
    float s, r;
    sigmoid_pair(tanh_arg2(x), s, r);
    return x * s;
}
__device__ __forceinline__ float silu_sigmoid_f(float x) {
    float s, r;
    sigmoid_pair(x, s, r);
    return x * s;
}
// The slopes. A term x * (something that has reached 0) is 0 for any x,
// infinities too.
__device__ __forceinline__ float gelu_slope(float x) {
    float e;
    const float tail = normal_tail(x, e);
    const float phi = 0.39894228040143268f * e;
    return (x < 0.0f ? tail : 1.0f - tail) + (phi == 0.0f ? 0.0f : x * phi);
}
__device__ __forceinline__ float gelu_tanh_slope(float x) {
    float s, r;
    sigmoid_pair(tanh_arg2(x), s, r);
    const float sr = s * r;
    return s + (sr == 0.0f ? 0.0f : 2.0f * kTanhC0 * x * __builtin_fmaf(3.0f * kTanhC1 * x, x, 1.0f) * sr);
}
__device__ __forceinline__ float silu_slope(float x) {
    float s, r;
    sigmoid_pair(x, s, r);
    const float sr = s * r;
    return s + (sr == 0.0f ? 0.0f : x * sr);
}

// v = act(v), four values: one uniform branch for them.
__device__ __forceinline__ void activate4(int act, float (&v)[4]) {
#define MMH_EACH4(E) _Pragma("unroll") for (int j = 0; j < 4; ++j) E
    switch (act) {
        case MMH_ACT_RELU: MMH_EACH4(v[j] = v[j] < 0.0f ? 0.0f : v[j]); break;
        case MMH_ACT_GELU: MMH_EACH4(v[j] = gelu_f(v[j])); break;
        case MMH_ACT_GELU_TANH: MMH_EACH4(v[j] = gelu_tanh_f(v[j])); break;
        case MMH_ACT_SILU: MMH_EACH4(v[j] = silu_sigmoid_f(v[j])); break;
        default: break;
    }
}
// dh *= act'(x); a NaN of x or dh stays one in every activation's (relu's slope at 0 is
// 0, and the product with it is taken: an infinity of dh times 0 is a NaN)
__device__ __forceinline__ void activate_grad4(int act, const float (&x)[4], float (&dh)[4]) {
    switch (act) {
        case MMH_ACT_RELU: MMH_EACH4(dh[j] = x[j] > 0.0f ? dh[j] : x[j] <= 0.0f ? dh[j] * 0.0f : x[j]); break;
        case MMH_ACT_GELU: MMH_EACH4(dh[j] *= gelu_slope(x[j])); break;
        case MMH_ACT_GELU_TANH: MMH_EACH4(dh[j] *= gelu_tanh_slope(x[j])); break;
        case MMH_ACT_SILU: MMH_EACH4(dh[j] *= silu_slope(x[j])); break;
        default: break;
    }
#undef MMH_EACH4
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
// The words of values i .. i + 3 of an array: one block where they are its four
// words, else two that follow each other.
__device__ __forceinline__ void drop_words4(const Drop &d, int64_t i, uint32_t (&w)[4]) {
    const uint64_t block = d.offset + ((uint64_t)i >> 2);
    const uint4 a = philox(block, d.k0, d.k1);
    w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    const int first = (int)(i & 3);
    if (first) {
        const uint4 b = philox(block + 1, d.k0, d.k1);
        const uint32_t e[7] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z};
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = first == 1 ? e[j + 1] : first == 2 ? e[j + 2] : e[j + 3];
    }
}
__device__ __forceinline__ void drop4(const Drop &d, int64_t i, float (&v)[4]) {
    uint32_t w[4];
    drop_words4(d, i, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = drop_word(d, w[j], v[j]);
}

// Up to four neighbouring values of an array at any 4-byte alignment (gfx950
// moves 16 bytes at any dword); those past `count` read as 0 and are not written.
__device__ __forceinline__ void load4(const float *p, int count, float (&v)[4]) {
    if (count == 4) {
        __builtin_memcpy(v, p, 16);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = j < count ? p[j] : 0.0f;
    }
}
__device__ __forceinline__ void store4(float *p, int count, const float (&v)[4]) {
    if (count == 4) {
        __builtin_memcpy(p, v, 16);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < count) p[j] = v[j];
    }
}

// ---- the linear layer's epilogue ---------------------------------------------
// What follows the product in out = residual + dropout(act(product + bias)),
// out [rows, n] contiguous. Pointers that are not wanted are null.
struct LinearTail {
    const float *bias = nullptr, *residual = nullptr;
    float *pre = nullptr, *out = nullptr;
    int act = MMH_ACT_NONE;
    Drop drop;
};
// The part read from memory of columns col .. col + count - 1 of a row.
struct TailInputs {
    float b[4], r[4];
};
__device__ __forceinline__ void tail_load(const LinearTail &t, int64_t n, int64_t row, int64_t col,
                                          int count, TailInputs &in) {
    if (t.bias) load4(t.bias + col, count, in.b);
    if (t.residual) load4(t.residual + row * n + col, count, in.r);
}
// act and dropout of pre = v (stored where it is kept).
__device__ __forceinline__ void tail_values(const LinearTail &t, int64_t n, int64_t row, int64_t col,
                                            int count, float (&v)[4]) {
    const int64_t i = row * n + col;
    if (t.pre) store4(t.pre + i, count, v);
    activate4(t.act, v);
    if (t.drop.on) drop4(t.drop, i, v);
}
__device__ __forceinline__ void tail_finish(const LinearTail &t, int64_t n, int64_t row, int64_t col,
                                            int count, const TailInputs &in, float (&v)[4]) {
    if (t.bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] += in.b[j];
    }
    tail_values(t, n, row, col, count, v);
    if (t.residual) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = in.r[j] + v[j];
    }
    store4(t.out + row * n + col, count, v);
}

}  // namespace mmh
