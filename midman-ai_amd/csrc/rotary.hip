// Rotary positions: both pair layouts, a part of the head, given positions, and
// tables whose frequencies are scaled for contexts longer than the trained one.
//
//   (a, b) -> (a c - b s, b c + a s) for the pairs (i, i + width/2) or (2i, 2i + 1)
//   of a head's first `width` columns, c and s the table's row of the position;
//   the backward pass is the transpose (s negated). Products and sums round one by
//   one, so the half layout over a whole head has mmh_apply_rope's bits.
#include <algorithm>
#include <cmath>

#include "mmh_args.h"
#include "mmh_internal.h"

namespace mmh {
namespace {

struct RotaryTable {
    int64_t width, positions;
    double theta, factor, trained, low, high, amplitude;
    int scaling;
};

// The frequency of pair i, in f64.
__device__ double frequency(const RotaryTable &p, int64_t i) {
    const double base =
        p.scaling == MMH_ROTARY_BASE && p.width > 2 ? p.theta * pow(p.factor, (double)p.width / (double)(p.width - 2)) : p.theta;
    const double w = pow(base, -2.0 * (double)i / (double)p.width);
    if (p.scaling == MMH_ROTARY_LINEAR) return w / p.factor;
    if (p.scaling == MMH_ROTARY_PARTS) {
        const double turns = p.trained * w / 6.283185307179586476925;
        const double kept = fmin(fmax((turns - p.low) / (p.high - p.low), 0.0), 1.0);
        return w * (kept + (1.0 - kept) / p.factor);
    }
    return w;
}

__global__ __launch_bounds__(256) void rotary_tables_kernel(RotaryTable p, float *cos_t, float *sin_t) {
    const int64_t half = p.width / 2, n = p.positions * half;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < n; at += (int64_t)gridDim.x * 256) {
        double s, c;
        sincos((double)(at / half) * frequency(p, at % half), &s, &c);
        cos_t[at] = (float)(c * p.amplitude);
        sin_t[at] = (float)(s * p.amplitude);
    }
}

struct RotaryArgs {
    const float *q, *k, *cos_t, *sin_t;
    float *q_out, *k_out;
    const int32_t *positions;  // device [b, t], or null: 0 .. t-1
    int64_t b, h, hkv, t, hd, width;
    int interleaved;
    float sign;
};

__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p) {
    const int64_t half = p.width / 2, units = half + p.hd - p.width;
    const int64_t rows_q = p.q ? p.b * p.h * p.t : 0, rows_k = p.k ? p.b * p.hkv * p.t : 0;
    const int64_t n = (rows_q + rows_k) * units;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < n; at += (int64_t)gridDim.x * 256) {
        int64_t row = at / units;
        const int64_t u = at - row * units;
        const bool is_k = row >= rows_q;
        if (is_k) row -= rows_q;
        const float *x = (is_k ? p.k : p.q) + row * p.hd;
        float *out = (is_k ? p.k_out : p.q_out) + row * p.hd;
        if (u >= half) {
            out[u + half] = x[u + half];
            continue;
        }
        const int64_t t = row % p.t, b = row / (p.t * (is_k ? p.hkv : p.h));
        const int64_t at_row = (p.positions ? p.positions[b * p.t + t] : t) * half + u;
        const float c = p.cos_t[at_row], s = p.sin_t[at_row] * p.sign;
        const int64_t i0 = p.interleaved ? 2 * u : u, i1 = p.interleaved ? i0 + 1 : u + half;
        const float x0 = x[i0], x1 = x[i1];
        out[i0] = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, s));
        out[i1] = __fadd_rn(__fmul_rn(x1, c), __fmul_rn(x0, s));
    }
}

int32_t rotate(mmh_handle ctx, int32_t layout, const float *q, const float *k, const int32_t *positions, int64_t b,
               int64_t h, int64_t hkv, int64_t t, int64_t hd, int64_t width, int64_t table, const float *cos_dev,
               const float *sin_dev, float *q_out, float *k_out, float sign) {
    if (layout != MMH_ROTARY_HALF && layout != MMH_ROTARY_INTERLEAVED)
        fail(MMH_ERR_ARGUMENT, "rotary: unknown layout " + std::to_string(layout));
    need(cos_dev, "cos");
    need(sin_dev, "sin");
    if (!q && !k) fail(MMH_ERR_ARGUMENT, "rotary: neither q nor k is given");
    if (q) need(q_out, "q_out");
    if (k) need(k_out, "k_out");
    bounded(b, "batch");
    bounded(t, "time");
    bounded(hd, "head_dim");
    if (q) bounded(h, "n_heads");
    if (k) bounded(hkv, "n_kv_heads");
    bounded(table, "table");
    if (width < 2 || (width & 1) || width > hd)
        fail(MMH_ERR_SHAPE, "rotary: width must be even and 2 to " + std::to_string(hd) + ", got " + std::to_string(width));
    const int64_t places = extent(b, t, "positions");
    const int64_t nq = q ? extent(extent(places, h, "q"), hd, "q") : 0, nk = k ? extent(extent(places, hkv, "k"), hd, "k") : 0;
    if (!positions && t > table)
        fail(MMH_ERR_SHAPE, "rotary: " + std::to_string(t) + " positions but tables of " + std::to_string(table));
    if (positions) check_ids(positions, places, table, "rotary position");
    const int64_t nt = extent(table, width / 2, "tables");
    const Span sc{cos_dev, nt, "cos"}, ss{sin_dev, nt, "sin"}, sq{q, nq, "q"}, sk{k, nk, "k"};
    const Span oq{q ? q_out : nullptr, nq, "q_out"}, ok{k ? k_out : nullptr, nk, "k_out"};
    apart_or_same(oq, {sq});
    apart_or_same(ok, {sk});
    apart(oq, {sk, ok, sc, ss});
    apart(ok, {sq, sc, ss});
    Context &cx = context(ctx);
    RotaryArgs p{q, k, cos_dev, sin_dev, q_out, k_out, nullptr, b, h, hkv, t, hd, width, layout == MMH_ROTARY_INTERLEAVED, sign};
    if (positions) p.positions = cx.stage_ids(positions, places, 0);
    const int64_t n = (nq + nk) / hd * (hd - width / 2);
    hipLaunchKernelGGL(rotary_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 65536)), dim3(256), 0, cx.stream, p);
    check_hip(hipGetLastError(), "rotary launch");
    return MMH_OK;
}

}  // namespace
}  // namespace mmh

using namespace mmh;

extern "C" {

int32_t mmh_rotary_tables(mmh_handle ctx, int64_t width, int64_t positions, float theta, int32_t scaling, float factor,
                          int64_t trained, float low, float high, float amplitude, float *cos_dev, float *sin_dev) {
    return guard([&] {
        need(cos_dev, "cos");
        need(sin_dev, "sin");
        bounded(width, "width");
        if (width & 1) fail(MMH_ERR_SHAPE, "rotary_tables: width must be even, got " + std::to_string(width));
        bounded(positions, "positions");
        const int64_t n = extent(positions, width / 2, "tables");
        auto above_zero = [](float v, const char *what) {
            if (!(std::isfinite(v) && v > 0.0f))
                fail(MMH_ERR_ARGUMENT, std::string("rotary_tables: ") + what + " must be positive and finite");
        };
        above_zero(theta, "theta");
        above_zero(amplitude, "amplitude");
        if (scaling < MMH_ROTARY_NONE || scaling > MMH_ROTARY_PARTS)
            fail(MMH_ERR_ARGUMENT, "rotary_tables: unknown scaling " + std::to_string(scaling));
        if (scaling != MMH_ROTARY_NONE) above_zero(factor, "factor");
        if (scaling == MMH_ROTARY_PARTS) {
            bounded(trained, "trained length");
            if (!(std::isfinite(low) && std::isfinite(high) && low >= 0.0f && low < high))
                fail(MMH_ERR_ARGUMENT, "rotary_tables: low must be at least 0 and below high, both finite");
        }
        apart({cos_dev, n, "cos"}, {{sin_dev, n, "sin"}});
        Context &cx = context(ctx);
        const RotaryTable p{width, positions, theta, factor, (double)trained, low, high, amplitude, scaling};
        hipLaunchKernelGGL(rotary_tables_kernel, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 65536)), dim3(256),
                           0, cx.stream, p, cos_dev, sin_dev);
        check_hip(hipGetLastError(), "rotary tables launch");
        return MMH_OK;
    });
}

int32_t mmh_rotary(mmh_handle ctx, int32_t layout, const float *q, const float *k, const int32_t *positions_host,
                   int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t hd, int64_t width, int64_t table,
                   const float *cos_dev, const float *sin_dev, float *q_out, float *k_out) {
    return guard([&] {
        return rotate(ctx, layout, q, k, positions_host, b, h, hkv, t, hd, width, table, cos_dev, sin_dev, q_out, k_out, 1.0f);
    });
}

int32_t mmh_rotary_backward(mmh_handle ctx, int32_t layout, const float *dq, const float *dk,
                            const int32_t *positions_host, int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t hd,
                            int64_t width, int64_t table, const float *cos_dev, const float *sin_dev, float *dq_out,
                            float *dk_out) {
    return guard([&] {
        return rotate(ctx, layout, dq, dk, positions_host, b, h, hkv, t, hd, width, table, cos_dev, sin_dev, dq_out, dk_out, -1.0f);
    });
}

}  // extern "C"
