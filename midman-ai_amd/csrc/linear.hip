// The linear layer with its epilogue, and dropout.
//
//   pre = x op(W) + bias,  out = residual + dropout(act(pre))
//   dpre = dropout(dout) * act'(pre),  dbias = column sums of dpre,
//   dx = dpre op(W)^T,  dW = x^T dpre (or its transpose)
//
// Dropout's mask is drawn again wherever it is needed, from the call's key and
// counter, and never stored.
#include <algorithm>
#include <cmath>

#include "mmh_args.h"
#include "mmh_elementwise.h"
#include "mmh_internal.h"

namespace mmh {

Drop make_drop(float p, uint64_t seed, uint64_t offset) {
    if (!(p >= 0.0f && p <= 1.0f))
        fail(MMH_ERR_ARGUMENT, "dropout: p must be in [0, 1], got " + std::to_string(p));
    Drop d;
    const uint64_t t = (uint64_t)((double)p * 4294967296.0);
    d.on = t > 0;
    d.last = (uint32_t)(t - 1);
    d.scale = p < 1.0f ? (float)(1.0 / (1.0 - (double)p)) : 0.0f;
    d.k0 = (uint32_t)seed;
    d.k1 = (uint32_t)(seed >> 32);
    d.offset = offset;
    return d;
}

namespace {

bool al16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

unsigned grid_for(int64_t work, int per_block = 256) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((work + per_block - 1) / per_block, 65536));
}

// out = residual + dropout(x), four values and one generator block per step.
// Bound by its reads and writes.
template <bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(const float *x, const float *residual,
                                                      int64_t n, Drop d, float *out) {
    const int64_t groups = (n + 3) / 4;
    for (int64_t g = (int64_t)blockIdx.x * 256 + threadIdx.x; g < groups; g += (int64_t)gridDim.x * 256) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (d.on) w = philox(d.offset + (uint64_t)g, d.k0, d.k1);
        const int64_t i = 4 * g;
        if (VEC && i + 4 <= n) {
            float4 v = *reinterpret_cast<const float4 *>(x + i);
            if (d.on) {
                v.x = drop_word(d, w.x, v.x);
                v.y = drop_word(d, w.y, v.y);
                v.z = drop_word(d, w.z, v.z);
                v.w = drop_word(d, w.w, v.w);
            }
            if (residual) {
                const float4 r = *reinterpret_cast<const float4 *>(residual + i);
                v = make_float4(r.x + v.x, r.y + v.y, r.z + v.z, r.w + v.w);
            }
            *reinterpret_cast<float4 *>(out + i) = v;
            continue;
        }
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j >= n) break;
            float v = x[i + j];
            if (d.on) v = drop_word(d, ws[j], v);
            out[i + j] = residual ? residual[i + j] + v : v;
        }
    }
}

void launch_dropout(Context &ctx, const float *x, const float *residual, int64_t n, const Drop &d,
                    float *out) {
    const bool vec = al16(x) && al16(out) && (!residual || al16(residual));
    const dim3 grid(grid_for((n + 3) / 4));
    if (vec)
        hipLaunchKernelGGL(dropout_kernel<true>, grid, dim3(256), 0, ctx.stream, x, residual, n, d, out);
    else
        hipLaunchKernelGGL(dropout_kernel<false>, grid, dim3(256), 0, ctx.stream, x, residual, n, d, out);
    check_hip(hipGetLastError(), "dropout launch");
}

// out = residual + dropout(act(prod + bias)); pre (when wanted) = prod + bias.
__global__ __launch_bounds__(256) void linear_finish_kernel(const float *prod, const float *bias,
                                                            const float *residual, int64_t total,
                                                            int64_t n, int act, Drop d, float *pre,
                                                            float *out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float v = prod[i];
        if (bias) v += bias[i % n];
        if (pre) pre[i] = v;
        v = activate(act, v);
        if (d.on) v = drop_value(d, i, v);
        out[i] = residual ? residual[i] + v : v;
    }
}

// dpre = dropout(dout) * act'(pre)
__global__ __launch_bounds__(256) void linear_dpre_kernel(const float *dout, const float *pre,
                                                          int64_t total, int act, Drop d,
                                                          float *dpre) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        float v = dout[i];
        if (d.on) v = drop_value(d, i, v);
        dpre[i] = activate_grad(act, pre ? pre[i] : 0.0f, v);
    }
}

// Column sums of y [rows, n] in 64 bits, a thread per column.
__global__ __launch_bounds__(64) void column_sums_kernel(const float *y, int64_t rows, int64_t n,
                                                         float *out) {
    const int64_t j = (int64_t)blockIdx.x * 64 + threadIdx.x;
    if (j >= n) return;
    double s = 0.0;
    for (int64_t i = 0; i < rows; ++i) s += (double)y[i * n + j];
    out[j] = (float)s;
}

void check_linear(int32_t form, int64_t rows, int64_t k, int64_t n, int32_t act) {
    if (form != MMH_GEMM_NN && form != MMH_GEMM_NT)
        fail(MMH_ERR_ARGUMENT, "linear: form must be nn or nt, got " + std::to_string(form));
    bounded(rows, "rows");
    bounded(k, "k");
    bounded(n, "n");
    extent(rows, k, "x");
    extent(k, n, "w");
    extent(rows, n, "out");
    if (act < MMH_ACT_NONE || act > MMH_ACT_SILU)
        fail(MMH_ERR_ARGUMENT, "linear: unknown activation " + std::to_string(act));
}

void product(Context &cx, const float *a, bool ta, const float *b, bool tb, float *c, int64_t m,
             int64_t k, int64_t n) {
    GemmDesc g;
    g.a = a;
    g.ta = ta;
    g.lda = ta ? m : k;
    g.b = b;
    g.tb = tb;
    g.ldb = tb ? k : n;
    g.c = c;
    g.ldc = n;
    g.m = m;
    g.k = k;
    g.n = n;
    gemm(cx, g);
}

}  // namespace
}  // namespace mmh

using namespace mmh;

extern "C" {

int32_t mmh_dropout(mmh_handle ctx, const float *x, const float *residual, int64_t n, float p,
                    uint64_t seed, uint64_t offset, float *out) {
    return guard([&] {
        need(x, "x");
        need(out, "out");
        positive(n, "n");
        extent(n, 1, "x");
        const Drop d = make_drop(p, seed, offset);
        apart_or_same({out, n, "out"}, {{x, n, "x"}, {residual, n, "residual"}});
        Context &cx = context(ctx);
        launch_dropout(cx, x, residual, n, d, out);
        return MMH_OK;
    });
}

int32_t mmh_dropout_backward(mmh_handle ctx, const float *dout, int64_t n, float p, uint64_t seed,
                             uint64_t offset, float *dx) {
    return guard([&] {
        need(dout, "dout");
        need(dx, "dx");
        positive(n, "n");
        extent(n, 1, "dout");
        const Drop d = make_drop(p, seed, offset);
        apart_or_same({dx, n, "dx"}, {{dout, n, "dout"}});
        Context &cx = context(ctx);
        launch_dropout(cx, dout, nullptr, n, d, dx);
        return MMH_OK;
    });
}

int32_t mmh_linear(mmh_handle ctx, int32_t form, const float *x, const float *w, const float *bias,
                   const float *residual, int64_t rows, int64_t k, int64_t n, int32_t activation,
                   float p, uint64_t seed, uint64_t offset, float *pre, float *out) {
    return guard([&] {
        need(x, "x");
        need(w, "w");
        need(out, "out");
        check_linear(form, rows, k, n, activation);
        const Drop d = make_drop(p, seed, offset);
        const Span sx{x, rows * k, "x"}, sw{w, k * n, "w"}, sb{bias, n, "bias"},
            sr{residual, rows * n, "residual"}, so{out, rows * n, "out"};
        apart(so, {sx, sw, sb});
        apart_or_same(so, {sr});
        apart({pre, rows * n, "pre"}, {sx, sw, sb, sr, so});
        Context &cx = context(ctx);
        float *prod = pre ? pre : static_cast<float *>(cx.workspace(2, (size_t)(rows * n) * 4));
        product(cx, x, false, w, form == MMH_GEMM_NT, prod, rows, k, n);
        hipLaunchKernelGGL(linear_finish_kernel, dim3(grid_for(rows * n)), dim3(256), 0, cx.stream, prod,
                           bias, residual, rows * n, n, activation, d, pre, out);
        check_hip(hipGetLastError(), "linear epilogue launch");
        return MMH_OK;
    });
}

int32_t mmh_linear_backward(mmh_handle ctx, int32_t form, const float *x, const float *w,
                            const float *pre, const float *dout, int64_t rows, int64_t k, int64_t n,
                            int32_t activation, float p, uint64_t seed, uint64_t offset, float *dx,
                            float *dw, float *dbias) {
    return guard([&] {
        need(dout, "dout");
        check_linear(form, rows, k, n, activation);
        if (activation != MMH_ACT_NONE) need(pre, "pre (of an activation)");
        if (dx) need(w, "w");
        if (dw) need(x, "x");
        const Drop d = make_drop(p, seed, offset);
        const Span sx{x, rows * k, "x"}, sw{w, k * n, "w"}, sp{pre, rows * n, "pre"},
            sd{dout, rows * n, "dout"}, gx{dx, rows * k, "dx"}, gw{dw, k * n, "dw"},
            gb{dbias, n, "dbias"};
        apart(gx, {sx, sw, sp, sd, gw, gb});
        apart(gw, {sx, sw, sp, sd, gb});
        apart(gb, {sx, sw, sp, sd});
        Context &cx = context(ctx);
        if (!dx && !dw && !dbias) return MMH_OK;
        const bool nt = form == MMH_GEMM_NT;
        const float *dpre = dout;
        if (activation != MMH_ACT_NONE || d.on) {
            float *buf = static_cast<float *>(cx.workspace(2, (size_t)(rows * n) * 4));
            hipLaunchKernelGGL(linear_dpre_kernel, dim3(grid_for(rows * n)), dim3(256), 0, cx.stream, dout,
                               pre, rows * n, activation, d, buf);
            check_hip(hipGetLastError(), "linear dpre launch");
            dpre = buf;
        }
        if (dbias) {
            hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)((n + 63) / 64)), dim3(64), 0, cx.stream,
                               dpre, rows, n, dbias);
            check_hip(hipGetLastError(), "linear dbias launch");
        }
        if (dx) product(cx, dpre, false, w, !nt, dx, rows, n, k);
        if (dw && !nt) product(cx, x, true, dpre, false, dw, k, rows, n);
        if (dw && nt) product(cx, dpre, true, x, false, dw, n, rows, k);
        return MMH_OK;
    });
}

}  // extern "C"
