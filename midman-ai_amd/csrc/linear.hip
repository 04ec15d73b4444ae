// The linear layer with its epilogue, and dropout.
//
//   pre = x op(W) + bias,  out = residual + dropout(act(pre))
//   dpre = dropout(dout * act'(pre)),  dbias = column sums of dpre,
//   dx = dpre op(W)^T,  dW = x^T dpre (or its transpose)
//
// Dropout's mask is drawn again wherever it is needed, from the call's key and
// counter, and never stored.
#include <algorithm>

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
// Bound by its reads and writes (2^25 values with a residual 68 us, 5.9 TB/s).
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

// dpre = dropout(dout * act'(pre)) (written where WRITE) and the column sums of
// a strip of rows of it. A wave walks rows of 256 columns, four per lane: 16-byte
// accesses, one generator block per four values. Bound by its reads and writes (4096 x
// 5632: 59 us, 4.7 TB/s).
template <bool WRITE>
__global__ __launch_bounds__(256) void linear_dpre_kernel(const float *dout, const float *pre,
                                                          int64_t rows, int64_t n, int64_t strip,
                                                          int act, Drop d, float *dpre, float *sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 256 + 4 * lane;
    const int64_t first = (int64_t)blockIdx.y * strip, last = min(rows, first + strip);
    const int count = (int)max((int64_t)0, min(n - col, (int64_t)4));
    float acc[4] = {};
    if (count > 0) {
        for (int64_t row = first + wave; row < last; row += 4) {
            const int64_t i = row * n + col;
            float v[4], x[4] = {};
            load4(dout + i, count, v);
            if (act != MMH_ACT_NONE) load4(pre + i, count, x);
            // (drawn while the loads are on their way, applied last: a dropped value is 0
            // whatever dout and pre hold)
            uint32_t w[4] = {};
            if (d.on) drop_words4(d, i, w);
            activate_grad4(act, x, v);
            if (d.on) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = drop_word(d, w[j], v[j]);
            }
            if (WRITE) store4(dpre + i, count, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] += v[j];
        }
    }
    if (!sums) return;
    __shared__ __attribute__((aligned(16))) float part[4][256];
    __builtin_memcpy(&part[wave][4 * lane], acc, 16);
    __syncthreads();
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j < n) {
        const int t = threadIdx.x;
        sums[blockIdx.y * n + j] = (part[0][t] + part[1][t]) + (part[2][t] + part[3][t]);
    }
}

// Strips of rows for about four workgroups per CU, of 16 rows at least and 1024 at
// most (a lane then adds 256 values one after another, and the strips' sums follow
// in 16 chains: the bias gradient of 2^21 rows rounds about 400 times).
int64_t strip_rows(const Context &ctx, int64_t rows, int64_t n) {
    const int64_t cols = (n + 255) / 256, want = std::max<int64_t>(1, 4 * (int64_t)ctx.cu_count / cols);
    const int64_t strip = std::min<int64_t>(1024, std::max<int64_t>(16, (rows + want - 1) / want));
    return std::max(strip, (rows + 65534) / 65535);  // (a grid's y)
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

GemmDesc product(const float *a, bool ta, const float *b, bool tb, float *c, int64_t m, int64_t k,
                 int64_t n) {
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
    g.split_bytes = kTrainSplitBytes;
    return g;
}
GemmDesc dx_product(bool nt, const float *dpre, const float *w, float *dx, int64_t rows, int64_t k, int64_t n) {
    return product(dpre, false, w, !nt, dx, rows, n, k);
}
GemmDesc dw_product(bool nt, const float *x, const float *dpre, float *dw, int64_t rows, int64_t k, int64_t n) {
    return nt ? product(dpre, true, x, false, dw, n, rows, k) : product(x, true, dpre, false, dw, k, rows, n);
}

}  // namespace
}  // namespace mmh

using namespace mmh;

extern "C" {

// For the tests, not part of the C ABI: the tile (rows, columns) and the K splits of
// mmh_linear for arrays at `at` (forward), or the tile and the splits of dx and dw
// that mmh_linear_backward takes in one launch, zeros where it takes two.
int32_t mmh_test_linear_plan(mmh_handle ctx, int32_t form, float *at, int64_t rows, int64_t k, int64_t n,
                             int32_t backward, int32_t *plan) {
    return guard([&] {
        need(plan, "plan");
        check_linear(form, rows, k, n, MMH_ACT_NONE);
        Context &cx = context(ctx);
        const bool nt = form == MMH_GEMM_NT;
        LinearTail tail;
        tail.out = at;
        GemmDesc g = backward ? dx_product(nt, at, at, at, rows, k, n) : product(at, false, at, nt, nullptr, rows, k, n);
        g.plan = plan;
        if (backward) {
            gemm_pair(cx, g, dw_product(nt, at, at, at, rows, k, n));
        } else {
            g.epi = EPI_LINEAR;
            g.tail = &tail;
            gemm(cx, g);
        }
        return MMH_OK;
    });
}

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
        LinearTail tail;
        tail.bias = bias;
        tail.residual = residual;
        tail.pre = pre;
        tail.out = out;
        tail.act = activation;
        tail.drop = d;
        GemmDesc g = product(x, false, w, form == MMH_GEMM_NT, nullptr, rows, k, n);
        g.epi = EPI_LINEAR;
        g.tail = &tail;
        gemm(cx, g);
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
        const bool changes = activation != MMH_ACT_NONE || d.on;
        if (changes || dbias) {
            const int64_t strip = strip_rows(cx, rows, n), strips = (rows + strip - 1) / strip;
            const size_t values = changes ? ((size_t)(rows * n) + 63) / 64 * 64 : 0;
            const bool several = dbias && strips > 1;
            float *buf = static_cast<float *>(
                cx.workspace(2, (values + (several ? (size_t)(strips * n) : 0)) * 4));
            float *sums = several ? buf + values : dbias;
            const dim3 grid((unsigned)((n + 255) / 256), (unsigned)strips);
            if (changes) {
                hipLaunchKernelGGL(linear_dpre_kernel<true>, grid, dim3(256), 0, cx.stream, dout, pre, rows,
                                   n, strip, activation, d, buf, sums);
                dpre = buf;
            } else {
                hipLaunchKernelGGL(linear_dpre_kernel<false>, grid, dim3(256), 0, cx.stream, dout, pre, rows,
                                   n, strip, activation, d, nullptr, sums);
            }
            check_hip(hipGetLastError(), "linear dpre launch");
            if (several) launch_sum_rows(cx, sums, strips, n, dbias);
        }
        const GemmDesc to_x = dx_product(nt, dpre, w, dx, rows, k, n);
        const GemmDesc to_w = dw_product(nt, x, dpre, dw, rows, k, n);
        if (dx && dw) gemm_pair(cx, to_x, to_w);
        else if (dx) gemm(cx, to_x);
        else if (dw) gemm(cx, to_w);
        return MMH_OK;
    });
}

}  // extern "C"
