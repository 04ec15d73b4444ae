// Cross entropy of a linear head, straight from the hidden states:
//   z = x op(W), loss = mean over the kept rows of ln sum_j exp(z_j) - z_target,
//   dz = (softmax(z) - onehot) / kept, dx = dz op(W)^T, dW = x^T dz (or dz^T x).
//
// The logits are never whole in memory: the loss alone folds into the head's
// product (EPI_CE: a maximum and a sum per row and 128 columns), and the
// gradients take blocks of rows, whose logits become dz in place in a workspace
// of kLogitBytes. Rows whose target is `ignore` are left out before the first
// product, so nothing they hold (infinities, NaN) reaches a sum.
#include <algorithm>
#include <vector>

#include "mmh_args.h"
#include "mmh_internal.h"

namespace mmh {
namespace {

// The workspace of a block's logits, and the rows that a block has at least.
constexpr int64_t kLogitBytes = int64_t(256) << 20;
constexpr int64_t kMinRows = 128;

int64_t block_rows(int64_t n, int64_t row_bytes) {
    int64_t rows = std::max(kMinRows, kLogitBytes / row_bytes);
    if (rows >= n) return n;
    // blocks of one size (the last may be smaller), in whole tiles of 256 rows
    // where a block has as many
    const int64_t blocks = (n + rows - 1) / rows;
    rows = (n + blocks - 1) / blocks;
    return rows > 256 ? (rows + 255) / 256 * 256 : rows;
}

// dx[i] = from[map[i]], a row of zeros where map[i] < 0.
__global__ __launch_bounds__(256) void spread_rows_kernel(const float *__restrict__ from,
                                                          const int32_t *__restrict__ map,
                                                          int64_t n, int64_t d,
                                                          float *__restrict__ dx) {
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int32_t m = map[i];
        for (int64_t j = threadIdx.x; j < d; j += 256)
            dx[i * d + j] = m < 0 ? 0.0f : from[(int64_t)m * d + j];
    }
}

// A row's loss, max + ln(sum exp(z - max)) - z[target], and with GRAD dz =
// (exp(z - max) / sum - onehot) * scale in its place. One workgroup per row,
// rows of ld (a multiple of 4, 16-byte aligned) floats of which v are logits;
// the maximum first, so that a NaN anywhere reaches the sum.
template <bool GRAD>
__global__ __launch_bounds__(256) void loss_rows_kernel(float *z, const int32_t *targets, int64_t ld,
                                                        int64_t v, float scale, float *row_loss) {
    __shared__ float red_m[4], red_s[4];
    const int64_t row = blockIdx.x;
    float4 *z4 = reinterpret_cast<float4 *>(z + row * ld);
    const int64_t v4 = (v + 3) / 4;
    const int32_t t = targets[row];
    const float zt = z[row * ld + t];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    auto load = [&](int64_t q) {
        float4 a = z4[q];
        if (4 * q + 1 >= v) a.y = -INFINITY;
        if (4 * q + 2 >= v) a.z = -INFINITY;
        if (4 * q + 3 >= v) a.w = -INFINITY;
        return a;
    };
    float m = -INFINITY;
    for (int64_t q = threadIdx.x; q < v4; q += 256) {
        const float4 a = load(q);
        m = fmaxf(m, fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)));
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if (lane == 0) red_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
    float s = 0.0f;
    for (int64_t q = threadIdx.x; q < v4; q += 256) {
        const float4 a = load(q);
        s += (expf(a.x - m) + expf(a.y - m)) + (expf(a.z - m) + expf(a.w - m));
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if (lane == 0) red_s[wave] = s;
    __syncthreads();  // (z[target] has been read by every thread, too)
    s = (red_s[0] + red_s[1]) + (red_s[2] + red_s[3]);
    if (threadIdx.x == 0) row_loss[row] = (m + logf(s)) - zt;
    if (!GRAD) return;
    auto grad = [&](float x, int64_t j) {
        const float d = __fdiv_rn(expf(x - m), s) * scale;
        return j == t ? d - scale : d;
    };
    for (int64_t q = threadIdx.x; q < v4; q += 256) {
        float4 a = load(q);
        a.x = grad(a.x, 4 * q);
        a.y = grad(a.y, 4 * q + 1);
        a.z = grad(a.z, 4 * q + 2);
        a.w = grad(a.w, 4 * q + 3);
        z4[q] = a;
    }
}

template <bool GRAD>
void launch_loss_rows(Context &cx, float *z, const int32_t *targets, int64_t rows, int64_t ld, int64_t v,
                      float scale, float *row_loss) {
    hipLaunchKernelGGL(loss_rows_kernel<GRAD>, dim3((unsigned)rows), dim3(256), 0, cx.stream, z, targets,
                       ld, v, scale, row_loss);
    check_hip(hipGetLastError(), "loss launch");
}

// Floats of a row of stored logits: whole float4s, for the products too.
int64_t logit_row(int64_t vocab) { return (vocab + 31) / 32 * 32; }

// The rows that count.
struct Rows {
    int64_t kept = 0;
    const float *x = nullptr;          // [kept, d]
    const int32_t *targets = nullptr;  // device, [kept]
    const int32_t *map = nullptr;      // device, [n]: a row's place among the kept ones, or -1; null: all are kept
    std::vector<int32_t> host;         // what the upload reads
};

struct Head {
    int32_t form;
    const float *x, *w;
    const int32_t *targets;
    int64_t n, d, vocab;
    int32_t ignore;
};

void check_head(const Head &h) {
    if (h.form != MMH_GEMM_NN && h.form != MMH_GEMM_NT)
        fail(MMH_ERR_ARGUMENT, "linear_cross_entropy: form must be nn or nt, got " + std::to_string(h.form));
    need(h.x, "x");
    need(h.w, "w");
    need(h.targets, "target class");
    bounded(h.n, "rows");
    bounded(h.d, "d");
    bounded(h.vocab, "vocab");
    extent(h.n, h.d, "x");
    extent(h.d, h.vocab, "w");
    for (int64_t i = 0; i < h.n; ++i)
        if (h.targets[i] != h.ignore && (h.targets[i] < 0 || h.targets[i] >= h.vocab))
            fail(MMH_ERR_INDEX, "target class " + std::to_string(h.targets[i]) +
                                    " is out of range for " + std::to_string(h.vocab));
}

// Uploads the targets; with ignored rows also the kept rows' indexes and the
// map back, and packs those rows of x into `packed`.
void stage_rows(Context &cx, const Head &h, float *packed, Rows &r) {
    const int64_t pad = (h.n + 63) / 64 * 64;
    int32_t *dev = static_cast<int32_t *>(cx.workspace(1, (size_t)(3 * pad) * 4));
    r.targets = dev;
    if (r.kept == h.n) {
        check_hip(hipMemcpyAsync(dev, h.targets, (size_t)h.n * 4, hipMemcpyHostToDevice, cx.stream),
                  "targets upload");
        r.x = h.x;
        return;
    }
    r.host.assign((size_t)(3 * pad), 0);
    int32_t *t = r.host.data(), *index = t + pad, *map = index + pad;
    int32_t at = 0;
    for (int64_t i = 0; i < h.n; ++i) {
        const bool keep = h.targets[i] != h.ignore;
        map[i] = keep ? at : -1;
        if (!keep) continue;
        t[at] = h.targets[i];
        index[at++] = (int32_t)i;
    }
    check_hip(hipMemcpyAsync(dev, t, (size_t)(3 * pad) * 4, hipMemcpyHostToDevice, cx.stream),
              "targets upload");
    r.map = dev + 2 * pad;
    launch_embedding(cx, h.x, h.d, dev + pad, r.kept, packed);
    r.x = packed;
}

int64_t kept_rows(const Head &h) {
    return h.n - std::count(h.targets, h.targets + h.n, h.ignore);
}

GemmDesc head_product(const Head &h, const float *x, int64_t rows) {
    GemmDesc g;
    g.a = x;
    g.b = h.w;
    g.m = rows;
    g.k = h.d;
    g.n = h.vocab;
    g.lda = h.d;
    g.tb = h.form == MMH_GEMM_NT;
    g.ldb = g.tb ? h.d : h.vocab;
    return g;
}

size_t round64(int64_t floats) { return ((size_t)floats + 63) / 64 * 64; }

void finish_loss(Context &cx, float *loss_host) {
    check_hip(hipStreamSynchronize(cx.stream), "loss sync");
    *loss_host = cx.words[0];
}

void forward(Context &cx, const Head &h, float *loss_host) {
    Rows r;
    r.kept = kept_rows(h);
    if (r.kept == 0) {
        *loss_host = 0.0f;
        return;
    }
    const int64_t units = (h.vocab + 127) / 128;
    auto folds = [&](int64_t rows) { return gemm_ce_tiles(cx, head_product(h, h.x, rows)) > 0; };
    const int64_t ld = logit_row(h.vocab);
    const int64_t block = block_rows(r.kept, folds(r.kept) ? units * 8 : ld * 4);
    // a block's partials, or the logits of one too small for the product to fold them (the last, often)
    auto floats = [&](int64_t rows) { return rows * (folds(rows) ? units * 2 : ld); };
    const size_t packed = r.kept < h.n ? round64(r.kept * h.d) : 0;
    const size_t part = round64(std::max(floats(block), floats((r.kept - 1) % block + 1)));
    float *ws = static_cast<float *>(cx.workspace(2, (packed + part + round64(block)) * 4));
    float *row_loss = static_cast<float *>(cx.workspace(3, round64(r.kept) * 4));
    stage_rows(cx, h, ws, r);
    float *buf = ws + packed, *zt = buf + part;
    for (int64_t at = 0; at < r.kept; at += block) {
        const int64_t rows = std::min(block, r.kept - at);
        GemmDesc g = head_product(h, r.x + at * h.d, rows);
        if (folds(rows)) {
            g.epi = EPI_CE;
            g.ce_targets = r.targets + at;
            g.ce_part = buf;
            g.ce_zt = zt;
            gemm(cx, g);
            launch_ce_combine_rows(cx, buf, units, zt, rows, row_loss + at);
        } else {
            g.c = buf;
            g.ldc = ld;
            gemm(cx, g);
            launch_loss_rows<false>(cx, buf, r.targets + at, rows, ld, h.vocab, 0.0f, row_loss + at);
        }
    }
    launch_mean(cx, row_loss, r.kept, cx.words);
    finish_loss(cx, loss_host);
}

void backward(Context &cx, const Head &h, float *dx, float *dw, float *loss_host) {
    Rows r;
    r.kept = kept_rows(h);
    if (r.kept == 0) {
        if (loss_host) *loss_host = 0.0f;
        if (dx) launch_fill(cx, dx, h.n * h.d, 0.0f);
        if (dw) launch_fill(cx, dw, h.d * h.vocab, 0.0f);
        return;
    }
    const bool all = r.kept == h.n, nt = h.form == MMH_GEMM_NT;
    const int64_t ld = logit_row(h.vocab), block = block_rows(r.kept, ld * 4);
    const size_t packed = all ? 0 : round64(r.kept * h.d);
    float *ws = static_cast<float *>(
        cx.workspace(2, (packed * (dx ? 2 : 1) + round64(block * ld)) * 4));
    float *row_loss = static_cast<float *>(cx.workspace(3, round64(r.kept) * 4));
    stage_rows(cx, h, ws, r);
    float *z = ws + packed, *dxk = all ? dx : z + round64(block * ld);
    const float scale = 1.0f / (float)r.kept;
    for (int64_t at = 0; at < r.kept; at += block) {
        const int64_t rows = std::min(block, r.kept - at);
        GemmDesc g = head_product(h, r.x + at * h.d, rows);
        g.c = z;
        g.ldc = ld;
        gemm(cx, g);
        launch_loss_rows<true>(cx, z, r.targets + at, rows, ld, h.vocab, scale, row_loss + at);
        if (dx) {  // dz [rows, vocab] . op(W)^T
            GemmDesc p;
            p.a = z;
            p.b = h.w;
            p.c = dxk + at * h.d;
            p.m = rows;
            p.k = h.vocab;
            p.n = h.d;
            p.lda = ld;
            p.tb = !nt;
            p.ldb = nt ? h.d : h.vocab;
            p.ldc = h.d;
            gemm(cx, p);
        }
        if (dw) {  // x^T dz [d, vocab], or dz^T x [vocab, d]; later blocks are added
            GemmDesc p;
            p.a = nt ? z : r.x + at * h.d;
            p.b = nt ? r.x + at * h.d : z;
            p.c = dw;
            p.m = nt ? h.vocab : h.d;
            p.k = rows;
            p.n = nt ? h.d : h.vocab;
            p.ta = true;
            p.lda = nt ? ld : h.d;
            p.ldb = nt ? h.d : ld;
            p.ldc = p.n;
            p.epi = at ? EPI_ACCUM : EPI_STORE;
            gemm(cx, p);
        }
    }
    if (!all && dx) {
        hipLaunchKernelGGL(spread_rows_kernel, dim3((unsigned)std::min<int64_t>(h.n, 65536)), dim3(256), 0,
                           cx.stream, dxk, r.map, h.n, h.d, dx);
        check_hip(hipGetLastError(), "gradient rows launch");
    }
    if (loss_host) {
        launch_mean(cx, row_loss, r.kept, cx.words);
        finish_loss(cx, loss_host);
    } else {  // the upload has read the targets
        check_hip(hipStreamSynchronize(cx.stream), "targets upload sync");
    }
}

}  // namespace
}  // namespace mmh

using namespace mmh;

extern "C" {

int32_t mmh_linear_cross_entropy(mmh_handle ctx, int32_t form, const float *x, const float *w,
                                 const int32_t *targets_host, int64_t n, int64_t d, int64_t vocab,
                                 int32_t ignore, float *loss_host) {
    return guard([&] {
        const Head h{form, x, w, targets_host, n, d, vocab, ignore};
        check_head(h);
        need(loss_host, "loss");
        forward(context(ctx), h, loss_host);
        return MMH_OK;
    });
}

int32_t mmh_linear_cross_entropy_backward(mmh_handle ctx, int32_t form, const float *x,
                                          const float *w, const int32_t *targets_host, int64_t n,
                                          int64_t d, int64_t vocab, int32_t ignore, float *dx,
                                          float *dw, float *loss_host) {
    return guard([&] {
        const Head h{form, x, w, targets_host, n, d, vocab, ignore};
        check_head(h);
        const Span sx{x, n * d, "x"}, sw{w, d * vocab, "w"}, gx{dx, n * d, "dx"}, gw{dw, d * vocab, "dw"};
        apart(gx, {sx, sw, gw});
        apart(gw, {sx, sw});
        backward(context(ctx), h, dx, dw, loss_host);
        return MMH_OK;
    });
}

}  // extern "C"
