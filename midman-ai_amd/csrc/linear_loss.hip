// Cross entropy of a linear head, straight from the hidden states:
//   z = x op(W), loss = mean over the kept rows of ln sum_j exp(z_j) - z_target,
//   dz = (softmax(z) - onehot) / kept, dx = dz op(W)^T, dW = x^T dz (or dz^T x).
//
// The loss alone folds into the head's product (EPI_CE: a maximum and a sum per
// row and 128 columns) and stores no logits; the gradients take blocks of rows,
// whose logits become dz in place in a workspace of kLogitBytes (or kMinRows rows),
// however many rows there are. (Dropping them and forming them again for dx and dW
// would cost a fourth product, a third of the time.) A pass over them reads and
// writes each row once: up to kRowCols columns from registers; for wider rows the product
// leaves the same partials beside the logits (three passes over such rows instead:
// 817 x 1024 x 131071 4650 us, 4500 so). Rows whose target is `ignore` are left out
// before the first product, so nothing they hold (infinities, NaN) reaches a sum.
#include <algorithm>

#include "mmh_args.h"
#include "mmh_elementwise.h"
#include "mmh_internal.h"
#include "mmh_loss.h"

namespace mmh {
namespace {

// The rows that a block has at least, and at most (narrow vocabularies: a launch has
// less than 2^32 threads, a row up to 512).
constexpr int64_t kMinRows = 128, kMaxRows = int64_t(1) << 22;
// Up to so many rows the loss takes stored logits: the tiles that fold it have
// 128 rows at least, those of the plain product 32 or 64 (35 rows x 1344 x 153411
// 367 -> 266 us for the product, 64 rows 372 -> 274, 128 rows 384 -> 341 and 33
// for the stored logits' two ways).
constexpr int64_t kFewRows = 64;
// So few rows past a block's last whole 256 are a part of their own beside
// weights of kTailWeights values or more: in the tiles of 256 rows they would cost
// a whole one, and they read W again for less (817 rows x 1024 x 131071 4000 ->
// 3780 us, 545 x 2048 x 32000 1480 -> 1307, 1044 x 4096 x 16000 2330 -> 2065;
// with fewer weights the further launches take that back: 320 x 1024 x 40000 617 ->
// 621, the loss alone of 1044 x 768 x 50000 521 -> 565).
constexpr int64_t kTailWeights = int64_t(52) << 20;

// The rows of the part of a block that starts at `at` of its `rows`.
int64_t part_rows(int64_t rows, int64_t at, int64_t weights) {
    const int64_t tail = rows % 256;
    if (at > 0 || rows < 256 || tail > kFewRows || weights < kTailWeights) return rows - at;
    return rows - tail;
}

// Rows of a block of n rows of row_bytes each: all, or as many as `bytes` hold, but
// kMinRows at least. Blocks of one size (the last may be smaller), in whole tiles of
// 256 rows where a block has as many: rounded up where that still fits, else down
// where that takes a quarter more blocks at most (8192 x 1024 x 152064 with 768 rows
// 42.2 ms, with 820 45.1; 514 x 768 x 522000 with 256 10.0, with 257 10.5; where it
// takes more the two are even: 670 x 1024 x 400000 with 256 or 335 11.9).
int64_t block_rows(int64_t n, int64_t row_bytes, int64_t bytes) {
    const int64_t most = std::min(kMaxRows, std::max(kMinRows, bytes / row_bytes));
    if (most >= n) return n;
    const int64_t blocks = (n + most - 1) / most, rows = (n + blocks - 1) / blocks;
    if (rows <= 256) return rows;
    const int64_t down = rows / 256 * 256, up = down == rows ? rows : down + 256;
    return up <= most ? up : 4 * rows <= 5 * down ? down : rows;
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

// Rows of stored logits of up to kRowCols columns: the row's loss, max + ln(sum
// exp(z - max)) - z[target], and with GRAD dz = (exp(z - max) / sum - onehot) *
// scale in its place. A workgroup holds a row in registers, NV float4s per
// thread, so it passes through once; rows are ld (a multiple of 4, 16-byte
// aligned) floats of which v are logits. A NaN anywhere reaches the sum. Bound by
// the logits' read and write (4096 x 32000: 194 us, 5.4 TB/s).
constexpr int64_t kRowCols = 32768;
template <int NT, int NV, bool GRAD>
__global__ __launch_bounds__(NT) void loss_rows_kernel(float *z, const int32_t *targets, int64_t ld, int v,
                                                       float scale, float *row_loss) {
    __shared__ float red_m[NT / 64], red_s[NT / 64];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, v4 = (v + 3) / 4;
    float4 *z4 = reinterpret_cast<float4 *>(z + row * ld);
    const int t = targets[row];
    float4 e[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int q = tid + NT * i;
        e[i] = z4[min(q, v4 - 1)];
        if (4 * q >= v) e[i].x = -INFINITY;
        if (4 * q + 1 >= v) e[i].y = -INFINITY;
        if (4 * q + 2 >= v) e[i].z = -INFINITY;
        if (4 * q + 3 >= v) e[i].w = -INFINITY;
    }
    const float zt = tid == 0 ? z[row * ld + t] : 0.0f;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) m = fmaxf(m, fmaxf(fmaxf(e[i].x, e[i].y), fmaxf(e[i].z, e[i].w)));
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if (lane == 0) red_m[wave] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) m = fmaxf(m, red_m[i]);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        // (columns past the row hold -inf: exp gives 0)
        e[i] = make_float4(exp_neg(e[i].x - m), exp_neg(e[i].y - m), exp_neg(e[i].z - m),
                           exp_neg(e[i].w - m));
        s += (e[i].x + e[i].y) + (e[i].z + e[i].w);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if (lane == 0) red_s[wave] = s;
    __syncthreads();  // (z[target] has been read, too)
    s = red_s[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) s += red_s[i];
    if (tid == 0) row_loss[row] = (m + logf(s)) - zt;
    if constexpr (!GRAD) return;
    const float f = __fdiv_rn(scale, s);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int q = tid + NT * i;
        if (q >= v4) break;
        float4 a = make_float4(e[i].x * f, e[i].y * f, e[i].z * f, e[i].w * f);
        if (t >> 2 == q) {
            if ((t & 3) == 0) a.x -= scale;
            if ((t & 3) == 1) a.y -= scale;
            if ((t & 3) == 2) a.z -= scale;
            if ((t & 3) == 3) a.w -= scale;
        }
        z4[q] = a;
    }
}

template <bool GRAD>
void launch_loss_rows(Context &cx, float *z, const int32_t *targets, int64_t rows, int64_t ld, int64_t v,
                      float scale, float *row_loss) {
    auto launch = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(threads), 0, cx.stream, z, targets, ld, (int)v,
                           scale, row_loss);
    };
    if (v <= 1024) launch(loss_rows_kernel<256, 1, GRAD>, 256);
    else if (v <= 4096) launch(loss_rows_kernel<256, 4, GRAD>, 256);
    else if (v <= 8192) launch(loss_rows_kernel<512, 4, GRAD>, 512);
    else if (v <= 16384) launch(loss_rows_kernel<512, 8, GRAD>, 512);
    else if (v <= kRowCols) launch(loss_rows_kernel<512, 16, GRAD>, 512);
    else fail(MMH_ERR_OTHER, "linear_cross_entropy: rows of " + std::to_string(v) + " logits without partials");
    check_hip(hipGetLastError(), "loss launch");
}

// The (max, sum) of each kPartCols columns of stored logits, and the target's
// logit: the partials of wider rows where there are too few of them for the
// product's tiles to leave any (kFewRows). A workgroup has a row's piece in registers.
constexpr int64_t kPartCols = 8192;
__global__ __launch_bounds__(256) void loss_parts_kernel(const float *z, const int32_t *targets, int64_t ld,
                                                         int64_t v, int64_t units, float2 *part, float *zt) {
    __shared__ float red_m[4], red_s[4];
    const int64_t row = blockIdx.y, unit = blockIdx.x, c0 = unit * kPartCols;
    const float4 *z4 = reinterpret_cast<const float4 *>(z + row * ld + c0);
    const int tid = threadIdx.x, wave = tid >> 6, n = (int)min(v - c0, kPartCols);
    const int64_t t = targets[row] - c0;
    float4 e[8];
    float m = -INFINITY, s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int q = tid + 256 * i;
        e[i] = z4[min(q, (n + 3) / 4 - 1)];
        if (4 * q >= n) e[i].x = -INFINITY;
        if (4 * q + 1 >= n) e[i].y = -INFINITY;
        if (4 * q + 2 >= n) e[i].z = -INFINITY;
        if (4 * q + 3 >= n) e[i].w = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fmaxf(fmaxf(e[i].x, e[i].y), fmaxf(e[i].z, e[i].w)));
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    if ((tid & 63) == 0) red_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red_m[0], red_m[1]), fmaxf(red_m[2], red_m[3]));
    const float m0 = m == -INFINITY ? 0.0f : m;  // (then every exponential is 0, or NaN)
#pragma unroll
    for (int i = 0; i < 8; ++i)
        s += (exp_neg(e[i].x - m0) + exp_neg(e[i].y - m0)) + (exp_neg(e[i].z - m0) + exp_neg(e[i].w - m0));
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if ((tid & 63) == 0) red_s[wave] = s;
    __syncthreads();
    if (tid != 0) return;
    s = (red_s[0] + red_s[1]) + (red_s[2] + red_s[3]);
    // a NaN sum keeps its place beside any maximum (a piece of -inf and NaN has no other)
    part[row * units + unit] = make_float2(s != s ? s : m, s);
    if (t >= 0 && t < n) zt[row] = z[row * ld + c0 + t];
}

// dz in place of wider rows, whose product left (max, sum) per 128 columns beside
// the logits (EPI_CE_STORE) or which loss_parts_kernel has been through. A
// workgroup has a chunk of a row: it merges the row's partials (a few KB, read by
// each of the row's workgroups), then its columns pass through once. Bound by the
// logits' read and write (817 x 131071: 170 us, 5.0 TB/s).
__global__ __launch_bounds__(256) void loss_grad_kernel(float *z, const float2 *part,
                                                        const int32_t *targets, int64_t ld, int64_t v,
                                                        int64_t units, int64_t chunk, float scale,
                                                        float *row_loss) {
    __shared__ float red_m[4], red_s[4];
    const int64_t row = blockIdx.x, q0 = blockIdx.y * (chunk / 4);
    float4 *z4 = reinterpret_cast<float4 *>(z + row * ld);
    const int32_t t = targets[row];
    const bool has_t = t / chunk == (int64_t)blockIdx.y;
    const float zt = has_t ? z[row * ld + t] : 0.0f;
    float m = -INFINITY, s = 0.0f;
    for (int64_t j = threadIdx.x; j < units; j += 256) {
        const float2 a = part[row * units + j];
        lse_merge(m, s, a.x, a.y);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float m2 = __shfl_xor(m, off, 64), s2 = __shfl_xor(s, off, 64);
        lse_merge(m, s, m2, s2);
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
        red_m[wave] = m;
        red_s[wave] = s;
    }
    __syncthreads();  // (z[target] has been read by every thread, too)
    m = red_m[0];
    s = red_s[0];
    for (int i = 1; i < 4; ++i) lse_merge(m, s, red_m[i], red_s[i]);
    if (has_t && threadIdx.x == 0) row_loss[row] = (m + logf(s)) - zt;
    const float f = __fdiv_rn(scale, s);
    auto grad = [&](float x, int64_t j) {
        const float d = exp_neg(x - m) * f;
        return j == t ? d - scale : d;
    };
    const int64_t q1 = min((v + 3) / 4, q0 + chunk / 4);
    for (int64_t q = q0 + threadIdx.x; q < q1; q += 256) {
        float4 a = z4[q];  // (columns past v are padding of the row)
        a.x = grad(a.x, 4 * q);
        a.y = grad(a.y, 4 * q + 1);
        a.z = grad(a.z, 4 * q + 2);
        a.w = grad(a.w, 4 * q + 3);
        z4[q] = a;
    }
}

// Columns of a workgroup of loss_grad_kernel: whole rows where there are eight
// workgroups per CU of them, else parts of 8192 columns at least (a grid has at
// most 65535 in y).
int64_t grad_chunk(const Context &cx, int64_t rows, int64_t v) {
    const int64_t parts = std::max<int64_t>(1, std::min((8 * (int64_t)cx.cu_count + rows - 1) / rows, (v + 8191) / 8192));
    return std::max((v + parts - 1) / parts, v / 65535 + 1) / 4 * 4 + 4;
}

int64_t part_units(int64_t v) { return (v + kPartCols - 1) / kPartCols; }

void launch_loss_parts(Context &cx, const float *z, const int32_t *targets, int64_t rows, int64_t ld,
                       int64_t v, float *part, float *zt) {
    const int64_t units = part_units(v);
    hipLaunchKernelGGL(loss_parts_kernel, dim3((unsigned)units, (unsigned)rows), dim3(256), 0, cx.stream, z,
                       targets, ld, v, units, reinterpret_cast<float2 *>(part), zt);
    check_hip(hipGetLastError(), "loss partials launch");
}

__global__ __launch_bounds__(256) void copy_ids_kernel(const int32_t *host, int64_t n, int32_t *dev) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        dev[i] = host[i];
}

// Floats of a row of stored logits: whole float4s, for the products too.
int64_t logit_row(int64_t vocab) { return (vocab + 31) / 32 * 32; }

// The rows that count.
struct Rows {
    int64_t kept = 0;
    const float *x = nullptr;          // [kept, d]
    const int32_t *targets = nullptr;  // [kept], where kernels read them
    const int32_t *map = nullptr;      // device, [n]: a row's place among the kept ones, or -1; null: all are kept
    float *loss = nullptr;             // pinned, [kept]: the rows' terms
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

// The targets into pinned memory, which the kernels that read a row's target
// once take them from; into device memory for the product that reads them in
// every tile (`device`), and with ignored rows, where the kept rows' indexes and
// the map back go along and those rows of x are packed.
void stage_rows(Context &cx, const Head &h, bool device, float *packed, Rows &r) {
    const int64_t pad = (h.n + 63) / 64 * 64, total = r.kept == h.n ? h.n : 3 * pad;
    int32_t *t = static_cast<int32_t *>(cx.pinned_rows(((size_t)total + (size_t)r.kept) * 4));
    r.loss = reinterpret_cast<float *>(t + total);
    r.x = h.x;
    if (r.kept == h.n) {
        std::copy(h.targets, h.targets + h.n, t);
        r.targets = t;
        if (!device) return;
    } else {
        int32_t *index = t + pad, *map = index + pad, at = 0;
        std::fill(t, t + total, 0);
        for (int64_t i = 0; i < h.n; ++i) {
            const bool keep = h.targets[i] != h.ignore;
            map[i] = keep ? at : -1;
            if (!keep) continue;
            t[at] = h.targets[i];
            index[at++] = (int32_t)i;
        }
    }
    int32_t *dev = static_cast<int32_t *>(cx.workspace(1, (size_t)total * 4));
    r.targets = dev;
    hipLaunchKernelGGL(copy_ids_kernel, dim3((unsigned)std::min<int64_t>((total + 255) / 256, 65536)),
                       dim3(256), 0, cx.stream, t, total, dev);
    check_hip(hipGetLastError(), "targets launch");
    if (r.kept == h.n) return;
    r.map = dev + 2 * pad;
    for (int64_t at = 0; at < r.kept; at += kMaxRows)
        launch_embedding(cx, h.x, h.d, dev + pad + at, std::min(kMaxRows, r.kept - at), packed + at * h.d);
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
    g.split_bytes = kTrainSplitBytes;
    return g;
}

size_t round64(int64_t floats) { return ((size_t)floats + 63) / 64 * 64; }

void forward(Context &cx, const Head &h, float *loss_host) {
    Rows r;
    r.kept = kept_rows(h);
    if (r.kept == 0) {
        *loss_host = 0.0f;
        return;
    }
    const int64_t units = (h.vocab + 127) / 128;
    // (more columns than kRowCols always fill the tiles that fold the loss)
    auto folds = [&](int64_t rows) {
        return rows > kFewRows && (h.vocab > kRowCols || gemm_ce_tiles(cx, head_product(h, h.x, rows)) > 0);
    };
    const int64_t ld = logit_row(h.vocab);
    const int64_t block = block_rows(r.kept, folds(r.kept) ? units * 8 : ld * 4, cx.loss_block_bytes);
    // a block's partials, or the logits of one too small for the product to fold them (the last, often)
    auto floats = [&](int64_t rows) { return rows * (folds(rows) ? units * 2 : ld); };
    const int64_t weights = h.d * h.vocab, last = (r.kept - 1) % block + 1;
    int64_t most = 0;
    for (int64_t rows : {block, last})
        for (int64_t at = 0, n; at < rows; at += n) most = std::max(most, floats(n = part_rows(rows, at, weights)));
    const size_t packed = r.kept < h.n ? round64(r.kept * h.d) : 0;
    const size_t part = round64(most);
    const size_t parts_floats = round64(2 * kFewRows * part_units(h.vocab));
    float *ws = static_cast<float *>(cx.workspace(2, (packed + part + round64(block) + parts_floats) * 4));
    Drain drain{cx};
    stage_rows(cx, h, folds(block), ws, r);
    float *row_loss = r.loss;
    float *buf = ws + packed, *zt = buf + part, *stats = zt + round64(block);
    for (int64_t at = 0, rows; at < r.kept; at += rows) {
        rows = part_rows(std::min(block, r.kept - at / block * block), at % block, weights);
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
            if (h.vocab <= kRowCols) {
                launch_loss_rows<false>(cx, buf, r.targets + at, rows, ld, h.vocab, 0.0f, row_loss + at);
            } else {
                const int64_t parts = part_units(h.vocab);
                launch_loss_parts(cx, buf, r.targets + at, rows, ld, h.vocab, stats, zt);
                launch_ce_combine_rows(cx, stats, parts, zt, rows, row_loss + at);
            }
        }
    }
    *loss_host = mean_loss(drain, r.loss, r.kept, r.kept);
}

void backward(Context &cx, const Head &h, float *dx, float *dw, float *loss_host) {
    Rows r;
    r.kept = kept_rows(h);
    if (r.kept == 0) {
        if (loss_host) *loss_host = 0.0f;
        if (dx) launch_fill(cx, dx, h.n * h.d, 0.0f);
        if (dw) launch_fill(cx, dw, h.d * h.vocab, 0.0f);
        check_hip(hipStreamSynchronize(cx.stream), "loss sync");  // (like every other way out)
        return;
    }
    const bool all = r.kept == h.n, nt = h.form == MMH_GEMM_NT;
    const int64_t units = (h.vocab + 127) / 128;
    const int64_t ld = logit_row(h.vocab), block = block_rows(r.kept, ld * 4, cx.loss_block_bytes);
    const size_t packed = all ? 0 : round64(r.kept * h.d);
    float *ws = static_cast<float *>(
        cx.workspace(2, (packed * (dx ? 2 : 1) + round64(block * ld) + round64(block * units * 2) + kFewRows) * 4));
    Drain drain{cx};
    stage_rows(cx, h, false, ws, r);
    float *row_loss = r.loss;
    float *z = ws + packed, *part = z + round64(block * ld);
    float *zt = part + round64(block * units * 2), *dxk = all ? dx : zt + kFewRows;
    const float scale = 1.0f / (float)r.kept;
    // dz of the rows at .. at + rows in zp
    auto logits = [&](float *zp, int64_t at, int64_t rows) {
        GemmDesc g = head_product(h, r.x + at * h.d, rows);
        g.c = zp;
        g.ldc = ld;
        if (h.vocab > kRowCols) {
            int64_t stats = units;
            if (rows > kFewRows) {
                g.epi = EPI_CE_STORE;
                g.ce_part = part;
                gemm(cx, g);
            } else {
                stats = part_units(h.vocab);
                gemm(cx, g);
                launch_loss_parts(cx, zp, r.targets + at, rows, ld, h.vocab, part, zt);
            }
            const int64_t chunk = grad_chunk(cx, rows, h.vocab);
            const dim3 grid((unsigned)rows, (unsigned)((h.vocab + chunk - 1) / chunk));
            hipLaunchKernelGGL(loss_grad_kernel, grid, dim3(256), 0, cx.stream, zp,
                               reinterpret_cast<const float2 *>(part), r.targets + at, ld, h.vocab, stats,
                               chunk, scale, row_loss + at);
            check_hip(hipGetLastError(), "loss gradient launch");
        } else {
            gemm(cx, g);
            launch_loss_rows<true>(cx, zp, r.targets + at, rows, ld, h.vocab, scale, row_loss + at);
        }
    };
    // dx of the rows at .. at + rows: dz [rows, vocab] . op(W)^T
    auto dx_product = [&](const float *zp, int64_t at, int64_t rows) {
        GemmDesc p;
        p.a = zp;
        p.b = h.w;
        p.c = dxk + at * h.d;
        p.m = rows;
        p.k = h.vocab;
        p.n = h.d;
        p.lda = ld;
        p.tb = !nt;
        p.ldb = nt ? h.d : h.vocab;
        p.ldc = h.d;
        p.split_bytes = kTrainSplitBytes;
        return p;
    };
    // a block's share of dW: x^T dz [d, vocab], or dz^T x [vocab, d]; later blocks are added
    auto dw_product = [&](int64_t at, int64_t rows) {
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
        p.split_bytes = kTrainSplitBytes;
        p.epi = at ? EPI_ACCUM : EPI_STORE;
        return p;
    };
    const int64_t weights = h.d * h.vocab;
    for (int64_t at = 0; at < r.kept; at += block) {
        const int64_t rows = std::min(block, r.kept - at), most = part_rows(rows, 0, weights);
        logits(z, at, most);
        if (most < rows) logits(z + most * ld, at + most, rows - most);
        if (dx && dw && at == 0) {
            gemm_pair(cx, dx_product(z, at, most), dw_product(at, rows));
        } else {
            if (dx) gemm(cx, dx_product(z, at, most));
            if (dw) gemm(cx, dw_product(at, rows));
        }
        if (dx && most < rows) gemm(cx, dx_product(z + most * ld, at + most, rows - most));
    }
    if (!all && dx) {
        hipLaunchKernelGGL(spread_rows_kernel, dim3((unsigned)std::min<int64_t>(h.n, 65536)), dim3(256), 0,
                           cx.stream, dxk, r.map, h.n, h.d, dx);
        check_hip(hipGetLastError(), "gradient rows launch");
    }
    const float loss = mean_loss(drain, r.loss, r.kept, r.kept);  // (waits: the pinned targets have been read)
    if (loss_host) *loss_host = loss;
}

}  // namespace
}  // namespace mmh

using namespace mmh;

extern "C" {

// For the tests, not part of the C ABI: the rows of a block of n rows of row_bytes
// within `bytes`; the bytes that a context's blocks take (0: the ordinary ones).
int32_t mmh_test_loss_block_rows(int64_t n, int64_t row_bytes, int64_t bytes, int64_t *rows) {
    return guard([&] {
        need(rows, "rows");
        positive(n, "n");
        positive(row_bytes, "row_bytes");
        *rows = block_rows(n, row_bytes, bytes > 0 ? bytes : kLogitBytes);
        return MMH_OK;
    });
}
int32_t mmh_test_loss_block_bytes(mmh_handle ctx, int64_t bytes) {
    return guard([&] {
        context(ctx).loss_block_bytes = bytes > 0 ? bytes : kLogitBytes;
        return MMH_OK;
    });
}

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
        if (dx || dw) backward(context(ctx), h, dx, dw, loss_host);
        else if (loss_host) forward(context(ctx), h, loss_host);
        else context(ctx);
        return MMH_OK;
    });
}

}  // extern "C"
