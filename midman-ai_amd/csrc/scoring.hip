// Scoring tokens by a model's logits, and learning from a teacher's.
//
// With m the largest logit of a row, d = z - m and S(T) = sum exp(d / T):
//   logprob of token t   d_t - ln S(1)
//   entropy              ln S(1) - sum exp(d) d / S(1)
//   distillation         alpha T^2 sum_j q_j (ln q_j - (d_j / T - ln S(T)))
//                        + (1 - alpha) (ln S(1) - d_target),
//   q the softmax of the teacher's k logits over T. Their gradients are
//   dl (onehot - p) - dH p (ln p + H) and
//   alpha T (p_T - q) + (1 - alpha) (p - onehot), p and p_T the row's softmax at 1 and T.
//
// S is kept as 1 + rest, without one of the largest logits' terms, and its logarithm
// is log1p(rest): near a certain token the log probability and the entropy are as
// small as the rest, and keep all their bits.
#include <algorithm>

#include "mmh_args.h"
#include "mmh_elementwise.h"
#include "mmh_internal.h"
#include "mmh_loss.h"

namespace mmh {
namespace {

// A launch has less than 2^32 threads, a row up to 512.
constexpr int64_t kMaxRows = int64_t(1) << 22;
// Alternatives of a row, and slots of a teacher's, at most.
constexpr int64_t kMaxTop = 256;

// A row's sums in progress: m the largest logit (-inf: none yet), a the sum of
// exp((z - m) rate) without one term of m itself, u the sum of exp(z - m) (z - m)
// (SUMS_ENTROPY) or a at rate 1 (SUMS_BOTH).
enum Sums : int { SUMS_ONE = 0, SUMS_ENTROPY = 1, SUMS_BOTH = 2 };
struct RowSums {
    float m, a, u;
};

// exp(d rate), d <= 0.
__device__ __forceinline__ float exp_at(float d, float rate) { return exp_neg(d * rate); }

// (A NaN counts as +inf, which leaves a row without a distribution: see finish.)
__device__ __forceinline__ float logit(float z) { return z != z ? INFINITY : z; }

template <int SUMS>
__device__ __forceinline__ void merge(RowSums &x, const RowSums &y, float rate) {
    if (y.m == -INFINITY) return;
    if (x.m == -INFINITY) {
        x = y;
        return;
    }
    RowSums big = x, small = y;
    if (y.m > x.m) {
        big = y;
        small = x;
    }
    const float d = fmaxf(small.m - big.m, -1e30f), w = exp_at(d, rate);
    x.m = big.m;
    x.a = big.a + (1.0f + small.a) * w;
    if (SUMS == SUMS_ENTROPY) x.u = big.u + (small.u + d * (1.0f + small.a)) * w;
    if (SUMS == SUMS_BOTH) x.u = big.u + (1.0f + small.u) * exp_at(d, 1.0f);
}

// A row whose largest logit is not finite (nothing but -inf, an infinity or a NaN) has
// no distribution: its sums are NaN, and so is what is formed from them.
__device__ __forceinline__ void finish(RowSums &x) {
    if (!(fabsf(x.m) < INFINITY)) x.a = x.u = __builtin_nanf("");
}

template <int NT, int SUMS>
__device__ __forceinline__ RowSums block_sums(RowSums x, float rate, RowSums *lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const RowSums y{__shfl_xor(x.m, off, 64), __shfl_xor(x.a, off, 64), __shfl_xor(x.u, off, 64)};
        // (both lanes take the sums in one order: their results are the same)
        const bool low = (threadIdx.x & off) == 0;
        RowSums l = low ? x : y;
        merge<SUMS>(l, low ? y : x, rate);
        x = l;
    }
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
    for (int i = 1; i < NT / 64; ++i) merge<SUMS>(x, lds[i], rate);
    finish(x);
    return x;
}

template <int NT, int SUMS>
__device__ __forceinline__ RowSums row_sums(const float *z, int64_t v, float rate, RowSums *lds) {
    RowSums x{-INFINITY, 0.0f, 0.0f};
    for (int64_t j = threadIdx.x; j < v; j += NT) {
        const RowSums y{logit(z[j]), 0.0f, 0.0f};
        merge<SUMS>(x, y, rate);
    }
    return block_sums<NT, SUMS>(x, rate, lds);
}

// Values in the order of their logits, lower ids first among equals: a number that
// is larger for what comes first.
__device__ __forceinline__ uint32_t order_of(float z) {
    const uint32_t b = __float_as_uint(z + 0.0f);  // (-0 as 0)
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct ScoreArgs {
    const float *logits;
    const int32_t *targets;  // device, or null
    int64_t vocab;
    int32_t ignore;
    int k;
    float *logprobs, *entropy;
    int32_t *top_ids;
    float *top_logprobs;
};

__global__ __launch_bounds__(256) void scores_kernel(ScoreArgs p) {
    __shared__ RowSums lds[4];
    __shared__ unsigned long long best;
    const int64_t row = blockIdx.x;
    const float *z = p.logits + row * p.vocab;
    const int tid = threadIdx.x;
    const int32_t t = p.targets ? p.targets[row] : 0;
    if (p.targets && t == p.ignore) {
        if (tid == 0 && p.logprobs) p.logprobs[row] = 0.0f;
        if (tid == 0 && p.entropy) p.entropy[row] = 0.0f;
        for (int j = tid; j < p.k; j += 256) {
            p.top_ids[row * p.k + j] = -1;
            p.top_logprobs[row * p.k + j] = -INFINITY;
        }
        return;
    }
    const RowSums s = row_sums<256, SUMS_ENTROPY>(z, p.vocab, 1.0f, lds);
    const float rest = log1pf(s.a);
    if (tid == 0 && p.logprobs) p.logprobs[row] = (logit(z[t]) - s.m) - rest;
    if (tid == 0 && p.entropy) p.entropy[row] = rest - s.u / (1.0f + s.a);
    unsigned long long last = ~0ull;
    for (int j = 0; j < p.k; ++j) {
        if (tid == 0) best = 0;
        __syncthreads();
        unsigned long long mine = 0;
        for (int64_t i = tid; i < p.vocab; i += 256) {
            const unsigned long long key = (unsigned long long)order_of(logit(z[i])) << 32 | (uint32_t)~(uint32_t)i;
            if (key < last && key > mine) mine = key;
        }
        atomicMax(&best, mine);
        __syncthreads();
        last = best;
        const int32_t id = (int32_t) ~(uint32_t)last;
        if (tid == 0) {
            p.top_ids[row * p.k + j] = id;
            p.top_logprobs[row * p.k + j] = (logit(z[id]) - s.m) - rest;
        }
        __syncthreads();
    }
}

// dlogits of the log probabilities and entropies. dlogits may be the logits.
__global__ __launch_bounds__(256) void scores_grad_kernel(const float *logits, const int32_t *targets, int64_t v,
                                                          int32_t ignore, const float *dlogprobs,
                                                          const float *dentropy, float *dlogits) {
    __shared__ RowSums lds[4];
    const int64_t row = blockIdx.x;
    const float *z = logits + row * v;
    float *out = dlogits + row * v;
    const int64_t t = targets ? targets[row] : -1;
    if (targets && t == ignore) {
        for (int64_t j = threadIdx.x; j < v; j += 256) out[j] = 0.0f;
        return;
    }
    const RowSums s = row_sums<256, SUMS_ENTROPY>(z, v, 1.0f, lds);
    const float total = 1.0f + s.a, rest = log1pf(s.a), h = rest - s.u / total;
    const float dl = dlogprobs ? dlogprobs[row] : 0.0f, dh = dentropy ? dentropy[row] : 0.0f;
    for (int64_t j = threadIdx.x; j < v; j += 256) {
        const float d = fmaxf(logit(z[j]) - s.m, -1e4f), p = exp_neg(d) / total;
        const float g = p * (-dl - dh * ((d - rest) + h));
        out[j] = j == t ? dl + g : g;
    }
}

struct DistillArgs {
    const float *logits;
    const int32_t *targets;  // or null
    int64_t vocab;
    int32_t ignore;
    const int32_t *ids;
    const float *teacher;
    int k;
    float temperature, alpha, scale;  // scale: 1 / the rows that count
    float *row_loss;                  // [rows], 0 for a row that is left out
    int32_t *wrong;                   // receives an id beyond the vocabulary
    float *dlogits;
};

// The row's loss and (dlogits) its gradient. dlogits may be the logits.
__global__ __launch_bounds__(256) void distill_kernel(DistillArgs p) {
    __shared__ RowSums lds[4];
    __shared__ float q[kMaxTop], term[kMaxTop], zid[kMaxTop];
    __shared__ int32_t id[kMaxTop];
    const int64_t row = blockIdx.x, v = p.vocab;
    const float *z = p.logits + row * v;
    float *out = p.dlogits ? p.dlogits + row * v : nullptr;
    const int tid = threadIdx.x;
    const int64_t t = p.targets ? p.targets[row] : -1;
    if (p.targets && t == p.ignore) {
        if (tid == 0) p.row_loss[row] = 0.0f;
        if (out)
            for (int64_t j = tid; j < v; j += 256) out[j] = 0.0f;
        return;
    }
    const float rate = 1.0f / p.temperature;
    const RowSums s = row_sums<256, SUMS_BOTH>(z, v, rate, lds);
    const float zt = t >= 0 ? logit(z[t]) : 0.0f;
    if (tid < p.k) {
        const int32_t i = p.ids[row * p.k + tid];
        const bool ok = i >= 0 && i < v;
        if (i >= v) *p.wrong = 1;
        id[tid] = ok ? i : -1;
        q[tid] = ok ? logit(p.teacher[row * p.k + tid]) : -INFINITY;
        zid[tid] = ok ? logit(z[i]) : 0.0f;
    }
    __syncthreads();
    float top = -INFINITY;
    for (int j = 0; j < p.k; ++j) top = fmaxf(top, q[j]);
    float sum = 0.0f;
    if (top > -INFINITY)
        for (int j = 0; j < p.k; ++j) sum += exp_neg((q[j] - top) * rate);
    __syncthreads();
    if (tid < p.k) {
        const float u = (q[tid] - top) * rate, share = top > -INFINITY ? exp_neg(u) / sum : 0.0f;
        q[tid] = share;
        term[tid] = share == 0.0f ? 0.0f : share * ((u - logf(sum)) - ((zid[tid] - s.m) * rate - log1pf(s.a)));
    }
    __syncthreads();
    if (tid == 0) {
        float kl = 0.0f;
        for (int j = 0; j < p.k; ++j) kl += term[j];
        float loss = 0.0f;
        if (p.alpha > 0.0f) loss = p.alpha * p.temperature * p.temperature * kl;
        if (p.alpha < 1.0f) loss += (1.0f - p.alpha) * (log1pf(s.u) - (zt - s.m));
        p.row_loss[row] = loss;
    }
    if (!out) return;
    const float soft = p.alpha * p.temperature * p.scale, hard = (1.0f - p.alpha) * p.scale;
    for (int64_t j = tid; j < v; j += 256) {
        const float d = fmaxf(logit(z[j]) - s.m, -1e30f);
        float g = exp_neg(d * rate) / (1.0f + s.a) * soft + exp_neg(d) / (1.0f + s.u) * hard;
        for (int i = 0; i < p.k; ++i)
            if (id[i] == j) g -= soft * q[i];
        if (j == t) g -= hard;
        out[j] = g;
    }
}

void check_logits(const char *what, const float *logits, const int32_t *targets, int64_t n, int64_t vocab,
                  int32_t ignore) {
    need(logits, "logits");
    bounded(n, "rows");
    bounded(vocab, "vocab");
    extent(n, vocab, "logits");
    if (!targets) return;
    for (int64_t i = 0; i < n; ++i)
        if (targets[i] != ignore && (targets[i] < 0 || targets[i] >= vocab))
            fail(MMH_ERR_INDEX, std::string(what) + ": target " + std::to_string(targets[i]) +
                                    " is out of range for " + std::to_string(vocab));
}

struct Distill {
    const float *logits;
    const int32_t *targets;
    int64_t n, vocab;
    int32_t ignore;
    const int32_t *ids;
    const float *teacher;
    int64_t k;
    float temperature, alpha;
};

void check_distill(const Distill &d) {
    check_logits("distillation", d.logits, d.targets, d.n, d.vocab, d.ignore);
    need(d.ids, "teacher_ids");
    need(d.teacher, "teacher_logits");
    if (d.k < 1 || d.k > kMaxTop)
        fail(MMH_ERR_SHAPE, "distillation: k must be 1 to " + std::to_string(kMaxTop) + ", got " + std::to_string(d.k));
    if (!(d.temperature >= 0.001f && d.temperature <= 1000.0f))
        fail(MMH_ERR_ARGUMENT, "distillation: temperature must be in [0.001, 1000], got " + std::to_string(d.temperature));
    if (!(d.alpha >= 0.0f && d.alpha <= 1.0f))
        fail(MMH_ERR_ARGUMENT, "distillation: alpha must be in [0, 1], got " + std::to_string(d.alpha));
    if (d.alpha < 1.0f) need(d.targets, "targets (of alpha below 1)");
}

void distill(Context &cx, const Distill &d, float *dlogits, float *loss_host) {
    const int64_t kept = d.targets ? d.n - std::count(d.targets, d.targets + d.n, d.ignore) : d.n;
    int32_t *pinned = static_cast<int32_t *>(cx.pinned_rows((size_t)(2 * d.n + 16) * 4));
    Drain drain{cx};
    DistillArgs p;
    p.vocab = d.vocab;
    p.ignore = d.ignore;
    p.k = (int)d.k;
    p.temperature = d.temperature;
    p.alpha = d.alpha;
    p.scale = 1.0f / (float)std::max<int64_t>(1, kept);
    p.wrong = pinned;
    *pinned = 0;
    float *rows = reinterpret_cast<float *>(pinned + 16);
    int32_t *targets = pinned + 16 + d.n;
    if (d.targets) std::copy(d.targets, d.targets + d.n, targets);
    for (int64_t at = 0; at < d.n; at += kMaxRows) {
        const int64_t n = std::min(kMaxRows, d.n - at);
        p.logits = d.logits + at * d.vocab;
        p.targets = d.targets ? targets + at : nullptr;
        p.ids = d.ids + at * d.k;
        p.teacher = d.teacher + at * d.k;
        p.row_loss = rows + at;
        p.dlogits = dlogits ? dlogits + at * d.vocab : nullptr;
        hipLaunchKernelGGL(distill_kernel, dim3((unsigned)n), dim3(256), 0, cx.stream, p);
        check_hip(hipGetLastError(), "distillation launch");
    }
    const float mean = mean_loss(drain, rows, d.n, std::max<int64_t>(1, kept));
    if (*(volatile int32_t *)p.wrong)
        fail(MMH_ERR_INDEX, "distillation: a teacher's id is out of range for " + std::to_string(d.vocab));
    if (loss_host) *loss_host = mean;
}

}  // namespace
}  // namespace mmh

using namespace mmh;

extern "C" {

int32_t mmh_token_logprobs(mmh_handle ctx, const float *logits, const int32_t *targets_host, int64_t n,
                           int64_t vocab, int32_t ignore, int64_t k, float *logprobs, float *entropy,
                           int32_t *top_ids, float *top_logprobs) {
    return guard([&] {
        check_logits("token_logprobs", logits, targets_host, n, vocab, ignore);
        if (k < 0 || k > std::min(vocab, kMaxTop))
            fail(MMH_ERR_SHAPE, "token_logprobs: k must be 0 to " + std::to_string(std::min(vocab, kMaxTop)) +
                                    ", got " + std::to_string(k));
        if (logprobs) need(targets_host, "targets (of log probabilities)");
        if (k > 0) {
            need(top_ids, "top_ids");
            need(top_logprobs, "top_logprobs");
        } else {
            top_ids = nullptr;
            top_logprobs = nullptr;
        }
        const Span sz{logits, n * vocab, "logits"}, sl{logprobs, n, "logprobs"}, se{entropy, n, "entropy"},
            si{top_ids, n * k, "top_ids"}, st{top_logprobs, n * k, "top_logprobs"};
        apart(sl, {sz, se, si, st});
        apart(se, {sz, si, st});
        apart(si, {sz, st});
        apart(st, {sz});
        Context &cx = context(ctx);
        if (!logprobs && !entropy && k == 0) return MMH_OK;
        const int32_t *targets = targets_host ? cx.stage_ids(targets_host, n, 1) : nullptr;
        for (int64_t at = 0; at < n; at += kMaxRows) {
            const int64_t rows = std::min(kMaxRows, n - at);
            ScoreArgs p;
            p.logits = logits + at * vocab;
            p.targets = targets ? targets + at : nullptr;
            p.vocab = vocab;
            p.ignore = ignore;
            p.k = (int)k;
            p.logprobs = logprobs ? logprobs + at : nullptr;
            p.entropy = entropy ? entropy + at : nullptr;
            p.top_ids = top_ids + at * k;
            p.top_logprobs = top_logprobs + at * k;
            hipLaunchKernelGGL(scores_kernel, dim3((unsigned)rows), dim3(256), 0, cx.stream, p);
            check_hip(hipGetLastError(), "token_logprobs launch");
        }
        return MMH_OK;
    });
}

int32_t mmh_token_logprobs_backward(mmh_handle ctx, const float *logits, const int32_t *targets_host, int64_t n,
                                    int64_t vocab, int32_t ignore, const float *dlogprobs, const float *dentropy,
                                    float *dlogits) {
    return guard([&] {
        check_logits("token_logprobs", logits, targets_host, n, vocab, ignore);
        need(dlogits, "dlogits");
        if (dlogprobs) need(targets_host, "targets (of log probabilities)");
        const Span sz{logits, n * vocab, "logits"}, sl{dlogprobs, n, "dlogprobs"}, se{dentropy, n, "dentropy"},
            sd{dlogits, n * vocab, "dlogits"};
        apart_or_same(sd, {sz});
        apart(sd, {sl, se});
        Context &cx = context(ctx);
        const int32_t *targets = targets_host ? cx.stage_ids(targets_host, n, 1) : nullptr;
        for (int64_t at = 0; at < n; at += kMaxRows) {
            const int64_t rows = std::min(kMaxRows, n - at);
            hipLaunchKernelGGL(scores_grad_kernel, dim3((unsigned)rows), dim3(256), 0, cx.stream, logits + at * vocab,
                               targets ? targets + at : nullptr, vocab, ignore, dlogprobs ? dlogprobs + at : nullptr,
                               dentropy ? dentropy + at : nullptr, dlogits + at * vocab);
            check_hip(hipGetLastError(), "token_logprobs gradient launch");
        }
        return MMH_OK;
    });
}

int32_t mmh_distillation(mmh_handle ctx, const float *logits, const int32_t *targets_host, int64_t n, int64_t vocab,
                         int32_t ignore, const int32_t *teacher_ids, const float *teacher_logits, int64_t k,
                         float temperature, float alpha, float *loss_host) {
    return guard([&] {
        const Distill d{logits, targets_host, n, vocab, ignore, teacher_ids, teacher_logits, k, temperature, alpha};
        check_distill(d);
        need(loss_host, "loss");
        distill(context(ctx), d, nullptr, loss_host);
        return MMH_OK;
    });
}

int32_t mmh_distillation_backward(mmh_handle ctx, const float *logits, const int32_t *targets_host, int64_t n,
                                  int64_t vocab, int32_t ignore, const int32_t *teacher_ids,
                                  const float *teacher_logits, int64_t k, float temperature, float alpha,
                                  float *dlogits, float *loss_host) {
    return guard([&] {
        const Distill d{logits, targets_host, n, vocab, ignore, teacher_ids, teacher_logits, k, temperature, alpha};
        check_distill(d);
        need(dlogits, "dlogits");
        const Span sd{dlogits, n * vocab, "dlogits"};
        apart_or_same(sd, {{logits, n * vocab, "logits"}});
        apart(sd, {{teacher_ids, n * k, "teacher_ids"}, {teacher_logits, n * k, "teacher_logits"}});
        distill(context(ctx), d, dlogits, loss_host);
        return MMH_OK;
    });
}

}  // extern "C"
