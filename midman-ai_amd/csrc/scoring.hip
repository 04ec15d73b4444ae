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
// is log1p(rest): near a certain token the log probability, the entropy and the target's
// gradient are as small as the rest, and keep all their bits. (A teacher's share q does
// not: p_T - q is off by a rounding of q.)
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "mmh_args.h"
#include "mmh_elementwise.h"
#include "mmh_ids.h"
#include "mmh_internal.h"
#include "mmh_loss.h"

namespace mmh {
namespace {

// A launch has less than 2^32 threads, a row's workgroup up to 1024.
constexpr int64_t kMaxRows = int64_t(1) << 21;
// Alternatives of a row, and slots of a teacher's, at most.
constexpr int64_t kMaxTop = 256;

// (exp(-200) is 0 in f32: a masked token's difference has this in its place, so that
// its product with that 0 is one)
constexpr float kFar = -200.0f;

// A factor in two floats, both above 0.
struct Rate {
    float hi, lo;
};
inline Rate rate_of(double k) {
    float hi = (float)k;
    if ((double)hi > k) hi = std::nextafterf(hi, 0.0f);
    return Rate{hi, std::max((float)(k - (double)hi), hi * 0x1p-60f)};
}
// The product, rounded once. (An infinite d has its own sign in both.)
__device__ __forceinline__ float times(float d, const Rate &k) { return __builtin_fmaf(d, k.hi, d * k.lo); }
// log2 e / T, for exponentials of differences at temperature T = 1.
constexpr double kLog2e = 1.4426950408889634074;
constexpr Rate kPlain{1.44269502f, 1.92596303e-8f};  // rate_of(kLog2e)
// exp(d / T), d <= 0, off by up to (2 + |d| / T) 2^-24 of itself, to both sides alike: the
// exponent rounds once. (With one float for log2 e every term is too large by 0.22 |d|
// 2^-24, and ln S of 32000 logits by 7e-8; both cost the same within 1%. Carrying the
// exponent's rounding along as well would leave 2^-23 alone, beside the |d| / T 2^-24 of
// d's own rounding, and take longer: 4096 x 32000 with both terms 228 -> 257 us, log
// probabilities 109 -> 114.)
__device__ __forceinline__ float exp_of(float d, const Rate &k) { return __builtin_amdgcn_exp2f(times(d, k)); }

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// Over a wave, in every lane: within 16 lanes by DPP, then by halves. (Shuffles through
// LDS take several times as long, and a short row is little else.)
template <int CTRL>
__device__ __forceinline__ int32_t dpp(int32_t v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
template <class F>
__device__ __forceinline__ int32_t wave_fold(int32_t v, F &&f) {
    v = f(v, dpp<0xb1>(v));   // lane ^ 1
    v = f(v, dpp<0x4e>(v));   // lane ^ 2
    v = f(v, dpp<0x141>(v));  // mirrored within 8 lanes
    v = f(v, dpp<0x140>(v));  // and within 16
    auto c = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = f((int32_t)c[0], (int32_t)c[1]);
    c = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    return f((int32_t)c[0], (int32_t)c[1]);
}
__device__ __forceinline__ float wave_max(float v) {
    return __int_as_float(wave_fold(__float_as_int(v), [](int32_t a, int32_t b) {
        return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
    }));
}
__device__ __forceinline__ float wave_sum(float v) {
    return __int_as_float(wave_fold(__float_as_int(v), [](int32_t a, int32_t b) {
        return __float_as_int(__int_as_float(a) + __int_as_float(b));
    }));
}
__device__ __forceinline__ int wave_sum(int v) {
    return wave_fold(v, [](int32_t a, int32_t b) { return a + b; });
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    return (uint32_t)wave_fold((int32_t)v, [](int32_t a, int32_t b) { return (int32_t)max((uint32_t)a, (uint32_t)b); });
}

// ---- a stretch of a row in registers ------------------------------------------
// Rows begin at any 4-byte address. They are taken as if they began `shift` floats
// earlier, at a cache line, so that a wave's strips are whole lines (768 rows of 131071 as
// they lie 196 us, so 175, as rows of 131072); columns below are of that longer row.
constexpr int kLine = 32;
__device__ __forceinline__ int line_shift(const float *row) { return (int)(reinterpret_cast<uintptr_t>(row) >> 2 & (kLine - 1)); }

// NT threads hold NV strips of 4 NT columns of a stretch, thread t of strip i the columns
// 4 (t + NT i) and three on; of the stretch the columns lo .. cols - 1 are the row's (lo
// below kLine), the others -inf. Loads of whole float4s are unconditional (those that end
// outside start from within), so all of them are in flight at once.
template <int NT, int NV>
__device__ __forceinline__ void load_stretch(const float *z, int lo, int cols, float (&e)[NV][4], int tid = threadIdx.x) {
    static_assert(4 * NT >= kLine, "lo lies in the first strip");
    if (cols - lo >= 4) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = min(4 * (tid + NT * i), cols - 4);
            __builtin_memcpy(e[i], z + (i == 0 ? max(c, lo) : c), 16);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if ((i > 0 || lo == 0) && 4 * NT * (i + 1) <= cols) continue;
        const int c = 4 * (tid + NT * i);
        if (c >= lo && c + 4 <= cols) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) e[i][j] = c + j >= lo && c + j < cols ? z[c + j] : -INFINITY;
    }
}
// f of a stretch to `out`, each strip on its way as soon as it is formed. `stream`: past
// the caches, for outputs that they would not hold until they are read. (A branch for
// both ways at each store would hold them back until all is formed: 4096 x 32000 227 ->
// 237 us.)
template <bool STREAM, int NT, int NV, class F>
__device__ __forceinline__ void write_strips(float *out, int lo, int cols, const float (&e)[NV][4], int tid, F &&f) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = 4 * (tid + NT * i);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = f(e[i][j]);
        if ((i > 0 || c >= lo) && c + 4 <= cols) {
            float4u x;
            __builtin_memcpy(&x, v, 16);
            if (STREAM) __builtin_nontemporal_store(x, reinterpret_cast<float4u *>(out + c));
            else *reinterpret_cast<float4u *>(out + c) = x;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j >= lo && c + j < cols) out[c + j] = v[j];
        }
    }
}
template <int NT, int NV, class F>
__device__ __forceinline__ void write_stretch(float *out, int lo, int cols, bool stream, const float (&e)[NV][4], int tid, F &&f) {
    if (stream) write_strips<true, NT, NV>(out, lo, cols, e, tid, f);
    else write_strips<false, NT, NV>(out, lo, cols, e, tid, f);
}

// ---- a row's sums ---------------------------------------------------------------
// Of exp((z - m) rate), m the largest logit: `count` of the terms are 1 (z = m), a is
// the sum of the others, and u the sum of exp(z - m) (z - m) (KIND_SCORES) or of the
// others' terms at rate 1 (KIND_BOTH). A wave's lanes have one m.
enum Kind : int { KIND_SCORES = 0, KIND_ONE = 1, KIND_BOTH = 2 };
struct RowSums {
    float m, count, a, u;
};
__device__ __forceinline__ RowSums no_sums() { return RowSums{-INFINITY, 0.0f, 0.0f, 0.0f}; }

// Adds a stretch to a wave's running sums (per lane but for m). A NaN stays in a. The
// wave's largest logit lies in one group of strips as a rule: only there are its terms
// told from the others, by a branch that the whole wave takes.
template <int KIND, int NV>
__device__ __forceinline__ void add_stretch(RowSums &s, const float (&e)[NV][4], const Rate &k) {
    constexpr int G = NV < 16 ? (NV + 3) / 4 : 4;
    float top = -INFINITY, group[NV / G];
#pragma unroll
    for (int g = 0; g < NV / G; ++g) {
        group[g] = -INFINITY;
#pragma unroll
        for (int i = g * G; i < (g + 1) * G; ++i)
            group[g] = fmaxf(group[g], fmaxf(fmaxf(e[i][0], e[i][1]), fmaxf(e[i][2], e[i][3])));
        top = fmaxf(top, group[g]);
    }
    top = wave_max(top);
    if (top > s.m) {
        // what is there is scaled to the new largest logit; its ones are ordinary terms
        if (s.m > -INFINITY) {
            const float d = s.m - top, w = exp_of(d, k);
            if (KIND == KIND_SCORES) s.u = (s.u + fmaxf(d, kFar) * (s.a + s.count)) * w;
            if (KIND == KIND_BOTH) s.u = (s.u + s.count) * exp_of(d, kPlain);
            s.a = (s.a + s.count) * w;
        }
        s.m = top;
        s.count = 0.0f;
    }
    const float m = s.m == -INFINITY ? 0.0f : s.m;  // (nothing but -inf: terms of 0)
    auto add = [&](float z, bool look) __attribute__((always_inline)) {
        const float d = z - m;
        float x = exp_of(d, k), x1 = KIND == KIND_BOTH ? exp_of(d, kPlain) : 0.0f;
        if (look) {
            // (selected by arithmetic: a selection would become a branch around the exponentials)
            const float one = d == 0.0f ? 1.0f : 0.0f;
            s.count += one;
            x -= one;
            x1 -= one;
        }
        s.a += x;
        if (KIND == KIND_SCORES) s.u = __builtin_fmaf(x, fmaxf(d, kFar), s.u);
        if (KIND == KIND_BOTH) s.u += x1;
    };
#pragma unroll
    for (int g = 0; g < NV / G; ++g) {
        if (__any(group[g] == m)) {
            asm volatile("");  // (stays a branch of its own)
#pragma unroll
            for (int c = 0; c < 4 * G; ++c) add(e[g * G + c / 4][c % 4], true);
        } else {
#pragma unroll
            for (int c = 0; c < 4 * G; ++c) add(e[g * G + c / 4][c % 4], false);
        }
    }
}
// The wave's sums in every lane; a NaN among its logits makes m one.
__device__ __forceinline__ RowSums wave_sums(RowSums s) {
    s.count = wave_sum(s.count);
    s.a = wave_sum(s.a);
    s.u = wave_sum(s.u);
    if (s.a != s.a) s.m = s.a;
    return s;
}
// The sums of n parts of a row together. (A part of nothing but -inf adds nothing; inf -
// inf is NaN.)
template <int KIND>
__device__ __forceinline__ RowSums join_sums(const RowSums *parts, int n, const Rate &k) {
    RowSums s = no_sums();
    for (int i = 0; i < n; ++i) s.m = fmaxf(s.m, parts[i].m);
    for (int i = 0; i < n; ++i) {
        const RowSums p = parts[i];
        if (p.m == -INFINITY) continue;
        const float d = p.m - s.m;
        if (d == 0.0f) {
            s.count += p.count;
            s.a += p.a;
            s.u += p.u;
        } else {
            const float w = exp_of(d, k), all = p.a + p.count;
            s.a += all * w;
            if (KIND == KIND_SCORES) s.u += (p.u + fmaxf(d, kFar) * all) * w;
            if (KIND == KIND_BOTH) s.u += (p.u + p.count) * exp_of(d, kPlain);
        }
    }
    return s;
}
// (as wave_sums: a NaN shows in m, so that it is not taken for a part of -inf)
__device__ __forceinline__ RowSums with_nan(RowSums s) {
    if (s.a != s.a) s.m = s.a;
    return s;
}
// A whole row's: one whose largest logit is not finite (nothing but -inf, an infinity or
// a NaN) has no distribution, and what is formed from NaN sums is NaN.
__device__ __forceinline__ RowSums row_sums(RowSums s) {
    if (!(fabsf(s.m) < INFINITY)) s.a = s.u = __builtin_nanf("");
    return s;
}
// The sums of a row's n parts, by one wave: in every lane, in one order.
template <int KIND>
__device__ __forceinline__ RowSums wave_join(const RowSums *parts, int n, const Rate &k) {
    const int lane = threadIdx.x & 63;
    RowSums s = no_sums();
    for (int j = lane; j < n; j += 64) {
        const RowSums two[2] = {s, parts[j]};
        s = with_nan(join_sums<KIND>(two, 2, k));
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const RowSums o{__shfl_xor(s.m, off, 64), __shfl_xor(s.count, off, 64), __shfl_xor(s.a, off, 64), __shfl_xor(s.u, off, 64)};
        const RowSums two[2] = {lane & off ? o : s, lane & off ? s : o};
        s = with_nan(join_sums<KIND>(two, 2, k));
    }
    return s;
}
// S - 1: the sum without one of the largest logits' terms.
__device__ __forceinline__ float rest_of(const RowSums &s) { return s.a + (s.count - 1.0f); }

// Values in the order of their logits: a larger number for a larger one, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float z) {
    const uint32_t b = __float_as_uint(z + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
// (for the order of alternatives a NaN counts as +inf)
__device__ __forceinline__ float ranked(float z) { return z != z ? INFINITY : z; }

// ---- log probabilities, entropies and the most likely tokens -------------------------
// The k largest of a stretch, without sorting it: the k-th largest of the threads'
// maxima is no larger than the k-th largest logit, and only what is above it (a little
// more than k logits as a rule) goes to a list in LDS, where each entry's place is the
// number of larger ones.
// One read of the logits bounds it (4096 x 32000 without targets and alternatives 86 us,
// 6.1 TB/s); then the steps between barriers, of which two workgroups on a CU hide a part
// (k 16 93 us, 64 105, 128 123, 256 187; an argmax per alternative, as first built, k 64
// 7390).
struct ScoreArgs {
    const float *logits;
    HostIds targets;
    int64_t vocab;
    int32_t ignore;
    int k;
    float *logprobs, *entropy;
    int32_t *top_ids;
    float *top_logprobs;
    // rows over several workgroups: what a part leaves
    int64_t part;         // columns of a part, a multiple of kLine, some hundreds at least
    int parts;
    RowSums *sums;        // [rows, parts]
    uint64_t *best;       // [rows, parts, k], the largest first
};

constexpr int kList = 1024;  // entries of the list; kMaxTop at least
constexpr int kColBits = 15; // of a column within its stretch
// An entry of a stretch: larger for what comes first, the larger logit or the lower column.
// Below 2^53, so an f64 holds it: those compare at the vector rate, 64-bit integers do not.
__device__ __forceinline__ double entry_of(float z, int col) {
    return (double)order_of(z) * (1 << kColBits) + (double)((1 << kColBits) - 1 - col);
}
// The same of a whole row.
__device__ __forceinline__ uint64_t row_entry(double e, uint32_t first) {
    const uint64_t b = (uint64_t)e;
    const uint32_t col = (1u << kColBits) - 1 - (uint32_t)(b & ((1u << kColBits) - 1));
    return b >> kColBits << 32 | (uint32_t)~(first + col);
}

struct TopShared {
    // as they are found, a logit and its column; in their order, entry_of
    union __attribute__((aligned(16))) {
        float2 found[kList + 16];
        double list[kList + 16];
    };
    uint32_t maxima[512];  // of the threads, as orders
    int32_t rank[kList];    // of the list's entries
    int32_t count[16];
    int32_t n;              // entries of the list
    float above;            // logits above it are in the list
};

// The number, over the workgroup, of logits above t.
template <int NT, int NV>
__device__ __forceinline__ int count_above(const float (&e)[NV][4], float t, TopShared &sh) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) n += e[i][j] > t ? 1 : 0;
    n = wave_sum(n);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.count[threadIdx.x >> 6] = n;
    __syncthreads();
    n = 0;
    for (int i = 0; i < NT / 64; ++i) n += sh.count[i];
    return n;
}

// The k largest of a stretch (no NaN) to place(rank, entry), by every thread of the
// workgroup; fewer where it has fewer columns. Its column 0 is the row's `first`.
template <int NT, int NV, class F>
__device__ __forceinline__ void top_of(const float (&e)[NV][4], int lo_col, int cols, uint32_t first, int k, TopShared &sh, F &&place) {
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t lowest = order_of(-INFINITY);
    k = min(k, max(0, cols - lo_col));
    float mine = -INFINITY;
#pragma unroll
    for (int i = 0; i < NV; ++i) mine = fmaxf(mine, fmaxf(fmaxf(e[i][0], e[i][1]), fmaxf(e[i][2], e[i][3])));
    sh.maxima[tid] = order_of(mine);
    __syncthreads();
    if (tid < 64) {
        // A value that k threads' maxima reach, and a quarter and 8 more at most where they
        // differ. Their number falls by a factor for each step of the value, more or less, so a
        // line through its logarithm finds it in a few tries; halving the range of orders ends it
        // whatever the logits are.
        uint32_t m[NT / 64], lo = ~0u, hi = 0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) {
            m[i] = sh.maxima[lane + 64 * i];
            lo = min(lo, m[i]);
            hi = max(hi, m[i]);
        }
        lo = NT < k ? lowest : ~wave_max(~lo);
        hi = wave_max(hi) + 1;  // (lo is reached by k maxima or is the lowest, hi by none)
        float n_lo = (float)NT, n_hi = 0.5f;
        for (int tries = 0; hi - lo > 1; ++tries) {
            uint32_t mid = lo + (hi - lo) / 2;
            if (tries < 5) {
                const float v = value_of(lo), l = __builtin_amdgcn_logf(n_lo);
                const float share = (l - __builtin_amdgcn_logf((float)(k + k / 8 + 4))) / (l - __builtin_amdgcn_logf(n_hi));
                const float at = v + (value_of(hi - 1) - v) * share;
                if (at > v) mid = max(lo + 1, min(hi - 1, order_of(at)));  // (not of a NaN or infinities)
            }
            int n = 0;
#pragma unroll
            for (int i = 0; i < NT / 64; ++i) n += __popcll(__ballot(m[i] >= mid));
            if (n < k) {
                hi = mid;
                n_hi = fmaxf((float)n, 0.5f);
            } else {
                lo = mid;
                n_lo = (float)n;
            }
            if (n >= k && n <= k + k / 4 + 8) break;
        }
        if (tid == 0) {
            sh.above = value_of(lo);
            sh.n = 0;
        }
    }
    __syncthreads();
    float above = sh.above;
    // Each wave counts what it has, takes its places in the list at once and goes through
    // its registers again; strips in which no lane has any cost three operations.
    auto hits = [&](float over, auto &&f) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!__any(fmaxf(fmaxf(e[i][0], e[i][1]), fmaxf(e[i][2], e[i][3])) > over)) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint64_t hit = __ballot(e[i][j] > over);
                if (hit != 0) f(hit, e[i][j], 4 * (tid + NT * i) + j);
            }
        }
    };
    auto collect = [&] {
        float over = above;
        int count = 0, at = 0;
        hits(over, [&](uint64_t hit, float, int) { count += __popcll(hit); });
        if (count > 0) {
            if (lane == 0) at = atomicAdd(&sh.n, count);
            at = __builtin_amdgcn_readfirstlane(at);
            asm volatile("" : "+v"(over));  // (compared again: the masks kept would not fit the scalar registers)
            hits(over, [&](uint64_t hit, float z, int col) {
                const int to = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(hit >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)hit, 0));
                if (z > over && to < kList) sh.found[to] = make_float2(z, __int_as_float(col));
                at += __popcll(hit);
            });
        }
        __syncthreads();
    };
    collect();
    int n = sh.n;
    if (n > kList) {
        // Many of the largest logits are a few threads': the halving goes on over all of them,
        // until what is above fits, or above and below are neighbours.
        uint32_t lo = order_of(above), hi = 0;
        for (int i = 0; i < NT; ++i) hi = max(hi, sh.maxima[i]);  // (more than kList above lo, none above hi)
        while (n > kList && hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int c = count_above<NT, NV>(e, value_of(mid), sh);
            if (c < k) hi = mid;
            else lo = mid, n = c;
        }
        above = value_of(n > kList ? hi : lo);
        __syncthreads();
        if (tid == 0) sh.n = 0;
        __syncthreads();
        collect();
        n = sh.n;
    }
    if (n < k) {
        // Fewer than k are above it, so it is the k-th largest logit itself: the lowest columns
        // that hold it fill the list, strip by strip.
        int have = n;
        for (int i = 0; i < NV && have < k; ++i) {
            float x[4];
#pragma unroll
            for (int c = 0; c < NV; ++c)
                if (c == i) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = e[c][j];
                }
            const int c0 = 4 * (tid + NT * i);
            int before = have, here = 0;
            uint64_t hit[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                hit[j] = __ballot(x[j] == above && c0 + j >= lo_col && c0 + j < cols);
                here += __popcll(hit[j]);
            }
            __syncthreads();
            if (lane == 0) sh.count[tid >> 6] = here;
            __syncthreads();
            for (int w = 0; w < NT / 64; ++w) {
                if (w < tid >> 6) before += sh.count[w];
                have += sh.count[w];
            }
            // (columns run through the lanes, four to each)
            const uint64_t below = (1ull << lane) - 1;
#pragma unroll
            for (int j = 0; j < 4; ++j) before += __popcll(hit[j] & below);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (hit[j] >> lane & 1) {
                    if (before < k) sh.found[before] = make_float2(x[j], __int_as_float(c0 + j));
                    ++before;
                }
        }
        __syncthreads();
        n = k;
    }
    // Each wave compares its share of the list, read once for several entries of each lane, with
    // all of it: an entry's rank is the sum of what the waves find above it.
    constexpr int kWaves = NT / 64;
    const int share = (n + 2 * kWaves - 1) / (2 * kWaves) * 2, from = (tid >> 6) * share;
    for (int i = tid; i < n; i += NT) {
        sh.rank[i] = 0;
        const float2 x = sh.found[i];
        sh.list[i] = entry_of(x.x, __float_as_int(x.y));
    }
    if (tid < 16) sh.list[n + tid] = 0.0;  // (below every entry: the last reads end past it)
    __syncthreads();
    auto compare = [&](auto each) __attribute__((always_inline)) {
        constexpr int E = decltype(each)::value;
        const int to = min(n, from + share);
        for (int at = lane; at < n + lane; at += 64 * E) {
            double me[E];
            int above[E] = {};
#pragma unroll
            for (int i = 0; i < E; ++i) me[i] = at + 64 * i < n ? sh.list[at + 64 * i] : 0.0;
#pragma unroll 4
            for (int j = from; j < to; j += 2) {
                const double2 x = *reinterpret_cast<const double2 *>(&sh.list[j]);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    above[i] += x.x > me[i] ? 1 : 0;
                    above[i] += x.y > me[i] ? 1 : 0;
                }
            }
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (at + 64 * i < n && above[i]) atomicAdd(&sh.rank[at + 64 * i], above[i]);
        }
    };
    if (n <= 64) compare(std::integral_constant<int, 1>());
    else compare(std::integral_constant<int, 2>());
    __syncthreads();
    for (int i = tid; i < n; i += NT)
        if (sh.rank[i] < k) place(sh.rank[i], row_entry(sh.list[i], first));
}

__device__ __forceinline__ void score_left_out(const ScoreArgs &p, int64_t row, int threads) {
    if (threadIdx.x == 0 && p.logprobs) p.logprobs[row] = 0.0f;
    if (threadIdx.x == 0 && p.entropy) p.entropy[row] = 0.0f;
    for (int j = threadIdx.x; j < p.k; j += threads) {
        p.top_ids[row * p.k + j] = -1;
        p.top_logprobs[row * p.k + j] = -INFINITY;
    }
}

// A row of up to 4 NT NV columns, the shift's among them (PARTS: a part of one), in a
// workgroup's registers.
template <int NT, int NV, bool PARTS>
__global__ __launch_bounds__(NT, 4) void scores_kernel(ScoreArgs p) {
    __shared__ RowSums lds[NT / 64];
    __shared__ TopShared sh;
    const int64_t row = PARTS ? blockIdx.y : blockIdx.x, at = PARTS ? (int64_t)blockIdx.x * p.part : 0;
    const float *z = p.logits + row * p.vocab;
    const int tid = threadIdx.x, shift = line_shift(z);
    const int lo = PARTS ? (int)max((int64_t)0, shift - at) : shift;
    const int cols = (int)(PARTS ? min(p.part, p.vocab + shift - at) : p.vocab + shift);
    const int32_t t = p.targets.given ? p.targets.at(row) : 0;
    if (p.targets.given && t == p.ignore) {
        if (!PARTS) score_left_out(p, row, NT);
        return;
    }
    float e[NV][4];
    const float zt = !PARTS && p.logprobs && tid == 0 ? z[t] : 0.0f;
    load_stretch<NT, NV>(z + at - shift, lo, cols, e);
    RowSums s = no_sums();
    add_stretch<KIND_SCORES>(s, e, kPlain);
    s = wave_sums(s);
    if ((tid & 63) == 0) lds[tid >> 6] = s;
    __syncthreads();
    s = join_sums<KIND_SCORES>(lds, NT / 64, kPlain);
    const bool odd = s.a != s.a;
    float rest = 0.0f;
    if constexpr (PARTS) {
        if (tid == 0) p.sums[row * p.parts + blockIdx.x] = with_nan(s);
    } else {
        s = row_sums(s);
        const float a = rest_of(s);
        rest = log1pf(a);
        if (tid == 0 && p.logprobs) p.logprobs[row] = (zt - s.m) - rest;
        if (tid == 0 && p.entropy) p.entropy[row] = rest - s.u / (1.0f + a);
    }
    if (p.k == 0) return;
    if (odd) {
        // (for the order of alternatives a NaN counts as +inf)
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) e[i][j] = e[i][j] != e[i][j] ? INFINITY : e[i][j];
    }
    const float m = s.m;
    top_of<NT, NV>(e, lo, cols, (uint32_t)(at - shift), p.k, sh, [&](int rank, uint64_t entry) {
        if constexpr (PARTS) {
            p.best[(row * p.parts + blockIdx.x) * p.k + rank] = entry;
        } else {
            p.top_ids[row * p.k + rank] = (int32_t) ~(uint32_t)entry;
            p.top_logprobs[row * p.k + rank] = (value_of((uint32_t)(entry >> 32)) - m) - rest;
        }
    });
}

// The parts of a row together: their sums, and of their lists the k that come first, each
// entry's place the number of larger ones. Latency: 4 rows of 131071, k 20, 13 us in the
// two launches.
constexpr int kJoinEntries = 12 * 256;   // twelve of a thread: 48 KB for both lists
__global__ __launch_bounds__(256) void scores_join_kernel(ScoreArgs p) {
    __shared__ RowSums all;
    __shared__ uint64_t held[kJoinEntries], some[kJoinEntries];
    __shared__ int32_t count;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, k = p.k, parts = p.parts, entries = parts * k;
    const int32_t t = p.targets.given ? p.targets.at(row) : 0;
    if (p.targets.given && t == p.ignore) return score_left_out(p, row, 256);
    const uint64_t *best = p.best + row * entries;
    const bool in_lds = entries <= kJoinEntries && parts <= 256;
    if (in_lds)
        for (int i = tid; i < entries; i += 256) held[i] = best[i];
    if (tid == 0) count = 0;
    if (tid < 64) {
        const RowSums s = wave_join<KIND_SCORES>(p.sums + row * parts, parts, kPlain);
        if (tid == 0) all = s;
    }
    __syncthreads();
    const RowSums s = row_sums(all);
    const float a = rest_of(s), rest = log1pf(a);
    if (tid == 0 && p.logprobs) p.logprobs[row] = (p.logits[row * p.vocab + t] - s.m) - rest;
    if (tid == 0 && p.entropy) p.entropy[row] = rest - s.u / (1.0f + a);
    if (k == 0) return;
    // (the first and the last parts may have fewer columns, and a shorter list)
    const int shift = line_shift(p.logits + row * p.vocab);
    auto length = [&](int q) {
        const int64_t cols = min(p.part, p.vocab + shift - q * p.part) - (q == 0 ? shift : 0);
        return (int)min((int64_t)k, max((int64_t)0, cols));
    };
    auto larger = [](const uint64_t *list, int n, uint64_t than) {
        int lo = 0;
        while (lo < n) {
            const int mid = (lo + n) / 2;
            if (list[mid] > than) lo = mid + 1;
            else n = mid;
        }
        return lo;
    };
    auto place = [&](int rank, uint64_t entry) {
        p.top_ids[row * k + rank] = (int32_t) ~(uint32_t)entry;
        p.top_logprobs[row * k + rank] = (value_of((uint32_t)(entry >> 32)) - s.m) - rest;
    };
    if (!in_lds) {
        // Lists beyond LDS: each entry finds its place by halving every other list.
        for (int i = tid; i < entries; i += 256) {
            const int q = i / k;
            int rank = i - q * k;
            if (rank >= length(q)) continue;
            const uint64_t me = best[i];
            for (int o = 0; o < parts && rank < k; ++o)
                if (o != q) rank += larger(best + (int64_t)o * k, length(o), me);
            if (rank < k) place(rank, me);
        }
        return;
    }
    // With r of the entries of each part but the last (which have more columns than entries)
    // at or above `least` there are k of them: only those (some dozens more than k as a rule) are compared with each other.
    const int r = (k + parts - 2) / (parts - 1);
    uint64_t least = ~0ull;
    for (int q = 0; q < parts - 1; ++q) least = min(least, held[q * k + r - 1]);
    for (int i = tid; i < entries; i += 256)
        if (i % k < length(i / k) && held[i] >= least) some[atomicAdd(&count, 1)] = held[i];
    __syncthreads();
    const int n = count;
    for (int i = tid; i < n; i += 256) {
        const uint64_t me = some[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += some[j] > me ? 1 : 0;
        if (rank < k) place(rank, me);
    }
}

int64_t round_line(int64_t v) { return (v + kLine - 1) / kLine * kLine; }
// Columns of an array's rows with their shift, at most.
int64_t line_cols(const float *rows, int64_t v) {
    return (reinterpret_cast<uintptr_t>(rows) & (4 * kLine - 1)) == 0 && v % kLine == 0 ? v : v + kLine - 1;
}
// Columns of a part at most, of one at least (a row of one column more than a part makes
// three of 16384 at most: a third, in whole lines), and the bytes that the parts' lists
// may take.
constexpr int64_t kScoreCols = 32768, kPartLeast = (kScoreCols / 3 + kLine) / kLine * kLine, kScoreBytes = int64_t(64) << 20;
static_assert(kPartLeast == 10944, "as the header says");

template <bool PARTS>
void launch_scores(Context &cx, const ScoreArgs &p, dim3 grid, int64_t cols) {
    auto launch = [&](auto kernel, int threads) { hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, cx.stream, p); };
    if constexpr (PARTS) {  // (of kPartLeast columns at least)
        if (cols <= 16384) launch(scores_kernel<512, 8, true>, 512);
        else launch(scores_kernel<512, 16, true>, 512);
    } else {
        if (cols <= 1024) launch(scores_kernel<256, 1, false>, 256);
        else if (cols <= 4096) launch(scores_kernel<256, 4, false>, 256);
        else if (cols <= 8192) launch(scores_kernel<512, 4, false>, 512);
        else if (cols <= 16384) launch(scores_kernel<512, 8, false>, 512);
        else launch(scores_kernel<512, 16, false>, 512);
    }
    check_hip(hipGetLastError(), "token_logprobs launch");
}

ScoreArgs rows_from(ScoreArgs p, int64_t row) {
    p.logits += row * p.vocab;
    p.targets.skip(row);
    if (p.logprobs) p.logprobs += row;
    if (p.entropy) p.entropy += row;
    if (p.top_ids) p.top_ids += row * p.k;
    if (p.top_logprobs) p.top_logprobs += row * p.k;
    return p;
}

void scores(Context &cx, const ScoreArgs &all, int64_t n) {
    const int64_t v = all.vocab;
    const int64_t cols = line_cols(all.logits, v);
    if (cols <= kScoreCols) {
        for (int64_t at = 0; at < n; at += kMaxRows)
            launch_scores<false>(cx, rows_from(all, at), dim3((unsigned)std::min(kMaxRows, n - at)), cols);
        return;
    }
    // parts for two workgroups per CU, of 16384 columns or the few thousand less that parts of
    // one size come to, kPartLeast (of 4096: 4 x 131071 15.2 -> 17.9 us, 1 x 262144 15.6 ->
    // 24.5: more lists to join), whose lists fit the join's LDS
    const int64_t fit = std::min<int64_t>(256, kJoinEntries / std::max(1, all.k));
    const int64_t want = std::max((cols + kScoreCols - 1) / kScoreCols, std::min({(cols + 16383) / 16384, 2 * cx.cu_count / n, fit}));
    const int64_t part = round_line((cols + want - 1) / want), parts = (cols + part - 1) / part;
    const int64_t row_bytes = parts * ((int64_t)sizeof(RowSums) + 8 * all.k);
    const int64_t block = std::min({n, std::max<int64_t>(1, kScoreBytes / row_bytes), std::max<int64_t>(1, (int64_t(1) << 22) / parts), int64_t(65535)});
    char *ws = static_cast<char *>(cx.workspace(2, (size_t)(block * row_bytes)));
    for (int64_t at = 0; at < n; at += block) {
        ScoreArgs p = rows_from(all, at);
        const unsigned rows = (unsigned)std::min(block, n - at);
        p.part = part;
        p.parts = (int)parts;
        p.sums = reinterpret_cast<RowSums *>(ws);
        p.best = reinterpret_cast<uint64_t *>(ws + block * parts * (int64_t)sizeof(RowSums));
        launch_scores<true>(cx, p, dim3((unsigned)parts, rows), part);
        hipLaunchKernelGGL(scores_join_kernel, dim3(rows), dim3(256), 0, cx.stream, p);
        check_hip(hipGetLastError(), "token_logprobs launch");
    }
}

// ---- gradients of a row's logits, and the distillation loss -----------------------
// Every gradient here is exp(d rate) times a line in d (KIND_SCORES) or a constant,
// KIND_BOTH with a second exponential at rate 1, less a weight at a few tokens: the
// teacher's slots and the target. A row's logits stay in registers between the sums and
// the gradient, so that the logits are read and the gradient written once, which bounds
// it: 4096 x 32000 with both terms 208 us, 5.0 TB/s (a copy of as much 215), log
// probabilities' with a quarter of the rows left out 175, 5.2 TB/s; 817 rows of 131071 and 204
// left out 212, 4.6 TB/s.
struct RowArgs {
    const float *logits;
    HostIds targets;
    int64_t vocab;
    int32_t ignore;
    float *out;              // dlogits, which may be the logits; null: the loss alone
    const float *dlogprobs, *dentropy;  // KIND_SCORES, each may be null
    // distillation
    const int32_t *ids;
    const float *teacher;
    int k;
    float temperature, alpha, scale;  // scale: 1 / the rows that count
    Rate rate;                        // of the first exponential: at the temperature, or 1 (KIND_SCORES, alpha 0)
    Rate inverse;                     // 1 / temperature
    float *row_loss;                  // [rows], 0 for a row that is left out
    int32_t *wrong;                   // receives 1 for a teacher's id beyond the vocabulary
    bool stream;
    // a row over several workgroups (parts_kernel, parts_grad_kernel)
    int64_t part;     // columns of a part, a multiple of kLine
    int parts;
    RowSums *sums;    // [rows, parts]
    float *slot_z;    // [rows, k + 1]
};

// (log probabilities' is a constant)
template <int KIND>
__device__ __forceinline__ Rate rate_for(const RowArgs &p) {
    return KIND == KIND_SCORES ? kPlain : p.rate;
}

// What the threads of a row share after its sums are known.
struct RowShared {
    RowSums parts[16];
    int32_t filled[8];  // of the waves: whether one of their slots is the teacher's
    int32_t id[kMaxTop + 1];
    float weight[kMaxTop + 1], z[kMaxTop + 1];
    float own;           // the target's gradient but for the teacher's shares, if its logit is the largest
};

// The teacher's softmax over the slots in LDS (values in weight), by one wave: weight
// becomes soft q. Returns sum_j q_j (ln q_j - ln p_T(id_j)), `a` the S - 1 of p_T. Logits are
// subtracted from logits and the logarithm taken of the two sums' quotient, by what it
// differs from 1 where that is little: each ln q and ln p on its own is some 10, whose
// rounding T^2 would make larger than a small term. log_hard: ln(1 + hard), formed beside
// the others.
__device__ __forceinline__ float teacher_terms(RowShared &sh, int k, const Rate &rate, const Rate &inverse, float soft, float m,
                                               float a, float hard, float &log_hard) {
    const int lane = threadIdx.x & 63;
    float t[kMaxTop / 64], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kMaxTop / 64; ++i) {
        t[i] = lane + 64 * i < k ? sh.weight[lane + 64 * i] : -INFINITY;
        top = fmaxf(top, ranked(t[i]));
    }
    top = wave_max(top);
    // (a row of empty slots has no teacher: every share 0)
    const float base = top == -INFINITY ? 0.0f : top;
    float some = 0.0f, e[kMaxTop / 64];
    int count = 0;
#pragma unroll
    for (int i = 0; i < kMaxTop / 64; ++i) {
        t[i] -= base;
        e[i] = exp_of(t[i], rate);
        count += __popcll(__ballot(t[i] == 0.0f));
        some += t[i] == 0.0f ? 0.0f : e[i];
    }
    // (a lane to each logarithm: one after another, 2048 rows of 4096 11 -> 12 us. Elsewhere the
    // difference of two: logf of the quotient is off by half a step of f32 on average, 5e-8 of
    // losses over 4096 rows.)
    const float rest = wave_sum(some) + (float)(count - 1), off = (rest - a) / (1.0f + a);
    const float log = log1pf(lane == 0 ? rest : lane == 1 ? a : lane == 2 ? off : hard);
    auto log_of = [&](int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(log), i)); };
    const float f = top == -INFINITY ? 0.0f : 1.0f / (1.0f + rest);
    const float log_ratio = fabsf(off) < 0.5f ? log_of(2) : log_of(0) - log_of(1);
    log_hard = log_of(3);
    float kl = 0.0f;
#pragma unroll
    for (int i = 0; i < kMaxTop / 64; ++i) {
        const int j = lane + 64 * i;
        if (j >= k) break;
        const float q = e[i] * f;
        if (q != 0.0f) kl += q * (times(t[i] - (sh.z[j] - m), inverse) - log_ratio);
        sh.weight[j] = soft * q;
    }
    return wave_sum(kl);
}

// The slots of a row on their way to LDS: 0 .. k - 1 the teacher's, slot k its target.
// Their loads go out with the target's, before it is known whether the row counts.
template <int NT>
struct Slots {
    static constexpr int N = (kMaxTop + NT) / NT;
    int32_t id[N];
    float weight[N], z[N];
    __device__ __forceinline__ void load(const RowArgs &p, int64_t row, int k) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = threadIdx.x + NT * i;
            id[i] = j < k ? p.ids[row * k + j] : -1;
            weight[i] = j < k ? p.teacher[row * k + j] : 0.0f;
        }
    }
    // z_of(slot, id): the id's logit
    template <class F>
    __device__ __forceinline__ void gather(const RowArgs &p, int k, int32_t t, F &&z_of) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = threadIdx.x + NT * i;
            if (j == k) id[i] = t;
            if (id[i] >= p.vocab) {
                *p.wrong = 1;
                id[i] = -1;
            }
            z[i] = id[i] < 0 ? 0.0f : z_of(j, id[i]);
        }
    }
    __device__ __forceinline__ void store(int k, RowShared &sh) const {
        bool some = false;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = threadIdx.x + NT * i;
            if (j > k) break;
            sh.id[j] = id[i] < 0 ? -1 : id[i];
            sh.weight[j] = id[i] < 0 ? -INFINITY : weight[i];
            sh.z[j] = z[i];
            some |= j < k && id[i] >= 0 && weight[i] != -INFINITY;
        }
        some = __any(some);
        if ((threadIdx.x & 63) == 0) sh.filled[threadIdx.x >> 6] = some;
    }
};

// A row that is left out. Its columns at .. end - 1 of the output are zeros.
template <int NT>
__device__ __forceinline__ void left_out(const RowArgs &p, int64_t row, int64_t at, int64_t end) {
    if (p.row_loss && at == 0 && threadIdx.x == 0) p.row_loss[row] = 0.0f;
    if (!p.out) return;
    float *out = p.out + row * p.vocab;
    const float zero[4] = {};
    for (int64_t j = at + 4 * (int64_t)threadIdx.x; j < end; j += 4 * NT) store4(out + j, (int)min((int64_t)4, end - j), zero);
}
// The shift of a row that is read, or of the output's that is written.
__device__ __forceinline__ int row_shift(const RowArgs &p, int64_t row) {
    return line_shift((p.out ? p.out : p.logits) + row * p.vocab);
}

// A row's dense gradient exp((z - m) rate) (f0 + f1 (z - m)) (KIND_SCORES; KIND_ONE: f1 =
// 0; KIND_BOTH: f1 times the second exponential instead), and what its target has less.
struct Dense {
    Rate rate;
    float m, f0, f1, hit;
    template <int KIND>
    __device__ __forceinline__ float at(float x) const {
        const float d = x - m, e = exp_of(d, rate);
        if (KIND == KIND_SCORES) return e * __builtin_fmaf(fmaxf(d, kFar), f1, f0);
        const float g = e * f0;
        return KIND == KIND_BOTH ? __builtin_fmaf(exp_of(d, kPlain), f1, g) : g;
    }
};

// From the row's sums, by every thread; wave 0 turns the teacher's slots into shares,
// and its lane 0 writes the row's loss where `loss`.
template <int NT, int KIND>
__device__ __forceinline__ Dense coefficients(const RowArgs &p, int64_t row, int k, const RowSums &s, bool loss_too,
                                              RowShared &sh) {
    const float a = rest_of(s), total = 1.0f + a;
    Dense g{rate_for<KIND>(p), s.m, 0.0f, 0.0f, 0.0f};
    if constexpr (KIND == KIND_SCORES) {
        // (ln p + H is d - sum exp(d) d / S: what a certain token has there is as small as u)
        const float dl = p.dlogprobs ? p.dlogprobs[row] : 0.0f, dh = p.dentropy ? p.dentropy[row] : 0.0f;
        const float bent = dh * (s.u / total);
        g.f0 = (bent - dl) / total;
        g.f1 = -dh / total;
        g.hit = -dl;
        if (threadIdx.x == 0) sh.own = dl * (a / total) + bent / total;
    } else {
        // (the soft term's derivative is that of sum q (ln q - ln p_T), p_T times the sum of
        // q, less q: a row of empty slots has neither)
        int32_t filled = 0;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) filled |= sh.filled[i];
        const float soft = filled ? p.alpha * p.temperature * p.scale : 0.0f, hard = (1.0f - p.alpha) * p.scale;
        const float rest1 = s.u + (s.count - 1.0f);  // (KIND_BOTH)
        g.f0 = (KIND == KIND_BOTH ? soft : soft + hard) / total;
        if (KIND == KIND_BOTH) g.f1 = hard / (1.0f + rest1);
        g.hit = hard;
        const float other = KIND == KIND_BOTH ? rest1 : a;
        if (threadIdx.x == 0) sh.own = soft / total - hard * (other / (1.0f + other));
        if (threadIdx.x < 64) {
            float loss = 0.0f, log_hard;
            const float kl = teacher_terms(sh, k, p.rate, p.inverse, soft, s.m, a, other, log_hard);
            if (p.alpha > 0.0f) loss = p.alpha * p.temperature * p.temperature * kl;
            if (p.alpha < 1.0f) loss += (1.0f - p.alpha) * (log_hard - (sh.z[k] - s.m));
            // (without a distribution the loss is NaN, also where no term above has met it)
            if (a != a) loss = a;
            if (loss_too && threadIdx.x == 0) p.row_loss[row] = loss;
        }
    }
    return g;
}

// The few tokens' own values, for columns at .. end - 1, after the dense ones: an
// id's first slot takes the shares of all its slots. A target whose logit is the largest
// has 1 - p = rest / S, which keeps its bits where p is near 1.
template <int NT, int KIND>
__device__ __forceinline__ void patch(float *out, int64_t at, int64_t end, int k, const Dense &g, const RowShared &sh) {
    for (int j = threadIdx.x; j <= k; j += NT) {
        const int32_t id = sh.id[j];
        if (id < at || id >= end) continue;
        float w = 0.0f;
        bool first = true;
        for (int i = 0; i < k; ++i)
            if (sh.id[i] == id) {
                first = first && i >= j;
                w += sh.weight[i];
            }
        if (!first) continue;
        const float z = sh.z[j];
        const bool target = sh.id[k] == id;
        out[id] = target && z == g.m ? sh.own - w : g.at<KIND>(z) - (target ? w + g.hit : w);
    }
}

// A row of up to 4 NT NV columns, the shift's among them, in a workgroup's registers: read
// once.
template <int NT, int NV, int KIND>
__global__ __launch_bounds__(NT, 4) void rows_kernel(RowArgs p) {
    __shared__ RowShared sh;
    const int64_t row = blockIdx.x;
    const int v = (int)p.vocab, tid = threadIdx.x;
    const float *z = p.logits + row * p.vocab;
    const int k = KIND == KIND_SCORES ? 0 : p.k;
    Slots<NT> slots;
    slots.load(p, row, k);
    const int32_t t = p.targets.given ? p.targets.at(row) : -1;
    if (p.targets.given && t == p.ignore) return left_out<NT>(p, row, 0, v);
    slots.gather(p, k, t, [&](int, int32_t id) { return z[id]; });
    float e[NV][4];
    RowSums s = no_sums();
    const int shift = row_shift(p, row);
    load_stretch<NT, NV>(z - shift, shift, shift + v, e);
    slots.store(k, sh);
    add_stretch<KIND>(s, e, rate_for<KIND>(p));
    s = wave_sums(s);
    if ((tid & 63) == 0) sh.parts[tid >> 6] = s;
    __syncthreads();
    s = row_sums(join_sums<KIND>(sh.parts, NT / 64, rate_for<KIND>(p)));
    const Dense g = coefficients<NT, KIND>(p, row, k, s, true, sh);
    if (!p.out) return;
    float *out = p.out + row * p.vocab;
    // (addresses formed anew: kept from the loads they would take the row's registers)
    int me = tid;
    asm volatile("" : "+v"(me));
    write_stretch<NT, NV>(out - shift, shift, shift + v, p.stream, e, me, [&](float x) { return g.at<KIND>(x); });
    __syncthreads();
    patch<NT, KIND>(out, 0, v, k, g, sh);
}

// Wider rows, of 2048 R columns at least: 512 threads have a CU's registers, and hold the
// row's first R strips there and L after them in LDS (98304 and 32768 columns of f32 with
// 48 and 16). Only what follows those is read twice. (`some`, 8 strips at a time, is what
// passes through.)
template <int R, int L, int KIND>
__global__ __launch_bounds__(512, 2) void wide_rows_kernel(RowArgs p) {
    constexpr int NT = 512, S = 8, kSome = 4 * NT * S;
    static_assert(L % S == 0, "whole passes");
    __shared__ RowShared sh;
    __shared__ __attribute__((aligned(16))) float held[L ? L * NT * 4 : 4];
    const int64_t row = blockIdx.x, v = p.vocab;
    const float *z = p.logits + row * v;
    const int tid = threadIdx.x;
    const int k = KIND == KIND_SCORES ? 0 : p.k;
    Slots<NT> slots;
    slots.load(p, row, k);
    const int32_t t = p.targets.given ? p.targets.at(row) : -1;
    if (p.targets.given && t == p.ignore) return left_out<NT>(p, row, 0, v);
    slots.gather(p, k, t, [&](int, int32_t id) { return z[id]; });
    slots.store(k, sh);
    const Rate kx = rate_for<KIND>(p);
    RowSums s = no_sums();
    const int shift = row_shift(p, row);
    constexpr int64_t kHeld = 4 * NT * R, kKept = kHeld + 4 * NT * L;
    const int64_t total = v + shift;
    const int passes = (int)(max((int64_t)0, total - kKept + kSome - 1) / kSome);
    auto cols_at = [&](int64_t at, int64_t end) { return (int)max((int64_t)0, min((int64_t)kSome, min(total, end) - at)); };
    z -= shift;
    {
        float some[S][4];
        for (int i = 0; i < passes; ++i) {
            const int64_t at = kKept + (int64_t)i * kSome;
            load_stretch<NT, S>(z + at, 0, cols_at(at, total), some);
            add_stretch<KIND>(s, some, kx);
        }
#pragma unroll 1
        for (int i = 0; i < L / S; ++i) {
            const int64_t at = kHeld + (int64_t)i * kSome;
            if (at >= total) break;
            load_stretch<NT, S>(z + at, 0, cols_at(at, kKept), some);
            add_stretch<KIND>(s, some, kx);
#pragma unroll
            for (int r = 0; r < S; ++r) __builtin_memcpy(__builtin_assume_aligned(&held[((i * S + r) * NT + tid) * 4], 16), some[r], 16);
        }
    }
    const uint32_t lane_at = 16u * (uint32_t)tid;
    float e[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        // (columns below the shift: any of the row's in their place at first)
        const uint32_t from = r == 0 ? max(lane_at, 4u * (uint32_t)shift) : lane_at;
        __builtin_memcpy(e[r], reinterpret_cast<const char *>(z) + 16 * NT * r + from, 16);
        __builtin_amdgcn_sched_barrier(0);  // (one address at a time: no registers for more)
    }
    if (4 * tid < shift) {
#pragma unroll
        for (int j = 0; j < 4; ++j) e[0][j] = 4 * tid + j >= shift ? z[4 * tid + j] : -INFINITY;
    }
    add_stretch<KIND>(s, e, kx);
    s = wave_sums(s);
    if ((tid & 63) == 0) sh.parts[tid >> 6] = s;
    __syncthreads();
    s = row_sums(join_sums<KIND>(sh.parts, NT / 64, kx));
    const Dense g = coefficients<NT, KIND>(p, row, k, s, true, sh);
    if (!p.out) return;
    float *out = p.out + row * v - shift;
    // (the addresses from here on are formed anew: kept from the first pass they would
    // take the registers that hold the row)
    int me = tid;
    asm volatile("" : "+v"(me));
    auto turn = [&](float x) { return g.at<KIND>(x); };
    write_stretch<NT, R>(out, shift, (int)kHeld, p.stream, e, me, turn);
#pragma unroll 1
    for (int i = 0; i < L / S; ++i) {
        const int64_t at = kHeld + (int64_t)i * kSome;
        if (at >= total) break;
        float some[S][4];
#pragma unroll
        for (int r = 0; r < S; ++r) __builtin_memcpy(some[r], __builtin_assume_aligned(&held[((i * S + r) * NT + me) * 4], 16), 16);
        write_stretch<NT, S>(out + at, 0, cols_at(at, kKept), p.stream, some, me, turn);
    }
    for (int i = passes - 1; i >= 0; --i) {
        float some[S][4];
        const int64_t at = kKept + (int64_t)i * kSome;
        load_stretch<NT, S>(z + at, 0, cols_at(at, total), some, me);
        write_stretch<NT, S>(out + at, 0, cols_at(at, total), p.stream, some, me, turn);
    }
    __syncthreads();
    patch<NT, KIND>(out + shift, 0, v, k, g, sh);
}

// A row over several workgroups, one part of at most 4 NT NV columns each: first the
// parts' sums and the slots' logits (dlogits may be the logits, which the second
// launch overwrites), then the gradient. Latency: 4 rows of 131071 13 us in two launches.
template <int NT, int NV, int KIND>
__global__ __launch_bounds__(NT, 4) void parts_kernel(RowArgs p) {
    __shared__ RowSums parts[NT / 64];
    const int64_t row = blockIdx.y, at = (int64_t)blockIdx.x * p.part, v = p.vocab;
    const int32_t t = p.targets.given ? p.targets.at(row) : -1;
    if (p.targets.given && t == p.ignore) return;
    const float *z = p.logits + row * v;
    const int shift = row_shift(p, row), k = KIND == KIND_SCORES ? 0 : p.k;
    const int lo = (int)max((int64_t)0, shift - at), cols = (int)min(p.part, v + shift - at);
    for (int j = threadIdx.x; j <= k; j += NT) {
        const int32_t id = j < k ? p.ids[row * k + j] : t;
        if (id >= 0 && (int64_t)id + shift >= at && (int64_t)id + shift < at + cols) p.slot_z[row * (k + 1) + j] = z[id];
    }
    float e[NV][4];
    RowSums s = no_sums();
    load_stretch<NT, NV>(z + at - shift, lo, cols, e);
    add_stretch<KIND>(s, e, rate_for<KIND>(p));
    s = wave_sums(s);
    if ((threadIdx.x & 63) == 0) parts[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) p.sums[row * p.parts + blockIdx.x] = with_nan(join_sums<KIND>(parts, NT / 64, rate_for<KIND>(p)));
}

template <int NT, int NV, int KIND>
__global__ __launch_bounds__(NT, 4) void parts_grad_kernel(RowArgs p) {
    __shared__ RowShared sh;
    const int64_t row = blockIdx.y, at = (int64_t)blockIdx.x * p.part, v = p.vocab;
    const int shift = row_shift(p, row);
    const int lo = (int)max((int64_t)0, shift - at), cols = (int)min(p.part, v + shift - at);
    // (the row's own columns)
    const int64_t from = max((int64_t)0, at - shift), end = min(v, at - shift + p.part);
    const int32_t t = p.targets.given ? p.targets.at(row) : -1;
    if (p.targets.given && t == p.ignore) return left_out<NT>(p, row, from, end);
    const float *z = p.logits + row * v;
    const int k = KIND == KIND_SCORES ? 0 : p.k, tid = threadIdx.x;
    const Rate kx = rate_for<KIND>(p);
    float e[NV][4];
    if (p.out) load_stretch<NT, NV>(z + at - shift, lo, cols, e);
    Slots<NT> slots;
    slots.load(p, row, k);
    slots.gather(p, k, t, [&](int j, int32_t) { return p.slot_z[row * (k + 1) + j]; });
    slots.store(k, sh);
    if (tid < 64) {
        const RowSums all = wave_join<KIND>(p.sums + row * p.parts, p.parts, kx);
        if (tid == 0) sh.parts[0] = all;
    }
    __syncthreads();
    const RowSums s = row_sums(sh.parts[0]);
    const Dense g = coefficients<NT, KIND>(p, row, k, s, blockIdx.x == 0, sh);
    if (!p.out) return;
    float *out = p.out + row * v;
    write_stretch<NT, NV>(out + at - shift, lo, cols, p.stream, e, tid, [&](float x) { return g.at<KIND>(x); });
    __syncthreads();
    patch<NT, KIND>(out, from, end, k, g, sh);
}

// Outputs from this size on, what the GPU's last cache holds, pass the caches by. With what
// reads them next: distillation of 4096 x 32000 and a copy of dlogits 415 -> 406 us, and a
// product with it 682 -> 671; of 1024 x 32000 and a copy 115, so 122.
constexpr int64_t kStreamBytes = int64_t(256) << 20;
// Rows of up to kRowCols columns, the shift's among them, stay in one workgroup's registers.
constexpr int64_t kRowCols = 32768;
constexpr int kPartThreads = 256, kPartStrips = 8;
constexpr int64_t kPartCols = 4 * kPartThreads * kPartStrips;
// Rows by their parts in one pair of launches (their sums' workspace; a grid's y).
constexpr int64_t kPartRows = 4096;

// n rows from `row` on.
RowArgs rows_from(RowArgs p, int64_t row) {
    p.logits += row * p.vocab;
    p.targets.skip(row);
    if (p.out) p.out += row * p.vocab;
    if (p.dlogprobs) p.dlogprobs += row;
    if (p.dentropy) p.dentropy += row;
    if (p.ids) p.ids += row * p.k;
    if (p.teacher) p.teacher += row * p.k;
    if (p.row_loss) p.row_loss += row;
    return p;
}

int64_t row_cols(const RowArgs &p) { return line_cols(p.out ? p.out : p.logits, p.vocab); }

template <int KIND>
void launch_whole(Context &cx, const RowArgs &all, int64_t n) {
    const int64_t cols = row_cols(all);
    for (int64_t at = 0; at < n; at += kMaxRows) {
        const RowArgs p = rows_from(all, at);
        const int64_t rows = std::min(kMaxRows, n - at);
        auto launch = [&](auto kernel, int threads) {
            hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(threads), 0, cx.stream, p);
        };
        // (a row's columns with its shift; the wide kernels take what they do not hold in passes)
        if (cols <= 1024) launch(rows_kernel<256, 1, KIND>, 256);
        else if (cols <= 4096) launch(rows_kernel<256, 4, KIND>, 256);
        else if (cols <= 8192) launch(rows_kernel<512, 4, KIND>, 512);
        else if (cols <= 16384) launch(rows_kernel<512, 8, KIND>, 512);
        else if (cols <= kRowCols) launch(rows_kernel<512, 16, KIND>, 512);
        else if (p.vocab < 32768) launch(wide_rows_kernel<8, 16, KIND>, 512);
        else if (p.vocab < 65536) launch(wide_rows_kernel<16, 16, KIND>, 512);
        else if (p.vocab < 98304) launch(wide_rows_kernel<32, 16, KIND>, 512);
        else launch(wide_rows_kernel<48, 16, KIND>, 512);
        check_hip(hipGetLastError(), "rows launch");
    }
}

template <int KIND>
void launch_parts(Context &cx, const RowArgs &all, int64_t n) {
    const int64_t v = all.vocab, cols = row_cols(all), slots = KIND == KIND_SCORES ? 1 : all.k + 1;
    // parts for two workgroups per CU, of 1024 columns at least
    const int64_t want = std::max((cols + kPartCols - 1) / kPartCols, std::min((v + 1023) / 1024, 2 * cx.cu_count / n));
    const int64_t part = round_line((cols + want - 1) / want), parts = (cols + part - 1) / part;
    const int64_t block = std::min({n, kPartRows, std::max<int64_t>(1, (int64_t(1) << 23) / parts)});
    const size_t sums = (size_t)(block * parts) * sizeof(RowSums);
    char *ws = static_cast<char *>(cx.workspace(2, sums + (size_t)(block * slots) * 4));
    for (int64_t at = 0; at < n; at += block) {
        RowArgs p = rows_from(all, at);
        p.part = part;
        p.parts = (int)parts;
        p.sums = reinterpret_cast<RowSums *>(ws);
        p.slot_z = reinterpret_cast<float *>(ws + sums);
        const unsigned rows = (unsigned)std::min(block, n - at);
        hipLaunchKernelGGL((parts_kernel<kPartThreads, kPartStrips, KIND>), dim3((unsigned)parts, rows), dim3(kPartThreads), 0, cx.stream, p);
        check_hip(hipGetLastError(), "row parts launch");
        hipLaunchKernelGGL((parts_grad_kernel<kPartThreads, kPartStrips, KIND>), dim3(p.out ? (unsigned)parts : 1u, rows),
                           dim3(kPartThreads), 0, cx.stream, p);
        check_hip(hipGetLastError(), "row parts launch");
    }
}

// Rows by a workgroup each. A few wide ones, a quarter of the CUs at most, by their parts:
// 64 rows of 131071 26 -> 20 us for log probabilities' gradients, one 21 -> 11, but 128 rows
// 29 -> 34; rows of up to kRowCols never (one of 32000 9 -> 12).
// targets_host: of the n rows, where some may be left out.
template <int KIND>
void launch_rows(Context &cx, RowArgs p, int64_t n, const int32_t *targets_host) {
    p.stream = n * p.vocab * 4 >= kStreamBytes;
    if (row_cols(p) <= kRowCols) return launch_whole<KIND>(cx, p, n);
    int64_t kept = n;
    if (targets_host) kept -= std::count(targets_host, targets_host + n, p.ignore);
    if (kept <= cx.cu_count / 4) launch_parts<KIND>(cx, p, n);
    else launch_whole<KIND>(cx, p, n);
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
    RowArgs p{};
    p.vocab = d.vocab;
    p.ignore = d.ignore;
    p.k = d.alpha > 0.0f ? (int)d.k : 0;  // (the teacher has no share at alpha 0)
    p.temperature = d.temperature;
    p.alpha = d.alpha;
    p.rate = rate_of(kLog2e / (d.alpha > 0.0f ? (double)d.temperature : 1.0));
    p.inverse = rate_of(1.0 / (double)d.temperature);
    p.scale = 1.0f / (float)std::max<int64_t>(1, kept);
    p.wrong = pinned;
    *pinned = 0;
    float *rows = reinterpret_cast<float *>(pinned + 16);
    if (d.targets && d.n <= HostIds::kHere) {
        p.targets = host_ids(cx, d.targets, d.n, 1);
    } else if (d.targets) {
        // (the call waits: its kernels read them where they are)
        p.targets.given = 1;
        p.targets.ids = pinned + 16 + d.n;
        std::copy(d.targets, d.targets + d.n, pinned + 16 + d.n);
    }
    p.logits = d.logits;
    p.ids = d.ids;
    p.teacher = d.teacher;
    p.row_loss = rows;
    p.out = dlogits;
    // (with one temperature, or one term, one exponential serves both)
    if (d.alpha > 0.0f && d.alpha < 1.0f && d.temperature != 1.0f) launch_rows<KIND_BOTH>(cx, p, d.n, d.targets);
    else launch_rows<KIND_ONE>(cx, p, d.n, d.targets);
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
        ScoreArgs p{};
        p.logits = logits;
        p.targets = host_ids(cx, targets_host, n, 1);
        p.vocab = vocab;
        p.ignore = ignore;
        p.k = (int)k;
        p.logprobs = logprobs;
        p.entropy = entropy;
        p.top_ids = top_ids;
        p.top_logprobs = top_logprobs;
        scores(cx, p, n);
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
        RowArgs p{};
        p.logits = logits;
        p.targets = host_ids(cx, targets_host, n, 1);
        p.vocab = vocab;
        p.ignore = ignore;
        p.dlogprobs = dlogprobs;
        p.dentropy = dentropy;
        p.out = dlogits;
        launch_rows<KIND_SCORES>(cx, p, n, targets_host);
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
