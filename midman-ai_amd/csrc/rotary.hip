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
#include "mmh_elementwise.h"
#include "mmh_ids.h"
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

// sin and cos in f64 to a few 2^-53: the angle less the nearest multiple of pi / 2 (its
// f64 value and the next 53 bits of it), and their Taylor series to r^15 and r^16, whose
// next terms are below 2^-54 for |r| <= pi / 4. (libm's is made for every angle: 131072 x
// 64 31 us with it, 27.5 so.)
__device__ __forceinline__ void sin_cos(double angle, double &s, double &c) {
    if (!(fabs(angle) < 1e9)) {
        sincos(angle, &s, &c);
        return;
    }
    const double k = rint(angle * 0.63661977236758134308);
    const double r = fma(-k, 6.12323399573676603587e-17, fma(-k, 1.57079632679489661923, angle)), x = r * r;
    double p = -1.0 / 1307674368000.0, q = 1.0 / 20922789888000.0;
    p = fma(p, x, 1.0 / 6227020800.0);
    q = fma(q, x, -1.0 / 87178291200.0);
    p = fma(p, x, -1.0 / 39916800.0);
    q = fma(q, x, 1.0 / 479001600.0);
    p = fma(p, x, 1.0 / 362880.0);
    q = fma(q, x, -1.0 / 3628800.0);
    p = fma(p, x, -1.0 / 5040.0);
    q = fma(q, x, 1.0 / 40320.0);
    p = fma(p, x, 1.0 / 120.0);
    q = fma(q, x, -1.0 / 720.0);
    p = fma(p, x, -1.0 / 6.0);
    q = fma(q, x, 1.0 / 24.0);
    q = fma(q, x, -0.5);
    const double sr = fma(r * x, p, r), cr = fma(q, x, 1.0);
    const int quarter = (int)k;
    const double a = quarter & 1 ? cr : sr, b = quarter & 1 ? sr : cr;
    s = quarter & 2 ? -a : a;
    c = (quarter + 1) & 2 ? -b : b;
}

// Lanes of a row of n units: a power of two, 256 at most.
int lane_bits(int64_t n) {
    int bits = 0;
    while (bits < 8 && (int64_t(1) << bits) < n) ++bits;
    return bits;
}

// A thread has a pair's column, whose frequency (two powers in f64, as long as a score
// of angles) is formed once for the workgroup, and `rows` positions of it: 131072 x 64
// 25 us, 2.7 TB/s of writes (a frequency for each thread and 16 positions 27.5, 4 48; for
// each angle 139).
__global__ __launch_bounds__(256) void rotary_tables_kernel(RotaryTable p, int bits, int rows, float *cos_t, float *sin_t) {
    __shared__ double frequencies[256];
    const int64_t half = p.width / 2, step = 256 >> bits, lanes = int64_t(1) << bits;
    const int64_t first = (int64_t)blockIdx.x * rows * step + (threadIdx.x >> bits);
    for (int64_t col = 0; col < half; col += lanes) {
        __syncthreads();
        if (threadIdx.x < lanes && col + threadIdx.x < half) frequencies[threadIdx.x] = frequency(p, col + threadIdx.x);
        __syncthreads();
        const int64_t i = col + (threadIdx.x & (lanes - 1));
        if (i >= half) continue;
        const double w = frequencies[threadIdx.x & (lanes - 1)];
        for (int r = 0; r < rows; ++r) {
            const int64_t pos = first + r * step;
            if (pos >= p.positions) break;
            double s, c;
            sin_cos((double)pos * w, s, c);
            cos_t[pos * half + i] = (float)(c * p.amplitude);
            sin_t[pos * half + i] = (float)(s * p.amplitude);
        }
    }
}

struct RotaryArgs {
    const float *q, *k, *cos_t, *sin_t;
    float *q_out, *k_out;
    HostIds positions;
    int64_t hd, half, first;
    int32_t places, t, h, heads;  // places: b * t, from `first` on; heads: those of q (h) and k
    int32_t units, rotated;       // four columns (or pairs of columns) each; the others are copied
    float sign;
};

// Past the caches: the next kernel finds it in memory's own cache either way, and this
// one ends without their write-back (4 x 1024 tokens of 24 heads of 128 24 -> 17 us, with
// the attention after it 129.0 -> 128.8; 8 x 2048 82 -> 57, 794 -> 782).
__device__ __forceinline__ void stream4(float *p, int count, const float (&v)[4]) {
    typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
    if (count < 4) return store4(p, count, v);
    float4u x;
    __builtin_memcpy(&x, v, 16);
    __builtin_nontemporal_store(x, reinterpret_cast<float4u *>(p));
}

// A unit of four pairs (half layout), of two (interleaved) or of four columns that are
// copied, up to `count` columns of each of its float4s. H heads of one place at a
// time: the table's row and the loads of all of them go out together. Bound by its reads
// and writes (4 x 1024 tokens of 24 heads of 128 16 us, 6.3 TB/s; two or eight heads at a
// time no faster).
template <int H, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p, int bits) {
    const int64_t place = p.first + (int64_t)blockIdx.x * (256 >> bits) + (threadIdx.x >> bits);
    if (place >= p.places) return;
    const uint32_t b = (uint32_t)place / (uint32_t)p.t, t = (uint32_t)place - b * (uint32_t)p.t;
    const int64_t row = p.positions.given ? p.positions.at(place) : (int64_t)t;
    const int head0 = blockIdx.y * H;
    const int64_t hkv = p.heads - p.h;
    for (int u = threadIdx.x & ((1 << bits) - 1); u < p.units; u += 1 << bits) {
        const bool turn = u < p.rotated;
        // the unit's first column, and that of the pairs' other halves
        const int64_t width = 2 * p.half, c0 = turn ? 4 * (int64_t)u : width + 4 * (int64_t)(u - p.rotated), c1 = c0 + p.half;
        const int count = (int)min((int64_t)4, (turn ? (INTERLEAVED ? width : p.half) : p.hd) - c0);
        const bool both = turn && !INTERLEAVED;
        float c[4] = {}, s[4] = {}, x[H][4], y[H][4];
        if (turn) {
            const int64_t at = row * p.half + (INTERLEAVED ? 2 : 4) * (int64_t)u;
            load4(p.cos_t + at, INTERLEAVED ? count / 2 : count, c);
            load4(p.sin_t + at, INTERLEAVED ? count / 2 : count, s);
        }
        auto at_head = [&](int i, const float *&src, float *&dst) {
            const int64_t j = head0 + i;
            const bool is_k = j >= p.h;
            const int64_t at = ((is_k ? b * hkv + (j - p.h) : (int64_t)b * p.h + j) * p.t + t) * p.hd;
            src = (is_k ? p.k : p.q) + at;
            dst = (is_k ? p.k_out : p.q_out) + at;
        };
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if (head0 + i >= p.heads) break;
            const float *src;
            float *dst;
            at_head(i, src, dst);
            load4(src + c0, count, x[i]);
            if (both) load4(src + c1, count, y[i]);
        }
#pragma unroll
        for (int i = 0; i < H; ++i) {
            if (head0 + i >= p.heads) break;
            const float *src;
            float *dst;
            at_head(i, src, dst);
            float o[4], o1[4];
            if (INTERLEAVED && turn) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float sj = s[j] * p.sign, a = x[i][2 * j], d = x[i][2 * j + 1];
                    o[2 * j] = __fsub_rn(__fmul_rn(a, c[j]), __fmul_rn(d, sj));
                    o[2 * j + 1] = __fadd_rn(__fmul_rn(d, c[j]), __fmul_rn(a, sj));
                }
            } else if (both) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float sj = s[j] * p.sign;
                    o[j] = __fsub_rn(__fmul_rn(x[i][j], c[j]), __fmul_rn(y[i][j], sj));
                    o1[j] = __fadd_rn(__fmul_rn(y[i][j], c[j]), __fmul_rn(x[i][j], sj));
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = x[i][j];
            }
            stream4(dst + c0, count, o);
            if (both) stream4(dst + c1, count, o1);
        }
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
    if (q) positive(h, "n_heads");
    if (k) positive(hkv, "n_kv_heads");
    if ((q ? h : 0) > 32767 || (k ? hkv : 0) > 32767) fail(MMH_ERR_SHAPE, "rotary: at most 32767 heads");
    bounded(table, "table");
    if (width < 2 || (width & 1) || width > hd)
        fail(MMH_ERR_SHAPE, "rotary: width must be even and 2 to " + std::to_string(hd) + ", got " + std::to_string(width));
    const int64_t places = extent(b, t, "positions");
    bounded(places, "positions");
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
    const bool inter = layout == MMH_ROTARY_INTERLEAVED;
    RotaryArgs p;
    p.q = q;
    p.k = k;
    p.cos_t = cos_dev;
    p.sin_t = sin_dev;
    p.q_out = q_out;
    p.k_out = k_out;
    p.positions = host_ids(cx, positions, places, 0);
    p.hd = hd;
    p.half = width / 2;
    p.places = (int32_t)places;
    p.t = (int32_t)t;
    p.h = q ? (int32_t)h : 0;
    const int64_t heads = p.h + (k ? hkv : 0);
    p.heads = (int32_t)heads;
    p.rotated = (int32_t)(((inter ? width : width / 2) + 3) / 4);
    p.units = p.rotated + (int32_t)((hd - width + 3) / 4);
    p.sign = sign;
    const int bits = lane_bits(p.units);
    const int64_t blocks = (places + (256 >> bits) - 1) / (256 >> bits);
    auto launch = [&](auto kernel, int64_t group) {
        constexpr int64_t most = int64_t(1) << 23;  // (a launch has less than 2^32 threads)
        for (int64_t at = 0; at < blocks; at += most) {
            p.first = at * (256 >> bits);
            hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(most, blocks - at), (unsigned)((heads + group - 1) / group)), dim3(256),
                               0, cx.stream, p, bits);
            check_hip(hipGetLastError(), "rotary launch");
        }
    };
    // four heads of a place in a thread, where that leaves four workgroups for each CU
    const bool four = blocks * ((heads + 3) / 4) >= 4 * cx.cu_count;
    if (four && inter) launch(rotary_kernel<4, true>, 4);
    else if (four) launch(rotary_kernel<4, false>, 4);
    else if (inter) launch(rotary_kernel<1, true>, 1);
    else launch(rotary_kernel<1, false>, 1);
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
        const int bits = lane_bits(width / 2);
        // positions of a thread: 32, or as many as leave four workgroups for each CU
        const int64_t step = 256 >> bits, rows = std::max<int64_t>(1, std::min<int64_t>(32, positions / (step * 4 * cx.cu_count)));
        hipLaunchKernelGGL(rotary_tables_kernel, dim3((unsigned)((positions + rows * step - 1) / (rows * step))), dim3(256), 0,
                           cx.stream, p, bits, (int)rows, cos_dev, sin_dev);
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
