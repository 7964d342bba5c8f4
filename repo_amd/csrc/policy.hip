// The log-probabilities of chosen tokens and the clipped policy loss with a KL
// term, from logits, with the logits' gradient.
//
// A row z of logits, the chosen token a, the temperature T:
//   l = z_a / T - log sum_j exp(z_j / T)
// and, with old and reference log-probabilities and an advantage A,
//   r = exp(l - old),  d = ref - l
//   L = -min(r A, clamp(r, 1 - lo, 1 + hi) A) + beta (exp(d) - d - 1)
//   dL/dl = -A r (where the first is the smaller) + beta (1 - exp(d))
//   dL/dz_j = dL/dl (delta_ja - exp(z_j / T) / sum) / T
// The loss is the sum of w L over the rows that the mask leaves.
//
// Exponentials are powers of two: with k = log2(e) / T in fp32 and c = max(z),
// s = sum_j 2^((z_j - c) k).  The difference comes first: z k of a type's lowest value, which
// masks use, has no fp32 value.
// What follows once a row (l, the ratio, the KL term, the slopes) is in fp64: d and
// l - old are differences of numbers of size 10, and exp(d) - d - 1 of a small d
// has no digits left in fp32.  Sums over rows are in fp64 and of a fixed order.
//
// Bound: HBM, the logits read once and the gradient written once.  The loss makes the
// gradient for an incoming one while the row is in registers (a second launch in the
// backward pass finds that one and ends, or makes another's from the logits): a wave holds
// rows up to 8 KB, a workgroup up to 32 KB, and of 512 threads those of 47 to 64 KB.  Rows of 32 to
// 47 KB and above 64 KB are read twice, for the loss those above 160 KB by workgroups of 1024 threads,
// so that the rows in flight stay in the memory-side cache (8192 of 256 KB: 1008 us of 256 threads for
// 890).  Measured: 16x512x32768 bf16, 0.7 of the rows counting, loss
// and gradient 194 us (913 MB at 4.7 TB/s), 8x1024x131072 914 to 966 us (3.65 GB, 3.9 TB/s); scoring
// 16x511x32768 68 us (375 MB, 5.6 TB/s).  Writing past the caches was slower (by 16 and 36 us).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/cubicsplat_hip.h"

namespace {

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };
enum { kToken = 0, kSequence = 1, kSum = 2 };

constexpr int64_t kPlBlocks = 1 << 20;   // workgroups; rows beyond are taken in turns
constexpr double kLn2 = 0.69314718055994530942;

struct PlRows {
    const void* logits;
    const int64_t* tokens;
    const uint8_t* mask;     // NULL: all rows count
    int64_t rows, length, vocab, batch_stride, row_stride;
    float k;                 // log2(e) / temperature
    double inv_t;
};

struct PlLoss {
    const float* advantages;
    const float* old;
    const float* ref;        // NULL: no KL term
    const float* weights;    // of each sequence; NULL: `weight` of all
    float weight;
    int64_t adv_batch_stride, adv_stride;
    double lo, hi, beta, scale;
    float* slopes;           // [rows] dloss/dl
    double* terms;           // [rows][3]: loss, KL, clipped, weighted
};

struct PlOut {
    float* stats;            // [rows][2]: c, s
    float* logprobs;         // [rows]
    void* grad;              // [rows][vocab]
    const float* upstream;   // [rows] (backward)
    const float* factor;     // what the slopes are multiplied with, NULL: 1
    int32_t unless_one;      // nothing is done where *factor is 1
};

template <typename T> struct PlVec { static constexpr int n = 16 / sizeof(T); T v[n]; };

// 16 bytes at any element: rows of an odd vocabulary begin anywhere.
typedef float PlFour __attribute__((ext_vector_type(4)));
typedef PlFour PlAny __attribute__((aligned(2)));

template <typename T>
__device__ inline PlVec<T> pl_get(const T* p) {
    return __builtin_bit_cast(PlVec<T>, (PlFour) * reinterpret_cast<const PlAny*>(p));
}

// Value j of a row that begins at p, the same for a wave: one register an address.
template <typename T>
__device__ inline T* pl_place(T* p, uint32_t j) {
    return (T*)((uintptr_t)p + j * (uint32_t)sizeof(T));
}

template <typename T>
__device__ inline void pl_put(T* p, const PlVec<T>& x) {
    *reinterpret_cast<PlAny*>(p) = __builtin_bit_cast(PlFour, x);
}

struct PlSum { float c, s; };   // sum of 2^((z - c) k), c the largest z

__device__ inline float pl_power(float z, float c, float k) {
    return __builtin_amdgcn_exp2f((z - c) * k);
}

__device__ inline PlSum pl_join(PlSum a, PlSum b, float k) {
    // No value seen yet, or -inf alone: c = -inf and s = 0.
    if (a.s == 0.0f && a.c == -INFINITY) return b;
    if (b.s == 0.0f && b.c == -INFINITY) return a;
    const float c = __builtin_fmaxf(a.c, b.c);
    return {c, a.s * pl_power(a.c, c, k) + b.s * pl_power(b.c, c, k)};
}

// N values more.  While -inf alone has been seen the sum stays empty: a row of it has
// c = -inf at the end, and NaN for a log-probability, as its difference is.
template <int N>
__device__ inline void pl_add(PlSum& a, const float (&z)[N], float k) {
    float most = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) most = __builtin_fmaxf(most, z[i]);
    if (most > a.c) {
        a.s *= pl_power(a.c, most, k);
        a.c = most;
    }
    const float c = a.c == -INFINITY ? 0.0f : a.c;
#pragma unroll
    for (int i = 0; i < N; ++i) a.s += pl_power(z[i], c, k);
}

// The THREADS threads of a row: a wave, or a whole workgroup.
template <int THREADS>
struct PlTeam {
    static constexpr int kRows = THREADS == 64 ? 4 : 1;   // rows of a workgroup
    static constexpr int kBlock = THREADS * kRows;
    struct Lds {
        float c[THREADS / 64], s[THREADS / 64];
        double less;
        float slope;
    };
    Lds* lds;

    __device__ static int rank() { return THREADS > 64 ? threadIdx.x : threadIdx.x & 63; }
    __device__ static int64_t first_row() {   // the same in all lanes of a wave
        if (THREADS > 64) return blockIdx.x;
        return (int64_t)blockIdx.x * kRows + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    }
    __device__ static int64_t step_rows() { return (int64_t)gridDim.x * kRows; }
    __device__ static void sync() {
        if (THREADS > 64) __syncthreads();
    }

    __device__ float most(float x) const {
        for (int m = 1; m < 64; m <<= 1) x = __builtin_fmaxf(x, __shfl_xor(x, m));
        if (THREADS > 64) {
            if ((threadIdx.x & 63) == 0) lds->c[threadIdx.x >> 6] = x;
            __syncthreads();
            x = lds->c[0];
            for (int w = 1; w < THREADS / 64; ++w) x = __builtin_fmaxf(x, lds->c[w]);
        }
        return x;
    }
    __device__ float sum(float x) const {
        for (int m = 1; m < 64; m <<= 1) x += __shfl_xor(x, m);
        if (THREADS > 64) {
            if ((threadIdx.x & 63) == 0) lds->s[threadIdx.x >> 6] = x;
            __syncthreads();
            x = lds->s[0];
            for (int w = 1; w < THREADS / 64; ++w) x += lds->s[w];
        }
        return x;
    }
    __device__ PlSum join(PlSum a, float k) const {
        for (int m = 1; m < 64; m <<= 1)
            a = pl_join(a, {__shfl_xor(a.c, m), __shfl_xor(a.s, m)}, k);
        if (THREADS > 64) {
            if ((threadIdx.x & 63) == 0) {
                lds->c[threadIdx.x >> 6] = a.c;
                lds->s[threadIdx.x >> 6] = a.s;
            }
            __syncthreads();
            a = {lds->c[0], lds->s[0]};
            for (int w = 1; w < THREADS / 64; ++w) a = pl_join(a, {lds->c[w], lds->s[w]}, k);
        }
        return a;
    }
};

template <typename T>
__device__ inline const T* pl_row(const PlRows& a, int64_t r) {
    const int64_t b = r / a.length;
    return (const T*)a.logits + b * a.batch_stride + (r - b * a.length) * a.row_stride;
}

// e^x - 1: x = n ln 2 + r with |r| <= ln 2 / 2, the exponential's series to r^14 / 14! (2^-63 of r),
// then 2^n (e^r - 1) + (2^n - 1).  Within 2^-50 of it, relative; the library's function keeps
// 95 registers beside those that hold a row.  From 709.79 on e^x is beyond fp64: n is at most 1024,
// and half of the sum is taken first, whose terms then are finite, so that its double is infinity.
__device__ inline double pl_expm1(double x) {
    x = x > 710.0 ? 710.0 : x < -800.0 ? -800.0 : x;   // infinity and -1; NaN stays
    const double n = __builtin_rint(x * 1.4426950408889634074);
    // ln 2 as its first 32 bits, which n of 11 bits multiplies exactly, and the rest.
    constexpr double kHead = 2977044471.0 / 4294967296.0;
    double r = __builtin_fma(n, -kHead, x);
    r = __builtin_fma(n, -1.9082149292705877e-10, r);
    double p = 1.0 / 87178291200.0;
    p = __builtin_fma(p, r, 1.0 / 6227020800.0);
    p = __builtin_fma(p, r, 1.0 / 479001600.0);
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p * r, r, r);
    const int e = (int)n - 1;
    return 2.0 * (__builtin_ldexp(p, e) + (__builtin_ldexp(1.0, e) - 0.5));
}

// log s from the hardware's logarithm y (22 bits): log s = y + log(1 + d), d = s e^-y - 1.
__device__ inline double pl_log(float s) {
    const double y = (double)__builtin_amdgcn_logf(s) * kLn2;
    const double m = pl_expm1(-y);
    const double d = __builtin_fma((double)s, m, (double)s) - 1.0;
    return y + __builtin_fma(-0.5 * d, d, d);
}

// l of a row, of whose token `chosen` is the logit (NaN for a token outside the vocabulary).
__device__ inline double pl_logprob(const PlRows& a, float chosen, PlSum sum) {
    const double l = ((double)chosen - (double)sum.c) * a.inv_t - pl_log(sum.s);
    return l > 0.0 ? 0.0 : l;   // s is rounded, a probability is at most 1
}

template <typename T>
__device__ inline float pl_chosen(const PlRows& a, const T* z, int64_t token) {
    return token >= 0 && token < a.vocab ? (float)z[token] : __builtin_nanf("");
}

// What belongs to a row besides its logits, asked for before them.
struct PlRow {
    int64_t token;
    bool counts;
    float chosen, old, ref, adv, weight;

    template <typename T>
    __device__ void get(const PlRows& a, const PlLoss& f, int64_t r, const T* z, bool loss) {
        token = a.tokens[r];
        counts = !a.mask || a.mask[r];
        chosen = old = ref = adv = weight = 0.0f;
        if (!counts) return;
        chosen = pl_chosen(a, z, token);
        if (!loss) return;
        const int64_t b = r / a.length;
        old = f.old[r];
        if (f.ref) ref = f.ref[r];
        adv = f.advantages[b * f.adv_batch_stride + (r - b * a.length) * f.adv_stride];
        weight = f.weights ? f.weights[b] : f.weight;
    }
};

// What a row's gradient slope (delta_ja - p_j) / T is made of: q 2^((z_j - c) k), and `own` at its
// token, 1 - p without the difference.  none: zeros, and nothing of the row is read.
struct PlSlope {
    float q, own, c;
    bool none;
    __device__ PlSlope(const PlRows& a, PlSum sum, float slope, double less)   // less: p - 1
        : q(0.0f), own(0.0f), c(sum.c), none(slope == 0.0f) {
        if (none) return;
        const double by = -(double)slope * a.inv_t;
        q = (float)by / sum.s;
        own = (float)(by * less);
    }
};

template <typename T>
__device__ inline PlVec<T> pl_slopes(const PlVec<T>& x, const PlSlope& g, float k) {
    PlVec<T> y;
#pragma unroll
    for (int i = 0; i < PlVec<T>::n; ++i)
        y.v[i] = (T)(g.q * pl_power((float)x.v[i], g.c, k));
    return y;
}

template <typename T>
__device__ inline T pl_slope_of(float z, const PlSlope& g, float k, bool own) {
    return (T)(own ? g.own
               : g.none ? 0.0f
                        : g.q * pl_power(z, g.c, k));
}

// A row is whole vectors and less than one of single values, which the first threads take.
template <typename T, int THREADS>
struct PlTail {
    int64_t full;
    bool mine;
    __device__ explicit PlTail(int64_t vocab)
        : full(vocab - vocab % PlVec<T>::n),
          mine(PlTeam<THREADS>::rank() < (int)(vocab - full)) {}
    __device__ int64_t at() const { return full + PlTeam<THREADS>::rank(); }
};

// A row's gradient from a second reading.
template <typename T, int THREADS>
__device__ inline void pl_gradient(const PlRows& a, const T* z, T* grad, int64_t token,
                                   const PlSlope& g) {
    constexpr int V = PlVec<T>::n;
    const PlTail<T, THREADS> tail(a.vocab);
    for (int64_t j = (int64_t)PlTeam<THREADS>::rank() * V; j < tail.full; j += THREADS * V) {
        PlVec<T> y{};
        if (!g.none) y = pl_slopes(pl_get(z + j), g, a.k);
        pl_put(grad + j, y);
        // The same thread, in this order: its token's value is written last.
        if (token >= j && token < j + V) grad[token] = (T)g.own;
    }
    if (tail.mine)
        grad[tail.at()] =
            pl_slope_of<T>(g.none ? 0.0f : (float)z[tail.at()], g, a.k, tail.at() == token);
}

// What the loss makes of a row's l: its terms, and dloss/dl; `less`: the token's p - 1.  A wave's
// lanes 0 to 2 compute the exponentials side by side.
__device__ inline float pl_terms(const PlLoss& f, int64_t r, const PlRow& row, double l,
                                 double* less) {
    const int lane = threadIdx.x & 63;
    double* t = f.terms + 3 * r;
    *less = 0.0;
    if (!row.counts) {
        if (lane == 0) t[0] = t[1] = t[2] = 0.0;
        return 0.0f;
    }
    const double d = f.ref ? (double)row.ref - l : 0.0;
    const double e = pl_expm1(lane == 0 ? l - (double)row.old : lane == 1 ? d : l);
    const double ratio = __shfl(e, 0) + 1.0, ed = __shfl(e, 1);
    *less = __shfl(e, 2);
    const double w = (double)row.weight, adv = (double)row.adv;
    const double low = 1.0 - f.lo, high = 1.0 + f.hi;
    const bool clipped = adv >= 0.0 ? ratio > high : adv < 0.0 && ratio < low;
    // min(ratio A, clamp(ratio) A): the clamped where it is the smaller.
    const double gain = adv * (clipped ? (adv >= 0.0 ? high : low) : ratio);
    double slope = clipped ? 0.0 : -adv * ratio, loss = -gain, kl = 0.0;
    if (f.ref) {
        kl = ed - d;
        if (f.beta != 0.0) {
            loss += f.beta * kl;
            slope -= f.beta * ed;
        }
    }
    if (lane == 0) {
        t[0] = w * f.scale * loss;
        t[1] = w * kl;
        t[2] = clipped && adv != 0.0 ? w : 0.0;
    }
    return (float)(w * f.scale * slope);
}

// What follows a row's sum: its first wave writes the statistics and, for the loss, tells the
// others the slope.
template <int THREADS, bool LOSS>
__device__ inline PlSlope pl_row_done(const PlRows& a, const PlLoss& f, const PlOut& o,
                                      const PlTeam<THREADS>& team, int64_t r, const PlRow& row,
                                      PlSum sum) {
    double less = 0.0;
    float slope = 0.0f;
    if (THREADS == 64 || threadIdx.x < 64) {
        const double l = row.counts ? pl_logprob(a, row.chosen, sum) : 0.0;
        if (LOSS) slope = pl_terms(f, r, row, l, &less);
        if ((threadIdx.x & 63) == 0) {
            *(float2*)(o.stats + 2 * r) = make_float2(sum.c, sum.s);
            o.logprobs[r] = (float)l;
            if (LOSS) f.slopes[r] = slope;
            if (LOSS && THREADS > 64) {
                team.lds->less = less;
                team.lds->slope = slope;
            }
        }
    }
    if (LOSS && THREADS > 64 && o.grad) {
        __syncthreads();
        less = team.lds->less;
        slope = team.lds->slope;
    }
    return PlSlope(a, sum, slope, less);
}

// Rows of any length: an online sum, two vectors ahead; with LOSS the gradient from a second
// reading.
template <typename T, int THREADS, bool LOSS>
__global__ __launch_bounds__(PlTeam<THREADS>::kBlock, THREADS == 1024 ? 8 : 4) void k_rows(
    PlRows a, PlLoss f, PlOut o) {
    constexpr int V = PlVec<T>::n, U = 2;
    __shared__ typename PlTeam<THREADS>::Lds lds;
    const PlTeam<THREADS> team{&lds};
    for (int64_t r = team.first_row(); r < a.rows; r += team.step_rows()) {
        const T* z = pl_row<T>(a, r);
        PlRow row;
        row.get(a, f, r, z, LOSS);
        PlSum sum{-INFINITY, 0.0f};
        if (row.counts) {
            const PlTail<T, THREADS> tail(a.vocab);
            int64_t j = (int64_t)team.rank() * V;
            for (; j + (U - 1) * THREADS * V < tail.full; j += U * THREADS * V) {
                PlVec<T> x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = pl_get(z + j + u * THREADS * V);
                float v[U * V];
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int i = 0; i < V; ++i) v[u * V + i] = (float)x[u].v[i];
                pl_add(sum, v, a.k);
            }
            for (; j < tail.full; j += THREADS * V) {
                const PlVec<T> x = pl_get(z + j);
                float v[V];
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = (float)x.v[i];
                pl_add(sum, v, a.k);
            }
            if (tail.mine) {
                const float v[1] = {(float)z[tail.at()]};
                pl_add(sum, v, a.k);
            }
            sum = team.join(sum, a.k);
        }
        const PlSlope g = pl_row_done<THREADS, LOSS>(a, f, o, team, r, row, sum);
        if (LOSS && o.grad) pl_gradient<T, THREADS>(a, z, (T*)o.grad + r * a.vocab, row.token, g);
        team.sync();   // the next row's sums use the same places
    }
}

// A vector's values as they lie, not as floats that an earlier pass made of them, and only once the
// vector before is done with: otherwise the compiler keeps floats of many vectors at once.
template <typename T>
__device__ inline PlVec<T> pl_anew(PlFour& x) {
    __builtin_amdgcn_sched_barrier(0);
    __asm__ volatile("" : "+v"(x));
    return __builtin_bit_cast(PlVec<T>, x);
}

// Rows that the registers of their threads hold, N vectors each: read once.
template <typename T, int THREADS, int N, bool LOSS>
__global__ __launch_bounds__(PlTeam<THREADS>::kBlock, 4) void k_rows_held(PlRows a, PlLoss f, PlOut o) {
    constexpr int V = PlVec<T>::n;
    __shared__ typename PlTeam<THREADS>::Lds lds;
    const PlTeam<THREADS> team{&lds};
    const PlTail<T, THREADS> tail(a.vocab);
    const uint32_t full = (uint32_t)tail.full;
    for (int64_t r = team.first_row(); r < a.rows; r += team.step_rows()) {
        const T* z = pl_row<T>(a, r);
        PlRow row;
        row.get(a, f, r, z, LOSS);
        const int64_t token = row.token;
        PlSum sum{-INFINITY, 0.0f};
        // Places anew in each row and pass: the compiler would keep all of them from the first on.
        uint32_t at = team.rank() * V;
        __asm__ volatile("" : "+v"(at));
        // As they lie: registers hold a row's 16-bit values, not floats, from pass to pass.
        PlFour x[N];
        float last = -INFINITY;
        if (row.counts) {
            PlVec<T> nothing;
#pragma unroll
            for (int i = 0; i < V; ++i) nothing.v[i] = (T)-INFINITY;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const uint32_t j = at + n * THREADS * V;
                x[n] = __builtin_bit_cast(PlFour, nothing);
                if (j < full) x[n] = __builtin_bit_cast(PlFour, pl_get(pl_place(z, j)));
            }
            if (tail.mine) last = (float)z[tail.at()];
            float most = last;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const PlVec<T> v = pl_anew<T>(x[n]);
#pragma unroll
                for (int i = 0; i < V; ++i) most = __builtin_fmaxf(most, (float)v.v[i]);
            }
            sum.c = team.most(most);
            const float c = sum.c == -INFINITY ? 0.0f : sum.c;
            sum.s = pl_power(last, c, a.k);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const PlVec<T> v = pl_anew<T>(x[n]);
#pragma unroll
                for (int i = 0; i < V; ++i)
                    sum.s += pl_power((float)v.v[i], c, a.k);
            }
            sum.s = team.sum(sum.s);
        }
        const PlSlope g = pl_row_done<THREADS, LOSS>(a, f, o, team, r, row, sum);
        if (!LOSS || !o.grad) {
            team.sync();   // the next row's sums use the same places
            continue;
        }
        T* grad = (T*)o.grad + r * a.vocab;
        __asm__ volatile("" : "+v"(at));
        const uint32_t own = token >= 0 && token < full ? (uint32_t)token : ~0u;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const uint32_t j = at + n * THREADS * V;
            if (j >= full) continue;
            PlVec<T> y{};
            if (!g.none) y = pl_slopes(pl_anew<T>(x[n]), g, a.k);
            pl_put(pl_place(grad, j), y);
            // The same thread, in this order: its token's value is written last.
            if (own - j < V) grad[own] = (T)g.own;
        }
        if (tail.mine) grad[tail.at()] = pl_slope_of<T>(last, g, a.k, tail.at() == token);
        team.sync();   // the next row's sums use the same places
    }
}

template <typename T, int THREADS>
__global__ __launch_bounds__(PlTeam<THREADS>::kBlock) void k_gradient(PlRows a, PlOut o) {
    const float factor = o.factor ? *o.factor : 1.0f;
    if (o.unless_one && factor == 1.0f) return;
    typedef PlTeam<THREADS> Team;
    for (int64_t r = Team::first_row(); r < a.rows; r += Team::step_rows()) {
        const T* z = pl_row<T>(a, r);
        float slope = !a.mask || a.mask[r] ? o.upstream[r] * factor : 0.0f;
        const PlSum sum{o.stats[2 * r], o.stats[2 * r + 1]};
        const int64_t token = a.tokens[r];
        const double l = slope == 0.0f ? 0.0 : pl_logprob(a, pl_chosen(a, z, token), sum);
        if (token < 0 || token >= a.vocab) slope *= (float)l;   // NaN, unless nothing comes in
        const PlSlope g(a, sum, slope, slope == 0.0f ? 0.0 : pl_expm1(l));
        pl_gradient<T, THREADS>(a, z, (T*)o.grad + r * a.vocab, token, g);
    }
}

// The weight of a row of each sequence: 1, 1 / (rows that count), or 1 / (rows of the
// sequence that count) / (sequences with such rows).  One workgroup: a wave takes a sequence, or
// a thread one of less than a wave's rows.
constexpr int kPlWide = 1024;

__host__ __device__ inline double pl_weight(int reduction, int64_t mine, int64_t total) {
    const double all = (double)(total > 0 ? total : 1);
    if (reduction == kToken) return 1.0 / all;
    if (reduction == kSequence) return mine ? 1.0 / ((double)mine * all) : 0.0;
    return 1.0;
}

// How many of 16 bytes, or of the last of a sequence's, are not zero.
__device__ inline int pl_count(const uint8_t* p, int64_t left) {
    typedef uint32_t Four __attribute__((ext_vector_type(4)));
    typedef Four Any __attribute__((aligned(1)));
    int n = 0;
    if (left >= 16) {
        const Four x = *reinterpret_cast<const Any*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            n += __popc((((x[i] & 0x7F7F7F7Fu) + 0x7F7F7F7Fu) | x[i]) & 0x80808080u);
    } else {
        for (int i = 0; i < (int)left; ++i) n += p[i] != 0;
    }
    return n;
}

__global__ __launch_bounds__(kPlWide) void k_weights(const uint8_t* mask, int64_t batch,
                                                     int64_t length, int reduction, float* weights) {
    __shared__ int64_t lds[kPlWide / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // Counts go to `weights` as whole numbers below 2^32 first (bits, not values).
    uint32_t* count_of = (uint32_t*)weights;
    int64_t total = 0;
    if (length >= 64) {
        for (int64_t b = wave; b < batch; b += kPlWide / 64) {
            int64_t n = 0;
            for (int64_t t = lane * 16; t < length; t += 1024)
                n += pl_count(mask + b * length + t, length - t);
            for (int m = 1; m < 64; m <<= 1) n += __shfl_xor(n, m);
            if (lane == 0) {
                count_of[b] = (uint32_t)n;
                total += reduction == kSequence ? n != 0 : n;
            }
        }
    } else {
        for (int64_t b = threadIdx.x; b < batch; b += kPlWide) {
            int64_t n = 0;
            for (int64_t t = 0; t < length; t += 16)
                n += pl_count(mask + b * length + t, length - t);
            count_of[b] = (uint32_t)n;
            total += reduction == kSequence ? n != 0 : n;
        }
    }
    for (int m = 1; m < 64; m <<= 1) total += __shfl_xor(total, m);
    if (lane == 0) lds[wave] = total;
    __syncthreads();   // the counts are written too
    total = 0;
    for (int w = 0; w < kPlWide / 64; ++w) total += lds[w];
    for (int64_t b = threadIdx.x; b < batch; b += kPlWide)
        weights[b] = (float)pl_weight(reduction, count_of[b], total);
}

__global__ __launch_bounds__(kPlWide) void k_sum(const double* terms, int64_t rows, float* out) {
    __shared__ double lds[kPlWide / 64][3];
    double t[3] = {0.0, 0.0, 0.0};
    int64_t r = threadIdx.x;
    for (; r + 3 * kPlWide < rows; r += 4 * kPlWide) {
        double v[4][3];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 3; ++i) v[u][i] = terms[3 * (r + u * kPlWide) + i];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 3; ++i) t[i] += v[u][i];
    }
    for (; r < rows; r += kPlWide)
#pragma unroll
        for (int i = 0; i < 3; ++i) t[i] += terms[3 * r + i];
    for (int i = 0; i < 3; ++i)
        for (int m = 1; m < 64; m <<= 1) t[i] += __shfl_xor(t[i], m);
    if ((threadIdx.x & 63) == 0)
        for (int i = 0; i < 3; ++i) lds[threadIdx.x >> 6][i] = t[i];
    __syncthreads();
    if (threadIdx.x < 3) {
        double all = 0.0;
        for (int w = 0; w < kPlWide / 64; ++w) all += lds[w][threadIdx.x];
        out[threadIdx.x] = (float)all;
    }
}

bool pl_rows(PlRows* a, const void* logits, int64_t batch, int64_t length, int64_t vocab,
             int64_t batch_stride, int64_t row_stride, int32_t dtype, const int64_t* tokens,
             const uint8_t* mask, double temperature) {
    const int64_t most = (int64_t)1 << 44;
    if (!logits || !tokens || dtype < kF32 || dtype > kF16 || !(temperature > 0.0) || batch < 1 ||
        length < 1 || vocab < 1 || vocab > most || batch > most / length ||
        batch * length > most / vocab || length > 0xFFFFFFFFll || batch_stride < 0 ||
        row_stride < 0)
        return false;
    const double k = 1.4426950408889634074 / temperature;
    if (!(k > 1e-30 && k < 1e30)) return false;
    *a = PlRows{logits, tokens, mask, batch * length, length, vocab, batch_stride, row_stride,
                (float)k, (double)(float)k * kLn2};
    return true;
}

template <int THREADS>
dim3 pl_grid(const PlRows& a) {
    const int64_t blocks = (a.rows + PlTeam<THREADS>::kRows - 1) / PlTeam<THREADS>::kRows;
    return dim3((unsigned)(blocks < kPlBlocks ? blocks : kPlBlocks));
}

template <typename T, bool LOSS, int THREADS, int N>
bool pl_rows_held(const PlRows& a, const PlLoss& f, const PlOut& o, hipStream_t stream) {
    if (a.vocab / PlVec<T>::n > THREADS * N) return false;
    hipLaunchKernelGGL((k_rows_held<T, THREADS, N, LOSS>), pl_grid<THREADS>(a),
                       dim3(PlTeam<THREADS>::kBlock), 0, stream, a, f, o);
    return true;
}

template <typename T, bool LOSS, int THREADS>
void pl_rows_twice(const PlRows& a, const PlLoss& f, const PlOut& o, hipStream_t stream) {
    hipLaunchKernelGGL((k_rows<T, THREADS, LOSS>), pl_grid<THREADS>(a), dim3(THREADS), 0, stream, a,
                       f, o);
}

// The fewest threads that hold a row, as what a row costs besides its values (its arithmetic, the
// workgroup's barriers) is theirs: bf16, 32768 rows of 4096, loss / scoring, us: a wave 107 / 40, 128
// threads 106 / 41, 256 131 / 55, 512 by the longer rows' kernel 244 / 168.  Two to four thousand
// vectors, 10920 rows of 24576: 512 threads that hold them 199 / 96, 256 that read twice 201 / 92
// (13416 of 20000: 223 / 113, 207 / 93; 8192 of 32768: 186 / 86, 197 / 93).  Longer rows, 5456 of
// 49152: 512 threads that read twice 196 / 94, 1024 227 / 127, 1024 that hold them 237 / 162; 1336 of
// 200000: 512 229 / 102, 1024 223 / 103.
template <typename T, bool LOSS>
void pl_run_rows(const PlRows& a, const PlLoss& f, const PlOut& o, hipStream_t stream) {
    const int64_t vectors = a.vocab / PlVec<T>::n;
    if (pl_rows_held<T, LOSS, 64, 1>(a, f, o, stream) ||
        pl_rows_held<T, LOSS, 64, 2>(a, f, o, stream) ||
        pl_rows_held<T, LOSS, 64, 4>(a, f, o, stream) ||
        pl_rows_held<T, LOSS, 64, 8>(a, f, o, stream) ||
        pl_rows_held<T, LOSS, 128, 8>(a, f, o, stream) ||
        pl_rows_held<T, LOSS, 256, 8>(a, f, o, stream))
        return;
    if (vectors <= 3000) pl_rows_twice<T, LOSS, 256>(a, f, o, stream);
    else if (pl_rows_held<T, LOSS, 512, 8>(a, f, o, stream)) return;
    else if (!LOSS || vectors <= 10240) pl_rows_twice<T, LOSS, 512>(a, f, o, stream);
    else pl_rows_twice<T, LOSS, 1024>(a, f, o, stream);
}

template <typename T, int THREADS>
void pl_gradient_by(const PlRows& a, const PlOut& o, hipStream_t stream) {
    dim3 grid = pl_grid<THREADS>(a);
    // As many as are resident where the factor most likely is one: none of them does anything then.
    constexpr unsigned kMost = 2048 * 256 / PlTeam<THREADS>::kBlock;
    if (o.unless_one && grid.x > kMost) grid.x = kMost;
    hipLaunchKernelGGL((k_gradient<T, THREADS>), grid, dim3(PlTeam<THREADS>::kBlock), 0, stream, a,
                       o);
}

// Measured, 64 / 256 / 512 / 1024 threads, us: bf16, 65536 rows of 2048 95 / 152 / 276 / 635; 16384
// of 8192 106 / 97 / 118 / 206; 8192 of 32768 246 / 202 / 194 / 214; 2048 of 131072 260 / 235 / 212 / 204.
template <typename T>
void pl_run_gradient(const PlRows& a, const PlOut& o, hipStream_t stream) {
    const int64_t vectors = a.vocab / PlVec<T>::n;
    if (vectors <= 512) pl_gradient_by<T, 64>(a, o, stream);
    else if (vectors < 2048) pl_gradient_by<T, 256>(a, o, stream);
    else if (vectors < 8192) pl_gradient_by<T, 512>(a, o, stream);
    else pl_gradient_by<T, 1024>(a, o, stream);
}

}  // namespace

extern "C" size_t cs_policy_loss_workspace_elems(int64_t batch, int64_t length) {
    if (batch < 1 || length < 1 || batch > ((int64_t)1 << 44) / length) return 0;
    return (size_t)(6 * batch * length + batch);
}

extern "C" int cs_token_logprobs_forward(const void* logits, int64_t batch, int64_t length,
                                         int64_t vocab, int64_t batch_stride, int64_t row_stride,
                                         int32_t dtype, const int64_t* tokens, const uint8_t* mask,
                                         double temperature, float* stats, float* logprobs,
                                         hipStream_t stream) {
    PlRows a;
    if (!pl_rows(&a, logits, batch, length, vocab, batch_stride, row_stride, dtype, tokens, mask,
                 temperature) ||
        !stats || !logprobs)
        return CS_ERR_ARGS;
    PlOut o{};
    o.stats = stats;
    o.logprobs = logprobs;
    if (dtype == kF32) pl_run_rows<float, false>(a, PlLoss{}, o, stream);
    else if (dtype == kBF16) pl_run_rows<__bf16, false>(a, PlLoss{}, o, stream);
    else pl_run_rows<_Float16, false>(a, PlLoss{}, o, stream);
    return hipGetLastError() == hipSuccess ? CS_OK : CS_ERR_HIP;
}

extern "C" int cs_token_logprobs_backward(const void* logits, int64_t batch, int64_t length,
                                          int64_t vocab, int64_t batch_stride, int64_t row_stride,
                                          int32_t dtype, const int64_t* tokens,
                                          const uint8_t* mask, double temperature,
                                          const float* stats, const float* upstream,
                                          const float* factor, int32_t unless_one, void* grad,
                                          hipStream_t stream) {
    PlRows a;
    if (!pl_rows(&a, logits, batch, length, vocab, batch_stride, row_stride, dtype, tokens, mask,
                 temperature) ||
        !stats || !upstream || !grad || (unless_one && !factor))
        return CS_ERR_ARGS;
    PlOut o{};
    o.stats = const_cast<float*>(stats);
    o.grad = grad;
    o.upstream = upstream;
    o.factor = factor;
    o.unless_one = unless_one;
    if (dtype == kF32) pl_run_gradient<float>(a, o, stream);
    else if (dtype == kBF16) pl_run_gradient<__bf16>(a, o, stream);
    else pl_run_gradient<_Float16>(a, o, stream);
    return hipGetLastError() == hipSuccess ? CS_OK : CS_ERR_HIP;
}

extern "C" int cs_policy_loss(const void* logits, int64_t batch, int64_t length, int64_t vocab,
                              int64_t batch_stride, int64_t row_stride, int32_t dtype,
                              const int64_t* tokens, const uint8_t* mask, double temperature,
                              const float* advantages, int64_t adv_batch_stride,
                              int64_t adv_stride, const float* old_logprobs,
                              const float* ref_logprobs, double clip_low, double clip_high,
                              double kl_weight, int32_t reduction, double scale, float* workspace,
                              float* stats, float* slopes, float* logprobs, float* out, void* grad,
                              hipStream_t stream) {
    PlRows a;
    if (!pl_rows(&a, logits, batch, length, vocab, batch_stride, row_stride, dtype, tokens, mask,
                 temperature) ||
        !advantages || adv_batch_stride < 0 || adv_stride < 0 || !old_logprobs ||
        !(clip_low >= 0.0) || !(clip_high >= 0.0) || !(kl_weight >= 0.0) || reduction < kToken ||
        reduction > kSum || !workspace || ((uintptr_t)workspace & 7) || !stats || !slopes ||
        !logprobs || !out)
        return CS_ERR_ARGS;
    double* terms = (double*)workspace;
    float* weights = workspace + 6 * a.rows;
    if (mask)
        hipLaunchKernelGGL(k_weights, dim3(1), dim3(kPlWide), 0, stream, mask, batch, length,
                           reduction, weights);
    const float weight =
        (float)pl_weight(reduction, length, reduction == kSequence ? batch : a.rows);
    const PlLoss f{advantages, old_logprobs, ref_logprobs, mask ? weights : nullptr, weight,
                   adv_batch_stride, adv_stride, clip_low, clip_high, kl_weight, scale, slopes,
                   terms};
    PlOut o{};
    o.stats = stats;
    o.logprobs = logprobs;
    o.grad = grad;
    if (dtype == kF32) pl_run_rows<float, true>(a, f, o, stream);
    else if (dtype == kBF16) pl_run_rows<__bf16, true>(a, f, o, stream);
    else pl_run_rows<_Float16, true>(a, f, o, stream);
    hipLaunchKernelGGL(k_sum, dim3(1), dim3(kPlWide), 0, stream, terms, a.rows, out);
    return hipGetLastError() == hipSuccess ? CS_OK : CS_ERR_HIP;
}
