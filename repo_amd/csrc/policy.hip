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
// Exponentials are powers of two: with k = log2(e) / T and c = max(z) k, both
// rounded to fp32, s = sum_j 2^(z_j k - c), each difference one fused operation.
// What follows once a row (l, the ratio, the KL term, the slopes) is in fp64: d and
// l - old are differences of numbers of size 10, and exp(d) - d - 1 of a small d
// has no digits left in fp32.  Sums over rows are in fp64 and of a fixed order.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/cubicsplat_hip.h"

namespace {

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };
enum { kToken = 0, kSequence = 1, kSum = 2 };

constexpr int kPlThreads = 256;
constexpr int64_t kPlBlocks = 1 << 20;   // rows beyond are taken in turns
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
    const float* weights;    // of each sequence
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

template <typename T>
__device__ inline void pl_put(T* p, const PlVec<T>& x) {
    *reinterpret_cast<PlAny*>(p) = __builtin_bit_cast(PlFour, x);
}

struct PlSum { float c, s; };   // sum of 2^(z k - c), c the largest z k

__device__ inline PlSum pl_join(PlSum a, PlSum b) {
    // No value seen yet: c = -inf and s = 0.
    if (a.s == 0.0f && a.c == -INFINITY) return b;
    if (b.s == 0.0f && b.c == -INFINITY) return a;
    const float c = __builtin_fmaxf(a.c, b.c);
    return {c, a.s * __builtin_amdgcn_exp2f(a.c - c) + b.s * __builtin_amdgcn_exp2f(b.c - c)};
}

// N values more.  While -inf alone has been seen the sum stays empty: a row of it has
// c = -inf at the end, and NaN for a log-probability, as its difference is.
template <int N>
__device__ inline void pl_add(PlSum& a, const float (&z)[N], float k) {
    float most = z[0];
#pragma unroll
    for (int i = 1; i < N; ++i) most = __builtin_fmaxf(most, z[i]);
    most *= k;
    if (most > a.c) {
        a.s *= __builtin_amdgcn_exp2f(a.c - most);
        a.c = most;
    }
    const float c = a.c == -INFINITY ? 0.0f : a.c;
#pragma unroll
    for (int i = 0; i < N; ++i) a.s += __builtin_amdgcn_exp2f(__builtin_fmaf(z[i], k, -c));
}

__device__ inline PlSum pl_join_block(PlSum a, PlSum* lds) {
    for (int m = 1; m < 64; m <<= 1)
        a = pl_join(a, {__shfl_xor(a.c, m), __shfl_xor(a.s, m)});
    const int wave = threadIdx.x >> 6;
    __syncthreads();   // the last row's is read
    if ((threadIdx.x & 63) == 0) lds[wave] = a;
    __syncthreads();
    a = lds[0];
    for (int w = 1; w < kPlThreads / 64; ++w) a = pl_join(a, lds[w]);
    return a;
}

template <typename T>
__device__ inline const T* pl_row(const PlRows& a, int64_t r) {
    const int64_t b = r / a.length;
    return (const T*)a.logits + b * a.batch_stride + (r - b * a.length) * a.row_stride;
}

// l of a row; NaN where the token is none of the vocabulary.
template <typename T>
__device__ inline double pl_logprob(const PlRows& a, const T* z, int64_t token, PlSum sum) {
    if (token < 0 || token >= a.vocab) return __builtin_nan("");
    const double l = ((double)(float)z[token] * (double)a.k - (double)sum.c) * kLn2 -
                     log((double)sum.s);
    return l > 0.0 ? 0.0 : l;   // s is rounded, a probability is at most 1
}

// slope (delta_ja - p_j) / T over a row; l: its chosen token's log-probability.
template <typename T>
__device__ inline void pl_gradient(const PlRows& a, const T* z, T* grad, int64_t token, PlSum sum,
                                   float slope, double l) {
    constexpr int V = PlVec<T>::n;
    const bool none = slope == 0.0f;   // masked or clipped: nothing of the row is read
    const float q = none ? 0.0f : (float)(-(double)slope * a.inv_t) / sum.s;
    // 1 - p of the chosen token without the difference.
    const float own = none ? 0.0f : (float)(-(double)slope * a.inv_t * expm1(l));
    for (int64_t j = (int64_t)threadIdx.x * V; j < a.vocab; j += (int64_t)blockDim.x * V) {
        PlVec<T> y;
        if (j + V <= a.vocab) {
            if (none) {
                for (int i = 0; i < V; ++i) y.v[i] = (T)0.0f;
            } else {
                const PlVec<T> x = pl_get(z + j);
                for (int i = 0; i < V; ++i) {
                    float g = q * __builtin_amdgcn_exp2f(__builtin_fmaf((float)x.v[i], a.k, -sum.c));
                    y.v[i] = (T)(j + i == token ? own : g);
                }
            }
            pl_put(grad + j, y);
        } else {
            for (int64_t i = j; i < a.vocab; ++i) {
                const float g = none ? 0.0f : q * __builtin_amdgcn_exp2f(
                                                      __builtin_fmaf((float)z[i], a.k, -sum.c));
                grad[i] = (T)(i == token ? own : g);
            }
        }
    }
}

// What the loss makes of a row's l: its terms, and dloss/dl.
__device__ inline float pl_terms(const PlLoss& f, int64_t r, int64_t length, double l, bool counts) {
    double* t = f.terms + 3 * r;
    if (!counts) {
        t[0] = t[1] = t[2] = 0.0;
        return 0.0f;
    }
    const int64_t b = r / length;
    const double w = (double)f.weights[b];
    const double adv = (double)f.advantages[b * f.adv_batch_stride + (r - b * length) * f.adv_stride];
    const double ratio = exp(l - (double)f.old[r]);
    const double low = 1.0 - f.lo, high = 1.0 + f.hi;
    const bool clipped = adv >= 0.0 ? ratio > high : adv < 0.0 && ratio < low;
    // min(ratio A, clamp(ratio) A): the clamped where it is the smaller.
    const double gain = adv * (clipped ? (adv >= 0.0 ? high : low) : ratio);
    double slope = clipped ? 0.0 : -adv * ratio, loss = -gain, kl = 0.0;
    if (f.ref) {
        const double d = (double)f.ref[r] - l, e = expm1(d);
        kl = e - d;
        if (f.beta != 0.0) {
            loss += f.beta * kl;
            slope -= f.beta * e;
        }
    }
    t[0] = w * f.scale * loss;
    t[1] = w * kl;
    t[2] = clipped && adv != 0.0 ? w : 0.0;
    return (float)(w * f.scale * slope);
}

template <typename T, bool LOSS>
__global__ __launch_bounds__(kPlThreads) void k_rows(PlRows a, PlLoss f, PlOut o) {
    constexpr int V = PlVec<T>::n;
    __shared__ PlSum lds[kPlThreads / 64];
    __shared__ float slope_of;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const bool counts = !a.mask || a.mask[r];
        const T* z = pl_row<T>(a, r);
        PlSum sum{-INFINITY, 0.0f};
        double l = 0.0;
        const int64_t token = a.tokens[r];
        if (counts) {
            for (int64_t j = (int64_t)threadIdx.x * V; j < a.vocab; j += kPlThreads * V) {
                if (j + V <= a.vocab) {
                    const PlVec<T> x = pl_get(z + j);
                    float v[V];
                    for (int i = 0; i < V; ++i) v[i] = (float)x.v[i];
                    pl_add(sum, v, a.k);
                } else {
                    for (int64_t i = j; i < a.vocab; ++i) {
                        const float v[1] = {(float)z[i]};
                        pl_add(sum, v, a.k);
                    }
                }
            }
            sum = pl_join_block(sum, lds);
            l = pl_logprob(a, z, token, sum);
        }
        if (threadIdx.x == 0) {
            o.stats[2 * r] = sum.c;
            o.stats[2 * r + 1] = sum.s;
            o.logprobs[r] = (float)l;
            if (LOSS) f.slopes[r] = slope_of = pl_terms(f, r, a.length, l, counts);
        }
        if (LOSS && o.grad) {
            __syncthreads();
            const float slope = slope_of;
            pl_gradient(a, z, (T*)o.grad + r * a.vocab, token, sum, slope, l);
            __syncthreads();
        }
    }
}

template <typename T>
__global__ __launch_bounds__(kPlThreads) void k_gradient(PlRows a, PlOut o) {
    const float factor = o.factor ? *o.factor : 1.0f;
    if (o.unless_one && factor == 1.0f) return;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* z = pl_row<T>(a, r);
        float slope = !a.mask || a.mask[r] ? o.upstream[r] * factor : 0.0f;
        const PlSum sum{o.stats[2 * r], o.stats[2 * r + 1]};
        const int64_t token = a.tokens[r];
        const double l = slope == 0.0f ? 0.0 : pl_logprob(a, z, token, sum);
        if (token < 0 || token >= a.vocab) slope *= (float)l;   // NaN, unless nothing comes in
        pl_gradient(a, z, (T*)o.grad + r * a.vocab, token, sum, slope, l);
    }
}

// The weight of a row of each sequence: 1, 1 / (rows that count), or 1 / (rows of the
// sequence that count) / (sequences with such rows).
constexpr int kPlWide = 1024;

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
            for (int64_t t = lane; t < length; t += 64) n += mask ? mask[b * length + t] != 0 : 1;
            for (int m = 1; m < 64; m <<= 1) n += __shfl_xor(n, m);
            if (lane == 0) {
                count_of[b] = (uint32_t)n;
                total += reduction == kSequence ? n != 0 : n;
            }
        }
    } else {
        for (int64_t b = threadIdx.x; b < batch; b += kPlWide) {
            int64_t n = 0;
            for (int64_t t = 0; t < length; ++t) n += mask ? mask[b * length + t] != 0 : 1;
            count_of[b] = (uint32_t)n;
            total += reduction == kSequence ? n != 0 : n;
        }
    }
    for (int m = 1; m < 64; m <<= 1) total += __shfl_xor(total, m);
    if (lane == 0) lds[wave] = total;
    __syncthreads();   // the counts are written too
    total = 0;
    for (int w = 0; w < kPlWide / 64; ++w) total += lds[w];
    for (int64_t b = threadIdx.x; b < batch; b += kPlWide) {
        const uint32_t n = count_of[b];
        double w = 1.0;
        if (reduction == kToken) w = 1.0 / (double)(total > 0 ? total : 1);
        if (reduction == kSequence)
            w = n ? 1.0 / ((double)n * (double)(total > 0 ? total : 1)) : 0.0;
        weights[b] = (float)w;
    }
}

__global__ __launch_bounds__(kPlWide) void k_sum(const double* terms, int64_t rows, float* out) {
    __shared__ double lds[kPlWide / 64][3];
    double t[3] = {0.0, 0.0, 0.0};
    for (int64_t r = threadIdx.x; r < rows; r += kPlWide)
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

unsigned pl_grid(int64_t rows) { return (unsigned)(rows < kPlBlocks ? rows : kPlBlocks); }

template <bool LOSS>
void pl_run_rows(const PlRows& a, const PlLoss& f, const PlOut& o, int dtype, hipStream_t stream) {
    const dim3 grid(pl_grid(a.rows)), block(kPlThreads);
    if (dtype == kF32)
        hipLaunchKernelGGL((k_rows<float, LOSS>), grid, block, 0, stream, a, f, o);
    else if (dtype == kBF16)
        hipLaunchKernelGGL((k_rows<__bf16, LOSS>), grid, block, 0, stream, a, f, o);
    else
        hipLaunchKernelGGL((k_rows<_Float16, LOSS>), grid, block, 0, stream, a, f, o);
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
    pl_run_rows<false>(a, PlLoss{}, o, dtype, stream);
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
    const dim3 grid(pl_grid(a.rows)), block(kPlThreads);
    if (dtype == kF32)
        hipLaunchKernelGGL((k_gradient<float>), grid, block, 0, stream, a, o);
    else if (dtype == kBF16)
        hipLaunchKernelGGL((k_gradient<__bf16>), grid, block, 0, stream, a, o);
    else
        hipLaunchKernelGGL((k_gradient<_Float16>), grid, block, 0, stream, a, o);
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
    hipLaunchKernelGGL(k_weights, dim3(1), dim3(kPlWide), 0, stream, mask, batch, length,
                       reduction, weights);
    const PlLoss f{advantages, old_logprobs, ref_logprobs, weights, adv_batch_stride, adv_stride,
                   clip_low, clip_high, kl_weight, scale, slopes, terms};
    PlOut o{};
    o.stats = stats;
    o.logprobs = logprobs;
    o.grad = grad;
    pl_run_rows<true>(a, f, o, dtype, stream);
    hipLaunchKernelGGL(k_sum, dim3(1), dim3(kPlWide), 0, stream, terms, a.rows, out);
    return hipGetLastError() == hipSuccess ? CS_OK : CS_ERR_HIP;
}
