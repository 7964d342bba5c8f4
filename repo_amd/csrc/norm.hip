// Group norm with an activation over channels-last images, and its gradient.
//
// x is [N, S, C] (S the spatial positions of a sample), a group g the channels
// [g D, (g + 1) D) of one sample, M = D S values:
//   mean = E[x], r = 1 / sqrt(E[(x - mean)^2] + eps), xh = (x - mean) r,
//   z = xh w_c + b_c, y = act(z)
//   dz = dy act'(z), db_c = sum dz, dw_c = sum dz xh,
//   dx = r (w dz - E[w dz] - xh E[w dz xh])
// Everything is computed in fp32 and rounded once on storing.
//
// Two launches a direction: one sums, one applies.  A workgroup takes a slice of
// channels (whole groups, up to 256 vectors of 16 bytes wide; a group that is wider
// is cut into parts) over a chunk of rows (spatial positions); a thread keeps the
// same vector of channels over all of its rows, so what depends on the channel
// stays in its registers.  The sums of a chunk are written out, and each workgroup
// of the second launch joins the ones that it needs, or a small launch in between
// joins them once where they are many; always in a fixed order, without atomics.
// Small samples take one launch (below).
//
// Bound: HBM.  x (and dy) have to be read twice, as a group's statistics need all
// of it; what the second reading costs depends on how much the memory-side cache
// still holds.  An element costs 12 to 20 VALU slots (two of them transcendental, at
// a quarter of the rate), near what the bf16 rate leaves: bytes per element times
// the loads in flight decide, so loads go out four rows ahead.
//
// The variance is not formed from a sum of squares: each thread sums x and x^2
// relative to its first value per channel, and (count, mean, sum of squared
// deviations) are what is joined, so a mean far from zero costs nothing.
//
// Times at the kernels are means of a kernel trace; pairs that a rule is chosen by are
// whole passes, both sides in turn.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/cubicsplat_hip.h"

namespace cs {

constexpr int kGnThreads = 256;
constexpr int kGnMaxVec = 8;

enum { kGnF32 = 0, kGnBF16 = 1, kGnF16 = 2 };
enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

struct GnShape {
    int64_t s;             // rows of a sample
    int32_t c, groups, d;  // d = c / groups
    int32_t gs;            // groups of a slice (1 where a group has several parts)
    int32_t parts;         // slices of a group
    int32_t cs;            // channels of a slice (the last may have fewer)
    int32_t slices;
    int32_t chunks;        // of a sample, in the summing launch
    int64_t rows;          // of such a chunk
    int32_t apply_chunks;
    int64_t apply_rows;
};

struct GnArgs {
    GnShape h;
    const void* x;
    const void* dy;
    const void* weight;
    const void* bias;
    int32_t wdtype;
    float eps;
    float* partials;   // [n][chunk][group][part][2]
    float* channels;   // backward: [n][chunk][channel][2]
    float* mean;
    float* rstd;
    void* out;         // y or dx
    void* dweight;
    void* dbias;
    int32_t n;
    int32_t channel_blocks;  // of the backward's second (or third) launch, for dw and db
    int32_t joined;          // a launch in between has joined the sums
    float* groups_out;       // backward, joined: [n][group] E[w dz], E[w dz xh]
    int32_t act;             // of the one-launch kernels
    int32_t past;            // 1: the second launch stores past the caches, 2: it reads so too
};

template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) GnVec { T v[V]; };

template <int V, typename T>
__device__ inline GnVec<T, V> gn_raw(const T* p) {
    return *reinterpret_cast<const GnVec<T, V>*>(p);
}

// The same past the caches, for what is not read again.
typedef float GnFour __attribute__((ext_vector_type(4)));

template <int V, bool PAST, typename T>
__device__ inline GnVec<T, V> gn_raw_past(const T* p) {
    if constexpr (PAST && sizeof(GnVec<T, V>) == sizeof(GnFour)) {
        const GnFour v = __builtin_nontemporal_load(reinterpret_cast<const GnFour*>(p));
        return __builtin_bit_cast(GnVec<T, V>, v);
    } else {
        return gn_raw<V>(p);
    }
}

template <int V, typename T>
__device__ inline void gn_load(const T* p, float (&out)[V]) {
    const GnVec<T, V> x = gn_raw<V>(p);
#pragma unroll
    for (int k = 0; k < V; ++k) out[k] = (float)x.v[k];
}

template <int V, bool PAST, typename T>
__device__ inline void gn_store(T* p, const float (&in)[V]) {
    GnVec<T, V> x;
#pragma unroll
    for (int k = 0; k < V; ++k) x.v[k] = (T)in[k];
    if constexpr (PAST && sizeof(x) == sizeof(GnFour))
        __builtin_nontemporal_store(__builtin_bit_cast(GnFour, x), reinterpret_cast<GnFour*>(p));
    else
        *reinterpret_cast<GnVec<T, V>*>(p) = x;
}

// V parameters from channel c on (none: the value where there are none).  The type
// is asked for once, so that the loads go out together.
template <int V>
__device__ inline void gn_params(const void* p, int dtype, int c, float none, float (&out)[V]) {
    if (!p) {
#pragma unroll
        for (int k = 0; k < V; ++k) out[k] = none;
    } else if (dtype == kGnF32) {
#pragma unroll
        for (int k = 0; k < V; ++k) out[k] = ((const float*)p)[c + k];
    } else if (dtype == kGnBF16) {
#pragma unroll
        for (int k = 0; k < V; ++k) out[k] = (float)((const __bf16*)p)[c + k];
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) out[k] = (float)((const _Float16*)p)[c + k];
    }
}

// The groups of V consecutive channels, relative to the slice's first.
template <int V>
__device__ inline void gn_group_of(int chan, int d, int (&g)[V]) {
    int at = chan / d, left = d - (chan - at * d);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        g[k] = at;
        --left;
        at += left == 0;
        left = left == 0 ? d : left;
    }
}

__device__ inline void gn_store_param(void* p, int dtype, int c, float v) {
    if (dtype == kGnF32) ((float*)p)[c] = v;
    else if (dtype == kGnBF16) ((__bf16*)p)[c] = (__bf16)v;
    else ((_Float16*)p)[c] = (_Float16)v;
}

__device__ inline float gn_sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __expf(-z));
}

// The normal distribution's tail below -|z| and e = exp(-z^2 / 2): erfc(x) = t P(t)
// exp(-x^2), t = 1 / (1 + p x), Abramowitz and Stegun 7.1.26, within 1.5e-7 of it, and
// the exponential is the slope's too.  GELU is within 2.1e-7 for z < 0, relative to its
// value 3e-6 at -2, 5e-5 at -3 and 5e-4 at -4, where z (1 + erf) / 2 in fp32 has 9e-7,
// 1e-5 and 5e-4 (beyond that it loses all, and this does not).  With the library's erfc
// a pass forward and backward takes 427 us for 239 (24x24576x128 bf16) and 470 for 397
// (fp32).
__device__ inline float gn_tail(float z, float* e) {
    const float x = __builtin_fabsf(z);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(x, 0.3275911f * 0.70710678f, 1.0f));
    *e = __expf(-0.5f * z * z);
    float q = __builtin_fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
    q = __builtin_fmaf(t, q, 0.5f * 1.421413741f);
    q = __builtin_fmaf(t, q, 0.5f * -0.284496736f);
    q = __builtin_fmaf(t, q, 0.5f * 0.254829592f);
    return q * t * *e;
}

template <int ACT>
__device__ inline float gn_act(float z) {
    if (ACT == kActRelu) return z < 0.0f ? 0.0f : z;  // NaN stays
    if (ACT == kActSilu) return z * gn_sigmoid(z);
    if (ACT == kActGelu) {
        float e;
        const float q = z * gn_tail(z, &e);
        return z > 0.0f ? z - q : q;
    }
    return z;
}

template <int ACT>
__device__ inline float gn_slope(float z) {
    if (ACT == kActRelu) return z > 0.0f ? 1.0f : 0.0f;
    if (ACT == kActSilu) {
        const float p = gn_sigmoid(z);
        return __builtin_fmaf(p, __builtin_fmaf(-z, p, z), p);
    }
    if (ACT == kActGelu) {
        float e;
        const float q = gn_tail(z, &e);
        return __builtin_fmaf(z * 0.39894228f, e, z > 0.0f ? 1.0f - q : q);
    }
    return 1.0f;
}

// A workgroup's place: its slice's first channel and width, its thread's first
// channel and row, and the rows of a pass.
struct GnPlace {
    int c0, cs, vecs, passrows, row, chan;
    int g0, ng;  // the slice's groups
    int part;
    bool live;
};

template <int V>
__device__ inline GnPlace gn_place(const GnShape& h, int slice, int threads = kGnThreads) {
    GnPlace q;
    const int group = h.parts > 1 ? slice / h.parts : slice * h.gs;
    q.part = h.parts > 1 ? slice - group * h.parts : 0;
    q.g0 = group;
    q.c0 = group * h.d + q.part * h.cs;
    const int end = h.parts > 1 ? (group + 1) * h.d : h.c;
    q.cs = q.c0 + h.cs < end ? h.cs : end - q.c0;
    q.ng = h.parts > 1 ? 1 : q.cs / h.d;
    q.vecs = q.cs / V;
    q.passrows = threads / q.vecs;
    q.row = threadIdx.x / q.vecs;
    q.chan = (threadIdx.x - q.row * q.vecs) * V;
    q.live = q.row < q.passrows;
    return q;
}

// A thread's rows from r on, a pass apart: f(A, offset) takes A of them at once
// (`stride` elements apart), so that their loads are in flight together.
constexpr int kGnAhead = 4;

template <int N> struct GnInt { static constexpr int value = N; };

template <int A, typename F>
__device__ inline void gn_rows(int64_t r, int64_t end, int passrows, int64_t stride, int c,
                               F&& f) {
    int64_t at = r * c;
    int left = r < end ? (int)((end - r + passrows - 1) / passrows) : 0;
    for (; left >= A; left -= A, at += A * stride) f(GnInt<A>(), at);
    for (; left > 0; --left, at += stride) f(GnInt<1>(), at);
}

struct GnWhere { int n, chunk, slice; };

__device__ inline GnWhere gn_where(const GnShape& h, uint32_t block, int chunks) {
    GnWhere w;
    const uint32_t per = (uint32_t)h.slices * chunks;
    w.n = block / per;
    const uint32_t rest = block - w.n * per;
    w.chunk = rest / h.slices;
    w.slice = rest - w.chunk * h.slices;
    return w;
}

// Sums the threads' values of each channel over the rows of a pass, and leaves
// the slice's channel sums in buf[0 .. cs).
template <int V>
__device__ inline void gn_rows_sum(float* buf, const GnPlace& q, const float (&v)[V]) {
    __syncthreads();
    if (q.live) {
#pragma unroll
        for (int k = 0; k < V; ++k) buf[q.row * q.cs + q.chan + k] = v[k];
    }
    // Eight rows to one a step: a barrier costs more than the additions.
    int n = q.passrows * q.cs;
    while (n > q.cs) {
        const int m = (n / q.cs + 7) / 8 * q.cs;
        __syncthreads();
        for (int i = threadIdx.x; i < m; i += blockDim.x) {
            float s = buf[i];
            for (int j = i + m; j < n; j += m) s += buf[j];
            buf[i] = s;
        }
        n = m;
    }
    __syncthreads();
}

// Lanes that work on one group together: a power of two.
__device__ inline int gn_lanes(int ng) {
    int t = 64;
    while (t > 1 && t * ng > kGnThreads) t >>= 1;
    return t;
}

__device__ inline float gn_lanes_sum(float x, int t) {
    for (int m = t >> 1; m > 0; m >>= 1) x += __shfl_xor(x, m);
    return x;
}

// Group sums of buf[0 .. cs) into out[0 .. ng).
__device__ inline void gn_groups_sum(const float* buf, float* out, const GnPlace& q, int d) {
    const int t = gn_lanes(q.ng), lane = threadIdx.x & (t - 1), step = blockDim.x / t;
    const int width = q.ng == 1 ? q.cs : d;
    for (int base = 0; base < q.ng; base += step) {
        const int g = base + threadIdx.x / t;
        float s = 0.0f;
        if (g < q.ng)
            for (int k = lane; k < width; k += t) s += buf[g * width + k];
        s = gn_lanes_sum(s, t);
        if (g < q.ng && lane == 0) out[g] = s;
    }
    __syncthreads();
}

// ---- forward

// Mean and squared deviations of a slice's groups over a chunk.  Reads x once: 32 us
// of 24x24576x128 bf16 (4.7 TB/s), 67 us of 2766240x32 fp32 (5.3 TB/s).  Small tensors
// (8x6144x128 bf16, 12.6 MB: 10.6 us, 1.2 TB/s) wait for its four sums over the
// workgroup, which has four rows a thread to read.
template <typename T, int V>
__global__ __launch_bounds__(kGnThreads) void k_gn_stats(GnArgs a) {
    __shared__ float buf[kGnThreads * V];
    __shared__ float gsum[kGnThreads * V], gmean[kGnThreads * V];
    const GnShape& h = a.h;
    const GnWhere at_block = gn_where(h, blockIdx.x, h.chunks);
    const int n = at_block.n, chunk = at_block.chunk;
    const GnPlace q = gn_place<V>(h, at_block.slice);
    const int64_t begin = chunk * h.rows, end = begin + h.rows < h.s ? begin + h.rows : h.s;
    const T* x = (const T*)a.x + ((int64_t)n * h.s) * h.c + q.c0 + q.chan;
    const int64_t stride = (int64_t)q.passrows * h.c;
    float k0[V], s1[V], s2[V], cnt = 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) k0[k] = s1[k] = s2[k] = 0.0f;
    if (q.live && begin + q.row < end) {
        gn_load<V>(x + (begin + q.row) * h.c, k0);
        gn_rows<kGnAhead>(begin + q.row, end, q.passrows, stride, h.c, [&](auto ahead, int64_t r) {
            constexpr int A = decltype(ahead)::value;
            GnVec<T, V> v[A];
#pragma unroll
            for (int u = 0; u < A; ++u) v[u] = gn_raw<V>(x + r + u * stride);
#pragma unroll
            for (int u = 0; u < A; ++u)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float e = (float)v[u].v[k] - k0[k];
                    s1[k] += e;
                    s2[k] = __builtin_fmaf(e, e, s2[k]);
                }
            cnt += (float)A;
        });
    }
    // The thread's mean and squared deviations per channel.
    float mean[V], m2[V], w[V];
    const float inv = cnt > 0.0f ? 1.0f / cnt : 0.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const float e = s1[k] * inv;
        mean[k] = k0[k] + e;
        m2[k] = fmaxf(__builtin_fmaf(-s1[k], e, s2[k]), 0.0f);
        w[k] = cnt * mean[k];
    }
    gn_rows_sum<V>(buf, q, w);
    gn_groups_sum(buf, gsum, q, h.d);
    const int width = q.ng == 1 ? q.cs : h.d;
    const float total = (float)(end - begin) * (float)width;
    for (int g = threadIdx.x; g < q.ng; g += kGnThreads) gmean[g] = gsum[g] / total;
    __syncthreads();
    if (q.live) {
        int group[V];
        gn_group_of<V>(q.ng == 1 ? 0 : q.chan, q.ng == 1 ? V + 1 : h.d, group);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float e = mean[k] - gmean[group[k]];
            w[k] = __builtin_fmaf(cnt * e, e, m2[k]);
        }
    }
    gn_rows_sum<V>(buf, q, w);
    gn_groups_sum(buf, gsum, q, h.d);
    for (int g = threadIdx.x; g < q.ng; g += kGnThreads) {
        float* o = a.partials +
                   ((((int64_t)n * h.chunks + chunk) * h.groups + q.g0 + g) * h.parts + q.part) * 2;
        o[0] = gmean[g];
        o[1] = gsum[g];
    }
}

// The values that one partial result of a group stands for.
__device__ inline float gn_weight(const GnShape& h, int chunk, int part) {
    const int64_t left = h.s - chunk * h.rows;
    const int width = h.d - part * h.cs < h.cs ? h.d - part * h.cs : h.cs;
    return (float)(left < h.rows ? left : h.rows) * (float)(h.parts > 1 ? width : h.d);
}

// Joins a slice's partial means and deviations: mean and 1 / sqrt(var + eps)
// of its groups into LDS.  A lane holds HELD of them, so that they are loaded
// together and once; what is beyond is read twice.
constexpr int kGnHeld = 12, kGnHeldInline = 4;  // as many as there are, mostly

template <int HELD>
__device__ inline void gn_join_stats(const GnArgs& a, const GnPlace& q, int n, float* mean,
                                     float* rstd) {
    const GnShape& h = a.h;
    const int t = gn_lanes(q.ng), lane = threadIdx.x & (t - 1), step = kGnThreads / t;
    const int entries = h.chunks * h.parts;
    const float2* all = (const float2*)a.partials + (int64_t)n * h.chunks * h.groups * h.parts;
    const int64_t row = (int64_t)h.groups * h.parts;
    for (int base = 0; base < q.ng; base += step) {
        const int g = base + threadIdx.x / t;
        const bool in = g < q.ng;
        const float2* p = all + (int64_t)(q.g0 + g) * h.parts;
        float2 v[HELD];
        float w[HELD], sw = 0.0f, swm = 0.0f;
#pragma unroll
        for (int u = 0; u < HELD; ++u) {
            const int i = lane + u * t, chunk = i / h.parts, part = i - chunk * h.parts;
            v[u] = make_float2(0.0f, 0.0f);
            w[u] = 0.0f;
            if (in && i < entries) {
                v[u] = p[chunk * row + part];
                w[u] = gn_weight(h, chunk, part);
            }
        }
#pragma unroll
        for (int u = 0; u < HELD; ++u) {
            sw += w[u];
            swm = __builtin_fmaf(w[u], v[u].x, swm);
        }
        for (int i = lane + HELD * t; in && i < entries; i += t) {
            const int chunk = i / h.parts, part = i - chunk * h.parts;
            const float m = gn_weight(h, chunk, part);
            sw += m;
            swm = __builtin_fmaf(m, p[chunk * row + part].x, swm);
        }
        sw = gn_lanes_sum(sw, t);
        const float mu = gn_lanes_sum(swm, t) / sw;
        float m2 = 0.0f;
#pragma unroll
        for (int u = 0; u < HELD; ++u) {
            const float dm = v[u].x - mu;
            m2 += __builtin_fmaf(w[u] * dm, dm, v[u].y);
        }
        for (int i = lane + HELD * t; in && i < entries; i += t) {
            const int chunk = i / h.parts, part = i - chunk * h.parts;
            const float2 e = p[chunk * row + part];
            const float dm = e.x - mu;
            m2 += __builtin_fmaf(gn_weight(h, chunk, part) * dm, dm, e.y);
        }
        m2 = gn_lanes_sum(m2, t);
        if (in && lane == 0) {
            mean[g] = mu;
            rstd[g] = 1.0f / __builtin_sqrtf(m2 / sw + a.eps);
        }
    }
    __syncthreads();
}

// The joining as a launch of its own: four groups a workgroup, a wave each.
constexpr int kGnJoin = kGnThreads / 64;

__device__ inline GnPlace gn_join_place(const GnShape& h, uint32_t block, int* n) {
    const uint32_t per = (h.groups + kGnJoin - 1) / kGnJoin;
    GnPlace q;
    *n = block / per;
    q.g0 = (block - *n * per) * kGnJoin;
    q.ng = h.groups - q.g0 < kGnJoin ? h.groups - q.g0 : kGnJoin;
    return q;
}

__global__ __launch_bounds__(kGnThreads) void k_gn_join_stats(GnArgs a) {
    __shared__ float gmean[kGnThreads], grstd[kGnThreads];
    int n;
    const GnPlace q = gn_join_place(a.h, blockIdx.x, &n);
    gn_join_stats<kGnHeld>(a, q, n, gmean, grstd);
    for (int g = threadIdx.x; g < q.ng; g += kGnThreads) {
        a.mean[(int64_t)n * a.h.groups + q.g0 + g] = gmean[g];
        a.rstd[(int64_t)n * a.h.groups + q.g0 + g] = grstd[g];
    }
}

// y from x and the joined statistics.  Reads x, writes y: 51 us of 24x24576x128 bf16
// (6.0 TB/s), 105 us of 2766240x32 fp32 (6.7 TB/s).  PAST: 1 stores past the caches,
// 2 loads too.
template <typename T, int V, int ACT, int PAST>
__global__ __launch_bounds__(kGnThreads) void k_gn_apply(GnArgs a) {
    __shared__ float gmean[kGnThreads * V], grstd[kGnThreads * V];
    const GnShape& h = a.h;
    const GnWhere w = gn_where(h, blockIdx.x, h.apply_chunks);
    const int n = w.n, chunk = w.chunk;
    const GnPlace q = gn_place<V>(h, w.slice);
    float scale[V], bias[V];
    if (q.live) {
        gn_params<V>(a.weight, a.wdtype, q.c0 + q.chan, 1.0f, scale);
        gn_params<V>(a.bias, a.wdtype, q.c0 + q.chan, 0.0f, bias);
    }
    if (a.joined) {
        for (int g = threadIdx.x; g < q.ng; g += kGnThreads) {
            gmean[g] = a.mean[(int64_t)n * h.groups + q.g0 + g];
            grstd[g] = a.rstd[(int64_t)n * h.groups + q.g0 + g];
        }
        __syncthreads();
    } else {
        gn_join_stats<kGnHeldInline>(a, q, n, gmean, grstd);
    }
    if (a.mean && !a.joined && chunk == 0 && q.part == 0)
        for (int g = threadIdx.x; g < q.ng; g += kGnThreads) {
            a.mean[(int64_t)n * h.groups + q.g0 + g] = gmean[g];
            a.rstd[(int64_t)n * h.groups + q.g0 + g] = grstd[g];
        }
    if (!q.live) return;
    float mean[V];
    int group[V];
    gn_group_of<V>(q.ng == 1 ? 0 : q.chan, q.ng == 1 ? V + 1 : h.d, group);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        mean[k] = gmean[group[k]];
        scale[k] *= grstd[group[k]];
    }
    const int64_t begin = chunk * h.apply_rows;
    const int64_t end = begin + h.apply_rows < h.s ? begin + h.apply_rows : h.s;
    const int64_t at = ((int64_t)n * h.s) * h.c + q.c0 + q.chan;
    const int64_t stride = (int64_t)q.passrows * h.c;
    const T* x = (const T*)a.x + at;
    T* y = (T*)a.out + at;
    gn_rows<kGnAhead>(begin + q.row, end, q.passrows, stride, h.c, [&](auto ahead, int64_t r) {
        constexpr int A = decltype(ahead)::value;
        GnVec<T, V> raw[A];
#pragma unroll
        for (int u = 0; u < A; ++u) raw[u] = gn_raw_past<V, PAST == 2>(x + r + u * stride);
#pragma unroll
        for (int u = 0; u < A; ++u) {
            float v[V];
#pragma unroll
            for (int k = 0; k < V; ++k)
                v[k] = gn_act<ACT>(
                    __builtin_fmaf((float)raw[u].v[k] - mean[k], scale[k], bias[k]));
            gn_store<V, PAST != 0>(y + r + u * stride, v);
        }
    });
}

// ---- backward

// Sums of dz and dz xh per channel and, weighted, per group over a chunk.  Reads x and
// dy: 61 us of 24x24576x128 bf16 silu (5.0 TB/s; its arithmetic takes some 40 of
// them at the VALU's full rate), 81 with gelu, 126 us of 2766240x32 fp32 silu (5.6 TB/s);
// 13.3 us of 8x6144x128 bf16 (25 MB, 1.9 TB/s: as k_gn_stats).
template <typename T, int V, int ACT>
__global__ __launch_bounds__(kGnThreads) void k_gn_bwd_sums(GnArgs a) {
    __shared__ float buf[kGnThreads * V], chan_sums[2][kGnThreads * V], gsum[kGnThreads * V];
    const GnShape& h = a.h;
    const GnWhere at_block = gn_where(h, blockIdx.x, h.chunks);
    const int n = at_block.n, chunk = at_block.chunk;
    const GnPlace q = gn_place<V>(h, at_block.slice);
    const int64_t begin = chunk * h.rows, end = begin + h.rows < h.s ? begin + h.rows : h.s;
    const int64_t at = ((int64_t)n * h.s) * h.c + q.c0 + q.chan;
    const int64_t stride = (int64_t)q.passrows * h.c;
    const T* x = (const T*)a.x + at;
    const T* dy = (const T*)a.dy + at;
    // The sums are of dz and dz (x - mean); 1 / deviation is a factor of the latter.
    float mean[V], rstd[V], scale[V], bias[V], sa[V], sb[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sa[k] = sb[k] = rstd[k] = 0.0f;
    if (q.live) {
        gn_params<V>(a.weight, a.wdtype, q.c0 + q.chan, 1.0f, scale);
        gn_params<V>(a.bias, a.wdtype, q.c0 + q.chan, 0.0f, bias);
        int group[V];
        gn_group_of<V>(q.ng == 1 ? 0 : q.chan, q.ng == 1 ? V + 1 : h.d, group);
        const int64_t g0 = (int64_t)n * h.groups + q.g0;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            mean[k] = a.mean[g0 + group[k]];
            rstd[k] = a.rstd[g0 + group[k]];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) scale[k] *= rstd[k];
    }
    if (q.live)
        gn_rows<kGnAhead>(begin + q.row, end, q.passrows, stride, h.c, [&](auto ahead, int64_t r) {
            constexpr int A = decltype(ahead)::value;
            GnVec<T, V> v[A], t[A];
#pragma unroll
            for (int u = 0; u < A; ++u) {
                v[u] = gn_raw<V>(x + r + u * stride);
                t[u] = gn_raw<V>(dy + r + u * stride);
            }
#pragma unroll
            for (int u = 0; u < A; ++u)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const float e = (float)v[u].v[k] - mean[k];
                    const float dz =
                        (float)t[u].v[k] * gn_slope<ACT>(__builtin_fmaf(e, scale[k], bias[k]));
                    sa[k] += dz;
                    sb[k] = __builtin_fmaf(dz, e, sb[k]);
                }
        });
#pragma unroll
    for (int k = 0; k < V; ++k) sb[k] *= rstd[k];
    for (int w = 0; w < 2; ++w) {
        gn_rows_sum<V>(buf, q, w ? sb : sa);
        for (int c = threadIdx.x; c < q.cs; c += kGnThreads) {
            float s = buf[c], weight[1];
            gn_params<1>(a.weight, a.wdtype, q.c0 + c, 1.0f, weight);
            chan_sums[w][c] = s;
            buf[c] = s * weight[0];
        }
        __syncthreads();
        gn_groups_sum(buf, gsum, q, h.d);
        for (int g = threadIdx.x; g < q.ng; g += kGnThreads)
            a.partials[((((int64_t)n * h.chunks + chunk) * h.groups + q.g0 + g) * h.parts +
                        q.part) * 2 + w] = gsum[g];
    }
    if (a.channels)
        for (int c = threadIdx.x; c < q.cs; c += kGnThreads) {
            float2* o = (float2*)a.channels + ((int64_t)n * h.chunks + chunk) * h.c + q.c0 + c;
            *o = make_float2(chan_sums[0][c], chan_sums[1][c]);
        }
}

// dw and db of kGnChans channels: 32 threads a channel over the samples' chunks,
// eight loads in flight each.
constexpr int kGnChans = kGnThreads / 32;

__device__ inline void gn_channel_grads(const GnArgs& a, int block) {
    __shared__ double sums[2][32][kGnChans + 1];
    const GnShape& h = a.h;
    const int lane = threadIdx.x % kGnChans, row = threadIdx.x / kGnChans;
    const int c = block * kGnChans + lane, entries = a.n * h.chunks;
    double sa = 0.0, sb = 0.0;
    if (c < h.c) {
        const float2* p = (const float2*)a.channels + c;
        int i = row;
        for (; i + 7 * 32 < entries; i += 8 * 32) {
            float2 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = p[(int64_t)(i + k * 32) * h.c];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                sa += v[k].x;
                sb += v[k].y;
            }
        }
        for (; i < entries; i += 32) {
            const float2 v = p[(int64_t)i * h.c];
            sa += v.x;
            sb += v.y;
        }
    }
    sums[0][row][lane] = sa;
    sums[1][row][lane] = sb;
    __syncthreads();
    if (row < 2 && c < h.c) {
        double s = 0.0;
        for (int k = 0; k < 32; ++k) s += sums[row][k][lane];
        void* to = row ? a.dweight : a.dbias;
        if (to) gn_store_param(to, a.wdtype, c, (float)s);
    }
}

// E[w dz] and E[w dz xh] of a slice's groups.
template <int HELD>
__device__ inline void gn_join_sums(const GnArgs& a, const GnPlace& q, int n, float* g1,
                                    float* g2) {
    const GnShape& h = a.h;
    const int t = gn_lanes(q.ng), lane = threadIdx.x & (t - 1), step = kGnThreads / t;
    const int entries = h.chunks * h.parts;
    const float inv = 1.0f / ((float)h.s * (float)h.d);
    for (int base = 0; base < q.ng; base += step) {
        const int g = base + threadIdx.x / t;
        float sa = 0.0f, sb = 0.0f;
        const float2* p = (const float2*)a.partials +
                          ((int64_t)n * h.chunks * h.groups + q.g0 + g) * h.parts;
        const int64_t row = (int64_t)h.groups * h.parts;
        for (int first = lane; g < q.ng && first < entries; first += HELD * t) {
            float2 v[HELD];
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
                const int i = first + u * t, ch = i / h.parts, part = i - ch * h.parts;
                v[u] = make_float2(0.0f, 0.0f);
                if (i < entries) v[u] = p[ch * row + part];
            }
#pragma unroll
            for (int u = 0; u < HELD; ++u) {
                sa += v[u].x;
                sb += v[u].y;
            }
        }
        sa = gn_lanes_sum(sa, t);
        sb = gn_lanes_sum(sb, t);
        if (g < q.ng && lane == 0) {
            g1[g] = sa * inv;
            g2[g] = sb * inv;
        }
    }
    __syncthreads();
}

__global__ __launch_bounds__(kGnThreads) void k_gn_join_sums(GnArgs a) {
    __shared__ float g1[kGnThreads], g2[kGnThreads];
    if ((int)blockIdx.x < a.channel_blocks) {
        gn_channel_grads(a, blockIdx.x);
        return;
    }
    int n;
    const GnPlace q = gn_join_place(a.h, blockIdx.x - a.channel_blocks, &n);
    gn_join_sums<kGnHeld>(a, q, n, g1, g2);
    for (int g = threadIdx.x; g < q.ng; g += kGnThreads)
        ((float2*)a.groups_out)[(int64_t)n * a.h.groups + q.g0 + g] = make_float2(g1[g], g2[g]);
}

// dx from x, dy and the joined sums.  Reads x and dy, writes dx: 74 us of 24x24576x128
// bf16 silu (6.1 TB/s), 155 us of 2766240x32 fp32 (6.8 TB/s).  PAST as above.  The
// first workgroups join dw and db where no launch in between has done so.
template <typename T, int V, int ACT, int PAST>
__global__ __launch_bounds__(kGnThreads) void k_gn_bwd_apply(GnArgs a) {
    __shared__ float g1[kGnThreads * V], g2[kGnThreads * V];
    const GnShape& h = a.h;
    if ((int)blockIdx.x < a.channel_blocks) {
        gn_channel_grads(a, blockIdx.x);
        return;
    }
    const GnWhere at_block = gn_where(h, blockIdx.x - a.channel_blocks, h.apply_chunks);
    const int n = at_block.n, chunk = at_block.chunk;
    const GnPlace q = gn_place<V>(h, at_block.slice);
    if (a.joined) {
        for (int g = threadIdx.x; g < q.ng; g += kGnThreads) {
            const float2 v = ((const float2*)a.groups_out)[(int64_t)n * h.groups + q.g0 + g];
            g1[g] = v.x;
            g2[g] = v.y;
        }
        __syncthreads();
    } else {
        gn_join_sums<kGnHeldInline>(a, q, n, g1, g2);
    }
    if (!q.live) return;
    // dx = (r w) dz - r E[w dz] - (x - mean) r^2 E[w dz xh]
    float mean[V], rstd[V], scale[V], bias[V], e1[V], e2[V];
    gn_params<V>(a.weight, a.wdtype, q.c0 + q.chan, 1.0f, scale);
    gn_params<V>(a.bias, a.wdtype, q.c0 + q.chan, 0.0f, bias);
    int group[V];
    gn_group_of<V>(q.ng == 1 ? 0 : q.chan, q.ng == 1 ? V + 1 : h.d, group);
    const int64_t g0 = (int64_t)n * h.groups + q.g0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        mean[k] = a.mean[g0 + group[k]];
        rstd[k] = a.rstd[g0 + group[k]];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
        scale[k] *= rstd[k];
        e1[k] = -rstd[k] * g1[group[k]];
        e2[k] = -rstd[k] * (rstd[k] * g2[group[k]]);
    }
    const int64_t begin = chunk * h.apply_rows;
    const int64_t end = begin + h.apply_rows < h.s ? begin + h.apply_rows : h.s;
    const int64_t at = ((int64_t)n * h.s) * h.c + q.c0 + q.chan;
    const int64_t stride = (int64_t)q.passrows * h.c;
    const T* x = (const T*)a.x + at;
    const T* dy = (const T*)a.dy + at;
    T* dx = (T*)a.out + at;
    gn_rows<kGnAhead>(begin + q.row, end, q.passrows, stride, h.c, [&](auto ahead, int64_t r) {
        constexpr int A = decltype(ahead)::value;
        GnVec<T, V> v[A], t[A];
#pragma unroll
        for (int u = 0; u < A; ++u) {
            v[u] = gn_raw_past<V, PAST == 2>(x + r + u * stride);
            t[u] = gn_raw_past<V, PAST == 2>(dy + r + u * stride);
        }
#pragma unroll
        for (int u = 0; u < A; ++u) {
            float o[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float e = (float)v[u].v[k] - mean[k];
                const float dz =
                    (float)t[u].v[k] * gn_slope<ACT>(__builtin_fmaf(e, scale[k], bias[k]));
                o[k] = __builtin_fmaf(dz, scale[k], __builtin_fmaf(e, e2[k], e1[k]));
            }
            gn_store<V, PAST != 0>(dx + r + u * stride, o);
        }
    });
}

// ---- one launch: a workgroup keeps its slice of a sample in registers

// At most kGnWholeThreads threads with P vectors each; x (and dy) are read once.
// Bound: latency, of the launch (some 4 us of any kernel in a trace), one reading and
// two to four sums over the workgroup (1x384x256 bf16: 8.7 us forward and 10.6 backward,
// the two launches forward took 15; 4x1024x128 bf16: 9.8 and 13.5).
constexpr int kGnWholeThreads = 1024;

extern __shared__ float gn_lds[];

__device__ inline float gn_act_of(int act, float z) {
    switch (act) {
        case kActRelu: return gn_act<kActRelu>(z);
        case kActSilu: return gn_act<kActSilu>(z);
        case kActGelu: return gn_act<kActGelu>(z);
    }
    return z;
}

__device__ inline float gn_slope_of(int act, float z) {
    switch (act) {
        case kActRelu: return gn_slope<kActRelu>(z);
        case kActSilu: return gn_slope<kActSilu>(z);
        case kActGelu: return gn_slope<kActGelu>(z);
    }
    return 1.0f;
}

// Workgroups go to the eight XCDs in turn; each XCD takes a run of consecutive
// slices, so that the slices of a row, which share cache lines, share an L2.
constexpr int kGnXcds = 8;

__device__ inline int gn_by_xcd(int total) {
    const int per = gridDim.x / kGnXcds;
    const int id = (blockIdx.x % kGnXcds) * per + blockIdx.x / kGnXcds;
    return id < total ? id : -1;
}

template <typename T, int V, int P>
__global__ __launch_bounds__(kGnWholeThreads) void k_gn_whole(GnArgs a) {
    const GnShape& h = a.h;
    const int id = gn_by_xcd(a.n * h.slices);
    if (id < 0) return;
    const int n = id / h.slices, slice = id - n * h.slices;
    const GnPlace q = gn_place<V>(h, slice, blockDim.x);
    float* buf = gn_lds;
    float* gmean = buf + blockDim.x * V;
    float* grstd = gmean + q.cs;
    const int64_t at = (int64_t)n * h.s * h.c + (int64_t)q.row * h.c + q.c0 + q.chan;
    const int64_t stride = (int64_t)q.passrows * h.c;
    const T* x = (const T*)a.x + at;
    T* y = (T*)a.out + at;
    const int mine = q.live && q.row < h.s ? (int)((h.s - q.row + q.passrows - 1) / q.passrows) : 0;
    GnVec<T, V> raw[P];
#pragma unroll
    for (int u = 0; u < P; ++u)
        if (u < mine) raw[u] = gn_raw<V>(x + u * stride);
    float scale[V], bias[V], w[V], mean[V];
    if (q.live) {
        gn_params<V>(a.weight, a.wdtype, q.c0 + q.chan, 1.0f, scale);
        gn_params<V>(a.bias, a.wdtype, q.c0 + q.chan, 0.0f, bias);
    }
    int group[V];
    gn_group_of<V>(q.ng == 1 ? 0 : q.chan, q.ng == 1 ? V + 1 : h.d, group);
#pragma unroll
    for (int k = 0; k < V; ++k) w[k] = 0.0f;
#pragma unroll
    for (int u = 0; u < P; ++u)
        if (u < mine) {
#pragma unroll
            for (int k = 0; k < V; ++k) w[k] += (float)raw[u].v[k];
        }
    gn_rows_sum<V>(buf, q, w);
    gn_groups_sum(buf, gmean, q, h.d);
    const float inv = 1.0f / ((float)h.s * (float)h.d);
    if (q.live) {
#pragma unroll
        for (int k = 0; k < V; ++k) mean[k] = gmean[group[k]] * inv;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) w[k] = 0.0f;
#pragma unroll
    for (int u = 0; u < P; ++u)
        if (u < mine) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float e = (float)raw[u].v[k] - mean[k];
                w[k] = __builtin_fmaf(e, e, w[k]);
            }
        }
    gn_rows_sum<V>(buf, q, w);
    gn_groups_sum(buf, grstd, q, h.d);
    for (int g = threadIdx.x; g < q.ng; g += blockDim.x) {
        const float r = 1.0f / __builtin_sqrtf(grstd[g] * inv + a.eps);
        grstd[g] = r;
        if (a.mean) {
            a.mean[(int64_t)n * h.groups + q.g0 + g] = gmean[g] * inv;
            a.rstd[(int64_t)n * h.groups + q.g0 + g] = r;
        }
    }
    __syncthreads();
    if (!q.live) return;
#pragma unroll
    for (int k = 0; k < V; ++k) scale[k] *= grstd[group[k]];
#pragma unroll
    for (int u = 0; u < P; ++u)
        if (u < mine) {
            float v[V];
#pragma unroll
            for (int k = 0; k < V; ++k)
                v[k] = gn_act_of(
                    a.act, __builtin_fmaf((float)raw[u].v[k] - mean[k], scale[k], bias[k]));
            gn_store<V, false>(y + u * stride, v);
        }
}

template <typename T, int V, int P>
__global__ __launch_bounds__(kGnWholeThreads) void k_gn_bwd_whole(GnArgs a) {
    const GnShape& h = a.h;
    const int id = gn_by_xcd(a.n * h.slices);
    if (id < 0) return;
    const int n = id / h.slices, slice = id - n * h.slices;
    const GnPlace q = gn_place<V>(h, slice, blockDim.x);
    float* buf = gn_lds;
    float* g1 = buf + blockDim.x * V;
    float* g2 = g1 + q.cs;
    float* chan = g2 + q.cs;
    const int64_t at = (int64_t)n * h.s * h.c + (int64_t)q.row * h.c + q.c0 + q.chan;
    const int64_t stride = (int64_t)q.passrows * h.c;
    const T* x = (const T*)a.x + at;
    const T* dy = (const T*)a.dy + at;
    const int mine = q.live && q.row < h.s ? (int)((h.s - q.row + q.passrows - 1) / q.passrows) : 0;
    GnVec<T, V> v[P], t[P];
#pragma unroll
    for (int u = 0; u < P; ++u)
        if (u < mine) {
            v[u] = gn_raw<V>(x + u * stride);
            t[u] = gn_raw<V>(dy + u * stride);
        }
    float mean[V], rstd[V], scale[V], bias[V], sa[V], sb[V];
#pragma unroll
    for (int k = 0; k < V; ++k) sa[k] = sb[k] = rstd[k] = 0.0f;
    int group[V];
    gn_group_of<V>(q.ng == 1 ? 0 : q.chan, q.ng == 1 ? V + 1 : h.d, group);
    if (q.live) {
        gn_params<V>(a.weight, a.wdtype, q.c0 + q.chan, 1.0f, scale);
        gn_params<V>(a.bias, a.wdtype, q.c0 + q.chan, 0.0f, bias);
        const int64_t g0 = (int64_t)n * h.groups + q.g0;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            mean[k] = a.mean[g0 + group[k]];
            rstd[k] = a.rstd[g0 + group[k]];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) scale[k] *= rstd[k];
    }
#pragma unroll
    for (int u = 0; u < P; ++u)
        if (u < mine) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float e = (float)v[u].v[k] - mean[k];
                const float dz = (float)t[u].v[k] *
                                 gn_slope_of(a.act, __builtin_fmaf(e, scale[k], bias[k]));
                sa[k] += dz;
                sb[k] = __builtin_fmaf(dz, e, sb[k]);
            }
        }
#pragma unroll
    for (int k = 0; k < V; ++k) sb[k] *= rstd[k];
    for (int w = 0; w < 2; ++w) {
        gn_rows_sum<V>(buf, q, w ? sb : sa);
        for (int c = threadIdx.x; c < q.cs; c += blockDim.x) {
            float s = buf[c], weight[1];
            gn_params<1>(a.weight, a.wdtype, q.c0 + c, 1.0f, weight);
            buf[c] = s * weight[0];
            if (w == 0) {
                chan[c] = s;
            } else if (a.channels) {
                ((float2*)a.channels)[(int64_t)n * h.c + q.c0 + c] = make_float2(chan[c], s);
            } else {  // one sample: the sums are the gradients
                if (a.dbias) gn_store_param(a.dbias, a.wdtype, q.c0 + c, chan[c]);
                if (a.dweight) gn_store_param(a.dweight, a.wdtype, q.c0 + c, s);
            }
        }
        __syncthreads();
        gn_groups_sum(buf, w ? g2 : g1, q, h.d);
    }
    if (!q.live || !a.out) return;
    const float inv = 1.0f / ((float)h.s * (float)h.d);
    float e1[V], e2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        e1[k] = -rstd[k] * (g1[group[k]] * inv);
        e2[k] = -rstd[k] * (rstd[k] * (g2[group[k]] * inv));
    }
    T* dx = (T*)a.out + at;
#pragma unroll
    for (int u = 0; u < P; ++u)
        if (u < mine) {
            float o[V];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float e = (float)v[u].v[k] - mean[k];
                const float dz = (float)t[u].v[k] *
                                 gn_slope_of(a.act, __builtin_fmaf(e, scale[k], bias[k]));
                o[k] = __builtin_fmaf(dz, scale[k], __builtin_fmaf(e, e2[k], e1[k]));
            }
            gn_store<V, false>(dx + u * stride, o);
        }
}

// ---- host

static int gn_gcd(int a, int b) { return b ? gn_gcd(b, a % b) : a; }

// How n samples of s rows and c channels are cut, with vectors of `vec` channels
// (1 where no slice of whole groups and whole vectors fits 256 of them).
static GnShape gn_shape(int64_t n, int64_t s, int32_t c, int32_t groups, int* vec) {
    GnShape h;
    h.s = s;
    h.c = c;
    h.groups = groups;
    h.d = c / groups;
    h.parts = 1;
    int unit = *vec / gn_gcd(h.d, *vec);
    if (unit > 1 && (int64_t)unit * h.d > (int64_t)kGnThreads * *vec) *vec = unit = 1;
    const int most = kGnThreads * *vec;
    if (h.d > most) {
        h.gs = 1;
        h.parts = (h.d + most - 1) / most;
        h.cs = (h.d + h.parts - 1) / h.parts;
        h.cs = (h.cs + *vec - 1) / *vec * *vec;
        h.parts = (h.d + h.cs - 1) / h.cs;
        h.slices = groups * h.parts;
    } else {
        h.gs = most / h.d / unit * unit;
        if (h.gs > groups) h.gs = groups;
        h.cs = h.gs * h.d;
        h.slices = (groups + h.gs - 1) / h.gs;
    }
    const int64_t passrows = kGnThreads / (h.cs / *vec);
    auto cut = [&](int64_t blocks, int64_t passes, int64_t* rows) {
        int64_t chunks = blocks / (n * h.slices);
        if (chunks < 1) chunks = 1;
        const int64_t most_chunks = (s + passrows * passes - 1) / (passrows * passes);
        if (chunks > most_chunks) chunks = most_chunks;
        *rows = (s + chunks - 1) / chunks;
        return (int32_t)((s + *rows - 1) / *rows);
    };
    // Summing: three workgroups a CU, all resident at once (one more than fit
    // would run by itself; 24x24576x128 bf16 backward: 1032 of them 151 us, 768 of
    // them 135).  Applying: as many as keep every CU busy to the end.
    h.chunks = cut(768, 4, &h.rows);
    h.apply_chunks = cut(4096, 4, &h.apply_rows);
    return h;
}

// Whether the sums are joined by a launch of their own: where a workgroup of the
// second launch would read more of them than this, and a group has more than one.
constexpr int64_t kGnInline = 1024;

// (8192x8x2048 bf16, a channel a group, one partial result each: joined all the same, in
// 4 million workgroups, 9620 us forward and backward, 590 not.)
static bool gn_joined(const GnShape& h) {
    return (int64_t)h.chunks * h.parts > 1 && (int64_t)h.chunks * h.parts * h.gs > kGnInline;
}

static uint32_t gn_join_blocks(const GnArgs& a) {
    return (uint32_t)a.n * ((a.h.groups + kGnJoin - 1) / kGnJoin);
}

static int gn_widest(int dtype) { return dtype == kGnF32 ? 4 : kGnMaxVec; }

static bool gn_valid(int64_t n, int64_t s, int32_t c, int32_t groups, int32_t dtype) {
    return n > 0 && s > 0 && c > 0 && groups > 0 && c % groups == 0 && dtype >= kGnF32 &&
           dtype <= kGnF16 && s <= ((int64_t)1 << 40) / c &&
           n <= ((int64_t)1 << 44) / (s * c);
}

// Four channels a vector, of 16 bits too: eight would not leave registers for 16
// vectors, and narrower slices make more workgroups.
constexpr int kGnWholeVec = 4;

// The one-launch form, where a slice of a sample fits a workgroup's registers
// (`most` vectors a thread): the slice is the narrowest of whole groups and whole
// vectors that gives a workgroup 256 vectors.  Threads of a workgroup, or 0.
//
// A slice of few channels is a few bytes of each row, which the two-launch form
// reads whole: this form is for samples of few rows and tensors of a few MB (bf16,
// us of this form and the other: 1x384x512 9.1 and 13.3 forward, 10.9 and 14.6
// backward; 4x1536x128 10.0 and 13.3, 14.8 and 14.6; 4x6144x128 18.6 and 17.9, 29.8
// and 20.8; 24x1536x512, 36 MB, 39.3 and 34.0, 69.0 and 44.4).
constexpr int64_t kGnWholeBytes = (int64_t)24 << 20;
constexpr int64_t kGnWholeRowsForward = 2048, kGnWholeRowsBackward = 1024;

static int gn_whole(int64_t n, int64_t s, int32_t c, int32_t groups, int vec, int most,
                    int64_t rows, int size, GnShape* shape) {
    if (s > rows || n * s * c * size > kGnWholeBytes) return 0;
    GnShape h{};
    h.s = s;
    h.c = c;
    h.groups = groups;
    h.d = c / groups;
    h.parts = 1;
    h.chunks = 1;
    h.rows = s;
    const int unit = vec / gn_gcd(h.d, vec);
    const int64_t row_vecs = (int64_t)unit * h.d / vec;
    if (row_vecs > 256) return 0;
    int64_t wide = (256 + s * row_vecs - 1) / (s * row_vecs);
    if (wide * row_vecs > 256) wide = 256 / row_vecs;
    h.gs = (int32_t)(wide * unit < groups ? wide * unit : groups);
    h.cs = h.gs * h.d;
    h.slices = (groups + h.gs - 1) / h.gs;
    const int vecs = h.cs / vec;
    // Four vectors a thread, more where that takes too many threads.
    int64_t threads = (((s + 3) / 4) * vecs + 63) / 64 * 64;
    if (threads < 256) threads = 256;
    if (threads > kGnWholeThreads) threads = kGnWholeThreads;
    if ((s + threads / vecs - 1) / (threads / vecs) > most) return 0;
    if (n > ((int64_t)1 << 22) / h.slices) return 0;
    *shape = h;
    return (int)threads;
}

// A launch has fewer than 2^24 workgroups of 256 threads: those of the samples, 2^23 at
// most, and where dw or db is asked for those of the channels' sums beside them.  No product
// overflows, as n s c is at most 2^44.
static bool gn_fits(int64_t n, const GnShape& h, bool sums) {
    const int64_t chunks = h.chunks > h.apply_chunks ? h.chunks : h.apply_chunks;
    const int64_t join = gn_joined(h) ? n * ((h.groups + kGnJoin - 1) / kGnJoin) : 0;
    const int64_t blocks = n * h.slices * chunks > join ? n * h.slices * chunks : join;
    const int64_t channels = sums ? (h.c + (int64_t)kGnChans - 1) / kGnChans : 0;
    return blocks <= (int64_t)1 << 23 && blocks + channels < (int64_t)1 << 24;
}

// Stores go past the caches where the tensor is larger than the L2s together, the
// second reading of the inputs where they are too large to have stayed in the
// memory-side cache (bf16, 128 channels, forward/backward in us, plain and so:
// 48 MB 37.0/62.5 and 35.7/54.4 with stores, 144 MB 101/162 and 81/134 with both;
// 96 MB forward 58.0 with stores, 58.9 with both, backward 105 and 96).
static int gn_past(int64_t bytes, bool backward) {
    if (bytes > (int64_t)(backward ? 64 : 128) << 20) return 2;
    return bytes > (int64_t)32 << 20;
}

static bool gn_aligned(const void* p, int to) { return ((uintptr_t)p % to) == 0; }

}  // namespace cs

using namespace cs;

extern "C" size_t cs_group_norm_workspace_elems(int64_t n, int64_t s, int32_t c, int32_t groups,
                                                int32_t dtype, int32_t backward) {
    if (!gn_valid(n, s, c, groups, dtype)) return 0;
    size_t most = 0;
    for (int vec : {gn_widest(dtype), 1}) {
        if (c % vec) continue;
        const GnShape h = gn_shape(n, s, c, groups, &vec);
        size_t e = (size_t)n * h.chunks * groups * h.parts * 2;
        if (gn_joined(h)) e += (size_t)n * groups * 2;
        if (backward) e += (size_t)n * h.chunks * c * 2;
        most = e > most ? e : most;
    }
    return most;
}

namespace {

constexpr int kGnWholeForward = 16, kGnWholeBackward = 8;  // vectors a thread at most

template <typename T, int V, bool BACKWARD>
int gn_run_whole(const GnArgs& a, int threads, hipStream_t stream) {
    const GnShape& h = a.h;
    const dim3 grid((unsigned)((a.n * h.slices + kGnXcds - 1) / kGnXcds * kGnXcds));
    const dim3 block((unsigned)threads);
    const size_t lds = ((size_t)threads * V + (size_t)h.cs * (BACKWARD ? 3 : 2)) * sizeof(float);
    const int passrows = threads / (h.cs / V);
    const bool few = h.s <= 4 * (int64_t)passrows;
    if (!BACKWARD) {
        if (few)
            hipLaunchKernelGGL((k_gn_whole<T, V, 4>), grid, block, lds, stream, a);
        else
            hipLaunchKernelGGL((k_gn_whole<T, V, kGnWholeForward>), grid, block, lds, stream, a);
    } else {
        if (few)
            hipLaunchKernelGGL((k_gn_bwd_whole<T, V, 4>), grid, block, lds, stream, a);
        else
            hipLaunchKernelGGL((k_gn_bwd_whole<T, V, kGnWholeBackward>), grid, block, lds, stream,
                               a);
        if (a.channels)
            hipLaunchKernelGGL(k_gn_join_sums, dim3(a.channel_blocks), dim3(kGnThreads), 0, stream,
                               a);
    }
    return hipGetLastError() == hipSuccess ? CS_OK : CS_ERR_HIP;
}

template <bool BACKWARD>
int gn_dispatch_whole(const GnArgs& a, int dtype, int vec, int threads, hipStream_t stream) {
    if (dtype == kGnF32)
        return vec > 1 ? gn_run_whole<float, kGnWholeVec, BACKWARD>(a, threads, stream)
                       : gn_run_whole<float, 1, BACKWARD>(a, threads, stream);
    if (dtype == kGnBF16)
        return vec > 1 ? gn_run_whole<__bf16, kGnWholeVec, BACKWARD>(a, threads, stream)
                       : gn_run_whole<__bf16, 1, BACKWARD>(a, threads, stream);
    return vec > 1 ? gn_run_whole<_Float16, kGnWholeVec, BACKWARD>(a, threads, stream)
                   : gn_run_whole<_Float16, 1, BACKWARD>(a, threads, stream);
}

template <typename T, int V, int ACT>
int gn_forward_act(const GnArgs& a, hipStream_t stream) {
    const GnShape& h = a.h;
    const dim3 sums((unsigned)(a.n * h.slices * h.chunks));
    const dim3 apply((unsigned)(a.n * h.slices * h.apply_chunks)), block(kGnThreads);
    hipLaunchKernelGGL((k_gn_stats<T, V>), sums, block, 0, stream, a);
    if (a.joined)
        hipLaunchKernelGGL(k_gn_join_stats, dim3(gn_join_blocks(a)), block, 0, stream, a);
    if (V > 1 && a.past == 2)
        hipLaunchKernelGGL((k_gn_apply<T, V, ACT, (V > 1 ? 2 : 0)>), apply, block, 0, stream, a);
    else if (V > 1 && a.past == 1)
        hipLaunchKernelGGL((k_gn_apply<T, V, ACT, (V > 1 ? 1 : 0)>), apply, block, 0, stream, a);
    else
        hipLaunchKernelGGL((k_gn_apply<T, V, ACT, 0>), apply, block, 0, stream, a);
    return hipGetLastError() == hipSuccess ? CS_OK : CS_ERR_HIP;
}

template <typename T, int V, int ACT>
int gn_backward_act(GnArgs a, hipStream_t stream) {
    const GnShape& h = a.h;
    const dim3 sums((unsigned)(a.n * h.slices * h.chunks)), block(kGnThreads);
    hipLaunchKernelGGL((k_gn_bwd_sums<T, V, ACT>), sums, block, 0, stream, a);
    if (a.joined) {
        hipLaunchKernelGGL(k_gn_join_sums,
                           dim3(a.channel_blocks + (a.out ? gn_join_blocks(a) : 0)), block, 0,
                           stream, a);
        a.channel_blocks = 0;
    }
    const dim3 apply(
        (unsigned)(a.channel_blocks + (a.out ? a.n * h.slices * h.apply_chunks : 0)));
    if (apply.x == 0) {
    } else if (V > 1 && a.past == 2) {
        hipLaunchKernelGGL((k_gn_bwd_apply<T, V, ACT, (V > 1 ? 2 : 0)>), apply, block, 0, stream,
                           a);
    } else if (V > 1 && a.past == 1) {
        hipLaunchKernelGGL((k_gn_bwd_apply<T, V, ACT, (V > 1 ? 1 : 0)>), apply, block, 0, stream,
                           a);
    } else {
        hipLaunchKernelGGL((k_gn_bwd_apply<T, V, ACT, 0>), apply, block, 0, stream, a);
    }
    return hipGetLastError() == hipSuccess ? CS_OK : CS_ERR_HIP;
}

template <typename T, int V, bool BACKWARD>
int gn_run(const GnArgs& a, int act, hipStream_t stream) {
    switch (act) {
        case kActNone:
            return BACKWARD ? gn_backward_act<T, V, kActNone>(a, stream)
                            : gn_forward_act<T, V, kActNone>(a, stream);
        case kActRelu:
            return BACKWARD ? gn_backward_act<T, V, kActRelu>(a, stream)
                            : gn_forward_act<T, V, kActRelu>(a, stream);
        case kActSilu:
            return BACKWARD ? gn_backward_act<T, V, kActSilu>(a, stream)
                            : gn_forward_act<T, V, kActSilu>(a, stream);
        default:
            return BACKWARD ? gn_backward_act<T, V, kActGelu>(a, stream)
                            : gn_forward_act<T, V, kActGelu>(a, stream);
    }
}

template <bool BACKWARD>
int gn_dispatch(const GnArgs& a, int dtype, int vec, int act, hipStream_t stream) {
    if (dtype == kGnF32)
        return vec > 1 ? gn_run<float, 4, BACKWARD>(a, act, stream)
                       : gn_run<float, 1, BACKWARD>(a, act, stream);
    if (dtype == kGnBF16)
        return vec > 1 ? gn_run<__bf16, 8, BACKWARD>(a, act, stream)
                       : gn_run<__bf16, 1, BACKWARD>(a, act, stream);
    return vec > 1 ? gn_run<_Float16, 8, BACKWARD>(a, act, stream)
                   : gn_run<_Float16, 1, BACKWARD>(a, act, stream);
}

}  // namespace

extern "C" int cs_group_norm_forward(const void* x, int64_t n, int64_t s, int32_t c,
                                     int32_t groups, int32_t dtype, const void* weight,
                                     const void* bias, int32_t param_dtype, double eps,
                                     int32_t act, float* workspace, float* mean, float* rstd,
                                     void* y, hipStream_t stream) {
    if (!gn_valid(n, s, c, groups, dtype) || param_dtype < kGnF32 || param_dtype > kGnF16 ||
        act < kActNone || act > kActGelu || !(eps >= 0.0) || !x || !y || !workspace ||
        !mean != !rstd)
        return CS_ERR_ARGS;
    int vec = gn_widest(dtype);
    if (c % vec || !gn_aligned(x, 16) || !gn_aligned(y, 16)) vec = 1;
    GnArgs a{};
    const int whole_vec = vec > 1 || (c % kGnWholeVec == 0 && gn_aligned(x, 16) && gn_aligned(y, 16))
                              ? kGnWholeVec : 1;
    const int size = dtype == kGnF32 ? 4 : 2;
    const int whole = gn_whole(n, s, c, groups, whole_vec, kGnWholeForward, kGnWholeRowsForward,
                               size, &a.h);
    if (!whole) a.h = gn_shape(n, s, c, groups, &vec);
    if (!whole && !gn_fits(n, a.h, false)) return CS_ERR_ARGS;
    a.act = act;
    a.x = x;
    a.weight = weight;
    a.bias = bias;
    a.wdtype = param_dtype;
    a.eps = (float)eps;
    a.partials = workspace;
    a.mean = mean;
    a.rstd = rstd;
    a.out = y;
    a.n = (int32_t)n;
    if (whole) return gn_dispatch_whole<false>(a, dtype, whole_vec, whole, stream);
    a.past = gn_past(n * s * c * size, false);
    a.joined = gn_joined(a.h);
    if (a.joined && !mean) {
        a.mean = workspace + (size_t)n * a.h.chunks * groups * a.h.parts * 2;
        a.rstd = a.mean + (size_t)n * groups;
    }
    return gn_dispatch<false>(a, dtype, vec, act, stream);
}

extern "C" int cs_group_norm_backward(const void* x, const void* dy, int64_t n, int64_t s,
                                      int32_t c, int32_t groups, int32_t dtype,
                                      const void* weight, const void* bias, int32_t param_dtype,
                                      int32_t act, const float* mean, const float* rstd,
                                      float* workspace, void* dx, void* dweight, void* dbias,
                                      hipStream_t stream) {
    if (!gn_valid(n, s, c, groups, dtype) || param_dtype < kGnF32 || param_dtype > kGnF16 ||
        act < kActNone || act > kActGelu || !x || !dy || !mean || !rstd || !workspace ||
        !gn_aligned(workspace, 8))
        return CS_ERR_ARGS;
    if (!dx && !dweight && !dbias) return CS_OK;
    int vec = gn_widest(dtype);
    if (c % vec || !gn_aligned(x, 16) || !gn_aligned(dy, 16) || (dx && !gn_aligned(dx, 16))) vec = 1;
    GnArgs a{};
    const int whole_vec = vec > 1 || (c % kGnWholeVec == 0 && gn_aligned(x, 16) &&
                                      gn_aligned(dy, 16) && (!dx || gn_aligned(dx, 16)))
                              ? kGnWholeVec : 1;
    const int size = dtype == kGnF32 ? 4 : 2;
    const int whole = gn_whole(n, s, c, groups, whole_vec, kGnWholeBackward, kGnWholeRowsBackward,
                               size, &a.h);
    if (!whole) a.h = gn_shape(n, s, c, groups, &vec);
    if (!whole && !gn_fits(n, a.h, dweight || dbias)) return CS_ERR_ARGS;
    a.act = act;
    a.x = x;
    a.dy = dy;
    a.weight = weight;
    a.bias = bias;
    a.wdtype = param_dtype;
    a.partials = workspace;
    a.mean = const_cast<float*>(mean);
    a.rstd = const_cast<float*>(rstd);
    a.out = dx;
    a.dweight = dweight;
    a.dbias = dbias;
    a.n = (int32_t)n;
    if (whole) {
        if (n > 1 && (dweight || dbias)) {
            a.channels = workspace;
            a.channel_blocks = (c + kGnChans - 1) / kGnChans;
        }
        return gn_dispatch_whole<true>(a, dtype, whole_vec, whole, stream);
    }
    a.past = gn_past(n * s * c * size, true);
    a.joined = gn_joined(a.h);
    float* rest = workspace + (size_t)n * a.h.chunks * groups * a.h.parts * 2;
    if (a.joined) {
        a.groups_out = rest;
        rest += (size_t)n * groups * 2;
    }
    if (dweight || dbias) {
        a.channels = rest;
        a.channel_blocks = (c + kGnChans - 1) / kGnChans;
    }
    return gn_dispatch<true>(a, dtype, vec, act, stream);
}
