// AdamW over all tensors of a network, with fp32 or 8-bit states, and the
// global norm of their gradients.
//
// Per element (decoupled weight decay; t the step of the tensor):
//   g  = grad * clip
//   p  = p * (1 - lr * weight_decay)
//   m  = m + (1 - beta1) * (g - m)
//   v  = v * beta2 + (1 - beta2) * g * g
//   p -= lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
// in fp32.  A bf16 or fp16 parameter has an fp32 master copy, which is what
// the update moves; the parameter is the master rounded to nearest.
//
// 8-bit states.  A byte holds m as sign, 4 exponent bits and 3 mantissa bits,
// and a byte holds sqrt(v), not v, as 4 exponent and 4 mantissa bits: the root
// is what the update divides by, has half of v's exponent range and no sign.
// 128 consecutive values share one byte, the biased fp32 exponent E of the
// largest finite |value|: a code's exponent field e and mantissa f stand for
//   e > 0:  (1 + f / 2^M) 2^(e - 14) 2^(E - 127),   e = 0: f / 2^M 2^(-13) 2^(E - 127)
// so the largest value lies in the binade e = 14, and rounding up ends at
// e = 15, f = 0 at most.  The code with all exponent and mantissa bits set is
// NaN (and what infinity becomes).  The scale is a power of two, so that
// scaling is exact and the code is the scaled float's own top bits: the float
// x 2^(14 - E) has e in its exponent field, subnormals included.
//
// Rounding is stochastic: with beta2 near 1 a step changes v by a fraction of
// a code's spacing, and rounding to nearest would lose every such change (v
// would stop where 1 - beta2 times g^2 falls under half a spacing).  A 16-bit
// random number is added below the code's last bit before the lower bits are
// cut, so the expected value is the value.  The numbers are a hash of (seed,
// step, tensor, element), hence the same in every run and launch shape.  A
// root that is not zero never becomes zero: the update divides by it.
//
// Bound: HBM at 28 bytes an element with fp32 states and 16 with 8-bit ones, whose
// 80 or so VALU slots an element come near the hundred that the bandwidth leaves.  A
// launch takes up to 56 tensors, whose pointers travel in its arguments, so nothing
// of the step is uploaded; a workgroup takes one pass of 2048 elements of one tensor,
// found by one ballot over the tensors' first workgroups, and its loads go out
// together.  Measured (means of a kernel trace): fp32 states 897 us of 197M bf16 weights
// (6.1 TB/s), 69 us of 16.3M fp32 (6.6 TB/s); 8-bit states 525 us of 197M bf16 (6.0
// TB/s), 165 us of 60.0M bf16 (5.8 TB/s), 45 us of 16.3M fp32 (5.8 TB/s).  Tensors off 16
// bytes are read and written value by value: 16.7M, most of them off, 137 us fp32 and
// 153 us bf16 with fp32 states, where aligned ones take 70 and 74.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/cubicsplat_hip.h"

namespace cs {

constexpr int kAwThreads = 256;
constexpr int kAwMaxTensors = 56;  // one lane each, and 4 KB of kernel arguments
constexpr int kAwMaxSets = 12;
constexpr int kAwPass = kAwThreads * 8;  // elements of a chunk's unit: whole blocks of 128
constexpr int kBlk = CS_ADAMW_BLOCK;

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };

struct AwTensor {
    void* param;
    const void* grad;
    float* master;
    void* avg;
    void* sq;
    int64_t n;
    uint32_t first_block;
    uint32_t meta;  // dtype | eight << 4 | vector << 5 | set << 8
    uint32_t key;
    uint32_t pad;
};

struct AwSet {
    float decay, step_size, inv_bc2_sqrt, omb1, beta2, omb2, eps, pad;
};

struct AwArgs {
    AwTensor t[kAwMaxTensors];
    AwSet s[kAwMaxSets];
    const float* clip;
    int64_t chunk;
    int32_t n;
    int32_t out_dtype;
};

static_assert(sizeof(AwArgs) <= 4096, "kernel arguments");

__host__ __device__ inline uint32_t aw_mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x9E3779B9u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}

// The hash's argument for element i, a multiple of 4; the three after it follow.
__device__ inline uint32_t aw_key(uint32_t key, int64_t i) {
    return key + (uint32_t)i + (uint32_t)(i >> 32) * 0x3C6EF372u;
}

// The tensor this workgroup works on: lane k holds tensor k's first block.
__device__ inline int aw_find(const AwArgs& a) {
    const int lane = threadIdx.x & 63;
    const bool mine = lane < a.n && a.t[lane < a.n ? lane : 0].first_block <= blockIdx.x;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1);
}

template <int DT> struct AwType;
template <> struct AwType<kF32> { typedef float type; };
template <> struct AwType<kBF16> { typedef __bf16 type; };
template <> struct AwType<kF16> { typedef _Float16 type; };

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) AwVec { T v[N]; };

typedef float AwFour __attribute__((ext_vector_type(4)));
typedef float AwTwo __attribute__((ext_vector_type(2)));

// One vector of at most 16 bytes; PAST: past the caches.
template <bool PAST, typename T, int N>
__device__ inline AwVec<T, N> aw_get(const T* p) {
    if constexpr (PAST && sizeof(AwVec<T, N>) == sizeof(AwFour))
        return __builtin_bit_cast(AwVec<T, N>,
                                  __builtin_nontemporal_load(reinterpret_cast<const AwFour*>(p)));
    else if constexpr (PAST && sizeof(AwVec<T, N>) == sizeof(AwTwo))
        return __builtin_bit_cast(AwVec<T, N>,
                                  __builtin_nontemporal_load(reinterpret_cast<const AwTwo*>(p)));
    else
        return *reinterpret_cast<const AwVec<T, N>*>(p);
}

template <bool PAST, typename T, int N>
__device__ inline void aw_put(T* p, const AwVec<T, N>& x) {
    if constexpr (PAST && sizeof(x) == sizeof(AwFour))
        __builtin_nontemporal_store(__builtin_bit_cast(AwFour, x), reinterpret_cast<AwFour*>(p));
    else if constexpr (PAST && sizeof(x) == sizeof(AwTwo))
        __builtin_nontemporal_store(__builtin_bit_cast(AwTwo, x), reinterpret_cast<AwTwo*>(p));
    else
        *reinterpret_cast<AwVec<T, N>*>(p) = x;
}

// N consecutive elements at element i.  FULL: all of them are there, aligned;
// otherwise elements past n are 0 and not stored.
template <int N, bool FULL, bool PAST = false, typename T>
__device__ inline void aw_load(const T* src, int64_t i, int64_t n, float (&out)[N]) {
    if constexpr (FULL) {
        const AwVec<T, N> x = aw_get<PAST, T, N>(src + i);
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = (float)x.v[k];
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k) out[k] = i + k < n ? (float)src[i + k] : 0.0f;
    }
}

template <int N, bool FULL, bool PAST = false, typename T>
__device__ inline void aw_store(T* dst, int64_t i, int64_t n, const float (&in)[N]) {
    if constexpr (FULL) {
        AwVec<T, N> x;
#pragma unroll
        for (int k = 0; k < N; ++k) x.v[k] = (T)in[k];
        aw_put<PAST>(dst + i, x);
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (i + k < n) dst[i + k] = (T)in[k];
    }
}

// The passes of [begin, end): f(FULL, first element) by the whole workgroup, full
// where all of the pass's elements are there and `vec` (a uniform choice, as the
// lanes of a block work together).
template <bool B> struct AwBool { static constexpr bool value = B; };

template <typename F>
__device__ inline void aw_passes(int64_t begin, int64_t end, bool vec, F&& f) {
    int64_t base = begin;
    if (vec)
        for (; base + kAwPass <= end; base += kAwPass) f(AwBool<true>(), base);
    for (; base < end; base += kAwPass) f(AwBool<false>(), base);
}

__device__ inline void aw_moments(const AwSet& s, float g, float& m, float& v) {
    m = m + s.omb1 * (g - m);
    v = v * s.beta2 + s.omb2 * (g * g);
}

// p after the step.  The hardware's reciprocal (1 ulp): the quotient is a few
// roundings off, the sequence of a rounded division would double the instructions.
__device__ inline float aw_move(const AwSet& s, float p, float m, float root) {
    const float inv = __builtin_amdgcn_rcpf(__builtin_fmaf(root, s.inv_bc2_sqrt, s.eps));
    return p * s.decay - s.step_size * (m * inv);
}

// Square roots of four second moments.  Where all of a wave's are ordinary numbers,
// by a reciprocal root and one correction by its exact remainder, half the
// instructions of the general sequence and the same roundings.
__device__ inline void aw_roots(const float (&v)[4], float (&root)[4]) {
    uint32_t low = ~0u, high = 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t b = __float_as_uint(v[k]);   // no sign: in the numbers' order
        low = b < low ? b : low;
        high = b > high ? b : high;
    }
    if (__all(low >= 0x0F800000u && high < 0x7F800000u)) {   // 2^-96, infinity
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float r = __builtin_amdgcn_rsqf(v[k]);
            const float x = v[k] * r;
            root[k] = __builtin_fmaf(__builtin_fmaf(-x, x, v[k]), 0.5f * r, x);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) root[k] = __builtin_sqrtf(v[k]);
    }
}

// ---- 8-bit codes

template <int MB>
__device__ inline float aw_decode(uint32_t code, int e) {
    const uint32_t mag = code & ((1u << (4 + MB)) - 1u);
    const float x = __builtin_ldexpf(__uint_as_float(mag << (23 - MB)), e - 14);
    const float y = mag == (1u << (4 + MB)) - 1u ? __builtin_nanf("") : x;
    return MB == 3 && (code & 0x80u) ? -y : y;
}

// The codes of a lane's four values; every lane of the wave takes part.  Scaled, a
// number's bits begin with its code.  Below the lowest binade the scaling rounds to
// nearest; there the bits are cut off instead, as the random number goes on top of
// what is left: 3 values of 10,000 of a normal distribution, so that most waves skip it.
template <int MB, bool FLOOR>
__device__ inline void aw_encode(const float (&x)[4], int e, const uint32_t (&r16)[4],
                                 uint32_t (&c)[4]) {
    uint32_t t[4], low = ~0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        t[k] = __float_as_uint(__builtin_ldexpf(x[k], 14 - e)) & 0x7FFFFFFFu;
        low = t[k] < low ? t[k] : low;
    }
    if (__any(low <= 0x00800000u)) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (t[k] <= 0x00800000u)
                t[k] = (uint32_t)__builtin_ldexpf(__builtin_fabsf(x[k]), 14 - e + 149);
    }
    const uint32_t all = (1u << (4 + MB)) - 1u;   // infinity and NaN end above it
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        c[k] = (t[k] + (r16[k] << (7 - MB))) >> (23 - MB);
        if (FLOOR) {  // x has no sign: 1 where it is not zero
            const uint32_t b = __float_as_uint(x[k]), one = b < 1u ? b : 1u;
            c[k] = c[k] < one ? one : c[k];
        }
        c[k] = c[k] < all ? c[k] : all;
        if (MB == 3) c[k] |= (__float_as_uint(x[k]) >> 24) & 0x80u;
    }
}

// The largest of the 32 lanes that hold a block.
__device__ inline uint32_t aw_block_max(uint32_t x) {
#define CS_ROW_MAX(ctrl)                                                                    \
    {                                                                                       \
        const uint32_t o =                                                                  \
            (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, 0xF, 0xF, true);         \
        x = x > o ? x : o;                                                                  \
    }
    CS_ROW_MAX(0x128);  // row_ror:8
    CS_ROW_MAX(0x124);
    CS_ROW_MAX(0x122);
    CS_ROW_MAX(0x121);
#undef CS_ROW_MAX
    // Both rows of 16 have their own; the odd rows of one copy change places with the
    // even rows of the other.
    const auto both = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return both[0] > both[1] ? both[0] : both[1];
}

// The exponent field of a block's largest finite magnitude; every lane of the wave
// takes part.  Magnitudes compare as their bits do; blocks with infinities or NaN
// are looked at again without them.
__device__ inline int aw_shared_exponent(const float (&x)[4]) {
    uint32_t top = 0u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t a = __float_as_uint(x[k]) & 0x7FFFFFFFu;
        top = a > top ? a : top;
    }
    top = aw_block_max(top);
    if (__any(top >= 0x7F800000u)) {
        top = 0u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t a = __float_as_uint(x[k]) & 0x7FFFFFFFu;
            top = a > top && a < 0x7F800000u ? a : top;
        }
        top = aw_block_max(top);
    }
    return (int)(top >> 23);
}

// The four or eight bytes of a lane; the code arrays are whole blocks, so all exist
// wherever the lane's first element does.
template <int N>
__device__ inline void aw_load_codes(const uint8_t* src, int64_t i, bool in, uint32_t (&c)[N]) {
    uint32_t w[N / 4] = {};
    if (in) __builtin_memcpy(w, __builtin_assume_aligned(src + i, N), N);
#pragma unroll
    for (int k = 0; k < N; ++k) c[k] = (w[k / 4] >> (8 * (k & 3))) & 0xFFu;
}

__device__ inline void aw_store_codes(uint8_t* dst, int64_t i, bool in, const uint32_t (&c)[4]) {
    if (in)
        *reinterpret_cast<uint32_t*>(dst + i) = c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24;
}

__device__ inline int64_t aw_blocks(int64_t n) { return (n + kBlk - 1) / kBlk; }

// Encodes and stores a lane's four values of m and root; every lane of the wave
// takes part.
template <bool FULL>
__device__ inline void aw_hold(uint8_t* avg, uint8_t* sq, int64_t i, int64_t n,
                               const float (&m)[4], const float (&root)[4],
                               const uint32_t (&r)[4]) {
    const bool in = FULL || i < n;
    const int em = aw_shared_exponent(m), er = aw_shared_exponent(root);
    uint32_t lo[4], hi[4], cm[4], cr[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        lo[k] = r[k] & 0xFFFFu;
        hi[k] = r[k] >> 16;
    }
    aw_encode<3, false>(m, em, lo, cm);
    aw_encode<4, true>(root, er, hi, cr);
    aw_store_codes(avg, i, in, cm);
    aw_store_codes(sq, i, in, cr);
    if (in && (threadIdx.x & 31) == 0) {
        const int64_t b = aw_blocks(n) * kBlk + i / kBlk;
        avg[b] = (uint8_t)em;
        sq[b] = (uint8_t)er;
    }
}

template <bool FULL, int N>
__device__ inline void aw_held(const uint8_t* avg, const uint8_t* sq, int64_t i, int64_t n,
                               float (&m)[N], float (&root)[N]) {
    const bool in = FULL || i < n;
    const int64_t b = aw_blocks(n) * kBlk + i / kBlk;
    const int em = in ? avg[b] : 0, er = in ? sq[b] : 0;
    uint32_t cm[N], cr[N];
    aw_load_codes(avg, i, in, cm);
    aw_load_codes(sq, i, in, cr);
#pragma unroll
    for (int k = 0; k < N; ++k) {
        m[k] = aw_decode<3>(cm[k], em);
        root[k] = aw_decode<4>(cr[k], er);
    }
}

// ---- the step

template <int DT, int PAST>
__device__ inline void aw_step32(const AwTensor& t, const AwSet& s, float clip, int64_t begin,
                                 int64_t end) {
    typedef typename AwType<DT>::type T;
    const bool vec = (t.meta >> 5) & 1;
    float* main = DT == kF32 ? (float*)t.param : t.master;
    aw_passes(begin, end, vec, [&](auto full, int64_t base) {
        constexpr bool F = decltype(full)::value;
        // Two vectors a thread, their loads in flight together.
        float p[2][4], g[2][4], m[2][4], v[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t i = base + (u * kAwThreads + threadIdx.x) * 4;
            aw_load<4, F, PAST == 2>(main, i, end, p[u]);
            aw_load<4, F, PAST == 2>((const T*)t.grad, i, end, g[u]);
            aw_load<4, F, PAST != 0>((const float*)t.avg, i, end, m[u]);
            aw_load<4, F, PAST != 0>((const float*)t.sq, i, end, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t i = base + (u * kAwThreads + threadIdx.x) * 4;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                aw_moments(s, g[u][k] * clip, m[u][k], v[u][k]);
                p[u][k] = aw_move(s, p[u][k], m[u][k], __builtin_sqrtf(v[u][k]));
            }
            aw_store<4, F, PAST == 2>(main, i, end, p[u]);
            if (DT != kF32) aw_store<4, F, PAST == 2>((T*)t.param, i, end, p[u]);
            aw_store<4, F, PAST != 0>((float*)t.avg, i, end, m[u]);
            aw_store<4, F, PAST != 0>((float*)t.sq, i, end, v[u]);
        }
    });
}

template <int DT, int PAST>
__device__ inline void aw_step8(const AwTensor& t, const AwSet& s, float clip, int64_t begin,
                                int64_t end) {
    typedef typename AwType<DT>::type T;
    const bool vec = (t.meta >> 5) & 1;
    float* main = DT == kF32 ? (float*)t.param : t.master;
    aw_passes(begin, end, vec, [&](auto full, int64_t base) {
        constexpr bool F = decltype(full)::value;
        // Two vectors of four a thread, their loads in flight together.
        float p[2][4], g[2][4], m[2][4], root[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t i = base + (u * kAwThreads + threadIdx.x) * 4;
            aw_load<4, F, PAST != 0>(main, i, t.n, p[u]);
            aw_load<4, F, PAST != 0>((const T*)t.grad, i, t.n, g[u]);
            aw_held<F, 4>((const uint8_t*)t.avg, (const uint8_t*)t.sq, i, t.n, m[u], root[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t i = base + (u * kAwThreads + threadIdx.x) * 4;
            const uint32_t key = aw_key(t.key, i);
            uint32_t r[4];
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = root[u][k] * root[u][k];
                aw_moments(s, g[u][k] * clip, m[u][k], v[k]);
            }
            aw_roots(v, root[u]);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                p[u][k] = aw_move(s, p[u][k], m[u][k], root[u][k]);
                r[k] = aw_mix(key + k);
                // Elements past the end do not set a block's exponent.
                if (!F && i + k >= t.n) m[u][k] = root[u][k] = 0.0f;
            }
            aw_store<4, F, PAST != 0>(main, i, t.n, p[u]);
            if (DT != kF32) aw_store<4, F, PAST != 0>((T*)t.param, i, t.n, p[u]);
            aw_hold<F>((uint8_t*)t.avg, (uint8_t*)t.sq, i, t.n, m[u], root[u], r);
        }
    });
}

// PAST: 1 the moments of 32 bits, which nothing reads before the next step, go past
// the caches, and the weights and gradients of tensors with 8-bit ones, whose codes
// are the smaller part; 2 the weights and gradients of all.
template <int PAST>
__global__ __launch_bounds__(kAwThreads) void k_adamw(AwArgs a) {
    const int k = aw_find(a);
    const AwTensor& t = a.t[k];
    const AwSet& s = a.s[t.meta >> 8];
    const float clip = a.clip ? *a.clip : 1.0f;
    const int64_t begin = (int64_t)(blockIdx.x - t.first_block) * a.chunk;
    const int64_t end = begin + a.chunk < t.n ? begin + a.chunk : t.n;
    switch (t.meta & 0x1F) {
        case kF32: aw_step32<kF32, PAST>(t, s, clip, begin, end); break;
        case kBF16: aw_step32<kBF16, PAST>(t, s, clip, begin, end); break;
        case kF16: aw_step32<kF16, PAST>(t, s, clip, begin, end); break;
        case kF32 | 16: aw_step8<kF32, PAST>(t, s, clip, begin, end); break;
        case kBF16 | 16: aw_step8<kBF16, PAST>(t, s, clip, begin, end); break;
        case kF16 | 16: aw_step8<kF16, PAST>(t, s, clip, begin, end); break;
    }
}

// ---- state conversions

// fp32 m (avg) and v (sq) -> codes at param (m) and grad (root), to nearest.  Bound:
// HBM, 10 bytes an element; taken when a checkpoint is loaded.
__global__ __launch_bounds__(kAwThreads) void k_adamw_pack(AwArgs a) {
    const AwTensor& t = a.t[aw_find(a)];
    const bool vec = (t.meta >> 5) & 1;
    const int64_t begin = (int64_t)(blockIdx.x - t.first_block) * a.chunk;
    const int64_t end = begin + a.chunk < t.n ? begin + a.chunk : t.n;
    aw_passes(begin, end, vec, [&](auto full, int64_t base) {
        constexpr bool F = decltype(full)::value;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int64_t i = base + (u * kAwThreads + threadIdx.x) * 4;
            float m[4], root[4];
            uint32_t r[4];
            aw_load<4, F>((const float*)t.avg, i, t.n, m);
            aw_load<4, F>((const float*)t.sq, i, t.n, root);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                root[k] = __builtin_sqrtf(root[k]);
                r[k] = 0x80008000u;  // one half of a spacing: to nearest
            }
            aw_hold<F>((uint8_t*)t.param, (uint8_t*)t.grad, i, t.n, m, root, r);
        }
    });
}

// What the states stand for, in T.  Bound: HBM, 6 bytes an element from 8 bits to
// bf16: 226 us of 197M (5.2 TB/s), 17 us of 16.3M.  16-bit values go past the caches
// (bf16, us without and with: 54.5M values of each moment 63 and 50, 16.3M 21.9 and 16.9,
// 3.5M 6.7 and 5.4); fp32 values lie 32 bytes a lane, in two stores that only the cache
// joins.
template <typename T>
__device__ inline void aw_unpack(const AwTensor& t, int64_t begin, int64_t end) {
    const bool vec = (t.meta >> 5) & 1, eight = (t.meta >> 4) & 1;
    const int64_t n = (int64_t)(intptr_t)t.master;  // with what follows the values
    // Full passes end with the values, not with what follows them.
    const int64_t whole = t.n < end ? begin + (t.n - begin) / kAwPass * kAwPass : end;
    const auto pass = [&](auto full, int64_t base) {
        constexpr bool F = decltype(full)::value;
        const int64_t i = base + threadIdx.x * 8;
        float m[8], v[8];
        if (eight) {
            aw_held<F, 8>((const uint8_t*)t.avg, (const uint8_t*)t.sq, i, t.n, m, v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool in = F || i + k < t.n;
                m[k] = in ? m[k] : 0.0f;
                v[k] = in ? v[k] * v[k] : 0.0f;
            }
        } else {
            aw_load<8, F>((const float*)t.avg, i, t.n, m);
            aw_load<8, F>((const float*)t.sq, i, t.n, v);
        }
        aw_store<8, F, sizeof(T) == 2>((T*)t.param, i, n, m);
        aw_store<8, F, sizeof(T) == 2>((T*)const_cast<void*>(t.grad), i, n, v);
    };
    if (whole > begin) aw_passes(begin, whole, vec, pass);
    aw_passes(whole > begin ? whole : begin, end, false, pass);
}

__global__ __launch_bounds__(kAwThreads) void k_adamw_unpack(AwArgs a) {
    const AwTensor& t = a.t[aw_find(a)];
    const int64_t n = (int64_t)(intptr_t)t.master;
    const int64_t begin = (int64_t)(blockIdx.x - t.first_block) * a.chunk;
    const int64_t end = begin + a.chunk < n ? begin + a.chunk : n;
    switch (a.out_dtype) {
        case kF32: aw_unpack<float>(t, begin, end); break;
        case kBF16: aw_unpack<__bf16>(t, begin, end); break;
        case kF16: aw_unpack<_Float16>(t, begin, end); break;
    }
}

// ---- the gradients' norm

// One launch sums squares, up to 2048 workgroups over all tensors, and a workgroup
// of its own joins them in fp64.  Bound: HBM, reads the gradients: 68 us of 197M bf16
// (5.8 TB/s; 78 after the values of 8-bit states were written), 14 us of 16.3M fp32 (4.6
// TB/s), and 4 us for the joining launch.
struct NormTensor {
    const void* grad;
    int64_t n;
    uint32_t first_block;
    uint32_t meta;  // dtype | vector << 5
};

constexpr int kNormMaxTensors = 64;
constexpr int kNormBlocks = CS_GRAD_NORM_BLOCKS;

struct NormArgs {
    NormTensor t[kNormMaxTensors];
    double* partials;  // of this launch's blocks
    int64_t chunk;
    int32_t n;
};

// Vectors of 16 bytes, kNormAhead of them in flight a thread.
constexpr int kNormAhead = 4;
// A chunk is whole rounds of them (bf16; 2048 elements, so that most of a chunk may
// be less than a round: 5.4M weights 13.1 us for 9.6, 197M 78.7 for 71.5).
constexpr int64_t kNormPass = (int64_t)kAwThreads * kNormAhead * 8;

template <int DT>
__device__ inline float norm_squares(const NormTensor& t, int64_t begin, int64_t end) {
    typedef typename AwType<DT>::type T;
    constexpr int N = 16 / sizeof(T);
    constexpr int64_t step = (int64_t)kAwThreads * N;
    const T* src = (const T*)t.grad;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int64_t i = begin + threadIdx.x * N;
    if ((t.meta >> 5) & 1)
        for (; i + (kNormAhead - 1) * step + N <= end; i += kNormAhead * step) {
            AwVec<T, N> g[kNormAhead];
#pragma unroll
            for (int u = 0; u < kNormAhead; ++u)
                g[u] = *reinterpret_cast<const AwVec<T, N>*>(src + i + u * step);
#pragma unroll
            for (int u = 0; u < kNormAhead; ++u)
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const float x = (float)g[u].v[k];
                    s[k & 3] = __builtin_fmaf(x, x, s[k & 3]);
                }
        }
    if ((t.meta >> 5) & 1)
        for (; i + N <= end; i += step) {
            const AwVec<T, N> g = *reinterpret_cast<const AwVec<T, N>*>(src + i);
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const float x = (float)g.v[k];
                s[k & 3] = __builtin_fmaf(x, x, s[k & 3]);
            }
        }
    for (; i < end; i += step) {
        float g[N];
        aw_load<N, false>(src, i, end, g);
#pragma unroll
        for (int k = 0; k < N; ++k) s[k & 3] = __builtin_fmaf(g[k], g[k], s[k & 3]);
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__device__ inline double block_sum(double x, double* lds) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__global__ __launch_bounds__(kAwThreads) void k_grad_squares(NormArgs a) {
    __shared__ double lds[4];
    const int lane = threadIdx.x & 63;
    const bool mine = lane < a.n && a.t[lane < a.n ? lane : 0].first_block <= blockIdx.x;
    const NormTensor& t =
        a.t[__builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1)];
    const int64_t begin = (int64_t)(blockIdx.x - t.first_block) * a.chunk;
    const int64_t end = begin + a.chunk < t.n ? begin + a.chunk : t.n;
    float s = 0.0f;
    switch (t.meta & 0xF) {
        case kF32: s = norm_squares<kF32>(t, begin, end); break;
        case kBF16: s = norm_squares<kBF16>(t, begin, end); break;
        case kF16: s = norm_squares<kF16>(t, begin, end); break;
    }
    const double sum = block_sum((double)s, lds);
    if (threadIdx.x == 0) a.partials[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kAwThreads) void k_grad_norm(const double* partials, int32_t n,
                                                          float max_norm, float* out) {
    __shared__ double lds[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += kAwThreads) s += partials[i];
    s = block_sum(s, lds);
    if (threadIdx.x == 0) {
        const float norm = (float)__builtin_sqrt(s);
        const float c = max_norm / (norm + 1e-6f);
        out[0] = norm;
        out[1] = max_norm > 0.0f && !(c > 1.0f) ? c : 1.0f;  // a NaN norm stays one
    }
}

static bool aw_aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }

// Elements of a chunk: whole passes, and at most `blocks` of them over the total.
static int64_t aw_chunk(int64_t total, int64_t blocks, int64_t pass) {
    const int64_t per = (total + blocks - 1) / blocks;
    return (per + pass - 1) / pass * pass;
}

}  // namespace cs

using namespace cs;

namespace {

enum AwOp { kStep, kPack, kUnpack };

// One pass a workgroup (bf16, 197M weights, 8-bit states: 8192 workgroups of many
// passes 660 us, one pass each 617), more only beyond 2^32 elements.
constexpr int64_t kAwBlocks = (int64_t)1 << 21;

// The moments go past the caches where a step moves more than the memory-side cache
// holds (three states in turn, us without and with: fp32, 3.2M weights, 85 MB, 15.6 and
// 16.6; 6.4M, 171 MB, 30.7 and 29.2; 10.1M, 270 MB, 55.9 and 46.1); the weights and
// gradients too where they alone are more than it holds (us: nothing, the moments, all:
// fp32 16.3M 84.6, 76.0, 75.9; 36M 190, 180, 169; bf16 54.5M 286, 278, 257; 197M 1045,
// 1020, 987).  With 8-bit states the weights and gradients go past them above the first
// limit: bf16 197M 569 and 521, fp32 16.3M (249 MB) 51.9 and 46.9; below it the step
// gains little (10.1M, 154 MB, 32.6 and 30.9; 6.4M, 98 MB, 22.6 and 22.4), and what
// reads the weights next finds them in the caches.
constexpr int64_t kAwPastBytes = (int64_t)224 << 20;
constexpr int64_t kAwPastWeights = (int64_t)256 << 20;

// table: [n][8] = param, grad, master, exp_avg, exp_avg_sq, numel, dtype | eight << 4 |
// set << 8, ordinal.
int aw_run(AwOp op, int32_t ntensors, const int64_t* table, int32_t nsets, const float* sets,
           const uint32_t* set_keys, const float* clip, int32_t out_dtype,
           hipStream_t stream) {
    if (ntensors < 0 || (ntensors > 0 && !table) || out_dtype < kF32 || out_dtype > kF16)
        return CS_ERR_ARGS;
    int64_t total = 0, bytes = 0, weights = 0;
    for (int k = 0; k < ntensors; ++k) {
        const int64_t* row = table + 8 * (int64_t)k;
        const int64_t n = row[5], meta = row[6];
        const int dtype = (int)(meta & 0xF);
        const bool eight = (meta >> 4) & 1;
        if (n < 0 || n > (int64_t)1 << 48 || dtype > kF16 || (meta & ~(int64_t)0x7FFFFF1F))
            return CS_ERR_ARGS;
        if (n == 0) continue;
        if (!row[0] || !row[1] || !row[3] || !row[4]) return CS_ERR_ARGS;
        if (op == kUnpack && (row[2] < n || row[2] > (int64_t)1 << 48)) return CS_ERR_ARGS;
        if (op == kStep) {
            if ((meta >> 8) >= nsets || !sets || !set_keys) return CS_ERR_ARGS;
            if (dtype != kF32 && !row[2]) return CS_ERR_ARGS;
        }
        // The codes are read and written eight at a time.
        if ((op != kPack && eight &&
             (!aw_aligned((void*)row[3], 8) || !aw_aligned((void*)row[4], 8))) ||
            (op == kPack && (!aw_aligned((void*)row[0], 8) || !aw_aligned((void*)row[1], 8))))
            return CS_ERR_ARGS;
        total += op == kUnpack ? row[2] : n;
        bytes += n * (eight ? 16 : 28);
        weights += n * 8;
    }
    if (total == 0) return CS_OK;
    const int64_t chunk = aw_chunk(total, kAwBlocks, kAwPass);
    const int past = weights > kAwPastWeights ? 2 : bytes > kAwPastBytes;
    int k = 0;
    while (k < ntensors) {
        AwArgs a;
        int set_of[kAwMaxSets], used = 0;
        a.n = 0;
        uint64_t blocks = 0;
        for (; k < ntensors && a.n < kAwMaxTensors; ++k) {
            const int64_t* row = table + 8 * (int64_t)k;
            const int64_t n = row[5];
            if (n == 0) continue;
            const int dtype = (int)(row[6] & 0xF), set = (int)(row[6] >> 8);
            const bool eight = (row[6] >> 4) & 1;
            int at = 0;
            if (op == kStep) {
                while (at < used && set_of[at] != set) ++at;
                if (at == used) {
                    if (used == kAwMaxSets) break;
                    set_of[used++] = set;
                    const float* f = sets + 8 * (int64_t)set;
                    a.s[at] = AwSet{f[0], f[1], f[2], f[3], f[4], f[5], f[6], 0.0f};
                }
            }
            const uint64_t b = (uint64_t)(((op == kUnpack ? row[2] : n) + chunk - 1) / chunk);
            bool vec = true;
            for (int c = 0; c < 5; ++c)
                if (c != 2 || op == kStep) vec = vec && aw_aligned((void*)row[c], 16);
            AwTensor& t = a.t[a.n++];
            t.param = (void*)row[0];
            t.grad = (const void*)row[1];
            t.master = (float*)row[2];
            t.avg = (void*)row[3];
            t.sq = (void*)row[4];
            t.n = n;
            t.first_block = (uint32_t)blocks;
            t.meta = (uint32_t)(dtype | (eight ? 16 : 0) | (vec ? 32 : 0) | at << 8);
            t.key = op == kStep ? aw_mix(set_keys[set] + (uint32_t)row[7]) : 0u;
            t.pad = 0;
            blocks += b;
        }
        if (a.n == 0) continue;
        a.clip = clip;
        a.chunk = chunk;
        a.out_dtype = out_dtype;
        const dim3 grid((unsigned)blocks), block(kAwThreads);
        if (op == kStep && past == 2)
            hipLaunchKernelGGL((k_adamw<2>), grid, block, 0, stream, a);
        else if (op == kStep && past == 1)
            hipLaunchKernelGGL((k_adamw<1>), grid, block, 0, stream, a);
        else if (op == kStep)
            hipLaunchKernelGGL((k_adamw<0>), grid, block, 0, stream, a);
        else if (op == kPack)
            hipLaunchKernelGGL(k_adamw_pack, grid, block, 0, stream, a);
        else
            hipLaunchKernelGGL(k_adamw_unpack, grid, block, 0, stream, a);
        if (hipGetLastError() != hipSuccess) return CS_ERR_HIP;
    }
    return CS_OK;
}

}  // namespace

extern "C" int cs_adamw_step(int32_t ntensors, const int64_t* table, int32_t nsets,
                             const float* sets, const uint32_t* keys, const float* clip,
                             hipStream_t stream) {
    return aw_run(kStep, ntensors, table, nsets, sets, keys, clip, kF32, stream);
}

extern "C" int cs_adamw_pack_state(int32_t ntensors, const int64_t* table, hipStream_t stream) {
    return aw_run(kPack, ntensors, table, 0, nullptr, nullptr, nullptr, kF32, stream);
}

extern "C" int cs_adamw_unpack_state(int32_t ntensors, const int64_t* table, int32_t out_dtype,
                                     hipStream_t stream) {
    return aw_run(kUnpack, ntensors, table, 0, nullptr, nullptr, nullptr, out_dtype, stream);
}

extern "C" int cs_grad_norm(int32_t ntensors, const int64_t* table, double max_norm,
                            double* partials, float* out, hipStream_t stream) {
    if (ntensors < 0 || (ntensors > 0 && !table) || !partials || !out || !(max_norm >= 0.0))
        return CS_ERR_ARGS;
    int64_t total = 0;
    for (int k = 0; k < ntensors; ++k) {
        const int64_t* row = table + 8 * (int64_t)k;
        if (row[5] < 0 || row[5] > (int64_t)1 << 48 || (row[6] & 0xF) > kF16 ||
            (row[5] > 0 && !row[1]))
            return CS_ERR_ARGS;
        total += row[5];
    }
    // Each tensor ends with a part of a chunk, so the blocks are at most
    // kNormBlocks and one a tensor.
    const int64_t chunk = aw_chunk(total, kNormBlocks, kNormPass);
    int k = 0;
    int64_t done = 0;
    while (k < ntensors) {
        NormArgs a;
        a.n = 0;
        int64_t blocks = 0;
        for (; k < ntensors && a.n < kNormMaxTensors; ++k) {
            const int64_t* row = table + 8 * (int64_t)k;
            if (row[5] == 0) continue;
            NormTensor& t = a.t[a.n++];
            t.grad = (const void*)row[1];
            t.n = row[5];
            t.first_block = (uint32_t)blocks;
            t.meta = (uint32_t)(row[6] & 0xF) | (aw_aligned((void*)row[1], 16) ? 32u : 0u);
            blocks += (row[5] + chunk - 1) / chunk;
        }
        if (a.n == 0) break;
        a.partials = partials + done;
        a.chunk = chunk;
        hipLaunchKernelGGL(k_grad_squares, dim3((unsigned)blocks), dim3(kAwThreads), 0, stream, a);
        if (hipGetLastError() != hipSuccess) return CS_ERR_HIP;
        done += blocks;
    }
    hipLaunchKernelGGL(k_grad_norm, dim3(1), dim3(kAwThreads), 0, stream, partials, (int32_t)done,
                       (float)max_norm, out);
    return hipGetLastError() == hipSuccess ? CS_OK : CS_ERR_HIP;
}
