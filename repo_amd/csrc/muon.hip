// Orthogonalising matrices by Newton-Schulz steps, and the Muon step on them.
//
// X of m rows and n >= m columns (transposed otherwise), scaled to a Frobenius norm of
// one, takes `steps` steps of the odd polynomial a s + b s^3 + c s^5 on its singular
// values:  A = X X^T,  P = a I + b A + c A^2,  X <- P X.
//
// Within a phase of several steps X itself need not move: A <- P A P and Q <- P Q, and
// X <- Q X at the phase's end.  All of these are polynomials of one symmetric matrix, so
// they commute and are symmetric: half of each product is computed and mirrored.  A step
// then costs 4 m^3 instead of 3 m^2 n + m^3.  A's rounding grows by a^2 a step where
// singular values are small (X's own by a), so a phase ends after three steps: relative
// to float64, 1.0 to 1.4 times the error of the steps on X (fp32 products, spectra flat
// to 1 / k^2), where one phase of five steps has 5 to 80 times.
//
// Products.  A value v is held as two halves of 16 bits, h = fp16(v 2^e) and l =
// fp16(v 2^e - h), together 23 bits of v where h is normal: as much as fp32 has.  A
// product is h h' + h l' + l h' on the matrix cores, summed in fp32 (l l' lies 2^-24
// below).  The exponents e come from bounds of the singular values that the host
// computes from the coefficients alone, so that nothing leaves fp16's range.
// A "pair" matrix holds, for 32 values of a row, their 32 h and then their 32 l (128
// bytes), and is padded with zeros to whole tiles.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <memory>
#include <new>

#include "../../include/cubicsplat_hip.h"

namespace {

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };

constexpr int kMuMaxEntries = 20;  // of one chunk: a launch has at most two jobs of each
constexpr int kMuMaxJobs = 2 * kMuMaxEntries;
constexpr int kMuTile = 128;
constexpr int kMuThreads = 256;
constexpr int kMuPatch = 64;       // of the launch that makes pairs
constexpr int kMuParts = 256;      // partial sums of a matrix's norm
constexpr int kMuPass = 2048;
constexpr int kMuPhase = 3;        // steps of a phase
constexpr int kMuMaxSteps = 64;
constexpr int64_t kMuMaxPatches = CS_MUON_MAX_PATCHES;
static_assert(kMuMaxPatches * kMuMaxEntries * kMuThreads < ((int64_t)1 << 32), "a launch's threads");

typedef _Float16 Half8 __attribute__((ext_vector_type(8)));
typedef _Float16 Half4 __attribute__((ext_vector_type(4)));
typedef float Float4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ products

enum { kGram = 0, kPoly = 1, kApply = 2 };

// out[i][j] = scale * sum_k left[i][k] right[j][k] (+ poly_b A_ij + poly_a (i == j)).
// Offsets are in halves from the workspace's beginning; matrix b of a stack lies
// b * stride further.
struct MuJob {
    int64_t left, right, out, other, stride;
    int32_t k;            // padded, in values
    int32_t rows, cols;   // of tiles; cols 0: symmetric, the lower triangle's tiles
    int32_t ld_out, ld_other;
    uint32_t first;       // workgroup
    int32_t tiles;        // of a matrix
    int32_t mode;
    int32_t m;
    float scale, poly_a, poly_b;
};

struct MuJobs {
    MuJob j[kMuMaxJobs];
    _Float16* ws;
    int32_t n;
};
static_assert(sizeof(MuJobs) <= 4096, "kernel arguments");

// Where the last product goes: y of a type, or the Muon step on fp32 weights.
struct MuLast {
    MuJob job;
    void* out;            // y or the parameter
    float* master;        // Muon: fp32 weights of a 16-bit parameter
    int64_t out_stride;   // of a stack, in elements
    int32_t rows, cols;   // of out, as it lies in memory
    int32_t tall;         // out is n x m
    int32_t dtype, muon;
    float decay, lr;
    int32_t pad;
};

struct MuLasts {
    MuLast j[kMuMaxEntries];
    _Float16* ws;
    int32_t n;
};
static_assert(sizeof(MuLasts) <= 4096, "kernel arguments");

template <typename J>
__device__ inline int mu_find(const J& jobs, int n, uint32_t (*first)(const J&, int)) {
    const int lane = threadIdx.x & 63;
    const bool mine = lane < n && first(jobs, lane < n ? lane : 0) <= blockIdx.x;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine)) - 1);
}

__device__ inline void mu_split(float v, _Float16* h, _Float16* l) {
    *h = (_Float16)v;
    *l = (_Float16)(v - (float)*h);
}

// Where value j of a row of a pair matrix has its h; its l lies 32 halves further.
__device__ inline int64_t mu_at(int64_t row, int ld, int j) {
    return row * 2 * ld + (j >> 5) * 64 + (j & 31);
}

// Tile t of the lower triangle: row r >= column c.
__device__ inline void mu_triangle(int t, int* r, int* c) {
    int i = (int)((__builtin_sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    while (i * (i + 1) / 2 > t) --i;
    *r = i;
    *c = t - i * (i + 1) / 2;
}

__device__ inline void mu_to_lds(const _Float16* from, char* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// One tile's sums.  A fragment (16 rows, 32 values, h or l) lies in LDS in its lanes'
// order: lane r + 16 q holds row r's values 8 q to 8 q + 7.  acc[i][j] of wave (w >> 1, w & 1):
// lane's left row 16 i + (lane & 15), right rows 16 j + 4 (lane >> 4) + 0..3.
__device__ inline void mu_tile(const _Float16* left, const _Float16* right, int k, char* lds,
                               Float4 (&acc)[4][4]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t ld = 2 * (int64_t)k;
    // Waves 0 and 1 bring the left rows, 2 and 3 the right: 4 blocks of 16 each.
    const _Float16* from = (wave < 2 ? left : right) +
                           ((wave & 1) * 64 + (lane & 15)) * ld + (lane >> 4) * 8;
    char* to = lds + wave * 8192;
    const int stages = k >> 5;
    auto bring = [&](int s) {
        char* at = to + (s & 1) * 32768;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int p = 0; p < 2; ++p)
                mu_to_lds(from + i * 16 * ld + (int64_t)s * 64 + p * 32, at + (i * 2 + p) * 1024);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = Float4{0.0f, 0.0f, 0.0f, 0.0f};
    bring(0);
    for (int s = 0; s < stages; ++s) {
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();   // this stage is there, and the last one read
        if (s + 1 < stages) bring(s + 1);
        const char* at = lds + (s & 1) * 32768;
        const char* a = at + (wave >> 1) * 8192 + lane * 16;
        const char* b = at + 16384 + (wave & 1) * 8192 + lane * 16;
        Half8 ah[4], al[4], bh[4], bl[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ah[i] = *(const Half8*)(a + i * 2048);
            al[i] = *(const Half8*)(a + i * 2048 + 1024);
            bh[i] = *(const Half8*)(b + i * 2048);
            bl[i] = *(const Half8*)(b + i * 2048 + 1024);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bl[j], ah[i], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], al[i], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bh[j], ah[i], acc[i][j], 0, 0, 0);
    }
}

__device__ inline uint32_t mu_first_job(const MuJobs& a, int k) { return a.j[k].first; }
__device__ inline uint32_t mu_first_last(const MuLasts& a, int k) { return a.j[k].job.first; }

__global__ __launch_bounds__(kMuThreads, 2) void k_mu_product(MuJobs a) {
    __shared__ __attribute__((aligned(16))) char lds[65536];
    const MuJob& job = a.j[mu_find(a, a.n, mu_first_job)];
    const uint32_t at = blockIdx.x - job.first;
    const int b = at / job.tiles, t = at - b * job.tiles;
    int ti, tj;
    if (job.cols == 0) {
        mu_triangle(t, &ti, &tj);
    } else {
        ti = t / job.cols;
        tj = t - ti * job.cols;
    }
    _Float16* ws = a.ws + b * job.stride;
    const int64_t ld = 2 * (int64_t)job.k;
    Float4 acc[4][4];
    mu_tile(ws + job.left + ti * kMuTile * ld, ws + job.right + tj * kMuTile * ld, job.k, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row0 = ti * kMuTile + (wave >> 1) * 64 + (lane & 15);
    const int col0 = tj * kMuTile + (wave & 1) * 64 + (lane >> 4) * 4;
    // The mirrored tile of a symmetric product; X beside its transpose.
    const bool mirror = job.cols == 0 ? ti != tj : job.other >= 0;
    const int64_t mirrored = job.cols == 0 ? job.out : job.other;
    const int ld_mirrored = job.cols == 0 ? job.ld_out : job.ld_other;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row0 + 16 * i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = col0 + 16 * j;
            const int64_t o = mu_at(row, job.ld_out, col);
            Float4 v = acc[i][j] * job.scale;
            if (job.mode == kPoly) {
                const Half4 h = *(const Half4*)(ws + job.other + o);
                const Half4 l = *(const Half4*)(ws + job.other + o + 32);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] += job.poly_b * ((float)h[e] + (float)l[e]);
                    if (row == col + e && row < job.m) v[e] += job.poly_a;
                }
            }
            Half4 h, l;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                _Float16 x, y;
                mu_split(v[e], &x, &y);
                h[e] = x;
                l[e] = y;
            }
            *(Half4*)(ws + job.out + o) = h;
            *(Half4*)(ws + job.out + o + 32) = l;
            if (mirror) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t q = mirrored + mu_at(col + e, ld_mirrored, row);
                    ws[q] = h[e];
                    ws[q + 32] = l[e];
                }
            }
        }
    }
}

__device__ inline void mu_put(void* p, int dtype, int64_t at, float v) {
    if (dtype == kF32) ((float*)p)[at] = v;
    else if (dtype == kBF16) ((__bf16*)p)[at] = (__bf16)v;
    else ((_Float16*)p)[at] = (_Float16)v;
}

__device__ inline float mu_get(const void* p, int dtype, int64_t at) {
    if (dtype == kF32) return ((const float*)p)[at];
    if (dtype == kBF16) return (float)((const __bf16*)p)[at];
    return (float)((const _Float16*)p)[at];
}

// The last X, into y or the weights.
__global__ __launch_bounds__(kMuThreads, 2) void k_mu_last(MuLasts a) {
    __shared__ __attribute__((aligned(16))) char lds[65536];
    const MuLast& l = a.j[mu_find(a, a.n, mu_first_last)];
    const MuJob& job = l.job;
    const uint32_t at = blockIdx.x - job.first;
    const int b = at / job.tiles, t = at - b * job.tiles;
    const int ti = t / job.cols, tj = t - ti * job.cols;
    const _Float16* ws = a.ws + b * job.stride;
    const int64_t ld = 2 * (int64_t)job.k;
    Float4 acc[4][4];
    mu_tile(ws + job.left + ti * kMuTile * ld, ws + job.right + tj * kMuTile * ld, job.k, lds, acc);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row0 = ti * kMuTile + (wave >> 1) * 64 + (lane & 15);
    const int col0 = tj * kMuTile + (wave & 1) * 64 + (lane >> 4) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // Row `row0 + 16 i` of X's transpose.
                const int r = l.tall ? row0 + 16 * i : col0 + 16 * j + e;
                const int c = l.tall ? col0 + 16 * j + e : row0 + 16 * i;
                if (r >= l.rows || c >= l.cols) continue;
                const int64_t o = b * l.out_stride + (int64_t)r * l.cols + c;
                const float v = acc[i][j][e] * job.scale;
                if (!l.muon) {
                    mu_put(l.out, l.dtype, o, v);
                    continue;
                }
                float* w = l.dtype == kF32 ? (float*)l.out : l.master;
                const float moved = __builtin_fmaf(-l.lr, v, w[o] * l.decay);
                w[o] = moved;
                if (l.dtype != kF32) mu_put(l.out, l.dtype, o, moved);
            }
}

// ------------------------------------------------------- what goes into them

// A matrix, or a stack of them, as it lies in memory.  momentum: the Muon step's, and x
// is its gradient.
struct MuSource {
    const void* x;
    float* momentum;
    double* parts;         // [count][kMuParts]
    int64_t x_stride;      // of a stack, in elements
    int64_t pairs, flipped; // offsets of X and its transpose, or the other way round: pairs in
                           // the source's orientation
    int64_t stride;        // of a stack, in halves
    int64_t chunk;         // elements of a partial sum
    int32_t rows, cols;
    int32_t padded_rows, padded_cols;
    uint32_t first_sum, first_patch;
    int32_t nparts, patches, patch_cols;
    int32_t dtype;
    float mix, look;       // momentum: m += mix (g - m), u = m + look (g - m)
};

struct MuSources {
    MuSource s[kMuMaxEntries];
    _Float16* ws;
    double eps;
    float scale;
    int32_t n;
};
static_assert(sizeof(MuSources) <= 4096, "kernel arguments");

__device__ inline uint32_t mu_first_sum(const MuSources& a, int k) { return a.s[k].first_sum; }
__device__ inline uint32_t mu_first_patch(const MuSources& a, int k) { return a.s[k].first_patch; }

// u - the update before orthogonalising - from a gradient and the moved momentum.
__device__ inline float mu_update(float g, float m, float look) {
    return __builtin_fmaf(look, g - m, m);
}

// The momentum's move, and partial sums of the squares of each matrix, in fp64.
__global__ __launch_bounds__(kMuThreads) void k_mu_sums(MuSources a) {
    __shared__ double lds[kMuThreads / 64];
    const MuSource& s = a.s[mu_find(a, a.n, mu_first_sum)];
    const uint32_t at = blockIdx.x - s.first_sum;
    const int b = at / s.nparts, part = at - b * s.nparts;
    const int64_t size = (int64_t)s.rows * s.cols, from = part * s.chunk;
    const int64_t to = from + s.chunk < size ? from + s.chunk : size;
    double sum = 0.0;
    for (int64_t i = from + threadIdx.x; i < to; i += kMuThreads) {
        float u = mu_get(s.x, s.dtype, b * s.x_stride + i);
        if (s.momentum) {
            float m = s.momentum[i];
            m = __builtin_fmaf(s.mix, u - m, m);
            s.momentum[i] = m;
            u = mu_update(u, m, s.look);
        }
        sum = __builtin_fma((double)u, (double)u, sum);
    }
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kMuThreads / 64; ++w) sum += lds[w];
        s.parts[(int64_t)b * kMuParts + part] = sum;
    }
}

// X and its transpose as pairs, scaled to a norm of one (times 2^e), patch by patch.
__global__ __launch_bounds__(kMuThreads) void k_mu_pairs(MuSources a) {
    __shared__ float tile[kMuPatch][kMuPatch + 1];
    __shared__ double lds[kMuThreads / 64];
    const MuSource& s = a.s[mu_find(a, a.n, mu_first_patch)];
    const uint32_t at = blockIdx.x - s.first_patch;
    const int b = at / s.patches, t = at - b * s.patches;
    const int r0 = t / s.patch_cols * kMuPatch, c0 = t % s.patch_cols * kMuPatch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    static_assert(kMuParts == kMuThreads, "one partial sum a thread");
    double sum = (int)threadIdx.x < s.nparts ? s.parts[(int64_t)b * kMuParts + threadIdx.x] : 0.0;
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
    if (lane == 0) lds[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kMuThreads / 64; ++w) sum += lds[w];
    const double norm = sqrt(sum);
    const double by = (double)a.scale / (norm < a.eps ? a.eps : norm);   // NaN stays
    const int c = c0 + lane;
    for (int r = wave; r < kMuPatch; r += kMuThreads / 64) {
        float u = 0.0f;
        if (r0 + r < s.rows && c < s.cols) {
            const int64_t i = (int64_t)(r0 + r) * s.cols + c;
            u = mu_get(s.x, s.dtype, b * s.x_stride + i);
            if (s.momentum) u = mu_update(u, s.momentum[i], s.look);
            u = (float)((double)u * by);
        }
        tile[r][lane] = u;
    }
    __syncthreads();
    _Float16* ws = a.ws + b * s.stride;
    for (int r = wave; r < kMuPatch; r += kMuThreads / 64) {
        _Float16 h, l;
        if (r0 + r < s.padded_rows) {
            mu_split(tile[r][lane], &h, &l);
            const int64_t o = s.pairs + mu_at(r0 + r, s.padded_cols, c);
            ws[o] = h;
            ws[o + 32] = l;
        }
        if (c0 + r < s.padded_cols) {
            mu_split(tile[lane][r], &h, &l);
            const int64_t o = s.flipped + mu_at(c0 + r, s.padded_rows, r0 + lane);
            ws[o] = h;
            ws[o + 32] = l;
        }
    }
}

// ---------------------------------------------------------------------- host

// Coefficients, and bounds of the singular values before each step, from which the
// exponents follow.
struct MuPlan {
    int steps, phase;
    double a, b, c;
    double x[kMuMaxSteps + 1];
};

double mu_poly(const MuPlan& p, double s) { return p.a + s * s * (p.b + s * s * p.c); }

// max over [0, s] of |P(t^2)|, or of |t P(t^2)|: at the ends or where the slope is zero.
double mu_bound(const MuPlan& p, double s, bool odd) {
    double at[4] = {0.0, s, 0.0, 0.0};
    const double qa = odd ? 5.0 * p.c : 0.0, qb = odd ? 3.0 * p.b : 2.0 * p.c,
                 qc = odd ? p.a : p.b;
    if (qa != 0.0) {
        const double root = sqrt(std::max(0.0, qb * qb - 4.0 * qa * qc));
        at[2] = (-qb + root) / (2.0 * qa);
        at[3] = (-qb - root) / (2.0 * qa);
    } else if (qb != 0.0) {
        at[2] = -qc / qb;
    }
    double most = 0.0;
    for (int i = 0; i < 4; ++i) {
        const double t = i < 2 ? at[i] : at[i] > 0.0 ? std::min(s, sqrt(at[i])) : 0.0;
        most = std::max(most, fabs(mu_poly(p, t)) * (odd ? t : 1.0));
    }
    return most * 1.01;   // the steps' own roundings
}

// What is below `bound` is held times 2^e: below 2^14, where fp16 ends at 2^16.
int mu_exponent(double bound) { return 14 - (int)ceil(log2(std::max(bound, 1e-3))); }

bool mu_plan(MuPlan* p, int steps, double a, double b, double c) {
    if (steps < 1 || steps > kMuMaxSteps || !(fabs(a) <= 64.0) || !(fabs(b) <= 64.0) ||
        !(fabs(c) <= 64.0))
        return false;
    *p = MuPlan{steps, 1, a, b, c, {1.01}};
    for (int k = 0; k < steps; ++k) {
        p->x[k + 1] = mu_bound(*p, p->x[k], true);
        if (!(p->x[k + 1] <= 64.0)) return false;   // values that grow without end
    }
    // The rounding of A grows by a^2 a step of a phase.
    while (p->phase < kMuPhase && pow(fabs(a), 2.0 * p->phase) <= 200.0) ++p->phase;
    return true;
}

struct MuEntry {
    const void* x;
    void* out;
    float *master, *momentum;
    int64_t count, rows, cols;   // as they lie in memory
    int dtype;
    float decay, lr, mix, look;

    bool tall;
    int64_t m, n, mp, np;        // m <= n, and padded
    int phase;
    int64_t base, stride;        // halves
    int64_t X, XT[2], A, T, P, Q[2];
};

int64_t mu_round(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// The products of one matrix by steps on X, or by phases, in m^3.
double mu_cost(int steps, int phase, double ratio) {
    double cost = 0.0;
    for (int k = 0; k < steps; k += phase) {
        const int len = std::min(phase, steps - k);
        cost += 3.0 * ratio + 4.0 * len - 3.0;
    }
    return cost;
}

// Where an entry's matrices lie; their size in halves.
int64_t mu_layout(MuEntry* e, const MuPlan& p, int64_t base) {
    e->tall = e->rows > e->cols;
    e->m = e->tall ? e->cols : e->rows;
    e->n = e->tall ? e->rows : e->cols;
    e->mp = mu_round(e->m, kMuTile);
    e->np = mu_round(e->n, kMuTile);
    const double ratio = (double)e->np / (double)e->mp;
    e->phase = mu_cost(p.steps, p.phase, ratio) < mu_cost(p.steps, 1, ratio) ? p.phase : 1;
    const int64_t wide = 2 * e->mp * e->np, square = 2 * e->mp * e->mp;
    int64_t at = 0;
    auto take = [&](int64_t size) { const int64_t o = base + at; at += size; return o; };
    e->X = take(wide);
    e->XT[0] = take(wide);
    e->XT[1] = e->phase < p.steps ? take(wide) : -1;
    e->A = take(square);
    e->Q[0] = take(square);
    if (e->phase > 1) {
        e->T = take(square);
        e->P = take(square);
        e->Q[1] = take(square);
    }
    e->base = base;
    e->stride = at;
    return at * e->count;
}

int64_t mu_chunk_bytes(MuEntry* e, int n, const MuPlan& p) {
    int64_t halves = 0, parts = 0;
    for (int k = 0; k < n; ++k) {
        halves += mu_layout(e + k, p, halves);
        parts += e[k].count * kMuParts;
    }
    return halves * 2 + parts * 8;
}

struct MuOp { MuJob job; int slot; };

// The products of an entry, each with the launch that it goes into (up to two of them a launch),
// without the last.
struct MuSchedule {
    MuOp ops[8 * kMuMaxSteps];
    int n = 0, slots = 0;
    MuJob last;

    void make(const MuEntry& e, const MuPlan& p) {
        n = slots = 0;
        const double xs = p.x[0];
        int ex = mu_exponent(xs), xt = 0;
        for (int k = 0; k < p.steps; k += e.phase) {
            const int len = std::min(e.phase, p.steps - k);
            int ea = mu_exponent(p.x[k] * p.x[k]), eq = 0, q = 0;
            double pq = 1.0;
            sym(e, e.X, e.X, e.A, e.np, ea - 2 * ex);
            ++slots;
            for (int i = 0; i < len; ++i) {
                const double x = p.x[k + i], bound = mu_bound(p, x, false);
                const int ep = mu_exponent(bound);
                const int64_t P = i == 0 ? e.Q[0] : e.P;
                MuJob* j = sym(e, e.A, e.A, P, e.mp, 0);
                j->mode = kPoly;
                j->other = e.A;
                j->scale = (float)ldexp(p.c, ep - 2 * ea);
                j->poly_b = (float)ldexp(p.b, ep - ea);
                j->poly_a = (float)ldexp(p.a, ep);
                ++slots;
                pq *= bound;
                const int next = mu_exponent(pq);
                if (i == 0) eq = ep;
                const bool more = i + 1 < len;
                const int et = mu_exponent(x * x * bound);
                if (i > 0) {
                    sym(e, P, e.Q[q], e.Q[q ^ 1], e.mp, next - ep - eq);
                    q ^= 1;
                    eq = next;
                }
                if (more) sym(e, P, e.A, e.T, e.mp, et - ep - ea);
                if (i > 0 || more) ++slots;
                if (more) {
                    const int ea2 = mu_exponent(p.x[k + i + 1] * p.x[k + i + 1]);
                    sym(e, P, e.T, e.A, e.mp, ea2 - ep - et);
                    ea = ea2;
                    ++slots;
                }
            }
            const bool end = k + e.phase >= p.steps;
            const int ex2 = end ? 0 : mu_exponent(p.x[k + len]);
            MuJob j = job(e, e.XT[xt], e.Q[q], e.mp, ex2 - ex - eq);
            j.mode = kApply;
            j.rows = (int32_t)(e.np / kMuTile);
            j.cols = (int32_t)(e.mp / kMuTile);
            j.tiles = j.rows * j.cols;
            j.ld_out = (int32_t)e.mp;
            j.ld_other = (int32_t)e.np;
            if (end) {
                last = j;
                return;
            }
            j.out = e.XT[xt ^ 1];
            j.other = e.X;
            ops[n++] = MuOp{j, slots++};
            xt ^= 1;
            ex = ex2;
        }
    }

  private:
    static MuJob job(const MuEntry& e, int64_t left, int64_t right, int64_t k, int exponent) {
        MuJob j{};
        j.left = left;
        j.right = right;
        j.stride = e.stride;
        j.k = (int32_t)k;
        j.m = (int32_t)e.m;
        j.scale = (float)ldexp(1.0, exponent);
        return j;
    }

    MuJob* sym(const MuEntry& e, int64_t left, int64_t right, int64_t out, int64_t k,
               int exponent) {
        MuJob j = job(e, left, right, k, exponent);
        const int t = (int)(e.mp / kMuTile);
        j.out = out;
        j.tiles = t * (t + 1) / 2;
        j.ld_out = (int32_t)e.mp;
        ops[n] = MuOp{j, slots};
        return &ops[n++].job;
    }
};

bool mu_launched() { return hipGetLastError() == hipSuccess; }

int mu_chunk(MuEntry* e, int n, const MuPlan& p, double eps, void* workspace, MuSchedule* sched,
             hipStream_t stream) {
    MuSources src{};
    src.ws = (_Float16*)workspace;
    src.eps = eps;
    src.scale = (float)ldexp(1.0, mu_exponent(p.x[0]));
    src.n = n;
    int64_t sums = 0, patches = 0, halves = 0;
    for (int k = 0; k < n; ++k) halves += e[k].stride * e[k].count;
    double* parts = (double*)((char*)workspace + halves * 2);
    int slots = 0;
    for (int k = 0; k < n; ++k) {
        MuSource& s = src.s[k];
        const int64_t size = e[k].rows * e[k].cols;
        s.x = e[k].x;
        s.momentum = e[k].momentum;
        s.parts = parts;
        parts += e[k].count * kMuParts;
        s.x_stride = size;
        s.pairs = e[k].tall ? e[k].XT[0] : e[k].X;
        s.flipped = e[k].tall ? e[k].X : e[k].XT[0];
        s.stride = e[k].stride;
        s.chunk = mu_round((size + kMuParts - 1) / kMuParts, kMuPass);
        s.nparts = (int32_t)((size + s.chunk - 1) / s.chunk);
        s.rows = (int32_t)e[k].rows;
        s.cols = (int32_t)e[k].cols;
        s.padded_rows = (int32_t)(e[k].tall ? e[k].np : e[k].mp);
        s.padded_cols = (int32_t)(e[k].tall ? e[k].mp : e[k].np);
        s.patch_cols = s.padded_cols / kMuPatch;
        s.patches = s.padded_rows / kMuPatch * s.patch_cols;
        s.dtype = e[k].dtype;
        s.mix = e[k].mix;
        s.look = e[k].look;
        s.first_sum = (uint32_t)sums;
        s.first_patch = (uint32_t)patches;
        sums += s.nparts * e[k].count;
        patches += s.patches * e[k].count;
        sched[k].make(e[k], p);
        slots = std::max(slots, sched[k].slots);
    }
    const dim3 block(kMuThreads);
    hipLaunchKernelGGL(k_mu_sums, dim3((unsigned)sums), block, 0, stream, src);
    if (!mu_launched()) return CS_ERR_HIP;
    hipLaunchKernelGGL(k_mu_pairs, dim3((unsigned)patches), block, 0, stream, src);
    if (!mu_launched()) return CS_ERR_HIP;
    int at[kMuMaxEntries] = {};
    for (int slot = 0; slot < slots; ++slot) {
        MuJobs a{};
        a.ws = (_Float16*)workspace;
        int64_t blocks = 0;
        for (int k = 0; k < n; ++k)
            for (; at[k] < sched[k].n && sched[k].ops[at[k]].slot == slot; ++at[k]) {
                MuJob& j = a.j[a.n++];
                j = sched[k].ops[at[k]].job;
                if (j.mode != kApply) j.cols = 0;
                j.first = (uint32_t)blocks;
                blocks += j.tiles * e[k].count;
            }
        hipLaunchKernelGGL(k_mu_product, dim3((unsigned)blocks), block, 0, stream, a);
        if (!mu_launched()) return CS_ERR_HIP;
    }
    MuLasts l{};
    l.ws = (_Float16*)workspace;
    l.n = n;
    int64_t blocks = 0;
    for (int k = 0; k < n; ++k) {
        MuLast& y = l.j[k];
        y.job = sched[k].last;
        y.job.first = (uint32_t)blocks;
        blocks += y.job.tiles * e[k].count;
        y.out = e[k].out;
        y.master = e[k].master;
        y.out_stride = e[k].rows * e[k].cols;
        y.rows = (int32_t)e[k].rows;
        y.cols = (int32_t)e[k].cols;
        y.tall = e[k].tall;
        y.dtype = e[k].dtype;
        y.muon = e[k].momentum != nullptr;
        y.decay = e[k].decay;
        y.lr = e[k].lr;
    }
    hipLaunchKernelGGL(k_mu_last, dim3((unsigned)blocks), block, 0, stream, l);
    return mu_launched() ? CS_OK : CS_ERR_HIP;
}

// Rows of the tables, checked: how many entries have anything, or -1.
int mu_entries(int32_t ntensors, const int64_t* table, const float* scalars, bool muon,
               MuEntry* e) {
    int n = 0;
    for (int k = 0; k < ntensors; ++k) {
        const int64_t* row = table + 8 * (int64_t)k;
        MuEntry& x = e[n];
        x = MuEntry{};
        x.count = muon ? 1 : row[2];
        x.rows = row[4];
        x.cols = row[5];
        x.dtype = (int)row[6];
        const int64_t most = (int64_t)1 << 22;
        if (x.count < 0 || x.rows < 0 || x.cols < 0 || x.rows > most || x.cols > most ||
            x.count > most || x.dtype < kF32 || x.dtype > kF16)
            return -1;
        if (x.count == 0 || x.rows == 0 || x.cols == 0) continue;
        // A launch has fewer than 2^32 threads.
        const int64_t rt = mu_round(x.rows, kMuTile) / kMuPatch,
                      ct = mu_round(x.cols, kMuTile) / kMuPatch;
        if (x.count * rt > kMuMaxPatches / ct) return -1;
        if (!row[0] || !row[1]) return -1;
        if (muon) {
            x.x = (const void*)row[1];
            x.out = (void*)row[0];
            x.master = (float*)row[2];
            x.momentum = (float*)row[3];
            if (!x.momentum || (x.dtype != kF32 && !x.master)) return -1;
            const float* f = scalars + 4 * (int64_t)k;
            x.decay = f[0];
            x.lr = f[1];
            x.mix = f[2];
            x.look = f[3];
        } else {
            x.x = (const void*)row[0];
            x.out = (void*)row[1];
        }
        ++n;
    }
    return n;
}

int mu_run(int32_t ntensors, const int64_t* table, const float* scalars, bool muon, int32_t steps,
           double a, double b, double c, double eps, void* workspace, int64_t* bytes,
           hipStream_t stream) {
    MuPlan p;
    if (ntensors < 0 || (ntensors > 0 && (!table || (muon && !scalars))) || !(eps >= 0.0) ||
        !mu_plan(&p, steps, a, b, c))
        return CS_ERR_ARGS;
    if (!bytes && ntensors > 0 && (!workspace || ((uintptr_t)workspace & 127))) return CS_ERR_ARGS;
    std::unique_ptr<MuEntry[]> e(new (std::nothrow) MuEntry[ntensors + 1]);
    std::unique_ptr<MuSchedule[]> sched(bytes ? nullptr
                                              : new (std::nothrow) MuSchedule[kMuMaxEntries]);
    if (!e || (!bytes && !sched)) return CS_ERR_ARGS;
    const int n = mu_entries(ntensors, table, scalars, muon, e.get());
    if (n < 0) return CS_ERR_ARGS;
    for (int k = 0; k < n; ++k) mu_layout(&e[k], p, 0);
    // The longest sums first: they end last.
    std::stable_sort(e.get(), e.get() + n,
                     [](const MuEntry& x, const MuEntry& y) { return x.np > y.np; });
    if (bytes) *bytes = 0;
    for (int k = 0; k < n; k += kMuMaxEntries) {
        const int many = std::min(kMuMaxEntries, n - k);
        const int64_t need = mu_chunk_bytes(&e[k], many, p);
        if (bytes) {
            *bytes = std::max(*bytes, need);
        } else {
            const int rc = mu_chunk(&e[k], many, p, eps, workspace, sched.get(), stream);
            if (rc != CS_OK) return rc;
        }
    }
    return CS_OK;
}

int64_t mu_bytes(int32_t ntensors, const int64_t* table, const float* scalars, bool muon,
                 int32_t steps, double a, double b, double c) {
    int64_t bytes = 0;
    return mu_run(ntensors, table, scalars, muon, steps, a, b, c, 0.0, nullptr, &bytes, nullptr) ==
                   CS_OK ? bytes : -1;
}

}  // namespace

extern "C" int64_t cs_orthogonalize_workspace_bytes(int32_t ntensors, const int64_t* table,
                                                    int32_t steps, double a, double b, double c) {
    return mu_bytes(ntensors, table, nullptr, false, steps, a, b, c);
}

extern "C" int cs_orthogonalize(int32_t ntensors, const int64_t* table, int32_t steps, double a,
                                double b, double c, double eps, void* workspace,
                                hipStream_t stream) {
    return mu_run(ntensors, table, nullptr, false, steps, a, b, c, eps, workspace, nullptr, stream);
}

extern "C" int64_t cs_muon_workspace_bytes(int32_t ntensors, const int64_t* table,
                                           const float* scalars, int32_t steps, double a, double b,
                                           double c) {
    return mu_bytes(ntensors, table, scalars, true, steps, a, b, c);
}

extern "C" int cs_muon_step(int32_t ntensors, const int64_t* table, const float* scalars,
                            int32_t steps, double a, double b, double c, double eps,
                            void* workspace, hipStream_t stream) {
    return mu_run(ntensors, table, scalars, true, steps, a, b, c, eps, workspace, nullptr, stream);
}
