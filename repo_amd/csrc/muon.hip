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
// singular values are small (X's own by a), so phases are of two steps and one in turn for a
// = 3.4445: relative to float64 the result has 0.8 to 1.3 times the error of the steps on X in
// fp32 (spectra flat to 1 / k^2), where phases of three steps have up to 4.7 times and one of
// five up to 100 times.
//
// Products.  A value v is held as two halves of 16 bits, h = fp16(v 2^e) and l =
// fp16(v 2^e - h), together 23 bits of v where h is normal: as much as fp32 has.  A
// product is h h' + h l' + l h' on the matrix cores, summed in fp32 (l l' lies 2^-24
// below).  The exponents e come from bounds of the singular values that the host
// computes from the coefficients alone, so that nothing leaves fp16's range.
// A "pair" matrix holds, for 32 values of a row, their 32 h and then their 32 l (128
// bytes), and is padded with zeros to whole tiles.
//
// Bound: three matrix instructions for each pair of 32 values. Measured (means of a kernel
// trace): a 4096 x 4096 product 1.3 PFLOP/s of fp16 instructions with tiles of 256 (the matrix
// cores are busy 68% of the clock that they leave, 1.8 to 2.05 GHz; an instruction loop without
// operands' traffic reaches 2.3), a symmetric one 191 us and 34 to join its sums, cut in three, 272
// whole.  The 18 matrices of an encoder 256 to 2048 wide take 12.0 ms a step, those of one 64 to 512
// wide 0.6 ms; a matrix of 1021 x 765 185 us, 17 launches of some 11 us, of which loads alone and
// products alone take 9 to 10 each.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <exception>
#include <memory>
#include <vector>

#include "../../include/cubicsplat_hip.h"

namespace {

enum { kF32 = 0, kBF16 = 1, kF16 = 2 };

constexpr int kMuMaxEntries = 20;  // of one chunk: a launch has at most two jobs of each
constexpr int kMuMaxJobs = 2 * kMuMaxEntries;
constexpr int kMuThreads = 256;   // of all launches but the products'
constexpr int kMuPatch = 64;       // of the launch that makes pairs
constexpr int kMuParts = 256;      // partial sums of a matrix's norm
constexpr int kMuPass = 2048;
constexpr int kMuPhase = 3;        // most steps of a phase
constexpr int kMuUnit = 4096;      // halves, or floats of partial sums, that offsets count
constexpr int kMuMaxSteps = 64;
constexpr int kMuMostTile = 256;
constexpr int64_t kMuMaxPatches = CS_MUON_MAX_PATCHES;
static_assert(kMuMaxPatches * kMuMaxEntries * 512 < ((int64_t)1 << 32), "a launch's threads");

typedef _Float16 Half8 __attribute__((ext_vector_type(8)));
typedef _Float16 Half4 __attribute__((ext_vector_type(4)));
typedef float Float4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ products

enum { kGram = 0, kPoly = 1, kApply = 2 };

// out[i][j] = scale * sum_k left[i][k] right[j][k] (+ poly_b A_ij + poly_a (i == j)), A at
// `other`.  Offsets are from the workspace's beginning, in units; matrix b of a stack lies
// b * stride further.  A sum over a long k is cut into pieces, whose partial sums a launch
// of its own joins.
struct MuJob {
    int32_t left, right, out, other, stride;
    int32_t partial;      // pieces > 1: [matrix][tile][piece][T][T] floats
    int32_t pieces, piece_stages;
    int32_t k;            // padded, in values
    int32_t cols;         // of tiles; 0: symmetric, the lower triangle's tiles
    int32_t ld_out, ld_other;
    uint32_t first;       // workgroup
    int32_t tiles;        // of a matrix
    int32_t mode, m;
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
    int32_t rows, cols;   // of out, as it lies in memory
    void* out;            // y or the parameter
    float* master;        // Muon: fp32 weights of a 16-bit parameter
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

// Tiles of T x T by WR x WC waves, each of I x J blocks of 16 x 16; a stage brings 32 KS
// values of k of every row, and ST stages are there or on their way.  KW groups of such waves
// share a stage's k: a tile of 64 mostly has a CU to itself, where one group waits for its own
// reads (a stage of one took 0.63 us, 1021 x 765 219 us).
template <int TILE> struct MuShape;
template <> struct MuShape<256> { enum { T = 256, WR = 2, WC = 4, KS = 1, KW = 1, ST = 2 }; };
template <> struct MuShape<128> { enum { T = 128, WR = 2, WC = 2, KS = 1, KW = 1, ST = 2 }; };
template <> struct MuShape<64> { enum { T = 64, WR = 2, WC = 2, KS = 2, KW = 2, ST = 3 }; };

template <typename S> struct MuSizes {
    enum {
        kGroup = S::WR * S::WC,
        kWaves = kGroup * S::KW,
        kThreads = kWaves * 64,
        I = S::T / S::WR / 16,
        J = S::T / S::WC / 16,
        kSide = S::T / 16 * S::KS * 2048,   // bytes of a stage's left or right rows
        kStage = 2 * kSide,
        kLds = kStage * S::ST,
        kBlocks = S::T / 16 / (kWaves / 2),   // of 16 rows, that a wave brings
        kLoads = kBlocks * S::KS * 2
    };
};

template <int N> __device__ inline void mu_wait_barrier() {
    // What this wave has asked for up to its N newest loads is there, and what it reads is read.
    __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
}

__device__ inline Float4 mu_mfma(Half8 a, Half8 b, Float4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// One tile's sums over stages [from, to).  acc[i][j]: the lane's left row 16 i + (lane & 15) of
// its wave's, right rows 16 j + 4 (lane >> 4) + 0..3.  16 rows' 32 values lie in LDS row by row, 128
// bytes each, as in memory, so that eight lanes bring a whole line; a row's eight parts of 16
// bytes change places by its number, so that lanes that read the same part of different rows
// find it in different banks.  (Brought in the order in which lanes read it, 16 bytes here and there,
// a 4096 x 4096 matrix took 6.45 ms for 4.12 with tiles of 128.)
template <typename S>
__device__ inline void mu_tile(const _Float16* left, const _Float16* right, int k, int from, int to,
                               char* lds, Float4 (&acc)[MuSizes<S>::I][MuSizes<S>::J]) {
    typedef MuSizes<S> Z;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t ld = 2 * (int64_t)k;
    // The first half of the waves brings the left rows, the other the right ones.
    const int mine = (wave & (Z::kWaves / 2 - 1)) * Z::kBlocks;
    const _Float16* src = (wave < Z::kWaves / 2 ? left : right) + (mine * 16 + (lane >> 3)) * ld +
                          ((lane & 7) ^ (lane >> 3)) * 8;
    char* dst = lds + (wave < Z::kWaves / 2 ? 0 : Z::kSide) + mine * (S::KS * 2048);
    auto bring = [&](int s, int slot) {
        char* at = dst + slot * Z::kStage;
        const _Float16* p = src + (int64_t)s * (S::KS * 64);
#pragma unroll
        for (int i = 0; i < Z::kBlocks; ++i)
#pragma unroll
            for (int c = 0; c < S::KS * 2; ++c)
                mu_to_lds(p + (i * 16 + (c & 1) * 8) * ld + (c >> 1) * 64,
                          at + (i * S::KS * 2 + c) * 1024);
    };
#pragma unroll
    for (int i = 0; i < Z::I; ++i)
#pragma unroll
        for (int j = 0; j < Z::J; ++j) acc[i][j] = Float4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < S::ST - 1; ++s)
        if (from + s < to) bring(from + s, s);
    const int high = (lane & 15) * 128 + ((lane >> 4) ^ (lane & 7)) * 16, low = high ^ 64;
    const int member = wave & (Z::kGroup - 1);
    const char* a0 = lds + (member / S::WC) * (Z::I * S::KS * 2048);
    const char* b0 = lds + Z::kSide + (member % S::WC) * (Z::J * S::KS * 2048);
    int slot = 0;
    if constexpr (S::KS == 1 && S::ST == 2) {
        // The barrier comes before a step's last blocks, whose operands then are in registers:
        // the next step's first reads go out between their products.
        constexpr int kTail = 3, kMain = Z::I - kTail;
        Half8 bh[Z::J], bl[Z::J], ah[2], al[2], th[kTail], tl[kTail];
        mu_wait_barrier<0>();
        if (from + 1 < to) bring(from + 1, 1);
#pragma unroll
        for (int j = 0; j < Z::J; ++j) {
            bh[j] = *(const Half8*)(b0 + j * 2048 + high);
            bl[j] = *(const Half8*)(b0 + j * 2048 + low);
        }
        ah[0] = *(const Half8*)(a0 + high);
        al[0] = *(const Half8*)(a0 + low);
        for (int s = from; s < to; ++s) {
            const char* a = a0 + slot * Z::kStage;
#pragma unroll
            for (int i = 0; i < kMain; ++i) {
                if (i + 1 < kMain) {
                    ah[(i + 1) & 1] = *(const Half8*)(a + (i + 1) * 2048 + high);
                    al[(i + 1) & 1] = *(const Half8*)(a + (i + 1) * 2048 + low);
                } else {
#pragma unroll
                    for (int t = 0; t < kTail; ++t) {
                        th[t] = *(const Half8*)(a + (kMain + t) * 2048 + high);
                        tl[t] = *(const Half8*)(a + (kMain + t) * 2048 + low);
                    }
                }
#pragma unroll
                for (int j = 0; j < Z::J; ++j)
                    acc[i][j] = mu_mfma(bl[j], ah[i & 1], acc[i][j]);
#pragma unroll
                for (int j = 0; j < Z::J; ++j)
                    acc[i][j] = mu_mfma(bh[j], al[i & 1], acc[i][j]);
#pragma unroll
                for (int j = 0; j < Z::J; ++j)
                    acc[i][j] = mu_mfma(bh[j], ah[i & 1], acc[i][j]);
            }
            __builtin_amdgcn_sched_barrier(0);
            mu_wait_barrier<0>();
            __builtin_amdgcn_sched_barrier(0);
            if (s + 2 < to) bring(s + 2, slot);
            slot ^= 1;
            // Behind the last stage this reads what was there before it, for nothing.
            const char* an = a0 + slot * Z::kStage;
            const char* bn = b0 + slot * Z::kStage;
            ah[0] = *(const Half8*)(an + high);
            al[0] = *(const Half8*)(an + low);
#pragma unroll
            for (int j = 0; j < Z::J; ++j) {
#pragma unroll
                for (int t = 0; t < kTail; ++t)
                    acc[kMain + t][j] = mu_mfma(bl[j], th[t], acc[kMain + t][j]);
#pragma unroll
                for (int t = 0; t < kTail; ++t)
                    acc[kMain + t][j] = mu_mfma(bh[j], tl[t], acc[kMain + t][j]);
#pragma unroll
                for (int t = 0; t < kTail; ++t)
                    acc[kMain + t][j] = mu_mfma(bh[j], th[t], acc[kMain + t][j]);
                bh[j] = *(const Half8*)(bn + j * 2048 + high);
                bl[j] = *(const Half8*)(bn + j * 2048 + low);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        return;
    }
    for (int s = from; s < to; ++s) {
        // This stage is there; the one read last has been read, and is brought anew.
        if (s + S::ST - 1 <= to)
            mu_wait_barrier<(S::ST - 2) * Z::kLoads>();
        else
            mu_wait_barrier<0>();
        if (s + S::ST - 1 < to) bring(s + S::ST - 1, slot == 0 ? S::ST - 1 : slot - 1);
        const char* a = a0 + slot * Z::kStage;
        const char* b = b0 + slot * Z::kStage;
#pragma unroll
        for (int q = 0; q < S::KS / S::KW; ++q) {
            const int c = q * S::KW + wave / Z::kGroup;
            Half8 bh[Z::J], bl[Z::J];
#pragma unroll
            for (int j = 0; j < Z::J; ++j) {
                bh[j] = *(const Half8*)(b + (j * S::KS + c) * 2048 + high);
                bl[j] = *(const Half8*)(b + (j * S::KS + c) * 2048 + low);
            }
            Half8 ah[Z::I], al[Z::I];
#pragma unroll
            for (int i = 0; i < Z::I; ++i) {
                ah[i] = *(const Half8*)(a + (i * S::KS + c) * 2048 + high);
                al[i] = *(const Half8*)(a + (i * S::KS + c) * 2048 + low);
            }
            // A product waits for the last one into its sums: as many others between them as
            // there are.
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int i = 0; i < Z::I; ++i)
#pragma unroll
                    for (int j = 0; j < Z::J; ++j)
                        acc[i][j] = mu_mfma(p == 0 ? bl[j] : bh[j], p == 1 ? al[i] : ah[i],
                                            acc[i][j]);
        }
        slot = slot == S::ST - 1 ? 0 : slot + 1;
    }
    if constexpr (S::KW == 2) {
        // Each group ends with the whole sums of its half of the block rows.
        constexpr int kHalf = Z::I / 2;
        __syncthreads();
        const int group = wave / Z::kGroup;
        Float4* there = (Float4*)lds + (group * Z::kGroup + member) * (kHalf * Z::J * 64) + lane;
        const Float4* here =
            (Float4*)lds + ((group ^ 1) * Z::kGroup + member) * (kHalf * Z::J * 64) + lane;
#pragma unroll
        for (int i = 0; i < kHalf; ++i)
#pragma unroll
            for (int j = 0; j < Z::J; ++j)
                there[(i * Z::J + j) * 64] = group ? acc[i][j] : acc[i + kHalf][j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kHalf; ++i)
#pragma unroll
            for (int j = 0; j < Z::J; ++j) {
                if (group) acc[i + kHalf][j] = here[(i * Z::J + j) * 64] + acc[i + kHalf][j];
                else acc[i][j] += here[(i * Z::J + j) * 64];
            }
    }
}

// Whether block row i of a tile's sums is the wave's to store.
template <typename S>
__device__ inline bool mu_mine(int i) {
    typedef MuSizes<S> Z;
    return S::KW == 1 || i / (Z::I / S::KW) == (int)(threadIdx.x >> 6) / Z::kGroup;
}

// A workgroup's place: matrix b of the stack, tile (ti, tj), its number, its piece.
struct MuPlace { int b, t, ti, tj, piece; };

__device__ inline MuPlace mu_place(const MuJob& job, uint32_t at) {
    MuPlace p;
    p.piece = at % job.pieces;
    at /= job.pieces;
    p.b = at / job.tiles;
    p.t = at - p.b * job.tiles;
    if (job.cols == 0) {
        mu_triangle(p.t, &p.ti, &p.tj);
    } else {
        p.ti = p.t / job.cols;
        p.tj = p.t - p.ti * job.cols;
    }
    return p;
}

// N times four neighbours of a row, 16 columns apart, into `out`, and mirrored: the other tile of
// a symmetric product, or X beside its transpose.
template <int N>
__device__ inline void mu_store(const MuJob& job, _Float16* ws, int row, int col, Float4 (&v)[N],
                                bool mirror) {
    Half4 h[N], l[N];
    if (job.mode == kPoly) {
        const _Float16* a = ws + (int64_t)job.other * kMuUnit;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t o = mu_at(row, job.ld_out, col + 16 * j);
            h[j] = *(const Half4*)(a + o);
            l[j] = *(const Half4*)(a + o + 32);
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = v[j][e] * job.scale;
            if (job.mode == kPoly) {
                x += job.poly_b * ((float)h[j][e] + (float)l[j][e]);
                if (row == col + 16 * j + e && row < job.m) x += job.poly_a;
            }
            _Float16 y, z;
            mu_split(x, &y, &z);
            h[j][e] = y;
            l[j][e] = z;
        }
    }
    _Float16* out = ws + (int64_t)job.out * kMuUnit;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int64_t o = mu_at(row, job.ld_out, col + 16 * j);
        *(Half4*)(out + o) = h[j];
        *(Half4*)(out + o + 32) = l[j];
    }
    if (!mirror) return;
    const bool sym = job.cols == 0;
    const int ld = sym ? job.ld_out : job.ld_other;
    if (!sym) out = ws + (int64_t)job.other * kMuUnit;
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t q = mu_at(col + 16 * j + e, ld, row);
            out[q] = h[j][e];
            out[q + 32] = l[j][e];
        }
}

__device__ inline uint32_t mu_first_job(const MuJobs& a, int k) { return a.j[k].first; }
__device__ inline uint32_t mu_first_last(const MuLasts& a, int k) { return a.j[k].job.first; }

template <int TILE>
__global__ __launch_bounds__(MuSizes<MuShape<TILE>>::kThreads, 2) void k_mu_product(MuJobs a) {
    typedef MuShape<TILE> S;
    typedef MuSizes<S> Z;
    __shared__ __attribute__((aligned(16))) char lds[Z::kLds];
    const MuJob& job = a.j[mu_find(a, a.n, mu_first_job)];
    const MuPlace p = mu_place(job, blockIdx.x - job.first);
    _Float16* ws = a.ws + (int64_t)p.b * job.stride * kMuUnit;
    const int64_t ld = 2 * (int64_t)job.k;
    const int stages = job.k / (32 * S::KS), from = p.piece * job.piece_stages;
    const int to = from + job.piece_stages < stages ? from + job.piece_stages : stages;
    Float4 acc[Z::I][Z::J];
    mu_tile<S>(ws + (int64_t)job.left * kMuUnit + p.ti * S::T * ld,
               ws + (int64_t)job.right * kMuUnit + p.tj * S::T * ld, job.k, from, to, lds, acc);
    const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & (Z::kGroup - 1);
    const int row0 = (wave / S::WC) * (Z::I * 16) + (lane & 15);
    const int col0 = (wave % S::WC) * (Z::J * 16) + (lane >> 4) * 4;
    if (job.pieces > 1) {
        float* part = (float*)a.ws + (int64_t)job.partial * kMuUnit +
                      (((int64_t)p.b * job.tiles + p.t) * job.pieces + p.piece) * (S::T * S::T);
#pragma unroll
        for (int i = 0; i < Z::I; ++i)
#pragma unroll
            for (int j = 0; j < Z::J; ++j)
                if (mu_mine<S>(i))
                    *(Float4*)(part + (row0 + 16 * i) * S::T + col0 + 16 * j) = acc[i][j];
        return;
    }
    const bool mirror = job.cols == 0 ? p.ti != p.tj : job.other >= 0;
#pragma unroll
    for (int i = 0; i < Z::I; ++i)
        if (mu_mine<S>(i))
            mu_store(job, ws, p.ti * S::T + row0 + 16 * i, p.tj * S::T + col0, acc[i], mirror);
}

// The pieces' sums, in their order: a workgroup takes 64 x 64 values of a tile, a thread eight
// neighbours of a row, and for the mirrored tile of a column.
template <int TILE>
__global__ __launch_bounds__(kMuThreads) void k_mu_join(MuJobs a) {
    constexpr int kSide = TILE / kMuPatch;
    __shared__ float patch[kMuPatch][kMuPatch + 1];
    const MuJob& job = a.j[mu_find(a, a.n, mu_first_job)];
    const uint32_t at = blockIdx.x - job.first;
    MuJob whole = job;
    whole.pieces = 1;
    const MuPlace p = mu_place(whole, at / (kSide * kSide));
    const int r0 = at % (kSide * kSide) / kSide * kMuPatch, c0 = at % kSide * kMuPatch;
    _Float16* ws = a.ws + (int64_t)p.b * job.stride * kMuUnit;
    _Float16* out = ws + (int64_t)job.out * kMuUnit;
    const float* part = (const float*)a.ws + (int64_t)job.partial * kMuUnit +
                        ((int64_t)p.b * job.tiles + p.t) * job.pieces * (TILE * TILE);
    const int c8 = (threadIdx.x & 7) * 8;
    for (int r = threadIdx.x >> 3; r < kMuPatch; r += kMuThreads / 8) {
        const float* from = part + (r0 + r) * TILE + c0 + c8;
        Float4 x = *(const Float4*)from, y = *(const Float4*)(from + 4);
#pragma unroll 4
        for (int q = 1; q < job.pieces; ++q) {
            x += *(const Float4*)(from + (int64_t)q * (TILE * TILE));
            y += *(const Float4*)(from + (int64_t)q * (TILE * TILE) + 4);
        }
        const int row = p.ti * TILE + r0 + r, col = p.tj * TILE + c0 + c8;
        const int64_t o = mu_at(row, job.ld_out, col);
        Half8 h, l;
        if (job.mode == kPoly) {
            h = *(const Half8*)(ws + (int64_t)job.other * kMuUnit + o);
            l = *(const Half8*)(ws + (int64_t)job.other * kMuUnit + o + 32);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = (e < 4 ? x[e & 3] : y[e & 3]) * job.scale;
            if (job.mode == kPoly) {
                v += job.poly_b * ((float)h[e] + (float)l[e]);
                if (row == col + e && row < job.m) v += job.poly_a;
            }
            patch[r][c8 + e] = v;
            _Float16 f, g;
            mu_split(v, &f, &g);
            h[e] = f;
            l[e] = g;
        }
        *(Half8*)(out + o) = h;
        *(Half8*)(out + o + 32) = l;
    }
    if (p.ti == p.tj) return;
    __syncthreads();
    for (int c = threadIdx.x >> 3; c < kMuPatch; c += kMuThreads / 8) {
        Half8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 f, g;
            mu_split(patch[c8 + e][c], &f, &g);
            h[e] = f;
            l[e] = g;
        }
        const int64_t o = mu_at(p.tj * TILE + c0 + c, job.ld_out, p.ti * TILE + r0 + c8);
        *(Half8*)(out + o) = h;
        *(Half8*)(out + o + 32) = l;
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
template <int TILE>
__global__ __launch_bounds__(MuSizes<MuShape<TILE>>::kThreads, 2) void k_mu_last(MuLasts a) {
    typedef MuShape<TILE> S;
    typedef MuSizes<S> Z;
    __shared__ __attribute__((aligned(16))) char lds[Z::kLds];
    const MuLast& l = a.j[mu_find(a, a.n, mu_first_last)];
    const MuJob& job = l.job;
    const MuPlace p = mu_place(job, blockIdx.x - job.first);
    const _Float16* ws = a.ws + (int64_t)p.b * job.stride * kMuUnit;
    const int64_t ld = 2 * (int64_t)job.k;
    Float4 acc[Z::I][Z::J];
    mu_tile<S>(ws + (int64_t)job.left * kMuUnit + p.ti * S::T * ld,
               ws + (int64_t)job.right * kMuUnit + p.tj * S::T * ld, job.k, 0,
               job.k / (32 * S::KS), lds, acc);
    const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & (Z::kGroup - 1);
    const int row0 = p.ti * S::T + (wave / S::WC) * (Z::I * 16) + (lane & 15);
    const int col0 = p.tj * S::T + (wave % S::WC) * (Z::J * 16) + (lane >> 4) * 4;
    const int64_t first = (int64_t)p.b * l.rows * l.cols;
    float* weights = l.dtype == kF32 ? (float*)l.out : l.master;
    // Row `row0 + 16 i` of X's transpose; its weights are asked for together.
#pragma unroll
    for (int i = 0; i < Z::I; ++i) {
        if (!mu_mine<S>(i)) continue;
        int64_t at[Z::J][4];
        float w[Z::J][4] = {};
#pragma unroll
        for (int j = 0; j < Z::J; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = l.tall ? row0 + 16 * i : col0 + 16 * j + e;
                const int c = l.tall ? col0 + 16 * j + e : row0 + 16 * i;
                const bool in = r < l.rows && c < l.cols;
                at[j][e] = in ? first + (int64_t)r * l.cols + c : -1;
                if (l.muon && in) w[j][e] = weights[at[j][e]];
            }
#pragma unroll
        for (int j = 0; j < Z::J; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (at[j][e] < 0) continue;
                float v = acc[i][j][e] * job.scale;
                if (l.muon) {
                    v = __builtin_fmaf(-l.lr, v, w[j][e] * l.decay);
                    weights[at[j][e]] = v;
                    if (l.dtype == kF32) continue;
                }
                mu_put(l.out, l.dtype, at[j][e], v);
            }
    }
}

// ------------------------------------------------------- what goes into them

// A matrix, or a stack of them, as it lies in memory.  momentum: the Muon step's, and x
// is its gradient.
struct MuSource {
    const void* x;
    float* momentum;
    double* parts;         // [count][kMuParts]
    int64_t chunk;         // elements of a partial sum
    int32_t pairs, flipped; // X and its transpose, or the other way round: `pairs` has the source's
                           // orientation
    int32_t stride;        // of a stack, in units
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

typedef Float4 MuAny4 __attribute__((aligned(4)));    // at any element
typedef Float4 MuAny2 __attribute__((aligned(2)));

// Eight neighbours, at any element's address.
__device__ inline void mu_get8(const void* p, int dtype, int64_t at, float (&v)[8]) {
    if (dtype == kF32) {
        const Float4 x = *(const MuAny4*)((const float*)p + at);
        const Float4 y = *(const MuAny4*)((const float*)p + at + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = x[i]; v[4 + i] = y[i]; }
    } else if (dtype == kBF16) {
        typedef __bf16 B8 __attribute__((ext_vector_type(8)));
        const B8 x = __builtin_bit_cast(B8, (Float4) * (const MuAny2*)((const __bf16*)p + at));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
    } else {
        const Half8 x = __builtin_bit_cast(Half8, (Float4) * (const MuAny2*)((const _Float16*)p + at));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
    }
}

// The momentum's move, and partial sums of the squares of each matrix, in fp64.
__global__ __launch_bounds__(kMuThreads) void k_mu_sums(MuSources a) {
    __shared__ double lds[kMuThreads / 64];
    const MuSource& s = a.s[mu_find(a, a.n, mu_first_sum)];
    const uint32_t at = blockIdx.x - s.first_sum;
    const int b = at / s.nparts, part = at - b * s.nparts;
    const int64_t size = (int64_t)s.rows * s.cols, from = part * s.chunk, base = b * size;
    const int64_t to = from + s.chunk < size ? from + s.chunk : size;
    double sum = 0.0;
    for (int64_t i = from + threadIdx.x * 8; i < to; i += kMuThreads * 8) {
        if (i + 8 <= to) {
            float u[8];
            mu_get8(s.x, s.dtype, base + i, u);
            if (s.momentum) {
                float m[8];
                mu_get8(s.momentum, kF32, i, m);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    m[e] = __builtin_fmaf(s.mix, u[e] - m[e], m[e]);
                    u[e] = mu_update(u[e], m[e], s.look);
                }
                *(MuAny4*)(s.momentum + i) = Float4{m[0], m[1], m[2], m[3]};
                *(MuAny4*)(s.momentum + i + 4) = Float4{m[4], m[5], m[6], m[7]};
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = __builtin_fma((double)u[e], (double)u[e], sum);
        } else {
            for (int64_t e = i; e < to; ++e) {
                float u = mu_get(s.x, s.dtype, base + e);
                if (s.momentum) {
                    float m = s.momentum[e];
                    m = __builtin_fmaf(s.mix, u - m, m);
                    s.momentum[e] = m;
                    u = mu_update(u, m, s.look);
                }
                sum = __builtin_fma((double)u, (double)u, sum);
            }
        }
    }
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kMuThreads / 64; ++w) sum += lds[w];
        s.parts[(int64_t)b * kMuParts + part] = sum;
    }
}

// X and its transpose as pairs, scaled to a norm of one (times 2^e), patch by patch: a
// thread takes eight neighbours of a row, and then of a column.
__global__ __launch_bounds__(kMuThreads) void k_mu_pairs(MuSources a) {
    __shared__ float tile[kMuPatch][kMuPatch + 1];
    __shared__ double lds[kMuThreads / 64];
    const MuSource& s = a.s[mu_find(a, a.n, mu_first_patch)];
    const uint32_t at = blockIdx.x - s.first_patch;
    const int b = at / s.patches, t = at - b * s.patches;
    const int r0 = t / s.patch_cols * kMuPatch, c0 = t % s.patch_cols * kMuPatch;
    static_assert(kMuParts == kMuThreads, "one partial sum a thread");
    double sum = (int)threadIdx.x < s.nparts ? s.parts[(int64_t)b * kMuParts + threadIdx.x] : 0.0;
    for (int m = 1; m < 64; m <<= 1) sum += __shfl_xor(sum, m);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kMuThreads / 64; ++w) sum += lds[w];
    const double norm = sqrt(sum);
    const double by = (double)a.scale / (norm < a.eps ? a.eps : norm);   // NaN stays
    const int64_t base = (int64_t)b * s.rows * s.cols;
    _Float16* ws = a.ws + (int64_t)b * s.stride * kMuUnit;
    const int c8 = (threadIdx.x & 7) * 8;
    for (int r = threadIdx.x >> 3; r < kMuPatch; r += kMuThreads / 8) {
        float u[8] = {};
        const int row = r0 + r, col = c0 + c8;
        if (row < s.rows && col < s.cols) {
            const int64_t i = (int64_t)row * s.cols + col;
            if (col + 8 <= s.cols) {
                mu_get8(s.x, s.dtype, base + i, u);
                if (s.momentum) {
                    float m[8];
                    mu_get8(s.momentum, kF32, i, m);
#pragma unroll
                    for (int e = 0; e < 8; ++e) u[e] = mu_update(u[e], m[e], s.look);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col + e < s.cols) {
                        u[e] = mu_get(s.x, s.dtype, base + i + e);
                        if (s.momentum) u[e] = mu_update(u[e], s.momentum[i + e], s.look);
                    }
            }
        }
        Half8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = (float)((double)u[e] * by);
            tile[r][c8 + e] = v;
            _Float16 x, y;
            mu_split(v, &x, &y);
            h[e] = x;
            l[e] = y;
        }
        _Float16* o = ws + (int64_t)s.pairs * kMuUnit + mu_at(row, s.padded_cols, col);
        *(Half8*)o = h;
        *(Half8*)(o + 32) = l;
    }
    __syncthreads();
    for (int c = threadIdx.x >> 3; c < kMuPatch; c += kMuThreads / 8) {
        Half8 h, l;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 x, y;
            mu_split(tile[c8 + e][c], &x, &y);
            h[e] = x;
            l[e] = y;
        }
        _Float16* o = ws + (int64_t)s.flipped * kMuUnit + mu_at(c0 + c, s.padded_rows, r0 + c8);
        *(Half8*)o = h;
        *(Half8*)(o + 32) = l;
    }
}

// ------------------------------------------------------------ small matrices

// A matrix of at most 96 rows by one workgroup, all steps in one launch: X stays in registers.
// A wave holds 32 C columns n, as operands whose lane is n and whose k is m: lane r + 16 g of
// block b has n = 16 b + r, and of 32 values of m those with (m & 15) >> 2 = g, value i being
// m = 16 (i >> 2) + 4 g + (i & 3).  In that order a product's sums lie as its operands do (four
// neighbours of m in the lane of their n), so P X becomes the next X where it is.  For X X^T,
// whose k is n, the wave's columns go through LDS and come back transposed.  A and P lie in LDS
// as operands of the same order.
struct MuSmall {
    const void* x;
    void* out;
    float *master, *momentum;
    int32_t rows, cols;
    uint32_t first;
    int32_t dtype, tall;
    float decay, lr, mix, look;
    int32_t pad;
};

constexpr int kMuSmallWaves = 8;
constexpr int kMuSmallSteps = 32;   // whose numbers travel with the launch

struct MuSmalls {
    MuSmall s[kMuMaxEntries];
    float gram[kMuSmallSteps], square[kMuSmallSteps], linear[kMuSmallSteps], one[kMuSmallSteps],
        apply[kMuSmallSteps];
    double eps;
    float scale, unscale;
    int32_t steps, n;
};
static_assert(sizeof(MuSmalls) <= 4096, "kernel arguments");

__device__ inline uint32_t mu_first_small(const MuSmalls& a, int k) { return a.s[k].first; }

template <int MB> struct MuSmallLds {
    enum {
        B = 2 * MB,                       // blocks of 16 rows
        S = B * (B + 1) / 2,              // of the lower triangle
        kRow = 64 * MB + 8,               // bytes of a column on its way through LDS
        kTurn = 2 * 32 * kRow,            // h and l of a wave's 32 columns
        kPair = B * MB * 2048,            // A or P
        kTurns = kMuSmallWaves * kTurn,
        kSums = kMuSmallWaves / 2 * S * 1024,
        kWork = kTurns > kSums ? kTurns : kSums,
    };
};

// Block (bi, bj) of a symmetric matrix, rows 16 bi + 4 g + e of column 16 bj + (lane & 15), into
// the operands, and mirrored.
template <int MB>
__device__ inline void mu_small_put(char* pair, int bi, int bj, Float4 v) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    Half4 h, l;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        _Float16 x, y;
        mu_split(v[e], &x, &y);
        h[e] = x;
        l[e] = y;
    }
    char* to = pair + (bj * MB + (bi >> 1)) * 2048 + lane * 16 + (bi & 1) * 8;
    *(Half4*)to = h;
    *(Half4*)(to + 1024) = l;
    if (bi == bj) return;
    to = pair + (bi * MB + (bj >> 1)) * 2048 + (4 * g + 16 * (c >> 2)) * 16 +
         (4 * (bj & 1) + (c & 3)) * 2;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        *(_Float16*)(to + e * 16) = h[e];
        *(_Float16*)(to + e * 16 + 1024) = l[e];
    }
}

// Four neighbours in LDS of each lane: of 16 lanes, lane j gives the place of four of the 16
// columns of row j >> 2 and gets its column's values of the four rows.
__device__ inline Half4 mu_turned(const char* at) {
    typedef short Short4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(Half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                         (__attribute__((address_space(3))) Short4*)at));
}

// Sixteen values by their places; the type is asked for once, so that the loads go out together.
__device__ inline void mu_gather(const void* p, int dtype, int64_t first, const int (&at)[16],
                                 float (&v)[16]) {
    if (dtype == kF32) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = ((const float*)p)[first + at[e]];
    } else if (dtype == kBF16) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = (float)((const __bf16*)p)[first + at[e]];
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = (float)((const _Float16*)p)[first + at[e]];
    }
}

__device__ inline void mu_scatter(void* p, int dtype, int64_t first, const int (&at)[16],
                                  const bool (&in)[16], const float (&v)[16]) {
    if (dtype == kF32) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (in[e]) ((float*)p)[first + at[e]] = v[e];
    } else if (dtype == kBF16) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (in[e]) ((__bf16*)p)[first + at[e]] = (__bf16)v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (in[e]) ((_Float16*)p)[first + at[e]] = (_Float16)v[e];
    }
}

template <int MB, int C>
__global__ __launch_bounds__(kMuSmallWaves * 64, 2) void k_mu_small(MuSmalls a) {
    typedef MuSmallLds<MB> Z;
    constexpr int B = Z::B, S = Z::S;
    __shared__ __attribute__((aligned(16))) char lds[Z::kPair + Z::kWork];
    __shared__ double norms[kMuSmallWaves];
    char* const mat = lds;                 // A
    char* const work = lds + Z::kPair;     // columns on their way, sums, P
    const MuSmall& s = a.s[mu_find(a, a.n, mu_first_small)];
    const int64_t first = (int64_t)(blockIdx.x - s.first) * s.rows * s.cols;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = s.tall ? s.cols : s.rows, n = s.tall ? s.rows : s.cols;
    // A wave's columns through LDS, whose rows of memory its lanes read side by side, 16 at a
    // time: 32 lanes take neighbours, columns, or rows where X is tall.
    char* const turn = work + wave * Z::kTurn;
    constexpr int kFar = 2 * Z::kRow;   // bytes of a column of floats
    const int fast = lane & 31, slow = lane >> 5;
    float u[C][2][MB][8];
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int n0 = (c * kMuSmallWaves + wave) * 32;
        if (n0 < n) {
            for (int i = 0; i < 32 * MB; i += 32) {
                int at[16], to[16];
                bool in[16];
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = i + 2 * e + slow;
                    const int col = s.tall ? j & 31 : fast, row = s.tall ? (j & ~31) + fast : j;
                    in[e] = row < m && n0 + col < n;
                    at[e] = !in[e] ? 0 : s.tall ? (n0 + col) * s.cols + row : row * s.cols + n0 + col;
                    to[e] = col * kFar + row * 4;
                }
                mu_gather(s.x, s.dtype, first, at, v);
                if (s.momentum) {
                    float q[16];
                    mu_gather(s.momentum, kF32, 0, at, q);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        q[e] = __builtin_fmaf(s.mix, v[e] - q[e], q[e]);
                        v[e] = mu_update(v[e], q[e], s.look);
                        if (in[e]) s.momentum[at[e]] = q[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    v[e] = in[e] ? v[e] : 0.0f;
                    sum = __builtin_fma((double)v[e], (double)v[e], sum);
                    *(float*)(turn + to[e]) = v[e];
                }
            }
        }
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < MB; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    Float4 x = *(const Float4*)(turn + (16 * b + r) * kFar +
                                                (32 * k + 16 * e + 4 * g) * 4);
                    if (n0 >= n) x = Float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < 4; ++i) u[c][b][k][4 * e + i] = x[i];
                }
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    for (int q = 1; q < 64; q <<= 1) sum += __shfl_xor(sum, q);
    if (lane == 0) norms[wave] = sum;
    __syncthreads();
    sum = 0.0;
    for (int w = 0; w < kMuSmallWaves; ++w) sum += norms[w];
    const double norm = sqrt(sum);
    const double by = (double)a.scale / (norm < a.eps ? a.eps : norm);   // NaN stays
    Half8 h[C][2][MB], l[C][2][MB];
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < MB; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    _Float16 x, y;
                    mu_split((float)((double)u[c][b][k][i] * by), &x, &y);
                    h[c][b][k][i] = x;
                    l[c][b][k][i] = y;
                }

    for (int step = 0; step < a.steps; ++step) {
        // A = X X^T: each wave's columns, then the waves' sums.
        Float4 acc[S];
#pragma unroll
        for (int t = 0; t < S; ++t) acc[t] = Float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if ((c * kMuSmallWaves + wave) * 32 >= n) continue;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int k = 0; k < MB; ++k)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        char* to = turn + (16 * b + r) * Z::kRow + (32 * k + 16 * e + 4 * g) * 2;
                        const Half8 x = h[c][b][k], y = l[c][b][k];
                        *(Half4*)to = Half4{x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]};
                        *(Half4*)(to + Z::kTurn / 2) =
                            Half4{y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]};
                    }
            __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            Half8 fh[B], fl[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const char* from = turn + (4 * g + (r >> 2)) * Z::kRow + (16 * b + 4 * (r & 3)) * 2;
                const Half4 h0 = mu_turned(from), h1 = mu_turned(from + 16 * Z::kRow);
                const Half4 l0 = mu_turned(from + Z::kTurn / 2),
                            l1 = mu_turned(from + Z::kTurn / 2 + 16 * Z::kRow);
                fh[b] = __builtin_shufflevector(h0, h1, 0, 1, 2, 3, 4, 5, 6, 7);
                fl[b] = __builtin_shufflevector(l0, l1, 0, 1, 2, 3, 4, 5, 6, 7);
            }
            __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int q = 0; q < 3; ++q)
#pragma unroll
                for (int bi = 0; bi < B; ++bi)
#pragma unroll
                    for (int bj = 0; bj <= bi; ++bj) {
                        Float4& t = acc[bi * (bi + 1) / 2 + bj];
                        t = mu_mfma(q == 0 ? fl[bi] : fh[bi], q == 1 ? fl[bj] : fh[bj], t);
                    }
        }
        __syncthreads();   // nothing is on its way any more
        char* const mine = work + (wave & (kMuSmallWaves / 2 - 1)) * (S * 1024) + lane * 16;
        const bool half = C == 1 && n <= kMuSmallWaves / 2 * 32;   // of the waves have columns
        if (!half) {
            if (wave >= kMuSmallWaves / 2) {
#pragma unroll
                for (int t = 0; t < S; ++t) *(Float4*)(mine + t * 1024) = acc[t];
            }
            __syncthreads();
        }
        if (wave < kMuSmallWaves / 2) {
#pragma unroll
            for (int t = 0; t < S; ++t) {
                if (!half) acc[t] += *(const Float4*)(mine + t * 1024);
                *(Float4*)(mine + t * 1024) = acc[t];
            }
        }
        __syncthreads();
        for (int t = wave; t < S; t += kMuSmallWaves) {
            int bi, bj;
            mu_triangle(t, &bi, &bj);
            Float4 v = *(const Float4*)(work + t * 1024 + lane * 16);
            for (int w = 1; w < kMuSmallWaves / 2; ++w)
                v += *(const Float4*)(work + (w * S + t) * 1024 + lane * 16);
            mu_small_put<MB>(mat, bi, bj, v * a.gram[step]);
        }
        __syncthreads();   // A is there, and the sums read: P takes their place
        for (int t = wave; t < S; t += kMuSmallWaves) {
            int bi, bj;
            mu_triangle(t, &bi, &bj);
            Float4 v{0.0f, 0.0f, 0.0f, 0.0f}, v1 = v, v2 = v;
#pragma unroll
            for (int k = 0; k < MB; ++k) {
                const char* x = mat + (bi * MB + k) * 2048 + lane * 16;
                const char* y = mat + (bj * MB + k) * 2048 + lane * 16;
                const Half8 xh = *(const Half8*)x, xl = *(const Half8*)(x + 1024);
                const Half8 yh = *(const Half8*)y, yl = *(const Half8*)(y + 1024);
                v1 = mu_mfma(xl, yh, v1);
                v2 = mu_mfma(xh, yl, v2);
                v = mu_mfma(xh, yh, v);
            }
            v += v1 + v2;
            const char* own = mat + (bj * MB + (bi >> 1)) * 2048 + lane * 16 + (bi & 1) * 8;
            const Half4 oh = *(const Half4*)own, ol = *(const Half4*)(own + 1024);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * bi + 4 * g + e;
                v[e] = v[e] * a.square[step] + a.linear[step] * ((float)oh[e] + (float)ol[e]);
                if (row == 16 * bj + r && row < m) v[e] += a.one[step];
            }
            mu_small_put<MB>(work, bi, bj, v);
        }
        __syncthreads();
        // X <- P X, where it is.
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if ((c * kMuSmallWaves + wave) * 32 >= n) continue;
            Float4 y[2][B];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int t = 0; t < B; ++t) y[b][t] = Float4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < MB; ++k)
#pragma unroll
                for (int t = 0; t < B; t += 2) {
                    Half8 ph[2], pl[2];
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        const char* p = work + ((t + d) * MB + k) * 2048 + lane * 16;
                        ph[d] = *(const Half8*)p;
                        pl[d] = *(const Half8*)(p + 1024);
                    }
#pragma unroll
                    for (int q = 0; q < 3; ++q)
#pragma unroll
                        for (int d = 0; d < 2; ++d)
#pragma unroll
                            for (int b = 0; b < 2; ++b)
                                y[b][t + d] = mu_mfma(q == 0 ? pl[d] : ph[d],
                                                      q == 1 ? l[c][b][k] : h[c][b][k], y[b][t + d]);
                }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int t = 0; t < B; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        _Float16 x, z;
                        mu_split(y[b][t][e] * a.apply[step], &x, &z);
                        h[c][b][t >> 1][4 * (t & 1) + e] = x;
                        l[c][b][t >> 1][4 * (t & 1) + e] = z;
                    }
        }
        __syncthreads();   // P is read
    }

    // Out as it came: the two halves hold a value to 2^-24.
    float* const weights = s.dtype == kF32 ? (float*)s.out : s.master;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int n0 = (c * kMuSmallWaves + wave) * 32;
        if (n0 >= n) continue;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int k = 0; k < MB; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    Float4 x;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        x[i] = ((float)h[c][b][k][4 * e + i] + (float)l[c][b][k][4 * e + i]) *
                               a.unscale;
                    *(Float4*)(turn + (16 * b + r) * kFar + (32 * k + 16 * e + 4 * g) * 4) = x;
                }
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        for (int i = 0; i < 32 * MB; i += 32) {
            int at[16];
            bool in[16];
            float v[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = i + 2 * e + slow;
                const int col = s.tall ? j & 31 : fast, row = s.tall ? (j & ~31) + fast : j;
                in[e] = row < m && n0 + col < n;
                at[e] = !in[e] ? 0 : s.tall ? (n0 + col) * s.cols + row : row * s.cols + n0 + col;
                v[e] = *(const float*)(turn + col * kFar + row * 4);
            }
            if (s.momentum) {
                float w[16];
                mu_gather(weights, kF32, 0, at, w);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    v[e] = __builtin_fmaf(-s.lr, v[e], w[e] * s.decay);
                    if (in[e]) weights[at[e]] = v[e];
                }
                if (s.dtype == kF32) continue;
            }
            mu_scatter(s.out, s.dtype, first, at, in, v);
        }
        __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// ---------------------------------------------------------------------- host

// Coefficients, and bounds of the singular values before each step, from which the
// exponents follow.
struct MuPlan {
    int steps, phase;
    double a, b, c;
    double x[kMuMaxSteps + 1];
    double p[kMuMaxSteps];   // bounds of P's
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

// What is below `bound` is held times 2^e: at most 2^14, where fp16 ends at 2^16.
int mu_exponent(double bound) {
    int e;
    frexp(std::max(bound, 1e-3), &e);   // below 2^e
    return 14 - e;
}

bool mu_plan(MuPlan* p, int steps, double a, double b, double c) {
    if (steps < 1 || steps > kMuMaxSteps || !(fabs(a) <= 64.0) || !(fabs(b) <= 64.0) ||
        !(fabs(c) <= 64.0))
        return false;
    *p = MuPlan{steps, 1, a, b, c, {1.01}, {}};
    for (int k = 0; k < steps; ++k) {
        p->p[k] = mu_bound(*p, p->x[k], false);
        p->x[k + 1] = mu_bound(*p, p->x[k], true);
        if (!(p->x[k + 1] <= 64.0)) return false;   // values that grow without end
    }
    // The rounding of A grows by a^2 a step of a phase.
    while (p->phase < kMuPhase && pow(fabs(a), 2.0 * p->phase) <= 14.0) ++p->phase;
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
    int phase;                   // most steps of a phase
    int64_t stride;              // in units, as the offsets
    int64_t X, XT[2], A, T, P, Q[2];
};

int64_t mu_round(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Phases: the longest, one shorter, the longest, ...
int mu_len(int phase, int number, int left) {
    const int len = number & 1 ? std::max(1, phase - 1) : phase;
    return std::min(len, left);
}

// The products of one matrix, in m^3.
double mu_cost(int steps, int phase, double ratio) {
    double cost = 0.0;
    for (int k = 0, number = 0; k < steps; ++number) {
        const int len = mu_len(phase, number, steps - k);
        cost += 3.0 * ratio + 4.0 * len - 3.0;
        k += len;
    }
    return cost;
}

// Where an entry's matrices lie for a tile and phases of so many steps (where they save work),
// from `base` on; the units that it takes.
int64_t mu_layout(MuEntry* e, const MuPlan& p, int tile, int phase, int64_t base) {
    e->tall = e->rows > e->cols;
    e->m = e->tall ? e->cols : e->rows;
    e->n = e->tall ? e->rows : e->cols;
    e->mp = mu_round(e->m, tile);
    e->np = mu_round(e->n, tile);
    const double ratio = (double)e->np / (double)e->mp;
    e->phase = mu_cost(p.steps, phase, ratio) < mu_cost(p.steps, 1, ratio) ? phase : 1;
    const int64_t wide = 2 * e->mp * e->np / kMuUnit, square = 2 * e->mp * e->mp / kMuUnit;
    int64_t at = 0;
    // Each an even number of units, as partial sums behind them need it.
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
    e->stride = at;
    return at * e->count;
}

// A product: rows x cols values, or the lower triangle of a square (cols 0).
struct MuOp { MuJob job; int64_t rows, cols; int slot; };

// The products of an entry, each with the launch that it goes into (up to two of them a
// launch), without the last.
struct MuSchedule {
    MuOp ops[8 * kMuMaxSteps];
    int n, slots;
    MuOp last;

    void make(const MuEntry& e, const MuPlan& p) {
        n = slots = 0;
        int ex = mu_exponent(p.x[0]), xt = 0;
        for (int k = 0, number = 0;; ++number) {
            const int len = mu_len(e.phase, number, p.steps - k);
            int ea = mu_exponent(p.x[k] * p.x[k]), eq = 0, q = 0;
            double pq = 1.0;
            sym(e, e.X, e.X, e.A, e.np, ea - 2 * ex);
            ++slots;
            for (int i = 0; i < len; ++i) {
                const double x = p.x[k + i], bound = p.p[k + i];
                const int ep = mu_exponent(bound);
                const int64_t P = i == 0 ? e.Q[0] : e.P;
                MuJob* j = sym(e, e.A, e.A, P, e.mp, 0);
                j->mode = kPoly;
                j->other = (int32_t)e.A;
                j->scale = (float)ldexp(p.c, ep - 2 * ea);
                j->poly_b = (float)ldexp(p.b, ep - ea);
                j->poly_a = (float)ldexp(p.a, ep);
                ++slots;
                pq *= bound;
                if (i == 0) eq = ep;
                const bool more = i + 1 < len;
                const int et = mu_exponent(x * x * bound);
                if (i > 0) {
                    const int next = mu_exponent(pq);
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
            k += len;
            const bool end = k >= p.steps;
            const int ex2 = end ? 0 : mu_exponent(p.x[k]);
            MuJob j = job(e, e.XT[xt], e.Q[q], e.mp, ex2 - ex - eq);
            j.mode = kApply;
            j.ld_out = (int32_t)e.mp;
            j.ld_other = (int32_t)e.np;
            if (end) {
                last = MuOp{j, e.np, e.mp, slots};
                return;
            }
            j.out = (int32_t)e.XT[xt ^ 1];
            j.other = (int32_t)e.X;
            ops[n++] = MuOp{j, e.np, e.mp, slots++};
            xt ^= 1;
            ex = ex2;
        }
    }

  private:
    MuJob job(const MuEntry& e, int64_t left, int64_t right, int64_t k, int exponent) {
        MuJob j{};
        j.left = (int32_t)left;
        j.right = (int32_t)right;
        j.stride = (int32_t)e.stride;
        j.k = (int32_t)k;
        j.m = (int32_t)e.m;
        j.scale = (float)ldexp(1.0, exponent);
        return j;
    }

    MuJob* sym(const MuEntry& e, int64_t left, int64_t right, int64_t out, int64_t k,
               int exponent) {
        MuJob j = job(e, left, right, k, exponent);
        j.out = (int32_t)out;
        j.ld_out = (int32_t)e.mp;
        ops[n] = MuOp{j, e.mp, 0, slots};
        return &ops[n++].job;
    }
};

bool mu_launched() { return hipGetLastError() == hipSuccess; }

int64_t mu_tiles(const MuOp& o, int tile) {
    const int64_t r = o.rows / tile;
    return o.cols ? r * (o.cols / tile) : r * (r + 1) / 2;
}

// What a launch of products costs with a tile, in us, from measurements: `stage` values of k
// take `us` where the CU's `resident` workgroups share it, and at least `alone`; a workgroup's
// beginning and end take `ends`.  (Measured with one tile for all launches, 64 / 128 / 256:
// 1021 x 765 216 / 449 / 1165 us; 4096 x 4096 6.9 / 4.1 / 4.0 ms; the encoder 64 wide 0.96 / 1.24
// / 2.66 ms, 256 wide 21.9 / 13.8 / 13.0 ms; by these costs 0.22, 3.8, 0.59 and 12.0.)
struct MuTileCost { int tile, stage, resident; double us, alone, ends; };
const MuTileCost kMuTiles[] = {{64, 64, 1, 0.75, 0.65, 1.5}, {128, 32, 2, 1.4, 0.75, 4.0},
                               {256, 32, 1, 2.1, 2.1, 10.0}};
constexpr int kMuCus = 256;
constexpr double kMuLaunch = 4.0;       // a launch more
constexpr double kMuBytesPerUs = 4e6;   // of partial sums

// How a launch's sums are cut: its tile, the most stages of a piece, and what it costs.
struct MuCut {
    const MuTileCost* tile;
    int64_t piece;
    double us;
    int64_t partials;   // units

    int64_t stages(const MuJob& j) const { return j.k / tile->stage; }
    int64_t pieces(const MuOp& o) const {
        return o.cols ? 1 : (stages(o.job) + piece - 1) / piece;
    }
};

MuCut mu_cut(const MuOp* const* ops, const int64_t* counts, int n, int most_tile, bool may_split) {
    MuCut best{nullptr, 0, 1e30, 0};
    for (const MuTileCost& t : kMuTiles) {
        if (t.tile > most_tile) continue;
        MuCut c{&t, (int64_t)1 << 40, 0.0, 0};
        const double slots = kMuCus * t.resident;
        int64_t longest = 0, tiles[kMuMaxJobs];
        double work = 0.0;
        for (int i = 0; i < n; ++i) {
            tiles[i] = mu_tiles(*ops[i], t.tile) * counts[i];
            work += (double)(tiles[i] * c.stages(ops[i]->job));
            longest = std::max(longest, c.stages(ops[i]->job));
        }
        for (int cuts = 1; cuts <= (may_split ? 32 : 1); cuts += 1 + cuts / 4) {
            // Pieces as long as these cuts of the longest sum.
            c.piece = (longest + cuts - 1) / cuts;
            if (cuts > 1 && c.piece < 4) break;
            double blocks = 0.0;
            int64_t piece = 0;
            c.partials = 0;
            for (int i = 0; i < n; ++i) {
                const int64_t pieces = c.pieces(*ops[i]), st = c.stages(ops[i]->job);
                piece = std::max(piece, (st + pieces - 1) / pieces);
                blocks += (double)(tiles[i] * pieces);
                if (pieces > 1) c.partials += tiles[i] * pieces * (t.tile * t.tile / kMuUnit);
            }
            // Rounds of the longest pieces; pieces of all lengths fill the last round better.
            double rounds = work / (double)piece / slots, last = 0.0;
            if (blocks * (double)piece < 1.1 * work) {
                last = rounds - floor(rounds);
                rounds = std::max(1.0, floor(rounds) + (last > 0.02 ? 1.0 : 0.0));
            } else {
                last = std::min(1.0, rounds);
                rounds = std::max(1.0, rounds + 0.5);
            }
            c.us = t.ends * std::max(1.0, blocks / slots) +
                   (double)piece * ((rounds - 1.0) * t.us + t.alone + (t.us - t.alone) * last);
            if (c.partials) c.us += kMuLaunch + c.partials * (kMuUnit * 8.0) / kMuBytesPerUs;
            if (c.us < best.us && c.partials < (int64_t)1 << 17) best = c;
            if (cuts > 1 && !c.partials) break;
        }
    }
    return best;
}

// The products of a launch.
struct MuLaunch {
    const MuOp* op[kMuMaxJobs];
    int64_t count[kMuMaxJobs];
    int n = 0;
    MuCut cut;

    void add(const MuOp& o, int64_t c) {
        op[n] = &o;
        count[n++] = c;
    }
    // Of the same sizes: cut alike.
    bool like(const MuLaunch& o) const {
        if (n != o.n) return false;
        for (int i = 0; i < n; ++i)
            if (op[i]->rows != o.op[i]->rows || op[i]->cols != o.op[i]->cols ||
                op[i]->job.k != o.op[i]->job.k || count[i] != o.count[i])
                return false;
        return true;
    }
    void place(MuJob* j, int i, int64_t* blocks, int64_t* partial) const {
        *j = op[i]->job;
        const int tile = cut.tile->tile;
        j->cols = (int32_t)(op[i]->cols / tile);
        j->tiles = (int32_t)mu_tiles(*op[i], tile);
        j->pieces = (int32_t)cut.pieces(*op[i]);
        const int64_t stages = cut.stages(*j);
        j->piece_stages = (int32_t)((stages + j->pieces - 1) / j->pieces);
        // Rounded up, some pieces fewer may do.
        j->pieces = (int32_t)((stages + j->piece_stages - 1) / j->piece_stages);
        j->first = (uint32_t)*blocks;
        *blocks += j->tiles * count[i] * j->pieces;
        if (j->pieces > 1) {
            j->partial = (int32_t)*partial;
            *partial += j->tiles * count[i] * j->pieces * (tile * tile / kMuUnit);
        }
    }
};

template <int TILE>
bool mu_products(const MuJobs& a, int64_t blocks, const MuJobs& joins, int64_t join_blocks,
                 hipStream_t stream) {
    hipLaunchKernelGGL(k_mu_product<TILE>, dim3((unsigned)blocks),
                       dim3(MuSizes<MuShape<TILE>>::kThreads), 0, stream, a);
    if (!mu_launched()) return false;
    if (join_blocks == 0) return true;
    hipLaunchKernelGGL(k_mu_join<TILE>, dim3((unsigned)join_blocks), dim3(kMuThreads), 0, stream,
                       joins);
    return mu_launched();
}

template <int TILE>
bool mu_last(const MuLasts& a, int64_t blocks, hipStream_t stream) {
    hipLaunchKernelGGL(k_mu_last<TILE>, dim3((unsigned)blocks),
                       dim3(MuSizes<MuShape<TILE>>::kThreads), 0, stream, a);
    return mu_launched();
}

// Entries whose launches are shared: what they are padded to, and their launches.
struct MuChunk {
    MuEntry* e;
    int n, pad, phase;
    double us;
    int64_t units;      // of halves; behind them the partial sums of products, and of norms
    int64_t partials, parts;
    std::unique_ptr<MuSchedule[]> sched;
    std::vector<MuLaunch> launches;   // the last one is the last product's

    int64_t bytes() const { return (units * 2 + partials * 4) * kMuUnit + parts * 8; }

    void lay(const MuPlan& p, int pad_of, int phase_of) {
        pad = pad_of;
        phase = phase_of;
        units = partials = parts = 0;
        int slots = 0;
        us = 0.0;
        for (int k = 0; k < n; ++k) {
            units += mu_layout(e + k, p, pad, phase, units);
            parts += e[k].count * kMuParts;
            sched[k].make(e[k], p);
            slots = std::max(slots, sched[k].slots);
        }
        launches.assign(slots + 1, MuLaunch());
        for (int k = 0; k < n; ++k) {
            for (int i = 0; i < sched[k].n; ++i)
                launches[sched[k].ops[i].slot].add(sched[k].ops[i], e[k].count);
            launches[slots].add(sched[k].last, e[k].count);
        }
        for (int i = 0; i <= slots; ++i) {
            MuLaunch& l = launches[i];
            int same = 0;
            while (same < i && !l.like(launches[same])) ++same;
            l.cut = same < i && i < slots ? launches[same].cut
                                          : mu_cut(l.op, l.count, l.n, pad, i < slots);
            us += l.cut.us + kMuLaunch;
            partials = std::max(partials, l.cut.partials);
        }
    }

    // The padding that costs least, and phases or steps on X: phases save work where X is long,
    // steps on X launches.
    void choose(const MuPlan& p) {
        int best_pad = 0, best_phase = p.phase;
        double least = 1e30;
        auto look = [&](int tile, int by) {
            lay(p, tile, by);
            if (us >= least) return;
            least = us;
            best_pad = tile;
            best_phase = by;
        };
        for (const MuTileCost& t : kMuTiles) look(t.tile, p.phase);
        if (p.phase > 1) look(best_pad, 1);
        if (best_pad != pad || best_phase != phase) lay(p, best_pad, best_phase);
    }
};

int mu_chunk(const MuChunk& chunk, const MuPlan& p, double eps, void* workspace,
             hipStream_t stream) {
    const MuEntry* e = chunk.e;
    const int n = chunk.n;
    MuSources src{};
    src.ws = (_Float16*)workspace;
    src.eps = eps;
    src.scale = (float)ldexp(1.0, mu_exponent(p.x[0]));
    src.n = n;
    int64_t sums = 0, patches = 0;
    double* parts = (double*)((char*)workspace + (chunk.units * 2 + chunk.partials * 4) * kMuUnit);
    for (int k = 0; k < n; ++k) {
        MuSource& s = src.s[k];
        const int64_t size = e[k].rows * e[k].cols;
        s.x = e[k].x;
        s.momentum = e[k].momentum;
        s.parts = parts;
        parts += e[k].count * kMuParts;
        s.pairs = (int32_t)(e[k].tall ? e[k].XT[0] : e[k].X);
        s.flipped = (int32_t)(e[k].tall ? e[k].X : e[k].XT[0]);
        s.stride = (int32_t)e[k].stride;
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
    }
    const dim3 block(kMuThreads);
    hipLaunchKernelGGL(k_mu_sums, dim3((unsigned)sums), block, 0, stream, src);
    if (!mu_launched()) return CS_ERR_HIP;
    hipLaunchKernelGGL(k_mu_pairs, dim3((unsigned)patches), block, 0, stream, src);
    if (!mu_launched()) return CS_ERR_HIP;
    // Partial sums lie behind the pairs; offsets count units of 4096 halves there, and of as many
    // floats here, so they begin at an even unit.
    for (size_t i = 0; i + 1 < chunk.launches.size(); ++i) {
        const MuLaunch& l = chunk.launches[i];
        MuJobs a{}, joins{};
        a.ws = joins.ws = (_Float16*)workspace;
        a.n = l.n;
        int64_t blocks = 0, partial = chunk.units / 2, join_blocks = 0;
        const int tile = l.cut.tile->tile;
        for (int k = 0; k < l.n; ++k) {
            l.place(&a.j[k], k, &blocks, &partial);
            if (a.j[k].pieces > 1) {
                MuJob& j = joins.j[joins.n++];
                j = a.j[k];
                j.first = (uint32_t)join_blocks;
                join_blocks += j.tiles * l.count[k] * (tile * tile / kMuUnit);
            }
        }
        const bool ok = tile == 256 ? mu_products<256>(a, blocks, joins, join_blocks, stream)
                        : tile == 128 ? mu_products<128>(a, blocks, joins, join_blocks, stream)
                                      : mu_products<64>(a, blocks, joins, join_blocks, stream);
        if (!ok) return CS_ERR_HIP;
    }
    const MuLaunch& l = chunk.launches.back();
    MuLasts last{};
    last.ws = (_Float16*)workspace;
    last.n = n;
    int64_t blocks = 0, none = 0;
    for (int k = 0; k < n; ++k) {
        MuLast& y = last.j[k];
        l.place(&y.job, k, &blocks, &none);
        y.out = e[k].out;
        y.master = e[k].master;
        y.rows = (int32_t)e[k].rows;
        y.cols = (int32_t)e[k].cols;
        y.tall = e[k].tall;
        y.dtype = e[k].dtype;
        y.muon = e[k].momentum != nullptr;
        y.decay = e[k].decay;
        y.lr = e[k].lr;
    }
    const int tile = l.cut.tile->tile;
    const bool ok = tile == 256 ? mu_last<256>(last, blocks, stream)
                    : tile == 128 ? mu_last<128>(last, blocks, stream)
                                  : mu_last<64>(last, blocks, stream);
    return ok ? CS_OK : CS_ERR_HIP;
}

// The columns that a workgroup of small matrices holds are 256 C.
int mu_small_blocks(const MuEntry& e) { return (int)((std::min(e.rows, e.cols) + 31) / 32); }

int mu_small_columns(const MuEntry& e) {
    const int64_t need = (std::max(e.rows, e.cols) + 255) / 256;
    return need <= 4 ? (int)need : 8;
}

// What the registers hold beside the sums.  (64 x 576 takes 60 us for 96 in launches of products,
// 24 x 96 x 97 45 for 105.)
bool mu_is_small(const MuEntry& e, const MuPlan& p) {
    const int mb = mu_small_blocks(e);
    return p.steps <= kMuSmallSteps && mb <= 3 &&
           std::max(e.rows, e.cols) <= (mb == 1 ? 2048 : mb == 2 ? 1024 : 512);
}

template <int MB, int C>
bool mu_small_launch(const MuSmalls& a, int64_t blocks, hipStream_t stream) {
    hipLaunchKernelGGL((k_mu_small<MB, C>), dim3((unsigned)blocks), dim3(kMuSmallWaves * 64), 0,
                       stream, a);
    return mu_launched();
}

// All entries are small: a launch for each kind, of up to 20.
int mu_small(const std::vector<MuEntry>& e, int n, const MuPlan& p, double eps,
             hipStream_t stream) {
    MuSmalls a{};
    a.eps = eps;
    a.steps = p.steps;
    a.scale = (float)ldexp(1.0, mu_exponent(p.x[0]));
    for (int k = 0; k < p.steps; ++k) {
        const int ex = mu_exponent(p.x[k]), ea = mu_exponent(p.x[k] * p.x[k]);
        const int ep = mu_exponent(p.p[k]);
        const int next = mu_exponent(p.x[k + 1]);
        a.unscale = (float)ldexp(1.0, -next);
        a.gram[k] = (float)ldexp(1.0, ea - 2 * ex);
        a.square[k] = (float)ldexp(p.c, ep - 2 * ea);
        a.linear[k] = (float)ldexp(p.b, ep - ea);
        a.one[k] = (float)ldexp(p.a, ep);
        a.apply[k] = (float)ldexp(1.0, next - ep - ex);
    }
    for (int mb = 1; mb <= 3; ++mb)
        for (int c : {1, 2, 3, 4, 8}) {
            int64_t blocks = 0;
            a.n = 0;
            for (int k = 0; k <= n; ++k) {
                if (a.n == kMuMaxEntries || (k == n && a.n > 0)) {
                    const bool ok =
                        mb == 1 ? (c == 1   ? mu_small_launch<1, 1>(a, blocks, stream)
                                   : c == 2 ? mu_small_launch<1, 2>(a, blocks, stream)
                                   : c <= 4 ? mu_small_launch<1, 4>(a, blocks, stream)
                                            : mu_small_launch<1, 8>(a, blocks, stream))
                        : mb == 2 ? (c == 1   ? mu_small_launch<2, 1>(a, blocks, stream)
                                     : c == 2 ? mu_small_launch<2, 2>(a, blocks, stream)
                                     : c == 3 ? mu_small_launch<2, 3>(a, blocks, stream)
                                              : mu_small_launch<2, 4>(a, blocks, stream))
                                  : (c == 1 ? mu_small_launch<3, 1>(a, blocks, stream)
                                            : mu_small_launch<3, 2>(a, blocks, stream));
                    if (!ok) return CS_ERR_HIP;
                    a.n = 0;
                    blocks = 0;
                }
                if (k == n || mu_small_blocks(e[k]) != mb || mu_small_columns(e[k]) != c) continue;
                MuSmall& s = a.s[a.n++];
                s = MuSmall{e[k].x, e[k].out, e[k].master, e[k].momentum, (int32_t)e[k].rows,
                            (int32_t)e[k].cols, (uint32_t)blocks, e[k].dtype,
                            e[k].rows > e[k].cols, e[k].decay, e[k].lr, e[k].mix, e[k].look, 0};
                blocks += e[k].count;
            }
        }
    return CS_OK;
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
        const int64_t rt = mu_round(x.rows, kMuMostTile) / kMuPatch,
                      ct = mu_round(x.cols, kMuMostTile) / kMuPatch;
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
    try {
        std::vector<MuEntry> e((size_t)ntensors + 1);
        const int n = mu_entries(ntensors, table, scalars, muon, e.data());
        if (n < 0) return CS_ERR_ARGS;
        // The longest sums first: they end last.
        std::stable_sort(e.begin(), e.begin() + n, [](const MuEntry& x, const MuEntry& y) {
            return std::max(x.rows, x.cols) > std::max(y.rows, y.cols);
        });
        if (bytes) *bytes = 0;
        if (std::all_of(e.begin(), e.begin() + n,
                        [&](const MuEntry& x) { return mu_is_small(x, p); }))
            return bytes ? CS_OK : mu_small(e, n, p, eps, stream);
        if (!bytes && (!workspace || ((uintptr_t)workspace & 127))) return CS_ERR_ARGS;
        MuChunk chunk;
        chunk.sched.reset(new MuSchedule[kMuMaxEntries]);
        for (int k = 0; k < n; k += kMuMaxEntries) {
            chunk.e = &e[k];
            chunk.n = std::min(kMuMaxEntries, n - k);
            chunk.choose(p);
            if (chunk.units + 2 * chunk.partials > 0x7FFFFFFF) return CS_ERR_ARGS;
            if (bytes) {
                *bytes = std::max(*bytes, chunk.bytes());
            } else {
                const int rc = mu_chunk(chunk, p, eps, workspace, stream);
                if (rc != CS_OK) return rc;
            }
        }
    } catch (const std::exception&) {   // of memory or lengths
        return CS_ERR_ARGS;
    }
    return CS_OK;
}

}  // namespace

extern "C" int64_t cs_orthogonalize_workspace_bytes(int32_t ntensors, const int64_t* table,
                                                    int32_t steps, double a, double b, double c) {
    int64_t bytes = 0;
    return mu_run(ntensors, table, nullptr, false, steps, a, b, c, 0.0, nullptr, &bytes,
                  nullptr) == CS_OK ? bytes : -1;
}

extern "C" int cs_orthogonalize(int32_t ntensors, const int64_t* table, int32_t steps, double a,
                                double b, double c, double eps, void* workspace,
                                hipStream_t stream) {
    return mu_run(ntensors, table, nullptr, false, steps, a, b, c, eps, workspace, nullptr, stream);
}

extern "C" int cs_muon_step(int32_t ntensors, const int64_t* table, const float* scalars,
                            int32_t steps, double a, double b, double c, double eps,
                            void* workspace, hipStream_t stream) {
    return mu_run(ntensors, table, scalars, true, steps, a, b, c, eps, workspace, nullptr, stream);
}
