// Orthogonalised updates: momentum, five quintic Newton-Schulz steps on each weight matrix, decay and update.
//
//   u = g + mu m' (m' = mu m + g),  X_0 = u / (|u|_F + eps),
//   A = X X^T,  Q = a + b A + c A^2,  X <- Q X          (a, b, c) = (3.4445, -4.7750, 2.0315), n = rows <= m = columns
//
// which maps every singular value s of X through a s + b s^3 + c s^5, towards 1 (tall matrices are worked on transposed).
// Per step n^2 m + n^3 + 2 n^2 m operations: A and Q are symmetric, only tiles that reach the diagonal or lie below it are
// computed, and stored to both places.  The bound is the matrix pipe from n = 1024 up, the chain of dependent launches below.
//
// Arithmetic.  Matrices of either type go through the two-way fp16 split of this library (device_utils.hpp: split2h): every
// operand is hi + lo in fp16 scaled by 2^14, products lo hi + hi lo + hi hi accumulate in fp32, i.e. fp32 accuracy at three 16-bit
// matrix instructions (a library fp32 product reaches 153 TFLOP/s on this card, the fp16 one 1220).  The scale is safe
// without looking at the data: |u|_F = 1 bounds every singular value of X_0 by 1, the quintic maps [0, 1.21] into itself, so
// |X| <= 1.21, |A| <= 1.47, |Q| <= 3.4445 and 3.4445 * 2^14 < 65504.
// bf16 matrices are read exactly and rounded once, at the end: their result is the fp32 one's, rounded.  (The hi planes
// alone, one instruction per product, round X, A and Q to 11 bits each step and lose every direction weaker than 2^-11 of the
// strongest: up to 4e-2 off where four directions carry all but 1e-3.  3 x 777 x 2050: 259 us that way, 379 this.)
// X_0 is never rounded by the normalisation: its planes hold u times a power of two, the rest of the factor (in (1, 2])
// enters the first step's products in fp32.
//
// Planes are stored as the matrix instruction's operand fragments, [row tile of 16][k block of 32][lane 64][8], 1 KB in a
// row per fragment, so a tile is fetched into LDS lane by lane (global_load_lds) and read back without a bank conflict.  X is
// kept one way: k along m for A; for Q X, k along n, its fragments are read from LDS transposed.
// Measured (one layer of width 2048: four 2048 x 2048, three 8192 x 2048, a step): 5.36 ms, products at 1.1 of the 1.22
// PFLOP/s of a large library product; 72 us for the agent's five matrices in the one-workgroup form.
#include <limits.h>
#include <math.h>

#include <algorithm>

#include "device_utils.hpp"

namespace mctsq {

// Matrices per launch (kernel arguments hold their descriptions).  The agent's largest encoders have 19; 32 costs every launch
// 0.4 us more.
constexpr int MU_GROUP = 20;
constexpr int MU_PARTS = 256;       // workgroups that add up one matrix's squares
constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float PLANE = 16384.0f, UNPLANE = 1.0f / 16384.0f;        // 2^14
constexpr int FRAG = 512;           // halves in a fragment
constexpr int P = 2;                // planes of a matrix: hi and lo

enum { MU_F32 = 0, MU_BF16 = 1 };

struct MuMat {
    int n, m;                       // working shape, n <= m
    int np, mp;                     // padded to the tile
    int rows, cols;                 // the matrix as the caller has it; transposed when rows > cols
    float lrs;                      // learning rate times the shape's factor
    const void* x; int64_t ldx;     // gradient, or the matrix to orthogonalise
    float* mom;                     // momentum [rows][cols], NULL: orthogonalise x
    void* out; int64_t ldo;         // parameters (updated in place), or the result
    _Float16* ws;                   // X old and new, four n x n matrices (MuPlanes), each of two planes
    double* part;                   // MU_PARTS sums of squares
};
struct MuArgs {
    int count, xtype, otype;        // element types of x and, when orthogonalising, out
    float mu, decay; int nesterov;
    double eps;
    int first[MU_GROUP];            // the launch's first workgroup of each matrix (INT_MAX past the last)
    MuMat mat[MU_GROUP];
};
static_assert(sizeof(MuArgs) <= 3584, "kernel arguments");

// the matrix that workgroup b belongs to; without an early exit, so that the scalar loads go out together
__device__ __forceinline__ int mu_which(const MuArgs& a, int b) {
    int w = -1;
#pragma unroll
    for (int i = 0; i < MU_GROUP; ++i) w += a.first[i] <= b;
    return w;
}

__device__ __forceinline__ float mu_load(const void* p, int64_t i, int type) {
    if (type == MU_F32) return reinterpret_cast<const float*>(p)[i];
    return __uint_as_float((unsigned)reinterpret_cast<const unsigned short*>(p)[i] << 16);
}

// ---- momentum and squares ------------------------------------------------------------------------------------------
__device__ __forceinline__ float4 mu_load4(const void* p, int64_t i, int type) {
    if (type == MU_F32) return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    const uint2 b = *reinterpret_cast<const uint2*>(reinterpret_cast<const unsigned short*>(p) + i);
    return make_float4(__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16),
                       __uint_as_float(b.y & 0xffff0000u));
}
__device__ __forceinline__ float mu_update(const MuArgs& a, float g, float& m) {        // new momentum, and u
    m = fmaf(a.mu, m, g);
    return a.nesterov ? fmaf(a.mu, m, g) : m;
}

__global__ __launch_bounds__(256) void mu_norm_kernel(MuArgs a) {
    __shared__ double red[4];
    const MuMat& t = a.mat[blockIdx.y];
    const int64_t total = (int64_t)t.rows * t.cols, tid = (int64_t)blockIdx.x * 256 + threadIdx.x, nt = (int64_t)MU_PARTS * 256;
    double acc = 0.0;
    const int xa = a.xtype == MU_F32 ? 15 : 7;
    const bool flat = t.ldx == t.cols || t.rows == 1;
    int64_t tail = 0;
    if (flat && ((uintptr_t)t.x & xa) == 0 && ((uintptr_t)t.mom & 15) == 0) {
        tail = total & ~(int64_t)3;
        for (int64_t i = tid * 4; i < tail; i += nt * 4) {
            const float4 g = mu_load4(t.x, i, a.xtype);
            float u[4] = {g.x, g.y, g.z, g.w};
            if (t.mom) {
                float4 m4 = *reinterpret_cast<const float4*>(t.mom + i);
                u[0] = mu_update(a, g.x, m4.x); u[1] = mu_update(a, g.y, m4.y);
                u[2] = mu_update(a, g.z, m4.z); u[3] = mu_update(a, g.w, m4.w);
                *reinterpret_cast<float4*>(t.mom + i) = m4;
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) acc = fma((double)u[c], (double)u[c], acc);
        }
    }
    for (int64_t i0 = tail + tid; i0 < total; i0 += 4 * nt) {             // four elements under way
        float g[4], m[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = i0 + u * nt < total ? i0 + u * nt : i0, r = flat ? 0 : i / t.cols;
            g[u] = mu_load(t.x, r * t.ldx + (i - r * t.cols), a.xtype);
            m[u] = t.mom ? t.mom[i] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (i0 + u * nt >= total) continue;
            float v = g[u];
            if (t.mom) {
                v = mu_update(a, g[u], m[u]);
                t.mom[i0 + u * nt] = m[u];
            }
            acc = fma((double)v, (double)v, acc);
        }
    }
    for (int d = 32; d >= 1; d >>= 1) acc += __shfl_xor(acc, d, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) t.part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// From the sum of squares: up = the power of two that brings |u|_F into [1/2, 1), s = the rest of 1 / (|u|_F + eps)
__device__ __forceinline__ void mu_scale_of(double squares, double eps, double& up, float& s) {
    const double norm = sqrt(squares);
    int e = 0;
    if (norm > 0.0 && norm < INFINITY) (void)frexp(norm, &e);
    e = e > 600 ? 600 : (e < -600 ? -600 : e);
    up = ldexp(1.0, -e);
    s = norm == 0.0 ? 0.0f : (float)(ldexp(1.0, e) / (norm + eps));       // a zero matrix stays 0 whatever eps is
}
// the same from the parts of mu_norm_kernel; every lane of a wave gets it
__device__ __forceinline__ void mu_scale(const MuMat& t, double eps, double& up, float& s) {
    double acc = 0.0;
    for (int i = threadIdx.x & 63; i < MU_PARTS; i += 64) acc += t.part[i];
    for (int d = 32; d >= 1; d >>= 1) acc += __shfl_xor(acc, d, 64);
    mu_scale_of(acc, eps, up, s);
}

// ---- planes of X_0 -----------------------------------------------------------------------------------
// element (row, k) of a plane of K columns
__device__ __forceinline__ int64_t frag_at(int row, int k, int K) {
    return ((int64_t)(row >> 4) * (K >> 5) + (k >> 5)) * FRAG + (((row & 15) + 16 * ((k & 31) >> 3)) << 3) + (k & 7);
}
struct MuPlanes {                   // where a matrix's planes are: X twice (old and new), four n x n matrices
    int64_t xs, as;                 // halves from a plane to the next
    _Float16* base;
    __device__ MuPlanes(const MuMat& t) : xs((int64_t)t.np * t.mp), as((int64_t)t.np * t.np), base(t.ws) {}
    __device__ _Float16* X(int cur) const { return base + cur * P * xs; }
    __device__ _Float16* N(int i) const { return base + 2 * P * xs + i * P * as; }
};

__global__ __launch_bounds__(256) void mu_planes_kernel(MuArgs a) {
    __shared__ float tile[64][65];
    const int w = mu_which(a, blockIdx.x);
    const MuMat& t = a.mat[w];
    const int blk = blockIdx.x - a.first[w], nb = t.mp / 64, bi = blk / nb * 64, bj = blk % nb * 64;     // working coordinates
    const bool tr = t.rows > t.cols;
    double up; float s;
    mu_scale(t, a.eps, up, s);
    {
        // x runs along the caller's columns, four at a time
        const int x = (threadIdx.x & 15) * 4, c = (tr ? bi : bj) + x;
        const bool vec = ((uintptr_t)t.x & (a.xtype == MU_F32 ? 15 : 7)) == 0 && (t.ldx & 3) == 0 && (t.cols & 3) == 0
                         && ((uintptr_t)t.mom & 15) == 0;
        const double f = up * (double)PLANE;
#pragma unroll
        for (int y = threadIdx.x >> 4; y < 64; y += 16) {
            const int r = (tr ? bj : bi) + y;
            float u[4] = {0.f, 0.f, 0.f, 0.f};
            if (r < t.rows && c < t.cols) {
                if (vec) {
                    const float4 g = mu_load4(t.x, r * t.ldx + c, a.xtype);
                    u[0] = g.x; u[1] = g.y; u[2] = g.z; u[3] = g.w;
                    if (t.mom) {
                        const float4 m = *reinterpret_cast<const float4*>(t.mom + (int64_t)r * t.cols + c);
                        const float mm[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) u[k] = a.nesterov ? fmaf(a.mu, mm[k], u[k]) : mm[k];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (c + k < t.cols) {
                            u[k] = mu_load(t.x, r * t.ldx + c + k, a.xtype);
                            if (t.mom) {
                                const float m = t.mom[(int64_t)r * t.cols + c + k];
                                u[k] = a.nesterov ? fmaf(a.mu, m, u[k]) : m;
                            }
                        }
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float v = (float)((double)u[k] * f);
                if (tr) tile[x + k][y] = v;
                else tile[y][x + k] = v;
            }
        }
    }
    __syncthreads();
    const MuPlanes pl(t);
    const int lane = threadIdx.x & 63, row = lane & 15, k0 = (lane >> 4) * 8;
#pragma unroll
    for (int f = threadIdx.x >> 6; f < 8; f += 4) {
        const int rt = f >> 1, kb = f & 1;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = tile[rt * 16 + row][kb * 32 + k0 + e];
            hi[e] = (_Float16)v;
            lo[e] = (_Float16)(v - (float)hi[e]);
        }
        _Float16* dst = pl.X(0) + frag_at(bi + rt * 16, bj + kb * 32, t.mp) + lane * 8;
        *reinterpret_cast<f16x8*>(dst) = hi;
        *reinterpret_cast<f16x8*>(dst + pl.xs) = lo;
    }
}

// ---- the products ---------------------------------------------------------------------------------------------------------
// ST_SYM: a product of two n x n symmetric matrices that commute, or X X^T: symmetric.  ST_POLY: a + b A + c A^2.
// ST_NEXT: X <- N X.  ST_LAST: the same into the caller's matrix.
enum { ST_SYM = 0, ST_POLY = 1, ST_NEXT = 2, ST_LAST = 3 };
struct MuStage {
    int r, s, out;                  // the n x n matrices R, S and the result; r = -1: X X^T
    int cur;                        // which X is the old one
    int scaled;                     // X is still u times a power of two: the rest of the normalisation goes in here
    float unit, plane;              // of the operands' scales, of the result's
};

// tiles of an np x cols product; of a symmetric one the tiles that reach the diagonal or lie below it
template <int TI, int TJ>
__host__ __device__ inline int mu_row_tiles(int np, int ti) {
    const int last = ti * TI + TI < np ? ti * TI + TI : np;              // rows of this tile row end here
    return (last + TJ - 1) / TJ;
}
template <int TI, int TJ>
__host__ __device__ inline int mu_tiles(int np, int cols, bool sym) {
    const int nti = (np + TI - 1) / TI;
    if (!sym) return nti * ((cols + TJ - 1) / TJ);
    // full tile rows: (ti + 1) TI / TJ tiles each, the last one by its own end
    return nti * (nti - 1) / 2 * (TI / TJ) + mu_row_tiles<TI, TJ>(np, nti - 1);
}

// C[i][j] = sum_k R[i][k] S[j][k] over fragments of R and S: a TI x TJ tile by 2 x 2 waves, a k block of 32 at a time.
// Three LDS buffers: while block k is multiplied from registers, block k + 1 is read from LDS into a second set of registers,
// blocks k + 2 and k + 3 are on their way from memory.  The buffers are variables of their own, so that the compiler knows that
// a read of one does not touch what is being fetched into another.
template <int TI, int TJ>
struct MuTile {
    static constexpr int WI = TI / 32, WJ = TJ / 32;                     // 16 x 16 tiles of a wave
    static constexpr int FI = P * TI / 16, F = FI + P * TJ / 16;         // fragments of a k block: of R, of both
    static constexpr int L = F / 4;                                      // a wave's share of the fetch
    static constexpr int BUF = F * FRAG;                                 // halves in a buffer
    static constexpr int NB = 3;
    // epilogue: bytes of a 16 x 16 tile in LDS, and how many rows of them fit a wave's half buffer
    static constexpr int SUB = 1024 + 64;
    static constexpr int QI = BUF / SUB / WJ >= 4 && WI >= 4 ? 4 : BUF / SUB / WJ >= 2 && WI >= 2 ? 2 : 1;
    static_assert(QI * WJ * SUB <= BUF && WI % QI == 0, "epilogue");
    static_assert(F % 4 == 0 && NB * BUF * 2 <= 160 * 1024, "LDS");
};

// Reads, fetches and products of a step one by one among each other: in a row they hold the wave up
template <int D, int L, int M, int I = 0>
__device__ __forceinline__ void mu_interleave() {
    if constexpr (I < L) {
        constexpr int d0 = I * D / L, d1 = (2 * I + 1) * D / (2 * L), d2 = (I + 1) * D / L;
        constexpr int m0 = I * M / L, m1 = (2 * I + 1) * M / (2 * L), m2 = (I + 1) * M / L;
        if constexpr (d1 > d0) __builtin_amdgcn_sched_group_barrier(0x100, d1 - d0, 0);
        if constexpr (m1 > m0) __builtin_amdgcn_sched_group_barrier(0x008, m1 - m0, 0);
        if constexpr (d2 > d1) __builtin_amdgcn_sched_group_barrier(0x100, d2 - d1, 0);
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
        if constexpr (m2 > m1) __builtin_amdgcn_sched_group_barrier(0x008, m2 - m1, 0);
        mu_interleave<D, L, M, I + 1>();
    }
}

// TR: k runs over S's rows (X itself, in place of its transpose), `stiles` tiles of 16 columns wide.  Its fragments are
// read from LDS transposed, groups of 16 lanes taking four rows of 16; every other octet's rows are fetched four places
// on, so that such a group finds its 128 bytes in different banks.
template <int TI, int TJ, bool TR>
__device__ __forceinline__ void mu_tile(const _Float16* R, int64_t rs, int rtiles, const _Float16* S, int64_t ss, int stiles,
                                        int KB, int ti, int tj, f32x4 (&acc)[MuTile<TI, TJ>::WI][MuTile<TI, TJ>::WJ],
                                        _Float16* b0, _Float16* b1, _Float16* b2) {
    using C = MuTile<TI, TJ>;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wi = wave >> 1, wj = wave & 1;
    const int place = TR ? (((lane & 15) ^ ((lane >> 4 & 1) << 2)) + (lane & 48)) * 8 : lane * 8;
    const _Float16* src[C::L];                   // this wave's fragments of block 0; rows past the matrix: its last tile again
#pragma unroll
    for (int l = 0; l < C::L; ++l) {
        const int f = wave * C::L + l;
        if (f < C::FI) {
            const int p = f / (TI / 16), rt = min(ti * (TI / 16) + f % (TI / 16), rtiles - 1);
            src[l] = R + p * rs + (int64_t)rt * KB * FRAG;
        } else {
            const int g = f - C::FI, p = g / (TJ / 16), i = g % (TJ / 16);
            if constexpr (TR) {
                const int e = i / (TJ / 32), jb = min(tj * (TJ / 32) + i % (TJ / 32), stiles / 2 - 1);
                src[l] = S + p * ss + ((int64_t)e * (stiles / 2) + jb) * FRAG;
            } else src[l] = S + p * ss + (int64_t)min(tj * (TJ / 16) + i, stiles - 1) * KB * FRAG;
        }
    }
    auto fetch = [&](int kb, _Float16* buf) {
        kb = kb < KB ? kb : KB - 1;              // past the end: the last block again, so that the counts below hold
        const int64_t rk = (int64_t)kb * FRAG, sk = TR ? rk * stiles : rk;
#pragma unroll
        for (int l = 0; l < C::L; ++l)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(wave * C::L + l < C::FI ? src[l] + rk + lane * 8 : src[l] + sk + place),
                                             (__attribute__((address_space(3))) void*)(buf + (wave * C::L + l) * FRAG), 16, 0, 0);
    };
    struct Frags { u32x4 r[P][C::WI], s[P][C::WJ]; };
    // this lane's two places in a transposed read of the even 16 columns of a k block of X
    const int g = lane & 15, quad = lane >> 4, par = g >> 1 & 1;
    const int t0 = ((quad >> 1) * (TJ / 32)) * FRAG + ((quad & 1) * 8 + (g >> 2) + 16 * par) * 8 + (g & 1) * 4;
    const int tr0 = t0 + par * 32, tr1 = t0 + (1 - par) * 32;
    auto read = [&](Frags& f, _Float16* buf) {
        const u32x4* b = reinterpret_cast<const u32x4*>(buf) + lane;
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < C::WI; ++i) f.r[p][i] = b[(p * (TI / 16) + wi * C::WI + i) * 64];
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int j = 0; j < C::WJ; ++j) {
                if constexpr (TR) {
                    const int jt = wj * C::WJ + j;
                    typedef short s16x4 __attribute__((ext_vector_type(4)));
                    _Float16* at = buf + (C::FI + p * (TJ / 16) + jt / 2) * FRAG + (jt & 1) * 256;
                    union { s16x4 h[2]; u32x4 u; } v;
                    v.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + tr0));
                    v.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + tr1));
                    f.s[p][j] = v.u;
                } else f.s[p][j] = b[(C::FI + p * (TJ / 16) + wj * C::WJ + j) * 64];
            }
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int j = 0; j < C::WJ; ++j) {
#pragma unroll
            for (int i = 0; i < C::WI; ++i) acc[i][j] = mfma_h(f.r[1][i], f.s[0][j], acc[i][j]);
#pragma unroll
            for (int i = 0; i < C::WI; ++i) acc[i][j] = mfma_h(f.r[0][i], f.s[1][j], acc[i][j]);
#pragma unroll
            for (int i = 0; i < C::WI; ++i) acc[i][j] = mfma_h(f.r[0][i], f.s[0][j], acc[i][j]);
        }
    };
    // this wave's part of the oldest fetch under way has arrived, its own LDS reads are done; then everyone's are
    auto arrive = [&]() {
        __builtin_amdgcn_s_waitcnt((C::L & 15) | (C::L >> 4) << 14 | 0x0070);        // vmcnt(L), lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
    };
    // multiply block k (in `cur`), read block k + 1 from `next`, fetch block k + 3 into `free`, which held block k
    auto step = [&](int k, const Frags& cur, Frags& other, _Float16* next, _Float16* free) {
        arrive();
        fetch(k + 3, free);
        read(other, next);
        multiply(cur);
        mu_interleave<P * (C::WI + (TR ? 2 : 1) * C::WJ), C::L, 3 * C::WI * C::WJ>();
    };
#pragma unroll
    for (int i = 0; i < C::WI; ++i)
#pragma unroll
        for (int j = 0; j < C::WJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    Frags x, y;
    fetch(0, b0);
    fetch(1, b1);
    arrive();
    fetch(2, b2);
    read(x, b0);
    int k = 0;
    for (; k + 6 <= KB; k += 6) {
        step(k, x, y, b1, b0); step(k + 1, y, x, b2, b1); step(k + 2, x, y, b0, b2);
        step(k + 3, y, x, b1, b0); step(k + 4, x, y, b2, b1); step(k + 5, y, x, b0, b2);
    }
    if (k < KB) step(k, x, y, b1, b0);
    if (k + 1 < KB) step(k + 1, y, x, b2, b1);
    if (k + 2 < KB) step(k + 2, x, y, b0, b2);
    if (k + 3 < KB) step(k + 3, y, x, b1, b0);
    if (k + 4 < KB) step(k + 4, x, y, b2, b1);
    __builtin_amdgcn_s_waitcnt(0x0f70);          // nothing is under way into this workgroup's LDS when it ends
}

// four consecutive values along k of one row: stored as hi (and lo), and read back
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void split4(const float* v, f16x4& h, f16x4& l, float plane = PLANE) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        h[r] = (_Float16)(v[r] * plane);
        l[r] = (_Float16)(v[r] * plane - (float)h[r]);
    }
}
struct Quad4 { f16x4 p[P]; };
__device__ __forceinline__ Quad4 plane_load(const _Float16* at, int64_t ps) {
    Quad4 q;
#pragma unroll
    for (int p = 0; p < P; ++p) q.p[p] = *reinterpret_cast<const f16x4*>(at + p * ps);
    return q;
}
__device__ __forceinline__ float plane_value(const Quad4& q, int r) {
    return ((float)q.p[0][r] + (float)q.p[1][r]) * UNPLANE;
}

// `count` (at most four; four where vec is set) results in a row of the caller's matrix, from column c on
__device__ __forceinline__ void mu_put(const MuArgs& a, const MuMat& t, int row, int c, const float* v, bool vec, int count = 4) {
    if (row >= t.rows || c >= t.cols) return;
    const int64_t at = (int64_t)row * t.ldo + c;
    const int end = t.cols - c < count ? t.cols - c : count;
    if (t.mom) {
        float* p = reinterpret_cast<float*>(t.out) + at;
        if (vec) {
            float4 q = *reinterpret_cast<const float4*>(p);
            q.x = fmaf(q.x, a.decay, -t.lrs * v[0]); q.y = fmaf(q.y, a.decay, -t.lrs * v[1]);
            q.z = fmaf(q.z, a.decay, -t.lrs * v[2]); q.w = fmaf(q.w, a.decay, -t.lrs * v[3]);
            *reinterpret_cast<float4*>(p) = q;
        } else
#pragma unroll
            for (int k = 0; k < 4; ++k) if (k < end) p[k] = fmaf(p[k], a.decay, -t.lrs * v[k]);
    } else if (a.otype == MU_F32) {
        float* p = reinterpret_cast<float*>(t.out) + at;
        if (vec) *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else
#pragma unroll
            for (int k = 0; k < 4; ++k) if (k < end) p[k] = v[k];
    } else {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        __bf16* p = reinterpret_cast<__bf16*>(t.out) + at;
        bf16x4 q;
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = (__bf16)(k < count ? v[k] : 0.0f);
        if (vec) *reinterpret_cast<bf16x4*>(p) = q;
        else
#pragma unroll
            for (int k = 0; k < 4; ++k) if (k < end) p[k] = q[k];
    }
}

template <int TI, int TJ, int ST>
__global__ __launch_bounds__(256) void mu_product_kernel(MuArgs a, MuStage g) {
    using C = MuTile<TI, TJ>;
    __shared__ __attribute__((aligned(16))) _Float16 b0[C::BUF], b1[C::BUF], b2[C::BUF];
    constexpr bool sym = ST == ST_SYM || ST == ST_POLY;
    const int w = mu_which(a, blockIdx.x), n = mu_tiles<TI, TJ>(a.mat[w].np, sym ? a.mat[w].np : a.mat[w].mp, sym);
    // workgroups go round the eight XCDs: of every matrix each XCD gets a run of neighbouring tiles, which share operands
    // in its L2
    const int lb = blockIdx.x - a.first[w], q = n >> 3, rest = n & 7, x = lb & 7;
    const int b = x * q + (x < rest ? x : rest) + (lb >> 3);
    const MuMat& t = a.mat[w];
    const MuPlanes pl(t);
    int ti, tj;
    {
        const int nti = (t.np + TI - 1) / TI, ntj = (t.mp + TJ - 1) / TJ;
        if (sym) {                   // tile row ti has the tiles that reach below the diagonal
            int c = b;
            for (ti = 0; c >= mu_row_tiles<TI, TJ>(t.np, ti); ++ti) c -= mu_row_tiles<TI, TJ>(t.np, ti);
            tj = c;
        } else {                     // bands of 8 tile rows, column by column
            const int band = b / (8 * ntj), h = nti - band * 8 < 8 ? nti - band * 8 : 8, c = b - band * 8 * ntj;
            ti = band * 8 + c % h; tj = c / h;
        }
    }
    const int nt = t.np / 16, mt = t.mp / 16;
    f32x4 acc[C::WI][C::WJ];
    if constexpr (sym) {
        const bool gram = ST == ST_SYM && g.r < 0;                        // X X^T: k runs along m
        const _Float16 *R = gram ? pl.X(g.cur) : pl.N(g.r), *S = gram ? pl.X(g.cur) : pl.N(g.s);
        const int64_t ps = gram ? pl.xs : pl.as;
        mu_tile<TI, TJ, false>(R, ps, nt, S, ps, nt, (gram ? t.mp : t.np) / 32, ti, tj, acc, b0, b1, b2);
    } else mu_tile<TI, TJ, true>(pl.N(g.r), pl.as, nt, pl.X(g.cur), pl.xs, mt, t.np / 32, ti, tj, acc, b0, b1, b2);

    // Lane (quad, col) holds rows 4 quad .. + 3 of column col of every 16 x 16 tile.  The results go through LDS and leave it
    // in short loops: read eight along a row, two tiles at a time, they are whole fragments; as they lie they are four
    // neighbours along k of the mirrored place (half a fragment by the wave), which symmetric results need too.
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), quad = lane >> 4, col = lane & 15;
    float s = 1.0f;
    if (g.scaled) { double up; mu_scale(t, a.eps, up, s); }
    const float unit = g.unit * (sym ? s * s : s);
    const int lane4 = (col + 16 * (quad >> 1)) * 8 + (quad & 1) * 4;     // this lane's place in a half fragment
    const int i0 = ti * (TI / 16) + (wave >> 1) * C::WI, j0 = tj * (TJ / 16) + (wave & 1) * C::WJ;
    // the A that c A^2 is added to: all of this wave's loads at once, as nothing else hides them
    Quad4 old[ST == ST_POLY ? C::WI : 1][C::WJ];
    if constexpr (ST == ST_POLY)
#pragma unroll
        for (int i = 0; i < C::WI; ++i)
#pragma unroll
            for (int j = 0; j < C::WJ; ++j) {
                const int i16 = min(i0 + i, nt - 1), j16 = min(j0 + j, nt - 1);
                old[i][j] = plane_load(pl.N(g.r) + ((int64_t)j16 * (t.np >> 5) + (i16 >> 1)) * FRAG + (i16 & 1) * 256 + lane4, pl.as);
            }
    __syncthreads();                                                     // the operands in LDS are done with
    // a wave's own 16 x 16 tiles, QI rows of them at a time; 16 bytes after every 16 lanes and every tile starts 16 banks
    // on, so that neither way of reading runs into bank conflicts
    char* own = reinterpret_cast<char*>(wave & 1 ? b1 : b0) + (wave >> 1) * C::BUF;          // half a buffer
    const bool tr = t.rows > t.cols;
    const bool vec = ST == ST_LAST && (t.ldo & 3) == 0 && (t.cols & 3) == 0 && ((uintptr_t)t.out & (t.mom || a.otype == MU_F32 ? 15 : 7)) == 0;
#pragma unroll
    for (int c = 0; c < C::WI; c += C::QI) {
#pragma unroll
        for (int q = 0; q < C::QI; ++q)
#pragma unroll
            for (int j = 0; j < C::WJ; ++j) {
                f32x4 v = acc[c + q][j];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    v[r] *= unit;
                    if constexpr (ST == ST_POLY) {                       // A is symmetric: read as it lies, (column, row)
                        v[r] = fmaf(NS_C, v[r], NS_B * plane_value(old[c + q][j], r));
                        if (i0 + c + q == j0 + j && 4 * quad + r == col) v[r] += NS_A;
                    }
                }
                *reinterpret_cast<f32x4*>(own + (q * C::WJ + j) * C::SUB + lane * 16 + quad * 16) = v;
            }
        asm volatile("" ::: "memory");           // a wave's LDS accesses are served in order: only the compiler must keep it
        constexpr int N = C::QI * C::WJ, U = N >= 4 ? 4 : N;             // U tiles' LDS reads under way at once
        if (sym || (ST == ST_LAST && tr))
            for (int e0 = 0; e0 < N; e0 += U) {
                f32x4 v4[U];
#pragma unroll
                for (int u = 0; u < U; ++u) v4[u] = *reinterpret_cast<const f32x4*>(own + (e0 + u) * C::SUB + lane * 16 + quad * 16);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i16 = i0 + c + (e0 + u) / C::WJ, j16 = j0 + (e0 + u) % C::WJ;
                    const bool in = i16 < nt && j16 <= (sym ? i16 : mt - 1);
                    const float v[4] = {v4[u][0], v4[u][1], v4[u][2], v4[u][3]};
                    if constexpr (ST == ST_LAST) {
                        if (in) mu_put(a, t, j16 * 16 + col, i16 * 16 + 4 * quad, v, vec);
                    } else {
                        f16x4 h, l;
                        split4(v, h, l, g.plane);
                        _Float16* out = pl.N(g.out) + ((int64_t)j16 * (t.np >> 5) + (i16 >> 1)) * FRAG + (i16 & 1) * 256 + lane4;
                        if (in) {
                            *reinterpret_cast<f16x4*>(out) = h;
                            *reinterpret_cast<f16x4*>(out + pl.as) = l;
                        }
                    }
                }
            }
        constexpr int U2 = N / 2 >= 4 ? 4 : N / 2;
        if (ST != ST_LAST || !tr)
            for (int e0 = 0; e0 < N / 2; e0 += U2) {
                // fragments: row lane & 15, octet lane >> 4 of the 32 columns; the result matrix: four lanes to a row
                const int row = ST == ST_LAST ? lane >> 2 : lane & 15, oct = ST == ST_LAST ? lane & 3 : lane >> 4;
                const char* src = own + (2 * e0 + (oct >> 1)) * C::SUB + ((oct & 1) * 8 + 16 * (row >> 2)) * 16 + (row >> 2) * 16 + (row & 3) * 4;
                float v[U2][8];
#pragma unroll
                for (int u = 0; u < U2; ++u)
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[u][k] = *reinterpret_cast<const float*>(src + u * 2 * C::SUB + k * 16);
#pragma unroll
                for (int u = 0; u < U2; ++u) {
                    const int i16 = i0 + c + (e0 + u) / (C::WJ / 2), jp = j0 + (e0 + u) % (C::WJ / 2) * 2;
                    const bool in = i16 < nt && jp <= (sym ? i16 : mt - 1);
                    if constexpr (ST == ST_LAST) {
                        if (in) {
                            mu_put(a, t, i16 * 16 + row, jp * 16 + oct * 8, v[u], vec);
                            mu_put(a, t, i16 * 16 + row, jp * 16 + oct * 8 + 4, v[u] + 4, vec);
                        }
                    } else {
                        const float plane = sym ? g.plane : PLANE;
                        f16x8 h, l;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            h[k] = (_Float16)(v[u][k] * plane);
                            l[k] = (_Float16)(v[u][k] * plane - (float)h[k]);
                        }
                        _Float16* out = (sym ? pl.N(g.out) : pl.X(g.cur ^ 1)) + ((int64_t)i16 * ((sym ? t.np : t.mp) >> 5) + (jp >> 1)) * FRAG + lane * 8;
                        if (in && (!sym || jp + (lane >> 5) < i16)) {    // on the diagonal the loop above stored the whole tile
                            *reinterpret_cast<f16x8*>(out) = h;
                            *reinterpret_cast<f16x8*>(out + (sym ? pl.as : pl.xs)) = l;
                        }
                    }
                }
            }
        asm volatile("" ::: "memory");
    }
}

// ---- small matrices: all of it in one workgroup ---------------------------------------------------------------------
// X and A (then B over A) of one matrix stay in LDS as fragments, 16 waves share the products in blocks of 32 x 32, results
// wait in registers until everyone has read the operands they replace.  X is kept one way only: where k runs along its rows
// the fragments are read with the transposing LDS read.  One launch for norm, five steps and update; the launches of the
// general path cost 60 to 110 us whatever the size.  Measured, this way and that: 64 x 64 28 and 71 us, 64 x 192 37 and 80,
// 128 x 192 69 and 88, 32 x 1000 73 and 103; the agent's five matrices 73 and 110.  Of 128 x 192's step (25 k cycles) the
// products are half, bound by LDS reads; the rest is waiting for the slowest wave and storing.
constexpr int MU_SMALL_LDS = 160 * 1024;
constexpr int MU_SMALL_NEXT = 2, MU_SMALL_SYM = 1;       // most blocks a wave gets

struct MuOperands { u32x4 r[P][2], c[P][2]; };
// k blocks one after the other, the next one's operands read while the current one is multiplied
template <typename Load, typename Multiply>
__device__ __forceinline__ void mu_blocks(int K, const Load& load, const Multiply& multiply) {
    MuOperands x, y;
    load(x, 0);
#pragma unroll 1
    for (int k = 0; k < K; k += 2) {
        load(y, k + 1 < K ? k + 1 : k);
        multiply(x);
        if (k + 1 == K) break;
        load(x, k + 2 < K ? k + 2 : k);
        multiply(y);
    }
}

static bool mu_is_small(int64_t rows, int64_t cols) {
    const int64_t n = round_up(rows < cols ? rows : cols, 32), m = round_up(rows < cols ? cols : rows, 32);
    const int64_t ni = n / 32, mi = m / 32;
    return 2 * P * (n * m + n * n) <= MU_SMALL_LDS && ni * mi <= 16 * MU_SMALL_NEXT
           && ni * (ni + 1) / 2 <= 16 * MU_SMALL_SYM;
}

__global__ __launch_bounds__(1024) void mu_small_kernel(MuArgs a) {
    __shared__ __attribute__((aligned(16))) _Float16 lds[MU_SMALL_LDS / 2];
    const MuMat& t = a.mat[blockIdx.x];
    int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int np = (t.n + 31) & ~31, mp = (t.m + 31) & ~31, nb = np / 32, mb = mp / 32;
    const int xs = np * mp, as = np * np;                 // a plane's halves
    _Float16 *X = lds, *A = lds + P * xs;
    const bool tr = t.rows > t.cols;

    // momentum, norm; X's planes cleared meanwhile (padding stays 0)
    for (int i = threadIdx.x; i < P * xs / 8; i += 1024) reinterpret_cast<u32x4*>(X)[i] = u32x4{0, 0, 0, 0};
    // A wave takes every 16th row, a lane its columns: nothing to divide, rows' addresses are scalar.  Four rows under way at
    // once: one workgroup has nobody else to wait with.
    constexpr int U = 4;
    double acc64 = 0.0;
    for (int r0 = wave; r0 < t.rows; r0 += 16 * U)
        for (int c = lane; c < t.cols; c += 64) {
            float g[U], m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = min(r0 + 16 * u, t.rows - 1);
                g[u] = mu_load(t.x, r * t.ldx + c, a.xtype);
                m[u] = t.mom ? t.mom[r * t.cols + c] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r0 + 16 * u >= t.rows) continue;
                float v = g[u];
                if (t.mom) {
                    v = mu_update(a, g[u], m[u]);
                    t.mom[(r0 + 16 * u) * t.cols + c] = m[u];
                }
                acc64 = fma((double)v, (double)v, acc64);
            }
        }
    for (int d = 32; d >= 1; d >>= 1) acc64 += __shfl_xor(acc64, d, 64);
    double* red = reinterpret_cast<double*>(A);
    if (lane == 0) red[wave] = acc64;
    __syncthreads();
    double sum = 0.0;
    for (int i = 0; i < 16; ++i) sum += red[i];
    double up; float s;
    mu_scale_of(sum, a.eps, up, s);
    // up * 2^14 as two fp32 powers of two: the product is exact wherever it matters (below 2^-126 nothing is left of it)
    int e = (int)(__builtin_bit_cast(uint64_t, up) >> 52) - 1023 + 14;
    e = e < -250 ? -250 : (e > 250 ? 250 : e);
    const float f0 = pow2i(e >> 1), f1 = pow2i(e - (e >> 1));
    for (int r0 = wave; r0 < t.rows; r0 += 16 * U)
        for (int c = lane; c < t.cols; c += 64) {
            float g[U], m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = min(r0 + 16 * u, t.rows - 1);
                g[u] = mu_load(t.x, r * t.ldx + c, a.xtype);
                m[u] = t.mom ? t.mom[r * t.cols + c] : 0.0f;             // written by this thread above
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + 16 * u;
                if (r >= t.rows) continue;
                const float w = !t.mom ? g[u] : a.nesterov ? fmaf(a.mu, m[u], g[u]) : m[u], v = w * f0 * f1;
                const int row = tr ? c : r, k = tr ? r : c;
                _Float16* o = X + ((row >> 4) * mb + (k >> 5)) * FRAG + (((row & 15) + 16 * ((k & 31) >> 3)) << 3) + (k & 7);
                const _Float16 h = (_Float16)v;
                o[0] = h;
                o[xs] = (_Float16)(v - (float)h);
            }
        }
    __syncthreads();

    const int sym = nb * (nb + 1) / 2, full = nb * mb;
    // fragment (row tile, k block) of a plane whose k extent is K blocks
    auto frag = [&](const _Float16* p, int rt, int kb, int K) {
        return *reinterpret_cast<const u32x4*>(p + (rt * K + kb) * FRAG + lane * 8);
    };
    // rows j = 16 jt .. + 15, k = 32 ib .. + 31 of X transposed: groups of 16 lanes read four rows of 16 and get columns
    auto frag_tr = [&](const _Float16* p, int jt, int ib) {
        const int g = lane & 15, j = jt * 16 + (g & 3) * 4, rt = 2 * ib + (lane >> 5);
        const _Float16* at = p + (rt * mb + (j >> 5)) * FRAG + ((((lane >> 4) & 1) * 8 + (g >> 2)) + 16 * ((j & 31) >> 3)) * 8 + (j & 7);
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        union { s16x4 h[2]; u32x4 u; } r;
        r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
        r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at + 4 * 8));
        return r.u;
    };
    // lower-triangle block b of the symmetric products
    auto block = [&](int b, int& bi, int& bj) {
        for (bi = 0; b > bi; ++bi) b -= bi + 1;
        bj = b;
    };
#pragma unroll 1
    for (int it = 0; it < 5; ++it) {
        asm volatile("" : "+v"(lane));           // addresses are made anew: kept over the steps they spill
        const float sc = it == 0 ? s : 1.0f;
#pragma unroll 1
        for (int st = ST_SYM; st <= ST_POLY; ++st) {     // A = X X^T, then B = a + b A + c A^2 over it
            const _Float16* src = st == ST_SYM ? X : A;
            const int64_t ps = st == ST_SYM ? xs : as;
            const int K = st == ST_SYM ? mb : nb;
            f32x4 acc[MU_SMALL_SYM][2][2];
#pragma unroll
            for (int q = 0; q < MU_SMALL_SYM; ++q) {
                const int b = wave + 16 * q;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[q][e >> 1][e & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (b >= sym) continue;
                int bi, bj;
                block(b, bi, bj);
                auto load = [&](MuOperands& o, int k) {
#pragma unroll
                    for (int p = 0; p < P; ++p)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            o.r[p][e] = frag(src + p * ps, 2 * bi + e, k, K);
                            o.c[p][e] = frag(src + p * ps, 2 * bj + e, k, K);
                        }
                };
                mu_blocks(K, load, [&](const MuOperands& o) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[q][e >> 1][e & 1] = mfma_h(o.r[1][e >> 1], o.c[0][e & 1], acc[q][e >> 1][e & 1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[q][e >> 1][e & 1] = mfma_h(o.r[0][e >> 1], o.c[1][e & 1], acc[q][e >> 1][e & 1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[q][e >> 1][e & 1] = mfma_h(o.r[0][e >> 1], o.c[0][e & 1], acc[q][e >> 1][e & 1]);
                });
                const float unit = UNPLANE * UNPLANE * (st == ST_SYM ? sc * sc : 1.0f);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i16 = 2 * bi + (e >> 1), j16 = 2 * bj + (e & 1);
                    f32x4& v = acc[q][e >> 1][e & 1];
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] *= unit;
                    if (st == ST_POLY) {
                        const Quad4 o = plane_load(A + frag_at(j16 * 16 + (lane & 15), i16 * 16 + (lane >> 4) * 4, np), as);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            v[x] = fmaf(NS_C, v[x], NS_B * plane_value(o, x));
                            if (i16 == j16 && (lane >> 4) * 4 + x == (lane & 15)) v[x] += NS_A;
                        }
                    }
                }
            }
            __syncthreads();                              // everyone has read A
#pragma unroll
            for (int q = 0; q < MU_SMALL_SYM; ++q) {
                const int b = wave + 16 * q;
                if (b >= sym) continue;
                int bi, bj;
                block(b, bi, bj);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i16 = 2 * bi + (e >> 1), j16 = 2 * bj + (e & 1);
                    if (j16 > i16) continue;
                    const float v[4] = {acc[q][e >> 1][e & 1][0], acc[q][e >> 1][e & 1][1], acc[q][e >> 1][e & 1][2], acc[q][e >> 1][e & 1][3]};
                    f16x4 h, l;
                    split4(v, h, l);
                    _Float16* o = A + frag_at(j16 * 16 + (lane & 15), i16 * 16 + (lane >> 4) * 4, np);
                    *reinterpret_cast<f16x4*>(o) = h;
                    *reinterpret_cast<f16x4*>(o + as) = l;
                    if (i16 != j16) {
                        o = A + frag_at(i16 * 16 + (lane >> 4) * 4, j16 * 16 + (lane & 15), np);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {     // rows 8 halves apart
                            o[x * 8] = h[x];
                            o[x * 8 + as] = l[x];
                        }
                    }
                }
            }
            __syncthreads();
        }
        // X <- B X; the instruction's rows are X's columns, so that a lane ends with four neighbours of one row
        f32x4 acc[MU_SMALL_NEXT][2][2];
#pragma unroll
        for (int q = 0; q < MU_SMALL_NEXT; ++q) {
            const int b = wave + 16 * q, bi = b % nb, bj = b / nb;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[q][e >> 1][e & 1] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (b >= full) continue;
            auto load = [&](MuOperands& o, int k) {
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        o.r[p][e] = frag(A + p * as, 2 * bi + e, k, nb);
                        o.c[p][e] = frag_tr(X + p * xs, 2 * bj + e, k);
                    }
            };
            mu_blocks(nb, load, [&](const MuOperands& o) {
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[q][e >> 1][e & 1] = mfma_h(o.c[0][e & 1], o.r[1][e >> 1], acc[q][e >> 1][e & 1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[q][e >> 1][e & 1] = mfma_h(o.c[1][e & 1], o.r[0][e >> 1], acc[q][e >> 1][e & 1]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[q][e >> 1][e & 1] = mfma_h(o.c[0][e & 1], o.r[0][e >> 1], acc[q][e >> 1][e & 1]);
            });
        }
        __syncthreads();                                  // everyone has read X
        const bool vec = (t.ldo & 3) == 0 && (t.cols & 3) == 0 && ((uintptr_t)t.out & (t.mom || a.otype == MU_F32 ? 15 : 7)) == 0;
#pragma unroll
        for (int q = 0; q < MU_SMALL_NEXT; ++q) {
            const int b = wave + 16 * q, bi = b % nb, bj = b / nb;
            if (b >= full) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int gi = (2 * bi + (e >> 1)) * 16 + (lane & 15), gj = (2 * bj + (e & 1)) * 16 + (lane >> 4) * 4;
                float v[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) v[x] = acc[q][e >> 1][e & 1][x] * (UNPLANE * UNPLANE * sc);
                if (it < 4) {
                    f16x4 h, l;
                    split4(v, h, l);
                    _Float16* o = X + frag_at(gi, gj, mp);
                    *reinterpret_cast<f16x4*>(o) = h;
                    *reinterpret_cast<f16x4*>(o + xs) = l;
                } else if (!tr) mu_put(a, t, gi, gj, v, vec);
                else
#pragma unroll
                    for (int x = 0; x < 4; ++x) mu_put(a, t, gj + x, gi, v + x, false, 1);
            }
        }
        __syncthreads();
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
constexpr int MU_PAD = 64;          // sides are padded to this; larger tiles repeat the last rows and drop them

static int64_t mu_matrix_bytes(int64_t rows, int64_t cols) {
    const int64_t n = rows < cols ? rows : cols, m = rows < cols ? cols : rows;
    const int64_t np = round_up(n, MU_PAD), mp = round_up(m, MU_PAD);
    return round_up(2 * P * (2 * np * mp + 4 * np * np), 256) + MU_PARTS * 8;
}
static int64_t mu_group_bytes(const mctsq_muon_matrix* mats, int count) {
    int64_t o = 0;
    for (int i = 0; i < count; ++i) o += mu_matrix_bytes(mats[i].rows, mats[i].cols);
    return o;
}
static int mu_check_shapes(const mctsq_muon_matrix* mats, int64_t count) {
    MCTSQ_CHECK(count >= 0 && count <= (1 << 20) && (mats || count == 0), "bad matrix list");
    for (int64_t i = 0; i < count; ++i)
        MCTSQ_CHECK(mats[i].rows >= 1 && mats[i].cols >= 1 && mats[i].rows <= 65536 && mats[i].cols <= 65536,
                    "matrix %lld is %lld x %lld: sides must lie in 1..65536", (long long)i, (long long)mats[i].rows,
                    (long long)mats[i].cols);
    return 0;
}
static int64_t mu_bytes(const mctsq_muon_matrix* mats, int64_t count) {
    int64_t need = 0;                                    // the groups run one after the other in the same space
    for (int64_t g = 0; g < count; g += MU_GROUP) {
        const int64_t b = mu_group_bytes(mats + g, (int)(count - g < MU_GROUP ? count - g : MU_GROUP));
        need = b > need ? b : need;
    }
    return need < 256 ? 256 : need;
}

// One product stage as tiles of TI x TJ: workgroups, and an estimate of its time in us from what was measured (CUs work off
// `load` tiles each; a k block takes `step`, a tile's start and end `over`; up to `share` workgroups share a CU's pauses)
template <int TI, int TJ>
static double mu_stage(MuArgs& a, bool sym, bool gram, double step, double over, int share, int& tiles) {
    tiles = 0;
    double work = 0.0;
    for (int i = 0; i < MU_GROUP; ++i) {
        a.first[i] = i < a.count ? tiles : INT_MAX;
        if (i >= a.count) continue;
        const int n = mu_tiles<TI, TJ>(a.mat[i].np, sym ? a.mat[i].np : a.mat[i].mp, sym);
        tiles += n;
        work += (double)n * ((gram ? a.mat[i].mp : a.mat[i].np) / 32);
    }
    const int load = (tiles + 255) / 256;
    return work / tiles * step * load + over * ((load + share - 1) / share);
}
// Launches the stage on the tiles that the estimate prefers, or only estimates it.
template <int ST>
static double mu_product(MuArgs& a, const MuStage& g, hipStream_t st, bool launch) {
    constexpr bool sym = ST == ST_SYM || ST == ST_POLY;
    const bool gram = ST == ST_SYM && g.r < 0;
    // 256 x 128 tiles 0.87 us a k block (0.73 at the matrix pipe's rate) and 23 a tile, 128 x 128 0.50 and 15, 64 x 64 0.20 and
    // 8 with three to a CU
    int tiles;
    const double t256 = mu_stage<256, 128>(a, sym, gram, 0.87, 23, 1, tiles);
    const double t128 = mu_stage<128, 128>(a, sym, gram, 0.50, 15, 1, tiles);
    const double t64 = mu_stage<64, 64>(a, sym, gram, 0.20, 8, 3, tiles);              // a.first as for 64 x 64
    const double best = std::min(t64, std::min(t128, t256));
    if (!launch) return best;
    if (t64 == best) {
        hipLaunchKernelGGL((mu_product_kernel<64, 64, ST>), dim3(tiles), dim3(256), 0, st, a, g);
    } else if (t128 == best) {
        mu_stage<128, 128>(a, sym, gram, 0, 0, 1, tiles);
        hipLaunchKernelGGL((mu_product_kernel<128, 128, ST>), dim3(tiles), dim3(256), 0, st, a, g);
    } else {
        mu_stage<256, 128>(a, sym, gram, 0, 0, 1, tiles);
        hipLaunchKernelGGL((mu_product_kernel<256, 128, ST>), dim3(tiles), dim3(256), 0, st, a, g);
    }
    return best;
}

// `chain` steps at once, from X_cur to the other X (or the caller's matrix).  The A of a step is a polynomial of the A of the
// step before it, A' = Q A Q with Q = a + b A + c A^2, as X' = Q X; so the chain needs X only at its ends:
//   A = X X^T;  per step Q = a + b A + c A^2, N <- Q N, A <- (Q A) Q;  X <- N X
// 3 n^2 m + (4 chain - 3) n^3 in place of chain (3 n^2 m + n^3).  N's values reach 3.4445^chain, its planes 2^(16 - 2 chain).
static double mu_steps(MuArgs& a, int chain, int cur, bool scaled, bool last, hipStream_t st, bool launch) {
    const float u2 = UNPLANE * UNPLANE;
    // n x n matrices: 0 A, 1 .. 3 Q, N and Q A in turn
    double t = mu_product<ST_SYM>(a, MuStage{-1, -1, 0, cur, scaled, u2, PLANE}, st, launch);
    int q = 1, n = 1;
    float np = PLANE;
    t += mu_product<ST_POLY>(a, MuStage{0, 0, q, cur, 0, u2, PLANE}, st, launch);
    for (int k = 1; k < chain; ++k) {
        const int w = 6 - q - n == 4 ? 2 : 6 - q - n;                        // the one that is neither (any of two where q = n)
        t += mu_product<ST_SYM>(a, MuStage{q, 0, w, cur, 0, u2, PLANE}, st, launch);             // Q A
        t += mu_product<ST_SYM>(a, MuStage{w, q, 0, cur, 0, u2, PLANE}, st, launch);             // (Q A) Q
        q = w;
        t += mu_product<ST_POLY>(a, MuStage{0, 0, q, cur, 0, u2, PLANE}, st, launch);
        const int o = 6 - q - n;
        t += mu_product<ST_SYM>(a, MuStage{q, n, o, cur, 0, UNPLANE / np, np / 4}, st, launch);  // N
        n = o;
        np /= 4;
    }
    const MuStage end{n, -1, -1, cur, scaled, UNPLANE / np, PLANE};
    return t + (last ? mu_product<ST_LAST>(a, end, st, launch) : mu_product<ST_NEXT>(a, end, st, launch));
}

static void mu_launch(MuArgs& a, hipStream_t st) {
    bool small = true;
    for (int i = 0; i < a.count; ++i) small = small && mu_is_small(a.mat[i].rows, a.mat[i].cols);
    if (small) {
        hipLaunchKernelGGL(mu_small_kernel, dim3(a.count), dim3(1024), 0, st, a);
        return;
    }
    hipLaunchKernelGGL(mu_norm_kernel, dim3(MU_PARTS, a.count), dim3(256), 0, st, a);
    int blk = 0;
    for (int i = 0; i < MU_GROUP; ++i) {
        a.first[i] = i < a.count ? blk : INT_MAX;
        if (i < a.count) blk += (a.mat[i].np / 64) * (a.mat[i].mp / 64);
    }
    hipLaunchKernelGGL(mu_planes_kernel, dim3(blk), dim3(256), 0, st, a);
    // One step at a time; or two, one, two at once, or two and three, where the products that saves are worth more than the
    // launches it adds (large matrices, the wider the more).  Errors against 64 bits, fp32, worst of five shapes and three
    // spectra (elementary fp32 operations 5.6e-6 and 1.3e-4 where four directions carry all but 1e-3): one by one 3.6e-6
    // and 1.5e-4, two-one-two 3.1e-6 and 9.5e-5, two-three 4.4e-6 and 9.8e-5, the 4.4e-6 at 1000 x 1500, hence 2 n <= m.
    // The weights after a step, four of 2048 x 2048 and three of 8192 x 2048: one by one 6.1e-8 and 5.0e-8 to 7.8e-8 off in
    // 6.29 ms, two-one-two 1.1e-7 and 4.7e-8 to 6.9e-8 in 5.30 (elementary fp32 8.3e-8 and 6.8e-8 to 1.15e-7).
    static constexpr int PLAN[3][6] = {{1, 1, 1, 1, 1, 0}, {2, 1, 2, 0, 0, 0}, {2, 3, 0, 0, 0, 0}};
    double one = 0.0, cost[4];
    for (int c = 1; c <= 3; ++c) cost[c] = mu_steps(a, c, 0, false, false, st, false);
    bool wide = true;
    for (int i = 0; i < a.count; ++i) wide = wide && a.mat[i].m >= 2 * a.mat[i].n;
    int plan = 0;
    for (int i = 0; i < (wide ? 3 : 2); ++i) {
        double t = i == 0 ? 0.0 : 5.0;                                       // us of launches
        for (int c = 0; PLAN[i][c]; ++c) t += cost[PLAN[i][c]];
        if (i == 0 || t < 0.97 * one) { one = t; plan = i; }
    }
    for (int c = 0, cur = 0; PLAN[plan][c]; ++c, cur ^= 1)
        mu_steps(a, PLAN[plan][c], cur, c == 0, PLAN[plan][c + 1] == 0, st, true);
}

static int mu_run(const mctsq_muon_matrix* mats, int64_t count, MuArgs& a, double lr, int adjust, char* ws, hipStream_t st) {
    for (int64_t g = 0; g < count; g += MU_GROUP) {
        const int c = (int)(count - g < MU_GROUP ? count - g : MU_GROUP);
        int64_t o = 0, blk = 0;
        a.count = c;
        int order[MU_GROUP];                              // longest products first: the short ones fill the gaps at the end
        for (int i = 0; i < c; ++i) order[i] = i;
        std::sort(order, order + c, [&](int x, int y) {
            const int64_t lx = std::max(mats[g + x].rows, mats[g + x].cols), ly = std::max(mats[g + y].rows, mats[g + y].cols);
            return lx != ly ? lx > ly : x < y;
        });
        for (int i = 0; i < c; ++i) {
            const mctsq_muon_matrix& s = mats[g + order[i]];
            MuMat& t = a.mat[i];
            t = MuMat{};
            t.rows = (int)s.rows; t.cols = (int)s.cols;
            t.n = t.rows < t.cols ? t.rows : t.cols; t.m = t.rows < t.cols ? t.cols : t.rows;
            t.np = (int)round_up(t.n, MU_PAD); t.mp = (int)round_up(t.m, MU_PAD);
            t.x = s.d_x; t.ldx = s.ldx; t.mom = s.d_momentum; t.out = s.d_out; t.ldo = s.ldo;
            const double r = (double)s.rows, k = (double)s.cols;
            t.lrs = (float)(lr * (adjust == MCTSQ_MUON_SPECTRAL ? sqrt(r > k ? r / k : 1.0)
                                  : adjust == MCTSQ_MUON_RMS ? 0.2 * sqrt(r > k ? r : k) : 1.0));
            t.ws = (_Float16*)(ws + o);
            o += mu_matrix_bytes(s.rows, s.cols);
            t.part = (double*)(ws + o) - MU_PARTS;
            blk += (int64_t)(t.np / 64) * (t.mp / 64);
        }
        MCTSQ_CHECK(blk < ((int64_t)1 << 31), "the matrices of one group are too large");
        mu_launch(a, st);
        MCTSQ_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace mctsq

using namespace mctsq;

extern "C" int64_t mctsq_orthogonalize_workspace_bytes(const mctsq_muon_matrix* mats, int64_t count, int dtype) {
    if (int rc = mu_check_shapes(mats, count)) return rc;
    MCTSQ_CHECK(dtype == MU_F32 || dtype == MU_BF16, "dtype must be 0 (fp32) or 1 (bf16)");
    return mu_bytes(mats, count);
}
extern "C" int mctsq_orthogonalize(const mctsq_muon_matrix* mats, int64_t count, int dtype, double eps, void* d_ws,
                                   int64_t ws_bytes, void* stream) {
    const int64_t need = mctsq_orthogonalize_workspace_bytes(mats, count, dtype);
    if (need < 0) return (int)need;
    MCTSQ_CHECK(eps > 0.0, "eps must be positive");
    MCTSQ_CHECK(d_ws && ((uintptr_t)d_ws & 255) == 0 && ws_bytes >= need,
                "workspace must hold mctsq_orthogonalize_workspace_bytes(), 256-byte aligned");
    const int es = dtype == MU_F32 ? 4 : 2;
    for (int64_t i = 0; i < count; ++i) {
        MCTSQ_CHECK(mats[i].d_x && mats[i].d_out, "NULL device pointer");
        MCTSQ_CHECK(!mats[i].d_momentum, "orthogonalisation takes no momentum");
        MCTSQ_CHECK(mats[i].ldx >= mats[i].cols && mats[i].ldo >= mats[i].cols, "leading dimensions are smaller than the rows");
        MCTSQ_CHECK((((uintptr_t)mats[i].d_x | (uintptr_t)mats[i].d_out) & (es - 1)) == 0, "a matrix is not aligned to its element size");
    }
    MuArgs a{};
    a.xtype = a.otype = dtype; a.eps = eps;
    return mu_run(mats, count, a, 1.0, MCTSQ_MUON_NONE, (char*)d_ws, (hipStream_t)stream);
}

extern "C" int64_t mctsq_muon_workspace_bytes(const mctsq_muon_matrix* mats, int64_t count) {
    if (int rc = mu_check_shapes(mats, count)) return rc;
    return mu_bytes(mats, count);
}
extern "C" int mctsq_muon_step(const mctsq_muon_matrix* mats, int64_t count, int grad_dtype, double lr, double momentum,
                               int nesterov, double weight_decay, double eps, int adjust, void* d_ws, int64_t ws_bytes,
                               void* stream) {
    const int64_t need = mctsq_muon_workspace_bytes(mats, count);
    if (need < 0) return (int)need;
    MCTSQ_CHECK(grad_dtype == MU_F32 || grad_dtype == MU_BF16, "gradient dtype must be 0 (fp32) or 1 (bf16)");
    MCTSQ_CHECK(lr == lr && weight_decay == weight_decay, "lr / weight_decay is NaN");
    MCTSQ_CHECK(momentum >= 0.0 && momentum < 1.0, "momentum must lie in [0, 1)");
    MCTSQ_CHECK(eps > 0.0, "eps must be positive");
    MCTSQ_CHECK(adjust == MCTSQ_MUON_NONE || adjust == MCTSQ_MUON_SPECTRAL || adjust == MCTSQ_MUON_RMS, "unknown adjust");
    MCTSQ_CHECK(d_ws && ((uintptr_t)d_ws & 255) == 0 && ws_bytes >= need,
                "workspace must hold mctsq_muon_workspace_bytes(), 256-byte aligned");
    const int gs = grad_dtype == MU_F32 ? 4 : 2;
    for (int64_t i = 0; i < count; ++i) {
        MCTSQ_CHECK(mats[i].d_x && mats[i].d_out && mats[i].d_momentum, "NULL device pointer");
        MCTSQ_CHECK(mats[i].ldx >= mats[i].cols && mats[i].ldo >= mats[i].cols, "leading dimensions are smaller than the rows");
        MCTSQ_CHECK(((uintptr_t)mats[i].d_x & (gs - 1)) == 0 && (((uintptr_t)mats[i].d_out | (uintptr_t)mats[i].d_momentum) & 3) == 0,
                    "a matrix is not aligned to its element size");
    }
    MuArgs a{};
    a.xtype = grad_dtype; a.otype = MU_F32; a.eps = eps;
    a.mu = (float)momentum; a.nesterov = nesterov; a.decay = (float)(1.0 - lr * weight_decay);
    return mu_run(mats, count, a, lr, adjust, (char*)d_ws, (hipStream_t)stream);
}
