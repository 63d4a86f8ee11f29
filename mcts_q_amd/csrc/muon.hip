// Orthogonalised updates: momentum, five quintic Newton-Schulz steps on each weight matrix, decay and update.
//
//   u = g + mu m' (m' = mu m + g),  X_0 = u / (|u|_F + eps),
//   A = X X^T,  B = b A + c A^2,  X <- a X + B X        (a, b, c) = (3.4445, -4.7750, 2.0315), n = rows <= m = columns
//
// which maps every singular value s of X through a s + b s^3 + c s^5, towards 1 (tall matrices are worked on transposed).
// Per step n^2 m + n^3 + 2 n^2 m fused multiply-adds: A and B are symmetric, only tiles on and below the diagonal are
// computed and stored to both places.  The bound is the matrix pipe.
//
// Arithmetic.  fp32 matrices go through the two-way fp16 split of this library (device_utils.hpp: split2h): every operand is
// hi + lo in fp16 scaled by 2^14, products lo hi + hi lo + hi hi accumulate in fp32, i.e. fp32 accuracy at three 16-bit
// matrix instructions.  The scale is safe without looking at the data: |u|_F = 1 bounds every singular value of X_0 by 1,
// the quintic maps [0, 1.21] into itself, so |X| <= 1.21, |A| <= 1.47, |B| <= 2.81 and 2.81 * 2^14 < 65504.
// bf16 matrices use the hi plane alone: one matrix instruction per product; X, A and B are rounded to 11 bits each step,
// which leaves the result 1.2e-3 off in the mean against 1.7e-3 for its rounding to bf16.
// X_0 is never rounded by the normalisation: its planes hold u times a power of two, the rest of the factor (in (1, 2])
// enters the first step's products in fp32.
//
// Planes are stored as the matrix instruction's operand fragments, [row tile of 16][k block of 32][lane 64][8], 1 KB in a
// row per fragment, so a tile is fetched into LDS lane by lane (global_load_lds) and read back without a bank conflict.
// X is kept both ways (k along m for A, k along n for B X).
#include <math.h>

#include "device_utils.hpp"

namespace mctsq {

constexpr int MU_GROUP = 20;        // matrices per launch (kernel arguments hold their descriptions)
constexpr int MU_PARTS = 256;       // workgroups that add up one matrix's squares
constexpr float NS_A = 3.4445f, NS_B = -4.7750f, NS_C = 2.0315f;
constexpr float PLANE = 16384.0f, UNPLANE = 1.0f / 16384.0f;        // 2^14
constexpr int FRAG = 512;           // halves in a fragment

enum { MU_F32 = 0, MU_BF16 = 1 };

struct MuMat {
    int n, m;                       // working shape, n <= m
    int np, mp;                     // padded to the tile
    int rows, cols;                 // the matrix as the caller has it; transposed when rows > cols
    int sym0, full0, blk0;          // first tile / tile / 64 x 64 block of this matrix in the launch
    float lrs;                      // learning rate times the shape's factor
    const void* x; int64_t ldx;     // gradient, or the matrix to orthogonalise
    float* mom;                     // momentum [rows][cols], NULL: orthogonalise x
    void* out; int64_t ldo;         // parameters (updated in place), or the result
    _Float16* ws;                   // X0 X1 | XT0 XT1 | A | B, each of `planes` planes
    double* part;                   // MU_PARTS sums of squares
};
struct MuArgs {
    int count, xtype, otype;        // element types of x and, when orthogonalising, out
    float mu, decay; int nesterov;
    double eps;
    MuMat mat[MU_GROUP];
};
static_assert(sizeof(MuArgs) <= 3584, "kernel arguments");

__device__ __forceinline__ float mu_load(const void* p, int64_t i, int type) {
    if (type == MU_F32) return reinterpret_cast<const float*>(p)[i];
    return __uint_as_float((unsigned)reinterpret_cast<const unsigned short*>(p)[i] << 16);
}

// ---- momentum and squares ------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void mu_norm_kernel(MuArgs a) {
    __shared__ double red[4];
    const MuMat& t = a.mat[blockIdx.y];
    const int64_t total = (int64_t)t.rows * t.cols;
    double acc = 0.0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)MU_PARTS * 256) {
        const int64_t r = i / t.cols, c = i - r * t.cols;
        float u = mu_load(t.x, r * t.ldx + c, a.xtype);
        if (t.mom) {
            const float m = fmaf(a.mu, t.mom[i], u);
            t.mom[i] = m;
            u = a.nesterov ? fmaf(a.mu, m, u) : m;
        }
        acc += (double)u * u;
    }
    for (int d = 32; d >= 1; d >>= 1) acc += __shfl_xor(acc, d, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = acc;
    __syncthreads();
    if (threadIdx.x == 0) t.part[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// |u|_F from the parts (every lane of a wave gets it): up = the power of two that brings it into [1/2, 1), s = the rest
// of 1 / (|u| + eps)
__device__ __forceinline__ void mu_scale(const MuMat& t, double eps, double& up, float& s) {
    double acc = 0.0;
    for (int i = threadIdx.x & 63; i < MU_PARTS; i += 64) acc += t.part[i];
    for (int d = 32; d >= 1; d >>= 1) acc += __shfl_xor(acc, d, 64);
    const double norm = sqrt(acc);
    int e = 0;
    if (norm > 0.0 && norm < INFINITY) (void)frexp(norm, &e);
    e = e > 600 ? 600 : (e < -600 ? -600 : e);
    up = ldexp(1.0, -e);
    s = (float)(ldexp(1.0, e) / (norm + eps));
}

// ---- planes of X_0 and its transpose -----------------------------------------------------------------------------------
// element (row, k) of a plane of K columns
__device__ __forceinline__ int64_t frag_at(int row, int k, int K) {
    return ((int64_t)(row >> 4) * (K >> 5) + (k >> 5)) * FRAG + (((row & 15) + 16 * ((k & 31) >> 3)) << 3) + (k & 7);
}
template <int P>
struct MuPlanes {                   // where a matrix's planes are; plane p of X starts p * np * mp behind X
    int64_t xs, as;
    _Float16 *base, *A, *B;
    __device__ MuPlanes(const MuMat& t) {
        xs = (int64_t)t.np * t.mp; as = (int64_t)t.np * t.np;
        base = t.ws; A = base + 4 * P * xs; B = A + P * as;
    }
    __device__ _Float16* X(int cur) const { return base + cur * P * xs; }
    __device__ _Float16* XT(int cur) const { return base + (2 + cur) * P * xs; }
};

template <int P>
__global__ __launch_bounds__(256) void mu_planes_kernel(MuArgs a) {
    __shared__ float tile[64][65];
    int w = 0;
    while (w + 1 < a.count && (int)blockIdx.x >= a.mat[w + 1].blk0) ++w;
    const MuMat& t = a.mat[w];
    const int blk = blockIdx.x - t.blk0, nb = t.mp / 64, bi = blk / nb * 64, bj = blk % nb * 64;     // working coordinates
    const bool tr = t.rows > t.cols;
    double up; float s;
    mu_scale(t, a.eps, up, s);
    const int x = threadIdx.x & 63, y0 = threadIdx.x >> 6;
    for (int y = y0; y < 64; y += 4) {               // x runs along the caller's columns
        const int r = (tr ? bj : bi) + y, c = (tr ? bi : bj) + x;
        float u = 0.0f;
        if (r < t.rows && c < t.cols) {
            u = mu_load(t.x, r * t.ldx + c, a.xtype);
            if (t.mom) {
                const float m = t.mom[(int64_t)r * t.cols + c];
                u = a.nesterov ? fmaf(a.mu, m, u) : m;
            }
            u = (float)((double)u * up * (double)PLANE);
        }
        if (tr) tile[x][y] = u;
        else tile[y][x] = u;
    }
    __syncthreads();
    const MuPlanes<P> pl(t);
    const int lane = threadIdx.x & 63, row = lane & 15, k0 = (lane >> 4) * 8;
    for (int f = y0; f < 16; f += 4) {               // 8 fragments of X, 8 of its transpose
        const bool T = f >= 8;
        const int rt = (f & 7) >> 1, kb = f & 1;
        f16x8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int i = rt * 16 + row, k = kb * 32 + k0 + e;
            const float v = T ? tile[k][i] : tile[i][k];
            hi[e] = (_Float16)v;
            lo[e] = (_Float16)(v - (float)hi[e]);
        }
        _Float16* dst = (T ? pl.XT(0) + frag_at(bj + rt * 16, bi + kb * 32, t.np) : pl.X(0) + frag_at(bi + rt * 16, bj + kb * 32, t.mp)) + lane * 8;
        *reinterpret_cast<f16x8*>(dst) = hi;
        if (P == 2) *reinterpret_cast<f16x8*>(dst + pl.xs) = lo;
    }
}

// ---- the products ---------------------------------------------------------------------------------------------------------
enum { ST_GRAM = 0, ST_POLY = 1, ST_NEXT = 2, ST_LAST = 3 };

// C[i][j] = sum_k R[i][k] S[j][k] over fragments of R and S: a T x T tile, T = 128 or 64, four waves of T/2 x T/2.
// Two LDS buffers of one k block (32) each; the next block is fetched while the current one is multiplied.
template <int P, int T>
__device__ __forceinline__ void mu_tile(const _Float16* R, int64_t rs, const _Float16* S, int64_t ss, int KB, int ti, int tj,
                                        f32x4 (&acc)[T / 32][T / 32], _Float16* lds) {
    constexpr int RT = T / 16, F = 2 * P * RT, W = T / 32;       // row tiles, fragments of a k block, tiles per wave side
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wi = wave >> 1, wj = wave & 1;
    auto fetch = [&](int kb, int buf) {
#pragma unroll
        for (int f0 = 0; f0 < F; f0 += 4) {
            const int f = f0 + wave;
            const int side = f / (P * RT), p = f / RT % P, rt = f % RT;
            const _Float16* g = (side ? S + p * ss + ((int64_t)(tj * RT + rt) * KB + kb) * FRAG
                                      : R + p * rs + ((int64_t)(ti * RT + rt) * KB + kb) * FRAG) + lane * 8;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                             (__attribute__((address_space(3))) void*)(lds + ((int64_t)buf * F + f) * FRAG), 16, 0, 0);
        }
    };
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    fetch(0, 0);
    for (int kb = 0; kb < KB; ++kb) {
        __builtin_amdgcn_s_waitcnt(0x0f70);          // vmcnt(0): this wave's part of block kb has arrived
        __syncthreads();                             // ... and everyone's; nobody reads the other buffer any more
        if (kb + 1 < KB) fetch(kb + 1, (kb + 1) & 1);
        const u32x4* b = reinterpret_cast<const u32x4*>(lds + (int64_t)(kb & 1) * F * FRAG) + lane;
        u32x4 r[P][W], s[P];
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < W; ++i) r[p][i] = b[(p * RT + wi * W + i) * 64];
#pragma unroll
        for (int j = 0; j < W; ++j) {
#pragma unroll
            for (int p = 0; p < P; ++p) s[p] = b[(P * RT + p * RT + wj * W + j) * 64];
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if constexpr (P == 2) {
                    acc[i][j] = mfma_h(r[1][i], s[0], acc[i][j]);
                    acc[i][j] = mfma_h(r[0][i], s[1], acc[i][j]);
                }
                acc[i][j] = mfma_h(r[0][i], s[0], acc[i][j]);
            }
        }
    }
}

template <int P>
__device__ __forceinline__ float plane_value(const _Float16* p, int64_t ps, int64_t at) {
    float v = (float)p[at];
    if (P == 2) v += (float)p[at + ps];
    return v * UNPLANE;
}
// four values along k of one row (k a multiple of 4)
template <int P>
__device__ __forceinline__ void put4(_Float16* p, int64_t ps, int64_t at, const float* v) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    f16x4 h, l;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        h[r] = (_Float16)(v[r] * PLANE);
        l[r] = (_Float16)(v[r] * PLANE - (float)h[r]);
    }
    *reinterpret_cast<f16x4*>(p + at) = h;
    if (P == 2) *reinterpret_cast<f16x4*>(p + at + ps) = l;
}
template <int P>
__device__ __forceinline__ void put1(_Float16* p, int64_t ps, int64_t at, float v) {
    const _Float16 h = (_Float16)(v * PLANE);
    p[at] = h;
    if (P == 2) p[at + ps] = (_Float16)(v * PLANE - (float)h);
}

template <int P, int T, int ST>
__global__ __launch_bounds__(256) void mu_product_kernel(MuArgs a, int it) {
    constexpr int W = T / 32;
    __shared__ __attribute__((aligned(16))) _Float16 lds[2 * 2 * P * (T / 16) * FRAG];
    const bool sym = ST == ST_GRAM || ST == ST_POLY;
    int w = 0;
    while (w + 1 < a.count && (int)blockIdx.x >= (sym ? a.mat[w + 1].sym0 : a.mat[w + 1].full0)) ++w;
    const MuMat& t = a.mat[w];
    const MuPlanes<P> pl(t);
    const int b = blockIdx.x - (sym ? t.sym0 : t.full0);
    int ti, tj;
    if (sym) {                       // tile b of the lower triangle, row by row
        ti = (int)((sqrtf(8.0f * b + 1.0f) - 1.0f) * 0.5f);
        while ((ti + 1) * (ti + 2) / 2 <= b) ++ti;
        while (ti * (ti + 1) / 2 > b) --ti;
        tj = b - ti * (ti + 1) / 2;
    } else {
        ti = b % (t.np / T); tj = b / (t.np / T);
    }
    const int cur = it & 1;
    f32x4 acc[W][W];
    if (ST == ST_GRAM) mu_tile<P, T>(pl.X(cur), pl.xs, pl.X(cur), pl.xs, t.mp / 32, ti, tj, acc, lds);
    else if (ST == ST_POLY) mu_tile<P, T>(pl.A, pl.as, pl.A, pl.as, t.np / 32, ti, tj, acc, lds);
    else mu_tile<P, T>(pl.B, pl.as, pl.XT(cur), pl.xs, t.np / 32, ti, tj, acc, lds);

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane >> 4, col = lane & 15;
    float s = 1.0f;
    if (it == 0 && ST != ST_POLY) { double up; mu_scale(t, a.eps, up, s); }
    const float unit = UNPLANE * UNPLANE;
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int gi = ti * T + ((wave >> 1) * W + i) * 16 + 4 * q, gj = tj * T + ((wave & 1) * W + j) * 16 + col;
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = acc[i][j][r] * unit;
            if constexpr (ST == ST_GRAM) {
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] *= s * s;
            }
            if constexpr (ST == ST_POLY) {
#pragma unroll
                for (int r = 0; r < 4; ++r)              // A is symmetric: its (gj, gi + r) lie side by side
                    v[r] = fmaf(NS_C, v[r], NS_B * plane_value<P>(pl.A, pl.as, frag_at(gj, gi, t.np) + r));
            }
            if constexpr (sym) {
                _Float16* out = ST == ST_GRAM ? pl.A : pl.B;
                put4<P>(out, pl.as, frag_at(gj, gi, t.np), v);
                if (ti != tj)
#pragma unroll
                    for (int r = 0; r < 4; ++r) put1<P>(out, pl.as, frag_at(gi + r, gj, t.np), v[r]);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    v[r] = s * fmaf(NS_A, plane_value<P>(pl.XT(cur), pl.xs, frag_at(gj, gi, t.np) + r), v[r]);
                if constexpr (ST == ST_NEXT) {
                    put4<P>(pl.XT(cur ^ 1), pl.xs, frag_at(gj, gi, t.np), v);
#pragma unroll
                    for (int r = 0; r < 4; ++r) put1<P>(pl.X(cur ^ 1), pl.xs, frag_at(gi + r, gj, t.mp), v[r]);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (gi + r < t.n && gj < t.m) {
                            const bool tr = t.rows > t.cols;
                            const int64_t at = (int64_t)(tr ? gj : gi + r) * t.ldo + (tr ? gi + r : gj);
                            if (t.mom) {
                                float* p = reinterpret_cast<float*>(t.out);
                                p[at] = fmaf(p[at], a.decay, -t.lrs * v[r]);
                            } else if (a.otype == MU_F32) reinterpret_cast<float*>(t.out)[at] = v[r];
                            else reinterpret_cast<__bf16*>(t.out)[at] = (__bf16)v[r];
                        }
                }
            }
        }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
struct MuPlan { int T; int64_t bytes; };

static int64_t mu_planes_halves(int64_t n, int64_t m, int T, int P) {
    const int64_t np = round_up(n, T), mp = round_up(m, T);
    return P * (4 * np * mp + 2 * np * np);
}
// The tile of a group: 128 unless the launch would then leave CUs without a tile.
static int mu_tile_size(const mctsq_muon_matrix* mats, int count) {
    int64_t tiles = 0;
    for (int i = 0; i < count; ++i) {
        const int64_t n = mats[i].rows < mats[i].cols ? mats[i].rows : mats[i].cols;
        const int64_t t = (n + 127) / 128;
        tiles += t * (t + 1) / 2;
    }
    return tiles >= 256 ? 128 : 64;
}
static int64_t mu_group_bytes(const mctsq_muon_matrix* mats, int count, int P) {
    const int T = mu_tile_size(mats, count);
    int64_t o = 0;
    for (int i = 0; i < count; ++i) {
        const int64_t n = mats[i].rows < mats[i].cols ? mats[i].rows : mats[i].cols;
        const int64_t m = mats[i].rows < mats[i].cols ? mats[i].cols : mats[i].rows;
        o += round_up(mu_planes_halves(n, m, T, P) * 2, 256) + MU_PARTS * 8;
    }
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
static int64_t mu_bytes(const mctsq_muon_matrix* mats, int64_t count, int P) {
    int64_t need = 0;                                    // the groups run one after the other in the same space
    for (int64_t g = 0; g < count; g += MU_GROUP) {
        const int64_t b = mu_group_bytes(mats + g, (int)(count - g < MU_GROUP ? count - g : MU_GROUP), P);
        need = b > need ? b : need;
    }
    return need < 256 ? 256 : need;
}

template <int P, int T>
static void mu_launch(const MuArgs& a, int sym, int full, int blk, hipStream_t st) {
    hipLaunchKernelGGL(mu_norm_kernel, dim3(MU_PARTS, a.count), dim3(256), 0, st, a);
    hipLaunchKernelGGL(mu_planes_kernel<P>, dim3(blk), dim3(256), 0, st, a);
    for (int it = 0; it < 5; ++it) {
        hipLaunchKernelGGL((mu_product_kernel<P, T, ST_GRAM>), dim3(sym), dim3(256), 0, st, a, it);
        hipLaunchKernelGGL((mu_product_kernel<P, T, ST_POLY>), dim3(sym), dim3(256), 0, st, a, it);
        if (it < 4) hipLaunchKernelGGL((mu_product_kernel<P, T, ST_NEXT>), dim3(full), dim3(256), 0, st, a, it);
        else hipLaunchKernelGGL((mu_product_kernel<P, T, ST_LAST>), dim3(full), dim3(256), 0, st, a, it);
    }
}

static int mu_run(const mctsq_muon_matrix* mats, int64_t count, int P, MuArgs& a, double lr, int adjust, char* ws, hipStream_t st) {
    for (int64_t g = 0; g < count; g += MU_GROUP) {
        const int c = (int)(count - g < MU_GROUP ? count - g : MU_GROUP);
        const int T = mu_tile_size(mats + g, c);
        int64_t o = 0, sym = 0, full = 0, blk = 0;
        a.count = c;
        for (int i = 0; i < c; ++i) {
            const mctsq_muon_matrix& s = mats[g + i];
            MuMat& t = a.mat[i];
            t = MuMat{};
            t.rows = (int)s.rows; t.cols = (int)s.cols;
            t.n = t.rows < t.cols ? t.rows : t.cols; t.m = t.rows < t.cols ? t.cols : t.rows;
            t.np = (int)round_up(t.n, T); t.mp = (int)round_up(t.m, T);
            t.x = s.d_x; t.ldx = s.ldx; t.mom = s.d_momentum; t.out = s.d_out; t.ldo = s.ldo;
            const double r = (double)s.rows, k = (double)s.cols;
            t.lrs = (float)(lr * (adjust == MCTSQ_MUON_SPECTRAL ? sqrt(r > k ? r / k : 1.0)
                                  : adjust == MCTSQ_MUON_RMS ? 0.2 * sqrt(r > k ? r : k) : 1.0));
            t.ws = (_Float16*)(ws + o); o += round_up(mu_planes_halves(t.n, t.m, T, P) * 2, 256);
            t.part = (double*)(ws + o); o += MU_PARTS * 8;
            t.sym0 = (int)sym; t.full0 = (int)full; t.blk0 = (int)blk;
            const int64_t nt = t.np / T;
            sym += nt * (nt + 1) / 2; full += nt * (t.mp / T); blk += (int64_t)(t.np / 64) * (t.mp / 64);
        }
        MCTSQ_CHECK(blk < ((int64_t)1 << 31), "the matrices of one group are too large");
        if (P == 2) { if (T == 128) mu_launch<2, 128>(a, sym, full, blk, st); else mu_launch<2, 64>(a, sym, full, blk, st); }
        else { if (T == 128) mu_launch<1, 128>(a, sym, full, blk, st); else mu_launch<1, 64>(a, sym, full, blk, st); }
        MCTSQ_HIP(hipGetLastError());
    }
    return 0;
}

}  // namespace mctsq

using namespace mctsq;

extern "C" int64_t mctsq_orthogonalize_workspace_bytes(const mctsq_muon_matrix* mats, int64_t count, int dtype) {
    if (int rc = mu_check_shapes(mats, count)) return rc;
    MCTSQ_CHECK(dtype == MU_F32 || dtype == MU_BF16, "dtype must be 0 (fp32) or 1 (bf16)");
    return mu_bytes(mats, count, dtype == MU_F32 ? 2 : 1);
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
    return mu_run(mats, count, dtype == MU_F32 ? 2 : 1, a, 1.0, MCTSQ_MUON_NONE, (char*)d_ws, (hipStream_t)stream);
}

extern "C" int64_t mctsq_muon_workspace_bytes(const mctsq_muon_matrix* mats, int64_t count) {
    if (int rc = mu_check_shapes(mats, count)) return rc;
    return mu_bytes(mats, count, 2);
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
    return mu_run(mats, count, 2, a, lr, adjust, (char*)d_ws, (hipStream_t)stream);
}
