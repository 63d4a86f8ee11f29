// What a policy learns from: log-probabilities of given actions, the clipped policy-ratio loss with a KL term, and the
// paired log-ratio loss over preferred / rejected sequences, each with its gradient by the logits.
//
//   logp_i = z_i[a_i] - lse_i,   lse_i = log sum_j exp z_i[j],   d logp_i / d z_i[j] = [j = a_i] - p_i[j]
//
// so every loss here is a coefficient c_i = d loss / d logp_i per row and the gradient row c_i (one_hot(a_i) - p_i).
// The bound is HBM: each logit read once, each gradient element written once.  One workgroup owns a row at a time:
//   - the row is loaded ONCE into registers as the 16-byte vectors it arrives in (row_reg_kernel), every thread reduces
//     its own elements to (max, sum of exponentials), the pairs are joined over the workgroup with one barrier, thread 0
//     turns them into the coefficient, and the gradient is formed from the same registers;
//   - rows longer than the registers hold are read twice (row_stream_kernel), the second time from the caches;
//   - rows of at most 256 elements go to groups of 4 or 16 lanes (row_lane_kernel), many rows to a workgroup.
// Statistics: exponentials and per-thread sums in fp32 (at most 128 terms), everything joined across threads, the
// logarithm, ratio, KL term and loss in fp64: the clip decides on a ratio that two evaluations must agree on.
// Rows of weight 0 are padding: their logits, action, and statistics are not read, their outputs are exactly 0.
// An action outside [0, V) on a row that has weight makes that row's outputs and the loss NaN; nothing is read for it.
// Sums are joined in a fixed order: the same inputs give the same bits.
#include <float.h>
#include <math.h>

#include "device_utils.hpp"

namespace mctsq {

enum { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };
enum { MODE_LOGP = 0, MODE_POLICY = 1, MODE_GRAD = 2 };

struct RowArgs {
    const char* z; int64_t z_so, z_si;        // logits and their strides (elements): row i = (i / inner, i % inner)
    char* dz; int64_t d_so, d_si;             // gradient (may be the logits themselves), NULL: none
    int64_t rows, inner, V;
    const void* act; int act64;
    const float* w;                           // row weights, NULL: 1
    const float* pair_w; int64_t pairs;       // pair weights of the preference loss (row / inner = pair or pairs + pair)
    // policy
    const float* old_logp; const float* ref_logp; const float* adv; int64_t adv_div;
    double clip_lo, clip_hi, kl_coef, scale;
    float* logp; float* kl;
    double* loss_part;                        // one per workgroup
    // preference: statistics of pass 1 (read by pass 2), coefficient per sequence
    double* logp64; float* stat_m; float* stat_inv; const float* seq_coef;
};

template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int VE = 4;
    __device__ static float load(const char* p, int64_t i) { return reinterpret_cast<const float*>(p)[i]; }
    __device__ static void store(char* p, int64_t i, float v) { reinterpret_cast<float*>(p)[i] = v; }
    __device__ static void unpack(const u32x4& u, float* f) {
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = __uint_as_float(u[k]);
    }
    __device__ static u32x4 pack(const float* f) {
        u32x4 u;
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = __float_as_uint(f[k]);
        return u;
    }
    static constexpr unsigned NEG_INF = 0xff800000u;       // one word of -inf
};
template <typename T> struct Elem16 {
    static constexpr int VE = 8;
    typedef T T2 __attribute__((ext_vector_type(2)));
    __device__ static float load(const char* p, int64_t i) { return (float)reinterpret_cast<const T*>(p)[i]; }
    __device__ static void store(char* p, int64_t i, float v) { reinterpret_cast<T*>(p)[i] = (T)v; }
    __device__ static u32x4 pack(const float* f) {          // round to nearest even: the one rounding of the gradient
        u32x4 u;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            T2 t;
            t.x = (T)f[2 * k]; t.y = (T)f[2 * k + 1];
            u[k] = __builtin_bit_cast(unsigned, t);
        }
        return u;
    }
};
template <> struct Elem<__bf16> : Elem16<__bf16> {
    __device__ static void unpack(const u32x4& u, float* f) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            f[2 * k] = __uint_as_float(u[k] << 16);
            f[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
        }
    }
    static constexpr unsigned NEG_INF = 0xff80ff80u;
};
template <> struct Elem<_Float16> : Elem16<_Float16> {
    __device__ static void unpack(const u32x4& u, float* f) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned w = u[k];          // a copy: a bit cast of the vector element itself reads element 0
            const T2 t = __builtin_bit_cast(T2, w);
            f[2 * k] = (float)t.x; f[2 * k + 1] = (float)t.y;
        }
    }
    static constexpr unsigned NEG_INF = 0xfc00fc00u;
};

// A row as the 16-byte vectors of memory it covers: vector v holds the elements [v VE - mis, (v + 1) VE - mis).  The
// first and last may lie partly outside the row; those are loaded and stored element by element, so no access leaves
// the row whatever its alignment.
template <typename T>
struct RowView {
    const char* base;           // first element of the row
    int64_t V;
    int mis;                    // elements between the 16-byte boundary below the row and its start
    int64_t nvec;
    __device__ RowView(const char* b, int64_t v) : base(b), V(v) {
        mis = (int)(((uintptr_t)b & 15) / sizeof(T));
        nvec = (mis + V + Elem<T>::VE - 1) / Elem<T>::VE;
    }
    __device__ u32x4 load(int64_t v) const {
        constexpr int VE = Elem<T>::VE;
        const int64_t e0 = v * VE - mis;
        if (e0 >= 0 && e0 + VE <= V) return *reinterpret_cast<const u32x4*>(base + e0 * (int64_t)sizeof(T));
        u32x4 u;
        u[0] = u[1] = u[2] = u[3] = Elem<T>::NEG_INF;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const int64_t e = e0 + j;
            if (e >= 0 && e < V) {
                if constexpr (sizeof(T) == 4) u[j] = reinterpret_cast<const unsigned*>(base)[e];
                else {
                    const unsigned h = reinterpret_cast<const unsigned short*>(base)[e];
                    u[j >> 1] = (j & 1) ? ((u[j >> 1] & 0xffffu) | (h << 16)) : ((u[j >> 1] & 0xffff0000u) | h);
                }
            }
        }
        return u;
    }
    // the gradient's vector v, at the same element positions of another row; `aligned`: both rows start at the same
    // offset from a 16-byte boundary
    __device__ void store(char* out, bool aligned, int64_t v, const float* f) const {
        constexpr int VE = Elem<T>::VE;
        const int64_t e0 = v * VE - mis;
        if (aligned && e0 >= 0 && e0 + VE <= V) {
            *reinterpret_cast<u32x4*>(out + e0 * (int64_t)sizeof(T)) = Elem<T>::pack(f);
            return;
        }
#pragma unroll
        for (int j = 0; j < VE; ++j)
            if (e0 + j >= 0 && e0 + j < V) Elem<T>::store(out, e0 + j, f[j]);
    }
};

// max and sum of exp(x - max) of a set of values, joinable in any order.  An empty set or one of -inf only is (-inf, 0).
__device__ __forceinline__ float exp_diff(float x, float m) { return fast_exp2((x - m) * LOG2E); }
// The same with log2 e in two words.  LOG2E alone is 1.3e-8 short, which makes every exponential of a row err to the same
// side and shows in the sum of a long sequence's log-probabilities; one more fma per element in a pass bound by memory.
constexpr float LOG2E_LO = 1.92596299e-8f;
__device__ __forceinline__ float exp_diff_sum(float x, float m) {
    const float d = x - m;
    return fast_exp2(fmaf(d, LOG2E, d * LOG2E_LO));
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }

template <int VE>
__device__ __forceinline__ void accumulate(const float* f, float& m, float& s) {
    float bm = f[0];
#pragma unroll
    for (int j = 1; j < VE; ++j) bm = fmaxf(bm, f[j]);
    const float nm = fmaxf(m, bm), ref = finite_or_zero(nm);
    s *= exp_diff_sum(m, ref);                          // m = -inf: the factor is 0, and so is s
#pragma unroll
    for (int j = 0; j < VE; ++j) s += exp_diff_sum(f[j], ref);
    m = nm;
}

__device__ __forceinline__ double shfl_xor_f64(double v, int mask) { return __shfl_xor(v, mask, 64); }

// join over the lanes of groups of W (a power of two <= 64): every lane gets the group's max and fp64 sum
template <int W>
__device__ __forceinline__ void join_lanes(float& m, double& s) {
    float M = m;
#pragma unroll
    for (int d = W / 2; d >= 1; d >>= 1) M = fmaxf(M, __shfl_xor(M, d, 64));
    s *= (double)exp_diff_sum(m, finite_or_zero(M));        // m = -inf: the factor is 0, and so is s
    if (!(m > -INFINITY) && s == s) s = 0.0;            // (-inf) - 0 and an empty set
#pragma unroll
    for (int d = W / 2; d >= 1; d >>= 1) s += shfl_xor_f64(s, d);
    m = M;
}

__device__ __forceinline__ int64_t row_action(const RowArgs& a, int64_t row) {
    return a.act64 ? reinterpret_cast<const int64_t*>(a.act)[row] : (int64_t)reinterpret_cast<const int32_t*>(a.act)[row];
}
__device__ __forceinline__ float row_weight(const RowArgs& a, int64_t row) {
    if (a.pair_w) {
        const int64_t q = row / a.inner;
        if (a.pair_w[q < a.pairs ? q : q - a.pairs] == 0.0f) return 0.0f;
    }
    return a.w ? a.w[row] : 1.0f;
}
__device__ __forceinline__ int64_t row_offset(int64_t row, int64_t inner, int64_t so, int64_t si) {
    return (row / inner) * so + (row % inner) * si;
}

// The row's log-probability and, in the policy mode, its loss and coefficient; writes the per-row outputs.
// L(r) = -min(r A, clip(r, lo, hi) A), r = exp(logp - old);  k = exp(d) - d - 1, d = ref - logp (never negative, 0 at d = 0)
// d L / d logp = -r A where the unclipped product is the smaller one (or equal), else 0;  d k / d logp = 1 - exp(d)
template <int MODE>
__device__ __forceinline__ double row_result(const RowArgs& a, int64_t row, float w, float za, float m, double s,
                                             float& coef) {
    const double logp = ((double)za - (double)m) - log(s);
    a.logp[row] = (float)logp;
    if constexpr (MODE == MODE_POLICY) {
        const double A = (double)a.adv[row / a.adv_div];
        const double r = a.old_logp ? exp(logp - (double)a.old_logp[row]) : (logp == logp ? 1.0 : logp);
        const double un = r * A, cl = fmin(fmax(r, a.clip_lo), a.clip_hi) * A;
        double loss = -(un <= cl ? un : cl), c = un <= cl ? -un : 0.0, k = 0.0;
        if (un != un) loss = c = un;
        if (a.ref_logp) {
            const double d = (double)a.ref_logp[row] - logp, e = expm1(d);
            k = e - d;
            loss += a.kl_coef * k;
            c -= a.kl_coef * e;
        }
        a.kl[row] = (float)k;
        const double sw = a.scale * (double)w;
        coef = (float)(sw * c);
        return sw * loss;
    }
    return 0.0;
}

// outputs of a padding row, and of one whose action does not exist
template <int MODE>
__device__ __forceinline__ void row_const(const RowArgs& a, int64_t row, float v) {
    if constexpr (MODE == MODE_LOGP || MODE == MODE_POLICY) a.logp[row] = v;
    if constexpr (MODE == MODE_POLICY) a.kl[row] = v;
    if (MODE == MODE_LOGP && a.logp64) a.logp64[row] = (double)v;
}

template <typename T>
__device__ __forceinline__ void grad_vec(const RowView<T>& rv, char* out, bool aligned, int64_t v, const float* f,
                                         float m, float nci, int64_t a, float coef) {
    constexpr int VE = Elem<T>::VE;
    float g[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) g[j] = nci * exp_diff(f[j], m);
    const int64_t ja = a + rv.mis - v * VE;             // the action's place in this vector, if it is here
    if (ja >= 0 && ja < VE)
#pragma unroll
        for (int j = 0; j < VE; ++j) if (j == ja) g[j] += coef;
    rv.store(out, aligned, v, g);
}

template <typename T>
__device__ __forceinline__ void fill_row(char* out, int64_t V, float v, int tid, int nt) {
    const RowView<T> rv(out, V);
    float f[Elem<T>::VE];
#pragma unroll
    for (int j = 0; j < Elem<T>::VE; ++j) f[j] = v;
    for (int64_t i = tid; i < rv.nvec; i += nt) rv.store(out, true, i, f);
}

// One row per workgroup of NT threads at a time, in KV vectors of registers per thread (KV = 0: streamed twice).
template <typename T, int NT, int KV, int MODE>
__global__ __launch_bounds__(NT) void row_kernel(RowArgs a) {
    constexpr int NW = NT / 64, VE = Elem<T>::VE, U = 4;
    __shared__ float s_m[NW];
    __shared__ double s_s[NW];
    __shared__ float s_coef;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    double loss = 0.0;                                                    // thread 0's
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float w = row_weight(a, row);
        char* out = a.dz ? a.dz + row_offset(row, a.inner, a.d_so, a.d_si) * (int64_t)sizeof(T) : nullptr;
        int64_t act = -1;
        bool bad = false;
        if (w != 0.0f) {
            act = row_action(a, row);
            bad = act < 0 || act >= a.V;
        }
        if (w == 0.0f || bad) {                                           // the whole workgroup agrees
            const float v = bad ? NAN : 0.0f;
            if (out) fill_row<T>(out, a.V, v, tid, NT);
            if (tid == 0) {
                row_const<MODE>(a, row, v);
                if (bad) loss = NAN;
            }
            continue;
        }
        const RowView<T> rv(a.z + row_offset(row, a.inner, a.z_so, a.z_si) * (int64_t)sizeof(T), a.V);
        const bool aligned = out && (((uintptr_t)out ^ (uintptr_t)rv.base) & 15) == 0;
        float za = 0.0f, m = -INFINITY, inv = 0.0f, coef = 0.0f;
        u32x4 x[KV > 0 ? KV : 1];
        if constexpr (KV > 0) {
#pragma unroll
            for (int k = 0; k < KV; ++k) {
                const int64_t v = tid + k * NT;
                if (v < rv.nvec) x[k] = rv.load(v);
                else x[k][0] = x[k][1] = x[k][2] = x[k][3] = Elem<T>::NEG_INF;
            }
        }
        if constexpr (MODE != MODE_GRAD) {
            if (tid == 0) za = Elem<T>::load(rv.base, act);
            float s = 0.0f;
            if constexpr (KV > 0) {
                float f[VE];
#pragma unroll
                for (int k = 0; k < KV; ++k) {
                    Elem<T>::unpack(x[k], f);
#pragma unroll
                    for (int j = 0; j < VE; ++j) m = fmaxf(m, f[j]);
                }
                const float ref = finite_or_zero(m);
#pragma unroll
                for (int k = 0; k < KV; ++k) {
                    Elem<T>::unpack(x[k], f);
#pragma unroll
                    for (int j = 0; j < VE; ++j) s += exp_diff_sum(f[j], ref);
                }
            } else {
                for (int64_t v0 = tid; v0 < rv.nvec; v0 += U * NT) {
                    u32x4 y[U];
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (v0 + u * NT < rv.nvec) y[u] = rv.load(v0 + u * NT);
                        else y[u][0] = y[u][1] = y[u][2] = y[u][3] = Elem<T>::NEG_INF;
                    }
                    float f[U * VE];
#pragma unroll
                    for (int u = 0; u < U; ++u) Elem<T>::unpack(y[u], f + u * VE);
                    accumulate<U * VE>(f, m, s);
                }
            }
            double sd = (double)s;
            join_lanes<64>(m, sd);
            if constexpr (NW > 1) {
                if (lane == 0) { s_m[wave] = m; s_s[wave] = sd; }
                __syncthreads();
                m = lane < NW ? s_m[lane] : -INFINITY;
                sd = lane < NW ? s_s[lane] : 0.0;
                join_lanes<NW>(m, sd);
                m = __shfl(m, 0, 64);
                sd = __shfl(sd, 0, 64);
            }
            inv = (float)(1.0 / sd);
            if (tid == 0) {
                loss += row_result<MODE>(a, row, w, za, m, sd, coef);
                if (MODE == MODE_LOGP && a.logp64) {
                    a.logp64[row] = ((double)za - (double)m) - log(sd);
                    a.stat_m[row] = m; a.stat_inv[row] = inv;
                }
                s_coef = coef;
            }
        } else {
            m = a.stat_m[row]; inv = a.stat_inv[row];
            coef = w * a.seq_coef[row / a.inner];
        }
        if (MODE != MODE_LOGP && out) {
            if constexpr (MODE == MODE_POLICY) { __syncthreads(); coef = s_coef; }
            const float nci = -coef * inv;
            float f[VE];
            if constexpr (KV > 0) {
#pragma unroll
                for (int k = 0; k < KV; ++k) {
                    const int64_t v = tid + k * NT;
                    if (v < rv.nvec) {
                        Elem<T>::unpack(x[k], f);
                        grad_vec<T>(rv, out, aligned, v, f, m, nci, act, coef);
                    }
                }
            } else {
                for (int64_t v0 = tid; v0 < rv.nvec; v0 += U * NT) {
                    u32x4 y[U];
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (v0 + u * NT < rv.nvec) y[u] = rv.load(v0 + u * NT);
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        if (v0 + u * NT < rv.nvec) {
                            Elem<T>::unpack(y[u], f);
                            grad_vec<T>(rv, out, aligned, v0 + u * NT, f, m, nci, act, coef);
                        }
                }
            }
        }
        if constexpr (MODE != MODE_GRAD) __syncthreads();   // s_m / s_s / s_coef are free for the next row
    }
    if (MODE == MODE_POLICY && tid == 0) a.loss_part[blockIdx.x] = loss;
}

// Short rows: G lanes to a row, EPL elements to a lane, 256 / G rows to a workgroup pass.
template <typename T, int G, int EPL, int MODE>
__global__ __launch_bounds__(256) void row_lane_kernel(RowArgs a) {
    __shared__ double s_loss[256 / G];
    constexpr int RPB = 256 / G;
    const int g = threadIdx.x & (G - 1), grp = threadIdx.x / G;
    double loss = 0.0;
    const int64_t step = (int64_t)gridDim.x * RPB, top = (a.rows + RPB - 1) / RPB * RPB;
    for (int64_t row0 = (int64_t)blockIdx.x * RPB + grp; row0 < top; row0 += step) {
        const bool in = row0 < a.rows;
        const int64_t row = in ? row0 : 0;                                // every lane takes part in the exchanges
        const float w = in ? row_weight(a, row) : 0.0f;
        const int64_t act = w != 0.0f ? row_action(a, row) : 0;
        const bool bad = act < 0 || act >= a.V, live = w != 0.0f && !bad;
        const char* z = a.z + row_offset(row, a.inner, a.z_so, a.z_si) * (int64_t)sizeof(T);
        float x[EPL], m = -INFINITY, inv, coef = 0.0f, za = 0.0f, s = 0.0f;
#pragma unroll
        for (int k = 0; k < EPL; ++k) {
            x[k] = live && g + k * G < a.V ? Elem<T>::load(z, g + k * G) : -INFINITY;
            m = fmaxf(m, x[k]);
        }
        if constexpr (MODE != MODE_GRAD) {
            if (live) za = Elem<T>::load(z, act);
            const float ref = finite_or_zero(m);
#pragma unroll
            for (int k = 0; k < EPL; ++k) s += exp_diff_sum(x[k], ref);
            double sd = (double)s;
            join_lanes<G>(m, sd);
            inv = (float)(1.0 / sd);
            if (in && g == 0) {
                if (live) {
                    loss += row_result<MODE>(a, row, w, za, m, sd, coef);
                    if (MODE == MODE_LOGP && a.logp64) {
                        a.logp64[row] = ((double)za - (double)m) - log(sd);
                        a.stat_m[row] = m; a.stat_inv[row] = inv;
                    }
                } else {
                    row_const<MODE>(a, row, bad ? NAN : 0.0f);
                    if (bad) loss = NAN;
                }
            }
            if constexpr (MODE == MODE_POLICY) coef = __shfl(coef, (threadIdx.x & 63) & ~(G - 1), 64);
        } else {
            m = live ? a.stat_m[row] : 0.0f; inv = live ? a.stat_inv[row] : 0.0f;
            coef = live ? w * a.seq_coef[row / a.inner] : 0.0f;
        }
        if (MODE != MODE_LOGP && in && a.dz) {
            char* out = a.dz + row_offset(row, a.inner, a.d_so, a.d_si) * (int64_t)sizeof(T);
            const float nci = -coef * inv;
#pragma unroll
            for (int k = 0; k < EPL; ++k) {
                const int64_t e = g + k * G;
                if (e < a.V) {
                    const float v = nci * exp_diff(x[k], m) + (e == act ? coef : 0.0f);
                    Elem<T>::store(out, e, live ? v : (bad ? NAN : 0.0f));
                }
            }
        }
    }
    if constexpr (MODE == MODE_POLICY) {
        if (g == 0) s_loss[grp] = loss;
        __syncthreads();
        if (threadIdx.x == 0) {
            double t = 0.0;
            for (int i = 0; i < RPB; ++i) t += s_loss[i];
            a.loss_part[blockIdx.x] = t;
        }
    }
}

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
    const int nw = blockDim.x >> 6;
    for (int d = 32; d >= 1; d >>= 1) v += shfl_xor_f64(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < nw; ++i) t += red[i];
    return t;
}

__global__ __launch_bounds__(1024) void loss_sum_kernel(const double* __restrict__ part, int64_t n, float* __restrict__ loss) {
    __shared__ double red[16];
    double acc = 0.0;
    for (int64_t i0 = threadIdx.x; i0 < n; i0 += 8 * 1024) {              // eight loads in flight, added in index order
        double v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = i0 + u * 1024 < n ? part[i0 + u * 1024] : 0.0;
#pragma unroll
        for (int u = 0; u < 8; ++u) acc += v[u];
    }
    acc = block_sum_f64(acc, red);
    if (threadIdx.x == 0) *loss = (float)acc;
}

// One workgroup per pair: the two sequences' weighted sums of log-probabilities, the margin
//   h = beta ((S_c - R_c) - (S_r - R_r)),
// the pair's loss -(1 - e) log sigmoid(h) - e log sigmoid(-h) and d loss / d S_c = -d loss / d S_r
//   = beta scale u (e - sigmoid(-h)),  u the pair's weight.
struct PairArgs {
    const double* logp64; const float* w; const float* ref; const float* pair_w;
    int64_t P, T;
    double beta, smooth, scale;
    float* seq_logp; float* margin; float* seq_coef; double* pair_loss;
};
__global__ __launch_bounds__(256) void pair_kernel(PairArgs a) {
    __shared__ double red[4];
    const int64_t p = blockIdx.x;
    double S[2];
    for (int side = 0; side < 2; ++side) {
        const int64_t r0 = (p + side * a.P) * a.T;
        double acc = 0.0;
        for (int64_t t = threadIdx.x; t < a.T; t += 256) {
            const float w = a.w ? a.w[r0 + t] : 1.0f;
            if (w != 0.0f) acc += (double)w * a.logp64[r0 + t];
        }
        S[side] = block_sum_f64(acc, red);
    }
    if (threadIdx.x == 0) {
        const double h = a.beta * ((S[0] - (double)a.ref[p]) - (S[1] - (double)a.ref[p + a.P]));
        const double t = log1p(exp(-fabs(h))), up = t + fmax(-h, 0.0), down = t + fmax(h, 0.0);
        const double u = a.pair_w ? (double)a.pair_w[p] : 1.0, sw = a.scale * u;
        const double dn = 1.0 / (1.0 + exp(h));                            // sigmoid(-h)
        const bool live = u != 0.0;
        const double c = live ? a.beta * sw * (a.smooth - dn) : 0.0;
        a.seq_logp[p] = (float)S[0]; a.seq_logp[p + a.P] = (float)S[1];
        a.margin[p] = live ? (float)h : 0.0f;
        a.seq_coef[p] = (float)c; a.seq_coef[p + a.P] = (float)-c;
        double l = sw * ((1.0 - a.smooth) * up + a.smooth * down);
        if (h != h) l = h * sw;
        a.pair_loss[p] = live ? l : 0.0;
    }
}

constexpr int64_t MAX_GRID = 16384;

template <typename T, int MODE>
static int64_t launch_rows(const RowArgs& a, hipStream_t st, bool dry) {
    constexpr int VE = Elem<T>::VE;
    int64_t grid;
#define MCTSQ_ROWS(kernel, nt, per)                                                               \
    do {                                                                                          \
        grid = (a.rows + (per) - 1) / (per);                                                      \
        if (grid > MAX_GRID) grid = MAX_GRID;                                                     \
        if (!dry) hipLaunchKernelGGL((kernel), dim3((unsigned)grid), dim3(nt), 0, st, a);         \
        return grid;                                                                              \
    } while (0)
#define MCTSQ_COMMA ,
    // nvec <= V / VE + 2 whatever the alignment
    const int64_t nv = a.V / VE + 2;
    if (a.V <= 32) MCTSQ_ROWS(row_lane_kernel<T MCTSQ_COMMA 4 MCTSQ_COMMA 8 MCTSQ_COMMA MODE>, 256, 64);
    if (a.V <= 256) MCTSQ_ROWS(row_lane_kernel<T MCTSQ_COMMA 16 MCTSQ_COMMA 16 MCTSQ_COMMA MODE>, 256, 16);
    if (nv <= 64 * 4) MCTSQ_ROWS(row_kernel<T MCTSQ_COMMA 64 MCTSQ_COMMA 4 MCTSQ_COMMA MODE>, 64, 1);
    if (nv <= 256 * 4) MCTSQ_ROWS(row_kernel<T MCTSQ_COMMA 256 MCTSQ_COMMA 4 MCTSQ_COMMA MODE>, 256, 1);
    if (nv <= 1024 * 4) MCTSQ_ROWS(row_kernel<T MCTSQ_COMMA 1024 MCTSQ_COMMA 4 MCTSQ_COMMA MODE>, 1024, 1);
    if (nv <= 1024 * 8) MCTSQ_ROWS(row_kernel<T MCTSQ_COMMA 1024 MCTSQ_COMMA 8 MCTSQ_COMMA MODE>, 1024, 1);
    MCTSQ_ROWS(row_kernel<T MCTSQ_COMMA 1024 MCTSQ_COMMA 0 MCTSQ_COMMA MODE>, 1024, 1);
#undef MCTSQ_ROWS
#undef MCTSQ_COMMA
}

template <int MODE>
static int64_t launch_rows(int dtype, const RowArgs& a, hipStream_t st, bool dry = false) {
    if (dtype == DT_F32) return launch_rows<float, MODE>(a, st, dry);
    if (dtype == DT_BF16) return launch_rows<__bf16, MODE>(a, st, dry);
    return launch_rows<_Float16, MODE>(a, st, dry);
}

// shapes and strides every entry point shares; fills the logits part of `a`
static int fill_rows(RowArgs& a, const void* d_logits, int dtype, int64_t rows, int64_t inner, int64_t stride_outer,
                     int64_t stride_inner, int64_t vocab, const void* d_act, int act_bytes, const float* d_weight) {
    MCTSQ_CHECK(dtype >= 0 && dtype <= 2, "logits dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    MCTSQ_CHECK(rows >= 0 && vocab >= 1 && inner >= 1, "rows must not be negative, vocab and inner at least 1");
    MCTSQ_CHECK(rows % inner == 0, "rows must be a multiple of the inner extent");
    MCTSQ_CHECK(act_bytes == 4 || act_bytes == 8, "actions must be 4- or 8-byte integers");
    MCTSQ_CHECK(rows == 0 || (d_logits && d_act), "NULL device pointer");
    const int es = dtype == DT_F32 ? 4 : 2;
    MCTSQ_CHECK(((uintptr_t)d_logits & (es - 1)) == 0, "logits are not aligned to their element size");
    MCTSQ_CHECK((inner == 1 || stride_inner >= 0) && (rows == inner || stride_outer >= 0), "negative strides");
    a = RowArgs{};
    a.z = (const char*)d_logits; a.z_so = stride_outer; a.z_si = stride_inner;
    a.rows = rows; a.inner = inner; a.V = vocab;
    a.act = d_act; a.act64 = act_bytes == 8; a.w = d_weight; a.adv_div = 1;
    return 0;
}
static int fill_grad(RowArgs& a, void* d_dlogits, int dtype, int64_t so, int64_t si) {
    const int es = dtype == DT_F32 ? 4 : 2;
    MCTSQ_CHECK(((uintptr_t)d_dlogits & (es - 1)) == 0, "dlogits is not aligned to its element size");
    // rows of the gradient must not share memory
    MCTSQ_CHECK((a.inner == 1 || si >= a.V) && (a.rows <= a.inner || so >= (a.inner - 1) * si + a.V || (a.inner == 1 && so >= a.V)
                 || (so >= a.V && si >= (a.rows / a.inner - 1) * so + a.V)), "gradient rows overlap");
    a.dz = (char*)d_dlogits; a.d_so = so; a.d_si = si;
    return 0;
}

static int64_t pref_ws(int64_t seqs, int64_t T, int64_t* off) {
    const int64_t rows = seqs * T;
    int64_t o = 0;
    auto take = [&](int64_t bytes) { const int64_t at = o; o += round_up(bytes, 16); return at; };
    off[0] = take(rows * 8);            // logp64
    off[1] = take(rows * 4);            // stat_m
    off[2] = take(rows * 4);            // stat_inv
    off[3] = take(rows * 4);            // logp (fp32, when the caller wants none)
    off[4] = take(seqs * 4);            // seq_coef
    off[5] = take(seqs / 2 * 8);        // pair_loss
    return o < 16 ? 16 : o;
}

}  // namespace mctsq

using namespace mctsq;

extern "C" int mctsq_token_logprobs(const void* d_logits, int dtype, int64_t rows, int64_t inner, int64_t stride_outer,
                                    int64_t stride_inner, int64_t vocab, const void* d_act, int act_bytes,
                                    const float* d_weight, float* d_logp, void* stream) {
    RowArgs a;
    if (int rc = fill_rows(a, d_logits, dtype, rows, inner, stride_outer, stride_inner, vocab, d_act, act_bytes, d_weight)) return rc;
    if (rows == 0) return 0;
    MCTSQ_CHECK(d_logp, "NULL device pointer");
    a.logp = d_logp;
    launch_rows<MODE_LOGP>(dtype, a, (hipStream_t)stream);
    MCTSQ_HIP(hipGetLastError());
    return 0;
}

extern "C" int64_t mctsq_policy_loss_workspace_bytes(int64_t rows) {
    MCTSQ_CHECK(rows >= 0, "negative row count");
    return 8 * (rows < 1 ? 1 : (rows < MAX_GRID ? rows : MAX_GRID));
}

extern "C" int mctsq_policy_loss(const void* d_logits, int dtype, int64_t rows, int64_t inner, int64_t stride_outer,
                                 int64_t stride_inner, int64_t vocab, const void* d_act, int act_bytes,
                                 const float* d_old_logp, const float* d_ref_logp, const float* d_adv, int64_t adv_div,
                                 const float* d_weight, double clip_low, double clip_high, double kl_coef,
                                 double loss_scale, float* d_loss, float* d_logp, float* d_kl, void* d_dlogits,
                                 int64_t dstride_outer, int64_t dstride_inner, void* d_ws, int64_t ws_bytes, void* stream) {
    RowArgs a;
    if (int rc = fill_rows(a, d_logits, dtype, rows, inner, stride_outer, stride_inner, vocab, d_act, act_bytes, d_weight)) return rc;
    MCTSQ_CHECK(d_loss && (rows == 0 || (d_adv && d_logp && d_kl)), "NULL device pointer");
    MCTSQ_CHECK(adv_div >= 1, "adv_div must be at least 1");
    MCTSQ_CHECK(clip_low >= 0.0 && clip_high >= 0.0, "clip ranges must not be negative");
    MCTSQ_CHECK(kl_coef == kl_coef && loss_scale == loss_scale, "kl_coef / loss_scale is NaN");
    MCTSQ_CHECK(d_ws && ((uintptr_t)d_ws & 7) == 0 && ws_bytes >= mctsq_policy_loss_workspace_bytes(rows),
                "workspace must hold mctsq_policy_loss_workspace_bytes(rows), 8-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    int64_t parts = 0;
    if (rows > 0) {
        if (d_dlogits) { if (int rc = fill_grad(a, d_dlogits, dtype, dstride_outer, dstride_inner)) return rc; }
        a.old_logp = d_old_logp; a.ref_logp = d_ref_logp; a.adv = d_adv; a.adv_div = adv_div;
        a.clip_lo = 1.0 - clip_low; a.clip_hi = 1.0 + clip_high; a.kl_coef = kl_coef; a.scale = loss_scale;
        a.logp = d_logp; a.kl = d_kl; a.loss_part = (double*)d_ws;
        parts = launch_rows<MODE_POLICY>(dtype, a, st);
    }
    hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, st, (const double*)d_ws, parts, d_loss);
    MCTSQ_HIP(hipGetLastError());
    return 0;
}

extern "C" int64_t mctsq_preference_loss_workspace_bytes(int64_t pairs, int64_t tokens) {
    MCTSQ_CHECK(pairs >= 0 && tokens >= 0, "negative size");
    int64_t off[6];
    return pref_ws(2 * pairs, tokens, off);
}

extern "C" int mctsq_preference_loss(const void* d_logits, int dtype, int64_t pairs, int64_t tokens, int64_t stride_outer,
                                     int64_t stride_inner, int64_t vocab, const void* d_act, int act_bytes,
                                     const float* d_ref_logp, const float* d_weight, const float* d_pair_weight,
                                     double beta, double label_smoothing, double loss_scale, float* d_loss,
                                     float* d_seq_logp, float* d_margin, void* d_dlogits, int64_t dstride_outer,
                                     int64_t dstride_inner, void* d_ws, int64_t ws_bytes, void* stream) {
    MCTSQ_CHECK(pairs >= 0 && tokens >= 0 && pairs <= ((int64_t)1 << 30), "pairs / tokens out of range");
    const int64_t rows = 2 * pairs * tokens;
    RowArgs a;
    if (int rc = fill_rows(a, d_logits, dtype, rows, tokens > 0 ? tokens : 1, stride_outer, stride_inner, vocab, d_act, act_bytes, d_weight)) return rc;
    MCTSQ_CHECK(d_loss && (pairs == 0 || (d_ref_logp && d_seq_logp && d_margin)), "NULL device pointer");
    MCTSQ_CHECK(beta == beta && loss_scale == loss_scale, "beta / loss_scale is NaN");
    MCTSQ_CHECK(label_smoothing >= 0.0 && label_smoothing <= 0.5, "label_smoothing must lie in [0, 0.5]");
    MCTSQ_CHECK(d_ws && ((uintptr_t)d_ws & 15) == 0 && ws_bytes >= mctsq_preference_loss_workspace_bytes(pairs, tokens),
                "workspace must hold mctsq_preference_loss_workspace_bytes(pairs, tokens), 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    int64_t off[6];
    pref_ws(2 * pairs, tokens, off);
    char* ws = (char*)d_ws;
    a.logp64 = (double*)(ws + off[0]); a.stat_m = (float*)(ws + off[1]); a.stat_inv = (float*)(ws + off[2]);
    a.logp = (float*)(ws + off[3]);
    a.pair_w = d_pair_weight; a.pairs = pairs;
    if (rows > 0) {
        if (d_dlogits) { if (int rc = fill_grad(a, d_dlogits, dtype, dstride_outer, dstride_inner)) return rc; }
        RowArgs f = a;
        f.dz = nullptr;
        launch_rows<MODE_LOGP>(dtype, f, st);
    }
    PairArgs p{};
    p.logp64 = a.logp64; p.w = d_weight; p.ref = d_ref_logp; p.pair_w = d_pair_weight; p.P = pairs; p.T = tokens;
    p.beta = beta; p.smooth = label_smoothing; p.scale = loss_scale;
    p.seq_logp = d_seq_logp; p.margin = d_margin; p.seq_coef = (float*)(ws + off[4]); p.pair_loss = (double*)(ws + off[5]);
    if (pairs > 0) hipLaunchKernelGGL(pair_kernel, dim3((unsigned)pairs), dim3(256), 0, st, p);
    hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, st, (const double*)p.pair_loss, pairs, d_loss);
    if (rows > 0 && d_dlogits) {
        a.seq_coef = p.seq_coef;
        launch_rows<MODE_GRAD>(dtype, a, st);
    }
    MCTSQ_HIP(hipGetLastError());
    return 0;
}
