// What a policy learns from: log-probabilities of given actions, the clipped policy-ratio loss with a KL term, and the
// paired log-ratio loss over preferred / rejected sequences, each with its gradient by the logits.
//
//   logp_i = z_i[a_i] - lse_i,   lse_i = log sum_j exp z_i[j],   d logp_i / d z_i[j] = [j = a_i] - p_i[j]
//
// so every loss here is a coefficient c_i = d loss / d logp_i per row and the gradient row c_i (one_hot(a_i) - p_i).
// The bound is HBM: each logit read once, each gradient element written once; the exponentials are the next one.
//   - rows of more than 256 elements: RW waves own a row at a time and take it in 16-byte vectors, U of them in flight per
//     lane, every lane with a running (max, sum of exponentials); the pairs are joined over the waves with one barrier, one
//     thread turns them into the coefficient.  Where U vectors a lane hold the whole row (HOLD), the exponentials stay in
//     registers and the gradient is one product per element; longer rows are read a second time, now from the caches.
//   - rows of at most 256 elements go to groups of 1, 4 or 16 lanes and stay in registers, many rows to a workgroup.
// Statistics: exponentials in fp32, added in fp64, of many 16-bit rows four at a time in fp32 first (a sum of fp32 steps shows
// where one action has nearly all the probability and its logarithm is small; see sum_exp); the joins across lanes, the logarithm, ratio, KL term
// and loss in fp64: the clip decides on a ratio that two evaluations must agree on.
// Rows of weight 0 are padding: their logits, action, and statistics are not read, their outputs are exactly 0.
// An action outside [0, V) on a row that has weight makes that row's outputs and the loss NaN; nothing is read for it.
// Sums are joined in a fixed order: the same inputs give the same bits.
// Measured (a large copy reaches 5.15 TB/s, a read 6.05): log-probabilities of 4096 x 32000 bf16 5.9 TB/s, fp32 5.4; policy
// loss and gradient of 8192 x 16000 bf16 5.0, 4096 x 32000 fp32 5.2, 4096 x 131072 bf16 with a third of the rows padding
// 404 us (343 at the copy's rate); preference loss of 16 x 511 x 50257 bf16 392 us (359 with its second reading).
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
    int one_group;                            // inner == all rows: nothing to divide
    const void* act; int act64;
    const float* w;                           // row weights, NULL: 1
    const float* pair_w; int64_t pairs;       // pair weights of the preference loss (row / inner = pair or pairs + pair)
    // policy
    const float* old_logp; const float* ref_logp; const float* adv; int64_t adv_div;
    double clip_lo, clip_hi, kl_coef, scale;
    float* logp; float* kl;
    double* loss_part; float* loss;           // one part per workgroup, or the loss itself from a launch of one
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
        u32x4 c;                                            // element by element, all loads at once
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const int64_t e = e0 + j;
            const bool in = e >= 0 && e < V;
            const int64_t at = in ? e : 0;
            if constexpr (sizeof(T) == 4) c[j] = reinterpret_cast<const unsigned*>(base)[at];
            else {
                const unsigned h = reinterpret_cast<const unsigned short*>(base)[at];
                c[j >> 1] = (j & 1) ? (c[j >> 1] | (h << 16)) : h;
            }
            constexpr int sh = sizeof(T) == 4 ? 0 : 1;
            const unsigned mask = sizeof(T) == 4 ? 0xffffffffu : (j & 1) ? 0xffff0000u : 0xffffu;
            if (in) u[j >> sh] = (u[j >> sh] & ~mask) | (c[j >> sh] & mask);
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
// The same, and in r what its argument lost in rounding (3e-7 of the exponential at x - m = -10): exp(x - m) = e (1 + r log 2).
// Far below, where e is 0, r must not be NaN.
constexpr float LN2 = 0.6931471805599453f;
__device__ __forceinline__ float exp_diff_rest(float x, float m, float& r) {
    const float d = __builtin_elementwise_maximum(x - m, -200.0f), t = d * LOG2E_LO, y = fmaf(d, LOG2E, t);   // NaN stays NaN
    r = fmaf(d, LOG2E, -y) + t;
    return fast_exp2(y);
}
template <bool ACC>
__device__ __forceinline__ double exp_factor(float x, float m) {
    if constexpr (!ACC) return (double)exp_diff_sum(x, m);
    float r;
    const float e = exp_diff_rest(x, m, r);
    return (double)e * fma((double)r, (double)LN2, 1.0);
}
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }

// Sum of exp(f - ref) over N values, left in f: four at a time in fp32, those sums in fp64 -- or, ACC, each in fp64 together
// with what the exponentials' arguments lost.  Two log-probabilities' difference, rows of 32000 to 81298, rms against 64 bits:
// 2.9e-8, ACC 1.0e-8 (what is left is the exponential instruction's own).  Either is below what a log-probability beyond -1/2
// loses when it is stored in fp32, so a row in a short and in a long call gives the same value or its neighbour; a preference
// margin and a ratio see the 64-bit value.  ACC is for fp32 logits (4096 x 32000: 92 -> 97 us, with the gradient 202 -> 198) and
// for at most a row per CU, where the call around the launch takes longer than the kernel (48 x 32000 bf16: 5.8 -> 7.2 us on the
// device, the call 10 either way).  Many 16-bit rows would pay for it: log-probabilities of 6 x 1023 x 50257 bf16 84 -> 106 us,
// policy loss of 3 x 333 x 50257 fp16 51 -> 64, preference loss of 4 pairs x 61 x 32000 bf16 25.5 -> 28.4.
template <int N, bool ACC>
__device__ __forceinline__ double sum_exp(float* f, float ref) {
    double s = 0.0, t = 0.0;
#pragma unroll
    for (int j = 0; j < N; j += 4) {
        if constexpr (ACC) {
            float c = 0.0f;
#pragma unroll
            for (int k = j; k < j + 4; ++k) {
                float r;
                f[k] = exp_diff_rest(f[k], ref, r);
                c = fmaf(f[k], r, c);
            }
            s += (double)f[j];
            t += (double)f[j + 1];
            s += (double)f[j + 2];
            t += (double)f[j + 3];
            s += (double)(c * LN2);
        } else {
#pragma unroll
            for (int k = j; k < j + 4; ++k) f[k] = exp_diff_sum(f[k], ref);
            s += (double)((f[j] + f[j + 1]) + (f[j + 2] + f[j + 3]));
        }
    }
    return ACC ? s + t : s;
}
template <int N, bool ACC>
__device__ __forceinline__ void accumulate(float* f, float& m, double& s) {
    float nm = m;
#pragma unroll
    for (int j = 0; j < N; ++j) nm = fmaxf(nm, f[j]);
    const float ref = finite_or_zero(nm);
    s *= exp_factor<ACC>(m, ref);                       // m = -inf: the factor is 0, and so is s
    s += sum_exp<N, ACC>(f, ref);
    m = nm;
}

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CTRL, 0xf, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, ((uint64_t)(unsigned)hi << 32) | (unsigned)lo);
}
__device__ __forceinline__ float lane_f32(float v, int l) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
__device__ __forceinline__ double lane_f64(double v, int l) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)b, l);
    const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(b >> 32), l);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// a pair (m, s) as it counts under the joint maximum M
template <bool ACC>
__device__ __forceinline__ double rescaled(float m, double s, float M) {
    const double r = s * exp_factor<ACC>(m, finite_or_zero(M));
    return m > -INFINITY || s != s ? r : 0.0;            // an empty set, or one of -inf only; NaN stays
}
// join over groups of W = 1, 4, 16 or 64 consecutive lanes: every lane gets the group's max and sum
template <int W, bool ACC>
__device__ __forceinline__ void join_lanes(float& m, double& s) {
    if constexpr (W == 1) return;
    float M = m;
    if constexpr (W == 4) {
        M = fmaxf(M, dpp_row<0xB1>(M));                  // quad_perm [1,0,3,2], [2,3,0,1]
        M = fmaxf(M, dpp_row<0x4E>(M));
    } else if constexpr (W > 1) M = row16_max_dpp(M);
    if constexpr (W == 64) M = fmaxf(fmaxf(lane_f32(M, 0), lane_f32(M, 16)), fmaxf(lane_f32(M, 32), lane_f32(M, 48)));
    s = rescaled<ACC>(m, s, M);
    if constexpr (W == 4) {
        s += dpp_f64<0xB1>(s);
        s += dpp_f64<0x4E>(s);
    } else {
        s += dpp_f64<0x128>(s);                          // rotations within rows of 16
        s += dpp_f64<0x124>(s);
        s += dpp_f64<0x122>(s);
        s += dpp_f64<0x121>(s);
    }
    if constexpr (W == 64) s = (lane_f64(s, 0) + lane_f64(s, 16)) + (lane_f64(s, 32) + lane_f64(s, 48));
    m = M;
}

__device__ __forceinline__ int64_t row_action(const RowArgs& a, int64_t row) {
    return a.act64 ? reinterpret_cast<const int64_t*>(a.act)[row] : (int64_t)reinterpret_cast<const int32_t*>(a.act)[row];
}
__device__ __forceinline__ int64_t row_group(const RowArgs& a, int64_t row) {      // row / inner; both fit 32 bits
    return a.one_group ? 0 : (int64_t)((unsigned)row / (unsigned)a.inner);
}
__device__ __forceinline__ float row_weight(const RowArgs& a, int64_t row) {
    if (a.pair_w) {
        const int64_t q = row_group(a, row);
        if (a.pair_w[q < a.pairs ? q : q - a.pairs] == 0.0f) return 0.0f;
    }
    return a.w ? a.w[row] : 1.0f;
}
__device__ __forceinline__ int64_t row_offset(const RowArgs& a, int64_t row, int64_t so, int64_t si) {
    const int64_t q = row_group(a, row);
    return q * so + (row - q * a.inner) * si;
}

// Logarithm and exponential in fp64 by their series, to about 1e-14 relative.  One lane of a row evaluates them while the
// row's other waves wait, so they are short, and their constants are set in scalar registers on the spot (scalar_const;
// left alone the compiler keeps them in vector registers over the loop of rows: 125 to 155 registers with the library's
// functions inlined, which halves the waves that hide the loads).
__device__ __forceinline__ double scalar_const(double c) {
    asm volatile("" : "+s"(c));
    return c;
}
// log s for s >= 1/2: s = 2^k f, f in [sqrt 1/2, sqrt 2), t = (f - 1) / (f + 1), log f = 2 (t + t^3 / 3 + t^5 / 5 + ...), |t| < 0.172
__device__ __forceinline__ double log_f64(double s) {
    const uint64_t b = __builtin_bit_cast(uint64_t, s);
    int k = (int)(b >> 52) - 1023;
    double f = __builtin_bit_cast(double, (b & 0x000fffffffffffffull) | 0x3ff0000000000000ull);
    if (f > scalar_const(1.4142135623730951)) { f *= 0.5; ++k; }
    const double d = f + 1.0;
    double r = __builtin_amdgcn_rcp(d);
    r = fma(r, fma(-d, r, 1.0), r);
    r = fma(r, fma(-d, r, 1.0), r);
    const double t = (f - 1.0) * r, w = t * t;
    double p = scalar_const(1.0 / 15);
#pragma unroll
    for (int i = 13; i >= 1; i -= 2) p = fma(p, w, scalar_const(1.0 / i));
    const double v = fma((double)k, scalar_const(0.6931471805599453), 2.0 * t * p);
    return s > 0.0 ? v : (s == 0.0 ? -INFINITY : s);            // NaN stays NaN
}
// e^x = 2^k (1 + p), p = e^r - 1 by its series, |r| <= log(2) / 2
__device__ __forceinline__ double exp_parts(double x, int& k) {
    const double lim = scalar_const(1100.0), c = fmin(fmax(x, -lim), lim), n = rint(c * scalar_const(1.4426950408889634));
    // log 2 as its first 32 bits after the point, which n times are exact, and the rest
    const double r = fma(-n, scalar_const(1.9082149292705877e-10), fma(-n, scalar_const(0.6931471803691238), c));
    constexpr double fact[13] = {1, 1, 2, 6, 24, 120, 720, 5040, 40320, 362880, 3628800, 39916800, 479001600};
    double p = scalar_const(1.0 / fact[12]);
#pragma unroll
    for (int i = 11; i >= 1; --i) p = fma(p, r, scalar_const(1.0 / fact[i]));
    k = (int)n;
    return p * r;
}
__device__ __forceinline__ double exp_f64(double x) {
    int k;
    const double p = exp_parts(x, k);
    return x == x ? ldexp(1.0 + p, k) : x;
}
__device__ __forceinline__ double expm1_f64(double x) {
    int k;
    const double p = exp_parts(x, k);
    // from 2^60 on the 1 is below half a step; two parts of unlike signs would meet as infinities further up
    const double v = k > 60 ? ldexp(1.0 + p, k) : ldexp(p, k) + (ldexp(1.0, k) - 1.0);
    return x == x ? v : x;
}

// The row's log-probability and, in the policy mode, its loss and coefficient; writes the per-row outputs.
// L(r) = -min(r A, clip(r, lo, hi) A), r = exp(logp - old);  k = exp(d) - d - 1, d = ref - logp (never negative, 0 at d = 0)
// d L / d logp = -r A where the unclipped product is the smaller one (or equal), else 0;  d k / d logp = 1 - exp(d)
template <int MODE>
__device__ __forceinline__ double row_result(const RowArgs& a, int64_t row, float w, float za, float m, double s, float inv,
                                             float& coef) {
    const double logp = ((double)za - (double)m) - log_f64(s);
    a.logp[row] = (float)logp;
    if (MODE == MODE_LOGP && a.logp64) {
        a.logp64[row] = logp;
        a.stat_m[row] = m; a.stat_inv[row] = inv;
    }
    if constexpr (MODE == MODE_POLICY) {
        const double A = (double)a.adv[a.adv_div == 1 ? row : a.adv_div == a.inner ? row_group(a, row) : row / a.adv_div];
        const double r = a.old_logp ? exp_f64(logp - (double)a.old_logp[row]) : (logp == logp ? 1.0 : logp);
        // 0 where A is 0 and r infinite (a behaviour policy that gave the action no probability)
        const double un = A == 0.0 && r == r ? 0.0 : r * A, cl = A == 0.0 ? 0.0 : fmin(fmax(r, a.clip_lo), a.clip_hi) * A;
        double loss = -(un <= cl ? un : cl), c = un <= cl ? -un : 0.0, k = 0.0;
        if (un != un) loss = c = un;
        if (a.ref_logp) {
            const double d = (double)a.ref_logp[row] - logp, e = expm1_f64(d);
            k = e == INFINITY ? e : e - d;                               // d may be infinite
            if (a.kl_coef != 0.0) {                                      // else k is only reported
                loss += a.kl_coef * k;
                c -= a.kl_coef * e;
            }
        }
        a.kl[row] = (float)k;
        const double sw = a.scale * (double)w;
        coef = (float)(sw * c);
        return sw * loss;
    }
    return 0.0;
}

// a workgroup's share of the loss; a launch of one workgroup needs nobody to add them up
__device__ __forceinline__ void put_loss(const RowArgs& a, double loss) {
    if (gridDim.x == 1) *a.loss = (float)loss;
    else a.loss_part[blockIdx.x] = loss;
}

// outputs of a padding row, and of one whose action does not exist
template <int MODE>
__device__ __forceinline__ void row_const(const RowArgs& a, int64_t row, float v) {
    if constexpr (MODE == MODE_LOGP || MODE == MODE_POLICY) a.logp[row] = v;
    if constexpr (MODE == MODE_POLICY) a.kl[row] = v;
    if (MODE == MODE_LOGP && a.logp64) a.logp64[row] = (double)v;
}

// the action's own element, c - c p; of an infinite coefficient the formula's c (1 - p)
__device__ __forceinline__ float at_action(float g, float coef) { return fabsf(coef) < INFINITY ? g + coef : coef; }

// vector v of the gradient: g holds -c p, the action's own element gets its c
template <typename T>
__device__ __forceinline__ void put_grad(const RowView<T>& rv, char* out, bool aligned, int64_t v, float* g, int64_t a, float coef) {
    constexpr int VE = Elem<T>::VE;
    const int64_t ja = a + rv.mis - v * VE;             // the action's place in this vector, if it is here
    if (ja >= 0 && ja < VE)
#pragma unroll
        for (int j = 0; j < VE; ++j) if (j == ja) g[j] = at_action(g[j], coef);
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

// Long rows: RW waves to a row; one row at a time, or four rows to a workgroup where a wave has its own (RW = 1).
template <typename T, int RW, int U, bool HOLD, int MODE, bool ACC>
__global__ __launch_bounds__(RW == 1 ? 256 : RW * 64) void row_kernel(RowArgs a) {
    constexpr int NT = RW * 64, RPB = RW == 1 ? 4 : 1, VE = Elem<T>::VE;
    static_assert(!HOLD || MODE == MODE_POLICY, "only the one-launch gradient keeps a row");
    __shared__ float s_m[16];
    __shared__ double s_s[16];
    __shared__ float s_coef;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = RW == 1 ? lane : threadIdx.x;
    double loss = 0.0;                                                    // lane 0's of the row's first wave
    for (int64_t row = (int64_t)blockIdx.x * RPB + (RW == 1 ? wave : 0); row < a.rows; row += (int64_t)gridDim.x * RPB) {
        const float w = row_weight(a, row);
        char* out = a.dz ? a.dz + row_offset(a, row, a.d_so, a.d_si) * (int64_t)sizeof(T) : nullptr;
        int64_t act = -1;
        bool bad = false;
        if (w != 0.0f) {
            act = row_action(a, row);
            bad = act < 0 || act >= a.V;
        }
        if (w == 0.0f || bad) {                                           // all of the row's threads agree
            const float v = bad ? NAN : 0.0f;
            if (out) fill_row<T>(out, a.V, v, tid, NT);
            if (tid == 0) {
                row_const<MODE>(a, row, v);
                if (bad) loss = NAN;
            }
            continue;
        }
        const RowView<T> rv(a.z + row_offset(a, row, a.z_so, a.z_si) * (int64_t)sizeof(T), a.V);
        const bool aligned = out && (((uintptr_t)out ^ (uintptr_t)rv.base) & 15) == 0;
        float za = 0.0f, m = -INFINITY, inv = 0.0f, coef = 0.0f;
        float ex[HOLD ? U * VE : 1], lane_m = 0.0f;
        if constexpr (MODE != MODE_GRAD) {
            if (tid == 0) za = Elem<T>::load(rv.base, act);
            double sd = 0.0;
            if constexpr (HOLD) {
                u32x4 y[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (tid + u * NT < rv.nvec) y[u] = rv.load(tid + u * NT);
                    else y[u][0] = y[u][1] = y[u][2] = y[u][3] = Elem<T>::NEG_INF;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) Elem<T>::unpack(y[u], ex + u * VE);
#pragma unroll
                for (int j = 0; j < U * VE; ++j) m = fmaxf(m, ex[j]);
                sd = sum_exp<U * VE, ACC>(ex, finite_or_zero(m));
                lane_m = m;
            } else for (int64_t v0 = tid; v0 < rv.nvec; v0 += U * NT) {
                u32x4 y[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (v0 + u * NT < rv.nvec) y[u] = rv.load(v0 + u * NT);
                    else y[u][0] = y[u][1] = y[u][2] = y[u][3] = Elem<T>::NEG_INF;
                }
                float f[U * VE];
#pragma unroll
                for (int u = 0; u < U; ++u) Elem<T>::unpack(y[u], f + u * VE);
                accumulate<U * VE, ACC>(f, m, sd);
            }
            join_lanes<64, ACC>(m, sd);
            if constexpr (RW > 1) {
                if (lane == 0) { s_m[wave] = m; s_s[wave] = sd; }
                __syncthreads();
                m = (lane & 15) < RW ? s_m[lane & 15] : -INFINITY;
                sd = (lane & 15) < RW ? s_s[lane & 15] : 0.0;
                join_lanes<16, ACC>(m, sd);
            }
            inv = fast_rcp((float)sd);
            if (tid == 0) {
                loss += row_result<MODE>(a, row, w, za, m, sd, inv, coef);
                if (RW > 1) s_coef = coef;
            }
        } else {
            m = a.stat_m[row]; inv = a.stat_inv[row];
            coef = w * a.seq_coef[row_group(a, row)];
        }
        if (MODE != MODE_LOGP && out) {
            if constexpr (MODE == MODE_POLICY) {
                if constexpr (RW > 1) { __syncthreads(); coef = s_coef; }
                else coef = lane_f32(coef, 0);
            }
            const float nci = -coef * inv;
            float f[VE];
            if constexpr (HOLD) {
                const float scale = nci * exp_diff(lane_m, m);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (tid + u * NT < rv.nvec) {
#pragma unroll
                        for (int j = 0; j < VE; ++j) f[j] = scale * ex[u * VE + j];
                        put_grad<T>(rv, out, aligned, tid + u * NT, f, act, coef);
                    }
            } else for (int64_t v0 = tid; v0 < rv.nvec; v0 += U * NT) {
                u32x4 y[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (v0 + u * NT < rv.nvec) y[u] = rv.load(v0 + u * NT);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (v0 + u * NT < rv.nvec) {
                        Elem<T>::unpack(y[u], f);
#pragma unroll
                        for (int j = 0; j < VE; ++j) f[j] = nci * exp_diff(f[j], m);
                        put_grad<T>(rv, out, aligned, v0 + u * NT, f, act, coef);
                    }
            }
        }
        if constexpr (MODE != MODE_GRAD && RW > 1) __syncthreads();       // s_m / s_s / s_coef are free for the next row
    }
    if constexpr (MODE == MODE_POLICY) {
        if constexpr (RW == 1) {
            if (lane == 0) s_s[wave] = loss;
            __syncthreads();
            loss = (s_s[0] + s_s[1]) + (s_s[2] + s_s[3]);
        }
        if (threadIdx.x == 0) put_loss(a, loss);
    }
}

// sum over the workgroup in a fixed order, every thread gets it; `red` holds one word per wave
__device__ __forceinline__ double wave_sum_f64(double s) {
    s += dpp_f64<0x128>(s);
    s += dpp_f64<0x124>(s);
    s += dpp_f64<0x122>(s);
    s += dpp_f64<0x121>(s);
    return (lane_f64(s, 0) + lane_f64(s, 16)) + (lane_f64(s, 32) + lane_f64(s, 48));
}
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
    const int nw = blockDim.x >> 6;
    v = wave_sum_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double t = 0.0;
    for (int i = 0; i < nw; ++i) t += red[i];
    return t;
}

// Short rows: G lanes to a row, EPL elements to a lane, NT / G rows to a pass of the workgroup.
template <typename T, int G, int EPL, int NT, int MODE>
__global__ __launch_bounds__(NT) void row_lane_kernel(RowArgs a) {
    __shared__ double s_loss[NT / 64];
    constexpr int RPB = NT / G;
    const int g = threadIdx.x & (G - 1), grp = threadIdx.x / G;
    double loss = 0.0;
    const int64_t step = (int64_t)gridDim.x * RPB, top = (a.rows + RPB - 1) / RPB * RPB;
    for (int64_t row0 = (int64_t)blockIdx.x * RPB + grp; row0 < top; row0 += step) {
        const bool in = row0 < a.rows;
        const int64_t row = in ? row0 : 0;                                // every lane takes part in the exchanges
        const float w = in ? row_weight(a, row) : 0.0f;
        const int64_t act = w != 0.0f ? row_action(a, row) : 0;
        const bool bad = act < 0 || act >= a.V, live = w != 0.0f && !bad;
        const char* z = a.z + row_offset(a, row, a.z_so, a.z_si) * (int64_t)sizeof(T);
        float x[EPL], m = -INFINITY, lane_m = 0.0f, inv, coef = 0.0f, za = 0.0f;
#pragma unroll
        for (int k = 0; k < EPL; ++k) {
            x[k] = -INFINITY;
            if (k * G >= a.V) continue;                                   // the whole launch agrees
            if (live && g + k * G < a.V) x[k] = Elem<T>::load(z, g + k * G);
            m = fmaxf(m, x[k]);
        }
        if constexpr (MODE != MODE_GRAD) {
            if (live) za = Elem<T>::load(z, act);
            const float ref = finite_or_zero(m);
            double sd = 0.0;
            lane_m = m;
#pragma unroll
            for (int k = 0; k < EPL; ++k)
                if (k * G < a.V) {
                    float r;
                    x[k] = exp_diff_rest(x[k], ref, r);
                    sd += (double)x[k] * fma((double)r, (double)LN2, 1.0);
                }
            join_lanes<G, true>(m, sd);
            inv = fast_rcp((float)sd);
            if (in && g == 0) {
                if (live) loss += row_result<MODE>(a, row, w, za, m, sd, inv, coef);
                else {
                    row_const<MODE>(a, row, bad ? NAN : 0.0f);
                    if (bad) loss = NAN;
                }
            }
            if constexpr (MODE == MODE_POLICY && G > 1) coef = __shfl(coef, (threadIdx.x & 63) & ~(G - 1), 64);
        } else {
            m = live ? a.stat_m[row] : 0.0f; inv = live ? a.stat_inv[row] : 0.0f;
            coef = live ? w * a.seq_coef[row_group(a, row)] : 0.0f;
        }
        if (MODE != MODE_LOGP && in && a.dz) {
            char* out = a.dz + row_offset(a, row, a.d_so, a.d_si) * (int64_t)sizeof(T);
            float scale = -coef * inv;
            if (MODE != MODE_GRAD) scale *= exp_diff(lane_m, m);
#pragma unroll
            for (int k = 0; k < EPL; ++k) {
                const int64_t e = g + k * G;
                if (e < a.V) {
                    const float g0 = scale * (MODE == MODE_GRAD ? exp_diff(x[k], m) : x[k]), v = e == act ? at_action(g0, coef) : g0;
                    Elem<T>::store(out, e, live ? v : (bad ? NAN : 0.0f));
                }
            }
        }
    }
    if constexpr (MODE == MODE_POLICY) {
        const double t = block_sum_f64(loss, s_loss);                     // lanes other than a row's first hold 0
        if (threadIdx.x == 0) put_loss(a, t);
    }
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

// A workgroup takes 64 pairs: its 16 waves add up the two sequences' weighted log-probabilities of four pairs each, then
// 64 lanes evaluate a pair each: the margin
//   h = beta ((S_c - R_c) - (S_r - R_r)),
// the pair's loss -(1 - e) log sigmoid(h) - e log sigmoid(-h) and d loss / d S_c = -d loss / d S_r
//   = beta scale u (e - sigmoid(-h)),  u the pair's weight.
struct PairArgs {
    const double* logp64; const float* w; const float* ref; const float* pair_w;
    int64_t P, T;
    double beta, smooth, scale;
    float* seq_logp; float* margin; float* seq_coef; double* loss_part; float* loss;
};
constexpr int PAIRS = 64;
__global__ __launch_bounds__(1024) void pair_kernel(PairArgs a) {
    __shared__ double S[2 * PAIRS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t base = (int64_t)blockIdx.x * PAIRS;
    double acc[8];                                                        // [pair of four][side]
#pragma unroll
    for (int q = 0; q < 8; ++q) acc[q] = 0.0;
    bool live[4];                                                         // padding pairs: nothing of theirs counts
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int64_t p = base + wave + 16 * q;
        live[q] = p < a.P && !(a.pair_w && a.pair_w[p] == 0.0f);
    }
    for (int64_t t = lane; t < a.T; t += 64) {                            // eight loads under way, each sum in order
        double v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int64_t p = base + wave + 16 * (q >> 1), row = (p + (q & 1) * a.P) * a.T + t;
            const bool in = live[q >> 1];
            const float w = in ? (a.w ? a.w[row] : 1.0f) : 0.0f;
            const double l = in ? a.logp64[row] : 0.0;
            v[q] = w != 0.0f ? (double)w * l : 0.0;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] += v[q];
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const double s = wave_sum_f64(acc[q]);
        if (lane == 0) S[2 * (wave + 16 * (q >> 1)) + (q & 1)] = s;
    }
    __syncthreads();
    if (wave > 0) return;
    const int64_t p = base + lane;
    double l = 0.0;
    if (p < a.P) {
        const double Sc = S[2 * lane], Sr = S[2 * lane + 1];
        const double h = a.beta * ((Sc - (double)a.ref[p]) - (Sr - (double)a.ref[p + a.P]));
        const double t = log1p(exp(-fabs(h))), up = t + fmax(-h, 0.0), down = t + fmax(h, 0.0);
        const double u = a.pair_w ? (double)a.pair_w[p] : 1.0, sw = a.scale * u;
        const double dn = 1.0 / (1.0 + exp(h));                            // sigmoid(-h)
        const bool live = u != 0.0;
        const double c = live ? a.beta * sw * (a.smooth - dn) : 0.0;
        a.seq_logp[p] = (float)Sc; a.seq_logp[p + a.P] = (float)Sr;
        a.margin[p] = live ? (float)h : 0.0f;
        a.seq_coef[p] = (float)c; a.seq_coef[p + a.P] = (float)-c;
        l = sw * ((1.0 - a.smooth) * up + (a.smooth > 0.0 ? a.smooth * down : 0.0));      // h may be infinite
        if (h != h) l = h * sw;
        if (!live) l = 0.0;
    }
    l = wave_sum_f64(l);
    if (lane == 0) {
        if (gridDim.x == 1) *a.loss = (float)l;
        else a.loss_part[blockIdx.x] = l;
    }
}

constexpr int64_t MAX_GRID = 16384;

template <typename T, int MODE, bool ACC>
static int64_t launch_rows(const RowArgs& a, hipStream_t st) {
    int64_t grid;
#define MCTSQ_ROWS(nt, per, ...)                                                                  \
    do {                                                                                          \
        grid = (a.rows + (per) - 1) / (per);                                                      \
        if (grid > MAX_GRID) grid = MAX_GRID;                                                     \
        hipLaunchKernelGGL((__VA_ARGS__), dim3((unsigned)grid), dim3(nt), 0, st, a);              \
        return grid;                                                                              \
    } while (0)
    const int64_t bytes = a.V * (int64_t)sizeof(T);
    if (a.V <= 8) {
        // a lane per row.  Up to 1024 rows (a batch of 1024 over 5 actions) one workgroup takes them all and adds
        // its own loss up: one launch
        if (MODE == MODE_POLICY && a.rows <= 1024) {
            hipLaunchKernelGGL((row_lane_kernel<T, 1, 8, 1024, MODE>), dim3(1), dim3(1024), 0, st, a);
            return 1;
        }
        MCTSQ_ROWS(256, 256, row_lane_kernel<T, 1, 8, 256, MODE>);
    }
    if (a.V <= 32) MCTSQ_ROWS(256, 64, row_lane_kernel<T, 4, 8, 256, MODE>);
    if (a.V <= 256) MCTSQ_ROWS(256, 16, row_lane_kernel<T, 16, 16, 256, MODE>);
    // Measured (policy loss, 2 V bytes a bf16 row, 33 to 270 MB of logits; GB/s read + written): waves per row and vectors
    // per lane so that one row just fits keeps the most rows in flight -- V = 2040 RW 1 U 4 3900 (RW 2 2830), 8184 RW 2 U 8
    // 4780 (RW 4 3500), 16000 RW 4 U 8 5050 (RW 8 U 4 4340), 65000 RW 16 U 8 4660 (streamed 3880).  Between, 16-bit rows are
    // better streamed by 8 waves, as two held rows are all that fit a CU: calls of 67 MB of logits, streamed / held, 17000
    // 2960 / 2580, 20000 3110 / 2810, 24000 3440 / 3180, 28000 3510 / 3260, 32000 3550 / 3400; fp32 rows hold half as many
    // values per vector and have no such gap (32000: held 5220, streamed 4560).  131072 streamed by 16 waves 3840.
    // vectors of a row: at its worst alignment, unless every row starts on a vector
    const int64_t es = sizeof(T), starts = (int64_t)((uintptr_t)a.z & 15) | ((a.z_si | (a.one_group ? 0 : a.z_so)) * es & 15);
    const int64_t nv = (a.V + (starts ? 2 * Elem<T>::VE - 2 : Elem<T>::VE - 1)) / Elem<T>::VE;
    if (nv <= 64) MCTSQ_ROWS(256, 4, row_kernel<T, 1, 1, MODE == MODE_POLICY, MODE, ACC>);
    if (nv <= 128) MCTSQ_ROWS(256, 4, row_kernel<T, 1, 2, MODE == MODE_POLICY, MODE, ACC>);
    if constexpr (MODE == MODE_POLICY) {
        if (nv <= 256) MCTSQ_ROWS(256, 4, row_kernel<T, 1, 4, true, MODE, ACC>);
        if (nv <= 512) MCTSQ_ROWS(256, 4, row_kernel<T, 1, 8, true, MODE, ACC>);
        if (nv <= 1024) MCTSQ_ROWS(128, 1, row_kernel<T, 2, 8, true, MODE, ACC>);
        if (nv <= 2048) MCTSQ_ROWS(256, 1, row_kernel<T, 4, 8, true, MODE, ACC>);
        if (nv <= 4096) {
            if constexpr (sizeof(T) == 4) MCTSQ_ROWS(512, 1, row_kernel<T, 8, 8, true, MODE, ACC>);
            else MCTSQ_ROWS(512, 1, row_kernel<T, 8, 4, false, MODE, ACC>);
        }
        if (nv <= 8192) MCTSQ_ROWS(1024, 1, row_kernel<T, 16, 8, true, MODE, ACC>);
        MCTSQ_ROWS(1024, 1, row_kernel<T, 16, 4, false, MODE, ACC>);
    } else if constexpr (MODE == MODE_LOGP) {
        // one pass, few registers: a wave per row up to 16 KB, four above (32000 bf16: 4 waves 5190 GB/s, 16 waves 3480) --
        // unless there are too few rows to fill the chip that way, when the whole workgroup shortens each (64 rows of
        // 32000: 10.4 us against 15.7)
        if (a.rows * (bytes <= 16384 ? 1 : 4) < 2048 && nv > 256) MCTSQ_ROWS(1024, 1, row_kernel<T, 16, 4, false, MODE, ACC>);
        if (bytes <= 16384) MCTSQ_ROWS(256, 4, row_kernel<T, 1, 4, false, MODE, ACC>);
        MCTSQ_ROWS(256, 1, row_kernel<T, 4, 4, false, MODE, ACC>);
    } else {
        // statistics are known: a plain sweep
        if (bytes <= 8192) MCTSQ_ROWS(256, 4, row_kernel<T, 1, 4, false, MODE, ACC>);
        if (bytes <= 32768) MCTSQ_ROWS(128, 1, row_kernel<T, 2, 4, false, MODE, ACC>);
        MCTSQ_ROWS(512, 1, row_kernel<T, 8, 4, false, MODE, ACC>);
    }
#undef MCTSQ_ROWS
}

template <int MODE>
static int64_t launch_rows(int dtype, const RowArgs& a, hipStream_t st) {
    if (dtype == DT_F32) return launch_rows<float, MODE, MODE != MODE_GRAD>(a, st);
    if constexpr (MODE != MODE_GRAD)
        if (a.rows <= 256)
            return dtype == DT_BF16 ? launch_rows<__bf16, MODE, true>(a, st) : launch_rows<_Float16, MODE, true>(a, st);
    if (dtype == DT_BF16) return launch_rows<__bf16, MODE, false>(a, st);
    return launch_rows<_Float16, MODE, false>(a, st);
}

// shapes and strides every entry point shares; fills the logits part of `a`
static int fill_rows(RowArgs& a, const void* d_logits, int dtype, int64_t rows, int64_t inner, int64_t stride_outer,
                     int64_t stride_inner, int64_t vocab, const void* d_act, int act_bytes, const float* d_weight) {
    MCTSQ_CHECK(dtype >= 0 && dtype <= 2, "logits dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
    MCTSQ_CHECK(rows >= 0 && vocab >= 1 && inner >= 1, "rows must not be negative, vocab and inner at least 1");
    MCTSQ_CHECK(rows < ((int64_t)1 << 31) && vocab < ((int64_t)1 << 40), "at most 2^31 - 1 rows");
    MCTSQ_CHECK(rows % inner == 0, "rows must be a multiple of the inner extent");
    MCTSQ_CHECK(act_bytes == 4 || act_bytes == 8, "actions must be 4- or 8-byte integers");
    MCTSQ_CHECK(rows == 0 || (d_logits && d_act), "NULL device pointer");
    const int es = dtype == DT_F32 ? 4 : 2;
    MCTSQ_CHECK(((uintptr_t)d_logits & (es - 1)) == 0, "logits are not aligned to their element size");
    MCTSQ_CHECK((inner == 1 || stride_inner >= 0) && (rows == inner || stride_outer >= 0), "negative strides");
    a = RowArgs{};
    a.z = (const char*)d_logits; a.z_so = stride_outer; a.z_si = stride_inner;
    a.rows = rows; a.inner = inner; a.V = vocab;
    a.one_group = inner == rows;
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

// at most 2^58 rows: 20 bytes of workspace each and the sequences' own stay within 64 bits
static int check_pairs(int64_t pairs, int64_t tokens) {
    MCTSQ_CHECK(pairs >= 0 && tokens >= 0 && pairs <= ((int64_t)1 << 30) && tokens <= ((int64_t)1 << 31)
                && 2 * pairs * tokens <= ((int64_t)1 << 58), "pairs / tokens out of range");
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
    off[5] = take((seqs / 2 + PAIRS - 1) / PAIRS * 8);      // loss_part
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
        a.logp = d_logp; a.kl = d_kl; a.loss_part = (double*)d_ws; a.loss = d_loss;
        parts = launch_rows<MODE_POLICY>(dtype, a, st);
    }
    if (parts != 1) hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, st, (const double*)d_ws, parts, d_loss);
    MCTSQ_HIP(hipGetLastError());
    return 0;
}

extern "C" int64_t mctsq_preference_loss_workspace_bytes(int64_t pairs, int64_t tokens) {
    if (int rc = check_pairs(pairs, tokens)) return rc;
    int64_t off[6];
    return pref_ws(2 * pairs, tokens, off);
}

extern "C" int mctsq_preference_loss(const void* d_logits, int dtype, int64_t pairs, int64_t tokens, int64_t stride_outer,
                                     int64_t stride_inner, int64_t vocab, const void* d_act, int act_bytes,
                                     const float* d_ref_logp, const float* d_weight, const float* d_pair_weight,
                                     double beta, double label_smoothing, double loss_scale, float* d_loss,
                                     float* d_seq_logp, float* d_margin, void* d_dlogits, int64_t dstride_outer,
                                     int64_t dstride_inner, void* d_ws, int64_t ws_bytes, void* stream) {
    if (int rc = check_pairs(pairs, tokens)) return rc;
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
    if (rows > 0 && d_dlogits) { if (int rc = fill_grad(a, d_dlogits, dtype, dstride_outer, dstride_inner)) return rc; }
    a.seq_coef = (float*)(ws + off[4]);
    PairArgs p{};
    p.logp64 = a.logp64; p.w = d_weight; p.ref = d_ref_logp; p.pair_w = d_pair_weight; p.P = pairs; p.T = tokens;
    p.beta = beta; p.smooth = label_smoothing; p.scale = loss_scale;
    p.seq_logp = d_seq_logp; p.margin = d_margin; p.seq_coef = (float*)(ws + off[4]); p.loss_part = (double*)(ws + off[5]); p.loss = d_loss;
    // The gradient reads the logits again, from memory where they are larger than the caches (8 pairs of 102 MB: 398 us at
    // 5.15 TB/s for two readings and one writing would be 359; pairs sent through in groups of 32 to 224 MB so that the
    // second reading could find them cached took 485 to 529).
    if (rows > 0) {
        RowArgs f = a;
        f.dz = nullptr;
        launch_rows<MODE_LOGP>(dtype, f, st);
    }
    const int64_t pg = pairs > 0 ? (pairs + PAIRS - 1) / PAIRS : 1;        // no pairs: the launch writes loss 0
    hipLaunchKernelGGL(pair_kernel, dim3((unsigned)pg), dim3(1024), 0, st, p);
    if (rows > 0 && d_dlogits) launch_rows<MODE_GRAD>(dtype, a, st);
    if (pg > 1) hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, st, (const double*)p.loss_part, pg, d_loss);
    MCTSQ_HIP(hipGetLastError());
    return 0;
}
