// AdamW over many tensors at once, with moments in float32 or in 8 bits, and the global gradient norm that clips them.
//
//   norm = sqrt(sum g^2) over all tensors,  f = min(1, max_norm / (norm + 1e-6))       (f = 1 without clipping)
//   m <- b1 m + (1 - b1) f g,   v <- b2 v + (1 - b2) (f g)^2
//   p <- (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Every element is read and written once (28 bytes for float32 throughout), so the step is bound by memory: 240M float32 weights
// 1.07 ms (6.3 TB/s; a plain copy kernel runs at 6.5), clipped 1.20 ms with the gradient read twice.  The tensors
// are cut into chunks of 1024 or 2048 elements; a table that the caller keeps on the device says which tensor a chunk lies in, so
// one launch covers up to kMaxTensors tensors of any sizes; their addresses travel in the launch's arguments, because
// gradients move from step to step.  Moments and master weights are flat buffers in which each tensor starts at a multiple of kBlock.
//
// 8-bit moments: a block of kBlock = 128 elements shares one scale 2^(s - 127) (a byte; 255 = the block is not finite), and
// an element is one byte: m as sign + 4 bits of exponent + 3 of mantissa, v (never negative) as 5 bits of exponent + 3 of mantissa.
// Scales are powers of two, so decoding and scaling are exact and the only rounding is the one to the byte.  It rounds up
// with probability equal to the remainder, by a sequence over steps and elements that covers [0, 1) evenly:
// with b2 = 0.999 a moment changes by less than half a code per step, and rounding to nearest would freeze it.
// The arithmetic is float64, whose products, sums and conversions issue as fast as integer operations here (4.4 to 5.4 cycles a
// wave; float32 additions 2.8): the top 20 bits of a double's mantissa hold the 3 bits of the code and 17 bits of remainder, so
// rounding is one integer addition on the double's upper word, and it is exact - the codes do not depend on how a compiler
// contracts a float32 expression.  60M float32 weights 171 us (16 bytes each, 5.6 TB/s), 240M bfloat16 weights 440 us (10 bytes, 5.5 TB/s:
// 56 vector instructions an element, 383 us of issue, no longer hide under 370 us of memory).
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "../../include/pinnjet.h"

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = PINN_ADAMW_BLOCK;        // elements that share a scale; also the layout's alignment
constexpr int kChunk32 = PINN_ADAMW_CHUNK32, kChunk8 = PINN_ADAMW_CHUNK8;   // elements a workgroup takes at a time
constexpr int kMaxTensors = PINN_ADAMW_MAX_TENSORS;
// Bytes of LDS that a step's workgroups ask for and do not use: 6 or 5 of them fit on a CU instead of 8.  More streams of reads and writes
// at once cost memory bandwidth.  float32 moments, 240M float32 weights (28 bytes each): 8 workgroups of 2048 elements 1186 us, 5 of them 1138,
// 5 of 1024 elements 1099, 6 of 1024 elements 1082 (6.2 TB/s), 3 of 1024 elements 1394.  8-bit moments, 240M float32 weights (16 bytes): free 673 us, 5 workgroups 653.
constexpr unsigned kPace32 = 27000, kPace8 = 32000;
constexpr int kNormTensors = PINN_NORM_TENSORS;
constexpr int kNormChunk = 8192;
constexpr int kMaxPartials = PINN_NORM_PARTIALS;
static_assert(sizeof(PinnAdamWChunk) == 32 && sizeof(PinnAdamWGroup) == 168, "the callers' layouts");
static_assert(kChunk32 == 4 * kThreads && kChunk8 == 8 * kThreads && kChunk32 % kBlock == 0, "a thread takes 4 or 8 elements of a chunk");

// N elements at any address that an element may have: the accesses stay wide, the hardware takes them unaligned.  Everything
// here is touched once per step: the non-temporal forms keep it from displacing what is used again (240M float32 weights, step with
// clipping, before the later changes: 1.60 ms plain, 1.53 ms with both; loads or stores alone 1.63, 1.60).
template <class T, int N>
using Vec = T __attribute__((ext_vector_type(N)));

template <int N, class T>
__device__ inline Vec<T, N> load(const T *p)
{
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    return __builtin_nontemporal_load((const V *)p);
}

template <int N, class T>
__device__ inline void store(T *p, Vec<T, N> x)
{
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    __builtin_nontemporal_store((V)x, (V *)p);
}

// the first `have` of N elements and zeros behind them; FULL: all are there
template <bool FULL, int N, class T>
__device__ inline Vec<T, N> load_some(const T *p, int have)
{
    if (FULL || have >= N) return load<N>(p);
    Vec<T, N> x = (T)0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < have) x[e] = p[e];
    return x;
}

template <bool FULL, int N, class T>
__device__ inline void store_some(T *p, Vec<T, N> x, int have)
{
    if (FULL || have >= N) return store<N>(p, x);
#pragma unroll
    for (int e = 0; e < N; ++e)
        if (e < have) p[e] = x[e];
}

// float32 rounded once to T.  The empty asm keeps the compiler from folding the conversion into what comes before it
// (v_fma_mixlo_f16 rounds the unrounded sum, and float64 by way of float32 becomes one conversion): a 16-bit weight is its
// float32 master's rounding, bit for bit.
template <class T>
__device__ inline T rounded(float x)
{
    if constexpr (!__is_same(T, float)) asm("" : "+v"(x));
    return (T)x;
}

struct StepArgs {
    void *p[kMaxTensors];
    const void *g[kMaxTensors];                 // null: no gradient, the tensor is left alone
};
typedef const __attribute__((address_space(4))) PinnAdamWChunk ConstChunk;   // read-only while the kernel runs: scalar loads
struct StepConst {
    const PinnAdamWChunk *chunks;
    const int32_t *rows;
    uint8_t *m, *v, *sm, *sv;                   // m, v: float32 or codes; sm, sv: scales
    float *master;
    double *state;                              // [tensor][3]: step, b1^t, b2^t
    uint32_t *ticket;
    const double *partials;
    float *norm_out;
    int64_t n_chunks;
    int32_t n_tensors, n_partials, skip_nonfinite, run;
    double max_norm, b1, b2, lr, eps, decay;
    float eps32, decay32;
};
static_assert(sizeof(StepArgs) + sizeof(StepConst) <= 4096, "a launch's arguments");

// The sum of the partial sums, in an order that depends on their number alone: every workgroup gets the same bits.
__device__ double sum_partials(const double *partials, int n)
{
    __shared__ double part[kThreads / 64];
    if (n == 1) return partials[0];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) s += partials[i];
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
    for (int w = 0; w < kThreads / 64; ++w) s += part[w];
    return s;
}

__device__ inline double clip_factor(double norm, double max_norm)
{
    const double f = max_norm / (norm + 1e-6);
    return f > 1.0 ? 1.0 : f;                   // NaN stays NaN, as min(1, NaN) would not
}

// The factor for float32 products, x * pre * f.  A norm is a float64 and may pass float32's largest value, and a factor below 2^-126
// would lose its digits: it is brought near 1 and x made smaller, which is exact for every x whose product is not itself below 2^-126.
// In a branch that no training takes: computed without one it costs 240M clipped float32 weights 8 us of 1205.
struct Factor {
    float pre = 1.0f, f;
    __device__ explicit Factor(double factor)
    {
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(factor < 0x1p-100), 0)) {
            const int down = 1023 - (__double2hiint(factor) >> 20), k = down < 140 ? down : 140;
            pre = ldexpf(1.0f, -k);
            factor = ldexp(factor, k);
        }
        f = (float)factor;
    }
    __device__ float operator*(float x) const { return x * pre * f; }
};

// ---- float32 moments -------------------------------------------------------------------------------------------
template <class F>
struct Scalars {
    F step_size, inv_bc2_sqrt;                  // float for float32 moments, double for 8 bits
    double p1, p2;
    uint32_t t;
};

// v_rcp_f64 and v_rsq_f64 are good to 2^-23 at least; one Newton step gives them twice the digits.  A full division and root
// are 60 instructions, which a workgroup of 2048 elements feels.
__device__ inline double reciprocal(double x)
{
    const double r = __builtin_amdgcn_rcp(x);
    return fma(r, fma(-x, r, 1.0), r);
}

__device__ inline double reciprocal_root(double x)
{
    const double r = __builtin_amdgcn_rsq(x);
    return fma(0.5 * r, fma(-x * r, r, 1.0), r);
}

template <class F>
__device__ inline Scalars<F> scalars_of(const double *row, double b1, double b2, double lr)
{
    Scalars<F> s;
    s.t = (uint32_t)(row[0] + 1.0);
    s.p1 = row[1] * b1;
    s.p2 = row[2] * b2;
    s.step_size = (F)(lr * reciprocal(1.0 - s.p1));
    s.inv_bc2_sqrt = (F)reciprocal_root(1.0 - s.p2);
    return s;
}

struct Hyper32 {
    float b2, omb1, omb2, eps, decay;
    Factor factor;
};

__device__ inline void update32(float &p, float g, float &m, float &v, const Scalars<float> &s, const Hyper32 &h)
{
    g = h.factor * g;
    p *= h.decay;
    m = fmaf(g - m, h.omb1, m);
    v = fmaf(h.omb2 * g, g, v * h.b2);
    const float denom = sqrtf(v) * s.inv_bc2_sqrt + h.eps;
    p = fmaf(-s.step_size, m / denom, p);
}

// Where a chunk's data lie.
template <class T>
struct At {
    T *p;
    const T *g;                                 // null: no gradient, nothing to do
    uint8_t *m, *v, *sm, *sv;
    float *master;
    uint32_t place;
    int count;
    const double *row;
};

template <bool FULL, bool MASTER, class T>
__device__ inline void chunk(const At<T> &at, const Scalars<float> &s, const Hyper32 &h)
{
    constexpr int N = 4;
    float *am = (float *)at.m, *av = (float *)at.v;
    const int i = (int)threadIdx.x * N, have = at.count - i;
    if (!FULL && have <= 0) return;
    const Vec<T, N> g = load_some<FULL, N>(at.g + i, have);
    Vec<T, N> p;
    Vec<float, N> w, m, v;
    if constexpr (MASTER) w = load_some<FULL, N>(at.master + i, have);
    else p = load_some<FULL, N>(at.p + i, have);
    m = load_some<FULL, N>(am + i, have);
    v = load_some<FULL, N>(av + i, have);
#pragma unroll
    for (int e = 0; e < N; ++e) {
        float we = MASTER ? w[e] : (float)p[e], me = m[e], ve = v[e];
        update32(we, (float)g[e], me, ve, s, h);
        w[e] = we;
        m[e] = me;
        v[e] = ve;
        p[e] = rounded<T>(we);
    }
    store_some<FULL, N>(at.p + i, p, have);
    if constexpr (MASTER) store_some<FULL, N>(at.master + i, w, have);
    store_some<FULL, N>(am + i, m, have);
    store_some<FULL, N>(av + i, v, have);
}

// ---- 8-bit moments ---------------------------------------------------------------------------------------------
struct Format {
    int shift;        // the smallest normal code's exponent against float64's (2^-1022): value * 2^-shift puts the code on top of the upper word
    int shift32;      // the same against float32's 2^-126, for decoding
    int top;          // exponent of the largest code's magnitude, 1.75 * 2^top
    int most_scale;   // largest scale byte: the largest code stays finite in float32
    uint32_t most_code;
};
constexpr Format kM = {1016, 120, 8, 246, 126u};
constexpr Format kV = {1008, 112, 16, 238, 254u};

__device__ inline double pow2(int e)            // 2^e, e within float64's normal range
{
    return __hiloint2double((e + 1023) << 20, 0);
}

__device__ inline uint32_t row_max(uint32_t x)  // the largest over the 16 lanes of a DPP row, in all of them
{
#define PINN_ROR(N) { const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + N, 0xf, 0xf, false); x = y > x ? y : x; }
    PINN_ROR(8) PINN_ROR(4) PINN_ROR(2) PINN_ROR(1)
#undef PINN_ROR
    return x;
}

// scale byte of a block whose largest magnitude has the upper word `hi` (sign off): the largest code's mantissa is 1.75,
// so a mantissa of 1.75 or more takes the next power of two and rounding up can never pass the largest code
__device__ inline int scale_of(uint32_t hi, const Format &f)
{
    if (hi >= 0x7ff00000u) return 255;
    const int s = (int)((hi + 0x40000u) >> 20) - 1023 - f.top + 127;
    return s < 0 ? 0 : s > f.most_scale ? f.most_scale : s;
}

// x's magnitude as a code before it is held to the largest: 3 mantissa bits and what the remainder adds to them.  `near` collects how far
// the sum's lower 17 bits came.
__device__ inline uint32_t code_of(double x, int exponent, uint32_t w, uint32_t &near)
{
    const uint32_t t = (uint32_t)__double2hiint(ldexp(fabs(x), exponent)) + (w >> 15 | 1u);
    near = t << 15 > near ? t << 15 : near;
    return t >> 17;
}

// The place y on the codes' scale (8 times the exponent field plus 8 times the fraction) is a float64 too, and the larger it is the fewer
// of x's last bits it has.  An x so near below a multiple of 2^-17 codes that y is rounded up to it takes that value.  It only
// matters where the sum lacks one to the next code (all 17 bits are set): about one wave in 130 looks.
__device__ inline double settled(double x, int exponent)
{
    const uint32_t hi = (uint32_t)__double2hiint(x), lo = (uint32_t)__double2loint(x);
    const int field = (int)((hi & 0x7fffffffu) >> 20) + exponent;
    const uint32_t half = field >= 16 ? 8u : field >= 8 ? 4u : field >= 4 ? 2u : field >= 2 ? 1u : 0u;   // half a unit of y's last place, in x's
    return half && lo >= 0u - half ? __hiloint2double((int)(hi + 1), 0) : x;
}

// the sequences that round: golden ratio, sqrt(2) over the elements; the two-dimensional analogue of the golden ratio over the steps
constexpr uint32_t kPlaceM = 0x9E3779B9u, kStepM = 0xC13FA9A9u, kPlaceV = 0x6A09E667u, kStepV = 0x91E10DA5u;

struct Hyper8 {
    double b1, b2, g1, g2;                      // g1 = (1 - b1) f, g2 = (1 - b2) f^2
    double eps, decay;
};

// a b + c d with each operation rounded by itself.  Codes are compared with where the remainder lies, and (9 m + g) / 10 lies on such a
// border more often than chance: m has 4 bits and g 24.  Which way 0.9 m + 0.1 g falls there is a matter of float64's last
// bit, so the order of rounding is fixed: with fma, one or two codes in 5M differ from what the formula gives step by step.
__device__ inline double product_sum(double a, double b, double c, double d)
{
#pragma clang fp contract(off)
    const double x = a * b, y = c * d;
    return x + y;
}

// A lane's 8 elements of a block: two runs of 4, APART elements from each other.  16-bit weights without masters: one run of 8
// (16 bytes).  With float32 among them the runs are half a block apart, so that 16 lanes read 256 bytes in a row and not every
// other 16 (240M float32 weights: 652 us, with one run of 8 766).
template <bool FULL, int APART, class T>
__device__ inline Vec<T, 8> load_runs(const T *p, int have)
{
    if constexpr (APART == 4) return load_some<FULL, 8>(p, have);
    const Vec<T, 4> a = load_some<FULL, 4>(p, have), b = load_some<FULL, 4>(p + APART, have - APART);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

template <bool FULL, int APART, class T>
__device__ inline void store_runs(T *p, Vec<T, 8> x, int have)
{
    if constexpr (APART == 4) return store_some<FULL, 8>(p, x, have);
    store_some<FULL, 4>(p, __builtin_shufflevector(x, x, 0, 1, 2, 3), have);
    store_some<FULL, 4>(p + APART, __builtin_shufflevector(x, x, 4, 5, 6, 7), have - APART);
}

template <bool FULL, bool MASTER, class T>
__device__ inline void chunk(const At<T> &at, const Scalars<double> &s, const Hyper8 &h)
{
    constexpr int N = 8, APART = sizeof(T) == 4 || MASTER ? kBlock / 2 : 4;
    const int lane = (int)threadIdx.x & 15, blk = (int)threadIdx.x >> 4;    // a block is 16 lanes, a DPP row
    const int i = blk * kBlock + lane * (APART == 4 ? 8 : 4), have = at.count - i;
    if (!FULL && blk * kBlock >= at.count) return;     // rows behind the tensor's end leave together
    Vec<uint32_t, 2> cm, cv;
    if constexpr (APART == 4) {
        cm = load<2>((const uint32_t *)(at.m + i));
        cv = load<2>((const uint32_t *)(at.v + i));
    } else {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            cm[r] = load<1>((const uint32_t *)(at.m + i + r * APART))[0];
            cv[r] = load<1>((const uint32_t *)(at.v + i + r * APART))[0];
        }
    }
    const int s0m = at.sm[blk], s0v = at.sv[blk];
    const Vec<T, N> g = load_runs<FULL, APART>(at.g + i, have);
    Vec<T, N> p;
    Vec<float, N> w;
    if constexpr (MASTER) w = load_runs<FULL, APART>(at.master + i, have);
    else p = load_runs<FULL, APART>(at.p + i, have);
    double um = h.b1 * pow2(s0m - 127), uv = h.b2 * pow2(s0v - 127 + kV.shift32);
    if (s0m == 255) um = __hiloint2double(0x7ff80000, 0);
    if (s0v == 255) uv = __hiloint2double(0x7ff80000, 0);
    asm("" : "+v"(um), "+v"(uv));               // or the compiler makes the NaN a choice behind every product
    // both terms of the denominator over the step size: the update is one product
    const double per_step = s.step_size == 0.0 ? 1e300 : reciprocal(s.step_size), root = s.inv_bc2_sqrt * per_step, eps = h.eps * per_step;
    const float decay32 = (float)h.decay;
    double md[N], vd[N];
    uint32_t hm = 0, hv = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        // m's codes are the hardware's 8-bit floats (OCP E4M3; its NaN, 127, is never written)
        const int pair = (int)cm[e / 4];
        const float fm = (e & 2 ? __builtin_amdgcn_cvt_pk_f32_fp8(pair, true) : __builtin_amdgcn_cvt_pk_f32_fp8(pair, false))[e & 1];
        const float fv = __uint_as_float((e & 3) == 3 ? cv[e / 4] >> 4 & 0x0ff00000u : cv[e / 4] << (20 - 8 * (e & 3)) & 0x0ff00000u);
        const double gd = (double)(float)g[e];
        md[e] = product_sum((double)fm, um, h.g1, gd);
        vd[e] = product_sum((double)fv, uv, h.g2 * gd, gd);
        const uint32_t am = (uint32_t)__double2hiint(md[e]) & 0x7fffffffu, av = (uint32_t)__double2hiint(vd[e]);
        hm = am > hm ? am : hm;
        hv = av > hv ? av : hv;
        // The denominator may be anything that a root of g^2 is: in float32 v_rcp_f32 gives 0 for the largest and infinity for
        // subnormals.  v_sqrt_f64 and v_rcp_f64 are good to 2^-23 of the update at least, which does not show beside the weight's own
        // rounding.  float32 weights and masters are rounded once, from float64.  A 16-bit weight's rounding is 2^13 times as coarse
        // or more and hides the two of float32 (240M bfloat16 weights, the step with its read-out: 840 us, in float64 to the end 892).
        const double update = md[e] * __builtin_amdgcn_rcp(fma(__builtin_amdgcn_sqrt(vd[e]), root, eps));
        float we;
        if constexpr (sizeof(T) == 4 || MASTER) we = (float)fma((double)(MASTER ? w[e] : (float)p[e]), h.decay, -update);
        else we = fmaf((float)p[e], decay32, (float)-update);
        w[e] = we;
        p[e] = rounded<T>(we);
    }
    store_runs<FULL, APART>(at.p + i, p, have);
    if constexpr (MASTER) store_runs<FULL, APART>(at.master + i, w, have);
    const int s1m = scale_of(row_max(hm), kM), s1v = scale_of(row_max(hv), kV);
    const int xm = 127 - s1m - kM.shift, xv = 127 - s1v - kV.shift;
    const uint32_t place = at.place + i;
    uint32_t w0m = place * kPlaceM + s.t * kStepM, w0v = place * kPlaceV + s.t * kStepV;
    Vec<uint32_t, 2> om, ov;
    // behind the tensor's end gradients and codes are zero, and so are the codes that come out
#pragma unroll 1
    for (bool again = false;;) {
        asm("" : "+v"(w0m), "+v"(w0v));         // or all 16 of the sums below are made before the loop, which would take registers that are not there
        uint32_t near = 0;
        om = 0;
        ov = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint32_t off = e < 4 ? e : APART + e - 4;
            uint32_t a = code_of(md[e], xm, w0m + off * kPlaceM, near), b = code_of(vd[e], xv, w0v + off * kPlaceV, near);
            a = a > kM.most_code ? kM.most_code : a;
            a |= (uint32_t)__double2hiint(md[e]) >> 24 & 128u;
            // 1 where v is not zero (written out: as a comparison it takes twice the instructions): a v that vanished under a live m would divide it by eps alone
            uint32_t live;
            asm("v_min_u32 %0, 1, %1" : "=v"(live) : "v"(__double2hiint(vd[e])));
            asm("v_med3_u32 %0, %1, %2, %3" : "=v"(b) : "v"(b), "v"(live), "s"(kV.most_code));
            om[e / 4] |= a << (8 * (e & 3));
            ov[e / 4] |= b << (8 * (e & 3));
        }
        if (__builtin_expect(again || near < 0xffff8000u, 1)) break;
        again = true;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            md[e] = settled(md[e], xm);
            vd[e] = settled(vd[e], xv);
        }
    }
    if (s1m == 255) om = 0;
    if (s1v == 255) ov = 0;
    if constexpr (APART == 4) {
        store<2>((uint32_t *)(at.m + i), om);
        store<2>((uint32_t *)(at.v + i), ov);
    } else {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            store<1>((uint32_t *)(at.m + i + r * APART), Vec<uint32_t, 1>(om[r]));
            store<1>((uint32_t *)(at.v + i + r * APART), Vec<uint32_t, 1>(ov[r]));
        }
    }
    if (lane == 0) {
        at.sm[blk] = (uint8_t)s1m;
        at.sv[blk] = (uint8_t)s1v;
    }
}

constexpr unsigned kTickets = 64, kTicketStride = 32;
static_assert((kTickets + 1) * kTicketStride == PINN_ADAMW_TICKET_WORDS, "the callers' buffer");

__device__ inline uint32_t draw(uint32_t *word)
{
    return __hip_atomic_fetch_add(word, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ inline void put_back(uint32_t *word)
{
    __hip_atomic_store(word, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <class T>
__device__ inline At<T> locate(const StepArgs &a, const StepConst &c, int64_t ch, int bits)
{
    ConstChunk &r = ((ConstChunk *)(uintptr_t)c.chunks)[ch];
    const int64_t base = r.base, place = r.place;
    const int k = r.tensor;
    const int bytes = bits == 32 ? 4 : 1;
    At<T> at;
    at.g = (const T *)a.g[k] ? (const T *)a.g[k] + base : nullptr;
    at.p = (T *)a.p[k] + base;
    at.m = c.m + place * bytes;
    at.v = c.v + place * bytes;
    at.sm = c.sm + place / kBlock;
    at.sv = c.sv + place / kBlock;
    at.master = c.master + place;
    at.place = (uint32_t)place;
    at.count = r.count;
    at.row = c.state + 3 * (int64_t)r.row;
    return at;
}

// Workgroup b takes the chunks b * run .. b * run + run - 1.
template <class T, bool MASTER, int BITS>
__global__ __launch_bounds__(kThreads, BITS == 32 ? 6 : 5) void k_adamw_group(const StepArgs a, const StepConst c)
{
    double factor = 1.0;
    if (c.n_partials) {
        const double norm = sqrt(sum_partials(c.partials, c.n_partials));
        if (c.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *c.norm_out = (float)norm;
        if (c.skip_nonfinite && !((float)norm < __uint_as_float(0x7f800000u))) return;   // as it is reported; in all workgroups alike: nothing is written, the tickets stay
        if (c.max_norm >= 0.0) factor = clip_factor(norm, c.max_norm);
    }
    const Hyper32 h32 = {(float)c.b2, (float)(1.0 - c.b1), (float)(1.0 - c.b2), c.eps32, c.decay32, Factor(factor)};
    const Hyper8 h8 = {c.b1, c.b2, (1.0 - c.b1) * factor, (1.0 - c.b2) * factor * factor, c.eps, c.decay};
    typedef std::conditional_t<BITS == 32, float, double> F;
    Scalars<F> s;
    const double *row = nullptr;
    const int64_t first = (int64_t)blockIdx.x * c.run, end = first + c.run < c.n_chunks ? first + c.run : c.n_chunks;
    for (int64_t ch = first; ch < end; ++ch) {
        const At<T> at = locate<T>(a, c, ch, BITS);
        if (!at.g) continue;
        if (at.row != row) s = scalars_of<F>(at.row, c.b1, c.b2, c.lr);
        row = at.row;
        if constexpr (BITS == 32) {
            if (at.count == kChunk32) chunk<true, MASTER>(at, s, h32);
            else chunk<false, MASTER>(at, s, h32);
        } else {
            if (at.count == kChunk8) chunk<true, MASTER>(at, s, h8);
            else chunk<false, MASTER>(at, s, h8);
        }
    }
    // The workgroup that finishes last advances the counters: every other one has used what it read of them by then.  Nothing
    // else passes between workgroups, so the tickets need no fence (a device-wide one writes the caches back, once per workgroup).
    // Atomics on one word take 11 ns each, one after the other (2048 of them 23 us, a third of a step of 5M weights): a
    // workgroup of a large grid draws from one of kTickets words on lines of their own, and the last of those draws from the first word.
    __shared__ bool last_of_all;
    __syncthreads();
    if (threadIdx.x == 0) {
        if (gridDim.x <= kTickets) {
            last_of_all = draw(c.ticket) == gridDim.x - 1;
        } else {
            const unsigned j = blockIdx.x % kTickets;
            uint32_t *mine = c.ticket + (1 + j) * kTicketStride;
            last_of_all = false;
            if (draw(mine) == (gridDim.x - j + kTickets - 1) / kTickets - 1) {
                put_back(mine);
                last_of_all = draw(c.ticket) == kTickets - 1;
            }
        }
        if (last_of_all) put_back(c.ticket);
    }
    __syncthreads();
    if (!last_of_all) return;
    for (int k = threadIdx.x; k < c.n_tensors; k += kThreads)
        if (a.g[k]) {
            double *row = c.state + 3 * (int64_t)c.rows[k];
            const Scalars<F> n = scalars_of<F>(row, c.b1, c.b2, c.lr);
            row[0] += 1.0;
            row[1] = n.p1;
            row[2] = n.p2;
        }
}

// Moments as float32: what the codes stand for.  One workgroup for 1024 elements, in order: 240M elements 384 us (10 bytes each, 6.25
// TB/s); 8192 workgroups in a loop 486 us.  A launch holds fewer than 2^32 threads.
constexpr int64_t kMomentsLaunch = (int64_t)1 << 33;
static_assert(kMomentsLaunch / 4 < (int64_t)1 << 32 && kMomentsLaunch % kBlock == 0, "threads of a launch; scales begin with it");
__global__ __launch_bounds__(kThreads) void k_moments(const uint8_t *m, const uint8_t *v, const uint8_t *sm, const uint8_t *sv, float *mo,
                                                            float *vo, int64_t n)
{
    const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4;
    if (i >= n) return;
    const uint32_t cm = load<1>((const uint32_t *)(m + i))[0], cv = load<1>((const uint32_t *)(v + i))[0];
    const int s0m = sm[i / kBlock], s0v = sv[i / kBlock];
    Vec<float, 4> x, y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t a = cm >> (8 * e) & 255u, b = cv >> (8 * e) & 255u;
        x[e] = ldexpf(__uint_as_float((a & 127u) << 20 | (a & 128u) << 24), s0m - 127 + kM.shift32);
        y[e] = ldexpf(__uint_as_float(b << 20), s0v - 127 + kV.shift32);
        if (s0m == 255) x[e] = __uint_as_float(0x7fc00000u);
        if (s0v == 255) y[e] = __uint_as_float(0x7fc00000u);
    }
    store<4>(mo + i, x);
    store<4>(vo + i, y);
}

// ---- the global norm -------------------------------------------------------------------------------------------
// Squares are summed in float64: no gradient that float32 can hold overflows or vanishes there, so no pass looks for a scale first.
// Workgroup b always takes the same chunks and its sum has its own place, so the norm is the same bits on every run.  The workgroups
// sweep the tensors together, 8192 elements each at a time with all loads of a chunk under way: 240M float32 elements 143 us (6.7 TB/s);
// each in a region of its own 176 us, chunks of 4096 152 us, of 2048 199 us.
// Whole words only: from an index into bytes the compiler may make a scalar load whose base and offset are each unaligned (base + k, offset
// 7 k for word pair k), and scalar loads drop the lowest two bits of each by itself.
struct NormArgs {
    void *x[kNormTensors];
    int32_t first_chunk[kNormTensors + 1];
    uint32_t kind[kNormTensors];                // elements of a tensor's last chunk, 1 .. kNormChunk, and its type above 16 bits
    int32_t n_tensors, first_partial;
    __host__ __device__ int tail(int k) const { return (int)(kind[k] & 0xffffu); }
    __host__ __device__ int dtype(int k) const { return (int)(kind[k] >> 16); }
};
static_assert(sizeof(NormArgs) + 48 <= 4096, "a launch's arguments");

__device__ inline int find_tensor(const NormArgs &a, int64_t ch)
{
    int lo = 0, hi = a.n_tensors;               // the last tensor whose first chunk is at or before ch
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.first_chunk[mid] <= ch) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <class T, int N>
__device__ inline void add_squares(double &s, Vec<T, N> x)
{
#pragma unroll
    for (int e = 0; e < N; ++e) s = fma((double)(float)x[e], (double)(float)x[e], s);
}

template <class T>
__device__ inline double chunk_sumsq(const T *x, int count)
{
    constexpr int N = 16 / sizeof(T), J = kNormChunk / (N * kThreads);
    double s = 0.0;
    if (count == kNormChunk) {
        Vec<T, N> t[J];                         // all loads of the chunk are under way before the first sum
#pragma unroll
        for (int j = 0; j < J; ++j) t[j] = load<N>(x + (j * kThreads + threadIdx.x) * N);
#pragma unroll
        for (int j = 0; j < J; ++j) add_squares<T, N>(s, t[j]);
    } else {
        for (int i = threadIdx.x * N; i + N <= count; i += kThreads * N) add_squares<T, N>(s, load<N>(x + i));
        const int i = count / N * N + (int)threadIdx.x;
        if (i < count) s = fma((double)(float)x[i], (double)(float)x[i], s);
    }
    return s;
}

__global__ __launch_bounds__(kThreads) void k_grad_sumsq(const NormArgs a, double *partials)
{
    double s = 0.0;
    const int64_t n_chunks = a.first_chunk[a.n_tensors];
    for (int64_t ch = blockIdx.x; ch < n_chunks; ch += gridDim.x) {
        const int k = find_tensor(a, ch);
        const int64_t base = (ch - a.first_chunk[k]) * kNormChunk;
        const int count = ch + 1 == a.first_chunk[k + 1] ? a.tail(k) : kNormChunk;
        if (a.dtype(k) == PINN_F32) s += chunk_sumsq((const float *)a.x[k] + base, count);
        else if (a.dtype(k) == PINN_BF16) s += chunk_sumsq((const __bf16 *)a.x[k] + base, count);
        else s += chunk_sumsq((const _Float16 *)a.x[k] + base, count);
    }
    __shared__ double part[kThreads / 64];
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < kThreads / 64; ++w) s += part[w];
        partials[a.first_partial + blockIdx.x] = s;
    }
}

__global__ __launch_bounds__(kThreads) void k_fold(double *partials, int n)
{
    const double s = sum_partials(partials, n);     // read by all before the barrier in there
    if (threadIdx.x == 0) partials[0] = s;
}

__global__ __launch_bounds__(kThreads) void k_norm_of(const double *partials, int n, float *norm)
{
    const double s = sum_partials(partials, n);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

template <class T>
__device__ inline void chunk_scale(T *x, int count, Factor f)
{
    constexpr int N = 16 / sizeof(T);
#pragma unroll 4
    for (int i = threadIdx.x * N; i + N <= count; i += kThreads * N) {
        Vec<T, N> t = load<N>(x + i);
#pragma unroll
        for (int e = 0; e < N; ++e) t[e] = (T)(f * (float)t[e]);
        store<N>(x + i, t);
    }
    const int i = count / N * N + (int)threadIdx.x;
    if (i < count) x[i] = (T)(f * (float)x[i]);
}

// 240M float32 elements, norm and scaling: 478 us (2.88 GB, 6.0 TB/s); where the norm is small enough nothing is scaled: 143 us.  The
// workgroups of the sums take the chunks in turn: one for each chunk scales 240M bfloat16 elements in 170 us instead of 181 (float32 336
// and 365), but where nothing is to be scaled, which only the kernel knows, they take 26 us to start and leave, not 4.6.
__global__ __launch_bounds__(kThreads) void k_grad_clip(const NormArgs a, const double *partials, int n_partials, double max_norm, float *norm_out)
{
    const double norm = sqrt(sum_partials(partials, n_partials));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const Factor f(clip_factor(norm, max_norm));
    if (f.f == 1.0f && f.pre == 1.0f) return;   // the gradients stay as they are: nothing to write
    const int64_t n_chunks = a.first_chunk[a.n_tensors];
    for (int64_t ch = blockIdx.x; ch < n_chunks; ch += gridDim.x) {
        const int k = find_tensor(a, ch);
        const int64_t base = (ch - a.first_chunk[k]) * kNormChunk;
        const int count = ch + 1 == a.first_chunk[k + 1] ? a.tail(k) : kNormChunk;
        if (a.dtype(k) == PINN_F32) chunk_scale((float *)a.x[k] + base, count, f);
        else if (a.dtype(k) == PINN_BF16) chunk_scale((__bf16 *)a.x[k] + base, count, f);
        else chunk_scale((_Float16 *)a.x[k] + base, count, f);
    }
}

// Few elements: ONE workgroup forms the norm and, with max_norm >= 0, scales.  A launch is 3.7 us at the host, so for a small net the second one
// is a quarter of the call (10 tensors: clipping 10.4 us, in two launches 13.2).  The tensors are cut into runs of 256 elements, which the 16
// waves take in turn: up to 32768 elements the kernel hides behind the host's next call, with 65536 a call takes 17.6 us, with 131072 31.7.
constexpr int kSmallThreads = 1024, kSmallTensors = PINN_NORM_SMALL_TENSORS, kRun = 256;
constexpr int64_t kSmallElements = PINN_NORM_SMALL_ELEMENTS;
static_assert(kSmallTensors == 64, "a lane for each tensor");

__device__ inline int length_of(const NormArgs &a, int k)
{
    return (a.first_chunk[k + 1] - a.first_chunk[k] - 1) * kNormChunk + a.tail(k);
}

// f(elements of a lane, how many there are, their address) for all runs; first[k]: runs before tensor k
template <class F>
__device__ inline void over_runs(const NormArgs &a, const int *first, F f)
{
    const int lane = threadIdx.x & 63, upto = first[lane + 1], total = first[kSmallTensors];
    for (int j = threadIdx.x >> 6; j < total; j += kSmallThreads / 64) {
        const int k = __popcll(__ballot(upto <= j));           // the tensors that end before run j
        const int i = (j - first[k]) * kRun + lane * 4, have = length_of(a, k) - i;
        if (a.dtype(k) == PINN_F32) f(load_some<false, 4>((float *)a.x[k] + i, have), have, (float *)a.x[k] + i);
        else if (a.dtype(k) == PINN_BF16) f(load_some<false, 4>((__bf16 *)a.x[k] + i, have), have, (__bf16 *)a.x[k] + i);
        else f(load_some<false, 4>((_Float16 *)a.x[k] + i, have), have, (_Float16 *)a.x[k] + i);
    }
}

__global__ __launch_bounds__(kSmallThreads) void k_norm_small(const NormArgs a, double max_norm, float *norm_out)
{
    __shared__ int first[kSmallTensors + 1];
    __shared__ double part[kSmallThreads / 64];
    if (threadIdx.x < kSmallTensors) {
        const int k = threadIdx.x;
        int runs = k < a.n_tensors ? (length_of(a, k) + kRun - 1) / kRun : 0;
        for (int d = 1; d < 64; d <<= 1) {
            const int before = __shfl_up(runs, d);
            if (k >= d) runs += before;
        }
        first[k + 1] = runs;
        if (k == 0) first[0] = 0;
    }
    __syncthreads();
    double s = 0.0;
    over_runs(a, first, [&](auto x, int, auto *) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fma((double)(float)x[e], (double)(float)x[e], s);
    });
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
    for (int w = 0; w < kSmallThreads / 64; ++w) s += part[w];
    const double norm = sqrt(s);
    if (threadIdx.x == 0) *norm_out = (float)norm;
    if (max_norm < 0.0) return;
    const Factor f(clip_factor(norm, max_norm));
    if (f.f == 1.0f && f.pre == 1.0f) return;
    over_runs(a, first, [&](auto x, int have, auto *at) {
        typedef std::remove_reference_t<decltype(*at)> T;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (T)(f * (float)x[e]);
        store_some<false, 4>(at, x, have);
    });
}

// ---- host ------------------------------------------------------------------------------------------------------
bool valid_dtype(int32_t d) { return d == PINN_F32 || d == PINN_BF16 || d == PINN_F16; }

int launch_error() { return hipGetLastError() == hipSuccess ? PINN_OK : PINN_ERR_HIP; }

template <class T, bool MASTER>
void launch_step(const StepArgs &a, StepConst c, int bits, hipStream_t st)
{
    // 10 bytes an element (8-bit moments, 16-bit weights without masters) leave so little to wait for that the instructions count: such
    // workgroups take 4 chunks each, which spreads the scalars of a step over more elements, and are not held back.  240M bfloat16
    // weights: 1 chunk 518 us, 2 451, 4 432, 8 446; held to 5 workgroups 560 (lists that do not fill the card have not been compared).  All others are bound by memory and go fastest when workgroups
    // come and go in the order of the addresses: 240M float32 weights, 8-bit moments: 1 chunk 773 us, 2 854, 4 957.
    const bool lean = bits == 8 && sizeof(T) == 2 && !MASTER;
    c.run = lean ? 4 : 1;
    const unsigned grid = (unsigned)((c.n_chunks + c.run - 1) / c.run), pace = lean ? 0 : bits == 32 ? kPace32 : kPace8;
    if (bits == 32) hipLaunchKernelGGL((k_adamw_group<T, MASTER, 32>), dim3(grid), dim3(kThreads), pace, st, a, c);
    else hipLaunchKernelGGL((k_adamw_group<T, MASTER, 8>), dim3(grid), dim3(kThreads), pace, st, a, c);
}

// the tables of one launch after another over a list of tensors, and how many partial sums each writes
struct NormPlan {
    int next = 0;          // first tensor of the next launch
    int partials = 0;      // partial sums of the launches so far
    unsigned grid = 0;
    bool advance(NormArgs &a, void *const *x, const int64_t *numel, const int32_t *dtype, int n)
    {
        int64_t chunks = 0;
        a.n_tensors = 0;
        a.first_partial = partials;
        for (; next < n && a.n_tensors < kNormTensors; ++next) {
            if (numel[next] == 0) continue;
            const int64_t more = (numel[next] + kNormChunk - 1) / kNormChunk;
            if (chunks + more > INT32_MAX) break;
            const int k = a.n_tensors++;
            a.x[k] = x[next];
            a.kind[k] = (uint32_t)(numel[next] - (more - 1) * kNormChunk) | (uint32_t)dtype[next] << 16;
            a.first_chunk[k] = (int32_t)chunks;
            chunks += more;
        }
        a.first_chunk[a.n_tensors] = (int32_t)chunks;
        grid = (unsigned)(chunks < kMaxPartials ? chunks : kMaxPartials);
        partials += (int)grid;
        return a.n_tensors > 0;
    }
};

int check_list(const void *const *x, const int64_t *numel, const int32_t *dtype, int32_t n)
{
    if (n < 0) return PINN_ERR_INVALID_DESC;
    if (n > 0 && (!x || !numel || !dtype)) return PINN_ERR_NULL;
    for (int32_t i = 0; i < n; ++i) {
        if (numel[i] < 0 || !valid_dtype(dtype[i])) return PINN_ERR_INVALID_DESC;
        if (numel[i] > (int64_t)INT32_MAX * kNormChunk) return PINN_ERR_TOO_LARGE;
        if (numel[i] > 0 && !x[i]) return PINN_ERR_NULL;
    }
    return PINN_OK;
}

// do two tensors share memory?  (scaling them in place would scale it twice, in no order)
int check_apart(void *const *x, const int64_t *numel, const int32_t *dtype, int32_t n)
{
    struct Span { uintptr_t begin, end; };
    Span *s = (Span *)malloc(sizeof(Span) * (size_t)(n > 0 ? n : 1));
    if (!s) return PINN_ERR_ALLOC;
    int m = 0;
    for (int32_t i = 0; i < n; ++i)
        if (numel[i] > 0) s[m++] = {(uintptr_t)x[i], (uintptr_t)x[i] + (uintptr_t)numel[i] * (dtype[i] == PINN_F32 ? 4 : 2)};
    const auto before = [](const Span &a, const Span &b) { return a.begin < b.begin; };
    if (!std::is_sorted(s, s + m, before)) std::sort(s, s + m, before);
    int rc = PINN_OK;
    for (int i = 1; i < m; ++i)
        if (s[i].begin < s[i - 1].end) rc = PINN_ERR_OVERLAP;
    free(s);
    return rc;
}

// the whole list in one workgroup's launch, if it is small enough
bool small_list(NormArgs &a, void *const *x, const int64_t *numel, const int32_t *dtype, int n)
{
    int64_t total = 0;
    for (int i = 0; i < n; ++i) {
        total += numel[i] <= kSmallElements ? numel[i] : kSmallElements + 1;
        if (total > kSmallElements) return false;
    }
    NormPlan plan;
    return (n <= kSmallTensors || total == 0) && (plan.advance(a, x, numel, dtype, n), true);
}

int launch_sumsq(const void *const *grads, const int64_t *numel, const int32_t *dtype, int n_tensors, double *partials, int64_t n_reserved,
                 int32_t *n_partials, void *stream)
{
    NormArgs a;
    NormPlan plan;
    while (plan.advance(a, (void *const *)grads, numel, dtype, n_tensors)) {
        if (plan.partials > n_reserved) return PINN_ERR_TOO_LARGE;
        hipLaunchKernelGGL(k_grad_sumsq, dim3(plan.grid), dim3(kThreads), 0, (hipStream_t)stream, a, partials);
        *n_partials = plan.partials;
    }
    return launch_error();
}

void fold(double *partials, int32_t &n_partials, void *stream)
{
    hipLaunchKernelGGL(k_fold, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, partials, (int)n_partials);
    n_partials = 1;
}

}  // namespace

// FNV-1a
static constexpr int32_t name_hash(const char *s)
{
    uint32_t h = 2166136261u;
    for (; *s; ++s) h = (h ^ (uint8_t)*s) * 16777619u;
    return (int32_t)h;
}

extern "C" int32_t pinn_layout(int32_t *out, int32_t n)
{
#define AT(S, F) name_hash(#F), (int32_t)offsetof(S, F)
#define CHUNK(F) AT(PinnAdamWChunk, F)
#define GROUP(F) AT(PinnAdamWGroup, F)
    static constexpr int32_t layout[] = {
        (int32_t)sizeof(pinn_desc), AT(pinn_desc, eq), AT(pinn_desc, n_lin), AT(pinn_desc, widths), AT(pinn_desc, lb), AT(pinn_desc, ub),
        AT(pinn_desc, coef), AT(pinn_desc, kernel), AT(pinn_desc, reserved),
        (int32_t)sizeof(PinnAdamWChunk), CHUNK(base), CHUNK(place), CHUNK(count), CHUNK(tensor), CHUNK(row), CHUNK(reserved),
        (int32_t)sizeof(PinnAdamWGroup), GROUP(chunks), GROUP(rows), GROUP(n_chunks), GROUP(n_tensors), GROUP(dtype), GROUP(state_bits),
        GROUP(skip_nonfinite), GROUP(exp_avg), GROUP(exp_avg_sq), GROUP(exp_avg_scale), GROUP(exp_avg_sq_scale), GROUP(master),
        GROUP(device_state), GROUP(ticket), GROUP(partials), GROUP(n_partials), GROUP(reserved), GROUP(norm), GROUP(max_norm), GROUP(lr),
        GROUP(beta1), GROUP(beta2), GROUP(eps), GROUP(weight_decay),
        PINN_ADAMW_BLOCK, PINN_ADAMW_CHUNK32, PINN_ADAMW_CHUNK8, PINN_ADAMW_MAX_TENSORS, PINN_ADAMW_MAX_CHUNKS, PINN_ADAMW_TICKET_WORDS,
        PINN_NORM_SMALL_TENSORS, PINN_NORM_SMALL_ELEMENTS, PINN_ERR_OVERLAP};
#undef GROUP
#undef CHUNK
#undef AT
    const int32_t count = (int32_t)(sizeof(layout) / sizeof(layout[0]));
    for (int32_t i = 0; out && i < n && i < count; ++i) out[i] = layout[i];
    return count;
}

extern "C" int64_t pinn_grad_norm_partials(int32_t n_tensors)
{
    return n_tensors < 0 ? PINN_ERR_INVALID_DESC : (int64_t)((n_tensors + kNormTensors - 1) / kNormTensors) * kMaxPartials;
}

extern "C" int pinn_grad_sumsq(const void *const *grads, const int64_t *numel, const int32_t *dtype, int32_t n_tensors, double *partials,
                               int64_t n_reserved, int32_t *n_partials, void *stream)
{
    if (const int rc = check_list(grads, numel, dtype, n_tensors)) return rc;
    if (!n_partials || !partials) return PINN_ERR_NULL;
    *n_partials = 0;
    if (const int rc = launch_sumsq(grads, numel, dtype, n_tensors, partials, n_reserved, n_partials, stream)) return rc;
    // Every workgroup of the step adds the partial sums up for itself.  Up to two loads a thread that costs less than a launch (5M
    // weights); beyond, there are thousands of workgroups and they are added once (60M float32 weights, 8-bit moments: 285 -> 255 us).
    if (*n_partials > 2 * kThreads) fold(partials, *n_partials, stream);
    return launch_error();
}

extern "C" int pinn_grad_norm(const void *const *grads, const int64_t *numel, const int32_t *dtype, int32_t n_tensors, double *partials,
                              int64_t n_reserved, float *norm, void *stream)
{
    if (const int rc = check_list(grads, numel, dtype, n_tensors)) return rc;
    if (!norm) return PINN_ERR_NULL;
    NormArgs a;
    if (small_list(a, (void *const *)grads, numel, dtype, n_tensors)) {
        hipLaunchKernelGGL(k_norm_small, dim3(1), dim3(kSmallThreads), 0, (hipStream_t)stream, a, -1.0, norm);
        return launch_error();
    }
    if (!partials) return PINN_ERR_NULL;
    int32_t n_partials = 0;
    if (const int rc = launch_sumsq(grads, numel, dtype, n_tensors, partials, n_reserved, &n_partials, stream)) return rc;
    hipLaunchKernelGGL(k_norm_of, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, partials, (int)n_partials, norm);
    return launch_error();
}

extern "C" int pinn_grad_clip(void *const *grads, const int64_t *numel, const int32_t *dtype, int32_t n_tensors, double *partials,
                              int64_t n_reserved, double max_norm, float *norm, void *stream)
{
    if (const int rc = check_list((const void *const *)grads, numel, dtype, n_tensors)) return rc;
    if (!norm) return PINN_ERR_NULL;
    if (!(max_norm >= 0.0)) return PINN_ERR_INVALID_DESC;
    if (const int rc = check_apart(grads, numel, dtype, n_tensors)) return rc;
    NormArgs a;
    if (small_list(a, grads, numel, dtype, n_tensors)) {
        hipLaunchKernelGGL(k_norm_small, dim3(1), dim3(kSmallThreads), 0, (hipStream_t)stream, a, max_norm, norm);
        return launch_error();
    }
    if (!partials) return PINN_ERR_NULL;
    int32_t n_partials = 0;
    if (const int rc = launch_sumsq((const void *const *)grads, numel, dtype, n_tensors, partials, n_reserved, &n_partials, stream)) return rc;
    // As in the step, but a launch counts for more beside these short ones: from 3 launches of the scaling on (2000 bfloat16 tensors of 60M
    // elements: 8 launches of 15.4 us, with the sums added once 11.1 and 8.6 for that; 300 tensors of 33M: 2 of 17.8, then 16.1 and 3.1).
    if (n_partials > 2 * kMaxPartials) fold(partials, n_partials, stream);
    NormPlan plan;
    for (float *out = norm; plan.advance(a, grads, numel, dtype, n_tensors); out = nullptr)
        hipLaunchKernelGGL(k_grad_clip, dim3(plan.grid), dim3(kThreads), 0, (hipStream_t)stream, a, partials, (int)n_partials, max_norm, out);
    return launch_error();
}

extern "C" int pinn_adamw_group_step(const PinnAdamWGroup *d, void *const *params, const void *const *grads, void *stream)
{
    if (!d || !params || !grads) return PINN_ERR_NULL;
    if (d->n_tensors < 0 || d->n_tensors > kMaxTensors || d->n_chunks < 0 || !valid_dtype(d->dtype) ||
        (d->state_bits != 32 && d->state_bits != 8) || d->n_partials < 0 || (d->master && d->dtype == PINN_F32))
        return PINN_ERR_INVALID_DESC;
    if (d->n_chunks > PINN_ADAMW_MAX_CHUNKS) return PINN_ERR_TOO_LARGE;
    if (d->n_tensors == 0 || d->n_chunks == 0) return PINN_OK;
    if (!d->chunks || !d->rows || !d->exp_avg || !d->exp_avg_sq || !d->device_state || !d->ticket) return PINN_ERR_NULL;
    if (d->state_bits == 8 && (!d->exp_avg_scale || !d->exp_avg_sq_scale)) return PINN_ERR_NULL;
    if (d->n_partials && !d->partials) return PINN_ERR_NULL;
    StepArgs a;
    bool any = false;
    for (int k = 0; k < d->n_tensors; ++k) {
        a.p[k] = params[k];
        a.g[k] = grads[k];
        if (grads[k] && !params[k]) return PINN_ERR_NULL;
        any |= grads[k] != nullptr;
    }
    if (!any) return PINN_OK;
    StepConst c;
    c.chunks = d->chunks;
    c.rows = d->rows;
    c.m = (uint8_t *)d->exp_avg;
    c.v = (uint8_t *)d->exp_avg_sq;
    c.sm = d->exp_avg_scale;
    c.sv = d->exp_avg_sq_scale;
    c.master = d->master;
    c.state = d->device_state;
    c.ticket = d->ticket;
    c.partials = d->partials;
    c.norm_out = d->norm;
    c.n_chunks = d->n_chunks;
    c.n_tensors = d->n_tensors;
    c.n_partials = d->n_partials;
    c.skip_nonfinite = d->skip_nonfinite;
    c.max_norm = d->max_norm;
    c.b1 = d->beta1;
    c.b2 = d->beta2;
    c.lr = d->lr;
    c.eps = d->eps;
    c.decay = 1.0 - d->lr * d->weight_decay;
    c.eps32 = (float)c.eps;
    c.decay32 = (float)c.decay;
    const hipStream_t st = (hipStream_t)stream;
    if (d->dtype == PINN_F32) launch_step<float, false>(a, c, d->state_bits, st);
    else if (d->dtype == PINN_BF16) {
        if (d->master) launch_step<__bf16, true>(a, c, d->state_bits, st);
        else launch_step<__bf16, false>(a, c, d->state_bits, st);
    } else {
        if (d->master) launch_step<_Float16, true>(a, c, d->state_bits, st);
        else launch_step<_Float16, false>(a, c, d->state_bits, st);
    }
    return launch_error();
}

extern "C" int pinn_adamw_moments(const uint8_t *exp_avg, const uint8_t *exp_avg_sq, const uint8_t *exp_avg_scale, const uint8_t *exp_avg_sq_scale,
                                  float *exp_avg_out, float *exp_avg_sq_out, int64_t n, void *stream)
{
    if (n < 0 || n % kBlock) return PINN_ERR_INVALID_DESC;
    if (n == 0) return PINN_OK;
    if (!exp_avg || !exp_avg_sq || !exp_avg_scale || !exp_avg_sq_scale || !exp_avg_out || !exp_avg_sq_out) return PINN_ERR_NULL;
    if (n > (int64_t)INT32_MAX * 4 * kThreads) return PINN_ERR_TOO_LARGE;
    for (int64_t at = 0; at < n; at += kMomentsLaunch) {
        const int64_t more = std::min(n - at, kMomentsLaunch), groups = (more / 4 + kThreads - 1) / kThreads;
        hipLaunchKernelGGL(k_moments, dim3((unsigned)groups), dim3(kThreads), 0, (hipStream_t)stream, exp_avg + at, exp_avg_sq + at,
                           exp_avg_scale + at / kBlock, exp_avg_sq_scale + at / kBlock, exp_avg_out + at, exp_avg_sq_out + at, more);
    }
    return launch_error();
}
