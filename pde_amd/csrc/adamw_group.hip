// AdamW over many tensors at once, with moments in float32 or in 8 bits, and the global gradient norm that clips them.
//
//   norm = sqrt(sum g^2) over all tensors,  f = min(1, max_norm / (norm + 1e-6))       (f = 1 without clipping)
//   m <- b1 m + (1 - b1) f g,   v <- b2 v + (1 - b2) (f g)^2
//   p <- (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Every element is read and written once (28 bytes for float32 throughout), so the step is bound by memory.  The tensors
// are cut into chunks of kChunk elements; a table that the caller keeps on the device says which tensor a chunk lies in, so
// one launch covers up to kMaxTensors tensors of any sizes; their addresses travel in the launch's arguments, because
// gradients move from step to step.  Moments and master weights are flat buffers in which each tensor starts at a multiple of kBlock.
//
// 8-bit moments: a block of kBlock = 128 elements shares one scale 2^(s - 127) (a byte; 255 = the block is not finite), and
// an element is one byte: m as sign + 4 bits of exponent + 3 of mantissa, v (never negative) as 5 bits of exponent + 3 of mantissa.
// Scales are powers of two, so decoding and scaling are exact and the only rounding is the one to the byte.  It rounds up
// with probability equal to the remainder, by a sequence over steps and elements that covers [0, 1) evenly:
// with b2 = 0.999 a moment changes by less than half a code per step, and rounding to nearest would freeze it.
// The arithmetic is float64 (as fast as unpacked float32 on this hardware): the top 20 bits of a double's mantissa hold the
// 3 bits of the code and 17 bits of remainder, so rounding is one integer addition on the double's upper word, and it is exact -
// the codes do not depend on how a compiler contracts a float32 expression.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdlib.h>

#include <algorithm>

#include "../../include/pinnjet.h"

namespace {

constexpr int kThreads = 256;
constexpr int kBlock = PINN_ADAMW_BLOCK;        // elements that share a scale; also the layout's alignment
constexpr int kChunk = PINN_ADAMW_CHUNK;        // elements a workgroup takes at a time
constexpr int kMaxTensors = PINN_ADAMW_MAX_TENSORS;
constexpr int kNormTensors = 160;
constexpr int kNormChunk = 8192;
constexpr int kMaxPartials = PINN_NORM_PARTIALS;
static_assert(sizeof(PinnTensorSpan) == 32 && sizeof(PinnAdamWGroup) == 168, "the callers' layouts");
static_assert(kChunk == 8 * kThreads && kChunk % kBlock == 0, "a thread takes 8 elements of a chunk");

// N elements at any address that an element may have: the loads stay wide, the hardware takes them unaligned
template <class T, int N>
__device__ inline void load(const T *p, T (&out)[N])
{
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    const V x = *(const V *)p;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = x[i];
}

template <class T, int N>
__device__ inline void store(T *p, const T (&in)[N])
{
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    V x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = in[i];
    *(V *)p = x;
}

// float32 rounded once to T.  The empty asm keeps the compiler from folding a float16 conversion into the fma before it
// (v_fma_mixlo_f16 rounds the unrounded sum): a 16-bit weight is its float32 master's rounding, bit for bit.
template <class T>
__device__ inline T rounded(float x)
{
    if constexpr (sizeof(T) == 2) asm("" : "+v"(x));
    return (T)x;
}

struct StepArgs {
    void *p[kMaxTensors];
    const void *g[kMaxTensors];                 // null: no gradient, the tensor is left alone
};
struct StepConst {
    const PinnTensorSpan *span;
    const uint16_t *chunk_tensor;
    uint8_t *m, *v, *sm, *sv;                   // m, v: float32 or codes; sm, sv: scales
    float *master;
    double *state;                              // [tensor][3]: step, b1^t, b2^t
    uint32_t *ticket;
    const double *partials;
    float *norm_out;
    int64_t n_chunks;
    int32_t n_tensors, n_partials, skip_nonfinite;
    double max_norm, b1, b2, lr;
    float eps, decay;
};
static_assert(sizeof(StepArgs) + sizeof(StepConst) <= 4096, "a launch's arguments");

// The sum of the partial sums, in an order that depends on their number alone: every workgroup gets the same bits.
__device__ double sum_partials(const double *partials, int n)
{
    __shared__ double part[kThreads / 64];
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

// ---- float32 moments -------------------------------------------------------------------------------------------
struct Scalars {
    float step_size, inv_bc2_sqrt;
    double p1, p2;
    uint32_t t;
};

__device__ inline Scalars scalars_of(const double *row, double b1, double b2, double lr)
{
    Scalars s;
    const double t0 = row[0];
    s.p1 = (t0 == 0.0 ? 1.0 : row[1]) * b1;
    s.p2 = (t0 == 0.0 ? 1.0 : row[2]) * b2;
    s.t = (uint32_t)(int64_t)(t0 + 1.0);
    s.step_size = (float)(lr / (1.0 - s.p1));
    s.inv_bc2_sqrt = (float)(1.0 / sqrt(1.0 - s.p2));
    return s;
}

struct Hyper32 {
    float b2, omb1, omb2, eps, decay, factor;
};

__device__ inline void update32(float &p, float g, float &m, float &v, const Scalars &s, const Hyper32 &h)
{
    g *= h.factor;
    p *= h.decay;
    m = fmaf(g - m, h.omb1, m);
    v = fmaf(h.omb2 * g, g, v * h.b2);
    const float denom = sqrtf(v) * s.inv_bc2_sqrt + h.eps;
    p = fmaf(-s.step_size, m / denom, p);
}

template <class T, bool MASTER>
__device__ inline void chunk32(T *p, const T *g, float *m, float *v, float *master, int64_t left, const Scalars &s, const Hyper32 &h)
{
    constexpr int N = 4, J = kChunk / (N * kThreads);
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int64_t i = (int64_t)(j * kThreads + threadIdx.x) * N;
        if (i + N <= left) {
            T pt[N], gt[N];
            float pf[N], mf[N], vf[N];
            load(g + i, gt);
            if constexpr (MASTER) load(master + i, pf);
            else load(p + i, pt);
            load(m + i, mf);
            load(v + i, vf);
#pragma unroll
            for (int e = 0; e < N; ++e) {
                if constexpr (!MASTER) pf[e] = (float)pt[e];
                update32(pf[e], (float)gt[e], mf[e], vf[e], s, h);
                pt[e] = rounded<T>(pf[e]);
            }
            store(p + i, pt);
            if constexpr (MASTER) store(master + i, pf);
            store(m + i, mf);
            store(v + i, vf);
        } else {
            for (int64_t e = i; e < left; ++e) {
                float pf = MASTER ? master[e] : (float)p[e], mf = m[e], vf = v[e];
                update32(pf, (float)g[e], mf, vf, s, h);
                p[e] = rounded<T>(pf);
                if constexpr (MASTER) master[e] = pf;
                m[e] = mf;
                v[e] = vf;
            }
        }
    }
}

// ---- 8-bit moments ---------------------------------------------------------------------------------------------
struct Format {
    int shift;        // the smallest normal code's exponent against float64's (2^-1022): value * 2^-shift puts code bits on top of the upper word
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

__device__ inline uint32_t code_of(double x, int scale, uint32_t w, const Format &f)
{
    const uint32_t hi = (uint32_t)__double2hiint(ldexp(x, 127 - scale - f.shift)) & 0x7fffffffu;
    const uint32_t c = (hi + (w >> 15 | 1u)) >> 17;
    return c > f.most_code ? f.most_code : c;
}

// the sequences that round: golden ratio, sqrt(2) over the elements; the two-dimensional analogue of the golden ratio over the steps
constexpr uint32_t kPlaceM = 0x9E3779B9u, kStepM = 0xC13FA9A9u, kPlaceV = 0x6A09E667u, kStepV = 0x91E10DA5u;

struct Hyper8 {
    double b1, b2, omb1, omb2, factor;
    float eps, decay;
};

template <class T, bool MASTER>
__device__ inline void chunk8(T *p, const T *g, uint8_t *m, uint8_t *v, uint8_t *sm, uint8_t *sv, float *master, int64_t place, int64_t left,
                              const Scalars &s, const Hyper8 &h)
{
    constexpr int N = 8;
    const int i = (int)threadIdx.x * N;         // a block is 16 lanes: a DPP row
    if ((int64_t)(i & ~(kBlock - 1)) >= left) return;   // whole rows leave together
    const int have = left - i >= N ? N : left - i <= 0 ? 0 : (int)(left - i);
    T gt[N], pt[N];
    float pf[N];
    if (have == N) {
        load(g + i, gt);
        if constexpr (MASTER) load(master + i, pf);
        else load(p + i, pt);
    } else {
        for (int e = 0; e < N; ++e) {
            gt[e] = e < have ? g[i + e] : (T)0.0f;
            if constexpr (MASTER) pf[e] = e < have ? master[i + e] : 0.0f;
            else pt[e] = e < have ? p[i + e] : (T)0.0f;
        }
    }
    const uint2 cm = *(const uint2 *)(m + i), cv = *(const uint2 *)(v + i);
    const int blk = i / kBlock;
    const int s0m = sm[blk], s0v = sv[blk];
    const double nan = __hiloint2double(0x7ff80000, 0);
    const double um = s0m == 255 ? nan : h.b1 * pow2(s0m - 127 + kM.shift32);
    const double uv = s0v == 255 ? nan : h.b2 * pow2(s0v - 127 + kV.shift32);
    double md[N], vd[N];
    uint32_t hm = 0, hv = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const uint32_t bm = ((e < 4 ? cm.x : cm.y) >> (8 * (e & 3))) & 255u, bv = ((e < 4 ? cv.x : cv.y) >> (8 * (e & 3))) & 255u;
        const double gd = (double)(float)gt[e] * h.factor;
        md[e] = fma((double)__uint_as_float((bm & 127u) << 20 | (bm & 128u) << 24), um, h.omb1 * gd);
        vd[e] = fma((double)__uint_as_float(bv << 20), uv, h.omb2 * gd * gd);
        const uint32_t am = (uint32_t)__double2hiint(md[e]) & 0x7fffffffu, av = (uint32_t)__double2hiint(vd[e]) & 0x7fffffffu;
        hm = am > hm ? am : hm;
        hv = av > hv ? av : hv;
        if constexpr (!MASTER) pf[e] = (float)pt[e];
        const float denom = sqrtf((float)vd[e]) * s.inv_bc2_sqrt + h.eps;
        pf[e] = fmaf(-s.step_size, (float)md[e] / denom, pf[e] * h.decay);
        pt[e] = rounded<T>(pf[e]);
    }
    const int s1m = scale_of(row_max(hm), kM), s1v = scale_of(row_max(hv), kV);
    const uint32_t at = (uint32_t)(place + i);
    uint32_t wm = at * kPlaceM + s.t * kStepM, wv = at * kPlaceV + s.t * kStepV;
    uint32_t om[2] = {0, 0}, ov[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < N; ++e, wm += kPlaceM, wv += kPlaceV) {
        uint32_t a = code_of(md[e], s1m, wm, kM) | ((uint32_t)__double2hiint(md[e]) >> 24 & 128u);
        uint32_t b = code_of(vd[e], s1v, wv, kV);
        if (b == 0 && vd[e] > 0.0) b = 1;       // a v that vanished under a live m would divide it by eps alone
        if (e >= have) a = b = 0;               // behind the tensor's end the codes stay zero
        om[e / 4] |= a << (8 * (e & 3));
        ov[e / 4] |= b << (8 * (e & 3));
    }
    if (s1m == 255) om[0] = om[1] = 0;
    if (s1v == 255) ov[0] = ov[1] = 0;
    *(uint2 *)(m + i) = make_uint2(om[0], om[1]);
    *(uint2 *)(v + i) = make_uint2(ov[0], ov[1]);
    if ((threadIdx.x & 15) == 0) {
        sm[blk] = (uint8_t)s1m;
        sv[blk] = (uint8_t)s1v;
    }
    if (have == N) {
        store(p + i, pt);
        if constexpr (MASTER) store(master + i, pf);
    } else {
        for (int e = 0; e < have; ++e) {
            p[i + e] = pt[e];
            if constexpr (MASTER) master[i + e] = pf[e];
        }
    }
}

template <class T, bool MASTER, int BITS>
__global__ __launch_bounds__(kThreads) void k_adamw_group(const StepArgs a, const StepConst c)
{
    double factor = 1.0;
    if (c.n_partials) {
        const double norm = sqrt(sum_partials(c.partials, c.n_partials));
        if (c.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *c.norm_out = (float)norm;
        if (c.skip_nonfinite && !(norm < __hiloint2double(0x7ff00000, 0))) return;   // in all workgroups alike: nothing is written, the ticket stays
        if (c.max_norm >= 0.0) factor = clip_factor(norm, c.max_norm);
    }
    Hyper32 h32;
    Hyper8 h8;
    if constexpr (BITS == 32) h32 = {(float)c.b2, (float)(1.0 - c.b1), (float)(1.0 - c.b2), c.eps, c.decay, (float)factor};
    else h8 = {c.b1, c.b2, 1.0 - c.b1, 1.0 - c.b2, factor, c.eps, c.decay};
    Scalars s;
    int last = -1;
    for (int64_t ch = blockIdx.x; ch < c.n_chunks; ch += gridDim.x) {
        const int k = c.chunk_tensor[ch];
        const T *g = (const T *)a.g[k];
        if (!g) continue;
        const PinnTensorSpan sp = c.span[k];
        const int64_t base = (ch - sp.first_chunk) * kChunk, left = sp.numel - base, at = sp.offset + base;
        if (k != last) s = scalars_of(c.state + 3 * (int64_t)sp.row, c.b1, c.b2, c.lr);
        last = k;
        T *p = (T *)a.p[k];
        if constexpr (BITS == 32)
            chunk32<T, MASTER>(p + base, g + base, (float *)c.m + at, (float *)c.v + at, c.master + at, left, s, h32);
        else
            chunk8<T, MASTER>(p + base, g + base, c.m + at, c.v + at, c.sm + at / kBlock, c.sv + at / kBlock, c.master + at, at, left, s, h8);
    }
    // the workgroup that finishes last advances the counters: every other one has read them by then
    __shared__ uint32_t done;
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        done = atomicAdd(c.ticket, 1u);
    }
    __syncthreads();
    if (done != gridDim.x - 1) return;
    for (int k = threadIdx.x; k < c.n_tensors; k += kThreads)
        if (a.g[k]) {
            double *row = c.state + 3 * (int64_t)c.span[k].row;
            const Scalars n = scalars_of(row, c.b1, c.b2, c.lr);
            row[0] += 1.0;
            row[1] = n.p1;
            row[2] = n.p2;
        }
    if (threadIdx.x == 0) __hip_atomic_store(c.ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// moments as float32: what the codes stand for
__global__ __launch_bounds__(kThreads) void k_moments(const uint8_t *m, const uint8_t *v, const uint8_t *sm, const uint8_t *sv, float *mo,
                                                            float *vo, int64_t n)
{
    for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * kThreads * 4) {
        const uint32_t cm = *(const uint32_t *)(m + i), cv = *(const uint32_t *)(v + i);
        const int s0m = sm[i / kBlock], s0v = sv[i / kBlock];
        float4 x, y;
        float *xs = (float *)&x, *ys = (float *)&y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t a = cm >> (8 * e) & 255u, b = cv >> (8 * e) & 255u;
            xs[e] = ldexpf(__uint_as_float((a & 127u) << 20 | (a & 128u) << 24), s0m - 127 + kM.shift32);
            ys[e] = ldexpf(__uint_as_float(b << 20), s0v - 127 + kV.shift32);
            if (s0m == 255) xs[e] = __uint_as_float(0x7fc00000u);
            if (s0v == 255) ys[e] = __uint_as_float(0x7fc00000u);
        }
        *(float4 *)(mo + i) = x;
        *(float4 *)(vo + i) = y;
    }
}

// ---- the global norm -------------------------------------------------------------------------------------------
// Squares are summed in float64: no gradient that float32 can hold overflows or vanishes there, so no pass looks for a scale first.
// Workgroup b always takes the same chunks and its sum has its own place, so the norm is the same bits on every run.
struct NormArgs {
    void *x[kNormTensors];
    int64_t numel[kNormTensors];
    int32_t first_chunk[kNormTensors + 1];
    uint8_t dtype[kNormTensors];
    int32_t n_tensors, first_partial;
};

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

template <class T>
__device__ inline double chunk_sumsq(const T *x, int64_t left)
{
    constexpr int N = 16 / sizeof(T);
    double s = 0.0;
    if (left >= kNormChunk) {
#pragma unroll
        for (int j = 0; j < kNormChunk / (N * kThreads); ++j) {
            T t[N];
            load(x + (j * kThreads + threadIdx.x) * N, t);
#pragma unroll
            for (int e = 0; e < N; ++e) s = fma((double)(float)t[e], (double)(float)t[e], s);
        }
    } else {
        for (int64_t i = threadIdx.x; i < left; i += kThreads) s = fma((double)(float)x[i], (double)(float)x[i], s);
    }
    return s;
}

__global__ __launch_bounds__(kThreads) void k_grad_sumsq(const NormArgs a, double *partials)
{
    double s = 0.0;
    const int64_t n_chunks = a.first_chunk[a.n_tensors];
    for (int64_t ch = blockIdx.x; ch < n_chunks; ch += gridDim.x) {
        const int k = find_tensor(a, ch);
        const int64_t base = (ch - a.first_chunk[k]) * kNormChunk, left = a.numel[k] - base;
        if (a.dtype[k] == PINN_F32) s += chunk_sumsq((const float *)a.x[k] + base, left);
        else if (a.dtype[k] == PINN_BF16) s += chunk_sumsq((const __bf16 *)a.x[k] + base, left);
        else s += chunk_sumsq((const _Float16 *)a.x[k] + base, left);
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

__global__ __launch_bounds__(kThreads) void k_norm_of(const double *partials, int n, float *norm)
{
    const double s = sum_partials(partials, n);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

template <class T>
__device__ inline void chunk_scale(T *x, int64_t left, float f)
{
    constexpr int N = 16 / sizeof(T);
    if (left >= kNormChunk) {
#pragma unroll
        for (int j = 0; j < kNormChunk / (N * kThreads); ++j) {
            T t[N], *at = x + (j * kThreads + threadIdx.x) * N;
            load(at, t);
#pragma unroll
            for (int e = 0; e < N; ++e) t[e] = (T)((float)t[e] * f);
            store(at, t);
        }
    } else {
        for (int64_t i = threadIdx.x; i < left; i += kThreads) x[i] = (T)((float)x[i] * f);
    }
}

__global__ __launch_bounds__(kThreads) void k_grad_clip(const NormArgs a, const double *partials, int n_partials, double max_norm, float *norm_out)
{
    const double norm = sqrt(sum_partials(partials, n_partials));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const float f = (float)clip_factor(norm, max_norm);
    if (f == 1.0f) return;                      // the gradients stay as they are: nothing to write
    const int64_t n_chunks = a.first_chunk[a.n_tensors];
    for (int64_t ch = blockIdx.x; ch < n_chunks; ch += gridDim.x) {
        const int k = find_tensor(a, ch);
        const int64_t base = (ch - a.first_chunk[k]) * kNormChunk, left = a.numel[k] - base;
        if (a.dtype[k] == PINN_F32) chunk_scale((float *)a.x[k] + base, left, f);
        else if (a.dtype[k] == PINN_BF16) chunk_scale((__bf16 *)a.x[k] + base, left, f);
        else chunk_scale((_Float16 *)a.x[k] + base, left, f);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------
bool valid_dtype(int32_t d) { return d == PINN_F32 || d == PINN_BF16 || d == PINN_F16; }

int launch_error() { return hipGetLastError() == hipSuccess ? PINN_OK : PINN_ERR_HIP; }

template <class T, bool MASTER>
void launch_step(const StepArgs &a, const StepConst &c, int bits, unsigned grid, hipStream_t st)
{
    if (bits == 32) hipLaunchKernelGGL((k_adamw_group<T, MASTER, 32>), dim3(grid), dim3(kThreads), 0, st, a, c);
    else hipLaunchKernelGGL((k_adamw_group<T, MASTER, 8>), dim3(grid), dim3(kThreads), 0, st, a, c);
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
            a.numel[k] = numel[next];
            a.dtype[k] = (uint8_t)dtype[next];
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
    std::sort(s, s + m, [](const Span &a, const Span &b) { return a.begin < b.begin; });
    int rc = PINN_OK;
    for (int i = 1; i < m; ++i)
        if (s[i].begin < s[i - 1].end) rc = PINN_ERR_OVERLAP;
    free(s);
    return rc;
}

}  // namespace

extern "C" int64_t pinn_grad_norm_partials(int32_t n_tensors)
{
    return n_tensors < 0 ? PINN_ERR_INVALID_DESC : (int64_t)((n_tensors + kNormTensors - 1) / kNormTensors) * kMaxPartials;
}

extern "C" int pinn_grad_sumsq(const void *const *grads, const int64_t *numel, const int32_t *dtype, int32_t n_tensors, double *partials,
                               int64_t n_reserved, int32_t *n_partials, void *stream)
{
    if (const int rc = check_list(grads, numel, dtype, n_tensors)) return rc;
    if (!n_partials || !partials) return PINN_ERR_NULL;
    NormArgs a;
    NormPlan plan;
    *n_partials = 0;
    while (plan.advance(a, (void *const *)grads, numel, dtype, n_tensors)) {
        if (plan.partials > n_reserved) return PINN_ERR_TOO_LARGE;
        hipLaunchKernelGGL(k_grad_sumsq, dim3(plan.grid), dim3(kThreads), 0, (hipStream_t)stream, a, partials);
        *n_partials = plan.partials;
    }
    return launch_error();
}

extern "C" int pinn_grad_norm(const double *partials, int32_t n_partials, float *norm, void *stream)
{
    if (!partials || !norm) return PINN_ERR_NULL;
    if (n_partials < 0) return PINN_ERR_INVALID_DESC;
    hipLaunchKernelGGL(k_norm_of, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, partials, (int)n_partials, norm);
    return launch_error();
}

extern "C" int pinn_grad_clip(void *const *grads, const int64_t *numel, const int32_t *dtype, int32_t n_tensors, const double *partials,
                              int32_t n_partials, double max_norm, float *norm, void *stream)
{
    if (const int rc = check_list((const void *const *)grads, numel, dtype, n_tensors)) return rc;
    if (!partials || !norm) return PINN_ERR_NULL;
    if (n_partials < 0 || !(max_norm >= 0.0)) return PINN_ERR_INVALID_DESC;
    if (const int rc = check_apart(grads, numel, dtype, n_tensors)) return rc;
    NormArgs a;
    NormPlan plan;
    float *out = norm;
    while (plan.advance(a, grads, numel, dtype, n_tensors)) {
        hipLaunchKernelGGL(k_grad_clip, dim3(plan.grid), dim3(kThreads), 0, (hipStream_t)stream, a, partials, (int)n_partials, max_norm, out);
        out = nullptr;
    }
    if (out) return pinn_grad_norm(partials, n_partials, norm, stream);   // nothing but empty tensors
    return launch_error();
}

extern "C" int pinn_adamw_group_step(const PinnAdamWGroup *d, void *const *params, const void *const *grads, void *stream)
{
    if (!d || !params || !grads) return PINN_ERR_NULL;
    if (d->n_tensors < 0 || d->n_tensors > kMaxTensors || d->n_chunks < 0 || !valid_dtype(d->dtype) ||
        (d->state_bits != 32 && d->state_bits != 8) || d->n_partials < 0 || (d->master && d->dtype == PINN_F32))
        return PINN_ERR_INVALID_DESC;
    if (d->n_tensors == 0 || d->n_chunks == 0) return PINN_OK;
    if (!d->spans || !d->chunk_tensor || !d->exp_avg || !d->exp_avg_sq || !d->device_state || !d->ticket) return PINN_ERR_NULL;
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
    c.span = d->spans;
    c.chunk_tensor = d->chunk_tensor;
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
    c.eps = (float)d->eps;
    c.decay = (float)(1.0 - d->lr * d->weight_decay);
    const unsigned grid = (unsigned)(d->n_chunks < PINN_ADAMW_GRID ? d->n_chunks : PINN_ADAMW_GRID);
    const hipStream_t st = (hipStream_t)stream;
    if (d->dtype == PINN_F32) launch_step<float, false>(a, c, d->state_bits, grid, st);
    else if (d->dtype == PINN_BF16) {
        if (d->master) launch_step<__bf16, true>(a, c, d->state_bits, grid, st);
        else launch_step<__bf16, false>(a, c, d->state_bits, grid, st);
    } else {
        if (d->master) launch_step<_Float16, true>(a, c, d->state_bits, grid, st);
        else launch_step<_Float16, false>(a, c, d->state_bits, grid, st);
    }
    return launch_error();
}

extern "C" int pinn_adamw_moments(const uint8_t *exp_avg, const uint8_t *exp_avg_sq, const uint8_t *exp_avg_scale, const uint8_t *exp_avg_sq_scale,
                                  float *exp_avg_out, float *exp_avg_sq_out, int64_t n, void *stream)
{
    if (n < 0 || n % kBlock) return PINN_ERR_INVALID_DESC;
    if (n == 0) return PINN_OK;
    if (!exp_avg || !exp_avg_sq || !exp_avg_scale || !exp_avg_sq_scale || !exp_avg_out || !exp_avg_sq_out) return PINN_ERR_NULL;
    const int64_t groups = (n / 4 + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(k_moments, dim3((unsigned)(groups < 8192 ? groups : 8192)), dim3(kThreads), 0, (hipStream_t)stream, exp_avg,
                       exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, exp_avg_out, exp_avg_sq_out, n);
    return launch_error();
}
