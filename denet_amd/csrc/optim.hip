// Optimizer operators over many tensors at once: the global L2 norm of a gradient list (with its clipping form) and the
// AdamW step with 32-bit or 8-bit states.
//
// A call takes a HOST array of tensor descriptors.  They travel as kernel arguments (at most 4 KB), so a launch covers
// up to OPT_SLOTS tensors and nothing has to be copied to the device first, kept between calls or re-validated: a
// captured graph holds its own copy.  The work is cut into chunks of CHUNK elements; `start[i]` is the first chunk of
// tensor i in the launch, and a block finds its tensor with one vector load and a ballot over the starts.
#include <math.h>
#include "denet_common.hpp"

// every operation of this file is rounded by itself (the AdamW step below says why); sums use explicit fma
#pragma clang fp contract(off)

#define OPT_THREADS 256
#define OPT_SLOTS 64                // one lane per tensor in the look-up
#define QBLOCK 256                  // consecutive elements that share a scale of the 8-bit states (one wave, 4 per lane)
#define NORM_PARTS 1024             // most partial sums of a norm: every block of the consumer adds them up itself
#define E4M3_MAX 448.f
#define SCALE_MIN 1.1754943508222875e-38f   // 2^-126

typedef float f32x4_u __attribute__((ext_vector_type(4), aligned(4)));      // views of a flat bucket start anywhere
typedef unsigned short u16x4_u __attribute__((ext_vector_type(4), aligned(2)));

// ---- four consecutive elements of a tensor -----------------------------------------------------------------------
template <typename T> struct Quad;
template <> struct Quad<float> {
    static __device__ __forceinline__ void load(const float* p, float x[4]) {
        const f32x4_u v = *reinterpret_cast<const f32x4_u*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e];
    }
    static __device__ __forceinline__ void store(float* p, const float x[4]) {
        *reinterpret_cast<f32x4_u*>(p) = f32x4_u{x[0], x[1], x[2], x[3]};
    }
};
template <> struct Quad<unsigned short> {
    static __device__ __forceinline__ void load(const unsigned short* p, float x[4]) {
        const u16x4_u v = *reinterpret_cast<const u16x4_u*>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = bf16_to_f32(v[e]);
    }
    static __device__ __forceinline__ void store(unsigned short* p, const float x[4]) {
        *reinterpret_cast<u16x4_u*>(p) = u16x4_u{f32_to_bf16(x[0]), f32_to_bf16(x[1]), f32_to_bf16(x[2]), f32_to_bf16(x[3])};
    }
};
// k = how many of the four exist (1..4)
template <typename T>
__device__ __forceinline__ void load4(const T* p, int k, float x[4]) {
    if (k == 4) { Quad<T>::load(p, x); return; }
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = e < k ? FeatIO<T>::load(p + e) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int k, const float x[4]) {
    if (k == 4) { Quad<T>::store(p, x); return; }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < k) FeatIO<T>::store(p + e, x[e]);
}

// The argument struct is read where the launch put it: indexing a by-value parameter would copy it to scratch first.
#define KARG(T) const __attribute__((address_space(4))) T
template <typename T>
__device__ __forceinline__ KARG(T)* kernel_args() {
    return (KARG(T)*)__builtin_amdgcn_kernarg_segment_ptr();
}

// the tensor that chunk `b` of a launch belongs to; starts[count..63] are not read into the vote
__device__ __forceinline__ int find_slot(KARG(int)* starts, int count, int b) {
    const int lane = threadIdx.x & 63;
    const bool before = lane < count && starts[lane] <= b;
    return __popcll(__ballot(before)) - 1;
}

// ---- the norm -----------------------------------------------------------------------------------------------------
// Sums of squares are kept in 64 bits from the first element on: fp32 squares overflow from |g| = 1.8e19 on, and long
// fp32 sums lose the small gradients.  The fp64 FMA runs at the fp32 rate on this chip, so the pass stays a read.
struct NormSlot { void* g; int64_t n; };          // n: bits 0..47 elements, bit 60: bf16
struct NormArgs {
    int start[OPT_SLOTS];
    NormSlot slot[OPT_SLOTS];
    double* part;
    int count, chunks;
};
#define OPT_N(x) ((x) & ((1ll << 48) - 1))
#define NORM_CHUNK 4096

__device__ __forceinline__ double block_sum(double v, double* red) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T>
__device__ __forceinline__ double chunk_sumsq(const T* g, int64_t left) {
    double s[4] = {0., 0., 0., 0.};
#pragma unroll
    for (int u = 0; u < NORM_CHUNK / (4 * OPT_THREADS); ++u) {
        const int64_t i = 4 * (u * OPT_THREADS + (int)threadIdx.x);
        if (i < left) {
            float x[4];
            load4(g + i, left - i < 4 ? (int)(left - i) : 4, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] = fma((double)x[e], (double)x[e], s[e]);
        }
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

__global__ __launch_bounds__(OPT_THREADS) void grad_sumsq_kernel(NormArgs by_value) {
    KARG(NormArgs)& a = *kernel_args<NormArgs>();
    __shared__ double red[4];
    double s = 0.;
    for (int b = blockIdx.x; b < a.chunks; b += gridDim.x) {
        const int i = __builtin_amdgcn_readfirstlane(find_slot(a.start, a.count, b));
        const int64_t n = a.slot[i].n, first = (int64_t)(b - a.start[i]) * NORM_CHUNK, left = OPT_N(n) - first;
        s += ((n >> 60) & 1) ? chunk_sumsq((const unsigned short*)a.slot[i].g + first, left)
                       : chunk_sumsq((const float*)a.slot[i].g + first, left);
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) a.part[blockIdx.x] = s;
}

struct ClipArgs { const double* part; double max_norm; float* norm; float* coef; int parts; };     // norm, coef: written where not NULL

// every block forms the same sum in the same order
__device__ __forceinline__ float clip_coef(const ClipArgs& c, double* red, bool write_norm) {
    double s = 0.;
    for (int i = threadIdx.x; i < c.parts; i += OPT_THREADS) s += c.part[i];
    const double n = sqrt(block_sum(s, red));
    if (write_norm && threadIdx.x == 0 && c.norm) *c.norm = (float)n;
    const double q = c.max_norm / (n + 1e-6);
    const float coef = q >= 1. ? 1.f : (float)q;        // a NaN norm makes a NaN coefficient, an infinite one 0
    if (write_norm && threadIdx.x == 0 && c.coef) *c.coef = coef;
    return coef;
}

__global__ __launch_bounds__(OPT_THREADS) void norm_finish_kernel(ClipArgs c) {
    __shared__ double red[4];
    (void)clip_coef(c, red, true);
}

#define SCALE_CHUNK 4096
struct ScaleArgs {
    int start[OPT_SLOTS];
    NormSlot slot[OPT_SLOTS];
    ClipArgs clip;
    int count, first_launch;
};
template <typename T>
__device__ __forceinline__ void chunk_scale(T* g, int64_t left, float c) {
#pragma unroll
    for (int u = 0; u < SCALE_CHUNK / (4 * OPT_THREADS); ++u) {
        const int64_t i = 4 * (u * OPT_THREADS + (int)threadIdx.x);
        if (i < left) {
            const int k = left - i < 4 ? (int)(left - i) : 4;
            float x[4];
            load4(g + i, k, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] *= c;
            store4(g + i, k, x);
        }
    }
}
__global__ __launch_bounds__(OPT_THREADS) void grad_scale_kernel(ScaleArgs by_value) {
    KARG(ScaleArgs)& a = *kernel_args<ScaleArgs>();
    __shared__ double red[4];
    const float c = clip_coef({a.clip.part, a.clip.max_norm, a.clip.norm, nullptr, a.clip.parts}, red, a.first_launch && blockIdx.x == 0);
    if (c == 1.f) return;                               // x * 1 = x for every x
    const int b = blockIdx.x, i = __builtin_amdgcn_readfirstlane(find_slot(a.start, a.count, b));
    const int64_t n = a.slot[i].n, first = (int64_t)(b - a.start[i]) * SCALE_CHUNK, left = OPT_N(n) - first;
    if ((n >> 60) & 1) chunk_scale((unsigned short*)a.slot[i].g + first, left, c);
    else chunk_scale((float*)a.slot[i].g + first, left, c);
}

// ---- AdamW ----------------------------------------------------------------------------------------------------------
//   g' = coef g;  m <- b1 m + (1-b1) g';  v <- b2 v + (1-b2) g'^2
//   p  <- (1 - lr wd) p - lr / (1-b1^t) * m / (sqrt(v) / sqrt(1-b2^t) + eps)
// Every operation is rounded by itself (no contraction, IEEE division and square root), so the step is the same fp32
// arithmetic as the formula written with elementary tensor operations, bit for bit.
struct AdamSlot {
    void* p; const void* g; void* m; void* v; float* ms; float* vs;
    int64_t n;                       // bits 0..47 elements, bit 60: bf16 parameter, bit 61: bf16 gradient
    float step_size, inv_bc2;        // lr / (1-b1^t), 1 / sqrt(1-b2^t)
    int index;                       // of the tensor in the caller's list (its place in the clock)
};
#define ADAM_SLOTS 52                // what fits into the 4 KB of kernel arguments
struct AdamArgs {
    int start[ADAM_SLOTS];
    AdamSlot slot[ADAM_SLOTS];
    ClipArgs clip;                   // clip.part NULL: no clipping
    const float* coef;               // coefficient that an earlier norm left; or NULL
    const float* clock;              // device-side step counters: decay, then {step_size, inv_bc2} per tensor; or NULL
    float decay, b1, c1, b2, c2, eps;
    int count, first_launch;
};
static_assert(sizeof(AdamArgs) <= 4096 && sizeof(ScaleArgs) <= 4096 && sizeof(NormArgs) <= 4096, "kernel arguments");

struct AdamC { float decay, b1, c1, b2, c2, eps, step_size, inv_bc2, coef; };

__device__ __forceinline__ void adam_moments(float g, float& m, float& v, const AdamC& c) {
    g = g * c.coef;
    m = m * c.b1 + g * c.c1;
    v = v * c.b2 + (g * g) * c.c2;
}
__device__ __forceinline__ float adam_update(float p, float m, float r, const AdamC& c) {
    const float denom = r * c.inv_bc2 + c.eps;
    return p * c.decay - (m / denom) * c.step_size;
}

template <typename PT, typename GT>
__device__ __forceinline__ void adam32_chunk(PT* p, const GT* g, float* m, float* v, int64_t left, int elems, const AdamC& c) {
    for (int i = 4 * (int)threadIdx.x; i < elems && i < left; i += 4 * OPT_THREADS) {
        const int k = left - i < 4 ? (int)(left - i) : 4;
        float xp[4], xg[4], xm[4], xv[4];
        load4(p + i, k, xp);
        load4(g + i, k, xg);
        load4(m + i, k, xm);
        load4(v + i, k, xv);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            adam_moments(xg[e], xm[e], xv[e], c);
            xp[e] = adam_update(xp[e], xm[e], sqrtf(xv[e]), c);
        }
        store4(m + i, k, xm);
        store4(v + i, k, xv);
        store4(p + i, k, xp);
    }
}

// 8-bit states: e4m3 codes of m / s and of sqrt(v) / s, s = max(absmax / 448, 2^-126) over QBLOCK elements.
//  - sqrt(v) and not v: half the range in octaves, so the 17.8 octaves of e4m3 span a factor of 2^35 in v.
//  - s is a full fp32 number and not a power of two: the largest entry of a block is then held to 2^-24, and with
//    it the block's slow drift (v moves by 1 - b2 = 0.1 % a step, far below half a code) is carried by the scale.
//  - sqrt(v) > 0 never gets code 0: rounding a denominator down to eps would blow its entry's update up.
//  - the update of p uses the moments of this step before they are rounded.
//  - an entry that is not finite takes the NaN code and is left out of absmax: its neighbours keep their values.
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a <= 3.4028234663852886e38f ? a : 0.f;
}
__device__ __forceinline__ float quant_scale(float amax) {
    const float s = amax * (1.f / E4M3_MAX);
    return s > SCALE_MIN ? s : SCALE_MIN;
}
__device__ __forceinline__ unsigned e4m3x4(const float y[4]) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
}
__device__ __forceinline__ void from_e4m3x4(unsigned w, float scale, float x[4]) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = lo[0] * scale; x[1] = lo[1] * scale; x[2] = hi[0] * scale; x[3] = hi[1] * scale;
}
__device__ __forceinline__ unsigned load_codes(const unsigned char* p, int k) {
    if (k == 4) return *reinterpret_cast<const unsigned*>(p);
    unsigned w = 0;
#pragma unroll
    for (int e = 0; e < 3; ++e) if (e < k) w |= (unsigned)p[e] << (8 * e);
    return w;
}
__device__ __forceinline__ void store_codes(unsigned char* p, int k, unsigned w) {
    if (k == 4) { *reinterpret_cast<unsigned*>(p) = w; return; }
#pragma unroll
    for (int e = 0; e < 3; ++e) if (e < k) p[e] = (unsigned char)(w >> (8 * e));
}

// one QBLOCK per wave: `left` elements from its first on
template <typename PT, typename GT>
__device__ __forceinline__ void adam8_block(PT* p, const GT* g, unsigned char* m, unsigned char* r, float* ms, float* rs,
                                            int64_t left, const AdamC& c) {
    const int i = 4 * (threadIdx.x & 63);
    const int k = left - i >= 4 ? 4 : left > i ? (int)(left - i) : 0;
    float xp[4] = {0.f, 0.f, 0.f, 0.f}, xg[4] = {0.f, 0.f, 0.f, 0.f}, xm[4] = {0.f, 0.f, 0.f, 0.f}, xr[4] = {0.f, 0.f, 0.f, 0.f};
    if (k) {
        load4(p + i, k, xp);
        load4(g + i, k, xg);
        from_e4m3x4(load_codes(m + i, k), *ms, xm);
        from_e4m3x4(load_codes(r + i, k), *rs, xr);
    }
    float am = 0.f, ar = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float v = xr[e] * xr[e];
        adam_moments(xg[e], xm[e], v, c);
        xr[e] = sqrtf(v);
        xp[e] = adam_update(xp[e], xm[e], xr[e], c);
        am = fmaxf(am, finite_abs(xm[e]));
        ar = fmaxf(ar, finite_abs(xr[e]));
    }
    const float sm = quant_scale(wave_max(am)), sr = quant_scale(wave_max(ar));
    const float im = 1.f / sm, ir = 1.f / sr;
    float ym[4], yr[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        ym[e] = fabsf(xm[e]) <= 3.4028234663852886e38f ? xm[e] * im : __builtin_nanf("");
        yr[e] = xr[e] <= 3.4028234663852886e38f ? xr[e] * ir : __builtin_nanf("");
        if (yr[e] > 0.f && yr[e] < 0.001953125f) yr[e] = 0.001953125f;       // 2^-9, the smallest code
    }
    if (k) {
        store_codes(m + i, k, e4m3x4(ym));
        store_codes(r + i, k, e4m3x4(yr));
        store4(p + i, k, xp);
    }
    if ((threadIdx.x & 63) == 0) { *ms = sm; *rs = sr; }
}

#define ADAM_CHUNK 4096
template <int BITS, typename PT, typename GT>
__device__ __forceinline__ void adam_chunk(const AdamSlot& s, int64_t first, int64_t left, const AdamC& c) {
    if constexpr (BITS == 32) {
        adam32_chunk((PT*)s.p + first, (const GT*)s.g + first, (float*)s.m + first, (float*)s.v + first, left, ADAM_CHUNK, c);
    } else {
        for (int b = threadIdx.x >> 6; b < ADAM_CHUNK / QBLOCK && (int64_t)b * QBLOCK < left; b += OPT_THREADS / 64) {
            const int64_t at = first + b * QBLOCK, q = at / QBLOCK;
            adam8_block((PT*)s.p + at, (const GT*)s.g + at, (unsigned char*)s.m + at, (unsigned char*)s.v + at, s.ms + q, s.vs + q,
                        left - b * QBLOCK, c);
        }
    }
}

template <int BITS>
__global__ __launch_bounds__(OPT_THREADS) void adamw_kernel(AdamArgs by_value) {
    KARG(AdamArgs)& a = *kernel_args<AdamArgs>();
    __shared__ double red[4];
    const int b = blockIdx.x, i = __builtin_amdgcn_readfirstlane(find_slot(a.start, a.count, b));
    KARG(AdamSlot)& k = a.slot[i];
    const AdamSlot s = {k.p, k.g, k.m, k.v, k.ms, k.vs, k.n, k.step_size, k.inv_bc2, k.index};
    const int64_t first = (int64_t)(b - a.start[i]) * ADAM_CHUNK, left = OPT_N(s.n) - first;
    AdamC c = {a.decay, a.b1, a.c1, a.b2, a.c2, a.eps, s.step_size, s.inv_bc2, 1.f};
    if (a.clock) {
        c.decay = a.clock[0];
        c.step_size = a.clock[1 + 2 * s.index];
        c.inv_bc2 = a.clock[2 + 2 * s.index];
    }
    if (a.coef) c.coef = *a.coef;
    if (a.clip.part) c.coef = clip_coef({a.clip.part, a.clip.max_norm, a.clip.norm, nullptr, a.clip.parts}, red, a.first_launch && b == 0);
    switch ((int)(s.n >> 60) & 3) {
        case 0: adam_chunk<BITS, float, float>(s, first, left, c); break;
        case 1: adam_chunk<BITS, unsigned short, float>(s, first, left, c); break;
        case 2: adam_chunk<BITS, float, unsigned short>(s, first, left, c); break;
        default: adam_chunk<BITS, unsigned short, unsigned short>(s, first, left, c); break;
    }
}

// Device-side step counters (updates that a captured graph replays): advances each and forms what the host forms otherwise
#define CLOCK_SLOTS 256
struct ClockArgs {
    int64_t* steps[CLOCK_SLOTS];     // NULL: an empty tensor without a counter
    double lr, wd, b1, b2;
    const float* lr_dev;
    float* clock;
    int count, base;
};
static_assert(sizeof(ClockArgs) <= 4096 && CLOCK_SLOTS == OPT_THREADS, "one block, one counter per thread");
__global__ __launch_bounds__(OPT_THREADS) void adamw_clock_kernel(ClockArgs by_value) {
    KARG(ClockArgs)& a = *kernel_args<ClockArgs>();
    const int i = threadIdx.x;
    const double lr = a.lr_dev ? (double)*a.lr_dev : a.lr;
    if (i == 0 && a.base == 0) a.clock[0] = (float)(1. - lr * a.wd);
    if (i >= a.count || !a.steps[i]) return;
    const int64_t t = ++*a.steps[i];
    a.clock[1 + 2 * (a.base + i)] = (float)(lr / (1. - pow(a.b1, (double)t)));
    a.clock[2 + 2 * (a.base + i)] = (float)(1. / sqrt(1. - pow(a.b2, (double)t)));
}

// ---- host side --------------------------------------------------------------------------------------------------------
static int64_t chunks_of(int64_t n, int64_t chunk) { return (n + chunk - 1) / chunk; }

static bool bad_grad(const denet_opt_tensor_t& t) {
    return t.n < 0 || t.n >= (1ll << 48) || (t.n > 0 && !t.grad) || (t.grad_dtype != DENET_F32 && t.grad_dtype != DENET_BF16) ||
           ((uintptr_t)t.grad & (t.grad_dtype == DENET_F32 ? 3 : 1));
}
static int check_grads(const denet_opt_tensor_t* t, int64_t count) {
    if (count < 0 || count > (1ll << 24) || (count > 0 && !t)) return DENET_E_BADARG;
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (bad_grad(t[i])) return DENET_E_BADARG;
        chunks += chunks_of(t[i].n, NORM_CHUNK);
        if (chunks >= (1ll << 31)) return DENET_E_UNSUPPORTED;
    }
    return DENET_OK;
}

// Partial sums of the whole list: at most NORM_PARTS over all launches, shared out by their chunks; -> how many were written.
static int launch_sumsq(const denet_opt_tensor_t* t, int64_t count, double* part, hipStream_t st, int* parts_out) {
    int64_t total = 0;
    for (int64_t i = 0; i < count; ++i) total += chunks_of(t[i].n, NORM_CHUNK);
    int parts = 0;
    NormArgs a;
    a.count = a.chunks = 0;
    for (int64_t i = 0; i <= count; ++i) {
        if (a.count == OPT_SLOTS || (i == count && a.count)) {
            // (the share is rounded up, so every launch has a block; the list has at most NORM_PARTS / 2 launches, see the workspace)
            int64_t grid = a.chunks;
            if (total > NORM_PARTS) grid = (int64_t)a.chunks * (NORM_PARTS - 1) / total + 1;
            a.part = part + parts;
            hipLaunchKernelGGL(grad_sumsq_kernel, dim3((unsigned)grid), dim3(OPT_THREADS), 0, st, a);
            DENET_CHECK_LAUNCH();
            parts += (int)grid;
            a.count = a.chunks = 0;
        }
        if (i == count || t[i].n == 0) continue;
        a.start[a.count] = a.chunks;
        a.slot[a.count] = {t[i].grad, t[i].n | ((int64_t)(t[i].grad_dtype == DENET_BF16) << 60)};
        a.chunks += (int)chunks_of(t[i].n, NORM_CHUNK);
        ++a.count;
    }
    *parts_out = parts;
    return DENET_OK;
}

// partial sums: NORM_PARTS, one more for each launch (their shares are rounded up); then the clock of a device-side step counter
static int64_t part_bytes(int64_t count) { return (NORM_PARTS + count / OPT_SLOTS + 1) * (int64_t)sizeof(double); }

extern "C" int64_t denet_opt_workspace(int64_t count) {
    if (count < 0 || count > (1ll << 24)) return DENET_E_BADARG;
    return part_bytes(count) + (2 * count + 2) * (int64_t)sizeof(float);
}

static int check_ws(const void* ws, int64_t ws_bytes, int64_t count) {
    if (!ws || ((uintptr_t)ws & 7)) return DENET_E_BADARG;
    return ws_bytes < denet_opt_workspace(count) ? DENET_E_WORKSPACE : DENET_OK;
}

extern "C" int denet_grad_norm(const denet_opt_tensor_t* tensors, int64_t count, double max_norm, float* norm, float* coef, void* ws,
                               int64_t ws_bytes, void* stream) {
    int rc = check_grads(tensors, count);
    if (rc == DENET_OK) rc = check_ws(ws, ws_bytes, count);
    if (rc != DENET_OK) return rc;
    if (!norm || (coef && !(max_norm >= 0.))) return DENET_E_BADARG;
    int parts = 0;
    rc = launch_sumsq(tensors, count, (double*)ws, (hipStream_t)stream, &parts);
    if (rc != DENET_OK) return rc;
    hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(OPT_THREADS), 0, (hipStream_t)stream,
                       ClipArgs{(const double*)ws, max_norm, norm, coef, parts});
    DENET_CHECK_LAUNCH();
    return DENET_OK;
}

extern "C" int denet_grad_clip(const denet_opt_tensor_t* tensors, int64_t count, double max_norm, float* norm, void* ws,
                               int64_t ws_bytes, void* stream) {
    int rc = check_grads(tensors, count);
    if (rc == DENET_OK) rc = check_ws(ws, ws_bytes, count);
    if (rc != DENET_OK) return rc;
    if (!norm || !(max_norm >= 0.)) return DENET_E_BADARG;
    hipStream_t st = (hipStream_t)stream;
    int parts = 0;
    rc = launch_sumsq(tensors, count, (double*)ws, st, &parts);
    if (rc != DENET_OK) return rc;
    if (!parts) return denet_grad_norm(tensors, count, max_norm, norm, nullptr, ws, ws_bytes, stream);      // nothing but empty tensors: norm 0
    ScaleArgs a;
    a.clip = {(const double*)ws, max_norm, norm, nullptr, parts};
    a.count = 0;
    a.first_launch = 1;
    int chunks = 0;
    for (int64_t i = 0; i <= count; ++i) {
        if (a.count == OPT_SLOTS || (i == count && a.count)) {
            hipLaunchKernelGGL(grad_scale_kernel, dim3((unsigned)chunks), dim3(OPT_THREADS), 0, st, a);
            DENET_CHECK_LAUNCH();
            a.first_launch = a.count = chunks = 0;
        }
        if (i == count || tensors[i].n == 0) continue;
        a.start[a.count] = chunks;
        a.slot[a.count] = {tensors[i].grad, tensors[i].n | ((int64_t)(tensors[i].grad_dtype == DENET_BF16) << 60)};
        chunks += (int)chunks_of(tensors[i].n, SCALE_CHUNK);
        ++a.count;
    }
    return DENET_OK;
}

static bool bad_tensor(const denet_opt_tensor_t& t, int bits, bool host_steps) {
    if (bad_grad(t) || (t.param_dtype != DENET_F32 && t.param_dtype != DENET_BF16)) return true;
    if (t.n == 0) return false;
    if (host_steps ? t.step < 1 : !t.step_dev || ((uintptr_t)t.step_dev & 7)) return true;
    if (!t.param || !t.exp_avg || !t.exp_avg_sq || ((uintptr_t)t.param & (t.param_dtype == DENET_F32 ? 3 : 1))) return true;
    if (((uintptr_t)t.exp_avg & 3) || ((uintptr_t)t.exp_avg_sq & 3)) return true;
    return bits == 8 && (!t.avg_scale || !t.sq_scale || ((uintptr_t)t.avg_scale & 3) || ((uintptr_t)t.sq_scale & 3));
}

extern "C" int denet_adamw_step(const denet_opt_tensor_t* tensors, int64_t count, int bits, const denet_adamw_t* h, float* norm,
                                void* ws, int64_t ws_bytes, void* stream) {
    if (!h || (bits != 32 && bits != 8)) return DENET_E_BADARG;
    if (!(h->lr >= 0.) || !(h->beta1 >= 0. && h->beta1 < 1.) || !(h->beta2 >= 0. && h->beta2 < 1.) || !(h->eps >= 0.) ||
        !(h->weight_decay >= 0.)) return DENET_E_BADARG;
    int rc = check_grads(tensors, count);
    if (rc != DENET_OK) return rc;
    for (int64_t i = 0; i < count; ++i)
        if (bad_tensor(tensors[i], bits, !h->device_steps)) return DENET_E_BADARG;
    if (h->max_norm != h->max_norm) return DENET_E_BADARG;
    const bool clip = h->max_norm >= 0.;
    if (clip || h->device_steps) {
        rc = check_ws(ws, ws_bytes, count);
        if (rc != DENET_OK) return rc;
    }
    if (clip && !norm) return DENET_E_BADARG;
    if ((h->lr_dev && !h->device_steps) || (clip && h->coef)) return DENET_E_BADARG;
    hipStream_t st = (hipStream_t)stream;
    AdamArgs a;
    a.clip = {nullptr, 0., nullptr, nullptr, 0};
    a.coef = h->coef;
    if (clip) {
        int parts = 0;
        rc = launch_sumsq(tensors, count, (double*)ws, st, &parts);
        if (rc != DENET_OK) return rc;
        if (!parts) {
            rc = denet_grad_norm(tensors, count, h->max_norm, norm, nullptr, ws, ws_bytes, stream);
            if (rc != DENET_OK) return rc;
        }
        a.clip = {(const double*)ws, h->max_norm, norm, nullptr, parts};
    }
    a.clock = nullptr;
    if (h->device_steps) {
        ClockArgs k;
        k.lr = h->lr; k.wd = h->weight_decay; k.b1 = h->beta1; k.b2 = h->beta2;
        k.lr_dev = h->lr_dev;
        k.clock = (float*)((char*)ws + part_bytes(count));
        for (int64_t i = 0; i < count; i += CLOCK_SLOTS) {
            k.base = (int)i;
            k.count = (int)(count - i < CLOCK_SLOTS ? count - i : CLOCK_SLOTS);
            for (int j = 0; j < k.count; ++j) k.steps[j] = tensors[i + j].n ? tensors[i + j].step_dev : nullptr;
            hipLaunchKernelGGL(adamw_clock_kernel, dim3(1), dim3(OPT_THREADS), 0, st, k);
            DENET_CHECK_LAUNCH();
        }
        a.clock = k.clock;
    }
    a.decay = (float)(1. - h->lr * h->weight_decay);
    a.b1 = (float)h->beta1;
    a.c1 = (float)(1. - h->beta1);
    a.b2 = (float)h->beta2;
    a.c2 = (float)(1. - h->beta2);
    a.eps = (float)h->eps;
    a.count = 0;
    a.first_launch = 1;
    int chunks = 0;
    int64_t t_last = 0;
    float step_size = 0.f, inv_bc2 = 0.f;
    for (int64_t i = 0; i <= count; ++i) {
        if (a.count == ADAM_SLOTS || (i == count && a.count)) {
            if (bits == 8) hipLaunchKernelGGL(adamw_kernel<8>, dim3((unsigned)chunks), dim3(OPT_THREADS), 0, st, a);
            else hipLaunchKernelGGL(adamw_kernel<32>, dim3((unsigned)chunks), dim3(OPT_THREADS), 0, st, a);
            DENET_CHECK_LAUNCH();
            a.first_launch = a.count = chunks = 0;
        }
        if (i == count || tensors[i].n == 0) continue;
        const denet_opt_tensor_t& t = tensors[i];
        if (!h->device_steps && t.step != t_last) {
            t_last = t.step;
            step_size = (float)(h->lr / (1. - pow(h->beta1, (double)t.step)));
            inv_bc2 = (float)(1. / sqrt(1. - pow(h->beta2, (double)t.step)));
        }
        a.start[a.count] = chunks;
        a.slot[a.count] = {t.param, t.grad, t.exp_avg, t.exp_avg_sq, t.avg_scale, t.sq_scale,
                           t.n | ((int64_t)(t.param_dtype == DENET_BF16) << 60) | ((int64_t)(t.grad_dtype == DENET_BF16) << 61),
                           step_size, inv_bc2, (int)i};
        chunks += (int)chunks_of(t.n, ADAM_CHUNK);
        ++a.count;
    }
    return DENET_OK;
}
