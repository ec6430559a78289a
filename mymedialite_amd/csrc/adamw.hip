// adamw.hip -- one AdamW step over the parameter tensors of a model (mml_adamw_step_device).
//
//   t <- t + 1
//   m <- beta1 m + (1 - beta1) g,   v <- beta2 v + (1 - beta2) g^2
//   p <- p - lr wd p - lr m / (1 - beta1^t) / (sqrt(v / (1 - beta2^t)) + eps)
//
// The moments are held in 32 bits, or in 8: blocks of 256 consecutive values of a tensor share one
// f32 scale = (largest magnitude) / 448 and every value is the e4m3 code of value / scale, rounded
// to nearest even.  The second moment is held as its root r = sqrt(v): e4m3 spans a factor of
// 2^17.8 in normal and subnormal values, for r a factor of 2^35 in v, and the step divides by r.  A
// root that is not zero never rounds to code 0 (it takes the smallest, 2^-9): a zero under a moment
// that is not zero would turn the step into m / eps.
//
// Codes alone do not follow the recurrences: a step moves a root by (1 - beta2) / 2 or so, 0.05 %, and
// half a code's spacing is 3 to 6 %, so rounding to nearest gives the old code back and the change is
// lost (over 5,000 steps roots up to 9 times too large and 2 times too small; first moments 1.5 times
// too large under a steady gradient).  So what a code leaves of its value, within half a spacing
// either way, is kept in a byte that both moments share (a caller may leave it out, to go on from a
// state of codes and scales alone): 3 bits for m in sixths of a spacing, 5 for the root in thirtieths.
// That is rounded with a dither, the fraction of a multiple of the golden ratio that goes with step and
// place, so that changes of less than a unit arrive on average; the same step gives the same bits.  Over 5,000 steps of steady, sparse, rising and falling gradients (beta2 = 0.999)
// roots then lie within 0.93 and 1.07 of theirs, 0.89 and 1.09 where half a block's gradients stop, first
// moments within 1.3 % of their size.
//
// Memory-bound: an f32 parameter takes 28 bytes with 32-bit moments (p, m, v read and written, g
// read), 18.06 with 8-bit ones, 16.06 without the rests.  71.5 M f32 values take 400, 267 and 231 us: 5.0,
// 4.8 and 5.0 TB/s (a large copy: 4.7).  With bf16 parameters 8-bit moments are bound by the vector
// instructions, some 100 a value with the rests: 232 us, 167 without (862 and 719 MB).  Small models take
// the 8 us of a launch.  One launch covers up to kMaxTensors tensors, whose addresses are kernel arguments
// (a captured graph replays with them); the step count lives on the device, so a replay counts on.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "mml_device.h"
#include "mml_internal.h"

namespace {

constexpr int kBlock = MML_ADAMW_BLOCK;  // values per scale
// Values per block of threads and turn: 2 groups of 4 a thread with 32-bit moments, 1 with 8-bit
// ones, whose arithmetic wants the waves instead (8 a SIMD; 71.5 M f32 values: 267 us against 320 with
// 5 to 7 waves, though 5 of a wave's registers are spilled; 64 M f32 values with 32-bit moments: 354 us
// with 2 groups, 367 with 1).
template <int BITS>
constexpr int kGroupsOf4 = BITS == 32 ? 2 : 1;
template <int BITS>
constexpr int kChunk = 1024 * kGroupsOf4<BITS>;
constexpr int kMaxTensors = 48;          // 80 bytes each: under the 4 KB of kernel arguments
constexpr float kPerMax = 1.0f / 448.0f;   // the largest e4m3 value
constexpr float kE4m3Min = 0.001953125f;   // the smallest that is not zero, 2^-9

constexpr int kGroups = 32, kLine = 32;  // 128-byte lines
static_assert(MML_ADAMW_STATE == kLine * (1 + kGroups), "step_state");

struct Tensor {
    void* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;
    uint8_t* rest;
    int64_t n;
    int64_t chunk0;  // the tensor's first chunk in the launch
    int16_t p_type, g_type;
    int32_t vec4;    // every array can be read and written 4 values at a time
};

struct Step {
    Tensor t[kMaxTensors];
    int64_t chunks;
    int32_t n_tensors, last;  // last: this launch ends the step (counts it)
    double lr, beta1, beta2, eps, decay;
    double log1, log2;  // log2 of the betas
    int32_t* state;  // [0] steps done, [1] groups that are through, [kLine (1 + g)] group g's blocks
};
static_assert(sizeof(Step) <= 4096, "kernel arguments");

__device__ __forceinline__ float load_as(const void* p, int type, int64_t i) {
    if (type == MML_DTYPE_F32) return ((const float*)p)[i];
    if (type == MML_DTYPE_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    return (float)((const _Float16*)p)[i];
}
__device__ __forceinline__ void store_as(void* p, int type, int64_t i, float x) {
    if (type == MML_DTYPE_F32) {
        ((float*)p)[i] = x;
    } else if (type == MML_DTYPE_BF16) {  // the parameter's one rounding, to nearest even
        const uint32_t b = __float_as_uint(x);
        ((uint16_t*)p)[i] = x != x ? 0x7FC0u : (uint16_t)((b + 0x7FFFu + ((b >> 16) & 1u)) >> 16);
    } else {
        ((_Float16*)p)[i] = (_Float16)x;
    }
}

using f32x4 = __attribute__((ext_vector_type(4))) float;
// Four values at i (a multiple of 4 from an aligned start)
__device__ __forceinline__ f32x4 load4(const void* p, int type, int64_t i) {
    if (type == MML_DTYPE_F32) return *(const f32x4*)((const float*)p + i);
    const uint2 q = *(const uint2*)((const uint16_t*)p + i);
    const uint32_t w[4] = {q.x & 0xFFFFu, q.x >> 16, q.y & 0xFFFFu, q.y >> 16};
    f32x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        x[e] = type == MML_DTYPE_BF16 ? __uint_as_float(w[e] << 16)
                                      : (float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
    return x;
}
__device__ __forceinline__ void store4(void* p, int type, int64_t i, f32x4 x) {
    if (type == MML_DTYPE_F32) {
        *(f32x4*)((float*)p + i) = x;
        return;
    }
    // one rounding each, to nearest even, two at a time
    using bf16x4 = __attribute__((ext_vector_type(4))) __bf16;
    using f16x4 = __attribute__((ext_vector_type(4))) _Float16;
    *(uint2*)((uint16_t*)p + i) =
        type == MML_DTYPE_BF16 ? __builtin_bit_cast(uint2, __builtin_convertvector(x, bf16x4))
                               : __builtin_bit_cast(uint2, __builtin_convertvector(x, f16x4));
}

// The update of one value; m and v come and go in f32.
struct Factors {
    float beta1, one1, beta2, one2, shrink, rate, root2, eps;
};
__device__ __forceinline__ void moments(const Factors& f, float g, float& m, float& v) {
    m = fmaf(f.one1, g, f.beta1 * m);
    v = fmaf(f.one2, g * g, f.beta2 * v);
}
// A square root rounded as sqrtf's from the reciprocal root in fewer instructions: one step of
// Goldschmidt's iteration for both sqrt(v) and 1 / (2 sqrt(v)), then the remainder (Markstein 2004).  For
// v from 2^-96 on (no term underflows).
__device__ __forceinline__ float normal_root(float v) {
    const float y = __builtin_amdgcn_rsqf(v);
    float g = v * y, h = 0.5f * y;
    const float r = fmaf(-h, g, 0.5f);
    g = fmaf(g, r, g);
    h = fmaf(h, r, h);
    return fmaf(fmaf(-g, g, v), h, g);
}
__device__ __forceinline__ float step_of(const Factors& f, float p, float m, float root) {
    // (the reciprocal is off by one unit in the last place of the step, which p rounds away)
    return fmaf(-f.rate, m * __builtin_amdgcn_rcpf(fmaf(root, f.root2, f.eps)), p * f.shrink);
}

__device__ __forceinline__ float decode(uint8_t c) {
    return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}
// value / scale as e4m3, to nearest even; not finite: the NaN code
__device__ __forceinline__ float quotient(float x, float scale) {
    return scale > 0.0f ? x / scale : 0.0f;
}
__device__ __forceinline__ uint8_t encode(float x, float scale) {
    if (!(fabsf(x) < INFINITY)) return 0x7F;
    return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(quotient(x, scale), 0.0f, 0, false) & 0xFF);
}
// A block's scale from its largest magnitude.  Not below the smallest normal number: a subnormal
// quotient is rounded by up to half of itself, and largest / scale would pass 464, from where on the
// conversion gives the NaN code.  (A first moment without gradients decays that far in 800 steps.)
__device__ __forceinline__ float scale_of(float largest) {
    return largest > 0.0f ? fmaxf(largest * kPerMax, 0x1p-126f) : 0.0f;
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.0f;  // (NaN too)
}

// The largest of a wave's values, in every lane: within rows of 16 by DPP, across them by the swaps.
// Magnitudes as their bits, which order as they do, with infinity and the NaNs above.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    const auto dpp = [](uint32_t v, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, 0xF, 0xF, true);
    };
    x = max(x, dpp(x, std::integral_constant<int, 0xB1>{}));   // quad_perm 1 0 3 2
    x = max(x, dpp(x, std::integral_constant<int, 0x4E>{}));   // quad_perm 2 3 0 1
    x = max(x, dpp(x, std::integral_constant<int, 0x141>{}));  // row_half_mirror
    x = max(x, dpp(x, std::integral_constant<int, 0x140>{}));  // row_mirror
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(b[0], b[1]);
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
constexpr uint32_t kInfinity = 0x7F800000u;
// What a code leaves.  8 spacings of the e4m3 numbers at a code's value d (under 2^-6 the subnormal
// ones'), and the value that a code and its rest stand for
__device__ __forceinline__ float spacings8(float d) {
    return __uint_as_float(max(__float_as_uint(d) & kInfinity, 121u << 23));
}
constexpr int kUnitsM = 6, kUnitsV = 30;  // units of the rests in a spacing: -3 .. 3 and -15 .. 15
template <int UNITS>
__device__ __forceinline__ float with_rest(float d, int32_t rest) {
    return fmaf((float)rest * (0.125f / UNITS), spacings8(d), d);
}
// The rest of the quotient q (value / scale) whose code stands for d, plus `bias` (so that cutting off
// rounds down); dither 0 .. 255 in 256ths of a unit and half a 256th more, which is 1/2 on average and
// under 1, so that what is a code's value exactly, 0 above all, stays it.  (The NaN code's rest does not
// matter.)
template <int UNITS>
__device__ __forceinline__ uint32_t rest_of(float q, float d, float dither, int bias) {
    const float units = __uint_as_float((254u << 23) - __float_as_uint(spacings8(d))) * (8.0f * UNITS);
    const int32_t r = (int32_t)fmaf(dither, 0x1p-8f, fmaf(q - d, units, (float)bias + 0x1p-9f));
    return (uint32_t)min(max(r, bias - UNITS / 2), bias + UNITS / 2);
}
// Both rests in a byte, m's in the low 3 bits, as two's complements.  Packed with biases of 4 and 16, whose
// removal is an exclusive or with kBiases.
constexpr int kBiasM = 4, kBiasV = 16;
constexpr uint32_t kBiases = 0x84848484u;
__device__ __forceinline__ uint32_t biased_rests(float qm, float dm, float qv, float dv, float dither) {
    return rest_of<kUnitsM>(qm, dm, dither, kBiasM) | rest_of<kUnitsV>(qv, dv, dither, kBiasV) << 3;
}
__device__ __forceinline__ int32_t rest_m(uint32_t byte) { return __builtin_amdgcn_sbfe((int)byte, 0, 3); }
__device__ __forceinline__ int32_t rest_v(uint32_t byte) { return __builtin_amdgcn_sbfe((int)byte, 3, 5); }
// Steps that leave no rest: v is the sum of so few terms then that a term moves it by a code's
// spacing or more, and codes and scales alone are the state of a run that short.
constexpr int kBareSteps = 4;
// The dithers of four values from the i-th on (a multiple of 4), a byte each: multiples of the golden
// ratio and of another fraction by step and place, as fractions of 2^32, whose bytes each run through all
// values.
__device__ __forceinline__ uint32_t dithers_at(int32_t step, int64_t i) {
    return (uint32_t)step * 0x9E3779B9u + (uint32_t)(i >> 2) * 0x85EBCA6Bu;
}

// Four finite values / scale as codes.  The quotients are rounded as a division rounds them: one
// division for the block's reciprocal y, then q = x y corrected by its remainder (Markstein 1990).
// Scales under 2^-100 are divided by.
__device__ __forceinline__ uint32_t encode4(const f32x4 x, float scale, float y, f32x4& q) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float z = x[e] * y;
        q[e] = fmaf(fmaf(-z, scale, x[e]), y, z);
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}
__device__ __forceinline__ f32x4 decode4(uint32_t w) {
    return f32x4{__builtin_amdgcn_cvt_f32_fp8((int)w, 0), __builtin_amdgcn_cvt_f32_fp8((int)w, 1),
                 __builtin_amdgcn_cvt_f32_fp8((int)w, 2), __builtin_amdgcn_cvt_f32_fp8((int)w, 3)};
}

template <int BITS, bool REST>
__global__ __launch_bounds__(256, BITS == 32 ? 1 : 8) void adamw_kernel(Step s) {
    constexpr int NU = kGroupsOf4<BITS>;
    const int t = threadIdx.x;
    const int32_t step = s.state[0] + 1;
    Factors f;
    bool ready = false;
    const auto prepare = [&] {  // behind the first chunk's loads
        if (ready) return;
        ready = true;
        // in 64 bits: 1 - beta and 1 - beta^t cancel for a beta near 1
        const double c1 = 1.0 - exp2(s.log1 * step);
        const double c2 = 1.0 - exp2(s.log2 * step);
        f.beta1 = (float)s.beta1;
        f.one1 = (float)(1.0 - s.beta1);
        f.beta2 = (float)s.beta2;
        f.one2 = (float)(1.0 - s.beta2);
        f.shrink = (float)(1.0 - s.lr * s.decay);
        f.rate = (float)(s.lr / c1);
        f.root2 = (float)(1.0 / sqrt(c2));
        f.eps = (float)s.eps;
    };
    int at = 0;
    for (int64_t c = blockIdx.x; c < s.chunks; c += gridDim.x) {
        while (at + 1 < s.n_tensors && c >= s.t[at + 1].chunk0) ++at;
        const Tensor& q = s.t[at];
        const int64_t base = (c - q.chunk0) * kChunk<BITS>;
        if (q.vec4 && base + kChunk<BITS> <= q.n) {  // a whole chunk
            f32x4 p[NU], g[NU], m[NU], v[NU];
            int64_t at[NU];
            uint32_t mq[NU], vq[NU], rq[NU] = {};
            float ms[NU], vs[NU];
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                // 8 bits: a wave's 256 values are a block
                at[u] = base + (BITS == 32 ? u * 1024 + 4 * t
                                           : ((t >> 6) * NU + u) * kBlock + 4 * (t & 63));
                p[u] = load4(q.p, q.p_type, at[u]);
                g[u] = load4(q.g, q.g_type, at[u]);
                if constexpr (BITS == 32) {
                    m[u] = *(const f32x4*)((const float*)q.m + at[u]);
                    v[u] = *(const f32x4*)((const float*)q.v + at[u]);
                } else {
                    mq[u] = *(const uint32_t*)((const uint8_t*)q.m + at[u]);
                    vq[u] = *(const uint32_t*)((const uint8_t*)q.v + at[u]);
                    if (REST) rq[u] = *(const uint32_t*)(q.rest + at[u]);
                    // (the same in all lanes: a scalar load)
                    const int64_t b = base / kBlock +
                                      __builtin_amdgcn_readfirstlane((t >> 6) * NU + u);
                    ms[u] = q.ms[b];
                    vs[u] = q.vs[b];
                }
            }
            prepare();
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                f32x4 r;
                if constexpr (BITS == 8) {
                    f32x4 dm = decode4(mq[u]), dv = decode4(vq[u]);
                    if constexpr (REST)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            dm[e] = with_rest<kUnitsM>(dm[e], rest_m(rq[u] >> (8 * e)));
                            dv[e] = with_rest<kUnitsV>(dv[e], rest_v(rq[u] >> (8 * e)));
                        }
                    m[u] = dm * ms[u];
                    const f32x4 root = dv * vs[u];
                    v[u] = root * root;
                }
                bool small = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float me = m[u][e], ve = v[u][e];
                    moments(f, g[u][e], me, ve);
                    m[u][e] = me;
                    v[u][e] = ve;
                    small = small || !(ve >= 0x1p-96f && ve < INFINITY);
                }
                if (__any(small)) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[e] = sqrtf(v[u][e]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[e] = normal_root(v[u][e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) p[u][e] = step_of(f, p[u][e], m[u][e], r[e]);
                store4(q.p, q.p_type, at[u], p[u]);
                if constexpr (BITS == 32) {
                    *(f32x4*)((float*)q.m + at[u]) = m[u];
                    *(f32x4*)((float*)q.v + at[u]) = v[u];
                } else {
                    uint32_t am = 0, ar = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        am = max(am, magnitude(m[u][e]));
                        ar = max(ar, magnitude(r[e]));
                    }
                    am = wave_max(am);
                    ar = wave_max(ar);
                    const bool odd = am >= kInfinity || ar >= kInfinity;  // in all lanes
                    if (odd) {  // the largest of the finite values
                        am = ar = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            am = max(am, magnitude(finite_abs(m[u][e])));
                            ar = max(ar, magnitude(finite_abs(r[e])));
                        }
                        am = wave_max(am);
                        ar = wave_max(ar);
                    }
                    const float nm = scale_of(__uint_as_float(am)), nr = scale_of(__uint_as_float(ar));
                    uint32_t cm, cv;
                    f32x4 qm, qr;  // the quotients
                    if (odd || !(nm > 0x1p-100f) || !(nr > 0x1p-100f)) {
                        const float least = kE4m3Min * nr;
                        cm = cv = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float root = r[e] > 0.0f && r[e] < least ? least : r[e];
                            cm |= (uint32_t)encode(m[u][e], nm) << (8 * e);
                            cv |= (uint32_t)encode(root, nr) << (8 * e);
                            qm[e] = quotient(m[u][e], nm);
                            qr[e] = quotient(r[e], nr);
                        }
                    } else {
                        cm = encode4(m[u], nm, 1.0f / nm, qm);
                        // code 1 at least for a root that is not zero (the codes of roots are < 128)
                        const uint32_t c = encode4(r, nr, 1.0f / nr, qr);
                        cv = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            cv |= max(c >> (8 * e) & 0xFFu, r[e] > 0.0f ? 1u : 0u) << (8 * e);
                    }
                    *(uint32_t*)((uint8_t*)q.m + at[u]) = cm;
                    *(uint32_t*)((uint8_t*)q.v + at[u]) = cv;
                    uint32_t rests = 0;
                    if (REST && step > kBareSteps) {
                        const f32x4 dm = decode4(cm), dv = decode4(cv);
                        const uint32_t dithers = dithers_at(step, at[u]);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            rests |= biased_rests(qm[e], dm[e], qr[e], dv[e],
                                                  (float)(dithers >> (8 * e) & 0xFFu)) << (8 * e);
                        rests ^= kBiases;
                    }
                    if (REST) *(uint32_t*)(q.rest + at[u]) = rests;
                    if ((t & 63) == 0) {
                        q.ms[at[u] / kBlock] = nm;
                        q.vs[at[u] / kBlock] = nr;
                    }
                }
            }
        } else if constexpr (BITS == 32) {
            prepare();
            for (int x = t; x < kChunk<BITS>; x += 256) {
                const int64_t i = base + x;
                if (i >= q.n) break;
                float m = ((float*)q.m)[i], v = ((float*)q.v)[i], root;
                moments(f, load_as(q.g, q.g_type, i), m, v);
                root = sqrtf(v);
                const float p = step_of(f, load_as(q.p, q.p_type, i), m, root);
                ((float*)q.m)[i] = m;
                ((float*)q.v)[i] = v;
                store_as(q.p, q.p_type, i, p);
            }
        } else {
            prepare();
            // a wave per block of 256: lane l holds values l, l + 64, l + 128, l + 192
            for (int blk = t >> 6; blk < kChunk<BITS> / kBlock; blk += 4) {
                const int64_t b0 = base + blk * kBlock;
                if (b0 >= q.n) break;
                const int64_t scale_at = b0 / kBlock;
                const float ms = q.ms[scale_at], vs = q.vs[scale_at];
                float m[4], r[4], am = 0.0f, ar = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t i = b0 + e * 64 + (t & 63);
                    m[e] = r[e] = 0.0f;
                    if (i < q.n) {
                        const uint32_t rest = REST ? q.rest[i] : 0;
                        m[e] = with_rest<kUnitsM>(decode(((uint8_t*)q.m)[i]), rest_m(rest)) * ms;
                        const float root =
                            with_rest<kUnitsV>(decode(((uint8_t*)q.v)[i]), rest_v(rest)) * vs;
                        float v = root * root;
                        moments(f, load_as(q.g, q.g_type, i), m[e], v);
                        r[e] = sqrtf(v);
                        const float p = step_of(f, load_as(q.p, q.p_type, i), m[e], r[e]);
                        store_as(q.p, q.p_type, i, p);
                        am = fmaxf(am, finite_abs(m[e]));
                        ar = fmaxf(ar, finite_abs(r[e]));
                    }
                }
#pragma unroll
                for (int d = 32; d > 0; d >>= 1) {
                    am = fmaxf(am, __shfl_xor(am, d));
                    ar = fmaxf(ar, __shfl_xor(ar, d));
                }
                const float nm = scale_of(am), nr = scale_of(ar);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t i = b0 + e * 64 + (t & 63);
                    if (i < q.n) {
                        const float least = kE4m3Min * nr;
                        const uint8_t cm = encode(m[e], nm);
                        const uint8_t cv = encode(r[e] > 0.0f && r[e] < least ? least : r[e], nr);
                        const float dither =
                            (float)(dithers_at(step, i) >> (8 * (int)(i & 3)) & 0xFFu);
                        ((uint8_t*)q.m)[i] = cm;
                        ((uint8_t*)q.v)[i] = cv;
                        if (REST)
                            q.rest[i] = step <= kBareSteps ? 0 : (uint8_t)(
                                biased_rests(quotient(m[e], nm), decode(cm), quotient(r[e], nr),
                                             decode(cv), dither) ^ kBiases);
                    }
                }
                if ((t & 63) == 0) {
                    q.ms[scale_at] = nm;
                    q.vs[scale_at] = nr;
                }
            }
        }
    }
    // The last block through counts the step: every block has read the count by then, which is all the
    // order there is, so the arrivals are relaxed (a fence here would write the XCD's L2 back once a
    // block: 80 us of 105 at 7 M values).  They arrive at kGroups counters, in lines of their own, and
    // the groups' last at one: arrivals at one address take 11.5 ns each, 23 us for 2,048 blocks.
    if (!s.last) return;
    __syncthreads();
    if (t == 0) {
        const int groups = min((int)gridDim.x, kGroups), g = blockIdx.x % groups;
        const int members = ((int)gridDim.x - g + groups - 1) / groups;
        const auto arrive = [](int32_t* at) {
            return __hip_atomic_fetch_add(at, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        };
        int32_t* mine = s.state + kLine * (1 + g);
        if (arrive(mine) == members - 1) {
            *mine = 0;
            if (arrive(s.state + 1) == groups - 1) {
                s.state[0] = step;
                s.state[1] = 0;
            }
        }
    }
}

void check_tensor(const mml_adamw_tensor& x, int32_t bits) {
    MML_REQUIRE(x.n >= 0, "a tensor's size is negative");
    MML_REQUIRE(x.param_dtype >= MML_DTYPE_F32 && x.param_dtype <= MML_DTYPE_F16 &&
                    x.grad_dtype >= MML_DTYPE_F32 && x.grad_dtype <= MML_DTYPE_F16,
                "unknown dtype");
    if (x.n == 0) return;
    MML_REQUIRE(x.param && x.grad && x.m && x.v, "a tensor's pointer is null");
    MML_REQUIRE(bits == 32 || (x.m_scale && x.v_scale), "8-bit moments without their scales");
}

}  // namespace

extern "C" mml_status mml_adamw_step_device(const mml_adamw_tensor* tensors, int32_t n_tensors,
                                            const mml_adamw_params* params, int32_t* step_state,
                                            int32_t device, void* stream) {
    return mml::guard([&] {
        MML_REQUIRE(params, "params is null");
        MML_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || tensors), "tensors is null");
        MML_REQUIRE(step_state, "step_state is null");
        const mml_adamw_params& a = *params;
        MML_REQUIRE(a.state_bits == 8 || a.state_bits == 32, "state_bits must be 8 or 32");
        MML_REQUIRE(a.learn_rate >= 0.0 && a.learn_rate < INFINITY && a.epsilon >= 0.0 &&
                        a.epsilon < INFINITY && a.weight_decay >= 0.0 && a.weight_decay < INFINITY,
                    "learn_rate, epsilon and weight_decay must be finite and not negative");
        MML_REQUIRE(a.beta1 >= 0.0 && a.beta1 < 1.0 && a.beta2 >= 0.0 && a.beta2 < 1.0,
                    "beta1 and beta2 must be in [0, 1)");
        int32_t sized = 0, with_rest = 0;
        for (int32_t i = 0; i < n_tensors; ++i) {
            check_tensor(tensors[i], a.state_bits);
            sized += tensors[i].n > 0;
            with_rest += tensors[i].n > 0 && tensors[i].rest;
        }
        MML_REQUIRE(a.state_bits == 32 || with_rest == 0 || with_rest == sized,
                    "rests of some tensors only");
        mml::DeviceScope on(device);
        Step s{};
        s.lr = a.learn_rate;
        s.beta1 = a.beta1;
        s.beta2 = a.beta2;
        s.eps = a.epsilon;
        s.decay = a.weight_decay;
        s.log1 = std::log2(a.beta1);
        s.log2 = std::log2(a.beta2);
        s.state = step_state;
        int32_t i = 0;
        do {
            s.n_tensors = 0;
            s.chunks = 0;
            for (; i < n_tensors && s.n_tensors < kMaxTensors; ++i) {
                const mml_adamw_tensor& x = tensors[i];
                if (x.n == 0) continue;
                const auto aligned = [](const void* q, size_t bytes) {
                    return (uintptr_t)q % bytes == 0;
                };
                const size_t moment = a.state_bits == 32 ? 16 : 4;
                const bool vec4 = aligned(x.param, x.param_dtype == MML_DTYPE_F32 ? 16 : 8) &&
                                  aligned(x.grad, x.grad_dtype == MML_DTYPE_F32 ? 16 : 8) &&
                                  aligned(x.m, moment) && aligned(x.v, moment) &&
                                  aligned(x.rest, 4);
                s.t[s.n_tensors++] = Tensor{x.param, x.grad, x.m, x.v, x.m_scale, x.v_scale, x.rest,
                                            x.n, s.chunks, (int16_t)x.param_dtype,
                                            (int16_t)x.grad_dtype, vec4};
                const int64_t chunk = a.state_bits == 32 ? kChunk<32> : kChunk<8>;
                s.chunks += (x.n + chunk - 1) / chunk;
            }
            s.last = i == n_tensors;
            const uint32_t blocks = (uint32_t)std::max<int64_t>(1, std::min<int64_t>(s.chunks, 2048));
            if (a.state_bits == 32)
                adamw_kernel<32, false><<<blocks, 256, 0, (hipStream_t)stream>>>(s);
            else if (with_rest)
                adamw_kernel<8, true><<<blocks, 256, 0, (hipStream_t)stream>>>(s);
            else
                adamw_kernel<8, false><<<blocks, 256, 0, (hipStream_t)stream>>>(s);
            MML_HIP(hipGetLastError());
        } while (i < n_tensors);
    });
}
