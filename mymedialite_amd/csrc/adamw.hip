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
// Memory-bound: an f32 parameter takes 28 bytes with 32-bit moments (p, m, v read and written, g
// read), 16.06 with 8-bit ones.  One launch covers up to kMaxTensors tensors, whose addresses are
// kernel arguments (a captured graph replays with them); the step count lives on the device, so a
// replay counts on.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "mml_device.h"
#include "mml_internal.h"

namespace {

constexpr int kBlock = MML_ADAMW_BLOCK;  // values per scale
constexpr int kChunk = 2048;             // values per block of threads and turn
constexpr int kMaxTensors = 40;          // 72 bytes each: under the 4 KB of kernel arguments
constexpr float kPerMax = 1.0f / 448.0f;   // the largest e4m3 value
constexpr float kE4m3Min = 0.001953125f;   // the smallest that is not zero, 2^-9

struct Tensor {
    void* p;
    const void* g;
    void *m, *v;
    float *ms, *vs;
    int64_t n;
    int64_t chunk0;  // the tensor's first chunk in the launch
    int32_t p_type, g_type;
};

struct Step {
    Tensor t[kMaxTensors];
    int64_t chunks;
    int32_t n_tensors, last;  // last: this launch ends the step (counts it)
    double lr, beta1, beta2, eps, decay;
    int32_t* state;  // [0] steps done, [1] blocks that are through
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

// The update of one value; m and v come and go in f32.
struct Factors {
    float beta1, one1, beta2, one2, shrink, rate, root2, eps;
};
__device__ __forceinline__ float update(const Factors& f, float p, float g, float& m, float& v,
                                        float& root) {
    m = fmaf(f.one1, g, f.beta1 * m);
    v = fmaf(f.one2, g * g, f.beta2 * v);
    root = sqrtf(v);
    return fmaf(-f.rate, m / fmaf(root, f.root2, f.eps), p * f.shrink);
}

__device__ __forceinline__ float decode(uint8_t c) {
    return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}
// value / scale as e4m3, to nearest even; not finite: the NaN code
__device__ __forceinline__ uint8_t encode(float x, float scale) {
    if (!(fabsf(x) < INFINITY)) return 0x7F;
    return scale > 0.0f ? (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(x / scale, 0.0f, 0, false) & 0xFF)
                        : 0;
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.0f;  // (NaN too)
}

template <int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(Step s) {
    const int t = threadIdx.x;
    const int32_t step = s.state[0] + 1;
    Factors f;
    {
        // in 64 bits: 1 - beta and 1 - beta^t cancel for a beta near 1
        const double c1 = 1.0 - pow(s.beta1, (double)step);
        const double c2 = 1.0 - pow(s.beta2, (double)step);
        f.beta1 = (float)s.beta1;
        f.one1 = (float)(1.0 - s.beta1);
        f.beta2 = (float)s.beta2;
        f.one2 = (float)(1.0 - s.beta2);
        f.shrink = (float)(1.0 - s.lr * s.decay);
        f.rate = (float)(s.lr / c1);
        f.root2 = (float)(1.0 / sqrt(c2));
        f.eps = (float)s.eps;
    }
    int at = 0;
    for (int64_t c = blockIdx.x; c < s.chunks; c += gridDim.x) {
        while (at + 1 < s.n_tensors && c >= s.t[at + 1].chunk0) ++at;
        const Tensor& q = s.t[at];
        const int64_t base = (c - q.chunk0) * kChunk;
        if constexpr (BITS == 32) {
            for (int x = t; x < kChunk; x += 256) {
                const int64_t i = base + x;
                if (i >= q.n) break;
                float m = ((float*)q.m)[i], v = ((float*)q.v)[i], root;
                const float p = update(f, load_as(q.p, q.p_type, i), load_as(q.g, q.g_type, i), m, v,
                                       root);
                ((float*)q.m)[i] = m;
                ((float*)q.v)[i] = v;
                store_as(q.p, q.p_type, i, p);
            }
        } else {
            // a wave per block of 256: lane l holds values l, l + 64, l + 128, l + 192
            for (int blk = t >> 6; blk < kChunk / kBlock; blk += 4) {
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
                        m[e] = decode(((uint8_t*)q.m)[i]) * ms;
                        const float root = decode(((uint8_t*)q.v)[i]) * vs;
                        float v = root * root;
                        const float p = update(f, load_as(q.p, q.p_type, i),
                                               load_as(q.g, q.g_type, i), m[e], v, r[e]);
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
                const float nm = am * kPerMax, nr = ar * kPerMax;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t i = b0 + e * 64 + (t & 63);
                    if (i < q.n) {
                        ((uint8_t*)q.m)[i] = encode(m[e], nm);
                        const float least = kE4m3Min * nr;
                        ((uint8_t*)q.v)[i] = encode(r[e] > 0.0f && r[e] < least ? least : r[e], nr);
                    }
                }
                if ((t & 63) == 0) {
                    q.ms[scale_at] = nm;
                    q.vs[scale_at] = nr;
                }
            }
        }
    }
    // The last block through counts the step: every block has read the count by then.
    if (!s.last) return;
    __syncthreads();
    if (t == 0) {
        __threadfence();
        if (atomicAdd(&s.state[1], 1) == (int)gridDim.x - 1) {
            s.state[0] = step;
            s.state[1] = 0;
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
        for (int32_t i = 0; i < n_tensors; ++i) check_tensor(tensors[i], a.state_bits);
        mml::DeviceScope on(device);
        Step s{};
        s.lr = a.learn_rate;
        s.beta1 = a.beta1;
        s.beta2 = a.beta2;
        s.eps = a.epsilon;
        s.decay = a.weight_decay;
        s.state = step_state;
        int32_t i = 0;
        do {
            s.n_tensors = 0;
            s.chunks = 0;
            for (; i < n_tensors && s.n_tensors < kMaxTensors; ++i) {
                const mml_adamw_tensor& x = tensors[i];
                if (x.n == 0) continue;
                s.t[s.n_tensors++] = Tensor{x.param, x.grad, x.m, x.v, x.m_scale, x.v_scale, x.n,
                                            s.chunks, x.param_dtype, x.grad_dtype};
                s.chunks += (x.n + kChunk - 1) / kChunk;
            }
            s.last = i == n_tensors;
            const uint32_t blocks = (uint32_t)std::max<int64_t>(1, std::min<int64_t>(s.chunks, 2048));
            if (a.state_bits == 32)
                adamw_kernel<32><<<blocks, 256, 0, (hipStream_t)stream>>>(s);
            else
                adamw_kernel<8><<<blocks, 256, 0, (hipStream_t)stream>>>(s);
            MML_HIP(hipGetLastError());
        } while (i < n_tensors);
    });
}
