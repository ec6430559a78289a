// item_softmax.hip -- the softmax over the catalogue of a matrix-factorization model: log
// probabilities of given items, the entropy, the top items (mml_item_log_probs_device) and the
// gradient of a loss on them (mml_item_log_probs_grad_device).
//
// For a row r (a user) and item j:  s_rj = <U_r, V_j> + b_j,  lse_r = log sum_j exp(s_rj),
// log p_rj = s_rj - lse_r,  H_r = -sum_j p_rj log p_rj.  With w_r = dL / d log p_r(given item t_r)
// and h_r = dL / dH_r:
//   G_rj = dL / ds_rj = w_r ([j = t_r] - p_rj) - h_r p_rj (log p_rj + H_r),
//   dL/dU = G V,  dL/dV = G^T U,  dL/db_j = sum_r G_rj.
// The R x N matrices s, p and G are never stored: 32 x 32 tiles of s are made on the matrix cores,
// used in registers and dropped (one pass with a running maximum m, sum l and sum of e y).
//
// f32 factors run on the f16 matrix cores at close to f32 accuracy: a value x, scaled by a power of
// two common to its matrix (largest magnitude just under 2^13), is hi + lo with hi = f16(x) and
// lo = f16(x - hi), 22 significant bits down to 2^-16 of the matrix' largest value and 2^-38 of it
// below; a product takes lo hi + hi lo + hi hi, accumulated in f32 (the dropped lo lo is below 2^-22
// of |a b|).  v_mfma_f32_32x32x16_f16 does 1,024 flops per cycle and SIMD against 64 of the f32
// form, so three products are 5 times as fast, and twice as fast as the six products that three bf16
// planes take -- which counts doubly, since the matrix cores run into the power limit first
// (1.6 PFLOP/s on random data against 2.3 on constants).  f16 factors are one f16 plane, bf16
// factors one bf16 plane.  G is split into two planes as well: f16 under a power of two that every
// kept row adapts to the largest |G| it has met (the sums are scaled along, as a running maximum's
// are), or bf16 for bf16 factors (17 bits against the result's 8: a result differs
// from that of G in f32 where the last 2^-18 of it turns a rounding, by one step).
//
// Tile layout.  v_mfma_f32_32x32x16: A (32 x 16), lane l holds row l % 32, k = 8 (l / 32) .. + 7;
// B (16 x 32) the same with the column; C: lane l holds column l % 32, register i row
// 8 (i / 4) + 4 (l / 32) + i % 4.  The streamed side is A, the side a wave keeps is B, so a lane
// owns one row of the kept side: in the forward pass and the users' gradient one user per lane
// pair (l, l + 32) and its softmax state needs no lane exchange; in the items' gradient one item.
// The next product contracts over the streamed side.  Its B operand (16 x 32) for step s takes, in
// lane l, the C registers 8 s .. 8 s + 7 as they are when the A operand's k order is
// 16 s + 8 (e / 4) + 4 (l / 32) + e % 4, which the "transposed" fragments are laid out for.
//
// A preparation kernel writes both sides as fragments in that order (16 bytes per lane, 1 KB per
// fragment), so every operand load is a linear 1 KB.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "mml_device.h"
#include "mml_internal.h"

namespace {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f32x2 = __attribute__((ext_vector_type(2))) float;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;
// A bias of this or less excludes its item; the score of an excluded item where scores are not scaled.
// Finite, so that e * y below is 0 * finite = 0 and not 0 * inf.
constexpr float kGone = -1e30f;
constexpr int kMaxTop = 128;

// Planes of a factor type: PS of the score product, PG of the gradient product's factors, GP of G;
// HALF: the planes are f16 (else bf16).
template <int T>
struct Planes {  // bf16 and f16 factors
    static constexpr int PS = 1, PG = 1, GP = 2;
    static constexpr bool HALF = T == MML_DTYPE_F16;
};
template <>
struct Planes<MML_DTYPE_F32> {
    static constexpr int PS = 2, PG = 2, GP = 2;
    static constexpr bool HALF = true;
};

template <int T>
__device__ __forceinline__ float load_factor(const void* p, int64_t i) {
    if constexpr (T == MML_DTYPE_F32) return ((const float*)p)[i];
    if constexpr (T == MML_DTYPE_BF16) return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    if constexpr (T == MML_DTYPE_F16) return (float)((const _Float16*)p)[i];
}
// Factors at .. at + 7, in loads of 16 bytes that need no more than an element's alignment
template <int T>
__device__ __forceinline__ void load_factors(const void* p, int64_t at, float (&v)[8]) {
    using f32x4_any = __attribute__((ext_vector_type(4), aligned(4))) float;
    using u32x4_any = __attribute__((ext_vector_type(4), aligned(2))) uint32_t;
    if constexpr (T == MML_DTYPE_F32) {
        const f32x4 lo = *(const f32x4_any*)((const float*)p + at);
        const f32x4 hi = *(const f32x4_any*)((const float*)p + at + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
    } else {
        const u32x4 w = *(const u32x4_any*)((const uint16_t*)p + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t b = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
            v[e] = T == MML_DTYPE_F16 ? (float)__builtin_bit_cast(_Float16, b)
                                      : __uint_as_float((uint32_t)b << 16);
        }
    }
}
__device__ __forceinline__ uint32_t bf16_rn(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;
}
template <int T>
__device__ __forceinline__ void store_factor(void* p, int64_t i, float x) {
    if constexpr (T == MML_DTYPE_F32) ((float*)p)[i] = x;
    if constexpr (T == MML_DTYPE_BF16)  // one rounding, to nearest; a NaN stays one
        ((uint16_t*)p)[i] = x != x ? 0x7FC0u : (uint16_t)bf16_rn(x);
    if constexpr (T == MML_DTYPE_F16) ((_Float16*)p)[i] = (_Float16)x;
}

// Factors f .. f + 3 of the row at `at`: one store where the rows allow it
template <int T>
__device__ __forceinline__ void store_factors(void* p, int64_t at, int f, int k, int vec4, f32x4 x) {
    if (f >= k) return;
    if (vec4) {  // k, the stride and the base are multiples of 4 factors
        if constexpr (T == MML_DTYPE_F32) {
            *(f32x4*)((float*)p + at + f) = x;
        } else {
            uint16_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) store_factor<T>(v, e, x[e]);
            *(uint2*)((uint16_t*)p + at + f) =
                make_uint2(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (f + e < k) store_factor<T>(p, at + f + e, x[e]);
}

// ------------------------------------------------------------------ arguments of the kernels
struct Side {  // one factor matrix as fragments
    const void* src;
    int64_t ld;
    const int32_t* index;  // row x of the side is src row index[x] (nullptr: x)
    int32_t n_src;         // rows of src
    int64_t n;             // rows of the side
    int32_t tiles;         // tiles of 32 rows written (>= ceil(n / 32))
    uint4* frag;           // [tiles][PS][KT][64]
    uint4* trans;          // [tiles][PG][MT][2][64] (nullptr: not needed)
    int32_t vec8;          // the rows begin at multiples of 16 bytes
};

struct RowMeta {  // per tile of the users' side, gradient only
    float lse2[32];   // lse * log2 e; 1e30 for a row without a gradient (p = 0)
    float c0[32], c1[32];  // G = p (c0 + c1 x) + [j = t] w,  x = log2 p
    int32_t t[32];    // the given item, -1: none
};

// Powers of two that the planes are scaled by (f32 factors; otherwise 1), so scores come out of the
// matrix cores as s 2^(eu + ev), and what follows from them.  Written by the preparation.
struct Scale {
    float kappa;  // log2 e / 2^(eu + ev)
    float unit;   // 2^-(eu + ev)
    float gone;   // the score of an excluded item: below every other
    float floor;  // where a running maximum starts: above gone, so that an excluded item's e is 0
                  // before the first score too (a row whose scores are all below it counts as empty)
    int32_t eu, ev;  // of the score's planes
    int32_t gu, gv;  // of the gradient products' (transposed) planes
};
__device__ __forceinline__ Scale plain_scale() {
    return Scale{kLog2e, 1.0f, kGone, kGone * 0.0625f, 0, 0, 0, 0};
}
// 2^86: scaled scores are below 2^35, so products beyond are far outside f32; and an excluded item's
// score times kappa, 2^40 2^86, is still finite.
constexpr int kLeastExponent = -86;
constexpr int kMaxParts = 512, kUserParts = 64;  // partial maxima of largest_factors

struct Job {
    Side u, v;
    float* parts;   // [kMaxParts]: largest |factor| each: kUserParts of the users', then the items'
    Scale* scale;
    const float* bias;   // items (nullptr: 0)
    float* vbias;        // [v.tiles * 32]: bias 2^(eu + ev), scale->gone for an excluded or padding
                         // item, NaN where the factors are not finite
    uint32_t* mask;      // [rows_pad][v.tiles]: bit i of word (r, tile): item 32 tile + i excluded
    int64_t rows_pad;    // u.tiles * 32
    const int64_t* ex_off;
    const int32_t* ex_items;
    int64_t n_ex;
    const int32_t* target;
    int32_t k, n_items;
    int64_t n_rows;
    int32_t splits;
    int32_t bias_vec4;  // the bias can be loaded 4 at a time
    int32_t direct;  // forward: no preparation
    // forward
    float* part;    // [3][rows_pad][splits]: m, l, w
    float* cmax;    // [rows_pad][cpad]: every tile's largest score (n_top > 0)
    int64_t cpad;
    int32_t n_top;
    float *log_probs, *log_norm, *entropy, *top_lp;
    int32_t* top_items;
    // gradient
    const float *in_norm, *in_entropy, *g_lp, *g_ent;
    RowMeta* meta;  // [u.tiles]
    float* w;       // [rows_pad]
    float *du_part, *dv_part, *db_part;
    int32_t vsplits;  // of the item tiles from vwhole on; those before have one block each
    int32_t vwhole;
    void *gu, *gv;
    int64_t ld_gu, ld_gv;
    int32_t gu_vec4, gv_vec4;
    float* gb;
};

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) {
    return x < lo ? lo : (x > hi ? hi : x);
}
__device__ __forceinline__ int64_t source_row(const Side& s, int64_t x) {  // -1: none
    if (x >= s.n) return -1;
    const int64_t r = s.index ? (int64_t)s.index[x] : x;
    return r >= 0 && r < s.n_src ? r : -1;
}

// ------------------------------------------------------------------ preparation
// The next plane of v, to nearest; v becomes what is left
template <int T>
__device__ __forceinline__ uint32_t take_plane(float& v) {
    if constexpr (Planes<T>::HALF) {
        const _Float16 h = (_Float16)v;
        v -= (float)h;
        return (uint32_t)__builtin_bit_cast(uint16_t, h);
    } else {
        const uint32_t b = bf16_rn(v);
        v -= __uint_as_float(b << 16);
        return b;
    }
}

// The exclusion lists as bits: a block makes up to kMaskWords words of a row in LDS and writes them.  The
// lists may be unsorted and may repeat an item (an OR of bits does not depend on the order); ids
// outside the catalogue and offsets outside the array are skipped.
constexpr int kMaskWords = 16128;  // with the kernel's other 16 bytes under 64 KB
__device__ __forceinline__ void make_mask(const Job& j, uint32_t block) {
    extern __shared__ __align__(16) uint32_t words[];
    const int parts = (j.v.tiles + kMaskWords - 1) / kMaskWords;
    const int64_t r = block / parts;
    const int w0 = (int)(block % parts) * kMaskWords, n = min(kMaskWords, j.v.tiles - w0);
    for (int x = threadIdx.x; x < n; x += 256) words[x] = 0;
    const int64_t u = source_row(j.u, r);
    int64_t b = 0, e = 0;
    if (u >= 0) b = clamp64(j.ex_off[u], 0, j.n_ex), e = clamp64(j.ex_off[u + 1], 0, j.n_ex);
    __syncthreads();
    for (int64_t x = b + threadIdx.x; x < e; x += 256) {
        const int32_t i = j.ex_items[x];
        const int at = (i >> 5) - w0;
        if (i >= 0 && i < j.n_items && at >= 0 && at < n) atomicOr(&words[at], 1u << (i & 31));
    }
    __syncthreads();
    uint32_t* out = j.mask + r * j.v.tiles + w0;
    for (int x = 4 * threadIdx.x; x < n; x += 1024)  // (the tiles are a multiple of 8)
        *(uint4*)(out + x) = *(const uint4*)(words + x);
}

// The largest finite magnitude of either matrix (the batch's users only, without the items that their
// bias excludes), in kMaxParts parts.
template <int T>
__device__ __forceinline__ void largest_factors(const Job& j, int block) {
    __shared__ float red[4];
    const bool users = block < kUserParts;
    const Side& s = users ? j.u : j.v;
    const int part = users ? block : block - kUserParts;
    const int parts = users ? kUserParts : kMaxParts - kUserParts;
    float m = 0.0f;
    const auto take = [&](float x) {
        const float a = fabsf(x);
        if (a < 3e38f) m = fmaxf(m, a);
    };
    const int lane = threadIdx.x & 63;
    const float* bias = users ? nullptr : j.bias;
    // the factors 4 at a time where they can be loaded so, else one by one
    const auto scan = [&](auto width) {
        constexpr int N = decltype(width)::value;
        const uint32_t per_row = (uint32_t)j.k / N;
        const int64_t n = s.n * per_row;
        const int64_t at = (int64_t)part * 256 + threadIdx.x, turn = (int64_t)parts * 256;
#pragma unroll 4
        for (int64_t x = at; x < n; x += turn) {
            const int64_t r = n >> 31 ? x / per_row : (int64_t)((uint32_t)x / per_row);
            const int64_t src = source_row(s, r);
            const float* p = (const float*)s.src + max(src, (int64_t)0) * s.ld + N * (x - r * per_row);
            float v[N];
            if constexpr (N == 4) {
                const f32x4 q = *(const f32x4*)p;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = q[e];
            } else {
                v[0] = *p;
            }
            const bool counts = src >= 0 && !(bias && bias[r] <= kGone);
#pragma unroll
            for (int e = 0; e < N; ++e) take(counts ? v[e] : 0.0f);
        }
    };
    if (s.vec8 && j.k % 4 == 0) {
        scan(std::integral_constant<int, 4>{});
    } else if (!s.index && s.ld == j.k && j.k >= 4 && (uintptr_t)s.src % 16 == 0) {
        // one array: 4 values belong to two rows at most (100 k x 150: 89 us one by one, 28 so)
        const float* src = (const float*)s.src;
        const uint32_t k = (uint32_t)j.k;
        const int64_t all = s.n * k, turn = (int64_t)parts * 1024;
        const auto counts = [&](int64_t r) { return !(bias && bias[r] <= kGone); };
#pragma unroll 4
        for (int64_t x = ((int64_t)part * 256 + threadIdx.x) * 4; x + 4 <= all; x += turn) {
            const int64_t r = all >> 31 ? x / k : (int64_t)((uint32_t)x / k), end = (r + 1) * k;
            const f32x4 v = *(const f32x4*)(src + x);
            const bool c0 = counts(r), c1 = counts(min(r + 1, s.n - 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) take((x + e < end ? c0 : c1) ? v[e] : 0.0f);
        }
        const int rest = (int)(all % 4);  // of the last row
        if (part == 0 && (int)threadIdx.x < rest)
            take(counts(s.n - 1) ? src[all - rest + threadIdx.x] : 0.0f);
    } else {
        scan(std::integral_constant<int, 1>{});
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0)
        j.parts[block] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}
// Both in one launch: kMaxParts blocks for the magnitudes (where j.parts is set), then the mask's.
template <int T>
__global__ __launch_bounds__(256) void softmax_start_kernel(Job j) {
    uint32_t block = blockIdx.x;
    if constexpr (T == MML_DTYPE_F32) {
        if (j.parts) {
            if (block < kMaxParts) return largest_factors<T>(j, (int)block);
            block -= kMaxParts;
        }
    }
    make_mask(j, block);
}

// The scales from the parts; all 256 threads of a block take part.  A matrix' largest magnitude comes
// out in [2^12, 2^13) -- for the scores only while eu + ev <= 24, so that biases of any size stay in f32
// when they are scaled along: what is lost of the smaller matrix then is below 2^-36 of a score of 1.
template <int T>
__device__ __forceinline__ Scale make_scale(const Job& j) {
    int eu = 0, ev = 0, gu = 0, gv = 0;
    if constexpr (T == MML_DTYPE_F32) {
        __shared__ float red[4], first;
        const int t = threadIdx.x;
        float v = j.parts[t], u = v;
        if (t < kUserParts) v = 0.0f;
        v = fmaxf(v, j.parts[t + 256]);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            v = fmaxf(v, __shfl_xor(v, d));
            u = fmaxf(u, __shfl_xor(u, d));
        }
        static_assert(kUserParts == 64, "the users' parts are wave 0's");
        if (t == 0) first = u;
        if ((t & 63) == 0) red[t >> 6] = v;
        __syncthreads();
        u = first;
        v = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        // (frexp: x = f 2^e, f in [0.5, 1); of 0 it is 0)
        eu = gu = 13 - __builtin_amdgcn_frexp_expf(u);
        ev = gv = 13 - __builtin_amdgcn_frexp_expf(v);
        if (eu + ev > 24) {
            if (eu > 12 && ev > 12) eu = ev = 12;
            else if (eu > 12) eu = 24 - ev;
            else ev = 24 - eu;
        }
    }
    Scale c;
    const int e = eu + ev;
    c.unit = ldexpf(1.0f, -e);
    c.kappa = ldexpf(kLog2e, -e);
    // (e <= 24: 1e30 2^24 is within f32; 2^40: products of scaled factors are below 2^35)
    c.gone = -fmaxf(ldexpf(1e30f, e), 1.0995116e12f);
    c.floor = c.gone * 0.0625f;
    if (e < kLeastExponent) c.unit = c.kappa = __builtin_nanf("");
    c.eu = eu;
    c.ev = ev;
    c.gu = gu;
    c.gv = gv;
    return c;
}

// A probability is 2^(s kappa - lse2), and lse is known to 2^-24 of itself: beyond this norm, where it
// is off by a tenth and more, a row's gradient is NaN.
constexpr float kMostNorm = 1e6f;
// The rows' constants of the gradient (thread t < 32 of a users' block: row r; bad: 1 = its factors are
// not finite, 2 = an unknown user).  A row without one -- both coefficients 0, no items left, an
// unknown user -- gets lse2 = 1e30, so that its p are 0.
__device__ __forceinline__ void make_meta(const Job& j, int64_t r, int bad) {
    float lse2 = 1e30f, c0 = 0.0f, c1 = 0.0f;
    int32_t given = -1;
    float w = 0.0f;
    if (r < j.n_rows && bad < 2) {
        const float lse = j.in_norm[r], h = j.g_ent ? j.g_ent[r] : 0.0f;
        int32_t t = j.target ? j.target[r] : -1;
        if (t < 0 || t >= j.n_items || (j.bias && j.bias[t] <= kGone) ||
            (j.mask && (j.mask[r * j.v.tiles + (t >> 5)] >> (t & 31) & 1u)))
            t = -1;
        w = t >= 0 && j.g_lp ? j.g_lp[r] : 0.0f;
        if ((w != 0.0f || h != 0.0f) && lse != -INFINITY) {
            const float H = h != 0.0f ? j.in_entropy[r] : 0.0f;
            lse2 = bad || !(fabsf(lse) <= kMostNorm) ? __builtin_nanf("") : lse * kLog2e;
            c0 = -(w + h * H);
            c1 = -h * kLn2;
            given = t;
        } else {
            w = 0.0f;
        }
    }
    RowMeta& m = j.meta[r >> 5];
    m.lse2[r & 31] = lse2;
    m.c0[r & 31] = c0;
    m.c1[r & 31] = c1;
    m.t[r & 31] = given;
    j.w[r] = w;
}

// Fragments of both sides, one block per tile of 32 rows (the users' tiles first).  A row with a
// value that is not finite is written as zeros and marked, so that 0 * NaN cannot reach the other
// rows' sums: an item that is not excluded gets the bias NaN, a user NaN results from the last kernel or
// NaN constants.  So is an item that its bias excludes, whose factors the scale does not count.  Bound by
// memory: 1 M items, k = 128 bf16 in 98 us (512 MB, 5.2 TB/s), 500 k with k = 256 and the transposed
// fragments in 155 us (768 MB).
template <int T, int KT>
__global__ __launch_bounds__(256) void softmax_prep_kernel(Job j) {
    using P = Planes<T>;
    constexpr int KP = KT * 16, MT = KT > 1 ? KT / 2 : 1, LD = KP + 4;
    __shared__ __align__(16) float tile[32 * LD];
    __shared__ int bad[32];
    const bool users = blockIdx.x < (uint32_t)j.u.tiles;
    const Side& s = users ? j.u : j.v;
    const int64_t tl = users ? blockIdx.x : blockIdx.x - j.u.tiles;
    const int t = threadIdx.x;
    const Scale sc = make_scale<T>(j);
    if (blockIdx.x == 0 && t == 0) *j.scale = sc;
    if (t < 32) {
        const int64_t row = tl * 32 + t;
        bad[t] = row >= s.n ? 0 : users ? 2 * (source_row(s, row) < 0)
                                        : 4 * (j.bias && j.bias[row] <= kGone);
    }
    __syncthreads();
    for (int x = t; x < 64 * KT; x += 256) {  // 8 factors each
        const int row = x / (2 * KT), f = 8 * (x % (2 * KT));
        const int64_t src = source_row(s, tl * 32 + row);
        float v[8] = {};
        if (src >= 0) {
            const int64_t at = src * s.ld + f;
            if (f + 8 <= j.k) {
                load_factors<T>(s.src, at, v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (f + e < j.k) v[e] = load_factor<T>(s.src, at + e);
            }
        }
        bool ok = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) ok = ok && fabsf(v[e]) < 3e38f;
        if (!ok) atomicOr(&bad[row], 1);
        *(f32x4*)&tile[row * LD + f] = f32x4{v[0], v[1], v[2], v[3]};
        *(f32x4*)&tile[row * LD + f + 4] = f32x4{v[4], v[5], v[6], v[7]};
    }
    __syncthreads();
    if (t < 32) {
        const int64_t row = tl * 32 + t;
        if (users) {
            if (j.meta) make_meta(j, row, bad[t]);
        } else {
            float b = row < s.n ? (j.bias ? j.bias[row] : 0.0f) : kGone;
            if (b <= kGone) b = sc.gone;
            else if (bad[t] || !(b < -kGone)) b = __builtin_nanf("");
            else b = fmaxf(ldexpf(b, sc.eu + sc.ev), sc.gone * 0.5f);
            j.vbias[row] = b;
        }
    }
    const int ex = users ? sc.eu : sc.ev, gx = users ? sc.gu : sc.gv;
    for (int x = t; x < KT * 64; x += 256) {
        const int ks = x >> 6, lane = x & 63, row = lane & 31;
        const f32x4* src = (const f32x4*)&tile[row * LD + ks * 16 + 8 * (lane >> 5)];
        const f32x4 lo = src[0], hi = src[1];
        uint32_t q[P::PS][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v = bad[row] ? 0.0f : ldexpf(e < 4 ? lo[e & 3] : hi[e & 3], ex);
#pragma unroll
            for (int p = 0; p < P::PS; ++p) q[p][e] = take_plane<T>(v);
        }
#pragma unroll
        for (int p = 0; p < P::PS; ++p)
            s.frag[((tl * P::PS + p) * KT + ks) * 64 + lane] =
                make_uint4(q[p][0] | q[p][1] << 16, q[p][2] | q[p][3] << 16,
                           q[p][4] | q[p][5] << 16, q[p][6] | q[p][7] << 16);
    }
    if (!s.trans) return;
    for (int x = t; x < MT * 128; x += 256) {
        const int mt = x >> 7, step = (x >> 6) & 1, lane = x & 63, f = 32 * mt + (lane & 31);
        uint32_t q[P::PG][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int row = 16 * step + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
            float v = f < KP && !bad[row] ? ldexpf(tile[row * LD + f], gx) : 0.0f;
#pragma unroll
            for (int p = 0; p < P::PG; ++p) q[p][e] = take_plane<T>(v);
        }
#pragma unroll
        for (int p = 0; p < P::PG; ++p)
            s.trans[((tl * P::PG + p) * MT * 2 + mt * 2 + step) * 64 + lane] =
                make_uint4(q[p][0] | q[p][1] << 16, q[p][2] | q[p][3] << 16,
                           q[p][4] | q[p][5] << 16, q[p][6] | q[p][7] << 16);
    }
}

// ------------------------------------------------------------------ staging
// One asynchronous copy of 16 bytes per active lane into LDS: lane i's 16 bytes at `from` go to
// to + 16 i (`to` is the same in all lanes).  Written in assembly, and not as the builtin, because
// the compiler makes every later LDS read wait for a builtin's copy to land, the reads of the other
// buffer too; stage_wait is the wait, and a __shared__ array filled here is only read behind one.
// (An SALU write of m0 needs a wait state before its use.)
__device__ __forceinline__ void copy_to_lds(const void* from, void* to) {
    const uint32_t at = __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)to);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 :
                 : "s"(at), "v"(from)
                 : "memory", "m0");
}
// n KB of fragments, the 1 KB pieces dealt over the block's waves.  stage_wait: this wave's copies
// have landed; with the barrier behind it, everyone's have.
template <int WAVES>
__device__ __forceinline__ void stage(const uint4* __restrict__ src, uint4* dst, int n) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int c = wave; c < n; c += WAVES) copy_to_lds(src + c * 64 + lane, dst + c * 64);
}
__device__ __forceinline__ void stage_wait() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// ------------------------------------------------------------------ tiles
template <int T>
__device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
    if constexpr (Planes<T>::HALF)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// The larger of the two values in lanes l and l + 32, in both
__device__ __forceinline__ float both_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// c + A B over the PS planes of KT steps (smallest products first).  A: fragments in LDS; B: the kept
// side's fragments in registers, the last LK steps' in LDS.
template <int T, int KT, int LK>
__device__ __forceinline__ f32x16 score_tile(const uint4* a,
                                             const uint4 (&b)[Planes<T>::PS][KT - LK],
                                             const uint4* kept, f32x16 c, int lane) {
    constexpr int PS = Planes<T>::PS;
#pragma unroll
    for (int ks = 0; ks < KT; ++ks) {
        uint4 x[PS], y[PS];
#pragma unroll
        for (int p = 0; p < PS; ++p) {
            x[p] = a[(p * KT + ks) * 64 + lane];
            y[p] = ks < KT - LK ? b[p][ks < KT - LK ? ks : 0]
                                : kept[(p * LK + ks - (KT - LK)) * 64 + lane];
        }
#pragma unroll
        for (int sum = PS - 1; sum >= 0; --sum)
#pragma unroll
            for (int p = sum; p >= 0; --p) c = mfma<T>(x[p], y[sum - p], c);
    }
    return c;
}
// The kept side's fragments of tile `tl`
template <int T, int KT, int LK>
__device__ __forceinline__ void load_kept(const uint4* __restrict__ frag, int64_t tl,
                                          uint4 (&b)[Planes<T>::PS][KT - LK], uint4* kept,
                                          int lane) {
    constexpr int PS = Planes<T>::PS;
#pragma unroll
    for (int p = 0; p < PS; ++p)
#pragma unroll
        for (int ks = 0; ks < KT; ++ks) {
            const uint4 x = frag[((tl * PS + p) * KT + ks) * 64 + lane];
            if (ks < KT - LK)
                b[p][ks < KT - LK ? ks : 0] = x;
            else
                kept[(p * LK + ks - (KT - LK)) * 64 + lane] = x;
        }
}

// Two values as two f16 planes, both rounded to nearest
__device__ __forceinline__ void split_pair(float x, float y, uint32_t& hi, uint32_t& lo) {
    float minus = -1.0f;  // unknown to the compiler, so that x - hi is one v_fma_mix_f32
    asm("" : "+s"(minus));
    const f16x2 h = __builtin_convertvector((f32x2{x, y}), f16x2);
    const f32x2 rest = {fmaf((float)h[0], minus, x), fmaf((float)h[1], minus, y)};
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, f16x2));
}
// The planes of G's registers 8 s .. 8 s + 7 as B operands, both rounded to nearest (the rest between
// them is exact).
template <int T>
__device__ __forceinline__ void split_g(const float (&g)[16], int step, uint4 (&q)[2]) {
    uint32_t w[2][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const f32x2 x = {g[8 * step + 2 * e], g[8 * step + 2 * e + 1]};
        if constexpr (Planes<T>::HALF) {
            split_pair(x[0], x[1], w[0][e], w[1][e]);
        } else {
            w[0][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(x, bf16x2));
            const f32x2 rest = {x[0] - __uint_as_float(w[0][e] << 16),
                                x[1] - __uint_as_float(w[0][e] & 0xFFFF0000u)};
            w[1][e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(rest, bf16x2));
        }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) q[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
}

// The power of two that a kept row's G and sums carry (f16 planes): |G| 2^e stays under 2^15.  Where
// a larger |G| comes, the exponent drops to bring it into [2^13, 2^14) and the sums follow, exactly.
// Both lanes of a row hold the same.
struct Shift {
    int32_t e = 100;
    float f = 1.2676506e30f;  // 2^e
};
template <int T, int MT>
__device__ __forceinline__ void scale_g(float (&g)[16], f32x16 (&acc)[MT], Shift& sh) {
    if constexpr (Planes<T>::HALF) {
        float most = fabsf(g[0]);
#pragma unroll
        for (int i = 1; i < 16; ++i) most = fmaxf(most, fabsf(g[i]));
        most = both_max(most);
        if (__any(most * sh.f > 32768.0f)) {
            const int e = most * sh.f > 32768.0f ? 14 - __builtin_amdgcn_frexp_expf(most) : sh.e;
            const float down = ldexpf(1.0f, max(e - sh.e, -126));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[mt][i] *= down;
            sh.e = e;
            sh.f = ldexpf(1.0f, e);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] *= sh.f;
    }
}
// What a sum is multiplied by in the end: the planes' scale 2^ex and G's undone
template <int T>
__device__ __forceinline__ float unscale(float x, const Shift& sh, int ex) {
    return Planes<T>::HALF ? ldexpf(x, -sh.e - ex) : x;
}

// acc[mt] += A B for the MT tiles of 32 factors: A the transposed fragments, B the planes of G
template <int T, int KT>
__device__ __forceinline__ void grad_tile(const uint4* a, const float (&g)[16],
                                          f32x16 (&acc)[(KT > 1 ? KT / 2 : 1)], int lane) {
    using P = Planes<T>;
    constexpr int MT = KT > 1 ? KT / 2 : 1, MAXSUM = P::PG > P::GP ? P::PG - 1 : P::GP - 1;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        uint4 q[P::GP];
        split_g<T>(g, s, q);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            uint4 x[P::PG];
#pragma unroll
            for (int p = 0; p < P::PG; ++p) x[p] = a[(p * MT * 2 + mt * 2 + s) * 64 + lane];
#pragma unroll
            for (int sum = MAXSUM; sum >= 0; --sum)
#pragma unroll
                for (int p = P::PG - 1; p >= 0; --p)
                    if (sum - p >= 0 && sum - p < P::GP) acc[mt] = mfma<T>(x[p], q[sum - p], acc[mt]);
        }
        // two tiles' LDS reads (0x100) ahead of their matrix instructions (0x008): 1,024 x 500 k, k = 256
        // bf16: the users' gradient in 664 us against 683; one or three ahead gain less
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * P::PG, 0);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            __builtin_amdgcn_sched_group_barrier(0x008, P::PG == 2 ? 3 : 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, P::PG, 0);
        }
    }
}

// The larger, or NaN if either is: what the instruction does without quieting its operands first
__device__ __forceinline__ float largest(float a, float b) { return __builtin_elementwise_maximum(a, b); }

__device__ __forceinline__ int reg_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// `gone` where the bits (shifted right by 4 h) say so.  The first empty asm keeps the compiler from
// taking the selects out of their branch: 32 instructions for every tile against 105 for the tile
// itself.  The other hides that `on` is 0 or -1: a bit field and a bitwise select, 2 instructions a
// score, instead of a comparison and a conditional move with the waits between them.
__device__ __forceinline__ void mask_tile(f32x16& c, uint32_t bits, float gone) {
    asm volatile("");
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        uint32_t on = (uint32_t)__builtin_amdgcn_sbfe((int)bits, reg_row(i, 0), 1);
        asm("" : "+v"(on));
        c[i] = __uint_as_float((on & __float_as_uint(gone)) | (~on & __float_as_uint(c[i])));
    }
}

// ------------------------------------------------------------------ forward
// Waves of a block: as many as the registers of two blocks' waves per SIMD allow, since the block
// shares each streamed tile.
template <int T, int KT>
constexpr int forward_waves() {
    return Planes<T>::PS * KT > 16 || (T == MML_DTYPE_F32 && KT == 8) ? 4 : 8;
}

template <int T, int KT>
constexpr int forward_per_simd() {
    return Planes<T>::PS * KT > 16 || (T == MML_DTYPE_F32 && KT == 8) ? 2 : 4;
}

// Tiles staged at a time: up to 8 in 32 KB.  Fewer barriers, and between two of them the waves
// drift apart, so that one's matrix work runs under another's exponentials.
template <int T, int KT>
constexpr int forward_tiles() {
    constexpr int n = 32 / (Planes<T>::PS * KT);
    return n >= 8 ? 8 : n >= 4 ? 4 : n >= 2 ? 2 : 1;
}
// Exponents are one fma, s kappa - m2, with m2 = m kappa rounded: off by 2^-24 of |m2|.  From this
// |m2| on (2^-15 off; from 2^31 on the exponentials would be infinite or 0) the maximum is subtracted
// first, exactly.
constexpr float kFar = 1024.0f;
constexpr int kTileGroup = 8;  // the streamed items are padded to a multiple of so many tiles

// A block's waves keep 32 users each and stream the item tiles of a split through LDS, TPS tiles a
// turn in two buffers: the next turn's tiles are on the way while this one's are used.  Lane l: user
// l % 32, 16 of a tile's 32 items.  m, l, w: the running maximum (of scaled scores), the sum of
// e = exp(s - m) and of e y, y = log2 e.
// Bound by instructions and power, not memory: 2,048 x 1 M, k = 128 bf16 takes 726 us, where the SIMDs
// issue about 450 cycles of vector instructions a tile (16 exponentials of 8 cycles, 80 others of 4), 64 % of
// the time, beside 256 of matrix instructions, at 1.95 GHz of 2.4: on zeros the same launch takes 500 us.
template <int T, int KT, bool TOP>
__global__ __launch_bounds__((forward_waves<T, KT>() * 64), (forward_per_simd<T, KT>())) void
softmax_forward_kernel(Job j) {
    constexpr int PS = Planes<T>::PS, WAVES = forward_waves<T, KT>(), TPS = forward_tiles<T, KT>();
    __shared__ uint4 buf[2][TPS * PS * KT * 64];
    __shared__ f32x4 bias[2][TPS * 8];
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
    const int split = blockIdx.x % j.splits;
    const int64_t ut = (int64_t)(blockIdx.x / j.splits) * WAVES + wave;
    // A wave behind the last tile of users has a loop of its own: a branch around the work in the common
    // one costs the others more than the work (the accumulators change registers at it).
    const bool mine = ut < j.u.tiles;
    const int64_t row = (mine ? ut : 0) * 32 + (lane & 31);
    uint4 b[PS][KT];
    load_kept<T, KT, 0>(j.u.frag, mine ? ut : 0, b, nullptr, lane);
    const int t0 = (int)((int64_t)(j.v.tiles / TPS) * split / j.splits) * TPS;
    const int t1 = (int)((int64_t)(j.v.tiles / TPS) * (split + 1) / j.splits) * TPS;
    const auto load = [&](int tl, int at) {
        stage<WAVES>(j.v.frag + (int64_t)tl * PS * KT * 64, buf[at], TPS * PS * KT);
        if (wave == WAVES - 1 && lane < TPS * 8)  // TPS * 32 floats
            copy_to_lds((const f32x4*)j.vbias + tl * 8 + lane, bias[at]);
    };
    const Scale sc = *j.scale;
    float m = sc.floor, m2 = m * sc.kappa, l = 0.0f, w = 0.0f, mx[TPS];
    bool far = false;  // in any lane
    uint32_t bits[TPS] = {}, next[TPS] = {};
    const auto load_bits = [&](int tl) {
#pragma unroll
        for (int x = 0; x < TPS; ++x) next[x] = j.mask[row * j.v.tiles + tl + x];
    };
    // A turn's maxima leave in the next turn, so that no wait meets the stores.  mx: of this lane's 16
    // items each; a swap joins the halves of two tiles, the first in the lower lanes.
    const auto store_max = [&](int tl) {
        if (!TOP) return;
        float* p = j.cmax + row * j.cpad + tl;
        if constexpr (TPS == 1) {
            const float most = both_max(mx[0]);
            if (h == 0) *p = most;
        } else {
            constexpr int N = TPS / 2;
            float q[N];
#pragma unroll
            for (int x = 0; x < N; ++x) {
                const auto s = __builtin_amdgcn_permlane32_swap(
                    __float_as_uint(mx[x]), __float_as_uint(mx[x + N]), false, false);
                q[x] = largest(__uint_as_float(s[0]), __uint_as_float(s[1]));
            }
            p += N * h;
            if constexpr (N == 4) *(f32x4*)p = f32x4{q[0], q[1], q[2], q[3]};
            else if constexpr (N == 2) *(f32x2*)p = f32x2{q[0], q[1]};
            else *p = q[0];
        }
    };
    if (t0 < t1) {
        load(t0, 0);
        if (j.mask) load_bits(t0);
    }
    if (!mine) {  // copies its share
        for (int ts = t0, at = 0; ts < t1; ts += TPS, at ^= 1) {
            stage_wait();
            if (ts + TPS < t1) load(ts + TPS, at ^ 1);
        }
        return;
    }
    for (int ts = t0, at = 0; ts < t1; ts += TPS, at ^= 1) {
        stage_wait();
#pragma unroll
        for (int x = 0; x < TPS; ++x) {
            // the wait for this load belongs before the next copies, not behind them
            asm volatile("" : "+v"(next[x]));
            bits[x] = next[x];
        }
        if (ts + TPS < t1) {
            load(ts + TPS, at ^ 1);
            if (j.mask) load_bits(ts + TPS);
        }
        if (ts > t0) store_max(ts - TPS);
#pragma unroll
        for (int x = 0; x < TPS; ++x) {
            f32x16 c;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 v = bias[at][x * 8 + 2 * q + h];
#pragma unroll
                for (int e = 0; e < 4; ++e) c[4 * q + e] = v[e];
            }
            c = score_tile<T, KT, 0>(buf[at] + x * PS * KT * 64, b, nullptr, c, lane);
            if (__any(bits[x])) mask_tile(c, bits[x] >> (4 * h), sc.gone);
            float mt = c[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) mt = largest(mt, c[i]);
            mx[x] = mt;
            if (__any(mt > m)) {
                const float mn = fmaxf(m, mt), d = (m - mn) * sc.kappa;
                const float f = __builtin_amdgcn_exp2f(d);
                w = f * fmaf(l, d, w);
                l *= f;
                m = mn;
                m2 = m * sc.kappa;
                far = __any(fabsf(m2) > kFar && m > sc.floor);
            }
            float from = m2;
            if (far) {
                asm volatile("");  // as in mask_tile
                from = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) c[i] -= m;
            }
            float sl, sw;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float y = fmaf(c[i], sc.kappa, -from), e = __builtin_amdgcn_exp2f(y);
                sl = i ? sl + e : e;
                sw = i ? fmaf(e, y, sw) : e * y;
            }
            l += sl;
            w += sw;
        }
    }
    if (t0 < t1) store_max(t1 - TPS);
    // the halves' states joined: lanes l and l + 32 hold the same user
    const float mn = both_max(m), d = (m - mn) * sc.kappa;
    const float f = __builtin_amdgcn_exp2f(d);
    w = f * fmaf(l, d, w);
    l *= f;
    w += __shfl_xor(w, 32);
    l += __shfl_xor(l, 32);
    if (h == 0) {
        float* p = j.part + row * j.splits + split;
        const int64_t next = j.rows_pad * j.splits;
        p[0] = mn;
        p[next] = l;
        p[2 * next] = w;
    }
}

// The forward pass for at most 32 rows, or for so little work that launches cost more: with one tile
// of users there is nothing to share and nothing to prepare.  A wave makes its fragments from the
// factors themselves, both sides', and the catalogue is read once (per tile of users).  f32: every tile
// of items has a scale of its own, 2^ev, and
// the scores are brought back before the bias is added (one instruction more per score, which the
// memory's pace hides: 25.6 MB of factors, one user, take 12 us, of which 5 are a large copy's rate and
// the rest the latency of a few loads one behind the other).  m, l, w as in
// the forward pass, in true units; the block's waves are joined before they are written.
constexpr int kDirectWaves = 4;

// Fragments of 32 rows from their source: row `row` of src in lanes l and l + 32.  Returns the
// exponent of the f32 planes' scale; finite: whether this lane's values are
template <int T, int KT>
__device__ __forceinline__ void load_rows(const Side& s, int64_t src, int k, int h,
                                          float (&v)[KT][8]) {
    if (k % 8 == 0) {
        // whole groups: every lane loads (a lane without a group row 0's), so that all loads are on
        // the way together
#pragma unroll
        for (int ks = 0; ks < KT; ++ks) {
            const int f = 16 * ks + 8 * h;
            load_factors<T>(s.src, src >= 0 && f < k ? src * s.ld + f : 0, v[ks]);
        }
#pragma unroll
        for (int ks = 0; ks < KT; ++ks) {
            const bool in = src >= 0 && 16 * ks + 8 * h < k;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[ks][e] = in ? v[ks][e] : 0.0f;
        }
    } else {
#pragma unroll
        for (int ks = 0; ks < KT; ++ks) {
            const int f0 = 16 * ks + 8 * h;
            if (KT > 1 && src >= 0 && f0 + 8 <= k) {
                load_factors<T>(s.src, src * s.ld + f0, v[ks]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[ks][e] = src >= 0 && f0 + e < k ? load_factor<T>(s.src, src * s.ld + f0 + e)
                                                      : 0.0f;
            }
        }
    }
}
// (What a row holds reaches its own scores only, so values that are not finite need no zeros here.)
template <int T, int KT>
__device__ __forceinline__ int make_planes(const float (&v)[KT][8], uint4 (&q)[Planes<T>::PS][KT],
                                           bool& finite) {
    using P = Planes<T>;
    float most = 0.0f, zero = 0.0f;
#pragma unroll
    for (int ks = 0; ks < KT; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            zero = fmaf(v[ks][e], 0.0f, zero);  // NaN from the first value that is not finite on
            if (T == MML_DTYPE_F32) most = fmaxf(most, fabsf(v[ks][e]));
        }
    finite = zero == 0.0f && most < 3e38f;
    int ex = 0;
    float mul = 1.0f;
    if constexpr (T == MML_DTYPE_F32) {
        if (!finite) most = 0.0f;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
        ex = min(100, 13 - __builtin_amdgcn_frexp_expf(most));  // (100: mul is finite)
        mul = ldexpf(1.0f, ex);
    }
#pragma unroll
    for (int ks = 0; ks < KT; ++ks) {
        uint32_t w[P::PS][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = v[ks][2 * e], y = v[ks][2 * e + 1];
            if constexpr (T == MML_DTYPE_F32) {
                split_pair(x * mul, y * mul, w[0][e], w[P::PS - 1][e]);
            } else if constexpr (T == MML_DTYPE_F16) {
                w[0][e] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)x, (_Float16)y});
            } else {
                w[0][e] = __float_as_uint(x) >> 16 | (__float_as_uint(y) & 0xFFFF0000u);
            }
        }
#pragma unroll
        for (int p = 0; p < P::PS; ++p) q[p][ks] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
    }
    return ex;
}

template <int T, int KT, bool TOP>
__global__ __launch_bounds__(kDirectWaves * 64) void softmax_direct_kernel(Job j) {
    constexpr int PS = Planes<T>::PS, W = kDirectWaves;
    __shared__ float state[W][3][32];
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6, col = lane & 31;
    const int split = blockIdx.x % j.splits;
    const int64_t row = (int64_t)(blockIdx.x / j.splits) * 32 + col;
    const int ways = j.splits * W, way = split * W + wave;
    const int t0 = (int)((int64_t)j.v.tiles * way / ways);
    const int t1 = (int)((int64_t)j.v.tiles * (way + 1) / ways);
    // a tile's factors are on the way while the one before is used (up to k = 128: registers)
    constexpr bool AHEAD = KT <= 8;
    float v[KT][8], u[KT][8];
    uint4 b[PS][KT];
    bool finite;
    load_rows<T, KT>(j.u, source_row(j.u, row), j.k, h, u);
    if (AHEAD && t0 < t1) load_rows<T, KT>(j.v, source_row(j.v, (int64_t)t0 * 32 + col), j.k, h, v);
    const int eu = make_planes<T, KT>(u, b, finite);
    const Scale sc = plain_scale();
    float m = sc.floor, l = 0.0f, w = 0.0f;
    for (int tl = t0; tl < t1; ++tl) {
        float bias[16];
        const bool whole = j.bias && j.bias_vec4 && tl * 32 + 32 <= j.n_items;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int64_t item = (int64_t)tl * 32 + 8 * q + 4 * h;
            if (whole) {
                const f32x4 x = *(const f32x4*)&j.bias[item];
#pragma unroll
                for (int e = 0; e < 4; ++e) bias[4 * q + e] = x[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    bias[4 * q + e] =
                        item + e < j.n_items ? (j.bias ? j.bias[item + e] : 0.0f) : kGone;
            }
        }
        const uint32_t bits =
            j.mask ? j.mask[row * (int64_t)j.v.tiles + tl] >> (4 * h) : 0;
        const int64_t own = (int64_t)tl * 32 + col;
        const bool off = j.bias && own < j.n_items && j.bias[own] <= kGone;
        uint4 a[PS][KT];
        if (!AHEAD) load_rows<T, KT>(j.v, source_row(j.v, (int64_t)tl * 32 + col), j.k, h, v);
        // an item that its bias excludes: its factors do not matter
        if (__any(off)) {
            asm volatile("");  // as in mask_tile
#pragma unroll
            for (int ks = 0; ks < KT; ++ks)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[ks][e] = off ? 0.0f : v[ks][e];
        }
        const int ev = make_planes<T, KT>(v, a, finite);
        uint64_t odd = __ballot(!finite);  // rows with a value that is not finite
        if (eu + ev < kLeastExponent) odd = ~0ull;
        if (AHEAD && tl + 1 < t1)
            load_rows<T, KT>(j.v, source_row(j.v, (int64_t)(tl + 1) * 32 + col), j.k, h, v);
        f32x16 c = {};
#pragma unroll
        for (int ks = 0; ks < KT; ++ks)
#pragma unroll
            for (int sum = PS - 1; sum >= 0; --sum)
#pragma unroll
                for (int p = sum; p >= 0; --p) c = mfma<T>(a[p][ks], b[sum - p][ks], c);
        const float unit = ldexpf(1.0f, -eu - ev);
        bool strange = odd != 0;  // a factor or a bias that is not finite: rarely
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            strange = strange || !(bias[i] < -kGone);
            c[i] = fmaxf(fmaf(c[i], unit, bias[i]), sc.gone);  // (an excluded item's bias is below)
        }
        if (__any(strange)) {
            asm volatile("");
            const uint32_t rows = (uint32_t)odd | (uint32_t)(odd >> 32);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (!(bias[i] < -kGone) || rows >> reg_row(i, h) & 1u) c[i] = __builtin_nanf("");
                if (bias[i] <= kGone) c[i] = sc.gone;
            }
        }
        if (__any(bits & 0x0F0F0F0Fu)) mask_tile(c, bits, sc.gone);
        float mt = c[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mt = fmaxf(mt, c[i]);
        if constexpr (TOP) {
            const float most = both_max(mt);
            if (h == 0 && row < j.n_rows) j.cmax[row * j.cpad + tl] = most;
        }
        const float mn = fmaxf(m, mt), d = (m - mn) * kLog2e, f = __builtin_amdgcn_exp2f(d);
        w = f * fmaf(l, d, w);
        l *= f;
        m = mn;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float y = (c[i] - m) * kLog2e, e = __builtin_amdgcn_exp2f(y);
            l += e;
            w = fmaf(e, y, w);
        }
    }
    {
        const float mn = both_max(m), d = (m - mn) * kLog2e, f = __builtin_amdgcn_exp2f(d);
        w = f * fmaf(l, d, w);
        l *= f;
        w += __shfl_xor(w, 32);
        l += __shfl_xor(l, 32);
        if (h == 0) state[wave][0][col] = mn, state[wave][1][col] = l, state[wave][2][col] = w;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        m = state[0][0][col];
#pragma unroll
        for (int x = 1; x < W; ++x) m = fmaxf(m, state[x][0][col]);
        l = w = 0.0f;
#pragma unroll
        for (int x = 0; x < W; ++x) {
            const float d = (state[x][0][col] - m) * kLog2e, f = __builtin_amdgcn_exp2f(d);
            w += f * fmaf(state[x][1][col], d, state[x][2][col]);
            l += f * state[x][1][col];
        }
        float* p = j.part + row * j.splits + split;
        const int64_t next = j.rows_pad * j.splits;
        p[0] = m;
        p[next] = l;
        p[2 * next] = w;
    }
}

// x of the lane whose number differs in one of the lowest two bits
template <int D>
__device__ __forceinline__ double neighbour(double x) {
    constexpr int ctrl = D == 1 ? 0xB1 : 0x4E;  // quad_perm 1 0 3 2, 2 3 0 1
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, ctrl, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), ctrl, 0xF, 0xF, true);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
// s_rj in 64 bits for the given and the top items: exact products, f64 sums.  LANES neighbouring
// lanes share an item (every lane gets the sum); u: the user's row in LDS.
template <int T, int LANES>
__device__ __forceinline__ double exact_score(const Job& j, const double* u, int64_t i, int lane) {
    double a = 0.0;
    const int64_t at = i * j.v.ld;
#pragma unroll 2
    for (int f = 8 * lane; f + 8 <= j.k; f += 8 * LANES) {
        float x[8];
        load_factors<T>(j.v.src, at + f, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) a = fma(u[f + e], (double)x[e], a);
    }
    for (int f = (j.k & ~7) + lane; f < j.k; f += LANES)
        a = fma(u[f], (double)load_factor<T>(j.v.src, at + f), a);
    if (LANES > 1) a += neighbour<1>(a);
    if (LANES > 2) a += neighbour<2>(a);
#pragma unroll
    for (int d = 4; d < LANES; d <<= 1) a += __shfl_xor(a, d);
    return a + (j.bias ? (double)j.bias[i] : 0.0);
}
__device__ __forceinline__ bool is_excluded(const Job& j, int64_t r, int64_t i) {
    return (j.bias && j.bias[i] <= kGone) ||
           (j.mask && (j.mask[r * j.v.tiles + (i >> 5)] >> (i & 31) & 1u));
}
// A double as an unsigned key in the same order (-inf is the smallest that occurs)
__device__ __forceinline__ uint64_t key_of(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double value_of(uint64_t k) {
    return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k));
}
__device__ __forceinline__ bool before(uint64_t va, int32_t ia, uint64_t vb, int32_t ib) {
    return va > vb || (va == vb && ia < ib);  // larger value first, then lower index
}
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b >> 31 ? ~b : b | 1u << 31;
}

constexpr int kListed = 1024;     // tiles that the selection below lists at most
constexpr int kCandidates = 512;  // and items, in the same memory

// A bound that at least `want` of the 256 keys reach and few more: the want-th largest key with its
// low bits cut off, found bit by bit.  One wave, four keys a lane.
__device__ __forceinline__ uint32_t bound_of(const uint32_t* key, int want) {
    uint32_t k[4], b = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = key[(threadIdx.x & 63) + 64 * i];
#pragma unroll 1
    for (int bit = 31; bit >= 12; --bit) {
        const uint32_t c = b | 1u << bit;
        int n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) n += __builtin_popcountll(__ballot(k[i] >= c));
        if (n >= want) b = c;
    }
    return b;
}
// A row's maxima as a block of NT threads reads them, four at a time (the tiles are a multiple of 8):
// the first groups of a thread stay in registers for the second pass: 256 threads hold 4,096 maxima
// (131 k items; 4,096 rows of 100 k items, top 10: 8 us less than with two reads).  Holding all of
// 1 M items' in 512 threads gained nothing: the registers leave too few blocks to score with.
template <int NT>
struct Maxima {
    static constexpr int kHeld = NT == 256 ? 4 : 1;
    const float* cm;
    int tiles;
    f32x4 held[kHeld];
    __device__ __forceinline__ void load() {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int x = 4 * (threadIdx.x + i * NT);
            held[i] = *(const f32x4*)(cm + (x < tiles ? x : 0));
        }
    }
    template <class F>
    __device__ __forceinline__ void each(F&& f) const {  // f(maximum, tile)
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int x = 4 * (threadIdx.x + i * NT);
            if (x < tiles)
#pragma unroll
                for (int e = 0; e < 4; ++e) f(held[i][e], x + e);
        }
#pragma unroll 4
        for (int x = 4 * (threadIdx.x + kHeld * NT); x < tiles; x += 4 * NT) {
            const f32x4 v = *(const f32x4*)(cm + x);
#pragma unroll
            for (int e = 0; e < 4; ++e) f(v[e], x + e);
        }
    }
};

// The `want` tiles with the largest maxima cm[0 .. tiles), ordered, the lower tile first among
// equals.  `least` is under the want-th largest of 256 partial maxima, which is a lower
// bound of the want-th largest maximum, so few tiles are at or above it: they are listed and ranked
// by counting.  Where more than kListed are (many equal maxima), they are taken one after another.
template <int NT>
__device__ __forceinline__ void select_tiles(const Maxima<NT>& maxima, int want, uint32_t least,
                                             int32_t* chosen, uint32_t* key, int32_t* index,
                                             int32_t& count) {
    const int t = threadIdx.x;
    const float* cm = maxima.cm;
    const int tiles = maxima.tiles;
    maxima.each([&](float most, int tile) {
        const uint32_t v = key_of(most);
        if (v < least) return;
        const int at = atomicAdd(&count, 1);
        if (at < kListed) {
            key[at] = v;
            index[at] = tile;
        }
    });
    __syncthreads();
    const int n = count;
    if (n <= kListed) {
        for (int x = t; x < n; x += NT) {
            const uint32_t v = key[x];
            const int32_t i = index[x];
            int r = 0;
#pragma unroll 4
            for (int y = 0; y < n; ++y) r += before(key[y], index[y], v, i);
            if (r < want) chosen[r] = i;
        }
        __syncthreads();
        return;
    }
    uint32_t lv = 0xFFFFFFFFu;
    int32_t li = -1;
    for (int c = 0; c < want; ++c) {
        uint32_t bv = 0;
        int32_t bi = 0x7FFFFFFF;
        for (int x = t; x < tiles; x += NT) {
            const uint32_t v = key_of(cm[x]);
            if (before(lv, li, v, x) && before(v, x, bv, bi)) bv = v, bi = x;
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const uint32_t v = (uint32_t)__shfl_xor((int)bv, d);
            const int32_t i = __shfl_xor(bi, d);
            if (before(v, i, bv, bi)) bv = v, bi = i;
        }
        __syncthreads();
        if ((t & 63) == 0) key[t >> 6] = bv, index[t >> 6] = bi;
        __syncthreads();
        bv = key[0], bi = index[0];
        for (int w = 1; w < NT / 64; ++w)
            if (before(key[w], index[w], bv, bi)) bv = key[w], bi = index[w];
        lv = bv, li = bi;
        if (t == 0) chosen[c] = bi;
    }
    __syncthreads();
}

// One block per row (64 threads; with top items 256, or 1,024 where the rows are too few to fill the
// GPU): the splits' states joined, the outputs, and the top items.  The n best items lie in the n
// tiles with the largest maxima (lower tile first among equals); two more tiles cover the rounding of
// the maxima.  Their items are scored again in 64 bits, so the order is that of the exact scores.  The
// n-th largest of the tiles' exact maxima bounds the n-th best score from below: the items at or above
// it are ranked by counting.  Dynamic LDS: the candidates' keys, 8 bytes each.
// Bound by memory: the maxima (2,048 rows of 1 M items: 256 MB, read twice, 86 of 124 us with the top
// 20) and the candidates' factors, 8 KB a tile at k = 64 (4,096 rows of 100 k items: 403 MB with the top
// 10, 54 us).  Waves hide its latencies better than loads in flight: 8 a SIMD and one item a turn take
// those 54 us, 6 and two items 60, 4 and four items 82 (from the top 50 on, where LDS leaves 4 to 6
// blocks a CU, it is the other way round by a tenth).  Without top items 5 us.
template <int T, int NT>
__global__ __launch_bounds__(NT, 8) void softmax_finish_kernel(Job j) {
    constexpr bool TOP = NT > 64;
    __shared__ double urow[256], joined[2];
    // the tiles' keys, later the candidates' (the listed ones' order is that of a counter: any)
    __shared__ uint64_t listed_key[TOP ? kCandidates : 1];
    static_assert(kListed * sizeof(uint32_t) == kCandidates * sizeof(uint64_t), "one array for both");
    __shared__ uint32_t least_tile;
    uint32_t* key = reinterpret_cast<uint32_t*>(listed_key);
    const int64_t r = blockIdx.x;
    const int t = threadIdx.x;
    const int64_t u = source_row(j.u, r);
    uint32_t mine = 0;
    Maxima<NT> maxima{j.cmax + r * j.cpad, j.v.tiles};
    if (TOP) {
        maxima.load();
        maxima.each([&](float most, int) { mine = max(mine, key_of(most)); });
        if (t < 256) key[t] = mine;
    }
    bool bad = u < 0;  // an unknown user, or factors that are not finite
    for (int f = t & 63; f < j.k; f += 64) {  // every wave checks the whole row, wave 0 keeps it
        const float x = u >= 0 ? load_factor<T>(j.u.src, u * j.u.ld + f) : 0.0f;
        bad = bad || !(fabsf(x) < 3e38f);
        if (t < 64) urow[f] = (double)x;
    }
    bad = __any(bad);
    if (t < 64) {  // the splits' states
        const Scale sc = j.scale ? *j.scale : plain_scale();
        const float* part = j.part + r * j.splits;
        const int64_t next = j.rows_pad * j.splits;
        float m = sc.floor;
#pragma unroll 4
        for (int s = t; s < j.splits; s += 64) m = fmaxf(m, part[s]);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
        double l = 0.0, w = 0.0;
#pragma unroll 4
        for (int s = t; s < j.splits; s += 64) {
            const double d = ((double)part[s] - m) * sc.unit * 1.4426950408889634;
            const double f = __builtin_amdgcn_exp2f((float)d), ls = part[s + next];
            w += f * ((double)part[s + 2 * next] + ls * d);
            l += f * ls;
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            l += __shfl_xor(l, d);
            w += __shfl_xor(w, d);
        }
        double lse = (double)m * sc.unit + log(l), H = log(l) - 0.69314718055994531 * w / l;
        if (m <= sc.floor && l == l) lse = -INFINITY, H = 0.0;  // no item left
        if (bad) lse = H = __builtin_nan("");
        if (t == 0) joined[0] = lse, joined[1] = H;
    }
    __syncthreads();
    if (NT > 256) {
        if (t >= 256) atomicMax(&key[t & 255], mine);
        __syncthreads();
    }
    const double lse = joined[0];
    if (t >= NT - 64) {  // the last wave
        const int32_t g = j.target ? j.target[r] : -1;
        double lp = 0.0;
        if (lse != lse) lp = lse;
        else if (g >= 0 && g < j.n_items)
            lp = lse == -INFINITY || is_excluded(j, r, g)
                     ? -INFINITY
                     : exact_score<T, 64>(j, urow, g, t & 63) - lse;
        if (t == NT - 1) {
            const double H = joined[1];
            j.log_probs[r] = (float)lp;
            j.log_norm[r] = (float)lse;
            j.entropy[r] = (float)(H < 0.0 ? 0.0 : H);
        }
    }
    if constexpr (TOP) {
        extern __shared__ uint64_t cand[];
        __shared__ int32_t index[kListed], chosen[kMaxTop + 2], count, found_tiles;
        __shared__ unsigned long long tmax[kMaxTop + 2], bound;
        const int n = j.n_top;
        if (lse != lse || lse == -INFINITY) {
            for (int x = t; x < n; x += NT) {
                j.top_items[r * n + x] = -1;
                j.top_lp[r * n + x] = (float)lse;
            }
            return;
        }
        const int want = min(n + 2, j.v.tiles);
        if (t < 64) {
            const uint32_t b = bound_of(key, want);
            if (t == 0) least_tile = b;
        }
        if (t < want) tmax[t] = 0;
        if (t == 0) count = found_tiles = 0, bound = 0;
        __syncthreads();
        select_tiles<NT>(maxima, want, least_tile, chosen, key, index, found_tiles);
        const uint64_t none = key_of(-INFINITY);
        const auto item_at = [&](int x) { return (int64_t)chosen[x >> 5] * 32 + (x & 31); };
        for (int x = t >> 2; x < want * 32; x += NT / 4) {
            const int64_t i = min(item_at(x), (int64_t)j.n_items - 1);
            const bool in = item_at(x) < j.n_items && !is_excluded(j, r, i);
            const double score = exact_score<T, 4>(j, urow, i, t & 3);
            if ((t & 3) == 0) cand[x] = in ? key_of(score) : none;
        }
        __syncthreads();
        for (int x = t; x < want * 4; x += NT) {  // 8 items each
            uint64_t most = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = max(most, cand[8 * x + ((e + x) & 7)]);
            atomicMax(&tmax[x >> 2], (unsigned long long)most);
        }
        __syncthreads();
        if (t < want) {  // the n-th largest of the tiles' maxima (none where there are fewer tiles)
            int rank = 0;
#pragma unroll 4
            for (int x = 0; x < want; ++x) rank += before(tmax[x], x, tmax[t], t);
            if (rank == n - 1) bound = tmax[t];
        }
        __syncthreads();
        uint64_t least = max((uint64_t)bound, none + 1);
        const auto list = [&] {
            for (int x = t; x < want * 32; x += NT)
                if (cand[x] >= least) {
                    const int at = atomicAdd(&count, 1);
                    if (at < kCandidates) {
                        listed_key[at] = cand[x];
                        index[at] = (int32_t)item_at(x);
                    }
                }
            __syncthreads();
        };
        list();
        if (count > kCandidates) {
            // Few tiles for so many items: the n-th largest key's upper half, bit by bit
            __shared__ int reach[32];
            uint32_t upper = 0;
            __syncthreads();  // (count is read by all)
            if (t < 32) reach[t] = 0;
            if (t == 0) count = 0;
            __syncthreads();
#pragma unroll 1
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t c = upper | 1u << bit;
                int mine = 0;
                for (int x = t; x < want * 32; x += NT)
                    mine += __builtin_popcountll(__ballot((uint32_t)(cand[x] >> 32) >= c));
                if ((t & 63) == 0 && mine) atomicAdd(&reach[bit], mine);
                __syncthreads();
                if (reach[bit] >= n) upper = c;
            }
            least = max(least, (uint64_t)upper << 32);
            list();
        }
        const int found = count;
        const auto place = [&](uint64_t v, int32_t i, int rank) {
            if (rank >= n) return;
            j.top_items[r * n + rank] = i;
            j.top_lp[r * n + rank] = (float)(value_of(v) - lse);
        };
        if (found <= kCandidates) {
            for (int y = t; y < found; y += NT) {
                const uint64_t v = listed_key[y];
                const int32_t i = index[y];
                int rank = 0;
#pragma unroll 4
                for (int z = 0; z < found; ++z) rank += before(listed_key[z], index[z], v, i);
                place(v, i, rank);
            }
        } else {
            for (int y = t; y < want * 32; y += NT) {
                const uint64_t v = cand[y];
                if (v < least) continue;
                const int32_t i = (int32_t)item_at(y);
                int rank = 0;
                for (int z = 0; z < want * 32; ++z) rank += before(cand[z], (int32_t)item_at(z), v, i);
                place(v, i, rank);
            }
        }
        for (int x = found + t; x < n; x += NT) {
            j.top_items[r * n + x] = -1;
            j.top_lp[r * n + x] = -INFINITY;
        }
    }
}

// ------------------------------------------------------------------ gradient
// Both kernels stage a tile's score fragments and its transposed ones.  Where two tiles' fit next to
// other blocks (k <= 128), in two buffers of both: the next tile's are on the way while this one's
// are used, one barrier a tile.  Else in one buffer of each: while the score fragments are used the
// transposed ones are on the way, and the other way round.  A block's waves share the
// streamed tile, and other blocks' waves fill the time at the barriers.  Waves of a block and waves
// per SIMD that the registers are held down to, measured (2048 x 100k, k = 64 f32; 1001 x 30k, k = 100
// f16; 1024 x 500k, k = 256 bf16): users 156 us with 8 and 4 against 199 with 8 and 2; items 206 with
// 4 and 3 against 236 with 8 and 4, which spills (a reload waits for the copies on the way); k > 128:
// users 729 with 4 and 2 against 1,221 with 4 and 1.
// Bound by the matrix cores and power: 1024 x 500k, k = 256 bf16 takes 3 products a side (the scores
// again, G's two planes), 786 Gflop, in 669 us (users) and 723 (items): 1.17 and 1.09 Pflop/s, where a
// large library product reaches 1.23.
template <int T, int KT>
constexpr int users_waves() {
    return KT > 4 ? 4 : 8;
}
template <int T, int KT>
constexpr int users_per_simd() {
    return KT <= 4 ? 4 : KT == 6 ? (T == MML_DTYPE_F32 ? 3 : 4) : KT <= 8 || T != MML_DTYPE_F32 ? 2 : 1;
}
template <int KT>
constexpr int tile_buffers() {
    return KT <= 8 ? 2 : 1;
}
// Steps of the kept fragments that stay in LDS, so that nothing is spilled at those waves per SIMD
template <int T, int KT>
constexpr int users_in_lds() {
    return KT == 16 && T == MML_DTYPE_F16 ? 4 : 0;
}
constexpr int kItemsWaves = 4;
template <int T, int KT>
constexpr int items_per_simd() {
    return KT <= 4 || (KT <= 8 && T != MML_DTYPE_F32) ? 3 : KT <= 8 || T != MML_DTYPE_F32 ? 2 : 1;
}
template <int T, int KT>
constexpr int items_in_lds() {
    return T == MML_DTYPE_F32 ? 0 : KT == 8 ? 4 : KT == 16 ? (T == MML_DTYPE_F16 ? 8 : 6) : 0;
}

// Users' side: as the forward pass, G in place of the softmax state, dU += G V.
template <int T, int KT>
__global__ __launch_bounds__((users_waves<T, KT>() * 64), (users_per_simd<T, KT>())) void
softmax_grad_users_kernel(Job j) {
    using P = Planes<T>;
    constexpr int PS = P::PS, MT = KT > 1 ? KT / 2 : 1, KP = MT * 32, WAVES = users_waves<T, KT>();
    constexpr int NS = PS * KT, NT = P::PG * MT * 2;  // KB of score and of transposed fragments
    constexpr int LK = users_in_lds<T, KT>();
    constexpr int NB = tile_buffers<KT>();
    __shared__ uint4 sbuf[NB][NS * 64], tbuf[NB][NT * 64], kept[WAVES][LK ? PS * LK * 64 : 1];
    __shared__ f32x4 bias[2][8];
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
    const int split = blockIdx.x % j.splits;
    const int64_t ut = (int64_t)(blockIdx.x / j.splits) * WAVES + wave;
    const bool mine = ut < j.u.tiles;  // as in the forward pass
    const int64_t row = (mine ? ut : 0) * 32 + (lane & 31);
    uint4 b[PS][KT - LK], *mykept = kept[wave];
    load_kept<T, KT, LK>(j.u.frag, mine ? ut : 0, b, mykept, lane);
    const RowMeta& meta = j.meta[mine ? ut : 0];
    const float lse2 = meta.lse2[lane & 31], c0 = meta.c0[lane & 31], c1 = meta.c1[lane & 31];
    const int32_t given = meta.t[lane & 31];
    const Scale sc = *j.scale;
    Shift sh;
    f32x16 acc[MT] = {};
    const int t0 = (int)((int64_t)j.v.tiles * split / j.splits);
    const int t1 = (int)((int64_t)j.v.tiles * (split + 1) / j.splits);
    uint32_t word = 0;
    const auto load_trans = [&](int tl, int at) {
        stage<WAVES>(j.v.trans + (int64_t)tl * NT * 64, tbuf[at], NT);
    };
    const auto load = [&](int tl, int at) {
        stage<WAVES>(j.v.frag + (int64_t)tl * NS * 64, sbuf[at], NS);
        if (wave == WAVES - 1 && lane < 8)
            copy_to_lds((const f32x4*)j.vbias + tl * 8 + lane, bias[tl & 1]);
        if (NB == 2) load_trans(tl, at);
        if (j.mask) word = j.mask[row * j.v.tiles + tl];
    };
    if (t0 < t1) load(t0, 0);
    if (!mine) {  // copies its share
        for (int tl = t0, at = 0; tl < t1; ++tl, at ^= NB - 1) {
            stage_wait();
            if (NB == 1) {
                load_trans(tl, 0);
                stage_wait();
            }
            if (tl + 1 < t1) load(tl + 1, NB == 1 ? 0 : at ^ 1);
        }
        return;
    }
    for (int tl = t0, at = 0; tl < t1; ++tl, at ^= NB - 1) {
        stage_wait();
        asm volatile("" : "+v"(word));  // the wait for this load belongs before the next copies
        const uint32_t bits = word >> (4 * h);
        if (NB == 1) load_trans(tl, 0);
        else if (tl + 1 < t1) load(tl + 1, at ^ 1);
        float g[16];
        f32x16 c;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 v = bias[tl & 1][2 * q + h];
#pragma unroll
            for (int e = 0; e < 4; ++e) c[4 * q + e] = v[e];
        }
        c = score_tile<T, KT, LK>(sbuf[at], b, mykept, c, lane);
        if (__any(bits & 0x0F0F0F0Fu)) mask_tile(c, bits, sc.gone);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = fmaf(c[i], sc.kappa, -lse2);
            g[i] = __builtin_amdgcn_exp2f(x) * fmaf(c1, x, c0);
        }
        // G is whole before it is split: w (1 - p) keeps the planes' bits where p is close to 1, which
        // -w p in two planes with w V_t added to the sum afterwards does not
        if (__any(given >> 5 == tl)) {  // a row's given item: rarely
            asm volatile("");  // as in mask_tile
            const float add = given >> 5 == tl ? j.w[row] : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) g[i] += (given & 31) - 4 * h == reg_row(i, 0) ? add : 0.0f;
        }
        if (NB == 1) {
            stage_wait();
            if (tl + 1 < t1) load(tl + 1, 0);
        }
        scale_g<T, MT>(g, acc, sh);
        grad_tile<T, KT>(tbuf[at], g, acc, lane);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[mt][i] = unscale<T>(acc[mt][i], sh, sc.gv);
    float* out = j.du_part + ((int64_t)split * j.rows_pad + row) * KP;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *(f32x4*)&out[32 * mt + 8 * q + 4 * h] =
                f32x4{acc[mt][4 * q], acc[mt][4 * q + 1], acc[mt][4 * q + 2], acc[mt][4 * q + 3]};
}

// Items' side: a wave keeps 32 items and streams the user tiles of its split; dV += G^T U,
// db = the sum of G.
template <int T, int KT>
__global__ __launch_bounds__((kItemsWaves * 64), (items_per_simd<T, KT>())) void
softmax_grad_items_kernel(Job j) {
    using P = Planes<T>;
    constexpr int PS = P::PS, MT = KT > 1 ? KT / 2 : 1, KP = MT * 32, WAVES = kItemsWaves;
    constexpr int NS = PS * KT, NT = P::PG * MT * 2;
    constexpr int LK = items_in_lds<T, KT>();
    constexpr int NB = tile_buffers<KT>();
    __shared__ uint4 sbuf[NB][NS * 64], tbuf[NB][NT * 64], kept[WAVES][LK ? PS * LK * 64 : 1];
    __shared__ __align__(16) RowMeta mbuf[2];
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
    const int whole = j.vwhole / WAVES, rest = (int)blockIdx.x - whole;
    const int splits = rest < 0 ? 1 : j.vsplits, split = rest < 0 ? 0 : rest % splits;
    const int64_t vt = (int64_t)(rest < 0 ? (int)blockIdx.x : whole + rest / splits) * WAVES + wave;
    const bool mine = vt < j.v.tiles;
    const int64_t item = (mine ? vt : 0) * 32 + (lane & 31);
    uint4 b[PS][KT - LK], *mykept = kept[wave];
    load_kept<T, KT, LK>(j.v.frag, mine ? vt : 0, b, mykept, lane);
    const float bias = j.vbias[item];
    const Scale sc = *j.scale;
    Shift sh;
    f32x16 acc[MT] = {};
    float db = 0.0f;
    const int t0 = (int)((int64_t)j.u.tiles * split / splits);
    const int t1 = (int)((int64_t)j.u.tiles * (split + 1) / splits);
    uint32_t next = 0;
    const auto load_trans = [&](int tl, int at) {
        stage<WAVES>(j.u.trans + (int64_t)tl * NT * 64, tbuf[at], NT);
    };
    const auto load = [&](int tl, int at) {
        stage<WAVES>(j.u.frag + (int64_t)tl * NS * 64, sbuf[at], NS);
        if (wave == WAVES - 1 && lane < 32)
            copy_to_lds((const uint4*)(j.meta + tl) + lane, &mbuf[tl & 1]);
        if (NB == 2) load_trans(tl, at);
        if (j.mask) next = j.mask[(tl * 32 + (lane & 31)) * (int64_t)j.v.tiles + (mine ? vt : 0)];
    };
    if (t0 < t1) load(t0, 0);
    for (int tl = t0, at = 0; tl < t1; ++tl, at ^= NB - 1) {
        stage_wait();
        asm volatile("" : "+v"(next));
        const uint32_t word = next;
        if (NB == 1) load_trans(tl, 0);
        else if (tl + 1 < t1) load(tl + 1, at ^ 1);
        float g[16];
        f32x16 c;
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] = bias;
        c = score_tile<T, KT, LK>(sbuf[at], b, mykept, c, lane);
        const RowMeta& meta = mbuf[tl & 1];
        if (__any(word)) {
            asm volatile("");  // as in mask_tile
#pragma unroll
            for (int i = 0; i < 16; ++i) {  // the rows of register i in the lower and upper lanes
                const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)word, reg_row(i, 0));
                const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)word, reg_row(i, 1));
                if (__builtin_amdgcn_inverse_ballot_w64(lo | hi << 32)) c[i] = sc.gone;
            }
        }
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x4 lse2 = *(const f32x4*)&meta.lse2[8 * q + 4 * h];
            const f32x4 c0 = *(const f32x4*)&meta.c0[8 * q + 4 * h];
            const f32x4 c1 = *(const f32x4*)&meta.c1[8 * q + 4 * h];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = fmaf(c[4 * q + e], sc.kappa, -lse2[e]);
                g[4 * q + e] = __builtin_amdgcn_exp2f(x) * fmaf(c1[e], x, c0[e]);
            }
        }
        const int32_t given = meta.t[lane & 31];
        uint32_t hits = (uint32_t)__ballot(given >> 5 == (int32_t)vt);
        while (hits) {  // a given item of the tile's rows among this wave's: rarely
            const int r = __builtin_ctz(hits);
            hits &= hits - 1;
            const bool here = (int32_t)item == __builtin_amdgcn_readlane(given, r);
            const float add = here ? j.w[tl * 32 + r] : 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) g[i] += r - 4 * h == reg_row(i, 0) ? add : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += g[i];
        db += sum;
        if (NB == 1) {
            stage_wait();
            if (tl + 1 < t1) load(tl + 1, 0);
        }
        scale_g<T, MT>(g, acc, sh);
        grad_tile<T, KT>(tbuf[at], g, acc, lane);
    }
    if (!mine) return;
    const int64_t items_pad = (int64_t)j.v.tiles * 32;
    db += __shfl_xor(db, 32);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[mt][i] = unscale<T>(acc[mt][i], sh, sc.gu);
    if (splits == 1) {  // nothing to join: the result itself
        if (item >= j.n_items) return;
        if (h == 0) j.gb[item] = db;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                store_factors<T>(j.gv, item * j.ld_gv, 32 * mt + 8 * q + 4 * h, j.k, j.gv_vec4,
                                 f32x4{acc[mt][4 * q], acc[mt][4 * q + 1], acc[mt][4 * q + 2],
                                       acc[mt][4 * q + 3]});
        return;
    }
    const int64_t first = (int64_t)j.vwhole * 32, parted = items_pad - first;
    float* out = j.dv_part + ((int64_t)split * parted + item - first) * KP;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *(f32x4*)&out[32 * mt + 8 * q + 4 * h] =
                f32x4{acc[mt][4 * q], acc[mt][4 * q + 1], acc[mt][4 * q + 2], acc[mt][4 * q + 3]};
    if (h == 0) j.db_part[split * parted + item - first] = db;
}

// Four factors of a row summed over the splits: `threads` neighbouring threads take every threads-th
// split and are joined in order, so the result is the same every time.
__host__ __device__ __forceinline__ int join_threads(int splits) {  // 1, 2, 4 or 8
    return splits >= 8 ? 8 : splits >= 4 ? 4 : splits >= 2 ? 2 : 1;
}
__device__ __forceinline__ f32x4 join_splits(const float* __restrict__ part, int64_t stride,
                                             int splits, int threads) {
    const int g = threadIdx.x & (threads - 1);
    f32x4 a = {};
#pragma unroll 4
    for (int s = g; s < splits; s += threads) a += *(const f32x4*)(part + s * stride);
    for (int d = 1; d < threads; d <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] += __shfl_xor(a[e], d);
    return a;
}
// The users' rows
template <int T>
__device__ __forceinline__ void join_users(const Job& j, int32_t kp, uint32_t block) {
    const int threads = join_threads(j.splits);
    const int64_t x = ((int64_t)block * 256 + threadIdx.x) / threads;
    const int quads = (j.k + 3) / 4;
    const bool in = x < j.n_rows * quads;  // (all lanes take part in the join)
    const int64_t r = in ? x / quads : 0;
    const int f = in ? 4 * (int)(x % quads) : 0;
    f32x4 a = join_splits(j.du_part + r * kp + f, j.rows_pad * kp, j.splits, threads);
    if (!in || (threadIdx.x & (threads - 1))) return;
    store_factors<T>(j.gu, r * j.ld_gu, f, j.k, j.gu_vec4, a);
}
template <int T>
__device__ __forceinline__ void join_items(const Job& j, int32_t kp, uint32_t block) {
    const int threads = join_threads(j.vsplits);
    const int64_t x = ((int64_t)block * 256 + threadIdx.x) / threads;
    const int64_t first = (int64_t)j.vwhole * 32, parted = (int64_t)j.v.tiles * 32 - first;
    const int quads = (j.k + 3) / 4;
    const bool in = x < (j.n_items - first) * quads;
    const int64_t i = in ? x / quads : 0;  // (from the first item in parts on)
    const int f = in ? 4 * (int)(x % quads) : 0;
    const f32x4 a = join_splits(j.dv_part + i * kp + f, parted * kp, j.vsplits, threads);
    if (!in || (threadIdx.x & (threads - 1))) return;
    store_factors<T>(j.gv, (first + i) * j.ld_gv, f, j.k, j.gv_vec4, a);
    if (f == 0) {
        float b = 0.0f;
        for (int s = 0; s < j.vsplits; ++s) b += j.db_part[s * parted + i];
        j.gb[first + i] = b;
    }
}
// Both in one launch: `users` blocks for the users' rows, then the items' (vsplits > 1).
template <int T>
__global__ __launch_bounds__(256) void softmax_join_kernel(Job j, int32_t kp, uint32_t users) {
    if (blockIdx.x < users) join_users<T>(j, kp, blockIdx.x);
    else join_items<T>(j, kp, blockIdx.x - users);
}

// ------------------------------------------------------------------ host side
int steps_of(int32_t k) {  // KT: the factors padded to 16, 32, 64, 96, 128, 192 or 256
    for (const int kt : {1, 2, 4, 6, 8, 12})
        if (k <= 16 * kt) return kt;
    return 16;
}

template <class F>
void dispatch(int T, int kt, F&& f) {
#define MML_KT(TT)                                                       \
    switch (kt) {                                                        \
        case 1: return f(std::integral_constant<int, TT>{}, std::integral_constant<int, 1>{});   \
        case 2: return f(std::integral_constant<int, TT>{}, std::integral_constant<int, 2>{});   \
        case 4: return f(std::integral_constant<int, TT>{}, std::integral_constant<int, 4>{});   \
        case 6: return f(std::integral_constant<int, TT>{}, std::integral_constant<int, 6>{});   \
        case 8: return f(std::integral_constant<int, TT>{}, std::integral_constant<int, 8>{});   \
        case 12: return f(std::integral_constant<int, TT>{}, std::integral_constant<int, 12>{}); \
        default: return f(std::integral_constant<int, TT>{}, std::integral_constant<int, 16>{}); \
    }
    switch (T) {
        case MML_DTYPE_F32: MML_KT(MML_DTYPE_F32)
        case MML_DTYPE_BF16: MML_KT(MML_DTYPE_BF16)
        default: MML_KT(MML_DTYPE_F16)
    }
#undef MML_KT
}

// How many splits of the streamed side: enough blocks to fill the 256 CUs with as many waves as fit,
// and short ones, so that the last blocks leave little idle; against a fixed cost per block (its kept
// fragments, the first tile) and the join of the splits' results.  kept / streamed: tiles of either
// side; matrix instructions per pair of tiles; bytes a split leaves per kept tile.  In cycles: a wave's
// tile takes 32 per matrix instruction and 500 besides; w waves on a SIMD take (w + 1.5) / 2.5 times as
// long as one (measured: 1.6 times the throughput from one to two, 1.2 from two to four); a block 6,000
// to start; results are written and read back at 8 KB a cycle (in the model's cycles, half the real ones
// a tile: with 2 KB, 1,001 x 30 k, k = 100 f16 took 118 us with 32 and 1 splits, with 8 KB 105 with 64
// and 2).  Above 8, a multiple of the 8 XCDs: block b runs on XCD b mod 8, so a split's blocks share an
// L2.
struct Splits {
    int32_t n = 1, whole = 0;  // kept tiles from `whole` on are split n ways, those before are not
    double cost = 0.0;
};
double block_time(int64_t per_cu, int waves, int instructions, int64_t tiles) {
    return (per_cu * waves / 4.0 + 1.5) / 2.5 * (instructions * 32.0 + 500.0) * tiles + 6000.0;
}
Splits choose_splits(int64_t kept, int64_t streamed, int waves, int per_simd, int instructions,
                     double bytes) {
    const int64_t row_blocks = std::max<int64_t>(1, (kept + waves - 1) / waves);
    const int64_t most_per_cu = std::max(1, per_simd * 4 / waves);
    Splits best;
    for (int64_t s = 1; s <= 1024 && s <= std::max<int64_t>(1, streamed); s += s < 8 ? 1 : 8) {
        const int64_t blocks = row_blocks * s;
        const int64_t per_cu = std::min(most_per_cu, (blocks + 255) / 256);
        const double one = block_time(per_cu, waves, instructions, (streamed + s - 1) / s);
        const double fill = (double)blocks / (256.0 * per_cu);
        const double cost = (fill <= 1.0 ? 1.0 : fill + 0.35) * one +
                            (s > 1 ? s * kept * bytes / 4096.0 : 0.0);
        if (s == 1 || cost < best.cost) best.cost = cost, best.n = (int32_t)s;
    }
    return best;
}
// The same with the kept tiles that fill the CUs a whole number of times left in one piece: a few
// blocks more than fit run alone at the end, and only they are split (2,048 x 100 k, k = 64, 782
// blocks in 768 places: 234 us for the items' gradient, 187 so).
Splits choose_splits_of_rest(int64_t kept, int64_t streamed, int waves, int per_simd,
                             int instructions, double bytes) {
    const Splits all = choose_splits(kept, streamed, waves, per_simd, instructions, bytes);
    const int64_t per_cu = std::max(1, per_simd * 4 / waves);
    const int64_t rounds = kept / waves / (256 * per_cu), whole = rounds * 256 * per_cu * waves;
    if (rounds == 0 || whole == kept) return all;
    Splits rest =
        choose_splits(kept - whole, streamed, waves, per_simd, instructions, bytes);
    rest.cost += rounds * block_time(per_cu, waves, instructions, streamed);
    rest.whole = (int32_t)whole;
    return rest.n > 1 && rest.cost < all.cost ? rest : all;
}

struct Carve {  // a workspace cut into arrays of 256-byte alignment (base null: sizes only)
    char* base;
    int64_t used = 0;
    template <class X>
    X* take(int64_t n) {
        X* p = base ? reinterpret_cast<X*>(base + used) : nullptr;
        used += (n * (int64_t)sizeof(X) + 255) & ~(int64_t)255;
        return p;
    }
};

void check_args(const mml_item_softmax_args* a) {
    MML_REQUIRE(a, "args is null");
    MML_REQUIRE(a->dtype >= MML_DTYPE_F32 && a->dtype <= MML_DTYPE_F16, "unknown dtype");
    MML_REQUIRE(a->num_factors >= 1 && a->num_factors <= 256, "num_factors must be in [1, 256]");
    MML_REQUIRE(a->n_rows >= 0 && a->n_rows <= (int64_t)1 << 30, "bad n_rows");
    MML_REQUIRE((a->n_users >= 1 || a->n_rows == 0) && a->n_items >= 1, "bad n_users or n_items");
    MML_REQUIRE(a->n_items <= 0x7FFFFF00, "n_items too large");
    MML_REQUIRE(a->users || a->n_rows <= a->n_users, "more rows than users");
    MML_REQUIRE(a->ld_users >= a->num_factors && a->ld_items >= a->num_factors,
                "a row stride is shorter than a row");
    MML_REQUIRE(a->n_top >= 0 && a->n_top <= kMaxTop, "n_top must be in [0, 128]");
    MML_REQUIRE(a->n_exclude >= 0, "bad n_exclude");
}

// The launch's numbers and its arrays in the workspace at `base` (nullptr: sizes only).
int64_t plan(const mml_item_softmax_args* a, bool grad, void* base, Job& j) {
    const int T = a->dtype, kt = steps_of(a->num_factors), mt = kt > 1 ? kt / 2 : 1;
    const int ps = T == MML_DTYPE_F32 ? 2 : 1, pg = ps;
    j = Job{};
    j.k = a->num_factors;
    j.n_items = a->n_items;
    j.n_rows = a->n_rows;
    j.n_top = grad ? 0 : a->n_top;
    j.u = Side{a->user_factors, a->ld_users, a->users, a->n_users, a->n_rows,
               (int32_t)((a->n_rows + 31) / 32), nullptr, nullptr, 0};
    j.v = Side{a->item_factors, a->ld_items, nullptr, a->n_items, a->n_items,
               (int32_t)(((int64_t)a->n_items + 32 * kTileGroup - 1) / (32 * kTileGroup) *
                         kTileGroup),
               nullptr, nullptr, 0};
    const int size = T == MML_DTYPE_F32 ? 4 : 2;
    j.u.vec8 = (uintptr_t)a->user_factors % 16 == 0 && a->ld_users * size % 16 == 0;
    j.v.vec8 = (uintptr_t)a->item_factors % 16 == 0 && a->ld_items * size % 16 == 0;
    j.rows_pad = (int64_t)j.u.tiles * 32;
    const int64_t items_pad = (int64_t)j.v.tiles * 32;
    j.bias = a->item_bias;
    j.bias_vec4 = (uintptr_t)a->item_bias % 16 == 0;
    j.target = a->items;
    j.ex_off = a->exclude_offsets;
    j.ex_items = a->exclude_items;
    j.n_ex = a->n_exclude;
    if (grad) {
        dispatch(T, kt, [&](auto tt, auto k) {
            constexpr int TT = decltype(tt)::value, KT = decltype(k)::value;
            constexpr int M = Planes<TT>::PS == 2 ? 6 * KT : 3 * KT;
            j.splits = choose_splits(j.u.tiles, j.v.tiles, users_waves<TT, KT>(),
                                     users_per_simd<TT, KT>(), M, mt * 4096.0).n;
            const Splits v = choose_splits_of_rest(j.v.tiles, j.u.tiles, kItemsWaves,
                                                   items_per_simd<TT, KT>(), M, mt * 4096.0);
            j.vsplits = v.n;
            j.vwhole = v.whole;
        });
    } else if (j.u.tiles <= 1 || (int64_t)j.u.tiles * j.v.tiles * kt <= 16384) {
        // no preparation: one tile of users, or as little work as 100 k items at k = 64 with one (37
        // users, 1,682 items, k = 10: 30 us a call against 36).  Two tiles of items or more a wave.
        j.direct = 1;
        j.splits = (int32_t)std::max<int64_t>(
            1, std::min<int64_t>((j.v.tiles + 2 * kDirectWaves - 1) / (2 * kDirectWaves), 2048));
    } else {
        dispatch(T, kt, [&](auto tt, auto k) {
            constexpr int TT = decltype(tt)::value, KT = decltype(k)::value;
            constexpr int M = Planes<TT>::PS == 2 ? 3 * KT : KT;
            j.splits = choose_splits(j.u.tiles, j.v.tiles / forward_tiles<TT, KT>(),
                                     forward_waves<TT, KT>(), forward_per_simd<TT, KT>(),
                                     M * forward_tiles<TT, KT>(), 384.0).n;
        });
    }
    Carve c{(char*)base};
    if (!j.direct) {
        j.scale = c.take<Scale>(1);
        if (T == MML_DTYPE_F32) j.parts = c.take<float>(kMaxParts);
        j.u.frag = c.take<uint4>((int64_t)j.u.tiles * ps * kt * 64);
        j.v.frag = c.take<uint4>((int64_t)j.v.tiles * ps * kt * 64);
        j.vbias = c.take<float>(items_pad);
    }
    if (a->exclude_offsets) j.mask = c.take<uint32_t>((int64_t)j.v.tiles * j.rows_pad);
    if (!grad) {
        j.part = c.take<float>((int64_t)j.splits * 3 * j.rows_pad);
        j.cpad = j.v.tiles;
        if (j.n_top) j.cmax = c.take<float>(j.rows_pad * j.cpad);
    } else {
        j.u.trans = c.take<uint4>((int64_t)j.u.tiles * pg * mt * 128);
        j.v.trans = c.take<uint4>((int64_t)j.v.tiles * pg * mt * 128);
        j.meta = c.take<RowMeta>(j.u.tiles);
        j.w = c.take<float>(j.rows_pad);
        j.du_part = c.take<float>((int64_t)j.splits * j.rows_pad * mt * 32);
        if (j.vsplits > 1) {
            const int64_t parted = items_pad - (int64_t)j.vwhole * 32;
            j.dv_part = c.take<float>(j.vsplits * parted * mt * 32);
            j.db_part = c.take<float>(j.vsplits * parted);
        }
    }
    return std::max<int64_t>(c.used, 256);
}

uint32_t grid_of(int64_t n) {
    if (n > 0x7FFFFFFF) mml::fail(MML_ERR_ARG, "too many rows or items for one launch");
    return (uint32_t)n;
}

// The mask, the scales and the fragments (direct: the mask only)
void prepare(const Job& j, int T, hipStream_t st) {
    dispatch(T, 1, [&](auto tt, auto) {
        const int64_t parts = (j.v.tiles + kMaskWords - 1) / kMaskWords;
        const int64_t blocks = (j.parts ? kMaxParts : 0) + (j.mask ? j.rows_pad * parts : 0);
        const size_t lds = j.mask ? std::min(j.v.tiles, kMaskWords) * sizeof(uint32_t) : 0;
        if (blocks)
            softmax_start_kernel<decltype(tt)::value><<<grid_of(blocks), 256, lds, st>>>(j);
    });
    if (j.direct) return;
    dispatch(T, steps_of(j.k), [&](auto tt, auto kt) {
        softmax_prep_kernel<decltype(tt)::value, decltype(kt)::value>
            <<<grid_of((int64_t)j.u.tiles + j.v.tiles), 256, 0, st>>>(j);
    });
}

void check_pointers(const mml_item_softmax_args* a, const void* ws, int64_t ws_bytes,
                    int64_t need) {
    MML_REQUIRE(a->user_factors && a->item_factors, "null factors");
    MML_REQUIRE(!a->exclude_offsets || a->n_exclude == 0 || a->exclude_items,
                "exclude_offsets without exclude_items");
    MML_REQUIRE(ws && ws_bytes >= need, "workspace too small");
    MML_REQUIRE((uintptr_t)ws % 256 == 0, "workspace must be aligned to 256 bytes");
}

}  // namespace

namespace mml {

void item_log_probs(const mml_item_softmax_args* a, float* log_probs, float* log_norm,
                    float* entropy, int32_t* top_items, float* top_log_probs, void* ws,
                    int64_t ws_bytes, hipStream_t st) {
    check_args(a);
    if (a->n_rows == 0) return;
    Job j;
    const int64_t need = plan(a, false, ws, j);
    check_pointers(a, ws, ws_bytes, need);
    MML_REQUIRE(log_probs && log_norm && entropy, "null output");
    MML_REQUIRE(a->n_top == 0 || (top_items && top_log_probs), "n_top without its outputs");
    j.log_probs = log_probs;
    j.log_norm = log_norm;
    j.entropy = entropy;
    j.top_items = top_items;
    j.top_lp = top_log_probs;
    prepare(j, a->dtype, st);
    const uint32_t direct_blocks = grid_of((int64_t)j.u.tiles * j.splits);
    dispatch(a->dtype, steps_of(j.k), [&](auto tt, auto kt) {
        constexpr int T = decltype(tt)::value, KT = decltype(kt)::value;
        constexpr int W = forward_waves<T, KT>();
        if (j.direct) {
            if (j.n_top)
                softmax_direct_kernel<T, KT, true><<<direct_blocks, kDirectWaves * 64, 0, st>>>(j);
            else
                softmax_direct_kernel<T, KT, false><<<direct_blocks, kDirectWaves * 64, 0, st>>>(j);
            return;
        }
        const uint32_t blocks = grid_of((int64_t)((j.u.tiles + W - 1) / W) * j.splits);
        if (j.n_top)
            softmax_forward_kernel<T, KT, true><<<blocks, W * 64, 0, st>>>(j);
        else
            softmax_forward_kernel<T, KT, false><<<blocks, W * 64, 0, st>>>(j);
    });
    const uint32_t lds = std::min(j.n_top + 2, j.v.tiles) * 32 * sizeof(uint64_t);
    dispatch(a->dtype, 1, [&](auto tt, auto) {
        constexpr int T = decltype(tt)::value;
        if (!j.n_top)
            softmax_finish_kernel<T, 64><<<grid_of(j.n_rows), 64, 0, st>>>(j);
        else if (j.n_rows <= 512)
            softmax_finish_kernel<T, 1024><<<grid_of(j.n_rows), 1024, lds, st>>>(j);
        else
            softmax_finish_kernel<T, 256><<<grid_of(j.n_rows), 256, lds, st>>>(j);
    });
    MML_HIP(hipGetLastError());
}

int64_t item_log_probs_workspace(const mml_item_softmax_args* a, bool grad) {
    check_args(a);
    Job j;
    return plan(a, grad, nullptr, j);
}

void item_log_probs_grad(const mml_item_softmax_args* a, const float* log_norm,
                         const float* entropy, const float* g_lp, const float* g_ent, void* gu,
                         int64_t ld_gu, void* gv, int64_t ld_gv, float* gb, void* ws,
                         int64_t ws_bytes, hipStream_t st) {
    check_args(a);
    Job j;
    const int64_t need = plan(a, true, ws, j);
    MML_REQUIRE(gv && gb && (gu || a->n_rows == 0), "null output");
    MML_REQUIRE(ld_gu >= a->num_factors && ld_gv >= a->num_factors,
                "a gradient's row stride is shorter than a row");
    if (a->n_rows > 0) {
        check_pointers(a, ws, ws_bytes, need);
        MML_REQUIRE(log_norm, "null log_norm");
        MML_REQUIRE(!g_ent || entropy, "grad_entropy without entropy");
        MML_REQUIRE(!g_lp || a->items, "grad_log_probs without items");
    } else {
        MML_REQUIRE(ws && ws_bytes >= need, "workspace too small");
    }
    j.in_norm = log_norm;
    j.in_entropy = entropy;
    j.g_lp = g_lp;
    j.g_ent = g_ent;
    j.gu = gu;
    j.gv = gv;
    j.ld_gu = ld_gu;
    j.ld_gv = ld_gv;
    j.gb = gb;
    const int size = a->dtype == MML_DTYPE_F32 ? 4 : 2;
    j.gu_vec4 = j.k % 4 == 0 && ld_gu % 4 == 0 && (uintptr_t)gu % (4 * size) == 0;
    j.gv_vec4 = j.k % 4 == 0 && ld_gv % 4 == 0 && (uintptr_t)gv % (4 * size) == 0;
    const int kt0 = steps_of(j.k), kp = std::max(32, kt0 * 16);
    if (a->n_rows > 0) prepare(j, a->dtype, st);
    const int64_t quads = (j.k + 3) / 4;
    const uint32_t ju = grid_of((j.n_rows * quads * join_threads(j.splits) + 255) / 256);
    const uint32_t ji =
        j.vsplits > 1
            ? grid_of(((j.n_items - (int64_t)j.vwhole * 32) * quads * join_threads(j.vsplits) + 255) / 256)
            : 0;
    dispatch(a->dtype, kt0, [&](auto tt, auto kt) {
        constexpr int T = decltype(tt)::value, KT = decltype(kt)::value, UW = users_waves<T, KT>();
        constexpr int IW = kItemsWaves;
        const uint32_t ub = grid_of((int64_t)((j.u.tiles + UW - 1) / UW) * j.splits);
        const uint32_t vb = grid_of(j.vwhole / IW +
                                    (int64_t)((j.v.tiles - j.vwhole + IW - 1) / IW) * j.vsplits);
        if (j.n_rows > 0) softmax_grad_users_kernel<T, KT><<<ub, UW * 64, 0, st>>>(j);
        softmax_grad_items_kernel<T, KT><<<vb, IW * 64, 0, st>>>(j);
        if (ju + ji) softmax_join_kernel<T><<<grid_of((int64_t)ju + ji), 256, 0, st>>>(j, kp, ju);
    });
    MML_HIP(hipGetLastError());
}

void check_model_log_probs(const int32_t* users, int64_t n, int32_t n_top, const float* log_probs,
                           const float* log_norm, const float* entropy, const int32_t* top_items,
                           const float* top_log_probs) {
    MML_REQUIRE(n >= 0 && n <= (int64_t)1 << 30, "bad n");
    MML_REQUIRE(n_top >= 0 && n_top <= kMaxTop, "n_top must be in [0, 128]");
    MML_REQUIRE(n == 0 || users, "null users");
    MML_REQUIRE(n == 0 || (log_probs && log_norm && entropy), "null output");
    MML_REQUIRE(n == 0 || n_top == 0 || (top_items && top_log_probs), "n_top without its outputs");
}

void model_log_probs(hipStream_t st, mml_item_softmax_args a, LogProbsWork& w, const int32_t* users,
                     const int32_t* items, int64_t n, int32_t n_top, float* log_probs,
                     float* log_norm, float* entropy, int32_t* top_items, float* top_log_probs) {
    int64_t rows = n;
    a.n_top = n_top;
    a.users = users;  // (only whether there are any matters to the size)
    a.items = items;
    for (;; rows = (rows / 2 + 31) / 32 * 32) {
        a.n_rows = rows;
        if (rows <= 32 || item_log_probs_workspace(&a, false) <= (int64_t)1 << 30) break;
    }
    w.ids.reserve(2 * rows);
    w.out.reserve((3 + 2 * (int64_t)n_top) * rows);
    for (int64_t r = 0; r < n; r += rows) {
        const int64_t m = std::min(rows, n - r);
        a.n_rows = m;
        const int64_t need = item_log_probs_workspace(&a, false);
        w.ws.reserve(need);
        float* out = w.out.get();
        int32_t* top = reinterpret_cast<int32_t*>(out + 3 * m);
        float* top_lp = out + (3 + n_top) * m;
        MML_HIP(hipMemcpyAsync(w.ids.get(), users + r, 4 * m, hipMemcpyHostToDevice, st));
        if (items)
            MML_HIP(hipMemcpyAsync(w.ids.get() + m, items + r, 4 * m, hipMemcpyHostToDevice, st));
        a.users = w.ids.get();
        a.items = items ? w.ids.get() + m : nullptr;
        item_log_probs(&a, out, out + m, out + 2 * m, top, top_lp, w.ws.get(), need, st);
        const auto copy = [&](void* to, const void* from, int64_t words) {
            if (words > 0) MML_HIP(hipMemcpyAsync(to, from, 4 * words, hipMemcpyDeviceToHost, st));
        };
        copy(log_probs + r, out, m);
        copy(log_norm + r, out + m, m);
        copy(entropy + r, out + 2 * m, m);
        copy(top_items + r * n_top, top, m * n_top);
        copy(top_log_probs + r * n_top, top_lp, m * n_top);
        MML_HIP(hipStreamSynchronize(st));
    }
}

}  // namespace mml

using mml::guard;

extern "C" mml_status mml_item_log_probs_workspace(const mml_item_softmax_args* args, int32_t grad,
                                                   int64_t* bytes) {
    return guard([&] {
        MML_REQUIRE(bytes, "bytes is null");
        *bytes = mml::item_log_probs_workspace(args, grad != 0);
    });
}

extern "C" mml_status mml_item_log_probs_device(const mml_item_softmax_args* args, float* log_probs,
                                                float* log_norm, float* entropy, int32_t* top_items,
                                                float* top_log_probs, void* workspace,
                                                int64_t workspace_bytes, int32_t device,
                                                void* stream) {
    return guard([&] {
        mml::DeviceScope on(device);
        mml::item_log_probs(args, log_probs, log_norm, entropy, top_items, top_log_probs, workspace,
                            workspace_bytes, (hipStream_t)stream);
    });
}

extern "C" mml_status mml_item_log_probs_grad_device(
    const mml_item_softmax_args* args, const float* log_norm, const float* entropy,
    const float* grad_log_probs, const float* grad_entropy, void* grad_users, int64_t ld_grad_users,
    void* grad_items, int64_t ld_grad_items, float* grad_bias, void* workspace,
    int64_t workspace_bytes, int32_t device, void* stream) {
    return guard([&] {
        mml::DeviceScope on(device);
        mml::item_log_probs_grad(args, log_norm, entropy, grad_log_probs, grad_entropy, grad_users,
                                 ld_grad_users, grad_items, ld_grad_items, grad_bias, workspace,
                                 workspace_bytes, (hipStream_t)stream);
    });
}
