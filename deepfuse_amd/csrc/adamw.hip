// adamw.hip -- the AdamW update (decoupled weight decay) over lists of tensors,
// its states in binary32 or in 8 bits (gfx950).
//
// Per element, every operation rounded to binary32 as written (no fused
// multiply-adds; IEEE division and square root):
//   g = grad * f                       f: the clip factor (1 when not clipping)
//   m = b1*m + (1-b1)*g;  v = b2*v + ((1-b2)*g)*g
//   p = p*(1 - lr*wd) - (lr*(m / (1-b1^t))) / (sqrt(v / (1-b2^t)) + eps)
//
// 8-bit states: 256 consecutive values of a tensor share a binary32 scale.
// m is kept as e4m3 codes of m / scale, scale = max|m| / 448 over the block's
// finite values; v as codes of sqrt(v), which the update needs anyway: e4m3
// spans 2^-9 to 448, so the square root covers 2^35 of v in one block.  A v
// above 0 never goes to code 0: the next step would divide its m by eps alone.
// The update itself uses the binary32 m and v; only what is kept is rounded, to
// 4 significant bits.
//
// To nearest, what one step keeps is off by at most 2^-4 of the value (or 2^-10
// of the scale), but the next step starts from there.  A step lowers a root by
// at most (1 - b2)/2 of itself, 2.5% at b2 = 0.95 and 0.05% at 0.999, and codes
// lie 6 to 12% apart: rounded to nearest, a falling root goes back to its code
// until the scale moves.  Half a block's gradients falling tenfold leave its
// roots up to ten times too large, for good where the gradients are steady.
// Dithered rounding (df_adamw_update_dithered) takes the upper of two codes with
// the probability of the value's place between them, so that a root moves as
// often as it should.  Its noise: a move of a share d of a code gap w is made with
// probability d, variance d w^2 at most, and dies away by b2 a step; with d w <= 2
// (1 - b2)/2 of the root (its own move and the scale's) and w <= 1/8 of it that is
// a variance of (1 - b2)/8 a step over 1 - b2^2, or 1 / (8 (1 + b2)): a standard
// deviation of a quarter of the root at most, however near b2 is to 1 (measured:
// 0.12 to 0.17, a third in the middle of a tenfold fall).  Two GPT-2 XL blocks (61.5M
// values) 214 us dithered, 194 to nearest.
//
// Bound by HBM: 24 bytes and the gradient per element with binary32 states,
// 12.1 and the gradient with 8-bit ones.  A wave takes 256 values at a time,
// four consecutive ones per lane, which is also the block of a scale: 16-byte
// accesses of p (m, v), 4-byte ones of codes, and the block's maxima fold
// across the wave's lanes (DPP) without leaving registers.
//
// Extends the reference's optimizer set, whose Adam couples the decay
// (dnn/optimizers/adam_optimizer.cu:24-30); no counterpart of the rest.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "df_common.hpp"

// Rounding of every operation as written: no fused multiply-adds.
#pragma clang fp contract(off)

namespace dfk {

namespace {

constexpr int kWThreads = 256;
constexpr int kUnit = 256;                              // values of a wave at a time, and of a scale
constexpr int kUnits = 4;                               // units whose loads are in flight together
constexpr int kRounds = 2;
constexpr int kWaves = kWThreads / 64;
constexpr int kSpan = kUnit * kUnits * kRounds * kWaves;  // values of a block
constexpr int kWList = 40;                              // tensors of a launch (their table is in the arguments)

struct WTensor {
    float* p;
    const void* g;
    void* m;
    void* v;
    float* ms;
    float* vs;
    uint16_t* copy;
    int64_t n;
};
struct WList {
    WTensor t[kWList];
    float wd[kWList];
    int first[kWList + 1];  // first block of each tensor; first[count] = blocks
    int idx[kWList];        // position in the caller's list
    int count;
};
struct WHyper {
    float lr, b1, b2, omb1, omb2, eps, max_norm;
    float bc1, bc2;         // 1 - beta^t, unless step is given
    int t;                  // likewise, and
    uint32_t seed;          // for the dither
    const float* lr_dev;
    const int* step;
    const float* norm;
    uint32_t* absmax;
};

// 1 - beta^t: beta^t by squaring in binary64, rounded once to binary32; the
// same operations on host and device, so both forms of the step agree
__host__ __device__ inline float bias_corr(float beta, int t) {
    double r = 1.0, b = beta;
    for (int k = t < 1 ? 1 : t; k > 0; k >>= 1) {
        if (k & 1) r = r * b;
        b = b * b;
    }
    return 1.0f - (float)r;
}

// 16, 8 or 4 bytes at element alignment (in structs: a template argument loses
// a type's alignment)
struct F4 { typedef f32x4 V __attribute__((aligned(4))); };
struct H4 { typedef u32x2 V __attribute__((aligned(2))); };
struct B4 { typedef uint32_t V __attribute__((aligned(1))); };

// Lists larger than the 256 MB Infinity Cache stream past it: two GPT-2 XL
// blocks (61.5M values, 8-bit states, 1 GB moved) 194 us against 205 with
// plain accesses.  Smaller ones stay in it for whoever reads the parameters
// next: one GPT-2 small block (7M values, 32-bit states) 30.6 us plain, 34.7
// past the cache.
constexpr int64_t kColdBytes = (int64_t)256 << 20;
template <bool NT, typename A> __device__ __forceinline__ auto ldv(const void* p) {
    const typename A::V* const q = static_cast<const typename A::V*>(p);
    if constexpr (NT) return __builtin_nontemporal_load(q);
    else return *q;
}
template <bool NT, typename A, typename X> __device__ __forceinline__ void stv(void* p, X v) {
    typename A::V* const q = static_cast<typename A::V*>(p);
    if constexpr (NT) __builtin_nontemporal_store(v, q);
    else *q = v;
}

// maximum over the wave (VALU only): rows of 16 lanes, then across them
__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
#define DF_DPP_MAX(CTRL) x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, true))
    DF_DPP_MAX(0x111);  // row_shr:1
    DF_DPP_MAX(0x112);  // row_shr:2
    DF_DPP_MAX(0x114);  // row_shr:4
    DF_DPP_MAX(0x118);  // row_shr:8: lane 15 of a row has the row's
    DF_DPP_MAX(0x142);  // row_bcast:15
    DF_DPP_MAX(0x143);  // row_bcast:31: lane 63 has the wave's
#undef DF_DPP_MAX
    return (uint32_t)__builtin_amdgcn_readlane((int)x, 63);
}

template <typename G> __device__ __forceinline__ float grad_one(const G* p);
template <> __device__ __forceinline__ float grad_one<float>(const float* p) { return *p; }
template <> __device__ __forceinline__ float grad_one<uint16_t>(const uint16_t* p) { return bf16_to_f32(*p); }
template <> __device__ __forceinline__ float grad_one<f16_t>(const f16_t* p) {
    return (float)__builtin_bit_cast(_Float16, p->bits);
}

// four gradients as loaded, and widened
template <typename G> struct Grad4 {
    u32x2 w;
    template <bool NT> __device__ __forceinline__ void load(const G* p) {
        w = ldv<NT, H4>(p);
    }
    __device__ __forceinline__ void widen(float* g) const {
        if constexpr (std::is_same<G, uint16_t>::value) {
            g[0] = __uint_as_float(w.x << 16); g[1] = __uint_as_float(w.x & 0xFFFF0000u);
            g[2] = __uint_as_float(w.y << 16); g[3] = __uint_as_float(w.y & 0xFFFF0000u);
        } else {
            g[0] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w.x & 0xFFFFu));
            g[1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w.x >> 16));
            g[2] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w.y & 0xFFFFu));
            g[3] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w.y >> 16));
        }
    }
};
template <> struct Grad4<float> {
    f32x4 w;
    template <bool NT> __device__ __forceinline__ void load(const float* p) {
        w = ldv<NT, F4>(p);
    }
    __device__ __forceinline__ void widen(float* g) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) g[e] = w[e];
    }
};

__device__ __forceinline__ void decode4(uint32_t w, float s, float* v) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = a.x * s; v[1] = a.y * s; v[2] = b.x * s; v[3] = b.y * s;
}

// the scale of a block whose largest finite magnitude is the pattern `am`
__device__ __forceinline__ float block_scale(uint32_t am) {
    const float a = __uint_as_float(am);
    return am ? __builtin_fmaxf(a / 448.0f, 0x1p-126f) : 1.0f;
}

// ---- dithered rounding ----
// 32 bits from 32: xor-shifts and odd multipliers in turn (the first digits of
// the square roots of 2 and 3).
__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    x *= 0xBB67AE85u;
    return x ^ (x >> 16);
}
// the draw of value i under a key of its own for each seed, step and tensor
__device__ __forceinline__ uint32_t draw(uint32_t key, int64_t i) {
    return mix(key + (uint32_t)i * 0x9E3779B9u + (uint32_t)(i >> 32) * 0xBB67AE85u);
}

// y to one of the e4m3 values next to it by 16 random bits r, at most 448: r is
// added below the 3 bits of mantissa that stay, and the others are cut.  Below
// 2^-6 e4m3 is even, in steps of 2^-9, as from 2^-6 to 2^-5: such a value goes
// there and back.  r stands for the middle of its interval, so that a value of
// e4m3 stays.
__device__ __forceinline__ float dither_e4m3(float y, uint32_t r) {
    const float a = __builtin_fabsf(y), up = a < 0x1p-6f ? 0x1p-6f : 0.0f;
    const float n = __uint_as_float((__float_as_uint(a + up) + (r << 4) + 8u) & 0xFFF00000u) - up;
    return __builtin_copysignf(__builtin_fminf(n, 448.0f), y);
}

template <int COPY> __device__ __forceinline__ uint32_t copy_bits(float v) {
    return COPY == DF_DTYPE_HALF ? f32_to_f16_rne(v) : f32_to_bf16_rne(v);
}

// ---- the same results in fewer operations ----
// An IEEE division is eleven instructions and a square root about fifteen, and
// the update of a value with 8-bit states has five and two: 249 us for two
// GPT-2 XL blocks (61.5M values) against the 192 us that its bytes take.  Where
// m and v of a wave's 256 values are zero or of ordinary size (kOdd below
// names the others, and 2^20 and more), shorter forms give the same bits:
//  - x / c for a divisor that the wave shares: RN(1/c) once, then Markstein's
//    two corrections (a faithful quotient, its exact remainder, and the last
//    fma rounds correctly).  x is first multiplied by 2^64, which is exact, so
//    that the remainders do not underflow.
//  - sqrt(x): the hardware's, good to a unit in the last place, and Tuckerman's
//    test: s is right when s*(s-) < x <= s*(s+), with s- and s+ its neighbours,
//    decided by the signs of two fma remainders; x again times 2^64, so the
//    root times 2^32.
// 2^64 and 2^32 then go out in multiplications that there are anyway.
constexpr int kOdd = 0x297;  // v_cmp_class: NaN, infinity, subnormal

struct ByShared {  // division by c
    float c, r;
    __device__ __forceinline__ float operator()(float x) const {
        const float y0 = x * r;
        const float y1 = __builtin_fmaf(__builtin_fmaf(-c, y0, x), r, y0);
        return __builtin_fmaf(__builtin_fmaf(-c, y1, x), r, y1);
    }
};

__device__ __forceinline__ float root_normal(float x) {  // x: 0 or in [2^-62, 2^124]
    const float s = __builtin_amdgcn_sqrtf(x);
    const float below = __uint_as_float(__float_as_uint(s) - 1u), above = __uint_as_float(__float_as_uint(s) + 1u);
    float y = __builtin_fmaf(-below, s, x) <= 0.0f ? below : s;
    y = __builtin_fmaf(-above, s, x) > 0.0f ? above : y;
    return x > 0.0f ? y : 0.0f;
}

// COPY: DF_DTYPE_BFLOAT16 or DF_DTYPE_HALF: the updated parameters are also
// written in that type; -1: not.  NT: the list is larger than the cache.
// DITHER: 8-bit states are rounded by dither.
template <typename G, bool S8, int COPY, bool NT, bool DITHER>
__global__ __launch_bounds__(kWThreads) void adamw_kernel(const WList L, const WHyper h) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo = 0, hi = L.count - 1;  // the tensor that owns this block: the last with first <= blockIdx.x
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (L.first[mid] <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const WTensor t = L.t[lo];
    const G* gp = static_cast<const G*>(t.g);
    float f = 1.0f;
    if (h.norm) {
        const float nv = h.norm[0];
        if (nv > h.max_norm) f = h.max_norm / nv;
    }
    const float lr = h.lr_dev ? h.lr_dev[0] : h.lr;
    float bc1 = h.bc1, bc2 = h.bc2;
    if (h.step) {
        bc1 = bias_corr(h.b1, h.step[0]);
        bc2 = bias_corr(h.b2, h.step[0]);
    }
    const float keep = 1.0f - lr * L.wd[lo];
    uint32_t am = 0;
    uint32_t key = 0;
    if constexpr (DITHER)
        key = mix(mix(mix(h.seed) + (uint32_t)(h.step ? max(h.step[0], 1) : h.t)) + (uint32_t)L.idx[lo]);

    const ByShared by1{bc1, 1.0f / bc1}, by2{bc2, 1.0f / bc2};
    const float lr64 = lr * 0x1p-64f;
    // the quotients' and roots' conditions on what the wave shares: 1 - beta^t
    // in [2^-40, 1], the rate's products above the smallest normal number
    const bool quick = bc1 >= 0x1p-40f && bc1 <= 1.0f && bc2 >= 0x1p-40f && bc2 <= 1.0f && lr >= 0x1p-40f &&
                       lr <= 0x1p40f;

    // new m and v; whether every value of the wave's takes the quick forms
    auto moments = [&](const float* g, float* m, float* v) __attribute__((always_inline)) -> bool {
        bool odd = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float ge = g[e] * f;
            m[e] = h.b1 * m[e] + h.omb1 * ge;
            v[e] = h.b2 * v[e] + h.omb2 * ge * ge;
            odd |= __builtin_amdgcn_classf(m[e], kOdd) | __builtin_amdgcn_classf(v[e], kOdd);
            odd |= __builtin_fmaxf(__builtin_fabsf(m[e]), v[e]) >= 0x1p20f;
        }
        return quick && __builtin_amdgcn_ballot_w64(odd) == 0;
    };
    // QUICK: root[e] is sqrt(v[e]) afterwards
    auto update = [&](auto how, float* p, const float* m, const float* v, float* root) __attribute__((always_inline)) {
        constexpr bool QUICK = decltype(how)::value;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (QUICK) {
                const float v64 = v[e] * 0x1p64f;
                // 2^32 times the root, a product that is exact, and one rounding: that of root + eps
                const float d = __builtin_fmaf(root_normal(by2(v64)), 0x1p-32f, h.eps);
                // (the corrections turn -0 into 0)
                p[e] = p[e] * keep - lr64 * __builtin_copysignf(by1(m[e] * 0x1p64f), m[e]) / d;
                if (S8) root[e] = root_normal(v64) * 0x1p-32f;
            } else {
                p[e] = p[e] * keep - lr * (m[e] / bc1) / (__builtin_sqrtf(v[e] / bc2) + h.eps);
                if (S8) root[e] = __builtin_sqrtf(v[e]);
            }
        }
        if (h.absmax) {
#pragma unroll
            for (int e = 0; e < 4; ++e) am = fold_f32(am, __float_as_uint(p[e]));
        }
    };
    // codes and scale of a unit's values; ROOT: roots, which above 0 go to code 1 at least
    auto encode = [&](const float* x, auto root, bool plain, float& s, const uint32_t* rnd)
                      __attribute__((always_inline)) -> uint32_t {
        constexpr bool ROOT = decltype(root)::value;
        uint32_t a = 0;
        if (plain) {  // no NaN or infinity among them
            a = __float_as_uint(__builtin_fmaxf(__builtin_fmaxf(__builtin_fabsf(x[0]), __builtin_fabsf(x[1])),
                                                __builtin_fmaxf(__builtin_fabsf(x[2]), __builtin_fabsf(x[3]))));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) a = fold_f32(a, __float_as_uint(x[e]));
        }
        s = block_scale(wave_umax(a));
        float y[4];
        if constexpr (DITHER) {
            const float inv = 1.0f / s;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = x[e] * inv;
                if (ROOT) y[e] = x[e] > 0.0f ? __builtin_fmaxf(y[e], 0x1p-9f) : y[e];
                const float z = dither_e4m3(y[e], ROOT ? rnd[e] >> 16 : rnd[e] & 0xFFFFu);
                y[e] = plain || __builtin_fabsf(y[e]) <= 448.0f ? z : y[e];  // others are saturated or NaN
            }
            if (plain) {
                const int lo2 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
                return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo2, true);
            }
            return encode2_hw<E4M3>(y[0], y[1]) | (encode2_hw<E4M3>(y[2], y[3]) << 16);
        }
        if (plain && s >= 0x1p-40f && s <= 0x1p40f) {
            // quotients of at most 448 (so no clamp); one whose remainders
            // underflow is below 2^-17 and goes to code 0 whatever its last bits
            const ByShared by{s, 1.0f / s};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = by(x[e]);
                if (ROOT) y[e] = x[e] > 0.0f ? __builtin_fmaxf(y[e], 0x1p-9f) : y[e];
                else y[e] = __builtin_copysignf(y[e], x[e]);  // the corrections turn -0 into 0
            }
            const int lo2 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo2, true);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            y[e] = x[e] / s;
            if (ROOT) y[e] = x[e] > 0.0f ? __builtin_fmaxf(y[e], 0x1p-9f) : y[e];
        }
        return encode2_hw<E4M3>(y[0], y[1]) | (encode2_hw<E4M3>(y[2], y[3]) << 16);
    };

    // the units base, base + STRIDE, ... of this wave, kUnits of them in flight
    const auto units = [&](auto by, const int64_t base) __attribute__((always_inline)) {
        constexpr int stride = decltype(by)::value;
        for (int round = 0; round < kRounds; ++round) {
            const int64_t u0 = base + (int64_t)round * kUnits * stride;
            if (u0 >= t.n) break;
            if (u0 + (kUnits - 1) * stride + kUnit <= t.n) {
                f32x4 rp[kUnits], rm[S8 ? 1 : kUnits], rv[S8 ? 1 : kUnits];
                uint32_t cm[S8 ? kUnits : 1], cv[S8 ? kUnits : 1];
                float sm[S8 ? kUnits : 1], sv[S8 ? kUnits : 1];
                Grad4<G> rg[kUnits];
#pragma unroll
                for (int u = 0; u < kUnits; ++u) {
                    const int64_t i = u0 + u * stride + lane * 4;
                    rg[u].template load<NT>(gp + i);
                    rp[u] = ldv<NT, F4>(t.p + i);
                    if constexpr (S8) {
                        cm[u] = ldv<NT, B4>(static_cast<const uint8_t*>(t.m) + i);
                        cv[u] = ldv<NT, B4>(static_cast<const uint8_t*>(t.v) + i);
                        sm[u] = t.ms[(u0 + u * stride) >> 8];
                        sv[u] = t.vs[(u0 + u * stride) >> 8];
                    } else {
                        rm[u] = ldv<NT, F4>(static_cast<const float*>(t.m) + i);
                        rv[u] = ldv<NT, F4>(static_cast<const float*>(t.v) + i);
                    }
                }
#pragma unroll
                for (int u = 0; u < kUnits; ++u) {
                    const int64_t i = u0 + u * stride + lane * 4;
                    float p[4], g[4], m[4], v[4];
                    rg[u].widen(g);
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = rp[u][e];
                    if constexpr (S8) {
                        decode4(cm[u], sm[u], m);
                        decode4(cv[u], sv[u], v);
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] *= v[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            m[e] = rm[u][e];
                            v[e] = rv[u][e];
                        }
                    }
                    float root[4];
                    const bool plain = moments(g, m, v);
                    if (plain) update(std::true_type{}, p, m, v, root);
                    else update(std::false_type{}, p, m, v, root);
                    stv<NT, F4>(t.p + i, f32x4{p[0], p[1], p[2], p[3]});
                    if constexpr (COPY >= 0)
                        stv<NT, H4>(t.copy + i,
                                u32x2{copy_bits<COPY>(p[0]) | (copy_bits<COPY>(p[1]) << 16),
                                      copy_bits<COPY>(p[2]) | (copy_bits<COPY>(p[3]) << 16)});
                    if constexpr (S8) {
                        float s0, s1;
                        uint32_t rnd[4] = {};
                        if constexpr (DITHER) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) rnd[e] = draw(key, i + e);
                        }
                        const uint32_t c0 = encode(m, std::false_type{}, plain, s0, rnd);
                        const uint32_t c1 = encode(root, std::true_type{}, plain, s1, rnd);
                        stv<NT, B4>(static_cast<uint8_t*>(t.m) + i, c0);
                        stv<NT, B4>(static_cast<uint8_t*>(t.v) + i, c1);
                        if (lane == 0) {
                            t.ms[(u0 + u * stride) >> 8] = s0;
                            t.vs[(u0 + u * stride) >> 8] = s1;
                        }
                    } else {
                        stv<NT, F4>(static_cast<float*>(t.m) + i, f32x4{m[0], m[1], m[2], m[3]});
                        stv<NT, F4>(static_cast<float*>(t.v) + i, f32x4{v[0], v[1], v[2], v[3]});
                    }
                }
                continue;
            }
            // the tensor's end: value by value; what lies past it counts as 0
            for (int64_t ub = u0; ub < t.n && ub < u0 + kUnits * stride; ub += stride) {
                float p[4], g[4], m[4], v[4];
                float s0 = 0.0f, s1 = 0.0f;
                if constexpr (S8) {
                    s0 = t.ms[ub >> 8];
                    s1 = t.vs[ub >> 8];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t i = ub + lane * 4 + e;
                    const bool in = i < t.n;
                    p[e] = in ? t.p[i] : 0.0f;
                    g[e] = in ? grad_one<G>(gp + i) : 0.0f;
                    if constexpr (S8) {
                        float d[4];
                        decode4(in ? static_cast<const uint8_t*>(t.m)[i] : 0u, s0, d);
                        m[e] = in ? d[0] : 0.0f;
                        decode4(in ? static_cast<const uint8_t*>(t.v)[i] : 0u, s1, d);
                        v[e] = in ? d[0] * d[0] : 0.0f;
                    } else {
                        m[e] = in ? static_cast<const float*>(t.m)[i] : 0.0f;
                        v[e] = in ? static_cast<const float*>(t.v)[i] : 0.0f;
                    }
                }
                const uint32_t before = am;
                float root[4];
                moments(g, m, v);
                update(std::false_type{}, p, m, v, root);
                uint32_t c0 = 0, c1 = 0;
                if constexpr (S8) {
                    // what lies past the end adds nothing to the maxima
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (ub + lane * 4 + e >= t.n) m[e] = root[e] = 0.0f;
                    uint32_t rnd[4] = {};
                    if constexpr (DITHER) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) rnd[e] = draw(key, ub + lane * 4 + e);
                    }
                    c0 = encode(m, std::false_type{}, false, s0, rnd);
                    c1 = encode(root, std::true_type{}, false, s1, rnd);
                    if (lane == 0) {
                        t.ms[ub >> 8] = s0;
                        t.vs[ub >> 8] = s1;
                    }
                }
                am = before;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int64_t i = ub + lane * 4 + e;
                    if (i >= t.n) continue;
                    t.p[i] = p[e];
                    if (h.absmax) am = fold_f32(am, __float_as_uint(p[e]));
                    if constexpr (COPY >= 0) t.copy[i] = (uint16_t)copy_bits<COPY>(p[e]);
                    if constexpr (S8) {
                        static_cast<uint8_t*>(t.m)[i] = (uint8_t)(c0 >> (8 * e));
                        static_cast<uint8_t*>(t.v)[i] = (uint8_t)(c1 >> (8 * e));
                    } else {
                        static_cast<float*>(t.m)[i] = m[e];
                        static_cast<float*>(t.v)[i] = v[e];
                    }
                }
            }
        }
    };
    // A wave's units lie side by side (206 us for two GPT-2 XL blocks, 8-bit
    // states; 220 with the waves taking units in turn), but in a tensor's last
    // block the waves take units in turn, so that several work on the few that
    // a small tensor has (two tensors of 771 values: 4.8 us against 9.5).
    const int64_t block0 = (int64_t)((int)blockIdx.x - L.first[lo]) * kSpan;
    if (block0 + kSpan <= t.n)
        units(std::integral_constant<int, kUnit>{}, block0 + (int64_t)wave * (kUnit * kUnits * kRounds));
    else
        units(std::integral_constant<int, kUnit * kWaves>{}, block0 + (int64_t)wave * kUnit);
    if (h.absmax) {
        // patterns of non-negative values order like unsigned integers: the
        // atomic maximum is exact in any order
        am = wave_umax(am);
        if (lane == 0 && am) atomicMax(h.absmax + L.idx[lo], am);
    }
}

enum Kept { kBits32, kBits8, kBits8Dithered };  // how states are kept

template <typename G, Kept K, bool NT>
void launch_copy(int copy_dtype, int blocks, const WList& L, const WHyper& h, hipStream_t st) {
    constexpr bool S8 = K != kBits32, D = K == kBits8Dithered;
    if (copy_dtype == DF_DTYPE_BFLOAT16)
        adamw_kernel<G, S8, DF_DTYPE_BFLOAT16, NT, D><<<blocks, kWThreads, 0, st>>>(L, h);
    else if (copy_dtype == DF_DTYPE_HALF)
        adamw_kernel<G, S8, DF_DTYPE_HALF, NT, D><<<blocks, kWThreads, 0, st>>>(L, h);
    else
        adamw_kernel<G, S8, -1, NT, D><<<blocks, kWThreads, 0, st>>>(L, h);
}

template <typename G, Kept K>
void launch_cold(bool cold, int copy_dtype, int blocks, const WList& L, const WHyper& h, hipStream_t st) {
    if (cold) launch_copy<G, K, true>(copy_dtype, blocks, L, h, st);
    else launch_copy<G, K, false>(copy_dtype, blocks, L, h, st);
}

template <typename G>
void launch_state(Kept kept, bool cold, int copy_dtype, int blocks, const WList& L, const WHyper& h, hipStream_t st) {
    if (kept == kBits32) launch_cold<G, kBits32>(cold, copy_dtype, blocks, L, h, st);
    else if (kept == kBits8) launch_cold<G, kBits8>(cold, copy_dtype, blocks, L, h, st);
    else launch_cold<G, kBits8Dithered>(cold, copy_dtype, blocks, L, h, st);
}

}  // namespace

}  // namespace dfk

using namespace dfk;

extern "C" int64_t df_adamw_scale_count(int64_t n) { return n <= 0 ? 0 : (n + kUnit - 1) / kUnit; }

static int update(const char* fn, bool dither, uint32_t seed, int count, const int64_t* sizes, float* const* params,
                  int grad_dtype, const void* const* grads, int state_dtype, void* const* m, void* const* v,
                  float* const* m_scale, float* const* v_scale, int copy_dtype, void* const* copies, float lr,
                  float beta1, float beta2, float eps, const float* weight_decay, int timestep, const float* lr_dev,
                  const int* timestep_dev, const float* clip_norm_dev, float max_norm, float* absmax_dev,
                  void* stream) {
    DF_CHECK(count >= 0, DF_ERR_INVALID, "%s: count = %d is negative", fn, count);
    DF_CHECK(grad_dtype == DF_DTYPE_FLOAT32 || grad_dtype == DF_DTYPE_BFLOAT16 || grad_dtype == DF_DTYPE_HALF,
             DF_ERR_UNSUPPORTED, "%s: gradient dtype %d not supported", fn, grad_dtype);
    DF_CHECK(state_dtype == DF_DTYPE_FLOAT32 || state_dtype == DF_DTYPE_FP8E4M3, DF_ERR_UNSUPPORTED,
             "%s: state dtype %d not supported", fn, state_dtype);
    DF_CHECK(!dither || state_dtype == DF_DTYPE_FP8E4M3, DF_ERR_UNSUPPORTED, "%s: only 8-bit states are dithered", fn);
    DF_CHECK(!copies || copy_dtype == DF_DTYPE_BFLOAT16 || copy_dtype == DF_DTYPE_HALF, DF_ERR_UNSUPPORTED,
             "%s: copy dtype %d not supported", fn, copy_dtype);
    const bool s8 = state_dtype == DF_DTYPE_FP8E4M3;
    DF_CHECK(count == 0 || (sizes && params && grads && m && v), DF_ERR_INVALID, "%s: an array is NULL", fn);
    DF_CHECK(count == 0 || !s8 || (m_scale && v_scale), DF_ERR_INVALID, "%s: 8-bit states without scales", fn);
    DF_CHECK(timestep_dev || timestep >= 1, DF_ERR_INVALID, "%s: timestep = %d (the first step is 1)", fn, timestep);
    DF_CHECK(aligned4(lr_dev) && aligned4(timestep_dev) && aligned4(clip_norm_dev) && aligned4(absmax_dev),
             DF_ERR_ALIGN, "%s: a device scalar is not 4-byte aligned", fn);
    const unsigned gmask = grad_dtype == DF_DTYPE_FLOAT32 ? 3u : 1u;
    int64_t total = 0, values = 0;
    for (int i = 0; i < count; ++i) {
        DF_CHECK(sizes[i] >= 0, DF_ERR_INVALID, "%s: sizes[%d] = %lld is negative", fn, i, (long long)sizes[i]);
        if (sizes[i] == 0) continue;
        total += (sizes[i] + kSpan - 1) / kSpan;
        values += sizes[i];
        DF_CHECK(total < (1ll << 31), DF_ERR_INVALID, "%s: too many elements", fn);
        DF_CHECK(params[i] && grads[i] && m[i] && v[i] && (!s8 || (m_scale[i] && v_scale[i])) && (!copies || copies[i]),
                 DF_ERR_INVALID, "%s: a pointer of tensor %d is NULL", fn, i);
        DF_CHECK(aligned4(params[i]) && ((uintptr_t)grads[i] & gmask) == 0 &&
                     (s8 ? aligned4(m_scale[i]) && aligned4(v_scale[i]) : aligned4(m[i]) && aligned4(v[i])) &&
                     (!copies || ((uintptr_t)copies[i] & 1u) == 0),
                 DF_ERR_ALIGN, "%s: a pointer of tensor %d is not aligned to its elements", fn, i);
    }
    WHyper h;
    h.lr = lr;
    h.b1 = beta1;
    h.b2 = beta2;
    h.omb1 = 1.0f - beta1;
    h.omb2 = 1.0f - beta2;
    h.eps = eps;
    h.max_norm = max_norm;
    h.bc1 = bias_corr(beta1, timestep);
    h.bc2 = bias_corr(beta2, timestep);
    h.t = timestep;
    h.seed = seed;
    h.lr_dev = lr_dev;
    h.step = timestep_dev;
    h.norm = clip_norm_dev;
    h.absmax = reinterpret_cast<uint32_t*>(absmax_dev);
    hipStream_t st = as_stream(stream);
    if (total == 0 && (!absmax_dev || count == 0)) return DF_OK;
    // bytes a value occupies, states and copy included
    const int64_t each = 4 + (s8 ? 2 : 8) + (grad_dtype == DF_DTYPE_FLOAT32 ? 4 : 2) + (copies ? 2 : 0);
    const bool cold = values * each > kColdBytes;
    if (absmax_dev) {
        const uint32_t zero = 0;
        if (int rc = df_fill(absmax_dev, count, 4, &zero, stream)) return rc;  // empty tensors stay at 0
    }
    for (int i = 0; i < count;) {
        WList L{};
        int blocks = 0, c = 0;
        for (; i < count && c < kWList; ++i) {
            if (sizes[i] == 0) continue;
            L.t[c] = WTensor{params[i], grads[i], m[i], v[i], s8 ? m_scale[i] : nullptr, s8 ? v_scale[i] : nullptr,
                             copies ? static_cast<uint16_t*>(copies[i]) : nullptr, sizes[i]};
            L.wd[c] = weight_decay ? weight_decay[i] : 0.0f;
            L.first[c] = blocks;
            L.idx[c] = i;
            blocks += (int)((sizes[i] + kSpan - 1) / kSpan);
            ++c;
        }
        if (c == 0) break;
        L.first[c] = blocks;
        L.count = c;
        const int cd = copies ? copy_dtype : -1;
        const Kept kept = !s8 ? kBits32 : dither ? kBits8Dithered : kBits8;
        if (grad_dtype == DF_DTYPE_FLOAT32) launch_state<float>(kept, cold, cd, blocks, L, h, st);
        else if (grad_dtype == DF_DTYPE_HALF) launch_state<f16_t>(kept, cold, cd, blocks, L, h, st);
        else launch_state<uint16_t>(kept, cold, cd, blocks, L, h, st);
    }
    return launch_status(fn);
}

extern "C" int df_adamw_update(int count, const int64_t* sizes, float* const* params, int grad_dtype,
                               const void* const* grads, int state_dtype, void* const* m, void* const* v,
                               float* const* m_scale, float* const* v_scale, int copy_dtype, void* const* copies,
                               float lr, float beta1, float beta2, float eps, const float* weight_decay, int timestep,
                               const float* lr_dev, const int* timestep_dev, const float* clip_norm_dev,
                               float max_norm, float* absmax_dev, void* stream) {
    clear_error();
    return update("df_adamw_update", false, 0, count, sizes, params, grad_dtype, grads, state_dtype, m, v,
                  m_scale, v_scale, copy_dtype, copies, lr, beta1, beta2, eps, weight_decay, timestep, lr_dev,
                  timestep_dev, clip_norm_dev, max_norm, absmax_dev, stream);
}

extern "C" int df_adamw_update_dithered(int count, const int64_t* sizes, float* const* params, int grad_dtype,
                                        const void* const* grads, int state_dtype, void* const* m, void* const* v,
                                        float* const* m_scale, float* const* v_scale, int copy_dtype,
                                        void* const* copies, float lr, float beta1, float beta2, float eps,
                                        const float* weight_decay, int timestep, const float* lr_dev,
                                        const int* timestep_dev, const float* clip_norm_dev, float max_norm,
                                        float* absmax_dev, uint32_t seed, void* stream) {
    clear_error();
    return update("df_adamw_update_dithered", true, seed, count, sizes, params, grad_dtype, grads, state_dtype, m, v,
                  m_scale, v_scale, copy_dtype, copies, lr, beta1, beta2, eps, weight_decay, timestep, lr_dev,
                  timestep_dev, clip_norm_dev, max_norm, absmax_dev, stream);
}
