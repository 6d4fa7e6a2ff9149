// moe.hip -- a mixture-of-experts layer for a few tokens (up to 64: generation),
// on e4m3 weights with a scale per 128 of the reduction (gfx950):
//   ids[t] = the top_k experts by the router's logits, ties to the lower index
//   w[t]   = softmax of their logits (over them, or over all experts)
//   y[t]   = sum over j of w[t][j] * W2[e] . act(W1[e] . x[t]),  e = ids[t][j]
// act: silu(gate) * up or gelu(gate) * up, W1 holding gate's rows, then up's; or
// gelu.
//
// Bound by reading the chosen experts' weights: at 48 tokens to two of 32 experts of
// 3 x 1600 x 1600 that is 240 MB.  A unit of an expert's tokens reads them, once from HBM
// and, where an expert has several, from L2 again.  So activations stay in 16 bits (no
// pass to quantize them), weights are widened in registers, 16 weight rows and 16
// tokens to a matrix instruction, and the launches are few: routing (for one token
// part of the next), W1 with the activation, W2 with the weighted sum.
//  - An expert's tokens are taken 16 at a time, a unit.  Routing lists the units
//    and their (token, choice) pairs, in order, in the workspace; one token's are
//    its choices as they are.
//  - W1: a block owns 16 inner values of a unit (both rows that make each); its
//    waves share the reduction.  The result, times the token's weight for the
//    expert, is kept as two bf16 values (hi + lo: 16 bits of significand, fp32's
//    range), so that it is not rounded to the output's type in between.
//  - W2: a block owns 16 columns of y for all tokens and all units; its waves take
//    equal shares of the units' steps and add what a unit's end gives to their own
//    sums in LDS, per token, which meet at the end in wave order.  No atomics on
//    values: results do not depend on timing.
// Measured: those 48 tokens 62 us (routing 5, W1 33 for 160 MB, W2 23 for 80 MB); one
// token to two of 32 experts (15 MB) 11.5, launches and the chain of a block's loads.
// Widening is exact (e4m3 to bf16 or f16), sums are fp32, scales are applied to each
// block's 128 products in fp32; W2's powers of two go into the widening to bf16, exact
// while codes times scales are multiples of 2^-133 below 2^128.
//
// The reference has no mixture of experts.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "block_scale.hpp"
#include "df_common.hpp"
#include "gemm_blocks.hpp"
#include "row_chunks.hpp"

namespace dfk {

namespace {

constexpr int kMoeTokens = 64, kMoeExperts = 256, kMoeTop = 16;
constexpr int kMoePairs = kMoeTokens * kMoeTop;
constexpr int kMoeUnits = kMoePairs / 4 + kMoeExperts;  // more than there can be, of either size
constexpr uint32_t kOOB = 0x80000000u;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// What routing leaves for the products, at the workspace's start: the pairs t * top + j
// by expert, then token, and lists of units, an expert's next few of them, for either
// product.
struct alignas(16) MoeUnit {  // (one load)
    int expert, first, count, none;  // (first: in `sorted`)
};
struct MoeUnits {
    MoeUnit unit[kMoeUnits];  // W1's are followed by units of no tokens, up to its grid's end
    int n;
};
struct MoePlan {
    MoeUnits up, down;
    int sorted[kMoePairs];
};

struct MoeArgs {
    const void* x; const void* logits;
    const uint8_t* W1; const void* s1; const uint8_t* W2; const void* s2;
    void* y; int* ids; float* weights;
    MoePlan* plan;
    uint16_t* hi; uint16_t* lo;  // [pairs][ldh] bf16
    float* part; int* arrived;   // W2 split: [splits][tokens][H16] sums, blocks done per column tile
    int tokens, H, N, experts, top, ldx, ldl, ldy, ldw1, ldw2, lds1, lds2, ldh, act, renormalize, x_dtype, l_dtype, splits, up_size, down_size, up_most;
};

// ------------------------------------------------------------------ routing --
__device__ __forceinline__ float load_as_float(const void* p, int dtype, int64_t i) {
    if (dtype == DF_DTYPE_FLOAT32) return static_cast<const float*>(p)[i];
    if (dtype == DF_DTYPE_HALF) return (float)__builtin_bit_cast(_Float16, static_cast<const uint16_t*>(p)[i]);
    return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}

// f over the 16 lanes of a DPP row, the same in each of them (a butterfly: quad_perm
// by 1 and 2, row_half_mirror, row_mirror)
template <typename T, typename F> __device__ __forceinline__ T row_fold(T v, const F& f) {
#define DF_FOLD(CTRL) \
    v = f(v, __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true)))
    DF_FOLD(0xB1);
    DF_FOLD(0x4E);
    DF_FOLD(0x141);
    DF_FOLD(0x140);
#undef DF_FOLD
    return v;
}

// 16 lanes (g: the lane among them): token t's choices, the j-th in lane j: its
// expert and weight, -1 and 0 where no more can be chosen (an expert whose logit is
// -infinity or NaN is none; tokens from a.tokens on have none).  PER: logits a lane.
template <int PER> __device__ __forceinline__ void route_token(const MoeArgs& a, int t, int g, int& id, float& weight) {
    float v[PER];
    uint32_t key[PER];  // order of the values; 0: cannot be chosen
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = g + 16 * i;
        v[i] = e < a.experts && t < a.tokens ? load_as_float(a.logits, a.l_dtype, (int64_t)t * a.ldl + e) : -__builtin_inff();
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const float z = v[i] == 0.0f ? 0.0f : v[i];  // -0 is 0
        const uint32_t u = __float_as_uint(z);
        key[i] = z > -__builtin_inff() ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;  // (NaN fails the test)
    }
    uint32_t mine = 0, first = 0;
    id = -1;
    for (int j = 0; j < a.top; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) best = max(best, key[i]);
        best = row_fold(best, [](uint32_t x, uint32_t y) { return max(x, y); });
        uint32_t who = 0xFFFFFFFFu;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) who = key[i] == best ? (uint32_t)(g + 16 * i) : who;
        who = row_fold(who, [](uint32_t x, uint32_t y) { return min(x, y); });
        if (j == 0) first = best;
        if (g == j && best) {
            id = (int)who;
            mine = best;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if ((uint32_t)(g + 16 * i) == who) key[i] = 0;
    }
    auto value = [](uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k); };
    const float most = value(first);
    // exp(l - most), right for infinities too
    auto part = [&](float x) { return x == most ? 1.0f : expf(x - most); };
    const float own = id >= 0 ? part(value(mine)) : 0.0f;
    float sum = own;
    if (!a.renormalize) {
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (v[i] > -__builtin_inff()) sum += part(v[i]);
    }
    sum = row_fold(sum, [](float x, float y) { return x + y; });
    weight = id >= 0 ? own / sum : 0.0f;
}
__device__ __forceinline__ void route_any(const MoeArgs& a, int t, int g, int& id, float& weight) {
    if (a.experts <= 64) route_token<4>(a, t, g, id, weight);
    else route_token<kMoeExperts / 16>(a, t, g, id, weight);
}

// One block: every token's choices, then the plan.
__global__ __launch_bounds__(1024) void moe_route_kernel(const MoeArgs a) {
    __shared__ int ids[kMoePairs];
    __shared__ uint32_t taken[kMoeExperts][kMoeTokens / 32];  // which tokens take an expert
    __shared__ int start[kMoeExperts], at_wave[3][4], up_units;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < kMoeExperts * (kMoeTokens / 32); i += 1024) (&taken[0][0])[i] = 0;
    __syncthreads();
    {
        const int t = threadIdx.x >> 4, g = threadIdx.x & 15;  // 64 tokens at once
        int e;
        float weight;
        route_any(a, t, g, e, weight);
        if (t < a.tokens && g < a.top) {
            const int p = t * a.top + g;
            ids[p] = e;
            a.ids[p] = e;
            a.weights[p] = weight;
            if (e >= 0) atomicOr(&taken[e][t >> 5], 1u << (t & 31));
        }
    }
    __syncthreads();
    // experts' pairs and units, added up in order of the experts
    const int e = threadIdx.x;
    int n = 0, sum[3] = {0, 0, 0};  // pairs, units of W1, of W2
    if (e < kMoeExperts) {
#pragma unroll
        for (int i = 0; i < kMoeTokens / 32; ++i) n += __builtin_popcount(taken[e][i]);
        sum[0] = n;
        sum[1] = (n + a.up_size - 1) / a.up_size;
        sum[2] = (n + a.down_size - 1) / a.down_size;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                const int o = __shfl_up(sum[i], off, 64);
                if (lane >= off) sum[i] += o;
            }
        }
        if (lane == 63)
            for (int i = 0; i < 3; ++i) at_wave[i][w] = sum[i];
    }
    __syncthreads();
    if (e < kMoeExperts) {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            for (int v = 0; v < w; ++v) sum[i] += at_wave[i][v];
        start[e] = sum[0] - n;
        auto list = [&](MoeUnits& u, int size, int upto) {
            const int k = upto - (n + size - 1) / size;
            for (int i = 0; i * size < n; ++i) {
                u.unit[k + i] = {e, sum[0] - n + size * i, min(n - size * i, size), 0};
            }
            if (e == kMoeExperts - 1) u.n = upto;
        };
        if (e == kMoeExperts - 1) up_units = sum[1];
        list(a.plan->up, a.up_size, sum[1]);
        list(a.plan->down, a.down_size, sum[2]);
    }
    __syncthreads();
    for (int i = up_units + threadIdx.x; i < a.up_most; i += 1024) a.plan->up.unit[i] = {0, 0, 0, 0};
    for (int p = threadIdx.x; p < a.tokens * a.top; p += 1024) {
        const int x = ids[p], t = p / a.top;
        if (x < 0) continue;
        int rank = 0;
#pragma unroll
        for (int i = 0; i < kMoeTokens / 32; ++i) {
            const uint32_t below = t >= 32 * (i + 1) ? ~0u : t > 32 * i ? (1u << (t - 32 * i)) - 1u : 0u;
            rank += __builtin_popcount(taken[x][i] & below);
        }
        a.plan->sorted[start[x] + rank] = p;
    }
}

// ----------------------------------------------------------------- products --
// eight codes widened to x's type, exact
template <typename V> __device__ __forceinline__ V widen_codes(uint32_t lo, uint32_t hi) {
    if constexpr (std::is_same<V, bf8>::value) {
        return widen8_scaled<E4M3>(lo, hi, 1.0f);
    } else {
        h2 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = i < 2 ? lo : hi;
            p[i] = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true)
                         : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        }
        return h8{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
    }
}
__device__ __forceinline__ v4f mfma16(bf8 a, bf8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ v4f mfma16(h8 a, h8 b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

template <bool E8> __device__ __forceinline__ float scale_value(uint32_t raw) {
    return E8 ? e8m0_value(raw) : __uint_as_float(raw);
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)bytes, 0x00020000);
}
// at a lane's offset and one for all lanes; the descriptor's range counts both, and past it
// 0 is read (kOOB: whatever the other)
template <bool E8> __device__ __forceinline__ uint32_t load_scale(__amdgpu_buffer_rsrc_t r, uint32_t at, int all) {
    if constexpr (E8) return __builtin_amdgcn_raw_buffer_load_b8(r, at, all, 0);
    else return __builtin_amdgcn_raw_buffer_load_b32(r, at, all, 0);
}
__device__ __forceinline__ u32x4 load16(__amdgpu_buffer_rsrc_t r, uint32_t at, int all) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, at, all, 0));
}

__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + expf(-v)); }
__device__ __forceinline__ float gelu(float v) {  // 0.5 v (1 + tanh(sqrt(2/pi) (v + 0.044715 v^3)))
    return v * sigmoid(1.5957691216057308f * (v + 0.044715f * v * v * v));
}

// W1 and the activation.  blockIdx.x: 16 inner values (32 without a gate), blockIdx.y:
// the unit.  Fragments go from memory to registers as the instruction wants them:
// lane l has weight row l%16 (or token l%16) and the 16-byte chunks l/16 and l/16 + 4
// of a step of 128 codes; U steps are loaded ahead.  Products are tokens x weight
// rows: lane l holds row l%16 and tokens 4*(l/16) .. +4, so a scale is one per lane.
template <typename V, bool E8, bool GATED, bool ALIGNED, int U>
__global__ __launch_bounds__(256) void moe_up_kernel(const MoeArgs a) {
    constexpr int W = 4, COLS = GATED ? 16 : 32, SZ = E8 ? 1 : 4;
    __shared__ float red[W][2][16][20];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * COLS, unit = blockIdx.y;
    // the next launch counts its blocks from 0
    if (blockIdx.y == 0)
        for (int i = blockIdx.x * 256 + threadIdx.x; a.splits > 1 && i < (a.H + 15) / 16; i += gridDim.x * 256) a.arrived[i] = 0;
    const int fr = lane & 15, fq = lane >> 4;
    int e, count, first = 0, pair = -1;
    float weight1 = 0.0f;
    if (a.tokens == 1) {  // the unit is a choice
        int id;
        float weight;
        route_any(a, 0, fr, id, weight);
        if (blockIdx.x == 0 && unit == 0 && (int)threadIdx.x < a.top) {
            a.ids[threadIdx.x] = id;
            a.weights[threadIdx.x] = weight;
        }
        e = __builtin_amdgcn_readlane(id, unit);
        weight1 = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), unit));
        if (e < 0) return;
        count = 1;
        if (fr == 0) pair = unit;
    } else {
        const MoeUnit u = a.plan->up.unit[unit];
        e = u.expert;
        count = u.count;
        first = u.first;
        if (count == 0) return;
        if (fr < count) pair = a.plan->sorted[first + fr];
    }
    if (n0 >= a.N) {  // only the zeros up to a step's end
        for (int i = threadIdx.x; i < count * COLS; i += 256) {
            const int p = a.tokens == 1 ? unit : a.plan->sorted[first + i / COLS];
            a.hi[(int64_t)p * a.ldh + n0 + i % COLS] = a.lo[(int64_t)p * a.ldh + n0 + i % COLS] = 0;
        }
        return;
    }
    const int rows1 = GATED ? 2 * a.N : a.N, blocks = (a.H + 127) >> 7;
    const int K16 = (a.H + 15) & ~15;
    // (up to the last row's codes: its leading dimension may reach past the tensor)
    const __amdgpu_buffer_rsrc_t rW = buffer(a.W1 + (int64_t)e * rows1 * a.ldw1, (int64_t)(rows1 - 1) * a.ldw1 + K16);
    const __amdgpu_buffer_rsrc_t rS =
        buffer(static_cast<const uint8_t*>(a.s1) + (int64_t)e * blocks * a.lds1 * SZ, (int64_t)blocks * a.lds1 * SZ);
    const __amdgpu_buffer_rsrc_t rX = buffer(a.x, ((int64_t)(a.tokens - 1) * a.ldx + a.H) * 2);
    // Offsets of a lane; a step adds the same to all of them.  Chunks behind the rows'
    // end are read from what follows and cleared before use, in the last step.
    uint32_t wo[2], so[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int n = n0 + (GATED ? 0 : 16 * g) + fr;
        const uint32_t row = (uint32_t)(n + (GATED ? g * a.N : 0));
        wo[g] = n < a.N ? row * (uint32_t)a.ldw1 + 16u * fq : kOOB;
        so[g] = n < a.N ? row * SZ : kOOB;
    }
    const uint32_t xo = pair >= 0 ? (uint32_t)(pair / a.top) * (uint32_t)a.ldx * 2u + 32u * fq : kOOB;
    const uint16_t* const xr = static_cast<const uint16_t*>(a.x) + (int64_t)(max(pair, 0) / a.top) * a.ldx;

    struct Step {
        u32x4 w[2][2], x[2][2];
        uint32_t s[2];
    };
    auto load_w = [&](Step& s, int step) {
        const bool live = step < blocks;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int g = 0; g < 2; ++g) s.w[g][h] = load16(rW, (live ? wo[g] : kOOB) + 64u * h, step * 128);
#pragma unroll
        for (int g = 0; g < 2; ++g) s.s[g] = load_scale<E8>(rS, live ? so[g] : kOOB, step * a.lds1 * SZ);
    };
    auto load_x = [&](Step& s, int step) {
        const bool live = step < blocks;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if constexpr (ALIGNED) s.x[h][c] = load16(rX, (live ? xo : kOOB) + 128u * h + 16u * c, step * 256);
                else s.x[h][c] = pair >= 0 && live ? load_chunk<uint16_t>(xr, step * 16 + 2 * fq + 8 * h + c, a.H) : u32x4{0, 0, 0, 0};
            }
    };
    v4f acc[2] = {};
    auto multiply = [&](Step& s, int step) {
        if (step * 128 + 128 > a.H) {  // the rows' end
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = step * 128 + 16 * fq + 64 * h;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    if constexpr (ALIGNED) {
                        if (k + 8 * c >= a.H) s.x[h][c] = u32x4{0, 0, 0, 0};
                    } else {  // its last chunk was loaded up to there
                        s.x[h][c] = place_chunk<uint16_t>(s.x[h][c], k / 8 + c, a.H);
                    }
                }
                if (k >= K16) s.w[0][h] = s.w[1][h] = u32x4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            v4f p = {};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    p = mfma16(__builtin_bit_cast(V, s.x[h][c]), widen_codes<V>(s.w[g][h][2 * c], s.w[g][h][2 * c + 1]), p);
            const float sc = scale_value<E8>(s.s[g]);
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[g][r] = __builtin_fmaf(p[r], sc, acc[g][r]);
        }
    };
    Step buf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load_w(buf[u], w + u * W);  // while `pair` is on its way
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) load_x(buf[u], w + u * W);
    for (int s = w; s < blocks; s += W * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u * W < blocks) multiply(buf[u], s + u * W);
            load_w(buf[u], s + (u + U) * W);
            load_x(buf[u], s + (u + U) * W);
        }
    }
#pragma unroll
    for (int g = 0; g < 2; ++g)
        *reinterpret_cast<v4f*>(&red[w][g][fr][4 * fq]) = acc[g];
    __syncthreads();
    const int c = threadIdx.x & 15, i = threadIdx.x >> 4;  // column, token of the unit
    if (i >= count) return;
    float v[2] = {0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int x = 0; x < W; ++x) v[g] += red[x][g][c][i];
    const int p = a.tokens == 1 ? unit : a.plan->sorted[first + i];
    const float weight = a.tokens == 1 ? weight1 : a.weights[p];
    auto put = [&](int n, float h) {
        h = n < a.N ? h * weight : 0.0f;  // zeros up to a step's end
        const uint32_t hi = f32_to_bf16_rne(h);
        // (an infinity has no rest)
        const float rest = h - bf16_to_f32(hi);
        a.hi[(int64_t)p * a.ldh + n] = (uint16_t)hi;
        a.lo[(int64_t)p * a.ldh + n] = (uint16_t)(__builtin_fabsf(h) < __builtin_inff() && __builtin_fabsf(rest) < __builtin_inff() ? f32_to_bf16_rne(rest) : 0u);
    };
    if constexpr (GATED) {
        put(n0 + c, (a.act == DF_ACT_SWIGLU ? v[0] * sigmoid(v[0]) : gelu(v[0])) * v[1]);
    } else {
        put(n0 + c, gelu(v[0]));
        put(n0 + 16 + c, gelu(v[1]));
    }
}

// How W2's product is laid out.  A memory instruction wants neighbouring lanes on
// neighbouring bytes, a matrix instruction a row each in them, and both get it from the
// parts of a row: a step is 256 codes, 16 chunks of 16, and lane l = 16 fq + 4 r + p
// loads chunk 4 fq + p of weight row r of four (the four rows' 256 bytes whole, in one
// load), and that part of token r of four.  As operands of the matrix instruction,
// rows are (token, p) and columns (weight row, p'); a result counts where p = p', and
// the four that do add up to a token and row's product.  The other twelve cost
// nothing: with 16 rows and tokens to an instruction, as in W1's, each group of four
// lanes reads from four rows, and where columns' blocks are few, as here, the address
// lookups of their CUs, 64 a load, bound the kernel (48 tokens to two of 32 experts:
// 26.4 us, 23.5 so; W1's blocks are many: whole lines through LDS took 31 us there in
// place of 33, and for two tokens 10.2 in place of 8.9).
// TG token groups of four share the weights' registers: units of 4 TG tokens.
constexpr int kStep = 256;

struct Lane {
    int fr, fq, r, p, chunk;  // chunk: this lane's first code of a step
};
__device__ __forceinline__ Lane lane_parts() {
    const int l = threadIdx.x & 63, fr = l & 15;
    return {fr, l >> 4, fr >> 2, fr & 3, 16 * (4 * (l >> 4) + (fr & 3))};
}

// A wave's load of 16 weight rows' scales of a step's two blocks, row l%16 and block
// (l/16)%2 in lane l, and what lane l needs of it: row 4 g + r of block b
__device__ __forceinline__ uint32_t scale_of(uint32_t raw, const Lane& l, int g, int b) {
    return (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (16 * b + 4 * g + l.r), (int)raw);
}

// 16 weight rows (w: four rows a load) times TG * 4 tokens over one step, into acc[tg][g].
// FOLD: scales are powers of two and V is bf16, they go into the widening; else each
// block of 128 is multiplied by itself, the other's half of x cleared.  x: PLANES values
// that add up to a token's.
template <bool E8, bool FOLD, typename V, int TG, int PLANES>
__device__ __forceinline__ void step_products(const u32x4 (&w)[4], uint32_t scales, const u32x4 (&x)[TG][PLANES][2],
                                              v4f (&acc)[TG][4], const Lane& l) {
    // the scales first, then four rows at a time: left to itself the compiler widens all
    // rows at once, at twice the registers
    uint32_t raw[4][FOLD ? 1 : 2];
#pragma unroll
    for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int b = 0; b < (FOLD ? 1 : 2); ++b) raw[g][b] = scale_of(scales, l, g, FOLD ? l.fq >> 1 : b);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (FOLD) {
            const float sc = e8m0_value(raw[g][0]);
            const V b0 = widen8_scaled<E4M3>(w[g][0], w[g][1], sc), b1 = widen8_scaled<E4M3>(w[g][2], w[g][3], sc);
#pragma unroll
            for (int t = 0; t < TG; ++t)
#pragma unroll
                for (int n = PLANES - 1; n >= 0; --n) {
                    acc[t][g] = mfma16(__builtin_bit_cast(V, x[t][n][0]), b0, acc[t][g]);
                    acc[t][g] = mfma16(__builtin_bit_cast(V, x[t][n][1]), b1, acc[t][g]);
                }
        } else {
            const V b0 = widen_codes<V>(w[g][0], w[g][1]), b1 = widen_codes<V>(w[g][2], w[g][3]);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float sc = scale_value<E8>(raw[g][b]);
                const uint32_t keep = (l.fq >> 1) == b ? ~0u : 0u;
#pragma unroll
                for (int t = 0; t < TG; ++t) {
                    v4f v = {};
#pragma unroll
                    for (int n = PLANES - 1; n >= 0; --n) {
                        v = mfma16(__builtin_bit_cast(V, x[t][n][0] & keep), b0, v);
                        v = mfma16(__builtin_bit_cast(V, x[t][n][1] & keep), b1, v);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t][g][i] = __builtin_fmaf(v[i], sc, acc[t][g][i]);
                }
            }
        }
    }
}

// token fq of a group times weight row 4 g + r, in every lane p: the four parts' sum
__device__ __forceinline__ float parts_sum(const v4f& a, const Lane& l) {
    const float even = l.p & 2 ? a[2] : a[0], odd = l.p & 2 ? a[3] : a[1];
    float v = l.p & 1 ? odd : even;
#define DF_QUAD(CTRL) \
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true))
    DF_QUAD(0xB1);  // quad_perm by 1, by 2
    DF_QUAD(0x4E);
#undef DF_QUAD
    return v;
}

// Blocks that meet: each puts its values (meeting_put), then arrives, and the last to
// arrive gets all (meeting_get).  Order rests on the hardware, not on the language's
// memory model: puts and gets are agent-scope atomics, which pass the caches of the XCDs,
// both ways, so a put that is done (vmcnt 0 in every wave, then the block's barrier) is
// seen by whoever sees the count that follows it.  What the model asks for, a release and
// an acquire, would write back and drop all of an XCD's L2, the weights with it: 48 tokens
// 124 us so, 42 this way.
__device__ __forceinline__ void meeting_put(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float meeting_get(const float* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// (the whole block; count is 0 before the first arrives)
__device__ __forceinline__ bool last_to_arrive(int* count, int blocks) {
    __shared__ int last;
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0);
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __syncthreads();
    if (threadIdx.x == 0) last = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == blocks - 1;
    __syncthreads();
    return last;
}

// W2 and the weighted sum.  blockIdx.x: 16 columns of y; blockIdx.y: a share of the
// units' steps, where there are more than 16 columns' blocks could keep under way.
// Shares leave fp32 sums in the workspace, and the last of a column's blocks to end
// adds them in order.
template <bool E8, int TG> __global__ __launch_bounds__(512) void moe_down_kernel(const MoeArgs a) {
    constexpr int W = 8, U = 2, SZ = E8 ? 1 : 4;
    __shared__ MoeUnit unit[kMoeUnits];
    __shared__ int sorted[kMoePairs];
    __shared__ float sums[W][kMoeTokens][17];
    const Lane l = lane_parts();
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h0 = blockIdx.x * 16, pairs = a.tokens * a.top;
    int units;
    if (a.tokens == 1) {
        units = a.top;
        if ((int)threadIdx.x < units) {
            const int id = a.ids[threadIdx.x];
            unit[threadIdx.x] = {id, (int)threadIdx.x, id >= 0, 0};
            sorted[threadIdx.x] = threadIdx.x;
        }
    } else {
        const MoeUnits& u = a.plan->down;
        static_assert(kMoeUnits == 512, "a thread takes one");
        unit[threadIdx.x] = u.unit[threadIdx.x];  // (of any value from u.n on: not waited for)
        units = u.n;
        for (int i = threadIdx.x; i < pairs; i += 512) sorted[i] = a.plan->sorted[i];
    }
    for (int i = threadIdx.x & 63; i < a.tokens * 17; i += 64) sums[w][i / 17][i % 17] = 0.0f;
    __syncthreads();
    const int blocks = (a.N + 127) >> 7, steps = a.ldh / kStep, K16 = (a.N + 15) & ~15;
    const int64_t bytes2 = (int64_t)a.H * a.ldw2, sbytes2 = (int64_t)blocks * a.lds2 * SZ;
    const int64_t range2 = (int64_t)(a.H - 1) * a.ldw2 + K16;  // (up to the last row's codes)
    const __amdgpu_buffer_rsrc_t rHi = buffer(a.hi, (int64_t)pairs * a.ldh * 2), rLo = buffer(a.lo, (int64_t)pairs * a.ldh * 2);
    uint32_t wo[4];
#pragma unroll
    for (int g = 0; g < 4; ++g)
        wo[g] = h0 + 4 * g + l.r < a.H ? (uint32_t)(h0 + 4 * g + l.r) * (uint32_t)a.ldw2 + (uint32_t)l.chunk : kOOB;
    const uint32_t so = h0 + l.fr < a.H ? (uint32_t)(h0 + l.fr + (l.fq & 1) * a.lds2) * SZ : kOOB;
    const int total = units * steps, shares = W * a.splits, share = blockIdx.y * W + w;
    const int lo_f = (int)((int64_t)total * share / shares), hi_f = (int)((int64_t)total * (share + 1) / shares);

    struct Step {
        u32x4 w[4], x[TG][2][2];  // x: the inner values' hi and lo
        uint32_t s;
    };
    // where loading is: step l_f, the l_s-th of unit l_u; its expert's weights, and the
    // rows of inner values of this lane's tokens
    int l_f = lo_f, l_u = lo_f / steps, l_s = lo_f - l_u * steps;
    __amdgpu_buffer_rsrc_t rW, rS;
    uint32_t ho[TG];
    auto enter = [&]() {
        const int u = min(l_u, units - 1);
        const int e = max(__builtin_amdgcn_readfirstlane(unit[u].expert), 0), n = __builtin_amdgcn_readfirstlane(unit[u].count);
        rW = buffer(a.W2 + (int64_t)e * bytes2, n ? range2 : 0);
        rS = buffer(static_cast<const uint8_t*>(a.s2) + (int64_t)e * sbytes2, n ? sbytes2 : 0);
#pragma unroll
        for (int t = 0; t < TG; ++t) {
            const int pair = 4 * t + l.r < n ? sorted[unit[u].first + 4 * t + l.r] : -1;
            ho[t] = pair >= 0 ? ((uint32_t)pair * (uint32_t)a.ldh + (uint32_t)l.chunk) * 2u : kOOB;
        }
    };
    auto load = [&](Step& s) {
        const bool live = l_f < hi_f;
#pragma unroll
        for (int t = 0; t < TG; ++t)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                s.x[t][0][c] = load16(rHi, (live ? ho[t] : kOOB) + 16u * c, l_s * kStep * 2);
                s.x[t][1][c] = load16(rLo, (live ? ho[t] : kOOB) + 16u * c, l_s * kStep * 2);
            }
#pragma unroll
        for (int g = 0; g < 4; ++g) s.w[g] = load16(rW, live ? wo[g] : kOOB, l_s * kStep);
        s.s = load_scale<E8>(rS, live && 2 * l_s + (l.fq & 1) < blocks ? so : kOOB, 2 * l_s * a.lds2 * SZ);
        ++l_f;
        if (++l_s == steps) {
            l_s = 0;
            ++l_u;
            enter();
        }
    };
    v4f acc[TG][4] = {};
    int m_u = l_u, m_s = l_s;  // the step that is multiplied
    auto multiply = [&](Step& s, bool last) {
        if (m_s == steps - 1 && m_s * kStep + l.chunk >= K16) {  // the rows' end (the inner values are 0 there)
#pragma unroll
            for (int g = 0; g < 4; ++g) s.w[g] = u32x4{0, 0, 0, 0};
        }
        step_products<E8, E8, bf8, TG, 2>(s.w, s.s, s.x, acc, l);
        if (++m_s == steps || last) {  // the unit's end, or this wave's
#pragma unroll
            for (int t = 0; t < TG; ++t) {
                float v[4];
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    v[g] = parts_sum(acc[t][g], l);
                    acc[t][g] = v4f{};
                }
                // lane p adds row 4 p + r
                const float even = l.p & 2 ? v[2] : v[0], odd = l.p & 2 ? v[3] : v[1];
                const int i = 4 * t + l.fq;
                if (i < unit[m_u].count) sums[w][sorted[unit[m_u].first + i] / a.top][4 * l.p + l.r] += l.p & 1 ? odd : even;
            }
            m_s = 0;
            ++m_u;
        }
    };
    if (lo_f < hi_f) {
        Step buf[U];
        enter();
#pragma unroll
        for (int u = 0; u < U; ++u) load(buf[u]);
        for (int f = lo_f; f < hi_f; f += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (f + u < hi_f) multiply(buf[u], f + u + 1 == hi_f);
                load(buf[u]);
            }
        }
    }
    __syncthreads();
    auto store = [&](int t, int c, float v) {
        const int64_t at = (int64_t)t * a.ldy + h0 + c;
        if (h0 + c >= a.H) return;
        if (a.x_dtype == DF_DTYPE_HALF) static_cast<f16_t*>(a.y)[at] = OutCvt<f16_t>::cvt(v);
        else static_cast<uint16_t*>(a.y)[at] = OutCvt<uint16_t>::cvt(v);
    };
    const int H16 = (a.H + 15) & ~15;
    for (int i = threadIdx.x; i < a.tokens * 16; i += 512) {
        const int t = i >> 4, c = i & 15;
        float v = 0.0f;
#pragma unroll
        for (int x = 0; x < W; ++x) v += sums[x][t][c];
        if (a.splits == 1) store(t, c, v);
        else meeting_put(a.part + ((int64_t)blockIdx.y * a.tokens + t) * H16 + h0 + c, v);
    }
    if (a.splits == 1 || !last_to_arrive(a.arrived + blockIdx.x, a.splits)) return;
    for (int i = threadIdx.x; i < a.tokens * 16; i += 512) {
        const int t = i >> 4, c = i & 15;
        float v = 0.0f;
        for (int x = 0; x < a.splits; ++x) v += meeting_get(a.part + ((int64_t)x * a.tokens + t) * H16 + h0 + c);
        store(t, c, v);
    }
}

template <typename V, bool E8> void launch_up(const MoeArgs& a, dim3 grid, hipStream_t st) {
    // 16-byte loads of x through a buffer descriptor, where its rows allow them
    const bool aligned = a.H % 8 == 0 && a.ldx % 8 == 0 && aligned16(a.x) &&
                         ((int64_t)(a.tokens - 1) * a.ldx + a.H) * 2 < (1ll << 31), gated = a.act != DF_ACT_GELU;
    if (gated && aligned && a.tokens == 1) moe_up_kernel<V, E8, true, true, 4><<<grid, 256, 0, st>>>(a);
    else if (gated && aligned) moe_up_kernel<V, E8, true, true, 2><<<grid, 256, 0, st>>>(a);
    else if (gated) moe_up_kernel<V, E8, true, false, 2><<<grid, 256, 0, st>>>(a);
    else if (aligned) moe_up_kernel<V, E8, false, true, 2><<<grid, 256, 0, st>>>(a);
    else moe_up_kernel<V, E8, false, false, 2><<<grid, 256, 0, st>>>(a);
}

// W2's units are of four tokens, or of 8 where experts get more than four on average:
// two groups then share the weights' registers.
bool many_tokens(int tokens, int experts, int top) { return (int64_t)tokens * top > 4 * (int64_t)experts; }

// at most this many units of `size` tokens, dealt in any way
int64_t most_units(int tokens, int experts, int top, int size) {
    const int64_t pairs = (int64_t)tokens * top;
    return tokens == 1 ? top : std::min<int64_t>(experts, pairs) + pairs / size;
}

// Blocks that share a column tile of W2: as many as make two of them for each of 256
// CUs, each wave with two steps at least; one, unless sharing spares a wave six steps, or
// more where more tokens' sums meet: a step takes 0.7 us, the blocks' meeting 4 for a few
// tokens and 7 for 64.  us with one and shared, powers of two, 1600 wide: 4 tokens to two
// of 32 experts (W2 alone) 9.0 and 10.8 with three, 8 tokens 14.6 and 12.4 with five; the
// layer, 64 tokens to eight of 8 experts 113 and 90 with five, to two of 8 45.6 and 45.5
// (fp32 scales 57.4 and 51.6), to four of 16 with N = 400 34.2 and 38.1 with four; 32
// tokens to two of 4, 768 and N = 3000, 37.2 and 34.6 with six.
int down_splits(int tokens, int H, int N, int experts, int top) {
    const int64_t tiles = (H + 15) / 16, pairs = (int64_t)tokens * top, size = many_tokens(tokens, experts, top) ? 8 : 4;
    // (dealt evenly: an expert's tokens may be several units)
    const int64_t units = tokens == 1 ? top : std::max(std::min<int64_t>(experts, pairs), (pairs + size - 1) / size);
    const int64_t steps = units * ((N + kStep - 1) / kStep), want = 512 / tiles, most = steps / (8 * 2);
    const int64_t n = std::max<int64_t>(1, std::min(want, most));
    return steps - steps / n < 8 * std::max<int64_t>(6, tokens / 6) ? 1 : (int)n;
}

template <bool E8> void launch(MoeArgs a, hipStream_t st) {
    const bool many = many_tokens(a.tokens, a.experts, a.top);
    a.up_size = 16;
    a.down_size = many ? 8 : 4;
    a.up_most = (int)most_units(a.tokens, a.experts, a.top, a.up_size);
    if (a.tokens > 1) moe_route_kernel<<<1, 1024, 0, st>>>(a);
    // (columns up to a step's end, for its zeros; a multiple of 8 blocks: an expert's
    // units share an XCD's L2)
    const dim3 up(a.ldh / (a.act != DF_ACT_GELU ? 16 : 32), (unsigned)a.up_most);
    const dim3 down((a.H + 15) / 16, a.splits);
    if (a.x_dtype == DF_DTYPE_HALF) launch_up<h8, E8>(a, up, st);
    else launch_up<bf8, E8>(a, up, st);
    if (many) moe_down_kernel<E8, 2><<<down, 512, 0, st>>>(a);
    else moe_down_kernel<E8, 1><<<down, 512, 0, st>>>(a);
}

constexpr size_t kPlanBytes = (sizeof(MoePlan) + 255) / 256 * 256;

}  // namespace

}  // namespace dfk

using namespace dfk;

// the plan, the inner values, the shares' sums and counts
extern "C" size_t df_moe_layer_workspace_bytes(int tokens, int H, int N, int experts, int top_k) {
    if (tokens <= 0 || tokens > kMoeTokens || top_k <= 0 || top_k > kMoeTop || H <= 0 || H > 0x7FFFFFF0 || N <= 0 ||
        N > 0x7FFFFF00 || experts < top_k || experts > kMoeExperts)
        return 0;
    const size_t H16 = ((size_t)H + 15) & ~(size_t)15, splits = down_splits(tokens, H, N, experts, top_k);
    return kPlanBytes + (size_t)tokens * top_k * (((size_t)N + kStep - 1) & ~(size_t)(kStep - 1)) * 4 +
           (splits > 1 ? splits * tokens * H16 * 4 + H16 / 16 * 4 : 0);
}

extern "C" int df_moe_layer(int dtype, const void* x, int ldx, int tokens, int H, int N, int experts, int top_k,
                            int logits_dtype, const void* logits, int ld_logits, int renormalize, int act,
                            const uint8_t* W1, int ldw1, const uint8_t* W2, int ldw2, int scale_kind, const void* s1,
                            int lds1, const void* s2, int lds2, void* y, int ldy, int* ids, float* weights, void* ws,
                            size_t ws_bytes, void* stream) {
    clear_error();
    const char* fn = "df_moe_layer";
    DF_CHECK(dtype == DF_DTYPE_BFLOAT16 || dtype == DF_DTYPE_HALF, DF_ERR_UNSUPPORTED, "%s: dtype %d not supported", fn, dtype);
    DF_CHECK(logits_dtype == DF_DTYPE_FLOAT32 || logits_dtype == DF_DTYPE_BFLOAT16 || logits_dtype == DF_DTYPE_HALF,
             DF_ERR_UNSUPPORTED, "%s: logits dtype %d not supported", fn, logits_dtype);
    DF_CHECK(tokens >= 0 && H >= 0 && N > 0 && experts > 0, DF_ERR_INVALID,
             "%s: bad sizes (tokens=%d, H=%d, N=%d, experts=%d)", fn, tokens, H, N, experts);
    DF_CHECK(tokens <= kMoeTokens && experts <= kMoeExperts, DF_ERR_UNSUPPORTED,
             "%s: %d tokens, %d experts (at most %d and %d)", fn, tokens, experts, kMoeTokens, kMoeExperts);
    DF_CHECK(top_k >= 1 && top_k <= experts && top_k <= kMoeTop, DF_ERR_INVALID, "%s: top_k=%d of %d experts (at most %d)", fn,
             top_k, experts, kMoeTop);
    DF_CHECK(act == DF_ACT_SWIGLU || act == DF_ACT_GEGLU || act == DF_ACT_GELU, DF_ERR_INVALID, "%s: bad activation %d", fn, act);
    DF_CHECK(scale_kind_ok(scale_kind), DF_ERR_INVALID, "%s: bad scale kind %d", fn, scale_kind);
    if (tokens == 0 || H == 0) return DF_OK;
    const int64_t rows1 = act == DF_ACT_GELU ? (int64_t)N : 2 * (int64_t)N;
    const int sz = scale_bytes(scale_kind);
    DF_CHECK(x && logits && W1 && W2 && s1 && s2 && y && ids && weights, DF_ERR_INVALID, "%s: NULL pointer", fn);
    DF_CHECK(ldx >= H && ldy >= H && ld_logits >= experts, DF_ERR_INVALID, "%s: a leading dimension is below its row", fn);
    DF_CHECK(((uintptr_t)x & 1u) == 0 && ((uintptr_t)y & 1u) == 0 &&
                 ((uintptr_t)logits & (logits_dtype == DF_DTYPE_FLOAT32 ? 3u : 1u)) == 0 && aligned4(ids) && aligned4(weights),
             DF_ERR_ALIGN, "%s: a pointer is not aligned to its elements", fn);
    DF_CHECK(ldw1 % 16 == 0 && ldw2 % 16 == 0 && ldw1 >= H && ldw2 >= N && aligned16(W1) && aligned16(W2), DF_ERR_ALIGN,
             "%s: weights need leading dimensions that are multiples of 16, >= %d and %d, and 16-byte alignment", fn, H, N);
    DF_CHECK(lds1 >= rows1 && lds2 >= H && (int64_t)lds1 * sz % 16 == 0 && (int64_t)lds2 * sz % 16 == 0 && aligned16(s1) &&
                 aligned16(s2),
             DF_ERR_ALIGN, "%s: scales need leading dimensions of whole 16 bytes, >= %lld and %d, and 16-byte alignment", fn,
             (long long)rows1, H);
    const int64_t limit = 1ll << 31;
    DF_CHECK(rows1 * ldw1 < limit && (int64_t)H * ldw2 < limit && (((int64_t)H + 127) / 128) * lds1 * sz < limit &&
                 (((int64_t)N + 127) / 128) * lds2 * sz < limit &&
                 (int64_t)tokens * top_k * (((int64_t)N + kStep - 1) & ~(int64_t)(kStep - 1)) * 2 < limit,
             DF_ERR_UNSUPPORTED, "%s: one expert's weights or scales, or the inner values of 2^31 bytes or more", fn);
    const size_t need = df_moe_layer_workspace_bytes(tokens, H, N, experts, top_k);
    DF_CHECK(ws && aligned16(ws) && ws_bytes >= need, DF_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu, or not 16-byte aligned",
             fn, ws ? ws_bytes : (size_t)0, need);
    const int ldh = (N + kStep - 1) & ~(kStep - 1);
    uint16_t* const hi = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(ws) + kPlanBytes);
    uint16_t* const lo = hi + (int64_t)tokens * top_k * ldh;
    float* const part = reinterpret_cast<float*>(lo + (int64_t)tokens * top_k * ldh);
    const int splits = down_splits(tokens, H, N, experts, top_k);
    int* const arrived = reinterpret_cast<int*>(part + (int64_t)splits * tokens * ((H + 15) & ~15));
    const MoeArgs a{x, logits, W1, s1, W2, s2, y, ids, weights, static_cast<MoePlan*>(ws), hi, lo, part,
                    arrived, tokens, H, N, experts, top_k, ldx, ld_logits, ldy, ldw1, ldw2, lds1, lds2, ldh, act, renormalize,
                    dtype, logits_dtype, splits, 0, 0, 0};
    if (scale_kind == DF_SCALE_E8M0) launch<true>(a, as_stream(stream));
    else launch<false>(a, as_stream(stream));
    return launch_status(fn);
}
