// moe.hip -- a mixture-of-experts layer for a few tokens (up to 64: generation),
// on e4m3 weights with a scale per 128 of the reduction (gfx950):
//   ids[t] = the top_k experts by the router's logits, ties to the lower index
//   w[t]   = softmax of their logits (over them, or over all experts)
//   y[t]   = sum over j of w[t][j] * W2[e] . act(W1[e] . x[t]),  e = ids[t][j]
// act: silu(gate) * up or gelu(gate) * up, W1 holding gate's rows, then up's; or
// gelu.
//
// Bound by reading the chosen experts' weights, each once: at 48 tokens to two of
// 32 experts of 3 x 1600 x 1600 that is 240 MB.  So activations stay in 16 bits (no
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
// Widening is exact (e4m3 to bf16 or f16), sums are fp32, scales are applied to each
// step's 128 products in fp32.
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
constexpr int kMoeUnits = kMoePairs / 16 + kMoeExperts;  // more than there can be
constexpr uint32_t kOOB = 0x80000000u;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// What routing leaves for the products, at the workspace's start.
struct MoePlan {
    int units;
    int expert[kMoeUnits], first[kMoeUnits], count[kMoeUnits];  // a unit's expert, its pairs in `sorted`
    int sorted[kMoePairs];                                      // pairs t * top + j by expert, then token
};

struct MoeArgs {
    const void* x; const void* logits;
    const uint8_t* W1; const void* s1; const uint8_t* W2; const void* s2;
    void* y; int* ids; float* weights;
    MoePlan* plan;
    uint16_t* hi; uint16_t* lo;  // [pairs][ldh] bf16
    int tokens, H, N, experts, top, ldx, ldl, ldy, ldw1, ldw2, lds1, lds2, ldh, act, renormalize, x_dtype, l_dtype;
};

// ------------------------------------------------------------------ routing --
__device__ __forceinline__ float load_as_float(const void* p, int dtype, int64_t i) {
    if (dtype == DF_DTYPE_FLOAT32) return static_cast<const float*>(p)[i];
    if (dtype == DF_DTYPE_HALF) return (float)__builtin_bit_cast(_Float16, static_cast<const uint16_t*>(p)[i]);
    return bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
}

template <typename F> __device__ __forceinline__ uint32_t wave_fold(uint32_t v, const F& f) {
#define DF_FOLD(CTRL) v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false))
    DF_FOLD(0x111);  // row_shr:1 .. 8, then row_bcast:15 and :31: lane 63 has the wave's
    DF_FOLD(0x112);
    DF_FOLD(0x114);
    DF_FOLD(0x118);
    DF_FOLD(0x142);
    DF_FOLD(0x143);
#undef DF_FOLD
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// One wave: token t's choices, the j-th in lane j: its expert and weight, -1 and 0
// where no more can be chosen (an expert whose logit is -infinity or NaN is none).
__device__ __forceinline__ void route_token(const MoeArgs& a, int t, int lane, int& id, float& weight) {
    constexpr int PER = kMoeExperts / 64;
    float v[PER];
    uint32_t key[PER];  // order of the values; 0: cannot be chosen
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 64 * i;
        v[i] = e < a.experts ? load_as_float(a.logits, a.l_dtype, (int64_t)t * a.ldl + e) : -__builtin_inff();
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
        best = wave_fold(best, [](uint32_t x, uint32_t y) { return max(x, y); });
        if (best == 0) break;
        uint32_t who = 0xFFFFFFFFu;
#pragma unroll
        for (int i = PER - 1; i >= 0; --i) who = key[i] == best ? (uint32_t)(lane + 64 * i) : who;
        who = wave_fold(who, [](uint32_t x, uint32_t y) { return min(x, y); });
        if (j == 0) first = best;
        if (lane == j) {
            id = (int)who;
            mine = best;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if ((uint32_t)(lane + 64 * i) == who) key[i] = 0;
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
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off, 64);
    weight = id >= 0 ? own / sum : 0.0f;
}

// One block: every token's choices, then the plan.
__global__ __launch_bounds__(1024) void moe_route_kernel(const MoeArgs a) {
    __shared__ int ids[kMoePairs];
    __shared__ uint32_t taken[kMoeExperts][kMoeTokens / 32];  // which tokens take an expert
    __shared__ int start[kMoeExperts], at_wave[2][4];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < kMoeExperts * (kMoeTokens / 32); i += 1024) (&taken[0][0])[i] = 0;
    __syncthreads();
    for (int t = w; t < a.tokens; t += 16) {
        int e;
        float weight;
        route_token(a, t, lane, e, weight);
        if (lane < a.top) {
            const int p = t * a.top + lane;
            ids[p] = e;
            a.ids[p] = e;
            a.weights[p] = weight;
            if (e >= 0) atomicOr(&taken[e][t >> 5], 1u << (t & 31));
        }
    }
    __syncthreads();
    // experts' pairs and units, added up in order of the experts
    const int e = threadIdx.x;
    int n = 0, units = 0, s = 0, u = 0;
    if (e < kMoeExperts) {
#pragma unroll
        for (int i = 0; i < kMoeTokens / 32; ++i) n += __builtin_popcount(taken[e][i]);
        units = (n + 15) / 16;
        s = n;
        u = units;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int so = __shfl_up(s, off, 64), uo = __shfl_up(u, off, 64);
            if (lane >= off) {
                s += so;
                u += uo;
            }
        }
        if (lane == 63) {
            at_wave[0][w] = s;
            at_wave[1][w] = u;
        }
    }
    __syncthreads();
    if (e < kMoeExperts) {
        for (int i = 0; i < w; ++i) {
            s += at_wave[0][i];
            u += at_wave[1][i];
        }
        start[e] = s - n;
        for (int i = 0; i < units; ++i) {
            const int k = u - units + i;
            a.plan->expert[k] = e;
            a.plan->first[k] = s - n + 16 * i;
            a.plan->count[k] = min(n - 16 * i, 16);
        }
        if (e == kMoeExperts - 1) a.plan->units = u;
    }
    __syncthreads();
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
template <bool E8> __device__ __forceinline__ uint32_t load_scale(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    if constexpr (E8) return __builtin_amdgcn_raw_buffer_load_b8(r, at, 0, 0);
    else return __builtin_amdgcn_raw_buffer_load_b32(r, at == kOOB ? kOOB : at * 4, 0, 0);
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
template <typename V, bool E8, bool GATED>
__global__ __launch_bounds__(256) void moe_up_kernel(const MoeArgs a) {
    constexpr int W = 4, U = 4, COLS = GATED ? 16 : 32;
    __shared__ float red[W][2][16][20];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * COLS, unit = blockIdx.y;
    if (n0 >= a.N) return;
    const int fr = lane & 15, fq = lane >> 4;
    int e, count, pair = -1;
    float weight1 = 0.0f;
    if (a.tokens == 1) {  // the unit is a choice
        int id;
        float weight;
        route_token(a, 0, lane, id, weight);
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
        if (unit >= a.plan->units) return;
        e = a.plan->expert[unit];
        count = a.plan->count[unit];
        if (fr < count) pair = a.plan->sorted[a.plan->first[unit] + fr];
    }
    const int rows1 = GATED ? 2 * a.N : a.N, blocks = (a.H + 127) >> 7;
    const __amdgpu_buffer_rsrc_t rW = buffer(a.W1 + (int64_t)e * rows1 * a.ldw1, (int64_t)rows1 * a.ldw1);
    const __amdgpu_buffer_rsrc_t rS =
        buffer(static_cast<const uint8_t*>(a.s1) + (int64_t)e * blocks * a.lds1 * (E8 ? 1 : 4), (int64_t)blocks * a.lds1 * (E8 ? 1 : 4));
    uint32_t row[2];
    bool ok[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int n = n0 + (GATED ? 0 : 16 * g) + fr;
        ok[g] = n < a.N;
        row[g] = (uint32_t)(n + (GATED ? g * a.N : 0));
    }
    const uint16_t* const xr = static_cast<const uint16_t*>(a.x) + (int64_t)(max(pair, 0) / a.top) * a.ldx;
    const int K16 = (a.H + 15) & ~15;

    struct Step {
        u32x4 w[2][2], x[2][2];
        uint32_t s[2];
    };
    auto load = [&](Step& s, int step) {
        const int k = step * 128 + 16 * fq;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool in = k + 64 * h < K16;
#pragma unroll
            for (int g = 0; g < 2; ++g)
                s.w[g][h] = __builtin_bit_cast(
                    u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                               rW, in && ok[g] ? row[g] * (uint32_t)a.ldw1 + (uint32_t)(k + 64 * h) : kOOB, 0, 0));
#pragma unroll
            for (int c = 0; c < 2; ++c)
                s.x[h][c] = pair >= 0 ? load_chunk<uint16_t>(xr, k / 8 + 8 * h + c, a.H) : u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int g = 0; g < 2; ++g)
            s.s[g] = load_scale<E8>(rS, ok[g] && step < blocks ? (uint32_t)step * (uint32_t)a.lds1 + row[g] : kOOB);
    };
    v4f acc[2] = {};
    auto multiply = [&](Step& s, int step) {
        if (step * 128 + 128 > a.H) {  // the row's end, which its last chunk was loaded up to
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    s.x[h][c] = place_chunk<uint16_t>(s.x[h][c], step * 16 + 2 * fq + 8 * h + c, a.H);
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
    for (int u = 0; u < U; ++u) load(buf[u], w + u * W);
    for (int s = w; s < blocks; s += W * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u * W < blocks) multiply(buf[u], s + u * W);
            load(buf[u], s + (u + U) * W);
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
    const int p = a.tokens == 1 ? unit : a.plan->sorted[a.plan->first[unit] + i];
    const float weight = a.tokens == 1 ? weight1 : a.weights[p];
    auto put = [&](int n, float h) {
        if (n >= a.ldh) return;
        h = n < a.N ? h * weight : 0.0f;  // zeros up to the next multiple of 16
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

// W2 and the weighted sum.  blockIdx.x: 16 columns of y.
template <bool E8> __global__ __launch_bounds__(512) void moe_down_kernel(const MoeArgs a) {
    constexpr int W = 8, U = 2;
    __shared__ int expert[kMoeUnits], first[kMoeUnits], count[kMoeUnits], sorted[kMoePairs];
    __shared__ float sums[W][kMoeTokens][17];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h0 = blockIdx.x * 16, pairs = a.tokens * a.top;
    int units;
    if (a.tokens == 1) {
        units = a.top;
        if ((int)threadIdx.x < units) {
            expert[threadIdx.x] = a.ids[threadIdx.x];
            first[threadIdx.x] = threadIdx.x;
            count[threadIdx.x] = a.ids[threadIdx.x] >= 0;
            sorted[threadIdx.x] = threadIdx.x;
        }
    } else {
        units = a.plan->units;
        for (int i = threadIdx.x; i < units; i += 512) {
            expert[i] = a.plan->expert[i];
            first[i] = a.plan->first[i];
            count[i] = a.plan->count[i];
        }
        for (int i = threadIdx.x; i < pairs; i += 512) sorted[i] = a.plan->sorted[i];
    }
    for (int i = lane; i < a.tokens * 17; i += 64) sums[w][i / 17][i % 17] = 0.0f;
    __syncthreads();
    const int fr = lane & 15, fq = lane >> 4;
    const int steps = (a.N + 127) >> 7, K16 = a.ldh;
    const int64_t bytes2 = (int64_t)a.H * a.ldw2, sbytes2 = (int64_t)steps * a.lds2 * (E8 ? 1 : 4);
    const __amdgpu_buffer_rsrc_t rHi = buffer(a.hi, (int64_t)pairs * a.ldh * 2), rLo = buffer(a.lo, (int64_t)pairs * a.ldh * 2);
    const bool ok = h0 + fr < a.H;
    const uint32_t row = (uint32_t)(h0 + fr);
    const int total = units * steps, lo_f = (int)((int64_t)total * w / W), hi_f = (int)((int64_t)total * (w + 1) / W);

    struct Step {
        u32x4 w[2], hi[2][2], lo[2][2];
        uint32_t s;
    };
    auto load = [&](Step& s, int f) {
        const bool live = f < hi_f;
        const int u = live ? f / steps : 0, step = f - u * steps;
        const int e = max(__builtin_amdgcn_readfirstlane(live ? expert[u] : 0), 0);
        const int n = __builtin_amdgcn_readfirstlane(live ? count[u] : 0);
        const int pair = fr < n ? sorted[first[u] + fr] : -1;
        const __amdgpu_buffer_rsrc_t rW = buffer(a.W2 + (int64_t)e * bytes2, bytes2);
        const __amdgpu_buffer_rsrc_t rS = buffer(static_cast<const uint8_t*>(a.s2) + (int64_t)e * sbytes2, sbytes2);
        const int k = step * 128 + 16 * fq;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool in = n > 0 && k + 64 * h < K16;
            s.w[h] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                         rW, in && ok ? row * (uint32_t)a.ldw2 + (uint32_t)(k + 64 * h) : kOOB, 0, 0));
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t at = in && pair >= 0 ? ((uint32_t)pair * (uint32_t)a.ldh + (uint32_t)(k + 64 * h + 8 * c)) * 2u : kOOB;
                s.hi[h][c] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rHi, at, 0, 0));
                s.lo[h][c] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rLo, at, 0, 0));
            }
        }
        s.s = load_scale<E8>(rS, ok && n > 0 ? (uint32_t)step * (uint32_t)a.lds2 + row : kOOB);
    };
    v4f acc = {};
    auto multiply = [&](const Step& s, int f) {
        v4f p = {};
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const bf8 v = widen8_scaled<E4M3>(s.w[h][2 * c], s.w[h][2 * c + 1], 1.0f);
                p = mfma16(__builtin_bit_cast(bf8, s.lo[h][c]), v, p);
                p = mfma16(__builtin_bit_cast(bf8, s.hi[h][c]), v, p);
            }
        const float sc = scale_value<E8>(s.s);
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[r] = __builtin_fmaf(p[r], sc, acc[r]);
        const int u = f / steps;
        if (f + 1 == hi_f || f + 1 == (u + 1) * steps) {  // the unit's end, or this wave's
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int i = 4 * fq + r;
                if (i < count[u]) sums[w][sorted[first[u] + i] / a.top][fr] += acc[r];
            }
            acc = v4f{};
        }
    };
    Step buf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(buf[u], lo_f + u);
    for (int f = lo_f; f < hi_f; f += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (f + u < hi_f) multiply(buf[u], f + u);
            load(buf[u], f + u + U);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.tokens * 16; i += 512) {
        const int t = i >> 4, c = i & 15;
        if (h0 + c >= a.H) continue;
        float v = 0.0f;
#pragma unroll
        for (int x = 0; x < W; ++x) v += sums[x][t][c];
        const int64_t at = (int64_t)t * a.ldy + h0 + c;
        if (a.x_dtype == DF_DTYPE_HALF) static_cast<f16_t*>(a.y)[at] = OutCvt<f16_t>::cvt(v);
        else static_cast<uint16_t*>(a.y)[at] = OutCvt<uint16_t>::cvt(v);
    }
}

template <bool E8> void launch(const MoeArgs& a, hipStream_t st) {
    const bool gated = a.act != DF_ACT_GELU;
    const int cols = gated ? 16 : 32;
    const int pairs = a.tokens * a.top;
    const int units = a.tokens == 1 ? a.top : std::min(a.experts, pairs) + pairs / 16;
    if (a.tokens > 1) moe_route_kernel<<<1, 1024, 0, st>>>(a);
    // columns' blocks to a multiple of 8: an expert's units then share an XCD's L2
    const dim3 grid((((a.N + cols - 1) / cols) + 7) / 8 * 8, units);
    if (a.x_dtype == DF_DTYPE_HALF) {
        if (gated) moe_up_kernel<h8, E8, true><<<grid, 256, 0, st>>>(a);
        else moe_up_kernel<h8, E8, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (gated) moe_up_kernel<bf8, E8, true><<<grid, 256, 0, st>>>(a);
        else moe_up_kernel<bf8, E8, false><<<grid, 256, 0, st>>>(a);
    }
    moe_down_kernel<E8><<<(a.H + 15) / 16, 512, 0, st>>>(a);
}

constexpr size_t kPlanBytes = (sizeof(MoePlan) + 255) / 256 * 256;

}  // namespace

}  // namespace dfk

using namespace dfk;

extern "C" size_t df_moe_layer_workspace_bytes(int tokens, int top_k, int N) {
    if (tokens <= 0 || tokens > kMoeTokens || top_k <= 0 || top_k > kMoeTop || N <= 0 || N > 0x7FFFFFF0) return 0;
    return kPlanBytes + (size_t)tokens * top_k * (((size_t)N + 15) & ~(size_t)15) * 4;
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
                 (int64_t)tokens * top_k * (((int64_t)N + 15) & ~15ll) * 2 < limit,
             DF_ERR_UNSUPPORTED, "%s: one expert's weights or scales, or the inner values of 2^31 bytes or more", fn);
    const size_t need = df_moe_layer_workspace_bytes(tokens, top_k, N);
    DF_CHECK(ws && aligned16(ws) && ws_bytes >= need, DF_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu, or not 16-byte aligned",
             fn, ws ? ws_bytes : (size_t)0, need);
    const int ldh = (N + 15) & ~15;
    uint16_t* const hi = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(ws) + kPlanBytes);
    const MoeArgs a{x, logits, W1, s1, W2, s2, y, ids, weights, static_cast<MoePlan*>(ws), hi,
                    hi + (int64_t)tokens * top_k * ldh, tokens, H, N, experts, top_k, ldx, ld_logits, ldy, ldw1, ldw2, lds1,
                    lds2, ldh, act, renormalize, dtype, logits_dtype};
    if (scale_kind == DF_SCALE_E8M0) launch<true>(a, as_stream(stream));
    else launch<false>(a, as_stream(stream));
    return launch_status(fn);
}
