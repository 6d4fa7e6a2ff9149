// rmsnorm.hip -- root-mean-square norm over rows, with the residual add in
// front of it: the forward that keeps rstd, its output in the element type or
// as fp8 codes with a scale per 128 columns, and the backward with the reduction
// of gamma's gradient (gfx950).
//
// Per row of n values, s = x + residual rounded to the element type:
//   rstd = 1/sqrt(sum(s^2)/n + eps),  y = s * rstd * gamma
// codes: q = y / scale of each 128 columns, from y in fp32 (not rounded to the
// element type first).  Backward, with xh = s * rstd and g = dy * gamma:
//   dx = rstd * (g - xh * mean(g * xh)) + dresidual,  dgamma = sum(dy * xh)
//
// Bound by HBM, each value read and written once: a row stays in registers from
// its load to its store, by the same division of rows over lanes as LayerNorm's
// (layernorm.hip).  The 128 columns of a scale are 16 lanes' chunks of 2-byte
// values (32 lanes' of fp32), so their absmax is a DPP row's maximum.  Sums
// are binary32, per lane in order, then in a fixed order over lanes and waves.
//
// Measured (bf16, residual in and sum out): 16384 x 1600 to codes in powers of two 38
// us (184 MB, 4.8 TB/s where a copy reaches 5.2), backward 41 (210 MB, 5.1 TB/s), of which
// 4 for the fold of gamma's partial sums; one row of 768 3.6, a launch.
//
// The reference has LayerNorm only (dnn/layers/layer_norm_layer.cu:26-90).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "block_scale.hpp"
#include "df_common.hpp"
#include "row_chunks.hpp"

namespace dfk {

namespace {

template <typename T> struct RmsFwd {
    const T* x; const T* res; T* sum; T* y; const T* gamma; float* rstd;
    uint8_t* q; void* s;  // codes [rows, ldq], scales [blocks, ldsc]
    int rows, cols, ldx, ldr, lds, ldy, ldq, ldsc, fmt;
    float eps;
};

// What is written beside y: nothing, or codes with scales of a kind
enum : int { OUT_Y = 0, OUT_E8 = 1, OUT_F32 = 2 };

// codes of E values (4 or 8) at block b
template <int FMT, bool E8, int E> __device__ __forceinline__ void put_codes(uint8_t* p, const float* v, const BlockDiv& b) {
    bool bad = !b.d.fast;
#pragma unroll
    for (int e = 0; e < E; e += 2) bad |= __builtin_isunordered(v[e], v[e + 1]);
    uint32_t w[E / 4];
    if (__builtin_amdgcn_ballot_w64(bad) == 0) {
#pragma unroll
        for (int e = 0; e < E; e += 4) w[e / 4] = block_quant4<FMT, E8, true>(v + e, b.d);
    } else {
#pragma unroll
        for (int e = 0; e < E; e += 4) w[e / 4] = block_quant4<FMT, E8, false>(v + e, b.d);
    }
    if constexpr (E == 8) *reinterpret_cast<u32x2*>(p) = u32x2{w[0], w[1]};
    else *reinterpret_cast<uint32_t*>(p) = w[0];
}

// ------------------------------------------------------------------ forward --
template <typename T, int RT, int CH, int OUT>
__global__ __launch_bounds__(RT == 64 ? 256 : RT) void rms_forward_kernel(const RmsFwd<T> a) {
    constexpr int E = El<T>::E;
    constexpr int RPB = RT == 64 ? 4 : 1;  // rows a block works on at once
    constexpr int GL = kScaleBlock / E;    // lanes that share a scale
    // The next row's loads before this row's arithmetic, gamma in registers; with codes
    // and a wave's four chunks a thread that took 158 registers, three waves a SIMD: no
    // row ahead then, and gamma in LDS (16384 x 1600: 43 us, 40 so)
    constexpr bool AHEAD = OUT == OUT_Y || CH < 4 || RT > 64;
    __shared__ u32x4 glds[AHEAD ? 1 : CH][AHEAD ? 1 : RT];
    __shared__ float red[2][2][1][RT / 64];
    const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
    RowSum<RT> rs{red};
    u32x4 gw[CH], nx[CH], nr[CH];
    const bool affine = a.gamma != nullptr, add = a.res != nullptr;
    auto fetch = [&](int r) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < CH; ++k) nx[k] = load_chunk<T>(a.x + (int64_t)r * a.ldx, t + RT * k, a.cols);
        if (add) {
#pragma unroll
            for (int k = 0; k < CH; ++k) nr[k] = load_chunk<T>(a.res + (int64_t)r * a.ldr, t + RT * k, a.cols);
        }
    };
    const int units = gridDim.x * RPB;
    const int unit = blockIdx.x * RPB + (RT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
    int r = unit;
    if (AHEAD && r < a.rows) fetch(r);
    if (affine) {
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const u32x4 w = place_chunk<T>(load_chunk<T>(a.gamma, t + RT * k, a.cols), t + RT * k, a.cols);
            if constexpr (AHEAD) gw[k] = w;
            else glds[k][t] = w;  // (every wave the same, its own lanes')
        }
    }
    // no wave stores of the first row before all have its loads on their way: a
    // row's last chunk holds values of the one before it, and the sum may lie over x
    if constexpr (RT > 64) __syncthreads();
    for (; r < a.rows; r += units) {
        if (!AHEAD) fetch(r);
        float v[CH][E];
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            El<T>::widen(place_chunk<T>(nx[k], t + RT * k, a.cols), v[k]);
            if (add) {
                float p[E];
                El<T>::widen(place_chunk<T>(nr[k], t + RT * k, a.cols), p);
#pragma unroll
                for (int e = 0; e < E; ++e) v[k][e] += p[e];
                const u32x4 w = El<T>::narrow(v[k]);  // the norm is that of the sum as stored
                El<T>::widen(w, v[k]);
                if (a.sum) store_chunk<T>(a.sum + (int64_t)r * a.lds, t + RT * k, a.cols, w);
            }
        }
        if (AHEAD && r + units < a.rows) fetch(r + units);
        float sq = 0.0f;
#pragma unroll
        for (int k = 0; k < CH; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) sq = __builtin_fmaf(v[k][e], v[k][e], sq);
        const float rstd = 1.0f / __builtin_sqrtf(rs.one(sq) / (float)a.cols + a.eps);
        if (t == 0 && a.rstd) a.rstd[r] = rstd;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const int c = (t + RT * k) * E;
#pragma unroll
            for (int e = 0; e < E; ++e) v[k][e] *= rstd;
            if (affine) {
                float g[E];
                if constexpr (AHEAD) El<T>::widen(gw[k], g);
                else El<T>::widen(glds[k][t], g);
#pragma unroll
                for (int e = 0; e < E; ++e) v[k][e] *= g[e];
            }
            if (OUT == OUT_Y || a.y) store_chunk<T>(a.y + (int64_t)r * a.ldy, t + RT * k, a.cols, El<T>::narrow(v[k]));
            if constexpr (OUT != OUT_Y) {
                // (values past the row's end are 0, unless the row's rstd or sum is
                // not finite: then they are NaN, and left out here)
                uint32_t most = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    if (c + e >= a.cols) v[k][e] = 0.0f;
                    most = fold_f32_biased(most, __float_as_uint(v[k][e]));
                }
                most = row16_max(unbias_f32(most));
                if constexpr (GL == 32) most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
                constexpr bool E8 = OUT == OUT_E8;
                auto codes = [&](auto fmt) {
                    constexpr int F = decltype(fmt)::value;
                    const BlockDiv b = block_div<F, E8>(most);
                    if (c < ((a.cols + 15) & ~15)) put_codes<F, E8, E>(a.q + (int64_t)r * a.ldq + c, v[k], b);
                    if ((t & (GL - 1)) == 0 && c < a.cols) {
                        const int64_t at = (int64_t)(c / kScaleBlock) * a.ldsc + r;
                        if constexpr (E8) static_cast<uint8_t*>(a.s)[at] = (uint8_t)b.byte;
                        else static_cast<float*>(a.s)[at] = b.d.s;
                    }
                };
                if (a.fmt == E4M3) codes(std::integral_constant<int, E4M3>{});
                else codes(std::integral_constant<int, E5M2>{});
            }
        }
    }
}

// Rows wider than a block's registers: a block reads its row twice; a wave
// quantizes 128 columns at a time.
constexpr int kWide = 1024;
template <typename T, int OUT> __global__ __launch_bounds__(kWide) void rms_forward_wide_kernel(const RmsFwd<T> a) {
    __shared__ float red[2][2][1][kWide / 64];
    RowSum<kWide> rs{red};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* xr = a.x + (int64_t)r * a.ldx;
        const T* rr = a.res ? a.res + (int64_t)r * a.ldr : nullptr;
        auto at = [&](int c) {
            float v = El<T>::one(xr + c);
            if (rr) {
                T p;
                El<T>::put(&p, v + El<T>::one(rr + c));
                v = El<T>::one(&p);
            }
            return v;
        };
        float sq = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kWide) {
            const float v = at(c);
            sq = __builtin_fmaf(v, v, sq);
        }
        const float rstd = 1.0f / __builtin_sqrtf(rs.one(sq) / (float)a.cols + a.eps);
        if (threadIdx.x == 0 && a.rstd) a.rstd[r] = rstd;
        const int blocks = (a.cols + kScaleBlock - 1) / kScaleBlock;
        for (int b = wave; b < blocks; b += kWide / 64) {
            const int c = b * kScaleBlock + 2 * lane;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            uint32_t most = 0;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (c + e >= a.cols) continue;
                const float s = at(c + e);
                v[e] = s * rstd;
                if (a.gamma) v[e] *= El<T>::one(a.gamma + c + e);
                if (rr && a.sum) El<T>::put(a.sum + (int64_t)r * a.lds + c + e, s);
                if (OUT == OUT_Y || a.y) El<T>::put(a.y + (int64_t)r * a.ldy + c + e, v[e]);
                most = fold_f32(most, __float_as_uint(v[e]));
            }
            if constexpr (OUT != OUT_Y) {
                most = row16_max(most);
                most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
                most = max(most, (uint32_t)__shfl_xor((int)most, 32, 64));
                constexpr bool E8 = OUT == OUT_E8;
                auto codes = [&](auto fmt) {
                    constexpr int F = decltype(fmt)::value;
                    const BlockDiv d = block_div<F, E8>(most);
                    if (c < ((a.cols + 15) & ~15))
                        *reinterpret_cast<uint16_t*>(a.q + (int64_t)r * a.ldq + c) = (uint16_t)block_quant4<F, E8, false>(v, d.d);
                    if (lane == 0) {
                        const int64_t p = (int64_t)b * a.ldsc + r;
                        if constexpr (E8) static_cast<uint8_t*>(a.s)[p] = (uint8_t)d.byte;
                        else static_cast<float*>(a.s)[p] = d.d.s;
                    }
                };
                if (a.fmt == E4M3) codes(std::integral_constant<int, E4M3>{});
                else codes(std::integral_constant<int, E5M2>{});
            }
        }
    }
}

// ----------------------------------------------------------------- backward --
template <typename T> struct RmsBwd {
    const T* dy; const T* x; const T* gamma; const float* rstd; const T* dres; T* dx;
    float* dgamma;  // written by the kernel itself when one block runs
    float* part;    // [blocks][cols]: each block's sums of dy * xh
    int rows, cols, lddy, ldx, lddr, lddx;
    float eps;
};

// As LayerNorm's: a block of NT threads works on NT / RT rows at once, a thread
// on the same columns of all its rows, so gamma's sums stay in its registers; the
// row groups' sums meet in LDS and leave as one partial per block, which
// rms_fold_kernel adds in block order.  SUMS: gamma's gradient is wanted.
constexpr int bwd_threads(int rt) { return rt > 512 ? rt : 512; }
template <typename T, int RT, int CH, bool SUMS>
__device__ __forceinline__ void backward_rows(const RmsBwd<T>& a, int blocks) {
    constexpr int E = El<T>::E;
    constexpr int GP = bwd_threads(RT) / RT;
    __shared__ float red[2][2][GP][RT / 64];
    const int t = threadIdx.x % RT, group = __builtin_amdgcn_readfirstlane(threadIdx.x / RT);
    RowSum<RT, GP> rs{red};
    // gamma in LDS: reading it there waits for no load under way
    __shared__ u32x4 gw[CH][bwd_threads(RT)];
    const bool affine = a.gamma != nullptr, add = a.dres != nullptr, given = a.rstd != nullptr;
    // The chunk in which the rows end holds this many values of the chunk before
    // it; they stay where they were loaded, gamma's likewise, count for no sum
    // and are not stored.
    auto borrowed = [&](int k) { return a.cols < E ? 0 : max(0, (t + RT * k) * E + E - a.cols); };
    float sg[CH][E];
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) sg[k][e] = 0.0f;
    const int step = blocks * GP;
    int r = blockIdx.x * GP + group;
    if (affine) {
#pragma unroll
        for (int k = 0; k < CH; ++k) gw[k][threadIdx.x] = load_chunk<T>(a.gamma, t + RT * k, a.cols);
    }
    const float inv = 1.0f / (float)a.cols;
    // the block's groups go round together (they share barriers); a group past
    // the last row works on zeros and stores nothing
    for (int base = blockIdx.x * GP; base < a.rows; base += step, r += step) {
        const bool live = GP == 1 || r < a.rows;
        u32x4 cx[CH], cy[CH], cr[CH];
        float rstd = 0.0f;
#pragma unroll
        for (int k = 0; k < CH; ++k) cx[k] = cy[k] = u32x4{0, 0, 0, 0};
        if (live) {
#pragma unroll
            for (int k = 0; k < CH; ++k) cx[k] = load_chunk<T>(a.x + (int64_t)r * a.ldx, t + RT * k, a.cols);
#pragma unroll
            for (int k = 0; k < CH; ++k) cy[k] = load_chunk<T>(a.dy + (int64_t)r * a.lddy, t + RT * k, a.cols);
            if (add) {
#pragma unroll
                for (int k = 0; k < CH; ++k) cr[k] = load_chunk<T>(a.dres + (int64_t)r * a.lddr, t + RT * k, a.cols);
            }
            if (given) rstd = a.rstd[r];
        }
        if (!given) {
            float sq = 0.0f;
#pragma unroll
            for (int k = 0; k < CH; ++k) {
                float v[E];
                El<T>::widen(place_chunk<T>(cx[k], t + RT * k, a.cols), v);
#pragma unroll
                for (int e = 0; e < E; ++e) sq = __builtin_fmaf(v[e], v[e], sq);
            }
            rstd = 1.0f / __builtin_sqrtf(rs.one(sq) / (float)a.cols + a.eps);
            if (GP > 1 && !live) rstd = 0.0f;
        }
        auto terms = [&](int k, float* xh, float* d, float* g) __attribute__((always_inline)) {
            El<T>::widen(cx[k], xh);
            El<T>::widen(cy[k], d);
            float w[E];
            if (affine) El<T>::widen(gw[k][threadIdx.x], w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[e] *= rstd;
                g[e] = affine ? d[e] * w[e] : d[e];
            }
        };
        float c2 = 0.0f;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            __builtin_amdgcn_sched_barrier(0);  // one chunk's terms at a time: registers
            float xh[E], d[E], g[E];
            terms(k, xh, d, g);
            const int over = borrowed(k);
            if (over > 0) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (e < over) g[e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (SUMS) sg[k][e] = __builtin_fmaf(d[e], xh[e], sg[k][e]);
                c2 = __builtin_fmaf(g[e], xh[e], c2);
            }
        }
        c2 = rs.one(c2) * inv;
        if (!live) continue;
        // the terms again from the row as loaded, not kept: registers
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            __builtin_amdgcn_sched_barrier(0);
            float xh[E], d[E], g[E], p[E];
            terms(k, xh, d, g);
            if (add) El<T>::widen(cr[k], p);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                g[e] = rstd * __builtin_fmaf(-xh[e], c2, g[e]);
                if (add) g[e] += p[e];
            }
            store_chunk<T>(a.dx + (int64_t)r * a.lddx, t + RT * k, a.cols,
                           place_chunk<T>(El<T>::narrow(g), t + RT * k, a.cols));
        }
    }
    if constexpr (SUMS) {
        float* const og = blocks == 1 ? a.dgamma : a.part + (int64_t)blockIdx.x * a.cols;
        if constexpr (GP > 1) {
            // halves onto halves; a thread's values lie RT apart: no bank conflicts
            __shared__ float slab[GP / 2][CH * E * RT];
#pragma unroll
            for (int half = GP / 2; half > 0; half >>= 1) {
                if (group >= half && group < 2 * half) {
#pragma unroll
                    for (int k = 0; k < CH; ++k)
#pragma unroll
                        for (int e = 0; e < E; ++e) slab[group - half][(k * E + e) * RT + t] = sg[k][e];
                }
                __syncthreads();
                if (group < half) {
#pragma unroll
                    for (int k = 0; k < CH; ++k)
#pragma unroll
                        for (int e = 0; e < E; ++e) sg[k][e] += slab[group][(k * E + e) * RT + t];
                }
                __syncthreads();
            }
            if (group != 0) return;
        }
#pragma unroll
        for (int k = 0; k < CH; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int c = (t + RT * k) * E + e - borrowed(k);
                if (e >= borrowed(k) && c < a.cols) og[c] = sg[k][e];
            }
    }
}

template <typename T, int RT, int CH, bool SUMS>
__global__ __launch_bounds__(bwd_threads(RT), 4) void rms_backward_kernel(const RmsBwd<T> a) {
    backward_rows<T, RT, CH, SUMS>(a, gridDim.x);
}

// Few rows, rstd given: dx and the column sums in one launch; the blocks behind
// the first `row_blocks` take a few columns each and read dy and x again, from
// the L2 that the rows' blocks fill (sizes as for LayerNorm's).
constexpr int kOnceLoads = 8;
constexpr int once_cols(int rt) { return rt <= 128 ? 16 : 32; }
template <typename T, int RT, int CH>
__global__ __launch_bounds__(bwd_threads(RT), 4) void rms_backward_once_kernel(const RmsBwd<T> a, int row_blocks) {
    if ((int)blockIdx.x < row_blocks) {
        backward_rows<T, RT, CH, false>(a, row_blocks);
        return;
    }
    constexpr int W = bwd_threads(RT) / 64, CW = once_cols(RT);
    __shared__ float red[W][CW];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = lane % CW;
    const int c = ((int)blockIdx.x - row_blocks) * CW + i;
    float sg = 0.0f;
    if (c < a.cols) {
        constexpr int STEP = 64 / CW * W;
        // kOnceLoads rows from r0; LAST: only those that there are
        auto rows = [&](int r0, auto last) __attribute__((always_inline)) {
            constexpr bool LAST = decltype(last)::value;
            float d[kOnceLoads], x[kOnceLoads], q[kOnceLoads];
#pragma unroll
            for (int k = 0; k < kOnceLoads; ++k) {
                const int r = LAST ? min(r0 + k * STEP, a.rows - 1) : r0 + k * STEP;
                d[k] = El<T>::one(a.dy + (int64_t)r * a.lddy + c);
                x[k] = El<T>::one(a.x + (int64_t)r * a.ldx + c);
                q[k] = a.rstd[r];
            }
#pragma unroll
            for (int k = 0; k < kOnceLoads; ++k)
                if (!LAST || r0 + k * STEP < a.rows) sg = __builtin_fmaf(d[k], x[k] * q[k], sg);
        };
        int r = threadIdx.x / CW;
        for (; r + (kOnceLoads - 1) * STEP < a.rows; r += kOnceLoads * STEP) rows(r, std::false_type{});
        if (r < a.rows) rows(r, std::true_type{});
    }
#pragma unroll
    for (int off = CW; off < 64; off <<= 1) sg += __shfl_xor(sg, off, 64);
    if (lane < CW) red[w][i] = sg;
    __syncthreads();
    if (w == 0 && lane < CW && c < a.cols) {
#pragma unroll
        for (int v = 1; v < W; ++v) sg += red[v][i];
        a.dgamma[c] = sg;
    }
}

// dgamma from `parts` partials of cols values: a block takes 32 columns, its
// half waves every 16th partial each, in order
constexpr int kFoldWaves = 8, kFoldCols = 32, kFoldParts = kFoldWaves * (64 / kFoldCols);
__global__ __launch_bounds__(64 * kFoldWaves) void rms_fold_kernel(const float* __restrict__ part, int parts, int cols,
                                                                   float* __restrict__ dgamma) {
    __shared__ float red[kFoldParts][kFoldCols];
    const int i = threadIdx.x % kFoldCols, mine = threadIdx.x / kFoldCols;
    const int64_t width = cols, c = (int64_t)blockIdx.x * kFoldCols + i;
    float s = 0.0f;
    if (c < width) {
        int p = mine;
        for (; p + 7 * kFoldParts < parts; p += 8 * kFoldParts) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = part[(p + k * kFoldParts) * width + c];
#pragma unroll
            for (int k = 0; k < 8; ++k) s += v[k];
        }
        for (; p < parts; p += kFoldParts) s += part[p * width + c];
    }
    red[mine][i] = s;
    __syncthreads();
    if (mine == 0 && c < width) {
#pragma unroll
        for (int k = 1; k < kFoldParts; ++k) s += red[k][i];
        dgamma[c] = s;
    }
}

// Rows wider than a block's registers: rstd where it is not given, the column
// sums (a thread per column, blockIdx.y's share of the rows), then dx, each from
// memory.
template <typename T>
__global__ __launch_bounds__(kWide) void rms_stats_wide_kernel(const T* x, int rows, int cols, int ldx, float eps,
                                                               float* rstd) {
    __shared__ float red[2][2][1][kWide / 64];
    RowSum<kWide> rs{red};
    for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + (int64_t)r * ldx;
        float sq = 0.0f;
        for (int c = threadIdx.x; c < cols; c += kWide) {
            const float v = El<T>::one(xr + c);
            sq = __builtin_fmaf(v, v, sq);
        }
        sq = rs.one(sq);
        if (threadIdx.x == 0) rstd[r] = 1.0f / __builtin_sqrtf(sq / (float)cols + eps);
    }
}
template <typename T> __global__ __launch_bounds__(256) void rms_colsum_wide_kernel(const RmsBwd<T> a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    float sg = 0.0f;
    for (int r = blockIdx.y; r < a.rows; r += gridDim.y)
        sg = __builtin_fmaf(El<T>::one(a.dy + (int64_t)r * a.lddy + c), El<T>::one(a.x + (int64_t)r * a.ldx + c) * a.rstd[r], sg);
    a.part[(int64_t)blockIdx.y * a.cols + c] = sg;
}
template <typename T> __global__ __launch_bounds__(kWide) void rms_dx_wide_kernel(const RmsBwd<T> a) {
    __shared__ float red[2][2][1][kWide / 64];
    RowSum<kWide> rs{red};
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* yr = a.dy + (int64_t)r * a.lddy;
        const T* xr = a.x + (int64_t)r * a.ldx;
        const float rstd = a.rstd[r];
        auto at = [&](int c, float& g, float& xh) {
            g = El<T>::one(yr + c);
            if (a.gamma) g *= El<T>::one(a.gamma + c);
            xh = El<T>::one(xr + c) * rstd;
        };
        float c2 = 0.0f, g, xh;
        for (int c = threadIdx.x; c < a.cols; c += kWide) {
            at(c, g, xh);
            c2 = __builtin_fmaf(g, xh, c2);
        }
        c2 = rs.one(c2) / (float)a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kWide) {
            at(c, g, xh);
            float d = rstd * __builtin_fmaf(-xh, c2, g);
            if (a.dres) d += El<T>::one(a.dres + (int64_t)r * a.lddr + c);
            El<T>::put(a.dx + (int64_t)r * a.lddx + c, d);
        }
    }
}

// -------------------------------------------------------------------- plans --
// Threads a row and chunks a thread; threads 0: too wide for registers.
struct RmsShape {
    int threads, chunks;
};
RmsShape fwd_shape(int cols, int esz) {
    const int n = (int)(((int64_t)cols * esz + 15) / 16);  // 16-byte chunks of a row
    if (n <= 64) return {64, 1};
    if (n <= 128) return {64, 2};
    if (n <= 256) return {64, 4};
    if (n <= 512) return {256, 2};
    if (n <= 1024) return {256, 4};
    if (n <= 2048) return {512, 4};
    return {0, 0};
}
RmsShape bwd_shape(int cols, int esz) {
    const int n = (int)(((int64_t)cols * esz + 15) / 16);
    if (n <= 64) return {64, 1};
    if (n <= 128) return {64, 2};
    if (n <= 256) return {128, 2};
    if (n <= 512) return {256, 2};
    if (n <= 1024) return {512, 2};
    if (n <= 2048) return {1024, 2};
    return {0, 0};
}

constexpr int kOnceRows = 1024;  // rows up to which dx and the column sums share a launch
constexpr int kMaxParts = 512;   // partial sums of gamma's gradient
constexpr int kWideParts = 64;

// blocks of the backward kernel: 16 waves per CU walk the rows
int bwd_blocks(int rows, const RmsShape& s) {
    if (s.threads == 0) return std::min(rows, kWideParts);
    const int nt = bwd_threads(s.threads), per = nt / s.threads;
    return std::min((rows + per - 1) / per, std::min(256 * 1024 / nt, std::max(256, rows / (4 * per))));
}

template <typename T, int OUT> void launch_forward(const RmsFwd<T>& a, hipStream_t st) {
    const RmsShape s = fwd_shape(a.cols, (int)sizeof(T));
    // 16 waves per CU walk the rows
    const int grid = s.threads == 64 ? std::min((a.rows + 3) / 4, 1024)
                                     : std::min(a.rows, s.threads == 0 ? 512 : 256 * 1024 / s.threads);
#define DF_RMS(RT, CH)                                                                   \
    if (s.threads == RT && s.chunks == CH) {                                             \
        rms_forward_kernel<T, RT, CH, OUT><<<grid, RT == 64 ? 256 : RT, 0, st>>>(a);     \
        return;                                                                          \
    }
    DF_RMS(64, 1)
    DF_RMS(64, 2)
    DF_RMS(64, 4)
    DF_RMS(256, 2)
    DF_RMS(256, 4)
    DF_RMS(512, 4)
#undef DF_RMS
    rms_forward_wide_kernel<T, OUT><<<grid, kWide, 0, st>>>(a);
}

// `stat`: room for rstd of every row (wide rows without a given one)
template <typename T> void launch_backward(RmsBwd<T> a, float* stat, hipStream_t st) {
    const RmsShape s = bwd_shape(a.cols, (int)sizeof(T));
    const int grid = bwd_blocks(a.rows, s);
    const bool sums = a.dgamma != nullptr;
    auto fold = [&](int parts) {
        const int blocks = (int)(((int64_t)a.cols + kFoldCols - 1) / kFoldCols);
        rms_fold_kernel<<<blocks, 64 * kFoldWaves, 0, st>>>(a.part, parts, a.cols, a.dgamma);
    };
    if (a.rows == 0) {
        if (sums) fold(0);
        return;
    }
    // rows and columns in one launch, unless dx lies over dy or x, which the
    // columns' blocks read: then these go first
    const bool once = sums && a.rstd && grid > 1 && s.threads > 0 && a.rows <= kOnceRows;
    const bool over = a.dx == a.dy || a.dx == a.x;
    if (s.threads == 0) {
        const int rgrid = std::min(a.rows, 512);
        if (!a.rstd) {
            rms_stats_wide_kernel<T><<<rgrid, kWide, 0, st>>>(a.x, a.rows, a.cols, a.ldx, a.eps, stat);
            a.rstd = stat;
        }
        if (sums) {  // before dx, which may lie over dy or x
            rms_colsum_wide_kernel<T><<<dim3((a.cols + 255) / 256, grid), 256, 0, st>>>(a);
            fold(grid);
        }
        rms_dx_wide_kernel<T><<<rgrid, kWide, 0, st>>>(a);
        return;
    }
#define DF_RMS(RT, CH)                                                          \
    if (s.threads == RT && s.chunks == CH) {                                    \
        constexpr int NT = bwd_threads(RT);                                     \
        if (once) {                                                             \
            const int cb = (a.cols + once_cols(RT) - 1) / once_cols(RT);        \
            if (over) {                                                         \
                rms_backward_once_kernel<T, RT, CH><<<cb, NT, 0, st>>>(a, 0);   \
                rms_backward_kernel<T, RT, CH, false><<<grid, NT, 0, st>>>(a);  \
            } else {                                                            \
                rms_backward_once_kernel<T, RT, CH><<<grid + cb, NT, 0, st>>>(a, grid); \
            }                                                                   \
            return;                                                             \
        }                                                                       \
        if (sums) rms_backward_kernel<T, RT, CH, true><<<grid, NT, 0, st>>>(a); \
        else rms_backward_kernel<T, RT, CH, false><<<grid, NT, 0, st>>>(a);     \
    }
    DF_RMS(64, 1)
    DF_RMS(64, 2)
    DF_RMS(128, 2)
    DF_RMS(256, 2)
    DF_RMS(512, 2)
    DF_RMS(1024, 2)
#undef DF_RMS
    if (sums && grid > 1) fold(grid);
}

bool el_dtype(int dtype) {
    return dtype == DF_DTYPE_FLOAT32 || dtype == DF_DTYPE_BFLOAT16 || dtype == DF_DTYPE_HALF;
}

// row and column counters step past the last by at most 2^13
constexpr int kMostRows = 0x7FFF0000;

// An output over an input: the same rows exactly, or a row would be written
// before another wave reads it.
bool same_rows(const void* out, int ldo, const void* in, int ldi, int rows) {
    return !out || out != in || ldo == ldi || rows == 1;
}

bool el_aligned(const void* p, int dtype) { return ((uintptr_t)p & (dtype == DF_DTYPE_FLOAT32 ? 3u : 1u)) == 0; }

// checks of a forward; `empty`: nothing to compute
int check_forward(const char* fn, int dtype, const void* x, int rows, int cols, int ldx, const void* residual, int ldr,
                  const void* sum, int lds, const void* gamma, float eps, const void* y, int ldy, const float* rstd,
                  bool& empty) {
    DF_CHECK(rows >= 0 && cols >= 0 && rows <= kMostRows && cols <= kMostRows, DF_ERR_INVALID,
             "%s: bad shape rows=%d cols=%d", fn, rows, cols);
    DF_CHECK(el_dtype(dtype), DF_ERR_UNSUPPORTED, "%s: dtype %d not supported", fn, dtype);
    DF_CHECK(eps >= 0.0f, DF_ERR_INVALID, "%s: eps < 0", fn);
    DF_CHECK(!sum || residual, DF_ERR_INVALID, "%s: sum without a residual", fn);
    empty = rows == 0 || cols == 0;
    if (empty) return DF_OK;
    DF_CHECK(x, DF_ERR_INVALID, "%s: x is NULL", fn);
    DF_CHECK(!sum || sum != y, DF_ERR_INVALID, "%s: sum and y are the same buffer", fn);
    DF_CHECK(ldx >= cols && (!y || ldy >= cols) && (!residual || ldr >= cols) && (!sum || lds >= cols), DF_ERR_INVALID,
             "%s: a leading dimension is below cols=%d", fn, cols);
    DF_CHECK(same_rows(sum, lds, x, ldx, rows) && same_rows(sum, lds, residual, ldr, rows) &&
                 same_rows(y, ldy, x, ldx, rows) && same_rows(y, ldy, residual, ldr, rows),
             DF_ERR_INVALID, "%s: an output lies over an input with another leading dimension", fn);
    for (const void* p : {x, residual, sum, gamma, y})
        DF_CHECK(el_aligned(p, dtype), DF_ERR_ALIGN, "%s: a pointer is not aligned to its elements", fn);
    DF_CHECK(aligned4(rstd), DF_ERR_ALIGN, "%s: rstd misaligned", fn);
    return DF_OK;
}

template <int OUT, typename Fill> void forward_as(int dtype, const Fill& fill, hipStream_t st) {
    auto go = [&](auto tag) {
        using T = decltype(tag);
        RmsFwd<T> a{};
        fill(a);
        launch_forward<T, OUT>(a, st);
    };
    if (dtype == DF_DTYPE_FLOAT32) go(float{});
    else if (dtype == DF_DTYPE_HALF) go(f16_t{});
    else go(uint16_t{});
}

}  // namespace

}  // namespace dfk

using namespace dfk;

extern "C" int df_rmsnorm_forward(int dtype, const void* x, int rows, int cols, int ldx, const void* residual, int ldr,
                                  void* sum, int lds, const void* gamma, float eps, void* y, int ldy, float* rstd,
                                  void* stream) {
    clear_error();
    const char* fn = "df_rmsnorm_forward";
    bool empty = false;
    if (int rc = check_forward(fn, dtype, x, rows, cols, ldx, residual, ldr, sum, lds, gamma, eps, y, ldy, rstd, empty))
        return rc;
    if (empty) return DF_OK;
    DF_CHECK(y, DF_ERR_INVALID, "%s: y is NULL", fn);
    forward_as<OUT_Y>(dtype, [&](auto& a) {
        using T = typename std::remove_reference<decltype(*a.y)>::type;
        a = {static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<T*>(sum), static_cast<T*>(y),
             static_cast<const T*>(gamma), rstd, nullptr, nullptr, rows, cols, ldx, ldr, lds, ldy, 0, 0, 0, eps};
    }, as_stream(stream));
    return launch_status(fn);
}

extern "C" int df_rmsnorm_quantize(int dtype, const void* x, int rows, int cols, int ldx, const void* residual, int ldr,
                                   void* sum, int lds, const void* gamma, float eps, void* y, int ldy, float* rstd,
                                   int fmt, uint8_t* q, int ldq, int scale_kind, void* scales, int ld_scales,
                                   void* stream) {
    clear_error();
    const char* fn = "df_rmsnorm_quantize";
    bool empty = false;
    DF_CHECK(fmt == DF_FMT_E4M3 || fmt == DF_FMT_E5M2, DF_ERR_INVALID, "%s: bad format %d", fn, fmt);
    DF_CHECK(scale_kind_ok(scale_kind), DF_ERR_INVALID, "%s: bad scale kind %d", fn, scale_kind);
    if (int rc = check_forward(fn, dtype, x, rows, cols, ldx, residual, ldr, sum, lds, gamma, eps, y, ldy, rstd, empty))
        return rc;
    if (empty) return DF_OK;
    DF_CHECK(q && scales, DF_ERR_INVALID, "%s: q or scales is NULL", fn);
    DF_CHECK(ldq % 16 == 0 && ldq >= cols && aligned16(q), DF_ERR_ALIGN,
             "%s: codes need a leading dimension that is a multiple of 16 and >= %d, and 16-byte alignment", fn, cols);
    DF_CHECK(ld_scales >= rows && (int64_t)ld_scales * scale_bytes(scale_kind) % 16 == 0 && aligned16(scales), DF_ERR_ALIGN,
             "%s: scales need a leading dimension of whole 16 bytes and >= %d, and 16-byte alignment", fn, rows);
    auto fill = [&](auto& a) {
        using T = typename std::remove_reference<decltype(*a.y)>::type;
        a = {static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<T*>(sum), static_cast<T*>(y),
             static_cast<const T*>(gamma), rstd, q, scales, rows, cols, ldx, ldr, lds, ldy, ldq, ld_scales, fmt, eps};
    };
    if (scale_kind == DF_SCALE_E8M0) forward_as<OUT_E8>(dtype, fill, as_stream(stream));
    else forward_as<OUT_F32>(dtype, fill, as_stream(stream));
    return launch_status(fn);
}

// the partial sums, then rstd of every row (wide rows), whatever the type
extern "C" size_t df_rmsnorm_backward_workspace_bytes(int rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return (size_t)std::min(rows, kMaxParts) * (size_t)cols * sizeof(float) + (size_t)rows * sizeof(float);
}

extern "C" int df_rmsnorm_backward(int dtype, const void* dy, int lddy, const void* x, int ldx, int rows, int cols,
                                   const void* gamma, const float* rstd, float eps, const void* dresidual, int lddr,
                                   void* dx, int lddx, float* dgamma, void* ws, size_t ws_bytes, void* stream) {
    clear_error();
    const char* fn = "df_rmsnorm_backward";
    DF_CHECK(rows >= 0 && cols >= 0 && rows <= kMostRows && cols <= kMostRows, DF_ERR_INVALID,
             "%s: bad shape rows=%d cols=%d", fn, rows, cols);
    DF_CHECK(el_dtype(dtype), DF_ERR_UNSUPPORTED, "%s: dtype %d not supported", fn, dtype);
    DF_CHECK(eps >= 0.0f, DF_ERR_INVALID, "%s: eps < 0", fn);
    if (cols == 0) return DF_OK;
    DF_CHECK(rows == 0 || (dy && x && dx), DF_ERR_INVALID, "%s: dy, x or dx is NULL", fn);
    DF_CHECK(rows == 0 || (lddy >= cols && ldx >= cols && lddx >= cols && (!dresidual || lddr >= cols)),
             DF_ERR_INVALID, "%s: a leading dimension is below cols=%d", fn, cols);
    DF_CHECK(same_rows(dx, lddx, dy, lddy, rows) && same_rows(dx, lddx, x, ldx, rows) &&
                 same_rows(dx, lddx, dresidual, lddr, rows),
             DF_ERR_INVALID, "%s: dx lies over an input with another leading dimension", fn);
    for (const void* p : {dy, x, gamma, dresidual, (const void*)dx})
        DF_CHECK(el_aligned(p, dtype), DF_ERR_ALIGN, "%s: a pointer is not aligned to its elements", fn);
    DF_CHECK(aligned4(rstd) && aligned4(dgamma), DF_ERR_ALIGN, "%s: rstd or dgamma misaligned", fn);
    const size_t need = df_rmsnorm_backward_workspace_bytes(rows, cols);
    DF_CHECK(need == 0 || (ws && aligned16(ws)), DF_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace", fn);
    DF_CHECK(ws_bytes >= need, DF_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu", fn, ws_bytes, need);
    float* part = static_cast<float*>(ws);
    float* stat = part ? part + (size_t)std::min(rows, kMaxParts) * (size_t)cols : nullptr;
    auto go = [&](auto tag) {
        using T = decltype(tag);
        launch_backward(RmsBwd<T>{static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const T*>(gamma), rstd,
                                  static_cast<const T*>(dresidual), static_cast<T*>(dx), dgamma, part, rows, cols, lddy,
                                  ldx, lddr, lddx, eps},
                        stat, as_stream(stream));
    };
    if (dtype == DF_DTYPE_FLOAT32) go(float{});
    else if (dtype == DF_DTYPE_HALF) go(f16_t{});
    else go(uint16_t{});
    return launch_status(fn);
}
