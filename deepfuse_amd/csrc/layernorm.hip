// layernorm.hip -- LayerNorm for training: the forward that keeps its row
// statistics, with the residual add in front of it, and the backward with the
// reductions of gamma's and beta's gradients (gfx950).
//
// Per row of n values, s = x + residual rounded to the element type:
//   mean = sum(s)/n, var = sum((s - mean)^2)/n, rstd = 1/sqrt(var + eps)
//   y = (s - mean) * rstd * gamma + beta
// and with xh = (s - mean) * rstd, g = dy * gamma, over the row
//   dx = rstd * (g - mean(g) - xh * mean(g * xh)) + dresidual
// and over the rows  dgamma = sum(dy * xh), dbeta = sum(dy).
//
// Both are bound by HBM: the forward reads x (and the residual) and writes y
// (and s), the backward reads dy and s (and the residual path's gradient) and
// writes dx, each once.  So a row stays in registers from its load to its
// store: a wave owns a row of up to 4 16-byte chunks per lane, wider rows take
// a block, and only rows beyond those (16384 two-byte values) are read in
// several passes.  16384 x 1600 bf16 with the residual (210 MB each way): forward
// 43.9 us, 4.8 TB/s, backward 50.6, 4.1 TB/s; a large copy reaches 5.1.  Sums are
// binary32: per lane in order, then a fixed
// butterfly, then waves in order, so results do not depend on timing.
//
// The reference's forward is layer_norm_forward_kernel
// (dnn/layers/layer_norm_layer.cu:26-63); its backward copies the incoming
// gradient (.cu:82-90), so the backward here has no counterpart.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "df_common.hpp"
#include "row_chunks.hpp"

namespace dfk {

namespace {

// mean and rstd of a row whose chunk k is get(k, values); values past the
// row's end, which are 0, take mean 0, so that they add nothing
template <typename T, int RT, int CH, typename Get, typename Sum>
__device__ __forceinline__ void row_stats(const Get& get, int t, int cols, float eps, Sum& rs, float& mean,
                                          float& rstd) {
    constexpr int E = El<T>::E;
    float s = 0.0f, sq = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        float v[E];
        get(k, v);
#pragma unroll
        for (int e = 0; e < E; ++e) s += v[e];
    }
    mean = rs.one(s) / (float)cols;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        const int c = (t + RT * k) * E;
        float v[E];
        get(k, v);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = v[e] - (c + e < cols ? mean : 0.0f);
            sq = __builtin_fmaf(d, d, sq);
        }
    }
    rstd = 1.0f / __builtin_sqrtf(rs.one(sq) / (float)cols + eps);
}

template <typename T> struct FwdArgs {
    const T* x; const T* res; T* sum; T* y;
    const T* gamma; const T* beta;
    float* mean; float* rstd;
    int rows, cols, ldx, ldr, lds, ldy;
    float eps;
};

// ------------------------------------------------------------------ forward --
template <typename T, int RT, int CH>
__global__ __launch_bounds__(RT == 64 ? 256 : RT) void ln_forward_kernel(const FwdArgs<T> a) {
    constexpr int E = El<T>::E;
    constexpr int RPB = RT == 64 ? 4 : 1;  // rows a block works on at once
    __shared__ float red[2][2][1][RT / 64];
    const int t = RT == 64 ? threadIdx.x & 63 : threadIdx.x;
    RowSum<RT> rs{red};
    u32x4 gw[CH], bw[CH], nx[CH], nr[CH];
    const bool affine = a.gamma != nullptr, add = a.res != nullptr;
    auto fetch = [&](int r) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < CH; ++k) nx[k] = load_chunk<T>(a.x + (int64_t)r * a.ldx, t + RT * k, a.cols);
        if (add) {
#pragma unroll
            for (int k = 0; k < CH; ++k) nr[k] = load_chunk<T>(a.res + (int64_t)r * a.ldr, t + RT * k, a.cols);
        }
    };
    const int step = gridDim.x * RPB;
    int r = blockIdx.x * RPB + (RT == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
    if (r < a.rows) fetch(r);
    if (affine) {
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            gw[k] = place_chunk<T>(load_chunk<T>(a.gamma, t + RT * k, a.cols), t + RT * k, a.cols);
            bw[k] = place_chunk<T>(load_chunk<T>(a.beta, t + RT * k, a.cols), t + RT * k, a.cols);
        }
    }
    // a row's last chunk is loaded with values of the chunk before it, which
    // another wave may own, and the sum may lie over x: no wave stores of the
    // first row before all have its loads on their way (later rows' loads come
    // before the barriers of the row before them)
    if constexpr (RT > 64) __syncthreads();
    for (; r < a.rows; r += step) {
        float v[CH][E];
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            El<T>::widen(place_chunk<T>(nx[k], t + RT * k, a.cols), v[k]);
            if (add) {
                float q[E];
                El<T>::widen(place_chunk<T>(nr[k], t + RT * k, a.cols), q);
#pragma unroll
                for (int e = 0; e < E; ++e) v[k][e] += q[e];
                // the statistics are those of the sum as stored
                const u32x4 w = El<T>::narrow(v[k]);
                El<T>::widen(w, v[k]);
                if (a.sum) store_chunk<T>(a.sum + (int64_t)r * a.lds, t + RT * k, a.cols, w);
            }
        }
        if (r + step < a.rows) fetch(r + step);
        float mean, rstd;
        row_stats<T, RT, CH>(
            [&](int k, float* o) {
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = v[k][e];
            },
            t, a.cols, a.eps, rs, mean, rstd);
        if (t == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
#pragma unroll
        for (int k = 0; k < CH; ++k) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[k][e] = (v[k][e] - mean) * rstd;
            if (affine) {
                float g[E], b[E];
                El<T>::widen(gw[k], g);
                El<T>::widen(bw[k], b);
#pragma unroll
                for (int e = 0; e < E; ++e) v[k][e] = __builtin_fmaf(v[k][e], g[e], b[e]);
            }
            store_chunk<T>(a.y + (int64_t)r * a.ldy, t + RT * k, a.cols, El<T>::narrow(v[k]));
        }
    }
}

// Rows wider than a block's registers: a block reads its row three times.
constexpr int kWide = 1024;
template <typename T> __global__ __launch_bounds__(kWide) void ln_forward_wide_kernel(const FwdArgs<T> a) {
    __shared__ float red[2][2][1][kWide / 64];
    RowSum<kWide> rs{red};
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* xr = a.x + (int64_t)r * a.ldx;
        const T* rr = a.res ? a.res + (int64_t)r * a.ldr : nullptr;
        auto at = [&](int c) {
            float v = El<T>::one(xr + c);
            if (rr) {
                T q;
                El<T>::put(&q, v + El<T>::one(rr + c));
                v = El<T>::one(&q);
            }
            return v;
        };
        float s = 0.0f, sq = 0.0f;
        for (int c = threadIdx.x; c < a.cols; c += kWide) s += at(c);
        const float mean = rs.one(s) / (float)a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kWide) {
            const float d = at(c) - mean;
            sq = __builtin_fmaf(d, d, sq);
        }
        const float rstd = 1.0f / __builtin_sqrtf(rs.one(sq) / (float)a.cols + a.eps);
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
        for (int c = threadIdx.x; c < a.cols; c += kWide) {
            const float v = at(c);
            float n = (v - mean) * rstd;
            if (a.gamma) n = __builtin_fmaf(n, El<T>::one(a.gamma + c), El<T>::one(a.beta + c));
            if (rr && a.sum) El<T>::put(a.sum + (int64_t)r * a.lds + c, v);
            El<T>::put(a.y + (int64_t)r * a.ldy + c, n);
        }
    }
}

// ----------------------------------------------------------------- backward --
template <typename T> struct BwdArgs {
    const T* dy; const T* x; const T* gamma; const float* mean; const float* rstd; const T* dres; T* dx;
    float* dgamma; float* dbeta;  // written by the kernel itself when one block runs
    float* part;                  // [blocks][2][cols]: each block's sums of dy * xh and dy
    int rows, cols, lddy, ldx, lddr, lddx;
    float eps;
};

// A block of NT threads works on NT / RT rows at once (512 threads, or 1024
// for the widest rows: two blocks or one per CU).  A thread keeps the same
// columns for all its rows, so gamma's and beta's sums stay in its registers;
// at the end the row groups' sums meet in LDS and leave as one partial per
// block (2 * cols values), which ln_fold_kernel adds in block order.
// Two chunks a thread and no row ahead: the sums leave no registers for more.
// Four chunks (a wave to a row of 1600 bf16 values) spilled 28 a lane, 98.5 us
// against 48.5 at 16384 rows; the next row's loads, of which the 16 waves of a
// CU hide as much, fewer: 1600 columns 54 against 51, 12800 467 against 333.
// SUMS: gamma's and beta's gradients are wanted.
constexpr int bwd_threads(int rt) { return rt > 512 ? rt : 512; }
template <typename T, int RT, int CH, bool SUMS>
__device__ __forceinline__ void backward_rows(const BwdArgs<T>& a, int blocks) {
    constexpr int E = El<T>::E;
    constexpr int GP = bwd_threads(RT) / RT;
    __shared__ float red[2][2][GP][RT / 64];
    const int t = threadIdx.x % RT, group = __builtin_amdgcn_readfirstlane(threadIdx.x / RT);
    RowSum<RT, GP> rs{red};
    // gamma, each thread's own chunks: in LDS, where reading them waits for no
    // load under way, and takes no registers from row to row
    __shared__ u32x4 gw[CH][bwd_threads(RT)];
    const bool affine = a.gamma != nullptr, add = a.dres != nullptr, given = a.mean != nullptr;
    // The chunk in which the rows end holds this many values of the chunk before
    // it (a chunk behind it: all).  They stay where they were loaded, gamma's
    // likewise (moving them cost registers that were spilled: 16384 x 1600 70 us
    // against 51), count for neither sum and are not stored.
    auto borrowed = [&](int k) { return a.cols < E ? 0 : max(0, (t + RT * k) * E + E - a.cols); };
    float sg[CH][E], sb[CH][E];
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) sg[k][e] = sb[k][e] = 0.0f;
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
        float mean = 0.0f, rstd = 0.0f;
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
            if (given) {
                mean = a.mean[r];
                rstd = a.rstd[r];
            }
        }
        if (!given)
            row_stats<T, RT, CH>([&](int k, float* o) { El<T>::widen(place_chunk<T>(cx[k], t + RT * k, a.cols), o); },
                                 t, a.cols, a.eps, rs, mean, rstd);
        if (GP > 1 && !live) mean = rstd = 0.0f;
        // xh and g = dy * gamma of chunk k.  Past the row's end dy is 0, so
        // what xh holds there adds nothing as long as it is finite: mean and
        // rstd of a row with an infinity or a NaN are not, and neither are
        // that row's sums.
        auto terms = [&](int k, float* xh, float* d, float* g) __attribute__((always_inline)) {
            El<T>::widen(cx[k], xh);
            El<T>::widen(cy[k], d);
            float w[E];
            if (affine) El<T>::widen(gw[k][threadIdx.x], w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[e] = (xh[e] - mean) * rstd;
                g[e] = affine ? d[e] * w[e] : d[e];
            }
        };
        float c1 = 0.0f, c2 = 0.0f;
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
                if (SUMS) {
                    sg[k][e] = __builtin_fmaf(d[e], xh[e], sg[k][e]);
                    sb[k][e] += d[e];
                }
                c1 += g[e];
                c2 = __builtin_fmaf(g[e], xh[e], c2);
            }
        }
        rs.two(c1, c2);
        c1 *= inv;
        c2 *= inv;
        if (!live) continue;
        // the terms again from the row as loaded, not kept: registers
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            __builtin_amdgcn_sched_barrier(0);
            float xh[E], d[E], g[E], q[E];
            terms(k, xh, d, g);
            if (add) El<T>::widen(cr[k], q);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                g[e] = rstd * (g[e] - __builtin_fmaf(xh[e], c2, c1));
                if (add) g[e] += q[e];
            }
            store_chunk<T>(a.dx + (int64_t)r * a.lddx, t + RT * k, a.cols,
                           place_chunk<T>(El<T>::narrow(g), t + RT * k, a.cols));
        }
    }
    if constexpr (SUMS) {
        float* og = a.part + (int64_t)blockIdx.x * 2 * a.cols;
        float* ob = og + a.cols;
        if (blocks == 1) {
            og = a.dgamma;
            ob = a.dbeta;
        }
        if constexpr (GP > 1) {
            // the groups' sums in LDS, halves onto halves; a thread's values
            // lie RT apart: no bank conflicts
            __shared__ float slab[GP / 2][2][CH * E * RT];
#pragma unroll
            for (int half = GP / 2; half > 0; half >>= 1) {
                if (group >= half && group < 2 * half) {
#pragma unroll
                    for (int k = 0; k < CH; ++k)
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            slab[group - half][0][(k * E + e) * RT + t] = sg[k][e];
                            slab[group - half][1][(k * E + e) * RT + t] = sb[k][e];
                        }
                }
                __syncthreads();
                if (group < half) {
#pragma unroll
                    for (int k = 0; k < CH; ++k)
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            sg[k][e] += slab[group][0][(k * E + e) * RT + t];
                            sb[k][e] += slab[group][1][(k * E + e) * RT + t];
                        }
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
                if (e >= borrowed(k) && c < a.cols) {
                    og[c] = sg[k][e];
                    ob[c] = sb[k][e];
                }
            }
    }
}

template <typename T, int RT, int CH, bool SUMS>
__global__ __launch_bounds__(bwd_threads(RT), 4) void ln_backward_kernel(const BwdArgs<T> a) {
    backward_rows<T, RT, CH, SUMS>(a, gridDim.x);
}

// Few rows, their statistics given: dx and the column sums in one launch.  The
// blocks behind the first `row_blocks` take a few columns each and read dy and
// x again (from the L2 the rows' blocks fill), a wave two or four rows at a
// time, so the sums need neither partials nor a second launch.  Eight rows'
// loads at a time, the last eight too: one by one, they took as long as the rest
// (1000 x 771 bf16 8.2 us, 6.7 so).  16 columns a block for narrow rows, which
// leave CUs idle (1024 x 768 7.2 us with 32, 6.7 with 16), 32 for wide ones
// (1024 x 6400 17.4 and 23.7).
constexpr int kOnceLoads = 8;
constexpr int once_cols(int rt) { return rt <= 128 ? 16 : 32; }
template <typename T, int RT, int CH>
__global__ __launch_bounds__(bwd_threads(RT), 4) void ln_backward_once_kernel(const BwdArgs<T> a, int row_blocks) {
    if ((int)blockIdx.x < row_blocks) {
        backward_rows<T, RT, CH, false>(a, row_blocks);
        return;
    }
    constexpr int W = bwd_threads(RT) / 64, CW = once_cols(RT);
    __shared__ float red[W][2][CW];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, i = lane % CW;
    const int c = ((int)blockIdx.x - row_blocks) * CW + i;
    float sg = 0.0f, sb = 0.0f;
    if (c < a.cols) {
        constexpr int STEP = 64 / CW * W;
        // kOnceLoads rows from r0; LAST: only those that there are
        auto rows = [&](int r0, auto last) __attribute__((always_inline)) {
            constexpr bool LAST = decltype(last)::value;
            float d[kOnceLoads], x[kOnceLoads], m[kOnceLoads], q[kOnceLoads];
#pragma unroll
            for (int k = 0; k < kOnceLoads; ++k) {
                const int r = LAST ? min(r0 + k * STEP, a.rows - 1) : r0 + k * STEP;
                d[k] = El<T>::one(a.dy + (int64_t)r * a.lddy + c);
                x[k] = El<T>::one(a.x + (int64_t)r * a.ldx + c);
                m[k] = a.mean[r];
                q[k] = a.rstd[r];
            }
#pragma unroll
            for (int k = 0; k < kOnceLoads; ++k) {
                if (!LAST || r0 + k * STEP < a.rows) {
                    sg = __builtin_fmaf(d[k], (x[k] - m[k]) * q[k], sg);
                    sb += d[k];
                }
            }
        };
        int r = threadIdx.x / CW;
        for (; r + (kOnceLoads - 1) * STEP < a.rows; r += kOnceLoads * STEP) rows(r, std::false_type{});
        if (r < a.rows) rows(r, std::true_type{});
    }
#pragma unroll
    for (int off = CW; off < 64; off <<= 1) {
        sg += __shfl_xor(sg, off, 64);
        sb += __shfl_xor(sb, off, 64);
    }
    if (lane < CW) {
        red[w][0][i] = sg;
        red[w][1][i] = sb;
    }
    __syncthreads();
    if (w == 0 && lane < CW && c < a.cols) {
#pragma unroll
        for (int v = 1; v < W; ++v) {
            sg += red[v][0][i];
            sb += red[v][1][i];
        }
        a.dgamma[c] = sg;
        a.dbeta[c] = sb;
    }
}

// dgamma and dbeta from `parts` partials of 2 * cols values: a block takes
// 32 of the 2 * cols columns, its half waves every 16th partial each, in order
// (16384 x 256 bf16 17.2 us with 64 columns, 15.6 with 32, 16.0 with 8).
constexpr int kFoldWaves = 8, kFoldCols = 32, kFoldParts = kFoldWaves * (64 / kFoldCols);
__global__ __launch_bounds__(64 * kFoldWaves) void ln_fold_kernel(const float* __restrict__ part, int parts, int cols,
                                                                  float* __restrict__ dgamma,
                                                                  float* __restrict__ dbeta) {
    __shared__ float red[kFoldParts][kFoldCols];
    const int i = threadIdx.x % kFoldCols, mine = threadIdx.x / kFoldCols;
    const int64_t width = 2 * (int64_t)cols, c = (int64_t)blockIdx.x * kFoldCols + i;
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
        if (c < cols) dgamma[c] = s;
        else dbeta[c - cols] = s;
    }
}

// Rows wider than a block's registers: the row statistics where they are not
// given, the column sums (a thread per column, blockIdx.y's share of the
// rows), then dx, each from memory.
template <typename T>
__global__ __launch_bounds__(kWide) void ln_stats_wide_kernel(const T* x, int rows, int cols, int ldx, float eps,
                                                              float* mean, float* rstd) {
    __shared__ float red[2][2][1][kWide / 64];
    RowSum<kWide> rs{red};
    for (int r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + (int64_t)r * ldx;
        float s = 0.0f, sq = 0.0f;
        for (int c = threadIdx.x; c < cols; c += kWide) s += El<T>::one(xr + c);
        const float m = rs.one(s) / (float)cols;
        for (int c = threadIdx.x; c < cols; c += kWide) {
            const float d = El<T>::one(xr + c) - m;
            sq = __builtin_fmaf(d, d, sq);
        }
        const float q = 1.0f / __builtin_sqrtf(rs.one(sq) / (float)cols + eps);
        if (threadIdx.x == 0) {
            mean[r] = m;
            rstd[r] = q;
        }
    }
}

template <typename T> __global__ __launch_bounds__(256) void ln_colsum_wide_kernel(const BwdArgs<T> a) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.cols) return;
    float sg = 0.0f, sb = 0.0f;
    for (int r = blockIdx.y; r < a.rows; r += gridDim.y) {
        const float d = El<T>::one(a.dy + (int64_t)r * a.lddy + c);
        const float xh = (El<T>::one(a.x + (int64_t)r * a.ldx + c) - a.mean[r]) * a.rstd[r];
        sg = __builtin_fmaf(d, xh, sg);
        sb += d;
    }
    float* o = a.part + (int64_t)blockIdx.y * 2 * a.cols + c;
    o[0] = sg;
    o[a.cols] = sb;
}

template <typename T> __global__ __launch_bounds__(kWide) void ln_dx_wide_kernel(const BwdArgs<T> a) {
    __shared__ float red[2][2][1][kWide / 64];
    RowSum<kWide> rs{red};
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* yr = a.dy + (int64_t)r * a.lddy;
        const T* xr = a.x + (int64_t)r * a.ldx;
        const float mean = a.mean[r], rstd = a.rstd[r];
        auto at = [&](int c, float& g, float& xh) {
            g = El<T>::one(yr + c);
            if (a.gamma) g *= El<T>::one(a.gamma + c);
            xh = (El<T>::one(xr + c) - mean) * rstd;
        };
        float c1 = 0.0f, c2 = 0.0f, g, xh;
        for (int c = threadIdx.x; c < a.cols; c += kWide) {
            at(c, g, xh);
            c1 += g;
            c2 = __builtin_fmaf(g, xh, c2);
        }
        rs.two(c1, c2);
        c1 /= (float)a.cols;
        c2 /= (float)a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kWide) {
            at(c, g, xh);
            float d = rstd * (g - __builtin_fmaf(xh, c2, c1));
            if (a.dres) d += El<T>::one(a.dres + (int64_t)r * a.lddr + c);
            El<T>::put(a.dx + (int64_t)r * a.lddx + c, d);
        }
    }
}

// -------------------------------------------------------------------- plans --
// Threads a row and chunks a thread; threads 0: too wide for registers.  The
// forward keeps a row in a wave while its registers hold it; the backward, with
// its sums, keeps two chunks a thread.
struct LnShape {
    int threads, chunks;
};
LnShape fwd_shape(int cols, int esz) {
    const int n = (int)(((int64_t)cols * esz + 15) / 16);  // 16-byte chunks of a row
    if (n <= 64) return {64, 1};
    if (n <= 128) return {64, 2};
    if (n <= 256) return {64, 4};
    if (n <= 512) return {256, 2};
    if (n <= 1024) return {256, 4};
    if (n <= 2048) return {512, 4};
    return {0, 0};
}
LnShape bwd_shape(int cols, int esz) {
    const int n = (int)(((int64_t)cols * esz + 15) / 16);
    if (n <= 64) return {64, 1};
    if (n <= 128) return {64, 2};
    if (n <= 256) return {128, 2};
    if (n <= 512) return {256, 2};
    if (n <= 1024) return {512, 2};
    if (n <= 2048) return {1024, 2};
    return {0, 0};
}

// Rows up to which dx and the column sums share a launch (us, two launches
// against one, bf16): 64 x 768 8.7 / 4.3, 512 x 768 10.3 / 4.9, 1024 x 768 10.0 /
// 6.7, 2048 x 768 11.5 / 13.2; 1024 x 6400 29.2 / 17.4, 4096 x 6400 61 / 82;
// 1024 x 12800 47.4 / 42.6, 2048 x 12800 66 / 82.
constexpr int kOnceRows = 1024;
constexpr int kMaxParts = 512;  // partial sums of gamma's and beta's gradients
constexpr int kWideParts = 64;

// blocks of the backward kernel: 16 waves per CU walk the rows
int bwd_blocks(int rows, const LnShape& s) {
    if (s.threads == 0) return std::min(rows, kWideParts);
    // (four times round at least before there are more than 256: each leaves
    // 2 * cols partial sums.  2048 x 1600 bf16: 16.7 us with 256 blocks, 19.4
    // with 512; 8192 x 1600: 35.7 and 33.6)
    const int nt = bwd_threads(s.threads), per = nt / s.threads;
    return std::min((rows + per - 1) / per, std::min(256 * 1024 / nt, std::max(256, rows / (4 * per))));
}

template <typename T> void launch_forward(const FwdArgs<T>& a, hipStream_t st) {
    const LnShape s = fwd_shape(a.cols, (int)sizeof(T));
    // 16 waves per CU walk the rows
    const int grid = s.threads == 64 ? std::min((a.rows + 3) / 4, 1024)
                                     : std::min(a.rows, s.threads == 0 ? 512 : 256 * 1024 / s.threads);
#define DF_LN(RT, CH)                                                 \
    if (s.threads == RT && s.chunks == CH) {                          \
        ln_forward_kernel<T, RT, CH><<<grid, RT == 64 ? 256 : RT, 0, st>>>(a); \
        return;                                                       \
    }
    DF_LN(64, 1)
    DF_LN(64, 2)
    DF_LN(64, 4)
    DF_LN(256, 2)
    DF_LN(256, 4)
    DF_LN(512, 4)
#undef DF_LN
    ln_forward_wide_kernel<T><<<grid, kWide, 0, st>>>(a);
}

// `stat`: room for mean and rstd of every row (wide rows without given ones)
template <typename T> void launch_backward(BwdArgs<T> a, float* stat, hipStream_t st) {
    const LnShape s = bwd_shape(a.cols, (int)sizeof(T));
    const int grid = bwd_blocks(a.rows, s);
    const bool sums = a.dgamma != nullptr;
    auto fold = [&](int parts) {
        const int blocks = (int)((2 * (int64_t)a.cols + kFoldCols - 1) / kFoldCols);
        ln_fold_kernel<<<blocks, 64 * kFoldWaves, 0, st>>>(a.part, parts, a.cols, a.dgamma, a.dbeta);
    };
    if (a.rows == 0) {
        if (sums) fold(0);
        return;
    }
    // rows and columns in one launch, unless dx lies over dy or x, which the
    // columns' blocks read: then these go first
    const bool once = sums && a.mean && grid > 1 && s.threads > 0 && a.rows <= kOnceRows;
    const bool over = a.dx == a.dy || a.dx == a.x;
    if (s.threads == 0) {
        const int rgrid = std::min(a.rows, 512);
        if (!a.mean) {
            ln_stats_wide_kernel<T><<<rgrid, kWide, 0, st>>>(a.x, a.rows, a.cols, a.ldx, a.eps, stat, stat + a.rows);
            a.mean = stat;
            a.rstd = stat + a.rows;
        }
        if (sums) {  // before dx, which may lie over dy or x
            ln_colsum_wide_kernel<T><<<dim3((a.cols + 255) / 256, grid), 256, 0, st>>>(a);
            fold(grid);
        }
        ln_dx_wide_kernel<T><<<rgrid, kWide, 0, st>>>(a);
        return;
    }
#define DF_LN(RT, CH)                                                          \
    if (s.threads == RT && s.chunks == CH) {                                   \
        constexpr int NT = bwd_threads(RT);                                    \
        if (once) {                                                            \
            const int cb = (a.cols + once_cols(RT) - 1) / once_cols(RT);       \
            if (over) {                                                        \
                ln_backward_once_kernel<T, RT, CH><<<cb, NT, 0, st>>>(a, 0);   \
                ln_backward_kernel<T, RT, CH, false><<<grid, NT, 0, st>>>(a);  \
            } else {                                                           \
                ln_backward_once_kernel<T, RT, CH><<<grid + cb, NT, 0, st>>>(a, grid); \
            }                                                                  \
            return;                                                            \
        }                                                                      \
        if (sums) ln_backward_kernel<T, RT, CH, true><<<grid, NT, 0, st>>>(a); \
        else ln_backward_kernel<T, RT, CH, false><<<grid, NT, 0, st>>>(a);     \
    }
    DF_LN(64, 1)
    DF_LN(64, 2)
    DF_LN(128, 2)
    DF_LN(256, 2)
    DF_LN(512, 2)
    DF_LN(1024, 2)
#undef DF_LN
    if (sums && grid > 1) fold(grid);
}

bool ln_dtype(int dtype) {
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

}  // namespace

}  // namespace dfk

using namespace dfk;

extern "C" int df_layernorm_forward(int dtype, const void* x, int rows, int cols, int ldx, const void* residual,
                                    int ldr, void* sum, int lds, const void* gamma, const void* beta, float eps,
                                    void* y, int ldy, float* mean, float* rstd, void* stream) {
    clear_error();
    const char* fn = "df_layernorm_forward";
    DF_CHECK(rows >= 0 && cols >= 0 && rows <= kMostRows && cols <= kMostRows, DF_ERR_INVALID,
             "%s: bad shape rows=%d cols=%d", fn, rows, cols);
    DF_CHECK(ln_dtype(dtype), DF_ERR_UNSUPPORTED, "%s: dtype %d not supported", fn, dtype);
    DF_CHECK((gamma == nullptr) == (beta == nullptr), DF_ERR_INVALID, "%s: gamma and beta go together", fn);
    DF_CHECK(eps >= 0.0f, DF_ERR_INVALID, "%s: eps < 0", fn);
    DF_CHECK(!sum || residual, DF_ERR_INVALID, "%s: sum without a residual", fn);
    if (rows == 0 || cols == 0) return DF_OK;
    DF_CHECK(x && y, DF_ERR_INVALID, "%s: x or y is NULL", fn);
    DF_CHECK(!sum || sum != y, DF_ERR_INVALID, "%s: sum and y are the same buffer", fn);
    DF_CHECK(ldx >= cols && ldy >= cols && (!residual || ldr >= cols) && (!sum || lds >= cols), DF_ERR_INVALID,
             "%s: a leading dimension is below cols=%d", fn, cols);
    DF_CHECK(same_rows(sum, lds, x, ldx, rows) && same_rows(sum, lds, residual, ldr, rows) &&
                 same_rows(y, ldy, x, ldx, rows) && same_rows(y, ldy, residual, ldr, rows),
             DF_ERR_INVALID, "%s: an output lies over an input with another leading dimension", fn);
    for (const void* p : {x, residual, (const void*)sum, gamma, beta, (const void*)y})
        DF_CHECK(el_aligned(p, dtype), DF_ERR_ALIGN, "%s: a pointer is not aligned to its elements", fn);
    DF_CHECK(aligned4(mean) && aligned4(rstd), DF_ERR_ALIGN, "%s: mean or rstd misaligned", fn);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        launch_forward(FwdArgs<T>{static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<T*>(sum),
                                  static_cast<T*>(y), static_cast<const T*>(gamma), static_cast<const T*>(beta), mean,
                                  rstd, rows, cols, ldx, ldr, lds, ldy, eps},
                       as_stream(stream));
    };
    if (dtype == DF_DTYPE_FLOAT32) go(float{});
    else if (dtype == DF_DTYPE_HALF) go(f16_t{});
    else go(uint16_t{});
    return launch_status(fn);
}

// the partial sums, then a row's statistics (wide rows), whatever the type
extern "C" size_t df_layernorm_backward_workspace_bytes(int rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return (size_t)std::min(rows, kMaxParts) * 2 * (size_t)cols * sizeof(float) + 2 * (size_t)rows * sizeof(float);
}

extern "C" int df_layernorm_backward(int dtype, const void* dy, int lddy, const void* x, int ldx, int rows, int cols,
                                     const void* gamma, const float* mean, const float* rstd, float eps,
                                     const void* dresidual, int lddr, void* dx, int lddx, float* dgamma, float* dbeta,
                                     void* ws, size_t ws_bytes, void* stream) {
    clear_error();
    const char* fn = "df_layernorm_backward";
    DF_CHECK(rows >= 0 && cols >= 0 && rows <= kMostRows && cols <= kMostRows, DF_ERR_INVALID,
             "%s: bad shape rows=%d cols=%d", fn, rows, cols);
    DF_CHECK(ln_dtype(dtype), DF_ERR_UNSUPPORTED, "%s: dtype %d not supported", fn, dtype);
    DF_CHECK((mean == nullptr) == (rstd == nullptr), DF_ERR_INVALID, "%s: mean and rstd go together", fn);
    DF_CHECK((dgamma == nullptr) == (dbeta == nullptr), DF_ERR_INVALID, "%s: dgamma and dbeta go together", fn);
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
    DF_CHECK(aligned4(mean) && aligned4(rstd) && aligned4(dgamma) && aligned4(dbeta), DF_ERR_ALIGN,
             "%s: mean, rstd, dgamma or dbeta misaligned", fn);
    const size_t need = df_layernorm_backward_workspace_bytes(rows, cols);
    DF_CHECK(need == 0 || (ws && aligned16(ws)), DF_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace", fn);
    DF_CHECK(ws_bytes >= need, DF_ERR_WORKSPACE, "%s: workspace %zu bytes < %zu", fn, ws_bytes, need);
    float* part = static_cast<float*>(ws);
    float* stat = part ? part + (size_t)std::min(rows, kMaxParts) * 2 * (size_t)cols : nullptr;
    auto go = [&](auto tag) {
        using T = decltype(tag);
        launch_backward(BwdArgs<T>{static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const T*>(gamma),
                                   mean, rstd, static_cast<const T*>(dresidual), static_cast<T*>(dx), dgamma, dbeta,
                                   part, rows, cols, lddy, ldx, lddr, lddx, eps},
                        stat, as_stream(stream));
    };
    if (dtype == DF_DTYPE_FLOAT32) go(float{});
    else if (dtype == DF_DTYPE_HALF) go(f16_t{});
    else go(uint16_t{});
    return launch_status(fn);
}
