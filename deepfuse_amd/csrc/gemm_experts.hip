// gemm_experts.hip -- the fp8 products of a Linear whose rows are dealt to
// experts (a mixture of experts): rows sorted by expert, expert e owning rows
// off[e] .. off[e+1) of the tokens, with weights of its own:
//   forward  Y[i]  = X[i]  . W[e]^T * sx  * sw[e]      (e4m3 x e4m3)
//   dX       dX[i] = dY[i] . W[e]   * sdy * sw[e]      (e5m2 x e4m3)
//   dW       dW[e] = sum over e's rows of dY^T . X * sdy * sx   (e5m2 x e4m3)
// The offsets are read on the device, so nothing waits for the host to learn
// how the rows were dealt.  ROWS calls (forward, dX) cut the rows of each
// expert into tiles; SUMS calls (dW) reduce over the tokens, whose range for
// an expert starts and ends at any byte of the transposed operands' rows: the
// bytes of the neighbouring experts in the first and last 16-byte chunk are
// cleared on both operands (a neighbour's NaN would outlive a zero on one).
//
// Two ways to multiply.  The fp8 matrix instructions add their products in
// groups of eight along K and drop what lies 13 bits below the largest of a
// group (measured: 2^16 + 2^3 keeps both, 2^16 + 2^2 loses the second; across
// groups and into the accumulator 23 bits are kept).  That is up to 7 * 2^-13
// of a group's largest product, in random data about 1e-5 of a result: below a
// 2-byte output's rounding, but not below an fp32 output's.  So calls with a
// 2-byte output use them, and calls with an fp32 output widen the codes to
// bf16 (exact, v_cvt_scalef32_pk_bf16_*) in registers, whose products the bf16
// instructions add with all 23 bits, at half the matrix rate.
//
// Offsets are clamped into [0, rows] and to be non-decreasing per expert, so a
// wrong one gives wrong values but no access outside the operands.
//
// The reference has no mixture of experts; per expert this is
// fully_connected_forward_kernel, fc_backward_input and fc_backward_weights
// (dnn/layers/fully_connected_layer.cu:14-89).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "df_common.hpp"
#include "gemm_common.hpp"
#include "gemm_experts.hpp"

namespace dfk {

namespace {

// ------------------------------------------------------------ small tiles --
// Row tile v of all experts' tiles of ROWS rows, counted through: its expert,
// that one's rows [lo, hi) and the tile's first; false behind the last.  The
// same for every lane of the wave (a lane counts an expert's tiles).  v is below
// most_tiles(): up to the first lane past it the counts are right even where
// later ones of overlapping offsets pass 32 bits.
template <int ROWS>
__device__ __forceinline__ bool row_tile(const ExpertArgs& g, int v, int lane, int& e, int& lo, int& hi, int& m0) {
    for (int base = 0; base < g.experts; base += 64) {
        int a = 0, b = 0;
        if (base + lane < g.experts) expert_rows(g.off, base + lane, g.rows, a, b);
        const int mine = (b - a + ROWS - 1) / ROWS;
        int upto = mine;  // summed up over the lanes: within rows of 16, then across them
#define DF_SCAN(CTRL, ROWS_IN) upto += __builtin_amdgcn_update_dpp(0, upto, CTRL, ROWS_IN, 0xF, false)
        DF_SCAN(0x111, 0xF);  // row_shr:1
        DF_SCAN(0x112, 0xF);
        DF_SCAN(0x114, 0xF);
        DF_SCAN(0x118, 0xF);  // row_shr:8
        DF_SCAN(0x142, 0xA);  // row_bcast:15 into the second and fourth row
        DF_SCAN(0x143, 0xC);  // row_bcast:31 into the upper half
#undef DF_SCAN
        const uint64_t past = __builtin_amdgcn_ballot_w64(upto > v);
        if (past) {
            const int l = __builtin_ctzll(past);
            e = base + l;
            lo = __builtin_amdgcn_readlane(a, l);
            hi = __builtin_amdgcn_readlane(b, l);
            m0 = lo + (v - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(mine, l))) * ROWS;
            return true;
        }
        v -= __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// As gemm_small.hip's kernel: a block owns a 16*MT x 16*NT tile, its W waves
// take the 128-byte K steps in turn and add up through LDS, in wave order.
// ROWS: blockIdx.x is the column tile.  Tiles of 16 rows, for experts of a few
// rows: blockIdx.y is the expert.  Tiles of 32: all experts' row tiles, counted
// through, are the block's from blockIdx.y in steps of gridDim.y, so that an
// expert that got most rows keeps no block longer than others (936 rows over 45
// experts, 300 of them one's, 1408 -> 448: 30.5 us with blocks bound to experts,
// 14.8 so; even shares mostly take 0.3 us more, and up to 15% where blocks side
// by side read the same weights from memory.  Counted in order of the tiles'
// place in their expert, or with a column's tiles on one XCD: slower elsewhere).
// SUMS: blockIdx.x is the tile, blockIdx.y the expert.
// WIDE: codes are multiplied as bf16, eight of a lane's 32 at a time: which K
// an instruction takes together is free as long as A and B agree.
template <int FA, int FB, int MT, int NT, int W, int U, bool SUMS, bool WIDE>
__global__ __launch_bounds__(64 * W) void experts_small_kernel(const ExpertArgs g, int c_dtype) {
    constexpr int ROWS = 16 * MT, COLS = 16 * NT;
    constexpr int NL = 2 * (MT + NT);  // loads of 8 rows x 128 bytes per step
    constexpr int SLAB = NL * 1024;    // a wave's step: A rows, then B rows
    constexpr int RSTR = COLS + 4;     // row of a partial tile (floats)
    constexpr int RED = ROWS * RSTR * 4;
    constexpr uint32_t kOOB = 0x80000000u;
    constexpr bool COUNTED = !SUMS && MT > 1;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[W * (SLAB > RED ? SLAB : RED)];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_n = (g.N + COLS - 1) / COLS;
    const int n0 = (SUMS ? (int)(blockIdx.x % tiles_n) : (int)blockIdx.x) * COLS;

    // loads: lane l takes 16-byte chunk l%8 of row l/8 of each 8-row group
    const int lr = lane >> 3, lc = (lane & 7) * 16;
    const uint32_t oa = (uint32_t)lr * (uint32_t)g.lda + (uint32_t)lc;
    const uint32_t ob = (uint32_t)lr * (uint32_t)g.ldb + (uint32_t)lc;
    // slab: rows of 128 bytes, 16-byte chunk c of row r in slot c ^ (r/2 % 8)
    uint8_t* const slab = lds + w * SLAB;
    const int wr_even = lr * 128 + (((lane & 7) ^ (lr >> 1)) << 4);
    const int wr_odd = wr_even ^ 64;
    const int fr = lane & 15, fq = (lane >> 4) * 2, fs = (fr >> 1) & 7;
    const int rd0 = fr * 128 + ((fq ^ fs) << 4), rd1 = fr * 128 + (((fq + 1) ^ fs) << 4);
    // the lanes of a wave hand chunks to each other through the slab: LDS
    // operations of a wave execute in order, the compiler must keep that order
    auto lanes_meet = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
    };

    const int most = COUNTED ? most_tiles(g.rows, g.experts, ROWS) : 0;
    for (int v = COUNTED ? (int)blockIdx.y : 0;; v += COUNTED ? (int)gridDim.y : 1) {
        int e, lo, hi, m0;
        if constexpr (COUNTED) {
            if (v >= most || !row_tile<ROWS>(g, v, lane, e, lo, hi, m0)) return;  // the whole block
        } else {
            e = blockIdx.y;
            expert_rows(g.off, e, g.rows, lo, hi);
            m0 = SUMS ? (int)(blockIdx.x / tiles_n) * ROWS : lo + v * ROWS;
            if (!SUMS && m0 >= hi) return;
        }
        // the reduction's bytes [k_lo, k_hi) of the operands' rows, in steps of 128 from kb
        const int kb = SUMS ? lo & ~127 : 0, k_lo = SUMS ? lo : 0, k_hi = SUMS ? hi : g.K;
        const int nk = (k_hi - kb + 127) >> 7;
        const uint8_t* const Be = g.B + (SUMS ? 0 : (int64_t)e * g.N * g.ldb) + (int64_t)n0 * g.ldb;
        const __amdgpu_buffer_rsrc_t rB = __builtin_amdgcn_make_buffer_rsrc(
            (void*)Be, (short)0, min(g.N - n0, COLS) * g.ldb, 0x00020000);
        const float sab = g.sa[0] * g.sb[SUMS ? 0 : e];
        const int mrows = min((SUMS ? g.M : hi) - m0, ROWS);
        const __amdgpu_buffer_rsrc_t rA = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(g.A + (int64_t)m0 * g.lda), (short)0, mrows * g.lda, 0x00020000);
        u32x4 buf[U][NL];
        auto load = [&](u32x4* b, int s) {
            const int k = kb + s * 128;  // past the last step: every chunk out of range
            const bool in = k + lc < k_hi && (!SUMS || k + lc + 16 > k_lo);
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i)
                b[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                    rA, in ? oa + (uint32_t)(8 * i) * (uint32_t)g.lda + (uint32_t)k : kOOB, 0, 0));
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i)
                b[2 * MT + i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                    rB, in ? ob + (uint32_t)(8 * i) * (uint32_t)g.ldb + (uint32_t)k : kOOB, 0, 0));
        };
        v4f acc[MT][NT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        // fragment t (16 rows) of a step in registers, through its part of the slab
        auto frag = [&](const u32x4* b, int t) -> v8i {
            *reinterpret_cast<u32x4*>(slab + t * 2048 + wr_even) = b[2 * t];
            *reinterpret_cast<u32x4*>(slab + t * 2048 + 1024 + wr_odd) = b[2 * t + 1];
            lanes_meet();
            const u32x4 x = *reinterpret_cast<const u32x4*>(slab + t * 2048 + rd0);
            const u32x4 y = *reinterpret_cast<const u32x4*>(slab + t * 2048 + rd1);
            v8i f;
            f[0] = (int)x.x; f[1] = (int)x.y; f[2] = (int)x.z; f[3] = (int)x.w;
            f[4] = (int)y.x; f[5] = (int)y.y; f[6] = (int)y.z; f[7] = (int)y.w;
            return f;
        };
        auto step = [&](u32x4* b, int s) {
            if (SUMS && (s == 0 || s == nk - 1)) {  // the neighbours' bytes of the edge chunks
                const int k = kb + s * 128 + lc;
                u32x4 keep;
#pragma unroll
                for (int d = 0; d < 4; ++d) keep[d] = keep_bytes(k + 4 * d, k_lo, k_hi);
#pragma unroll
                for (int i = 0; i < NL; ++i) b[i] &= keep;
            }
            lanes_meet();  // the step before has read the slab
            v8i fb[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) fb[j] = frag(b, MT + j);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const v8i fa = frag(b, i);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if constexpr (WIDE) {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                widen8<FB>((uint32_t)fb[j][2 * q], (uint32_t)fb[j][2 * q + 1]),
                                widen8<FA>((uint32_t)fa[2 * q], (uint32_t)fa[2 * q + 1]), acc[i][j], 0, 0, 0);
                    } else {
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], FB, FA, 0,
                                                                                     0, 0, 0);
                    }
                }
            }
        };
#pragma unroll
        for (int u = 0; u < U; ++u) load(buf[u], w + u * W);
        for (int s = w; s < nk; s += W * U) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (s + u * W < nk) step(buf[u], s + u * W);
                load(buf[u], s + (u + U) * W);
            }
        }
        // accumulators are C^T: lane l holds row l%16 and columns 4*(l/16) .. +4
        __syncthreads();
        float* const red = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
                *reinterpret_cast<v4f*>(red + (w * ROWS + 16 * i + fr) * RSTR + 16 * j + 4 * (lane >> 4)) = acc[i][j];
        __syncthreads();
        for (int x = threadIdx.x; x < ROWS * COLS / 4; x += 64 * W) {
            const int r = x / (COLS / 4), c = (x % (COLS / 4)) * 4, col = n0 + c;
            if (r >= mrows || col >= g.N) continue;
            v4f t = *reinterpret_cast<const v4f*>(red + r * RSTR + c);
#pragma unroll
            for (int v = 1; v < W; ++v) t += *reinterpret_cast<const v4f*>(red + (v * ROWS + r) * RSTR + c);
            float o[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) o[y] = t[y] * sab;
            auto put = [&](auto* p) {
                using T = typename std::remove_reference<decltype(*p)>::type;
                if (g.vec_out && col + 3 < g.N) {
                    store4(p, o);
                } else {
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        if (col + y < g.N) p[y] = OutCvt<T>::cvt(o[y]);
                }
            };
            const int64_t at = ((SUMS ? (int64_t)e * g.M : 0) + m0 + r) * g.ldc + col;
            if (c_dtype == DF_DTYPE_FLOAT32) put(static_cast<float*>(g.C) + at);
            else if (c_dtype == DF_DTYPE_HALF) put(static_cast<f16_t*>(g.C) + at);
            else put(static_cast<uint16_t*>(g.C) + at);
        }
        if (SUMS) return;
        __syncthreads();  // the partial tiles are read before slabs go over them
    }
}

template <int FA, bool SUMS, bool WIDE> void launch_small(const ExpertArgs& g, int c_dtype, hipStream_t st) {
    if constexpr (SUMS) {
        const dim3 grid(((g.N + 31) / 32) * ((g.M + 31) / 32), g.experts);
        experts_small_kernel<FA, E4M3, 2, 2, 4, 2, true, WIDE><<<grid, 256, 0, st>>>(g, c_dtype);
    } else {
        if ((g.rows + g.experts - 1) / g.experts <= 16) {
            const dim3 grid((g.N + 15) / 16, g.experts);
            experts_small_kernel<FA, E4M3, 1, 1, 4, 4, false, WIDE><<<grid, 256, 0, st>>>(g, c_dtype);
        } else {
            // at most this many row tiles; blocks behind the last return at once
            const dim3 grid((g.N + 31) / 32, std::min(most_tiles(g.rows, g.experts, 32), 65535));
            experts_small_kernel<FA, E4M3, 2, 2, 4, 2, false, WIDE><<<grid, 256, 0, st>>>(g, c_dtype);
        }
    }
}

// Which kernel a call takes; the host knows the rows, not how they were dealt,
// and counts row tiles as if dealt evenly.
//  ROWS: by the time either would take, in us, a step being 128 of K.  Large
//    tiles: 5 + 1.2 for each wide step (0.72 for a narrow one; 2.05 times as much
//    on bf16 instructions) and round of blocks over the CUs, with 3 steps of
//    overhead a tile (2.8 narrow).  Small tiles of 32 x 32: 4 + 0.12 for each
//    step (its latency) + 0.35e-3 for each tile and step, with 10 steps of
//    overhead a tile.  Measured, us a call, small against large:
//      bf16 out, 1 expert 4160 -> 2112: per 48 9.0 / 27.4, per 320 17.9 / 35.6;
//      8 experts 1600 -> 6400: per 24 25.5 / 34.3, per 96 50.2 / 30.6; 1600 ->
//      1600: per 48 14.3 / 15.5, per 96 18.3 / 16.7; 16 experts 768 -> 256: per
//      160 8.4 / 10.4, per 320 13.1 / 11.1.  fp32 out, 8 experts 1600 -> 6400:
//      per 48 40.0 / 47.3, per 160 77 / 46; 1600 -> 1600: per 160 24.8 / 26.8.
//  SUMS: large tiles write dW in whole row segments: 8 experts 6400 x 1600,
//    per 16: 220 / 74; few outputs of long reductions want more blocks: 8 experts
//    256 x 256, per 1024: 9.2 / 20.9; 64 experts 256 x 256 (4096 small tiles),
//    per 256: 20.1 / 15.4; 64 experts 128 x 128 (1024): 9.2 / 12.7.
// 256 x 128 tiles where the rounds of blocks over the CUs come out cheaper, as
// for the dense products.  8 experts 6400 -> 1600, per 64: 54.7 / 39.3 wide
// against narrow; 1600 -> 6400, per 2048: 172 / 211.
struct TilePlan {
    bool tiles, narrow;
    int grid;
};
TilePlan plan(const ExpertArgs& g, bool sums, bool wide_codes) {
    const int per = (g.rows + g.experts - 1) / g.experts;
    const int cus = std::max(device_cu_count(), 1);
    TilePlan p{false, false, 0};
    const int64_t wn = (g.N + kPBN - 1) / kPBN, sn = (g.N + 127) / 128;
    // row tiles: ROWS end each expert with a partial one, half of one on average
    const int64_t some = std::min(g.experts, g.rows);
    auto row_tiles = [&](int tile) { return std::max(some, g.rows / tile + (some + 1) / 2); };
    const int64_t mt = sums ? (int64_t)g.experts * ((g.M + kPBM - 1) / kPBM) : row_tiles(kPBM);
    const int64_t steps = ((sums ? per : g.K) + kPKB - 1) / kPKB + (sums ? 1 : 0);
    const int64_t wr = (mt * wn + cus - 1) / cus, sr = (mt * sn + cus - 1) / cus;
    const double wide = (double)wr * ((double)steps + 3.0), narrow = (double)sr * (0.6 * (double)steps + 2.0);
    p.narrow = narrow < wide;
    if (sums) {
        p.tiles = (int64_t)g.experts * ((g.M + 31) / 32) * ((g.N + 31) / 32) > 8 * (int64_t)cus;
    } else {
        const double small = 4.0 + 0.12 * (double)steps +
                             0.35e-3 * (double)(row_tiles(32) * ((g.N + 31) / 32)) * ((double)steps + 10.0);
        p.tiles = 5.0 + (wide_codes ? 2.46 : 1.2) * std::min(wide, narrow) < small;
    }
    if (!p.tiles) return p;
    // at most this many units; blocks without one return at once
    const int64_t most = (sums ? mt : most_tiles(g.rows, g.experts, kPBM)) * (p.narrow ? sn : wn);
    p.grid = (int)std::min<int64_t>(most, cus);
    return p;
}

template <int FA, bool SUMS> void launch(ExpertArgs& g, int c_dtype, hipStream_t st) {
    const int64_t ldc_bytes = (int64_t)g.ldc * (c_dtype == DF_DTYPE_FLOAT32 ? 4 : 2);
    const TilePlan p = plan(g, SUMS, c_dtype == DF_DTYPE_FLOAT32);
    if (p.tiles) {
        g.vec_out = epi_store_mode(g.C, ldc_bytes);
        launch_expert_tiles(FA, SUMS, p.narrow, c_dtype, g, p.grid, st);
        return;
    }
    g.vec_out = ldc_bytes % 16 == 0 && aligned16(g.C);
    if (c_dtype == DF_DTYPE_FLOAT32) launch_small<FA, SUMS, true>(g, c_dtype, st);
    else launch_small<FA, SUMS, false>(g, c_dtype, st);
}

// Checks of one call; `empty`: nothing to compute.
int check_call(const char* fn, const ExpertArgs& g, int K, bool sums, int c_dtype, bool& empty) {
    DF_CHECK(g.rows >= 0 && g.M >= 0 && g.N >= 0 && K >= 0 && g.experts >= 0, DF_ERR_INVALID,
             "%s: a negative size (rows=%d, experts=%d)", fn, g.rows, g.experts);
    DF_CHECK(g.rows <= 0x7FFF0000, DF_ERR_INVALID, "%s: %d rows", fn, g.rows);  // row counters step past the last
    DF_CHECK(g.experts <= kMaxExperts, DF_ERR_UNSUPPORTED, "%s: %d experts (at most %d)", fn, g.experts, kMaxExperts);
    DF_CHECK(c_dtype == DF_DTYPE_FLOAT32 || c_dtype == DF_DTYPE_BFLOAT16 || c_dtype == DF_DTYPE_HALF,
             DF_ERR_UNSUPPORTED, "%s: output dtype %d not supported", fn, c_dtype);
    DF_CHECK((int64_t)((g.N + 15) / 16) * (sums ? (g.M + 15) / 16 : 1) < (1ll << 31) &&
                 (int64_t)((g.N + 127) / 128) *
                         (sums ? (int64_t)g.experts * ((g.M + 255) / 256) : (int64_t)g.rows / 256 + g.experts) <
                     (1ll << 31),
             DF_ERR_INVALID, "%s: output too large", fn);
    empty = g.experts == 0 || g.N == 0 || (sums ? g.M == 0 : g.rows == 0);
    if (empty) return DF_OK;
    DF_CHECK(g.ldc >= g.N, DF_ERR_INVALID, "%s: output leading dimension %d < %d", fn, g.ldc, g.N);
    DF_CHECK(g.C && g.off && g.sa && g.sb, DF_ERR_INVALID, "%s: NULL pointer", fn);
    const int red = sums ? g.rows : K;
    DF_CHECK((g.A && g.B) || red == 0, DF_ERR_INVALID, "%s: NULL operand", fn);
    DF_CHECK(red == 0 || (g.lda >= red && g.ldb >= red && g.lda % 16 == 0 && g.ldb % 16 == 0), DF_ERR_ALIGN,
             "%s: operand leading dimensions %d and %d must be multiples of 16 and >= %d", fn, g.lda, g.ldb, red);
    DF_CHECK(g.lda >= 0 && g.ldb >= 0 && g.lda < (1 << 23) && g.ldb < (1 << 23), DF_ERR_UNSUPPORTED,
             "%s: operand leading dimensions %d and %d (below 2^23)", fn, g.lda, g.ldb);
    DF_CHECK(aligned16(g.A) && aligned16(g.B), DF_ERR_ALIGN, "%s: operands must be 16-byte aligned", fn);
    DF_CHECK(aligned4(g.off) && aligned4(g.sa) && aligned4(g.sb), DF_ERR_ALIGN, "%s: offsets or scales misaligned", fn);
    DF_CHECK(((uintptr_t)g.C & (c_dtype == DF_DTYPE_FLOAT32 ? 3u : 1u)) == 0, DF_ERR_ALIGN,
             "%s: output is not aligned to its elements", fn);
    return DF_OK;
}

}  // namespace

}  // namespace dfk

using namespace dfk;

extern "C" int df_fp8_experts_fwd(const uint8_t* Xq, int ldx, const uint8_t* Wq, int ldw, int rows, int N, int K,
                                  int experts, const int* offsets_dev, const float* sx_dev, const float* sw_dev,
                                  int y_dtype, void* Y, int ldy, void* stream) {
    clear_error();
    const char* fn = "df_fp8_experts_fwd";
    ExpertArgs g{Xq, Wq, Y, offsets_dev, sx_dev, sw_dev, ldx, ldw, ldy, rows, 0, N, (K + 15) & ~15, experts, 0};
    bool empty = false;
    if (int rc = check_call(fn, g, K, false, y_dtype, empty)) return rc;
    if (empty) return DF_OK;
    launch<E4M3, false>(g, y_dtype, as_stream(stream));
    return launch_status(fn);
}

extern "C" int df_fp8_experts_dx(const uint8_t* dYq, int lddy, const uint8_t* Wtq, int ldwt, int rows, int N, int K,
                                 int experts, const int* offsets_dev, const float* sdy_dev, const float* sw_dev,
                                 int dx_dtype, void* dX, int lddx, void* stream) {
    clear_error();
    const char* fn = "df_fp8_experts_dx";
    ExpertArgs g{dYq, Wtq, dX, offsets_dev, sdy_dev, sw_dev, lddy, ldwt, lddx, rows, 0, K, (N + 15) & ~15, experts, 0};
    bool empty = false;
    if (int rc = check_call(fn, g, N, false, dx_dtype, empty)) return rc;
    if (empty) return DF_OK;
    launch<E5M2, false>(g, dx_dtype, as_stream(stream));
    return launch_status(fn);
}

extern "C" int df_fp8_experts_dw(const uint8_t* dYtq, int lddyt, const uint8_t* Xtq, int ldxt, int rows, int N, int K,
                                 int experts, const int* offsets_dev, const float* sdy_dev, const float* sx_dev,
                                 int dw_dtype, void* dW, int lddw, void* stream) {
    clear_error();
    const char* fn = "df_fp8_experts_dw";
    ExpertArgs g{dYtq, Xtq, dW, offsets_dev, sdy_dev, sx_dev, lddyt, ldxt, lddw, rows, N, K, 0, experts, 0};
    bool empty = false;
    if (int rc = check_call(fn, g, 0, true, dw_dtype, empty)) return rc;
    if (empty) return DF_OK;
    launch<E5M2, true>(g, dw_dtype, as_stream(stream));
    return launch_status(fn);
}
