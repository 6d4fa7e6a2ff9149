// gemm_blocks.hip -- fp8 products with a scale per 128 of the reduction (gfx950):
//   C[m][n] = sum over blocks b of sa[b][m] * sb[b][n] * sum over k in b of
//             A[m][k] * B[n][k], plus bias[n]
// with A e4m3 or e5m2 and B e4m3: the forward, dX and dW of a Linear.  A block of
// the reduction is one step of every kernel here (128 bytes of a row), so a scale
// is used once per row and step.
//
// Power-of-two scales (DF_SCALE_E8M0) go into the matrix instruction
// (v_mfma_scale_f32_*_f8f6f4 takes one per row and 32 of K) and cost no VALU work;
// with an fp32 output they go into the codes' widening to bf16 instead
// (v_cvt_scalef32_pk_bf16_*), whose products the bf16 instructions add exactly,
// for the reason given in gemm_experts.hip.  fp32 scales cannot: a step's product
// is made from zero and added to the sum by the VALU, times sa * sb (in binary64
// where B's are far, gemm_blocks.hpp).
//
// Few rows are bound by latency and by reading B once (16 x 4800 x 1600 with 7.7 MB of
// weights: 4.4 us, 3 of them a launch), many by the matrix units (gemm_blocks_tiles.hip).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gemm_blocks.hpp"

namespace dfk {

namespace {

// ------------------------------------------------------------ small tiles --
// A block owns a 16*MT x 16*NT tile; its W waves take the 128-byte steps in turn
// and add up through LDS, in wave order.  Loads take 8 rows x 128 bytes, eight lanes
// a row; each wave passes them to its fragments (lane l: row l%16, 32 bytes of K)
// through a slab of LDS of its own.  Straight from memory a fragment's load has four
// rows to every four lanes, 64 address lookups (16 x 4800 x 1600 with tiles of 16 x
// 16: 5.7 us, 5.1 so).  U steps are loaded ahead; with two of them registers are kept to
// three waves a SIMD (1000 x 1037 x 771, fp32 scales and outputs: 11.7 us with two, 9.8).
template <int FA, bool E8, bool WIDE, int MT, int NT, int W, int U>
__global__ __launch_bounds__(64 * W, W == 4 && U == 2 ? 3 : 1)
void blocks_small_kernel(const BlocksArgs g, int c_dtype, int extent_a, int extent_b) {
    constexpr int FB = E4M3;
    constexpr int ROWS = 16 * MT, COLS = 16 * NT;
    constexpr int RSTR = COLS + 4;  // row of a partial tile (floats)
    constexpr uint32_t kOOB = 0x80000000u;
    constexpr int SZ = E8 ? 1 : 4;
    constexpr int NL = 2 * (MT + NT);  // loads of 8 rows x 128 bytes per step
    constexpr int SLAB = NL * 1024;    // a wave's step: A rows, then B rows
    constexpr int RED = ROWS * RSTR * 4;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[W * (SLAB > RED ? SLAB : RED)];
    float* const red = reinterpret_cast<float*>(lds);
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // tiles in order of rows within a column of tiles, an XCD's (every eighth
    // block's) tiles next to each other: they share B in its L2
    const int tiles_m = (g.M + ROWS - 1) / ROWS, P = gridDim.x;
    const int q = P >> 3, rr = P & 7, xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
    const int tile = xcd < rr ? xcd * (q + 1) + idx : rr * (q + 1) + (xcd - rr) * q + idx;
    const int m0 = (tile % tiles_m) * ROWS, n0 = (tile / tiles_m) * COLS;

    const int fr = lane & 15, fq = lane >> 4;
    auto rsrc = [](const void* p, int bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, 0x00020000);
    };
    const __amdgpu_buffer_rsrc_t rA = rsrc(g.A + (int64_t)m0 * g.lda, min(g.M - m0, ROWS) * g.lda);
    const __amdgpu_buffer_rsrc_t rB = rsrc(g.B + (int64_t)n0 * g.ldb, min(g.N - n0, COLS) * g.ldb);
    // (bytes behind a matrix's last row of scales read as 0, and so do its codes)
    const __amdgpu_buffer_rsrc_t rSA = rsrc(static_cast<const uint8_t*>(g.sa) + (int64_t)m0 * SZ, max(extent_a - m0 * SZ, 0));
    const __amdgpu_buffer_rsrc_t rSB = rsrc(static_cast<const uint8_t*>(g.sb) + (int64_t)n0 * SZ, max(extent_b - n0 * SZ, 0));
    // loads: lane l takes 16-byte chunk l%8 of row l/8 of each 8-row group
    const int lr = lane >> 3, lc = (lane & 7) * 16;
    const uint32_t oa = (uint32_t)lr * (uint32_t)g.lda + (uint32_t)lc, ob = (uint32_t)lr * (uint32_t)g.ldb + (uint32_t)lc;
    // slab: rows of 128 bytes, 16-byte chunk c of row r in slot c ^ (r/2 % 8)
    uint8_t* const slab = lds + w * SLAB;
    const int wr_even = lr * 128 + (((lane & 7) ^ (lr >> 1)) << 4), wr_odd = wr_even ^ 64;
    const int fs = (fr >> 1) & 7;
    const int rd0 = fr * 128 + (((2 * fq) ^ fs) << 4), rd1 = fr * 128 + (((2 * fq + 1) ^ fs) << 4);
    // the lanes of a wave hand chunks to each other through the slab: LDS operations of
    // a wave execute in order, the compiler must keep that order
    auto lanes_meet = [] {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
    };

    struct Step {
        u32x4 raw[NL];
        uint32_t sa[MT];
        typename std::conditional<E8, uint32_t, u32x4>::type sb[NT];
        uint32_t column;  // fp32: the scale of column `lane`, if there is one
    };
    const uint32_t oc = lane < min(g.N - n0, COLS) ? (uint32_t)lane * 4 : kOOB;
    auto load_column = [&](Step& s, int step) {
        if constexpr (!E8)
            s.column = __builtin_amdgcn_raw_buffer_load_b32(
                rSB, step * 128 < g.K && oc != kOOB ? (uint32_t)step * (uint32_t)g.ldsb * SZ + oc : kOOB, 0, 0);
    };
    // (the first of 24 loads, or the last of a few: 1024 x 1600 x 6400 26.2 us and 27.4, but 16 x
    // 4800 x 1600 4.28 and 4.19)
    constexpr bool COL_FIRST = MT == 4;
    auto load = [&](Step& s, int step) {
        const int k = step * 128;
        if constexpr (COL_FIRST) load_column(s, step);
        const bool in = k + lc < g.K;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)
            s.raw[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                           rA, in ? oa + (uint32_t)(8 * i) * (uint32_t)g.lda + (uint32_t)k : kOOB, 0, 0));
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i)
            s.raw[2 * MT + i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                    rB, in ? ob + (uint32_t)(8 * i) * (uint32_t)g.ldb + (uint32_t)k : kOOB, 0, 0));
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint32_t sc = k < g.K ? ((uint32_t)step * (uint32_t)g.ldsa + 16 * i + fr) * SZ : kOOB;
            if constexpr (E8) s.sa[i] = __builtin_amdgcn_raw_buffer_load_b8(rSA, sc, 0, 0);
            else s.sa[i] = __builtin_amdgcn_raw_buffer_load_b32(rSA, sc, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint32_t sc = (uint32_t)step * (uint32_t)g.ldsb + 16 * j;
            if constexpr (E8) s.sb[j] = __builtin_amdgcn_raw_buffer_load_b8(rSB, k < g.K ? sc + fr : kOOB, 0, 0);
            else s.sb[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                              rSB, k < g.K ? (sc + 4 * fq) * SZ : kOOB, 0, 0));
        }
        if constexpr (!COL_FIRST) load_column(s, step);
    };
    // accumulators are C^T: lane l holds row l%16 and columns 4*(l/16) .. +4
    v4f acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // fragment t (16 rows) of a step in registers, through its part of the slab
    auto frag = [&](const Step& s, int t) -> v8i {
        *reinterpret_cast<u32x4*>(slab + t * 2048 + wr_even) = s.raw[2 * t];
        *reinterpret_cast<u32x4*>(slab + t * 2048 + 1024 + wr_odd) = s.raw[2 * t + 1];
        lanes_meet();
        const u32x4 x = *reinterpret_cast<const u32x4*>(slab + t * 2048 + rd0);
        const u32x4 y = *reinterpret_cast<const u32x4*>(slab + t * 2048 + rd1);
        return v8i{(int)x[0], (int)x[1], (int)x[2], (int)x[3], (int)y[0], (int)y[1], (int)y[2], (int)y[3]};
    };
    auto multiply = [&](const Step& s, auto is_far) {
        constexpr bool FAR = decltype(is_far)::value;
        lanes_meet();  // the step before has read the slab
        v8i fb[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j) fb[j] = frag(s, MT + j);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const v8i fa = frag(s, i);
            bf8 wa[4];
            if constexpr (WIDE) {
                const float sa = E8 ? __uint_as_float(s.sa[i] << 23) : 1.0f;
#pragma unroll
                for (int x = 0; x < 4; ++x) wa[x] = widen8_scaled<FA>((uint32_t)fa[2 * x], (uint32_t)fa[2 * x + 1], sa);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                v4f p = E8 ? acc[i][j] : v4f{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (WIDE) {
                    float sb = 1.0f;
                    if constexpr (E8) sb = __uint_as_float(s.sb[j] << 23);
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            widen8_scaled<FB>((uint32_t)fb[j][2 * x], (uint32_t)fb[j][2 * x + 1], sb), wa[x], p, 0, 0, 0);
                } else if constexpr (E8) {
                    p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, p, FB, FA, 0, (int)s.sb[j], 0, (int)s.sa[i]);
                } else {
                    p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, p, FB, FA, 0, 0, 0, 0);
                }
                if constexpr (E8) {
                    acc[i][j] = p;
                } else {
                    const float sa = __uint_as_float(s.sa[i]);
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const float sb = __uint_as_float(s.sb[j][y]);
                        acc[i][j][y] = FAR ? add_scaled_far(p[y], sa, sb, acc[i][j][y]) : __builtin_fmaf(p[y] * sb, sa, acc[i][j][y]);
                    }
                }
            }
        }
    };
    const int nk = (g.K + 127) >> 7;
    bool odd = false;  // fp32: a scale of this lane's column was far
    Step buf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(buf[u], w + u * W);
    for (int s = w; s < nk; s += W * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u * W < nk) {
                if constexpr (!E8) odd |= scale_far(buf[u].column);
                multiply(buf[u], std::false_type{});
            }
            load(buf[u], s + (u + U) * W);
        }
    }
    // Once more, all steps, where some of B's scales were far.  (Told apart step by step in
    // the loop, their code took it 60 registers more, and a branch held the next step's
    // loads back, 1024 x 1600 x 6400 32.7 us; 26.2 so, 25.7 without a look.)
    if constexpr (!E8) {
        if (__builtin_amdgcn_ballot_w64(odd) != 0) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            for (int s = w; s < nk; s += W) {
                load(buf[0], s);
                multiply(buf[0], std::true_type{});
            }
        }
    }
    __syncthreads();  // the slabs are read before sums go over them
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
            *reinterpret_cast<v4f*>(red + (w * ROWS + 16 * i + fr) * RSTR + 16 * j + 4 * fq) = acc[i][j];
    __syncthreads();
    const int mrows = min(g.M - m0, ROWS);
    // the waves' sums in order, V columns of a row at a time: four, or one where rows of C
    // start anywhere, so that lanes' stores follow each other
    auto write = [&](auto width, auto* C) {
        constexpr int V = decltype(width)::value;
        using T = typename std::remove_reference<decltype(*C)>::type;
        static_assert(64 * W % (COLS / V) == 0, "a thread's columns are the same in all its rows");
        const int c = (threadIdx.x % (COLS / V)) * V, col = n0 + c;
        if (col >= g.N) return;
        float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (g.bias) {
#pragma unroll
            for (int y = 0; y < V; ++y)
                if (col + y < g.N) bias[y] = bias_at(g.bias, g.bias_dtype, col + y);
        }
        for (int r = threadIdx.x / (COLS / V); r < mrows; r += 64 * W / (COLS / V)) {
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int v = 0; v < W; ++v) {
                const float* t = red + (v * ROWS + r) * RSTR + c;
#pragma unroll
                for (int y = 0; y < V; ++y) o[y] = v == 0 ? t[y] : o[y] + t[y];
            }
            if (g.bias) {
#pragma unroll
                for (int y = 0; y < V; ++y) o[y] += bias[y];
            }
            T* const p = C + (int64_t)(m0 + r) * g.ldc + col;
            if (V == 4 && col + 3 < g.N) {
                store4(p, o);
            } else {
#pragma unroll
                for (int y = 0; y < V; ++y)
                    if (col + y < g.N) p[y] = OutCvt<T>::cvt(o[y]);
            }
        }
    };
    auto as = [&](auto* C) {
        if (g.vec_out) write(std::integral_constant<int, 4>{}, C);
        else write(std::integral_constant<int, 1>{}, C);
    };
    if constexpr (WIDE) as(static_cast<float*>(g.C));
    else if (c_dtype == DF_DTYPE_HALF) as(static_cast<f16_t*>(g.C));
    else as(static_cast<uint16_t*>(g.C));
}

// Which kernel a call takes, by the time each would take, in us; a step is 128 of K.
// Measured at M, N, K (bf16 out, powers of two; graph replays, a launch being 2.5 to 3
// of it):
//   16 x 16 tiles, while they are no more than the CUs: 32 x 1600 x 6400 5.8 (32 x 32:
//     7.6); up to 16 rows otherwise 16 x 32: 16 x 4800 x 1600 4.4 (16 x 16: 5.1)
//   32 x 32: 64 x 6400 x 1600 6.9, 256 x 6400 x 1600 16, 512 x 512 x 16384 16.3 (with
//     four waves in place of eight 7.1, 16, 19.9; 1000 x 1037 x 771, seven steps, 10.2
//     and 9.5)
//   64 x 64: 256 x 6400 x 1600 12.1, 1024 x 1600 x 6400 27.5
//   128 x 128: 256 x 6400 x 1600 10.1, 1024 x 1600 x 6400 25.7, 2048 x 6400 x 1600 35
//   256 x 256: 2048 x 6400 x 1600 25.2, 1024 x 1600 x 6400 60
// and likewise with fp32 outputs or scales, whose steps take longer on large tiles
// (128 x 128, 1024 x 1600 x 6400: 49 and 37.5; 64 x 64: 32 and 28.7).
struct BlocksPlan {
    int kernel;  // DF_BLOCKS_KERNEL_*
    int grid;
};
BlocksPlan plan(const BlocksArgs& g, bool e8, bool wide) {
    const int cus = std::max(device_cu_count(), 1);
    const double steps = (double)((g.K + 127) / 128);
    auto tiles = [&](int r, int c) { return (int64_t)((g.M + r - 1) / r) * ((g.N + c - 1) / c); };
    if (g.K == 0) return {DF_BLOCKS_KERNEL_32, (int)tiles(32, 32)};
    if (tiles(16, 16) <= cus) return {DF_BLOCKS_KERNEL_16, (int)tiles(16, 16)};
    if (g.M <= 16) return {DF_BLOCKS_KERNEL_16X32, (int)tiles(16, 32)};
    // fp32 scales, fp32 outputs: 0 to 3
    const int kind = (e8 ? 0 : 2) + (wide ? 1 : 0);
    const double slower[4] = {1.0, 1.08, 1.1, 1.2};
    double best = 3.2 + std::max(0.1 * steps, slower[kind] * (double)tiles(32, 32) * (0.56e-3 * steps + 1.9e-3));
    BlocksPlan p{g.K > 8 * 128 ? DF_BLOCKS_KERNEL_32_LONG : DF_BLOCKS_KERNEL_32, (int)tiles(32, 32)};
    auto offer = [&](int kernel, int64_t n, double t) {
        if (t < best) {
            best = t;
            p = {kernel, (int)n};
        }
    };
    if (kind != 3)
        offer(DF_BLOCKS_KERNEL_64, tiles(64, 64),
              3.5 + slower[kind] * (0.25 * steps + (double)tiles(64, 64) * (0.41e-3 * steps + 8.2e-3)));
    // rounds of blocks over the CUs, a step's time and a tile's besides
    auto large = [&](int kernel, int r, int c, const double* step, const double* over) {
        const int64_t n = tiles(r, c), rounds = (n + cus - 1) / cus;
        offer(kernel, std::min<int64_t>(n, cus), 3.0 + (double)rounds * (step[kind] * steps + over[kind]));
    };
    const double s1[4] = {0.39, 0.83, 0.62, 1.03}, o1[4] = {2.6, 3.0, 2.0, 3.0};
    const double s2[4] = {0.75, 1.28, 1.02, 1.75}, o2[4] = {3.0, 4.5, 2.5, 4.0};
    const double s4[2] = {1.1, 2.2}, o4[2] = {6.0, 8.0};
    large(DF_BLOCKS_KERNEL_128, 128, 128, s1, o1);
    large(DF_BLOCKS_KERNEL_256X128, 256, 128, s2, o2);
    if (e8) large(DF_BLOCKS_KERNEL_256, 256, 256, s4, o4);
    return p;
}

template <int FA, bool E8, bool WIDE>
void launch_small(const BlocksPlan& p, const BlocksArgs& g, int c_dtype, int ea, int eb, hipStream_t st) {
    if (p.kernel == DF_BLOCKS_KERNEL_16)
        blocks_small_kernel<FA, E8, WIDE, 1, 1, 8, 2><<<p.grid, 512, 0, st>>>(g, c_dtype, ea, eb);
    else if (p.kernel == DF_BLOCKS_KERNEL_16X32)
        blocks_small_kernel<FA, E8, WIDE, 1, 2, 8, 1><<<p.grid, 512, 0, st>>>(g, c_dtype, ea, eb);
    else if (p.kernel == DF_BLOCKS_KERNEL_32_LONG)
        blocks_small_kernel<FA, E8, WIDE, 2, 2, 8, 1><<<p.grid, 512, 0, st>>>(g, c_dtype, ea, eb);
    else if (p.kernel == DF_BLOCKS_KERNEL_32)
        blocks_small_kernel<FA, E8, WIDE, 2, 2, 4, 2><<<p.grid, 256, 0, st>>>(g, c_dtype, ea, eb);
    else if constexpr (E8 || !WIDE)
        blocks_small_kernel<FA, E8, WIDE, 4, 4, 4, 1><<<p.grid, 256, 0, st>>>(g, c_dtype, ea, eb);
}

}  // namespace

}  // namespace dfk

using namespace dfk;

// (blocks of small tiles: fewer than 2^32 threads; those of M <= 16 and of large tiles
// are fewer)
static bool tiles_fit(int M, int N) { return ((M + 31ll) / 32) * ((N + 31ll) / 32) < (1ll << 23); }

extern "C" int df_fp8_gemm_blocks_plan(int M, int N, int K, int scale_kind, int c_dtype, int* kernel) {
    clear_error();
    const char* fn = "df_fp8_gemm_blocks_plan";
    DF_CHECK(kernel, DF_ERR_INVALID, "%s: NULL output", fn);
    DF_CHECK(M > 0 && N > 0 && K >= 0, DF_ERR_INVALID, "%s: bad sizes (M=%d, N=%d, K=%d)", fn, M, N, K);
    DF_CHECK(scale_kind_ok(scale_kind), DF_ERR_INVALID, "%s: bad scale kind %d", fn, scale_kind);
    DF_CHECK(c_dtype == DF_DTYPE_FLOAT32 || c_dtype == DF_DTYPE_BFLOAT16 || c_dtype == DF_DTYPE_HALF, DF_ERR_UNSUPPORTED,
             "%s: output dtype %d not supported", fn, c_dtype);
    DF_CHECK(tiles_fit(M, N), DF_ERR_UNSUPPORTED, "%s: output of %d x %d too large", fn, M, N);
    BlocksArgs g{};
    g.M = M;
    g.N = N;
    g.K = (int)std::min(((int64_t)K + 15) & ~(int64_t)15, (int64_t)0x7FFFFFF0);
    *kernel = plan(g, scale_kind == DF_SCALE_E8M0, c_dtype == DF_DTYPE_FLOAT32).kernel;
    return DF_OK;
}

extern "C" int df_fp8_gemm_blocks(int fmt_a, const uint8_t* A, int lda, const uint8_t* B, int ldb, int M, int N, int K,
                                  int scale_kind, const void* sa, int ldsa, const void* sb, int ldsb, int bias_dtype,
                                  const void* bias, int c_dtype, void* C, int ldc, void* stream) {
    clear_error();
    const char* fn = "df_fp8_gemm_blocks";
    auto value_dtype = [](int d) { return d == DF_DTYPE_FLOAT32 || d == DF_DTYPE_BFLOAT16 || d == DF_DTYPE_HALF; };
    auto misaligned = [](const void* p, int d) { return ((uintptr_t)p & (d == DF_DTYPE_FLOAT32 ? 3u : 1u)) != 0; };
    DF_CHECK(M >= 0 && N >= 0 && K >= 0, DF_ERR_INVALID, "%s: a negative size (M=%d, N=%d, K=%d)", fn, M, N, K);
    DF_CHECK(fmt_a == DF_FMT_E4M3 || fmt_a == DF_FMT_E5M2, DF_ERR_INVALID, "%s: bad format %d", fn, fmt_a);
    DF_CHECK(scale_kind_ok(scale_kind), DF_ERR_INVALID, "%s: bad scale kind %d", fn, scale_kind);
    DF_CHECK(value_dtype(c_dtype), DF_ERR_UNSUPPORTED, "%s: output dtype %d not supported", fn, c_dtype);
    DF_CHECK(!bias || value_dtype(bias_dtype), DF_ERR_UNSUPPORTED, "%s: bias dtype %d not supported", fn, bias_dtype);
    DF_CHECK(tiles_fit(M, N), DF_ERR_UNSUPPORTED, "%s: output of %d x %d too large",
             fn, M, N);
    if (M == 0 || N == 0) return DF_OK;
    DF_CHECK(C && ldc >= N, DF_ERR_INVALID, "%s: output NULL or leading dimension %d < %d", fn, ldc, N);
    DF_CHECK(!misaligned(C, c_dtype) && !(bias && misaligned(bias, bias_dtype)), DF_ERR_ALIGN,
             "%s: output or bias is not aligned to its elements", fn);
    DF_CHECK(K == 0 || (A && B && sa && sb), DF_ERR_INVALID, "%s: NULL operand or scales", fn);
    DF_CHECK(K == 0 || (lda >= K && ldb >= K && lda % 16 == 0 && ldb % 16 == 0), DF_ERR_ALIGN,
             "%s: operand leading dimensions %d and %d must be multiples of 16 and >= %d", fn, lda, ldb, K);
    DF_CHECK(lda < (1 << 23) && ldb < (1 << 23), DF_ERR_UNSUPPORTED, "%s: operand leading dimensions %d and %d (below 2^23)",
             fn, lda, ldb);
    const int sz = scale_bytes(scale_kind);
    DF_CHECK(K == 0 || (ldsa >= M && ldsb >= N && (int64_t)ldsa * sz % 16 == 0 && (int64_t)ldsb * sz % 16 == 0), DF_ERR_ALIGN,
             "%s: scale leading dimensions %d and %d must be whole 16 bytes and >= %d and %d", fn, ldsa, ldsb, M, N);
    DF_CHECK(aligned16(A) && aligned16(B) && aligned16(sa) && aligned16(sb), DF_ERR_ALIGN,
             "%s: operands and scales must be 16-byte aligned", fn);
    const int64_t blocks = ((int64_t)K + 127) / 128;
    const int64_t ea = scales_extent(blocks, ldsa, M, sz), eb = scales_extent(blocks, ldsb, N, sz);
    DF_CHECK(ea < (1ll << 31) && eb < (1ll << 31), DF_ERR_UNSUPPORTED, "%s: scales of 2^31 bytes or more", fn);
    BlocksArgs g{A, B, C, sa, sb, bias, lda, ldb, ldc, ldsa, ldsb, M, N, (K + 15) & ~15, bias_dtype, 0};
    const int64_t ldc_bytes = (int64_t)ldc * (c_dtype == DF_DTYPE_FLOAT32 ? 4 : 2);
    if (K == 0) g.lda = g.ldb = g.ldsa = g.ldsb = 0;  // (not checked then, and nothing is read)
    const hipStream_t st = as_stream(stream);
    const bool wide = c_dtype == DF_DTYPE_FLOAT32, e8 = scale_kind == DF_SCALE_E8M0;
    const BlocksPlan p = plan(g, e8, wide);
    if (p.kernel >= DF_BLOCKS_KERNEL_128) {
        const int fm = p.kernel == DF_BLOCKS_KERNEL_128 ? 1 : p.kernel == DF_BLOCKS_KERNEL_256X128 ? 2 : 4;
        g.vec_out = epi_store_mode(C, ldc_bytes);
        launch_block_tiles(fmt_a, e8, fm, c_dtype, g, (int)ea, (int)eb, p.grid, st);
        return launch_status(fn);
    }
    g.vec_out = ldc_bytes % 16 == 0 && aligned16(C);
    auto go = [&](auto fa, auto e, auto wd) {
        launch_small<decltype(fa)::value, decltype(e)::value, decltype(wd)::value>(p, g, c_dtype, (int)ea, (int)eb, st);
    };
    auto as = [&](auto fa) {
        using Y = std::true_type;
        using X = std::false_type;
        if (e8 && wide) go(fa, Y{}, Y{});
        else if (e8) go(fa, Y{}, X{});
        else if (wide) go(fa, X{}, Y{});
        else go(fa, X{}, X{});
    };
    if (fmt_a == DF_FMT_E4M3) as(std::integral_constant<int, E4M3>{});
    else as(std::integral_constant<int, E5M2>{});
    return launch_status(fn);
}
