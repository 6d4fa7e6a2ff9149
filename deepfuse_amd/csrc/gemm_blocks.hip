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
// is made from zero and added to the sum by the VALU, times sa * sb.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gemm_blocks.hpp"

namespace dfk {

namespace {

// ------------------------------------------------------------ small tiles --
// A block owns a 16*MT x 16*NT tile; its W waves take the 128-byte steps in turn
// and add up through LDS, in wave order.  Fragments go from memory to registers
// as the instruction wants them: lane l has row l%16 and the 16-byte chunks l/16
// and l/16 + 4 of a step (which K a lane holds is free as long as A and B agree
// and share a scale).  U steps are loaded ahead.
template <int FA, bool E8, bool WIDE, int MT, int NT, int W, int U>
__global__ __launch_bounds__(64 * W) void blocks_small_kernel(const BlocksArgs g, int c_dtype, int extent_a, int extent_b) {
    constexpr int FB = E4M3;
    constexpr int ROWS = 16 * MT, COLS = 16 * NT;
    constexpr int RSTR = COLS + 4;  // row of a partial tile (floats)
    constexpr uint32_t kOOB = 0x80000000u;
    constexpr int SZ = E8 ? 1 : 4;
    __shared__ __attribute__((aligned(16))) float red[W * ROWS * RSTR];
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
    const uint32_t oa = (uint32_t)fr * (uint32_t)g.lda + 16u * fq, ob = (uint32_t)fr * (uint32_t)g.ldb + 16u * fq;

    struct Step {
        u32x4 a[MT][2], b[NT][2];
        uint32_t sa[MT];
        typename std::conditional<E8, uint32_t, u32x4>::type sb[NT];
    };
    auto load = [&](Step& s, int step) {
        const int k = step * 128, c = k + 16 * fq;
        const bool in0 = c < g.K, in1 = c + 64 < g.K;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const uint32_t at = oa + (uint32_t)(16 * i) * (uint32_t)g.lda + (uint32_t)k;
            s.a[i][0] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rA, in0 ? at : kOOB, 0, 0));
            s.a[i][1] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rA, in1 ? at + 64 : kOOB, 0, 0));
            const uint32_t sc = k < g.K ? ((uint32_t)step * (uint32_t)g.ldsa + 16 * i + fr) * SZ : kOOB;
            if constexpr (E8) s.sa[i] = __builtin_amdgcn_raw_buffer_load_b8(rSA, sc, 0, 0);
            else s.sa[i] = __builtin_amdgcn_raw_buffer_load_b32(rSA, sc, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const uint32_t at = ob + (uint32_t)(16 * j) * (uint32_t)g.ldb + (uint32_t)k;
            s.b[j][0] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rB, in0 ? at : kOOB, 0, 0));
            s.b[j][1] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rB, in1 ? at + 64 : kOOB, 0, 0));
            const uint32_t sc = (uint32_t)step * (uint32_t)g.ldsb + 16 * j;
            if constexpr (E8) s.sb[j] = __builtin_amdgcn_raw_buffer_load_b8(rSB, k < g.K ? sc + fr : kOOB, 0, 0);
            else s.sb[j] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                              rSB, k < g.K ? (sc + 4 * fq) * SZ : kOOB, 0, 0));
        }
    };
    // accumulators are C^T: lane l holds row l%16 and columns 4*(l/16) .. +4
    v4f acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    auto whole = [](const u32x4* p) {
        v8i f;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            f[x] = (int)p[0][x];
            f[4 + x] = (int)p[1][x];
        }
        return f;
    };
    auto multiply = [&](const Step& s) {
        if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float sb = 1.0f;
                if constexpr (E8) sb = __uint_as_float(s.sb[j] << 23);
                bf8 wb[4];
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    wb[x] = widen8_scaled<FB>(s.b[j][x >> 1][2 * (x & 1)], s.b[j][x >> 1][2 * (x & 1) + 1], sb);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const float sa = E8 ? __uint_as_float(s.sa[i] << 23) : 1.0f;
                    v4f p = E8 ? acc[i][j] : v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        p = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            wb[x], widen8_scaled<FA>(s.a[i][x >> 1][2 * (x & 1)], s.a[i][x >> 1][2 * (x & 1) + 1], sa), p, 0,
                            0, 0);
                    if constexpr (E8) {
                        acc[i][j] = p;
                    } else {
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            acc[i][j][y] = __builtin_fmaf(p[y] * __uint_as_float(s.sb[j][y]), __uint_as_float(s.sa[i]), acc[i][j][y]);
                    }
                }
            }
        } else {
            v8i fb[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) fb[j] = whole(s.b[j]);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const v8i fa = whole(s.a[i]);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    if constexpr (E8) {
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], FB, FA, 0,
                                                                                     (int)s.sb[j], 0, (int)s.sa[i]);
                    } else {
                        const v4f z = {0.0f, 0.0f, 0.0f, 0.0f};
                        const v4f p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, z, FB, FA, 0, 0, 0, 0);
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            acc[i][j][y] = __builtin_fmaf(p[y] * __uint_as_float(s.sb[j][y]), __uint_as_float(s.sa[i]), acc[i][j][y]);
                    }
                }
            }
        }
    };
    const int nk = (g.K + 127) >> 7;
    Step buf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) load(buf[u], w + u * W);
    for (int s = w; s < nk; s += W * U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u * W < nk) multiply(buf[u]);
            load(buf[u], s + (u + U) * W);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
            *reinterpret_cast<v4f*>(red + (w * ROWS + 16 * i + fr) * RSTR + 16 * j + 4 * fq) = acc[i][j];
    __syncthreads();
    const int mrows = min(g.M - m0, ROWS);
    for (int x = threadIdx.x; x < ROWS * COLS / 4; x += 64 * W) {
        const int r = x / (COLS / 4), c = (x % (COLS / 4)) * 4, col = n0 + c;
        if (r >= mrows || col >= g.N) continue;
        v4f t = *reinterpret_cast<const v4f*>(red + r * RSTR + c);
#pragma unroll
        for (int v = 1; v < W; ++v) t += *reinterpret_cast<const v4f*>(red + (v * ROWS + r) * RSTR + c);
        float o[4] = {t[0], t[1], t[2], t[3]};
        if (g.bias) {
#pragma unroll
            for (int y = 0; y < 4; ++y)
                if (col + y < g.N) o[y] += bias_at(g.bias, g.bias_dtype, col + y);
        }
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
        const int64_t at = (int64_t)(m0 + r) * g.ldc + col;
        if (c_dtype == DF_DTYPE_FLOAT32) put(static_cast<float*>(g.C) + at);
        else if (c_dtype == DF_DTYPE_HALF) put(static_cast<f16_t*>(g.C) + at);
        else put(static_cast<uint16_t*>(g.C) + at);
    }
}

template <int FA, bool E8, bool WIDE> void launch_small(const BlocksArgs& g, int c_dtype, int ea, int eb, hipStream_t st) {
    auto tiles = [&](int r, int c) { return (int)((int64_t)((g.M + r - 1) / r) * ((g.N + c - 1) / c)); };
    if (g.M <= 16 || g.N <= 16)
        blocks_small_kernel<FA, E8, WIDE, 1, 1, 4, 4><<<tiles(16, 16), 256, 0, st>>>(g, c_dtype, ea, eb);
    else
        blocks_small_kernel<FA, E8, WIDE, 2, 2, 4, 2><<<tiles(32, 32), 256, 0, st>>>(g, c_dtype, ea, eb);
}

// Which kernel a call takes, by the time each would take, in us; a step is 128 of
// K.  Large tiles: rounds of blocks over the CUs.
struct BlocksPlan {
    int fm;  // 0: small tiles
    int grid;
};
BlocksPlan plan(const BlocksArgs& g, bool e8, bool wide) {
    const int cus = std::max(device_cu_count(), 1);
    const double steps = (double)((g.K + 127) / 128);
    auto tiles = [&](int r, int c) { return (int64_t)((g.M + r - 1) / r) * ((g.N + c - 1) / c); };
    double best = 4.0 + 0.12 * steps + 0.35e-3 * (double)tiles(32, 32) * (steps + 10.0);
    BlocksPlan p{0, 0};
    if (g.K == 0) return p;
    auto offer = [&](int fm, int r, int c, double step, double over) {
        const int64_t n = tiles(r, c), rounds = (n + cus - 1) / cus;
        const double t = 5.0 + (double)rounds * (wide ? 2.05 : 1.0) * (step * steps + over);
        if (t < best) {
            best = t;
            p = {fm, (int)std::min<int64_t>(n, cus)};
        }
    };
    if (e8) {
        offer(4, 256, 256, 1.2, 3.6);
        offer(2, 256, 128, 0.72, 2.4);
        offer(1, 128, 128, 0.5, 1.8);
    } else {
        offer(2, 256, 128, 1.1, 2.4);
        offer(1, 128, 128, 0.7, 1.8);
    }
    return p;
}

}  // namespace

}  // namespace dfk

using namespace dfk;

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
    DF_CHECK((int64_t)((M + 15) / 16) * ((N + 15) / 16) < (1ll << 31), DF_ERR_INVALID, "%s: output too large", fn);
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
    if (p.fm) {
        g.vec_out = epi_store_mode(C, ldc_bytes);
        launch_block_tiles(fmt_a, e8, p.fm, c_dtype, g, (int)ea, (int)eb, p.grid, st);
        return launch_status(fn);
    }
    g.vec_out = ldc_bytes % 16 == 0 && aligned16(C);
    auto go = [&](auto fa, auto e, auto wd) {
        launch_small<decltype(fa)::value, decltype(e)::value, decltype(wd)::value>(g, c_dtype, (int)ea, (int)eb, st);
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
