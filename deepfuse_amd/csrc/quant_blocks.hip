// quant_blocks.hip -- a matrix to fp8 codes with a scale per 128 values (gfx950):
// row codes with a scale for 128 columns of a row, transposed codes with a scale
// for 128 rows of a column (each what the product that reduces over them reads),
// or both at one scale per 128 x 128 square.
//
// Bound by HBM: the matrix is read once and each kind of codes written once.  A
// block owns a 128 x 128 square, so that both directions' absmax and scales come
// from registers: a thread holds 8 x 8 values, 16 lanes (a DPP row) the 128
// columns of 8 rows; rows' maxima stay in a DPP row, columns' pass two lane
// exchanges and LDS.  Transposed codes leave through LDS in 16-byte stores of
// 128 consecutive rows.
//
// Measured (bf16, both kinds of codes, powers of two): 16384 x 6400 88 us, 4.8 TB/s
// where a copy reaches 5.2; with fp32 scales, whose quotients are divisions, 110.
// Calls of few squares take 6 to 10 us, a launch and a block's chain of load, maximum,
// exchange and stores; the rare paths (NaN, slow division) in loops instead of unrolled,
// 20 KB of code in place of 50, changed nothing there.
//
// No reference counterpart (the reference has no fp8).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "block_scale.hpp"
#include "df_common.hpp"
#include "row_chunks.hpp"

namespace dfk {

namespace {

struct BlockQuant {
    const void* x;
    uint8_t* q; void* s;    // row codes [rows, ldq], scales [column blocks, lds]
    uint8_t* qt; void* st;  // transposed codes [cols, ldqt], scales [row blocks, ldst]
    int rows, cols, ldx, ldq, lds, ldqt, ldst;
};

// eight scales that follow each other at p[at..], those below `end`
template <bool E8> __device__ __forceinline__ void put_scales(void* p, int64_t at, int n, const BlockDiv* b) {
    if constexpr (E8) {
        uint8_t* d = static_cast<uint8_t*>(p) + at;
        if (n >= 8) {
            u32x2 w = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i >> 2] |= b[i].byte << 8 * (i & 3);
            *reinterpret_cast<u32x2*>(d) = w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) d[i] = (uint8_t)b[i].byte;
        }
    } else {
        float* d = static_cast<float*>(p) + at;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) d[i] = b[i].d.s;
    }
}

// The absmax over finite values of 8 rows and 8 columns of values, without compares
// (fold_*_biased); 2-byte values two columns at a time.
template <typename T> struct Folds {  // bf16 and f16
    static constexpr bool BF = std::is_same<T, uint16_t>::value;
    static constexpr uint32_t bias = BF ? 0x00800080u : 0x04000400u;
    static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(df_short2, a), __builtin_bit_cast(df_short2, b)));
    }
    static __device__ __forceinline__ uint32_t value(int half) {  // a biased half as a binary32 pattern
        const uint32_t h = (uint32_t)max(half - (BF ? 0x80 : 0x400), 0);
        return BF ? h << 16 : __float_as_uint(f16_to_f32(h));
    }
    static __device__ __forceinline__ void fold(const u32x4 (&w)[8][1], uint32_t* rm, uint32_t* cm) {
        uint32_t col[4] = {0, 0, 0, 0};
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            uint32_t row = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = (w[p][0][i] & 0x7FFF7FFFu) + bias;  // not finite: negative
                row = larger(row, u);
                col[i] = larger(col[i], u);
            }
            rm[p] = value(max((int)(int16_t)(row >> 16), (int)(int16_t)(row & 0xFFFFu)));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cm[2 * i] = value((int)(int16_t)(col[i] & 0xFFFFu));
            cm[2 * i + 1] = value((int)(int16_t)(col[i] >> 16));
        }
    }
};
template <> struct Folds<float> {
    static __device__ __forceinline__ void fold(const u32x4 (&w)[8][2], uint32_t* rm, uint32_t* cm) {
#pragma unroll
        for (int e = 0; e < 8; ++e) cm[e] = 0;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            rm[p] = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                rm[p] = fold_f32_biased(rm[p], w[p][e >> 2][e & 3]);
                cm[e] = fold_f32_biased(cm[e], w[p][e >> 2][e & 3]);
            }
            rm[p] = unbias_f32(rm[p]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) cm[e] = unbias_f32(cm[e]);
    }
};

template <typename T, int FMT, bool E8, bool SQUARE>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(const BlockQuant a) {
    constexpr int E = El<T>::E, PITCH = 132;  // bytes of a transposed row in LDS: no bank conflicts in its writes
    __shared__ uint32_t colmax[4][kScaleBlock];
    __shared__ uint32_t tile[kScaleBlock * PITCH / 4];
    const int t = threadIdx.x, tr = t >> 4, tc = t & 15, w = t >> 6;
    const int64_t r0 = (int64_t)blockIdx.y * kScaleBlock;
    const int c0 = blockIdx.x * kScaleBlock, c = c0 + 8 * tc;
    const int64_t r = r0 + 8 * tr;
    // columns from the square before on: an offset in a row has 32 bits, its length more
    const int cb = max(c0 - kScaleBlock, 0), cols = a.cols - cb;
    const T* const x = static_cast<const T*>(a.x) + cb;

    u32x4 raw[8][8 / E];
#pragma unroll
    for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int h = 0; h < 8 / E; ++h)
            raw[p][h] = r + p < a.rows ? load_chunk<T>(x + (r + p) * a.ldx, (c - cb) / E + h, cols) : u32x4{0, 0, 0, 0};
    float v[8][8];
#pragma unroll
    for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int h = 0; h < 8 / E; ++h) {
            raw[p][h] = place_chunk<T>(raw[p][h], (c - cb) / E + h, cols);
            El<T>::widen(raw[p][h], v[p] + h * E);
        }

    bool nan = false;
#pragma unroll
    for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int e = 0; e < 8; e += 2) nan |= __builtin_isunordered(v[p][e], v[p][e + 1]);

    // absmax of the thread's rows and columns, as binary32 patterns
    uint32_t rm[8], cm[8];
    Folds<T>::fold(raw, rm, cm);
    if (!SQUARE) {
#pragma unroll
        for (int p = 0; p < 8; ++p) rm[p] = row16_max(rm[p]);
    }
    if constexpr (SQUARE) {
        uint32_t m = 0;
#pragma unroll
        for (int p = 0; p < 8; ++p) m = max(m, rm[p]);
        m = row16_max(m);
        m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        if ((t & 63) == 0) colmax[0][w] = m;
        __syncthreads();
        m = max(max(colmax[0][0], colmax[0][1]), max(colmax[0][2], colmax[0][3]));
#pragma unroll
        for (int p = 0; p < 8; ++p) rm[p] = cm[p] = m;
    } else if (a.qt) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            cm[e] = max(cm[e], (uint32_t)__shfl_xor((int)cm[e], 16, 64));
            cm[e] = max(cm[e], (uint32_t)__shfl_xor((int)cm[e], 32, 64));
            if ((t & 63) < 16) colmax[w][8 * tc + e] = cm[e];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e)
            cm[e] = max(max(colmax[0][8 * tc + e], colmax[1][8 * tc + e]),
                        max(colmax[2][8 * tc + e], colmax[3][8 * tc + e]));
    }

    if (a.q) {
        BlockDiv b[8];
        bool bad = nan;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            b[p] = block_div<FMT, E8>(rm[p]);
            bad |= !b[p].d.fast;
        }
        auto codes = [&](auto plain) {
#pragma unroll
            for (int p = 0; p < 8; ++p) {
                const u32x2 k = {block_quant4<FMT, E8, decltype(plain)::value>(v[p], b[p].d),
                                 block_quant4<FMT, E8, decltype(plain)::value>(v[p] + 4, b[p].d)};
                if (r + p < a.rows && c < ((a.cols + 15) & ~15)) *reinterpret_cast<u32x2*>(a.q + (r + p) * a.ldq + c) = k;
            }
        };
        if (__builtin_amdgcn_ballot_w64(bad) == 0) codes(std::true_type{});
        else codes(std::false_type{});
        if (tc == 0 && r < a.rows)
            put_scales<E8>(a.s, (int64_t)blockIdx.x * a.lds + r, (int)min<int64_t>(a.rows - r, 8), b);
    }
    if (a.qt) {
        BlockDiv b[8];
        bool bad = nan;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            b[e] = block_div<FMT, E8>(cm[e]);
            bad |= !b[e].d.fast;
        }
        auto codes = [&](auto plain) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float col[8] = {v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e]};
                uint32_t* p = tile + ((8 * tc + e) * PITCH + 8 * tr) / 4;
                p[0] = block_quant4<FMT, E8, decltype(plain)::value>(col, b[e].d);
                p[1] = block_quant4<FMT, E8, decltype(plain)::value>(col + 4, b[e].d);
            }
        };
        if (__builtin_amdgcn_ballot_w64(bad) == 0) codes(std::true_type{});
        else codes(std::false_type{});
        if (tr == 0 && c < a.cols) put_scales<E8>(a.st, (int64_t)blockIdx.y * a.ldst + c, min(a.cols - c, 8), b);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = i * 32 + (t >> 3), k = t & 7;
            const uint32_t* p = tile + (col * PITCH + 16 * k) / 4;
            const u32x4 o = {p[0], p[1], p[2], p[3]};
            // (rows up to the next multiple of 16 hold zero codes)
            if (c0 + col < a.cols && r0 + 16 * k < a.rows)
                *reinterpret_cast<u32x4*>(a.qt + (int64_t)(c0 + col) * a.ldqt + r0 + 16 * k) = o;
        }
    }
}

template <typename T, int FMT> void launch(const BlockQuant& a, bool e8, bool square, hipStream_t st) {
    const dim3 grid((a.cols + kScaleBlock - 1) / kScaleBlock, (a.rows + kScaleBlock - 1) / kScaleBlock);
    if (e8 && square) quantize_blocks_kernel<T, FMT, true, true><<<grid, 256, 0, st>>>(a);
    else if (e8) quantize_blocks_kernel<T, FMT, true, false><<<grid, 256, 0, st>>>(a);
    else if (square) quantize_blocks_kernel<T, FMT, false, true><<<grid, 256, 0, st>>>(a);
    else quantize_blocks_kernel<T, FMT, false, false><<<grid, 256, 0, st>>>(a);
}

}  // namespace

}  // namespace dfk

using namespace dfk;

extern "C" int df_quantize_blocks(int dtype, const void* x, int rows, int cols, int ldx, int fmt, int scale_kind,
                                  int square, uint8_t* q, int ldq, void* scales, int ld_scales, uint8_t* qt, int ldqt,
                                  void* scales_t, int ld_scales_t, void* stream) {
    clear_error();
    const char* fn = "df_quantize_blocks";
    DF_CHECK(rows >= 0 && cols >= 0 && rows <= 128 * 65535 && cols <= 0x7FFF0000, DF_ERR_INVALID,
             "%s: bad shape rows=%d cols=%d (at most %d rows)", fn, rows, cols, 128 * 65535);
    DF_CHECK(dtype == DF_DTYPE_FLOAT32 || dtype == DF_DTYPE_BFLOAT16 || dtype == DF_DTYPE_HALF, DF_ERR_UNSUPPORTED,
             "%s: dtype %d not supported", fn, dtype);
    DF_CHECK(fmt == DF_FMT_E4M3 || fmt == DF_FMT_E5M2, DF_ERR_INVALID, "%s: bad format %d", fn, fmt);
    DF_CHECK(scale_kind_ok(scale_kind), DF_ERR_INVALID, "%s: bad scale kind %d", fn, scale_kind);
    DF_CHECK(q || qt, DF_ERR_INVALID, "%s: neither row codes nor transposed ones are wanted", fn);
    DF_CHECK((!q || scales) && (!qt || scales_t), DF_ERR_INVALID, "%s: codes without their scales", fn);
    if (rows == 0 || cols == 0) return DF_OK;
    DF_CHECK(x, DF_ERR_INVALID, "%s: x is NULL", fn);
    DF_CHECK(ldx >= cols, DF_ERR_INVALID, "%s: ldx=%d < cols=%d", fn, ldx, cols);
    DF_CHECK(((uintptr_t)x & (dtype == DF_DTYPE_FLOAT32 ? 3u : 1u)) == 0, DF_ERR_ALIGN,
             "%s: x is not aligned to its elements", fn);
    DF_CHECK(!q || (ldq % 16 == 0 && ldq >= cols && aligned16(q)), DF_ERR_ALIGN,
             "%s: row codes need a leading dimension that is a multiple of 16 and >= %d, and 16-byte alignment", fn, cols);
    DF_CHECK(!qt || (ldqt % 16 == 0 && ldqt >= rows && aligned16(qt)), DF_ERR_ALIGN,
             "%s: transposed codes need a leading dimension that is a multiple of 16 and >= %d, and 16-byte alignment", fn,
             rows);
    const int sb = scale_bytes(scale_kind);
    DF_CHECK(!q || (ld_scales >= rows && (int64_t)ld_scales * sb % 16 == 0 && aligned16(scales)), DF_ERR_ALIGN,
             "%s: scales need a leading dimension of whole 16 bytes and >= %d, and 16-byte alignment", fn, rows);
    DF_CHECK(!qt || (ld_scales_t >= cols && (int64_t)ld_scales_t * sb % 16 == 0 && aligned16(scales_t)), DF_ERR_ALIGN,
             "%s: transposed scales need a leading dimension of whole 16 bytes and >= %d, and 16-byte alignment", fn, cols);
    const BlockQuant a{x, q, scales, qt, scales_t, rows, cols, ldx, ldq, ld_scales, ldqt, ld_scales_t};
    const bool e8 = scale_kind == DF_SCALE_E8M0;
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (fmt == DF_FMT_E4M3) launch<T, E4M3>(a, e8, square != 0, as_stream(stream));
        else launch<T, E5M2>(a, e8, square != 0, as_stream(stream));
    };
    if (dtype == DF_DTYPE_FLOAT32) go(float{});
    else if (dtype == DF_DTYPE_HALF) go(f16_t{});
    else go(uint16_t{});
    return launch_status(fn);
}
