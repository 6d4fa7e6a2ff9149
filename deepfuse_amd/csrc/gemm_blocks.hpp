// gemm_blocks.hpp -- what the products with a scale per 128 of the reduction share
// (gemm_blocks.hip: entry point, plan and small tiles; gemm_blocks_tiles.hip: large
// tiles).
#pragma once

#include "block_scale.hpp"
#include "df_common.hpp"
#include "gemm_common.hpp"

namespace dfk {

// C [M, ldc] = sum over blocks b of sa[b][m] * sb[b][n] * (A . B^T over block b) + bias;
// A [M, lda], B [N, ldb], K rounded up to 16, scales [blocks][ldsa / ldsb].
struct BlocksArgs {
    const uint8_t* A;
    const uint8_t* B;
    void* C;
    const void* sa;
    const void* sb;
    const void* bias;
    int lda, ldb, ldc, ldsa, ldsb, M, N, K, bias_dtype, vec_out;
};

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

// eight codes -> bf16, times the power of two `scale` (exact while the result is
// in bf16's range)
template <int FMT> __device__ __forceinline__ bf8 widen8_scaled(uint32_t lo, uint32_t hi, float scale) {
    bf2 p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? lo : hi;
        if constexpr (FMT == E4M3)
            p[i] = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true)
                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
        else
            p[i] = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, true)
                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, false);
    }
    return bf8{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
}

// fp32 scales.  A step's product p of 128 codes is 0 or 2^-25 to 2^32 in size: p * sb is in
// binary32's normal range unless B's scale is far (0 is not), and so is sa * sb if both lie
// in the middle.  A fused multiply-add with the other factor then rounds once.  Products at
// far scales take binary64, which holds all three factors'.
__device__ __forceinline__ bool scale_far(uint32_t bits) {  // not 0 nor 2^-100 .. 2^95, infinities and NaN too
    constexpr uint32_t least = 27u << 23, most = 222u << 23;
    bits &= 0x7FFFFFFFu;
    return bits != 0u && bits - least > most - least;
}
__device__ __forceinline__ bool scale_in_the_middle(uint32_t bits) {  // 2^-62 .. 2^62, positive
    constexpr uint32_t least = 65u << 23, most = 189u << 23;
    return bits - least <= most - least;
}
__device__ __forceinline__ float add_scaled_far(float p, float sa, float sb, float acc) {
    return (float)__builtin_fma((double)p * (double)sa, (double)sb, (double)acc);
}

// bytes of `blocks` blocks' scales of a matrix of `rows` rows: what may be read
inline int64_t scales_extent(int64_t blocks, int64_t ld, int64_t rows, int bytes) {
    const int64_t row = (rows * bytes + 15) & ~(int64_t)15;
    return blocks == 0 ? 0 : (blocks - 1) * ld * bytes + row;
}

__device__ __forceinline__ float bias_at(const void* bias, int dtype, int i) {
    if (dtype == DF_DTYPE_FLOAT32) return bias_ld(static_cast<const float*>(bias), i);
    if (dtype == DF_DTYPE_HALF) return bias_ld(static_cast<const f16_t*>(bias), i);
    return bias_ld(static_cast<const uint16_t*>(bias), i);
}

// gemm_blocks_tiles.hip: the persistent kernel on 256 x 256 (fm 4, power-of-two
// scales only), 256 x 128 (2) or 128 x 128 tiles (1); vec_out: an epi_store_mode.
void launch_block_tiles(int fmt_a, bool e8, int fm, int c_dtype, const BlocksArgs& g, int extent_a, int extent_b, int grid,
                        hipStream_t st);

}  // namespace dfk
