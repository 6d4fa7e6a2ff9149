// gemm_experts.hpp -- what the experts' products share (gemm_experts.hip:
// entry points and small tiles; gemm_experts_tiles.hip: large tiles).
#pragma once

#include "df_common.hpp"
#include "gemm_common.hpp"

namespace dfk {

constexpr int kMaxExperts = 1024;

// One call.  ROWS: A [rows, lda], B [experts][N][ldb], C [rows, ldc], reduction K.
// SUMS: A [M, lda], B [N, ldb], C [experts][M][ldc], reduction over the tokens.
struct ExpertArgs {
    const uint8_t* A;
    const uint8_t* B;
    void* C;
    const int* off;
    const float* sa;
    const float* sb;
    int lda, ldb, ldc, rows, M, N, K, experts, vec_out;
};

// expert e's rows, whatever the offsets hold
__device__ __forceinline__ void expert_rows(const int* off, int e, int rows, int& lo, int& hi) {
    lo = min(max(off[e], 0), rows);
    hi = min(max(off[e + 1], lo), rows);
}

// The most tiles of `tile` rows that experts' rows take, dealt in any way.
// Offsets that overlap may give more, up to one of all rows per expert: tiles
// from here on are not worked on, and counts of them may pass 32 bits.
__host__ __device__ __forceinline__ int most_tiles(int rows, int experts, int tile) {
    return rows / tile + (experts < rows ? experts : rows);
}

// bytes of a dword at byte position `pos` that lie in [lo, hi)
__device__ __forceinline__ uint32_t keep_bytes(int pos, int lo, int hi) {
    const int a = min(max(lo - pos, 0), 4) * 8, b = min(max(hi - pos, 0), 4) * 8;
    const uint32_t upto = b == 32 ? ~0u : (1u << b) - 1u, below = a == 32 ? ~0u : (1u << a) - 1u;
    return upto & ~below;
}

typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

// eight codes -> bf16, exact
template <int FMT> __device__ __forceinline__ bf8 widen8(uint32_t lo, uint32_t hi) {
    bf2 p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t w = i < 2 ? lo : hi;
        if constexpr (FMT == E4M3)
            p[i] = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true)
                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
        else
            p[i] = i & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, true)
                         : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, 1.0f, false);
    }
    return bf8{p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
}

// gemm_experts_tiles.hip: the persistent kernel on 256 x 256 or 256 x 128
// tiles (vec_out: an epi_store_mode).
void launch_expert_tiles(int fmt_a, bool sums, bool narrow, int c_dtype, const ExpertArgs& g, int grid,
                         hipStream_t st);

}  // namespace dfk
