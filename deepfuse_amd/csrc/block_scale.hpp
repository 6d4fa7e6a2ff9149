// block_scale.hpp -- fp8 codes with a scale per 128 values: the scales' two
// kinds and the encoders that quantize at them (quant_blocks.hip, rmsnorm.hip),
// and the scales as the products read them (gemm_blocks*.hip, moe.hip).
//
// A scale is fp32, absmax / fmax as for a whole tensor, or a power of two kept
// as its biased exponent, one byte: 2^(byte - 127), the smallest that keeps
// absmax / s within fmax.  A power of two costs no precision (codes are floating
// point: it moves their range, by less than one binade), multiplies exactly, and
// is what the matrix instructions apply by themselves.
#pragma once

#include "df_common.hpp"

namespace dfk {

constexpr int kScaleBlock = 128;  // values that share a scale

inline bool scale_kind_ok(int kind) { return kind == DF_SCALE_F32 || kind == DF_SCALE_E8M0; }
inline int scale_bytes(int kind) { return kind == DF_SCALE_F32 ? 4 : 1; }

// The byte for an absmax given as its binary32 pattern (finite): fmax is 1.75 *
// 2^8 (e4m3) or 1.75 * 2^15.  Below 2^-126 the exponent field is 0, and so is
// the byte; 0 itself gives scale 1.
template <int FMT> __device__ __forceinline__ uint32_t e8m0_of(uint32_t absmax) {
    constexpr int top = FMT == E4M3 ? 8 : 15;
    const int b = (int)(absmax >> 23) - top + ((absmax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return absmax == 0u ? 127u : (uint32_t)max(b, 0);
}
// 2^(127 - byte) of a byte that e8m0_of gives (at most 247)
__device__ __forceinline__ float e8m0_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ float e8m0_value(uint32_t byte) {
    return __uint_as_float(byte != 0u ? byte << 23 : 0x00400000u);
}

// What to quantize a block at: its scale and the reciprocal.  E8: the byte is
// left in `byte`, and x / s is x * r, exactly.
struct BlockDiv {
    QDiv d;
    uint32_t byte;
};
template <int FMT, bool E8> __device__ __forceinline__ BlockDiv block_div(uint32_t absmax) {
    BlockDiv b;
    if constexpr (E8) {
        b.byte = e8m0_of<FMT>(absmax);
        b.d.s = e8m0_value(b.byte);
        b.d.r = e8m0_inverse(b.byte);
        b.d.fast = true;
    } else {
        b.byte = 0;
        b.d = make_qdiv(absmax == 0u ? 1.0f : __uint_as_float(absmax) / Fp8<FMT>::fmax);
    }
    return b;
}

// Four values to four codes, a zero's being zero at any scale.  PLAIN: none is NaN and (fp32 scales) the division
// is in its fast range; the caller asks for a whole wave at once.
template <int FMT, bool E8, bool PLAIN>
__device__ __forceinline__ uint32_t block_quant4(const float* v, const QDiv& q) {
    if constexpr (!E8) {
        if constexpr (PLAIN) {
            return quant4_nonan<FMT>(v[0], v[1], v[2], v[3], q);
        } else {
            // (absmax / fmax is 0 below 2^-150 fmax, and 0 / 0 NaN: the zero itself then, as a
            // NaN is its own quotient)
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = qdiv(v[i], q);
                x[i] = x[i] != x[i] ? v[i] : x[i];
            }
            return encode2_hw<FMT>(x[0], x[1]) | (encode2_hw<FMT>(x[2], x[3]) << 16);
        }
    } else if constexpr (PLAIN) {
        constexpr float fm = Fp8<FMT>::fmax;
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_fmed3f(v[i] * q.r, -fm, fm);
        if constexpr (FMT == E4M3)
            return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false),
                                                             true);
        else
            return (uint32_t)__builtin_amdgcn_cvt_pk_bf8_f32(x[2], x[3], __builtin_amdgcn_cvt_pk_bf8_f32(x[0], x[1], 0, false),
                                                             true);
    } else {
        return encode2_hw<FMT>(v[0] * q.r, v[1] * q.r) | (encode2_hw<FMT>(v[2] * q.r, v[3] * q.r) << 16);
    }
}

// the maximum over 16 lanes (a DPP row), in each of them
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
#define DF_ROR_MAX(CTRL) v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true))
    DF_ROR_MAX(0x128);  // row_ror:8
    DF_ROR_MAX(0x124);
    DF_ROR_MAX(0x122);
    DF_ROR_MAX(0x121);
#undef DF_ROR_MAX
    return v;
}

}  // namespace dfk
