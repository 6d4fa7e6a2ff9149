// gemm_common.hpp -- what the fp8 GEMM sources share (gemm_fp8.hip,
// gemm_small.hip, gemm_experts*.hip): operand and accumulator vector types, the output
// conversions, the bias loads and the arguments of one NT GEMM.
#pragma once

#include "df_common.hpp"

namespace dfk {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

template <typename T> struct OutCvt;
template <> struct OutCvt<float> {
    static __device__ __forceinline__ float cvt(float v) { return v; }
};
template <> struct OutCvt<uint16_t> {  // bf16 bits
    static __device__ __forceinline__ uint16_t cvt(float v) { return (uint16_t)f32_to_bf16_rne(v); }
};
template <> struct OutCvt<f16_t> {
    static __device__ __forceinline__ f16_t cvt(float v) { return f16_t{(uint16_t)f32_to_f16_rne(v)}; }
};
__device__ __forceinline__ float bias_ld(const float* b, int i) { return b[i]; }
__device__ __forceinline__ float bias_ld(const uint16_t* b, int i) { return bf16_to_f32(b[i]); }
__device__ __forceinline__ float bias_ld(const f16_t* b, int i) { return f16_to_f32(b[i].bits); }

// 4 consecutive outputs of one row: one 16-byte (fp32) or 8-byte (bf16) store
__device__ __forceinline__ void store4(float* p, const float* v) {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ void store4(uint16_t* p, const float* v) {
    *reinterpret_cast<u32x2*>(p) = u32x2{f32_to_bf16_rne(v[0]) | (f32_to_bf16_rne(v[1]) << 16),
                                        f32_to_bf16_rne(v[2]) | (f32_to_bf16_rne(v[3]) << 16)};
}
__device__ __forceinline__ void store4(f16_t* p, const float* v) {
    *reinterpret_cast<u32x2*>(p) = u32x2{f32_to_f16_rne(v[0]) | (f32_to_f16_rne(v[1]) << 16),
                                        f32_to_f16_rne(v[2]) | (f32_to_f16_rne(v[3]) << 16)};
}

// ---- what the persistent kernels share ----
constexpr int kGroupM = 8;             // tile rows of a group of the tile order
constexpr int kPBM = 256, kPBN = 256;  // persistent block tile
constexpr int kPKB = 128;              // K bytes per DMA step
constexpr int kPStage = (kPBM + kPBN) * kPKB;
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pack_bf16_rne(float a, float b) {
    const v2f f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, v2bf));
}

// s_waitcnt immediate (gfx9 encoding): vmcnt(n), lgkmcnt(0), no expcnt wait
__device__ __forceinline__ constexpr int waitcnt_vm_lgkm0(int n) {
    return (n & 15) | ((n >> 4) << 14) | 0x70;
}

// The lane index, computed afresh where it is called.  The asm is opaque to
// the optimiser, so offsets derived from it stay where they are used: taken
// from threadIdx, the epilogue's per-lane offsets were hoisted out of the
// tile loop and, at the main loop's register pressure, spilled; each reload
// in the epilogue then waited on vmcnt(0), i.e. for the DMA in flight.
__device__ __forceinline__ int fresh_lane() {
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
    return l;
}

// Epilogue geometry for an output element of ES bytes: each 32-row block of
// a wave's FMR*32 x 64 part passes through an LDS slab of SR rows.
template <int ES, int FMR = 4>
struct EpiGeom {
    static constexpr int SR = ES == 2 ? 16 : 8;          // slab rows
    static constexpr int SROW = 64 * ES + 16;            // padded slab row (bytes)
    static constexpr int SLAB = SR * SROW;
    static constexpr int NPASS = 32 / SR;                // slab passes per 32-row block
    static constexpr int SPP = SR * 64 * ES / 1024;      // 16-byte stores per lane per pass
    static constexpr int NST = FMR * NPASS * SPP;        // epilogue stores per wave
};

// Store mode of the persistent kernel's epilogue: 0 element stores, 1
// 16-byte stores, 2 16-byte non-temporal stores.  One store instruction
// writes whole 64-column row segments (128 bytes of bf16, 256 of fp32);
// non-temporal stores are kept to rows that start on a 128-byte boundary, so
// that no cache line is written in parts by several non-temporal stores (in
// a probe that did so -- 8-byte non-temporal stores -- one output of sixteen
// came back different, where plain stores matched).
inline int epi_store_mode(const void* C, int64_t ldc_bytes) {
    if (ldc_bytes % 16 != 0 || !aligned16(C)) return 0;
    return (ldc_bytes % 128 == 0 && ((uintptr_t)C & 127u) == 0) ? 2 : 1;
}

template <typename T> struct Tag { using type = T; };

struct GemmArgs {
    const uint8_t* A; int lda;
    const uint8_t* B; int ldb;
    int M, N, K;
    const float* sa; const float* sb;
    const void* bias; void* C; int ldc;
    float* ws; size_t ws_bytes;
    hipStream_t st;
};

// The rounds cost model's unit, a 128-byte K step of a 256x256 tile, in
// microseconds on a partly filled chip (one or two rounds: 1.4-2.0 measured;
// the low end, so that the persistent kernel is left only where it is slower).
constexpr double kStepUs = 1.5;

// gemm_small.hip: the kernel on 16*mt x 16*nt tiles whose `waves` waves share
// the reduction, and the best such tiling of one GEMM (cost in steps).
struct SmallPlan {
    int mt, nt, waves;
    double cost;
};
SmallPlan small_plan(int M, int N, int K, int cus);
void launch_small(const SmallPlan& p, int fmt_a, int fmt_b, int bias_dtype, int c_dtype, const GemmArgs& g);

}  // namespace dfk
