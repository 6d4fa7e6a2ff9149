// row_chunks.hpp -- what the norms share (layernorm.hip, rmsnorm.hip): rows read
// and written as 16-byte chunks at any element's address, and sums over the
// threads that share a row.
#pragma once

#include "df_common.hpp"

namespace dfk {

// ------------------------------------------------- 16-byte chunks of a row --
typedef float lf2 __attribute__((ext_vector_type(2)));
typedef __bf16 lbf2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_el __attribute__((aligned(2)));  // 16 bytes at element alignment

template <typename T> struct El;
template <> struct El<float> {
    static constexpr int E = 4;
    static __device__ __forceinline__ void widen(const u32x4 w, float* v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ u32x4 narrow(const float* v) {
        return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
    static __device__ __forceinline__ void put(float* p, float v) { *p = v; }
};
template <> struct El<uint16_t> {  // bf16 bits
    static constexpr int E = 8;
    static __device__ __forceinline__ void widen(const u32x4 w, float* v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ u32x4 narrow(const float* v) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(lf2{v[2 * i], v[2 * i + 1]}, lbf2));
        return w;
    }
    static __device__ __forceinline__ float one(const uint16_t* p) { return bf16_to_f32(*p); }
    static __device__ __forceinline__ void put(uint16_t* p, float v) { *p = (uint16_t)f32_to_bf16_rne(v); }
};
template <> struct El<f16_t> {
    static constexpr int E = 8;
    static __device__ __forceinline__ void widen(const u32x4 w, float* v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] & 0xFFFFu));
            v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[i] >> 16));
        }
    }
    static __device__ __forceinline__ u32x4 narrow(const float* v) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i]) |
                   ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v[2 * i + 1]) << 16);
        return w;
    }
    static __device__ __forceinline__ float one(const f16_t* p) {
        return (float)__builtin_bit_cast(_Float16, p->bits);
    }
    static __device__ __forceinline__ void put(f16_t* p, float v) {
        p->bits = __builtin_bit_cast(uint16_t, (_Float16)v);
    }
};

// Chunk j of a row of `cols` values at any element-aligned address, as one
// load: where the row ends inside it, the 16 bytes up to the row's end, which
// place_chunk() moves down when the values are used.  Put together from single
// values at the load, the last chunk made its wave wait for all loads under way,
// the next row's too: 16384 x 2500 bf16 took 128 us backward and 105
// forward, and takes 81 and 67 so (2496 columns: 79 and 66).  Rows at odd
// addresses alone cost nothing.  Plain loads: non-temporal ones drop the lines
// that neighbouring rows share (1000 x 771 bf16 backward 11.4 us against 8.6).
template <typename T> __device__ __forceinline__ u32x4 load_chunk(const T* row, int j, int cols) {
    constexpr int E = El<T>::E;
    const int c = j * E;
    u32x4 w = {0, 0, 0, 0};
    if (cols >= E) {
        // (a 32-bit offset on the row's address, the same for every tensor: rows below 4 GiB)
        const uint32_t at = (uint32_t)min(c, cols - E) * (uint32_t)sizeof(T);
        if (c < cols) w = *reinterpret_cast<const u32x4_el*>(reinterpret_cast<const char*>(row) + at);
    } else if (j == 0) {  // a row shorter than a chunk
#pragma unroll
        for (int e = 0; e < E - 1; ++e) {
            if (e < cols) {
                if constexpr (sizeof(T) == 4) w[e] = __builtin_bit_cast(uint32_t, row[e]);
                else w[e >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, row[e]) << (16 * (e & 1));
            }
        }
    }
    return w;
}

// chunk j as load_chunk() gave it, its values in their places; those past the
// row's end are 0
template <typename T> __device__ __forceinline__ u32x4 place_chunk(u32x4 w, int j, int cols) {
    constexpr int E = El<T>::E;
    const int over = j * E + E - cols;  // values past the row's end, if 1 to E - 1
    if (over <= 0 || over >= E || cols < E) return w;
    const int half = sizeof(T) == 4 ? 2 * over : over;  // 16-bit places to move, 1 to 7
    if (half & 4) w = u32x4{w[2], w[3], 0, 0};
    if (half & 2) w = u32x4{w[1], w[2], w[3], 0};
    if (half & 1)
        w = u32x4{w[0] >> 16 | w[1] << 16, w[1] >> 16 | w[2] << 16, w[2] >> 16 | w[3] << 16, w[3] >> 16};
    return w;
}

template <typename T> __device__ __forceinline__ void store_chunk(T* row, int j, int cols, const u32x4 w) {
    constexpr int E = El<T>::E;
    const int c = j * E;
    if (c + E <= cols) {
        *reinterpret_cast<u32x4_el*>(row + c) = w;
    } else if (c < cols) {
#pragma unroll
        for (int e = 0; e < E - 1; ++e) {
            if (c + e < cols) {
                if constexpr (sizeof(T) == 4) row[c + e] = __builtin_bit_cast(T, (uint32_t)w[e]);
                else row[c + e] = __builtin_bit_cast(T, (uint16_t)(w[e >> 1] >> (16 * (e & 1))));
            }
        }
    }
}

// sum over the wave by DPP: within rows of 16 lanes, then across them into lane
// 63 (half the time of a butterfly through LDS)
__device__ __forceinline__ float wave_add(float v) {
#define DF_DPP_ADD(CTRL) \
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true))
    DF_DPP_ADD(0x111);  // row_shr:1
    DF_DPP_ADD(0x112);  // row_shr:2
    DF_DPP_ADD(0x114);  // row_shr:4
    DF_DPP_ADD(0x118);  // row_shr:8: lane 15 of a row has the row's
    DF_DPP_ADD(0x142);  // row_bcast:15
    DF_DPP_ADD(0x143);  // row_bcast:31: lane 63 has the wave's
#undef DF_DPP_ADD
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// Sum over the RT threads that share a row, in a block of GP such groups.  For
// rows wider than a wave the waves' sums meet in LDS, in one of two slots in
// turn: a slot is written again only after the barrier of the call between,
// which every wave reaches after its reads of that slot.
template <int RT, int GP = 1> struct RowSum {
    float (*red)[2][GP][RT / 64];  // [slot][which][group][wave], LDS (unused for a wave's row)
    int slot = 0;
    __device__ __forceinline__ void two(float& a, float& b) {
        a = wave_add(a);
        b = wave_add(b);
        if constexpr (RT > 64) {
            const int gi = GP == 1 ? 0 : threadIdx.x / RT, w = (threadIdx.x % RT) >> 6;  // (uniform in a wave)
            if ((threadIdx.x & 63) == 0) {
                red[slot][0][gi][w] = a;
                red[slot][1][gi][w] = b;
            }
            __syncthreads();
            if constexpr (RT >= 1024) {
                // a wave's sums to a lane: all 32 in every lane took registers that
                // the backward spilled (12800 bf16 columns: 627 us against 333)
                const int l = threadIdx.x & 63;
                a = wave_add(l < RT / 64 ? red[slot][0][gi][l] : 0.0f);
                b = wave_add(l < RT / 64 ? red[slot][1][gi][l] : 0.0f);
            } else {
                a = b = 0.0f;
#pragma unroll
                for (int i = 0; i < RT / 64; ++i) {
                    a += red[slot][0][gi][i];
                    b += red[slot][1][gi][i];
                }
            }
            slot ^= 1;
        }
    }
    __device__ __forceinline__ float one(float a) {
        float b = 0.0f;
        two(a, b);
        return a;
    }
};

}  // namespace dfk
