// gemm_experts_tiles.hip -- the experts' products (gemm_experts.hip) on
// 256 x 256 or 256 x 128 tiles: one persistent block per CU of eight waves,
// two per SIMD, each owning 128 x 64 (or 64 x 64) of the tile in fp32
// accumulators, operands by LDS DMA through two 64 KiB stages, as the
// persistent kernel of gemm_fp8.hip.  What differs:
//  - Which tiles there are is known only on the device.  ROWS: every block
//    first counts the experts' row tiles into LDS (a scan over the experts,
//    about 2 us once) and finds the expert of a tile there, two ballots deep.
//    SUMS: all experts have the same tiles, of different reductions.
//  - Operand buffers are set up per tile at the tile's first row (and its
//    expert's weights), so a tile's rows past its expert's end read as zero,
//    and no operand is too large for 32-bit buffer offsets.
//  - SUMS reduce over an expert's tokens, which start and end at any byte:
//    K steps start at the multiple of 128 below, 16-byte chunks outside the
//    range are not loaded, and the bytes of the neighbouring experts in the
//    two edge chunks are cleared in LDS, by one thread per operand row, before
//    the step is read.
//  - WIDE (fp32 outputs): fragments are widened to bf16 in registers and
//    multiplied by v_mfma_f32_32x32x16_bf16; see gemm_experts.hip for why.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "gemm_experts.hpp"

namespace dfk {

namespace {

// What a call reads at uniform indexes and nothing writes meanwhile: through
// the constant address space, by scalar loads, which do not wait for the DMA
// under way as vector loads would.
template <typename T> using Fixed = const __attribute__((address_space(4))) T*;
template <typename T> __device__ __forceinline__ Fixed<T> fixed(const T* p) { return (Fixed<T>)(uintptr_t)p; }

__device__ __forceinline__ void fixed_rows(const ExpertArgs& g, int e, int& lo, int& hi) {
    const Fixed<int> off = fixed(g.off);
    lo = min(max(off[e], 0), g.rows);
    hi = min(max(off[e + 1], lo), g.rows);
}

// Block-wide: tiles of 256 rows before each expert, into first[0..kMaxExperts]
// (INT_MAX behind the last).  Sums stay at kCountCap, so that overlapping offsets
// do not wrap them: each is right up to there, past most_tiles() (below 2^24).
constexpr int kCountCap = 0x3FFFFFFF;
__device__ __forceinline__ void count_tiles(const ExpertArgs& g, int* first, int* waves) {
    const int t = threadIdx.x, lane = t & 63, w = t >> 6;
    int c[2], sum = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int e = 2 * t + i;
        c[i] = 0;
        if (e < g.experts) {
            int a, b;
            expert_rows(g.off, e, g.rows, a, b);
            c[i] = (b - a + kPBM - 1) / kPBM;
        }
        sum += c[i];
    }
    int s = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(s, off, 64);
        if (lane >= off) s = min(s + o, kCountCap);
    }
    if (lane == 63) waves[w] = s;
    __syncthreads();
    for (int i = 0; i < w; ++i) s = min(s + waves[i], kCountCap);
    int at = s - sum;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int e = 2 * t + i;
        first[e] = e <= g.experts ? at : 0x7FFFFFFF;
        at += c[i];
    }
    if (t == 511) first[kMaxExperts] = g.experts == kMaxExperts ? at : 0x7FFFFFFF;
    __syncthreads();
}
static_assert(kMaxExperts == 2 * 512, "two experts per thread");

// the expert whose tiles hold row tile v: how many of first[1..] are <= v
__device__ __forceinline__ int find_expert(const int* first, int v, int lane) {
    const int n1 = __builtin_popcountll(__builtin_amdgcn_ballot_w64(first[16 * (lane + 1)] <= v));
    const uint64_t m = __builtin_amdgcn_ballot_w64(first[min(16 * n1 + lane + 1, kMaxExperts)] <= v);
    return 16 * n1 + __builtin_popcountll(m & 0xFFFFull);
}

typedef u32x4 u32x4_el __attribute__((aligned(2)));

template <int FA, int FB, typename OutT, bool SUMS, bool WIDE, bool NARROW>
__global__ __launch_bounds__(512, 1) void experts_tile_kernel(const ExpertArgs g) {
    constexpr int FM = NARROW ? 2 : 4, FN = 2;    // 32x32 MFMA tiles per wave
    constexpr int BN = NARROW ? 128 : kPBN;       // tile columns
    constexpr int WR = 32 * FM;                   // rows of a wave's part
    constexpr int NDA = 4, NDB = NARROW ? 2 : 4;  // A and B DMA instructions per wave and step
    constexpr int NF = FM + FN;
    using G = EpiGeom<(int)sizeof(OutT), FM>;
    constexpr int W_AFTER = G::NST > 63 ? 63 : G::NST;
    constexpr uint32_t kOOB = 0x80000000u;
    constexpr int kTable = SUMS ? 0 : 4 * (kMaxExperts + 1);
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * kPStage + 8 * G::SLAB + kTable];
    int* const first = reinterpret_cast<int*>(lds + 2 * kPStage + 8 * G::SLAB);  // [kMaxExperts + 1]

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = NARROW ? w >> 1 : w >> 2, wn = NARROW ? w & 1 : w & 3;
    uint8_t* const slab = lds + 2 * kPStage + w * G::SLAB;
    const int tiles_n = (g.N + BN - 1) / BN;
    const int tiles_m = SUMS ? (g.M + kPBM - 1) / kPBM : 0;
    if constexpr (!SUMS) count_tiles(g, first, reinterpret_cast<int*>(lds));
    const int nunits = SUMS ? g.experts * tiles_m * tiles_n
                            : min(__builtin_amdgcn_readfirstlane(first[g.experts]),
                                  most_tiles(g.rows, g.experts, kPBM)) * tiles_n;

    const int P = gridDim.x;
    const int q = P >> 3, rr = P & 7;
    const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
    const int bl = xcd < rr ? xcd * (q + 1) + idx : rr * (q + 1) + (xcd - rr) * q + idx;
    const int my_units = bl < nunits ? (nunits - bl + P - 1) / P : 0;
    if (my_units == 0) return;  // before any DMA; the whole block

    // unit r of this block: its expert, first row and column, the rows' end
    // (SUMS: M), and the reduction: steps of 128 from kb over bytes [k_lo, k_hi)
    struct Unit {
        int e, m0, mend, n0, kb, k_lo, k_hi, steps;
    };
    auto unit_of = [&](int r) {
        Unit u;
        const int n = bl + r * P;
        int tm_count, local;
        if constexpr (SUMS) {
            const int per = tiles_m * tiles_n;
            u.e = n / per;
            local = n - u.e * per;
            tm_count = tiles_m;
        } else {
            u.e = __builtin_amdgcn_readfirstlane(find_expert(first, n / tiles_n, lane));
            const int f = __builtin_amdgcn_readfirstlane(first[u.e]);
            tm_count = __builtin_amdgcn_readfirstlane(first[u.e + 1]) - f;
            local = n - f * tiles_n;
        }
        const int per_group = kGroupM * tiles_n;
        const int group = local / per_group;
        const int first_m = group * kGroupM;
        const int gsize = min(tm_count - first_m, kGroupM);
        const int in_group = local - group * per_group;
        u.m0 = (first_m + in_group % gsize) * kPBM;
        u.n0 = (in_group / gsize) * BN;
        if constexpr (SUMS) {
            u.mend = g.M;
            fixed_rows(g, u.e, u.k_lo, u.k_hi);
            u.kb = u.k_lo & ~(kPKB - 1);
        } else {
            int lo;
            fixed_rows(g, u.e, lo, u.mend);
            u.m0 += lo;
            u.k_lo = u.kb = 0;
            u.k_hi = g.K;
        }
        u.steps = max((u.k_hi - u.kb + kPKB - 1) / kPKB, 1);  // no reduction: one step of zeros
        return u;
    };

    // ---- DMA, as in gemm_fp8.hip: instruction d of wave w fills rows
    // (w*4+d)*8 + lane/8 of the stage's A (and (w*NDB+d)*8 + lane/8 of its B)
    // part, 16-byte chunk c of row r in slot c ^ ((r >> 1) & 7).  The cursor
    // (unit d_u, step d_k) runs two steps ahead of the products, across units.
    const int drow = lane >> 3;
    const int dch0 = ((lane & 7) ^ (lane >> 4)) << 4;
    const int dch1 = dch0 ^ 64;
    int d_unit = 0, d_k = 0, d_g = 0;
    Unit du = unit_of(0);
    __amdgpu_buffer_rsrc_t rA, rB;
    auto operands = [&]() {
        rA = __builtin_amdgcn_make_buffer_rsrc((void*)(g.A + (int64_t)du.m0 * g.lda), (short)0,
                                               min(du.mend - du.m0, kPBM) * g.lda, 0x00020000);
        rB = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(g.B + ((SUMS ? 0 : (int64_t)du.e * g.N) + du.n0) * g.ldb), (short)0, min(g.N - du.n0, BN) * g.ldb,
            0x00020000);
    };
    operands();
    uint32_t oa0, oa1, ob0, ob1;
    // SUMS: the edge chunks of the step in stage s that need clearing: bits
    // 0..3 first byte to keep of chunk 4..6 (bit 7: there is one), 8..11 first
    // byte not to keep of chunk 12..14 (bit 15)
    int edge0 = 0, edge1 = 0;
    auto dprep = [&]() {
        const bool live = d_unit < my_units;
        const int k0 = du.kb + d_k * kPKB + dch0, k1 = du.kb + d_k * kPKB + dch1;
        const bool in0 = live && k0 < du.k_hi && (!SUMS || k0 + 16 > du.k_lo);
        const bool in1 = live && k1 < du.k_hi && (!SUMS || k1 + 16 > du.k_lo);
        const uint32_t ra = (uint32_t)(w * 32 + drow), rb = (uint32_t)(w * 8 * NDB + drow);
        oa0 = in0 ? ra * (uint32_t)g.lda + (uint32_t)k0 : kOOB;
        oa1 = in1 ? (ra + 8u) * (uint32_t)g.lda + (uint32_t)k1 : kOOB;
        ob0 = in0 ? rb * (uint32_t)g.ldb + (uint32_t)k0 : kOOB;
        ob1 = in1 ? (rb + 8u) * (uint32_t)g.ldb + (uint32_t)k1 : kOOB;
        if constexpr (SUMS) {
            int x = 0;
            if (live && d_k == 0 && (du.k_lo & 15)) x |= 0x80 | (du.k_lo & 15) | (((du.k_lo >> 4) & 7) << 4);
            if (live && d_k == du.steps - 1 && (du.k_hi & 15))
                x |= 0x8000 | ((du.k_hi & 15) << 8) | (((du.k_hi >> 4) & 7) << 12);
            if (d_g & 1) edge1 = x;
            else edge0 = x;
        }
    };
    auto dissue_one = [&](int k) __attribute__((always_inline)) {
        uint8_t* base = lds + ((uint32_t)d_g & 1u) * kPStage;
        if (k < NDA)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rA, (__attribute__((address_space(3))) void*)(base + (w * 4 + k) * 1024), 16,
                ((k & 1) ? oa1 : oa0) + (uint32_t)(k >> 1) * 16u * (uint32_t)g.lda, 0, 0, 0);
        else
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rB, (__attribute__((address_space(3))) void*)(base + kPBM * kPKB + (w * NDB + k - NDA) * 1024), 16,
                (((k - NDA) & 1) ? ob1 : ob0) + (uint32_t)((k - NDA) >> 1) * 16u * (uint32_t)g.ldb, 0, 0, 0);
    };
    auto dadvance = [&]() {
        if (d_unit < my_units && ++d_k == du.steps) {
            d_k = 0;
            if (++d_unit < my_units) {
                du = unit_of(d_unit);
                operands();
            }
        }
        ++d_g;
        dprep();
    };
    // clears the neighbours' bytes of a step's edge chunks; thread t: row t of
    // the stage (A's 256, then B's)
    auto clear_edges = [&](int x, int stage) {
        if (threadIdx.x < kPBM + BN) {
            uint8_t* row = lds + stage * kPStage + threadIdx.x * kPKB;
            const int sw = (threadIdx.x >> 1) & 7;
            if (x & 0x80) {
                u32x4* p = reinterpret_cast<u32x4*>(row + ((((x >> 4) & 7) ^ sw) << 4));
                u32x4 v = *p;
#pragma unroll
                for (int d = 0; d < 4; ++d) v[d] &= keep_bytes(4 * d, x & 15, 16);
                *p = v;
            }
            if (x & 0x8000) {
                u32x4* p = reinterpret_cast<u32x4*>(row + ((((x >> 12) & 7) ^ sw) << 4));
                u32x4 v = *p;
#pragma unroll
                for (int d = 0; d < 4; ++d) v[d] &= keep_bytes(4 * d, 0, (x >> 8) & 15);
                *p = v;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    };

    // ---- fragments: lane l supplies row l%32 and K bytes 32*(l/32) .. +32 of
    // each 64: chunks 4e + 2*(l/32) and the next of K-half e
    const int fr = lane & 31;
    const int fsw = (fr >> 1) & 7;
    const int c0 = (lane >> 5) * 2;
    int foff[2][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        foff[e][0] = fr * kPKB + (((4 * e + c0) ^ fsw) << 4);
        foff[e][1] = fr * kPKB + (((4 * e + c0 + 1) ^ fsw) << 4);
    }
    // 16 bytes of fragment f (the wave's FM row blocks, then its FN column blocks)
    auto rd = [&](int stage, int f, int e, int h) -> u32x4 {
        const uint8_t* p = lds + stage * kPStage +
                           (f < FM ? (wm * WR + f * 32) * kPKB : (kPBM + wn * 64 + (f - FM) * 32) * kPKB);
        return *reinterpret_cast<const u32x4*>(p + foff[e][h]);
    };

    v16f acc[FM][FN];
    int after_epi = 0, c_g = 0;  // c_g: the step whose products are under way

    // Before the first read of step c_g + 1: this wave's part of it has landed
    // (after an epilogue its stores may still be under way: they were issued
    // later), then every wave's, and its edges are cleared.  Every wave has read
    // the last of step c_g, so the DMA of step c_g + 2 may go over it.
    auto next_step = [&]() __attribute__((always_inline)) {
        if (after_epi == 1) __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(W_AFTER));
        else __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(0));
        after_epi = 0;
        __builtin_amdgcn_s_barrier();
        if constexpr (SUMS) {
            const int x = (c_g + 1) & 1 ? edge1 : edge0;
            if (x) clear_edges(x, (c_g + 1) & 1);
        }
    };

    // ---- fp8 products: half-steps of 64 bytes; the MFMAs on (fa, fb) while
    // the next half-step's fragments are read into (na, nb); the order frozen
    // as in gemm_fp8.hip (reads under the first four MFMAs, the DMA of odd
    // half-steps spread over all)
    auto half = [&](auto zero, auto odd, v8i* fa, v8i* fb, v8i* na, v8i* nb) __attribute__((always_inline)) {
        constexpr bool ODD = decltype(odd)::value;
        __builtin_amdgcn_sched_barrier(0);
        if (ODD) next_step();
        const int stage = (ODD ? c_g + 1 : c_g) & 1;
        constexpr int NR = 2 * NF;
        u32x4 part[NR];
#pragma unroll
        for (int x = 0; x < FM * FN; ++x) {
            const int i = x >> 1, j = x & 1;
            if (decltype(zero)::value) {
                const v16f z = {};
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[j], fa[i], z, FB, FA, 0, 0, 0, 0);
            } else {
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[j], fa[i], acc[i][j], FB, FA, 0, 0,
                                                                            0, 0);
            }
            if (x < 4) {
#pragma unroll
                for (int r = (NR / 4) * x; r < (NR / 4) * (x + 1); ++r) part[r] = rd(stage, r >> 1, ODD ? 0 : 1, r & 1);
            }
            if (ODD) {
                if (NARROW) {
                    if (2 * x < NDA + NDB) dissue_one(2 * x);
                    if (2 * x + 1 < NDA + NDB) dissue_one(2 * x + 1);
                } else {
                    dissue_one(x);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const u32x4 lo = part[2 * f], hi = part[2 * f + 1];
            v8i r;
            r[0] = (int)lo.x; r[1] = (int)lo.y; r[2] = (int)lo.z; r[3] = (int)lo.w;
            r[4] = (int)hi.x; r[5] = (int)hi.y; r[6] = (int)hi.z; r[7] = (int)hi.w;
            if (f < FM) na[f] = r; else nb[f - FM] = r;
        }
        if (ODD) {
            ++c_g;
            dadvance();
        }
    };

    // ---- bf16 products: quarter-steps of 16 bytes per lane (32 of K); a
    // quarter's codes are widened eight at a time, the next quarter's read
    auto quarter = [&](auto zero, auto qq, const u32x4* cur, u32x4* nxt) __attribute__((always_inline)) {
        constexpr int Q = decltype(qq)::value;
        __builtin_amdgcn_sched_barrier(0);
        if (Q == 3) next_step();
        const int stage = (Q == 3 ? c_g + 1 : c_g) & 1;
#pragma unroll
        for (int f = 0; f < NF; ++f) nxt[f] = rd(stage, f, ((Q + 1) >> 1) & 1, (Q + 1) & 1);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            bf8 wb[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) wb[j] = widen8<FB>(cur[FM + j][2 * s], cur[FM + j][2 * s + 1]);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                const bf8 wa = widen8<FA>(cur[i][2 * s], cur[i][2 * s + 1]);
#pragma unroll
                for (int j = 0; j < FN; ++j) {
                    if (decltype(zero)::value && s == 0) {
                        const v16f z = {};
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j], wa, z, 0, 0, 0);
                    } else {
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j], wa, acc[i][j], 0, 0, 0);
                    }
                    const int x = (s * FM + i) * FN + j;
                    if (Q == 3 && x < NDA + NDB) dissue_one(x);
                }
            }
        }
        if (Q == 3) {
            ++c_g;
            dadvance();
        }
    };

    // Stores a finished unit: scale and conversion in registers, then each
    // 32-row block through the wave's LDS slab and out as 16-byte stores of
    // whole row segments (vec_out 2: non-temporal; see epi_store_mode).  Whether the wave's part
    // lay wholly inside the output, i.e. whether it issued all its stores.
    auto store_unit = [&](const Unit& u, float sab) __attribute__((always_inline)) -> bool {
        constexpr int ES = (int)sizeof(OutT);
        OutT* const C = static_cast<OutT*>(g.C) + (SUMS ? (int64_t)u.e * g.M * g.ldc : 0);
        const int el = fresh_lane(), efr = el & 31;
        const int rowb = u.m0 + wm * WR, colw = u.n0 + wn * 64;
        const int h4 = (el >> 5) * 4;
        constexpr int CPR = 64 * ES / 16;
        constexpr int RPS = 64 / CPR;
        const int srow = el / CPR, rc = el % CPR;
        const int scol = colw + rc * (16 / ES);
        const bool col_full = scol + 16 / ES <= g.N;
        const int my_sr = efr % G::SR, my_pass = efr / G::SR;
        typedef typename std::conditional<ES == 2, u32x2, f32x4>::type Pk;
        // LDS operations of one wave execute in order, so a pass's reads see
        // its writes and precede the next pass's writes; the empty asm
        // statements keep the compiler from reordering them.
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            Pk pk[FN][4];
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const v16f& a = acc[i][j];
                    const float v0 = a[4 * x] * sab, v1 = a[4 * x + 1] * sab, v2 = a[4 * x + 2] * sab,
                                v3 = a[4 * x + 3] * sab;
                    if constexpr (std::is_same<OutT, f16_t>::value)
                        pk[j][x] = u32x2{f32_to_f16_rne(v0) | (f32_to_f16_rne(v1) << 16),
                                         f32_to_f16_rne(v2) | (f32_to_f16_rne(v3) << 16)};
                    else if constexpr (ES == 2)
                        pk[j][x] = u32x2{pack_bf16_rne(v0, v1), pack_bf16_rne(v2, v3)};
                    else
                        pk[j][x] = f32x4{v0, v1, v2, v3};
                }
#pragma unroll
            for (int p = 0; p < G::NPASS; ++p) {
                if (my_pass == p) {
#pragma unroll
                    for (int j = 0; j < FN; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            *reinterpret_cast<Pk*>(slab + my_sr * G::SROW + (j * 32 + 8 * x + h4) * ES) = pk[j][x];
                }
                asm volatile("" ::: "memory");
#pragma unroll
                for (int s = 0; s < G::SPP; ++s) {
                    const int sr = s * RPS + srow;
                    const u32x4 val = *reinterpret_cast<const u32x4*>(slab + sr * G::SROW + rc * 16);
                    const int row = rowb + i * 32 + p * G::SR + sr;
                    if (row < u.mend) {
                        OutT* dst = C + (int64_t)row * g.ldc + scol;
                        if (col_full) {
                            // rows at any element's boundary: 16-byte stores all the same
                            if (g.vec_out == 2) __builtin_nontemporal_store(val, reinterpret_cast<u32x4*>(dst));
                            else *reinterpret_cast<u32x4_el*>(dst) = val;
                        } else {
                            const OutT* ev = reinterpret_cast<const OutT*>(&val);
#pragma unroll
                            for (int x = 0; x < 16 / ES; ++x)
                                if (scol + x < g.N) dst[x] = ev[x];
                        }
                    }
                }
                asm volatile("" ::: "memory");
            }
        }
        return rowb + WR <= u.mend && colw + 64 <= g.N;
    };

    // prologue: DMA steps 0 and 1; step 0's first fragments
    dprep();
    const int edge_first = edge0;
    for (int k = 0; k < NDA + NDB; ++k) dissue_one(k);
    dadvance();
    for (int k = 0; k < NDA + NDB; ++k) dissue_one(k);
    dadvance();
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(NDA + NDB));
    __builtin_amdgcn_s_barrier();
    if constexpr (SUMS) {
        if (edge_first) clear_edges(edge_first, 0);
    }

    using Z = std::true_type;
    using NZ = std::false_type;
    const float sa = fixed(g.sa)[0];
    if constexpr (WIDE) {
        u32x4 r0[NF], r1[NF];
        for (int f = 0; f < NF; ++f) r0[f] = rd(0, f, 0, 0);
        using Q0 = std::integral_constant<int, 0>;
        using Q1 = std::integral_constant<int, 1>;
        using Q2 = std::integral_constant<int, 2>;
        using Q3 = std::integral_constant<int, 3>;
        for (int r = 0; r < my_units; ++r) {
            const Unit u = unit_of(r);
            quarter(Z{}, Q0{}, r0, r1);
            quarter(NZ{}, Q1{}, r1, r0);
            quarter(NZ{}, Q2{}, r0, r1);
            quarter(NZ{}, Q3{}, r1, r0);
            for (int k = 1; k < u.steps; ++k) {
                quarter(NZ{}, Q0{}, r0, r1);
                quarter(NZ{}, Q1{}, r1, r0);
                quarter(NZ{}, Q2{}, r0, r1);
                quarter(NZ{}, Q3{}, r1, r0);
            }
            after_epi = store_unit(u, sa * fixed(g.sb)[SUMS ? 0 : u.e]) ? 1 : 2;
        }
    } else {
        v8i fa0[FM], fb0[FN], fa1[FM], fb1[FN];
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const u32x4 lo = rd(0, f, 0, 0), hi = rd(0, f, 0, 1);
            v8i r;
            r[0] = (int)lo.x; r[1] = (int)lo.y; r[2] = (int)lo.z; r[3] = (int)lo.w;
            r[4] = (int)hi.x; r[5] = (int)hi.y; r[6] = (int)hi.z; r[7] = (int)hi.w;
            if (f < FM) fa0[f] = r; else fb0[f - FM] = r;
        }
        for (int r = 0; r < my_units; ++r) {
            const Unit u = unit_of(r);
            half(Z{}, NZ{}, fa0, fb0, fa1, fb1);
            half(NZ{}, Z{}, fa1, fb1, fa0, fb0);
            for (int k = 1; k < u.steps; ++k) {
                half(NZ{}, NZ{}, fa0, fb0, fa1, fb1);
                half(NZ{}, Z{}, fa1, fb1, fa0, fb0);
            }
            after_epi = store_unit(u, sa * fixed(g.sb)[SUMS ? 0 : u.e]) ? 1 : 2;
        }
    }
    __builtin_amdgcn_s_waitcnt(0);  // every DMA has landed before the block's LDS is released
}

template <int FA, bool SUMS, bool NARROW> void launch(int c_dtype, const ExpertArgs& g, int grid, hipStream_t st) {
    if (c_dtype == DF_DTYPE_FLOAT32)
        experts_tile_kernel<FA, E4M3, float, SUMS, true, NARROW><<<grid, 512, 0, st>>>(g);
    else if (c_dtype == DF_DTYPE_HALF)
        experts_tile_kernel<FA, E4M3, f16_t, SUMS, false, NARROW><<<grid, 512, 0, st>>>(g);
    else
        experts_tile_kernel<FA, E4M3, uint16_t, SUMS, false, NARROW><<<grid, 512, 0, st>>>(g);
}

}  // namespace

void launch_expert_tiles(int fmt_a, bool sums, bool narrow, int c_dtype, const ExpertArgs& g, int grid,
                         hipStream_t st) {
    if (sums) {
        if (narrow) launch<E5M2, true, true>(c_dtype, g, grid, st);
        else launch<E5M2, true, false>(c_dtype, g, grid, st);
    } else if (fmt_a == E4M3) {
        if (narrow) launch<E4M3, false, true>(c_dtype, g, grid, st);
        else launch<E4M3, false, false>(c_dtype, g, grid, st);
    } else {
        if (narrow) launch<E5M2, false, true>(c_dtype, g, grid, st);
        else launch<E5M2, false, false>(c_dtype, g, grid, st);
    }
}

}  // namespace dfk
