// gemm_blocks_tiles.hip -- the products with a scale per 128 of the reduction
// (gemm_blocks.hip) on large tiles: one persistent block per CU of eight waves, two
// per SIMD, operands by LDS DMA through two stages of 128 bytes of K (three of the
// smallest tiles, whose steps are shorter than memory's latency), as the persistent
// kernel of gemm_fp8.hip.  A wave owns FM x 2 accumulators of 32 x 32.
// What differs:
//  - Scales come with each step by a DMA instruction of their own (waves 0 and 1),
//    into a ring of slots.  A lane needs the scales of its FM rows of A and 2 of
//    B, 32 accumulator rows apart; the operands' rows are laid into LDS so that these
//    are neighbours in memory (row FM * r + i of a wave's part is row r of its
//    accumulator i), and one LDS read gives the bytes of all, which the matrix
//    instruction picks by its operand select.
//  - E8, 2-byte outputs: v_mfma_scale_f32_32x32x64_f8f6f4 at full rate.
//  - E8, fp32 outputs (WIDE): scales go into the widening to bf16.
//  - fp32 scales: a step's products are made from zero and folded into the sums
//    while the next step's are under way: one fma a value, if B's scales are the
//    same over the wave's 64 columns (weights in squares), else a product more; in
//    binary64 before that, where some of B's are far (gemm_blocks.hpp).
// Bound by the matrix units' feed, as the persistent kernel without blocks, and by the
// last, partly filled round of tiles: 16384 x 6400 x 1600 (M, N, K), bf16 out, powers of
// two, 170 us (1.97 PFLOP/s; one scale per tensor: 164), 16384 x 1600 x 6400 161 (156).
// Four waves of 128 x 128 each, with half the LDS reads, took 225 and 176: a wave a SIMD
// leaves nothing to run behind an epilogue.
#include <hip/hip_runtime.h>

#include <type_traits>
#include <utility>

#include "gemm_blocks.hpp"

namespace dfk {

namespace {

template <int N, typename F, int... I> __device__ __forceinline__ void each_(const F& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
// f(0) .. f(N - 1), the indexes compile-time constants
template <int N, typename F> __device__ __forceinline__ void each(const F& f) {
    each_<N>(f, std::make_integer_sequence<int, N>{});
}

template <int FA, int FB, int OA, int OB>
__device__ __forceinline__ v16f mfma_scaled(v8i b, v8i a, v16f c, int sb, int sa) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b, a, c, FB, FA, OB, sb, OA, sa);
}

// the value is made before what follows
__device__ __forceinline__ void hold(v16f& v) { asm volatile("" : "+v"(v)); }

typedef __attribute__((address_space(3))) void* Lds;
typedef u32x4 u32x4_el __attribute__((aligned(2)));

// FM 4: 256 x 256 tiles, waves 2 x 4; 2: 256 x 128, waves 4 x 2; 1: 128 x 128, 4 x 2.
template <int FA, typename OutT, bool E8, int FM>
__global__ __launch_bounds__(512, 1) void blocks_tile_kernel(const BlocksArgs g, int extent_a, int extent_b) {
    constexpr int FB = E4M3;
    constexpr bool WIDE = sizeof(OutT) == 4;
    constexpr int FN = 2, NF = FM + FN;
    constexpr int WAVES_N = FM == 4 ? 4 : 2;
    constexpr int BM = (8 / WAVES_N) * 32 * FM, BN = 64 * WAVES_N;
    constexpr int WR = 32 * FM;                   // rows of a wave's part
    constexpr int NDA = BM / 64, NDB = BN / 64;   // DMA instructions per wave and step
    constexpr int ND = NDA + NDB;
    constexpr int STAGE = (BM + BN) * kPKB;
    constexpr int NS = FM == 1 ? 3 : 2;           // stages
    // Slots of scales: step c + 1 + NS is on its way while step c's are still folded in
    constexpr int SLOTS = NS == 2 ? 4 : 8;
    constexpr int SZ = E8 ? 1 : 4;
    constexpr int SLOT = 2 * 256 * SZ;            // one step's scales: A's, B's
    using G = EpiGeom<(int)sizeof(OutT), FM>;
    constexpr int W_AFTER = G::NST > 63 ? 63 : G::NST;
    constexpr uint32_t kOOB = 0x80000000u;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[NS * STAGE + SLOTS * SLOT + 8 * (G::SLAB + 256)];
    uint8_t* const ring = lds + NS * STAGE;

    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = w / WAVES_N, wn = w % WAVES_N;
    uint8_t* const slab = ring + SLOTS * SLOT + w * (G::SLAB + 256);
    float* const wbias = reinterpret_cast<float*>(slab + G::SLAB);  // the wave's 64 columns'
    const int tiles_n = (g.N + BN - 1) / BN, tiles_m = (g.M + BM - 1) / BM;
    const int nunits = tiles_m * tiles_n;
    const int steps = (g.K + kPKB - 1) / kPKB;

    const int P = gridDim.x;
    const int q = P >> 3, rr = P & 7;
    const int xcd = blockIdx.x & 7, idx = blockIdx.x >> 3;
    const int bl = xcd < rr ? xcd * (q + 1) + idx : rr * (q + 1) + (xcd - rr) * q + idx;
    const int my_units = bl < nunits ? (nunits - bl + P - 1) / P : 0;
    if (my_units == 0) return;  // before any DMA; the whole block

    struct Unit {
        int m0, n0;
    };
    auto unit_of = [&](int r) {
        Unit u;
        const int n = bl + r * P;
        const int per_group = kGroupM * tiles_n;
        const int group = n / per_group;
        const int first_m = group * kGroupM;
        const int gsize = min(tiles_m - first_m, kGroupM);
        const int in_group = n - group * per_group;
        u.m0 = (first_m + in_group % gsize) * BM;
        u.n0 = (in_group / gsize) * BN;
        return u;
    };

    // ---- DMA: instruction d of wave w fills rows (w*NDA+d)*8 + lane/8 of the
    // stage's A part (and (w*NDB+d)*8 + lane/8 of its B part), 16-byte chunk c of
    // row r in slot c ^ ((r >> 1) & 7).  Row 32*i + r of a wave's part holds the
    // operand's row FM*r + i of it (B: 2*r + j).  The cursor (unit d_unit, step d_k)
    // runs NS steps ahead of the products, across units.
    const int drow = lane >> 3;
    const int dch0 = ((lane & 7) ^ (lane >> 4)) << 4;
    const int dch1 = dch0 ^ 64;
    const int pa = w * 8 * NDA, pb = w * 8 * NDB;
    const uint32_t ra = (uint32_t)(pa - pa % WR + FM * (pa % 32 + drow) + pa % WR / 32);
    const uint32_t rb = (uint32_t)(pb - pb % 64 + FN * (pb % 32 + drow) + pb % 64 / 32);
    int d_unit = 0, d_k = 0, d_g = 0, d_st = 0;  // (step d_g goes to stage d_st = d_g % NS)
    Unit du = unit_of(0);
    __amdgpu_buffer_rsrc_t rA, rB, rS;
    auto rsrc = [](const void* p, int bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, 0x00020000);
    };
    auto operands = [&]() {
        rA = rsrc(g.A + (int64_t)du.m0 * g.lda, min(g.M - du.m0, BM) * g.lda);
        rB = rsrc(g.B + (int64_t)du.n0 * g.ldb, min(g.N - du.n0, BN) * g.ldb);
        rS = w == 0 ? rsrc(static_cast<const uint8_t*>(g.sa) + (int64_t)du.m0 * SZ, extent_a - du.m0 * SZ)
                    : rsrc(static_cast<const uint8_t*>(g.sb) + (int64_t)du.n0 * SZ, extent_b - du.n0 * SZ);
    };
    operands();
    uint32_t oa0, oa1, ob0, ob1;
    auto dprep = [&]() {
        const bool live = d_unit < my_units;
        const int k0 = d_k * kPKB + dch0, k1 = d_k * kPKB + dch1;
        const bool in0 = live && k0 < g.K, in1 = live && k1 < g.K;
        oa0 = in0 ? ra * (uint32_t)g.lda + (uint32_t)k0 : kOOB;
        oa1 = in1 ? (ra + 8u * FM) * (uint32_t)g.lda + (uint32_t)k1 : kOOB;
        ob0 = in0 ? rb * (uint32_t)g.ldb + (uint32_t)k0 : kOOB;
        ob1 = in1 ? (rb + 8u * FN) * (uint32_t)g.ldb + (uint32_t)k1 : kOOB;
        // 256 rows' scales (those of rows behind the tile are not read), a step's codes
        // ahead of the codes (step c's products done: step c + 1 + NS)
        if (w < 2) {
            const uint32_t os =
                live ? (uint32_t)d_k * (uint32_t)(w == 0 ? g.ldsa : g.ldsb) * SZ + (uint32_t)lane * (4 * SZ) : kOOB;
            uint8_t* const to = ring + (d_g & (SLOTS - 1)) * SLOT + w * 256 * SZ;
            if constexpr (E8) __builtin_amdgcn_raw_ptr_buffer_load_lds(rS, (Lds)to, 4, os, 0, 0, 0);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(rS, (Lds)to, 16, os, 0, 0, 0);
        }
    };
    auto dissue_one = [&](int k) __attribute__((always_inline)) {
        uint8_t* base = lds + d_st * STAGE;
        if (k < NDA)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rA, (Lds)(base + (w * NDA + k) * 1024), 16,
                                                     ((k & 1) ? oa1 : oa0) + (uint32_t)(k >> 1) * 16u * FM * (uint32_t)g.lda,
                                                     0, 0, 0);
        else if (k < ND)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                rB, (Lds)(base + BM * kPKB + (w * NDB + k - NDA) * 1024), 16,
                (((k - NDA) & 1) ? ob1 : ob0) + (uint32_t)((k - NDA) >> 1) * 16u * FN * (uint32_t)g.ldb, 0, 0, 0);
    };
    auto dadvance = [&]() {
        if (d_unit < my_units && ++d_k == steps) {
            d_k = 0;
            if (++d_unit < my_units) {
                du = unit_of(d_unit);
                operands();
            }
        }
        ++d_g;
        d_st = d_st + 1 == NS ? 0 : d_st + 1;
        dprep();
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
        const uint8_t* p =
            lds + stage * STAGE + (f < FM ? (wm * WR + f * 32) * kPKB : (BM + wn * 64 + (f - FM) * 32) * kPKB);
        return *reinterpret_cast<const u32x4*>(p + foff[e][h]);
    };
    // E8: the bytes of this lane's rows at a step, A's FM and B's 2
    auto rd_scales = [&](int step, int& a, int& b) {
        const uint8_t* p = ring + (step & (SLOTS - 1)) * SLOT;
        if constexpr (FM == 4) a = *reinterpret_cast<const int*>(p + wm * WR + 4 * fr);
        else if constexpr (FM == 2) a = *reinterpret_cast<const uint16_t*>(p + wm * WR + 2 * fr);
        else a = p[wm * WR + fr];
        b = *reinterpret_cast<const uint16_t*>(p + 256 + wn * 64 + 2 * fr);
    };

    v16f acc[FM][FN];
    int after_epi = 0, c_g = 0, c_st = 0;  // c_g: the step whose products are under way, in stage c_st

    // Before the first read of step c_g + 1: this wave's part of it has landed
    // (after an epilogue its stores may still be under way: they were issued
    // later), then every wave's.  Every wave has read the last of step c_g, so the
    // DMA of step c_g + NS may go over it.
    auto next_step = [&]() __attribute__((always_inline)) {
        if (NS == 2 && after_epi == 1) __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0(W_AFTER));
        else __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0((NS - 2) * ND));
        after_epi = 0;
        __builtin_amdgcn_s_barrier();
    };

    // ---- fp32 scales: one step's products, folded into acc times their scales
    // during the next step (its slot of the ring is not written before that one's end)
    v16f part[E8 ? 1 : FM][FN];
    float fsa[FM];
    float usb = 0.0f;
    // (not by what lies behind the output's rows and columns, which is of any value)
    bool same = false;  // B's scales are the same over the wave's columns, and all in the middle
    bool far = false;   // (if not same) some of B's are scale_far()
    uint64_t rows_in[FM], cols_in = 0;  // lanes whose row i, whose column is in the output
    float bcol = 0.0f;
    // a step's scales, read and looked at under its last products: its fold then waits for
    // neither
    auto read_scales = [&](int step) __attribute__((always_inline)) {
        const float* p = reinterpret_cast<const float*>(ring + (step & (SLOTS - 1)) * SLOT);
#pragma unroll
        for (int i = 0; i < FM; ++i) fsa[i] = p[wm * WR + FM * fr + i];
        bcol = p[256 + wn * 64 + lane];
    };
    auto see_scales = [&]() __attribute__((always_inline)) {
        const uint32_t bu = (uint32_t)__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, bcol));
        usb = __uint_as_float(bu);
        uint64_t odd = __builtin_amdgcn_ballot_w64(bcol != usb) & cols_in;
#pragma unroll
        for (int i = 0; i < FM; ++i)
            odd |= __builtin_amdgcn_ballot_w64(!scale_in_the_middle(__float_as_uint(fsa[i]))) & rows_in[i];
        same = odd == 0 && scale_in_the_middle(bu);
        far = !same && (__builtin_amdgcn_ballot_w64(scale_far(__float_as_uint(bcol))) & cols_in) != 0;
    };
    auto fold = [&](int step, int i) __attribute__((always_inline)) {
        if (same) {
            const float s = fsa[i] * usb;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_fmaf(part[i][j][e], s, acc[i][j][e]);
        } else {
            const float* p = reinterpret_cast<const float*>(ring + (step & (SLOTS - 1)) * SLOT) + 256 + wn * 64 + 8 * (lane >> 5);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 lo = *reinterpret_cast<const f32x4*>(p + 16 * x), hi = *reinterpret_cast<const f32x4*>(p + 16 * x + 4);
                const float s[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        acc[i][j][4 * x + y] =
                            __builtin_fmaf(part[i][j][4 * x + y] * s[2 * y + j], fsa[i], acc[i][j][4 * x + y]);
            }
        }
    };

    // A step with far scales is folded here; the fold that follows adds 0
    auto fold_far = [&](int step) __attribute__((always_inline)) {
        if (__builtin_expect(!far, 1)) return;
        const float* p = reinterpret_cast<const float*>(ring + (step & (SLOTS - 1)) * SLOT) + 256 + wn * 64 + 8 * (lane >> 5);
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int j = 0; j < FN; ++j)
#pragma unroll
                    for (int y = 0; y < 4; ++y)
                        acc[i][j][4 * x + y] =
                            add_scaled_far(part[i][j][4 * x + y], fsa[i], p[16 * x + 2 * y + j], acc[i][j][4 * x + y]);
            fsa[i] = 0.0f;
        }
        usb = 0.0f;
        same = true;
    };

    // ---- fp8 products: half-steps of 64 bytes; the MFMAs on (fa, fb) while the
    // next half-step's fragments are read into (na, nb); the order frozen as in
    // gemm_fp8.hip (reads under the first MFMAs, the DMA of odd half-steps spread
    // over all).  FIRST: the unit's first half-step.
    int sa = 0, sb = 0;
    auto half = [&](auto first, auto odd, v8i* fa, v8i* fb, v8i* na, v8i* nb) __attribute__((always_inline)) {
        constexpr bool ODD = decltype(odd)::value, FIRST = decltype(first)::value;
        constexpr int NM = FM * FN, RD_OVER = NM < 4 ? NM : 4;
        __builtin_amdgcn_sched_barrier(0);
        if (ODD) next_step();
        const int stage = ODD ? (c_st + 1 == NS ? 0 : c_st + 1) : c_st;
        constexpr int NR = 2 * NF;
        u32x4 frag[NR];
        int nsa = sa, nsb = sb;
        if constexpr (!E8 && ODD) read_scales(c_g);
        each<NM>([&](auto xc) __attribute__((always_inline)) {
            constexpr int x = decltype(xc)::value, i = x >> 1, j = x & 1;
            const v16f z = {};
            if constexpr (E8) {
                if constexpr (FIRST) acc[i][j] = mfma_scaled<FA, FB, i, j>(fb[j], fa[i], z, sb, sa);
                else acc[i][j] = mfma_scaled<FA, FB, i, j>(fb[j], fa[i], acc[i][j], sb, sa);
            } else {
                if constexpr (!ODD && !FIRST && j == 0) fold(c_g - 1, i);
                part[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[j], fa[i], ODD ? part[i][j] : z, FB, FA, 0, 0,
                                                                             0, 0);
            }
            if constexpr (x < RD_OVER) {
#pragma unroll
                for (int r = NR * x / RD_OVER; r < NR * (x + 1) / RD_OVER; ++r) frag[r] = rd(stage, r >> 1, ODD ? 0 : 1, r & 1);
                if constexpr (E8 && ODD && x == 0) rd_scales(c_g + 1, nsa, nsb);
            }
            if constexpr (ODD) {
#pragma unroll
                for (int d = ND * x / NM; d < ND * (x + 1) / NM; ++d) dissue_one(d);
            }
            if constexpr (!E8 && ODD && x == NM - 1) see_scales();
            __builtin_amdgcn_sched_barrier(0);
        });
#pragma unroll
        for (int f = 0; f < NF; ++f) {
            const u32x4 lo = frag[2 * f], hi = frag[2 * f + 1];
            v8i r;
            r[0] = (int)lo.x; r[1] = (int)lo.y; r[2] = (int)lo.z; r[3] = (int)lo.w;
            r[4] = (int)hi.x; r[5] = (int)hi.y; r[6] = (int)hi.z; r[7] = (int)hi.w;
            if (f < FM) na[f] = r; else nb[f - FM] = r;
        }
        if (ODD) {
            // The scaled products, unlike the others, are free to move: without this
            // the compiler sinks them behind the branches of dadvance(), next to the
            // following half-step's, and spills the fragments of both
            if constexpr (E8) {
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FN; ++j) hold(acc[i][j]);
            } else {
                fold_far(c_g);
            }
            sa = nsa;
            sb = nsb;
            ++c_g;
            c_st = stage;
            dadvance();
        }
    };

    // ---- bf16 products: quarter-steps of 16 bytes per lane (32 of K); a quarter's
    // codes are widened eight at a time, the next quarter's read
    float ws[NF];  // the widening's scales, of the FM rows and the FN columns
    auto wide_scales = [&](int step) {
        int a, b;
        rd_scales(step, a, b);
#pragma unroll
        for (int i = 0; i < FM; ++i) ws[i] = __uint_as_float(((uint32_t)a >> 8 * i & 0xFFu) << 23);
#pragma unroll
        for (int j = 0; j < FN; ++j) ws[FM + j] = __uint_as_float(((uint32_t)b >> 8 * j & 0xFFu) << 23);
    };
    if constexpr (!E8) {
#pragma unroll
        for (int f = 0; f < NF; ++f) ws[f] = 1.0f;
    }
    auto quarter = [&](auto first, auto qq, const u32x4* cur, u32x4* nxt) __attribute__((always_inline)) {
        constexpr int Q = decltype(qq)::value;
        constexpr bool FIRST = decltype(first)::value;
        __builtin_amdgcn_sched_barrier(0);
        if (Q == 3) next_step();
        const int stage = Q == 3 ? (c_st + 1 == NS ? 0 : c_st + 1) : c_st;
        if constexpr (!E8 && Q == 3) read_scales(c_g);
#pragma unroll
        for (int f = 0; f < NF; ++f) nxt[f] = rd(stage, f, ((Q + 1) >> 1) & 1, (Q + 1) & 1);
        // (read anew each step: kept from the step before, they took 80 registers' copies)
        if constexpr (E8 && Q == 0) wide_scales(c_g);
        each<2>([&](auto sc) __attribute__((always_inline)) {
            constexpr int s = decltype(sc)::value;
            bf8 wb[FN];
#pragma unroll
            for (int j = 0; j < FN; ++j) wb[j] = widen8_scaled<FB>(cur[FM + j][2 * s], cur[FM + j][2 * s + 1], ws[FM + j]);
            each<FM>([&](auto ic) __attribute__((always_inline)) {
                constexpr int i = decltype(ic)::value;
                const bf8 wa = widen8_scaled<FA>(cur[i][2 * s], cur[i][2 * s + 1], ws[i]);
                if constexpr (!E8 && Q == 0 && s == 0 && !FIRST) fold(c_g - 1, i);
                each<FN>([&](auto jc) __attribute__((always_inline)) {
                    constexpr int j = decltype(jc)::value, x = (s * FM + i) * FN + j;
                    const v16f z = {};
                    if constexpr (E8)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j], wa, FIRST && s == 0 ? z : acc[i][j], 0, 0, 0);
                    else
                        part[i][j] =
                            __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j], wa, Q == 0 && s == 0 ? z : part[i][j], 0, 0, 0);
                    if constexpr (Q == 3) {
                        constexpr int NM = 2 * FM * FN;
#pragma unroll
                        for (int d = ND * x / NM; d < ND * (x + 1) / NM; ++d) dissue_one(d);
                    }
                });
            });
        });
        if constexpr (!E8 && Q == 3) {
            see_scales();
            fold_far(c_g);
        }
        if (Q == 3) {
            ++c_g;
            c_st = stage;
            dadvance();
        }
    };

    // Stores a finished unit: bias and conversion in registers, then each 32-row
    // block through the wave's LDS slab and out as 16-byte stores of whole row
    // segments (vec_out 2: non-temporal; see epi_store_mode).  A lane holds row FM *
    // (lane % 32) + i of the wave's part and, for each x, its columns 16 x + 8 * (lane
    // / 32) .. +8.  Whether the wave's part lay wholly inside the output, i.e. whether
    // it issued all its stores.
    auto store_unit = [&](const Unit& u) __attribute__((always_inline)) -> bool {
        constexpr int ES = (int)sizeof(OutT);
        OutT* const C = static_cast<OutT*>(g.C);
        const int el = fresh_lane(), efr = el & 31;
        const int rowb = u.m0 + wm * WR, colw = u.n0 + wn * 64;
        const int h8 = (el >> 5) * 8;
        constexpr int CPR = 64 * ES / 16;
        constexpr int RPS = 64 / CPR;
        const int srow = el / CPR, rc = el % CPR;
        const int scol = colw + rc * (16 / ES);
        const bool col_full = scol + 16 / ES <= g.N;
        const int my_sr = efr % G::SR, my_pass = efr / G::SR;
        // LDS operations of one wave execute in order, so a pass's reads see its
        // writes and precede the next pass's writes; the empty asm statements keep
        // the compiler from reordering them.
#pragma unroll
        for (int i = 0; i < FM; ++i) {
#pragma unroll
            for (int p = 0; p < G::NPASS; ++p) {
                if (my_pass == p) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        float v[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = acc[i][e & 1][4 * x + (e >> 1)];
                        if (g.bias) {
                            const f32x4 lo = *reinterpret_cast<const f32x4*>(wbias + 16 * x + h8);
                            const f32x4 hi = *reinterpret_cast<const f32x4*>(wbias + 16 * x + h8 + 4);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                v[e] += lo[e];
                                v[4 + e] += hi[e];
                            }
                        }
                        uint8_t* d = slab + my_sr * G::SROW + (16 * x + h8) * ES;
                        if constexpr (ES == 4) {
                            *reinterpret_cast<f32x4*>(d) = f32x4{v[0], v[1], v[2], v[3]};
                            *reinterpret_cast<f32x4*>(d + 16) = f32x4{v[4], v[5], v[6], v[7]};
                        } else {
                            u32x4 o;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if constexpr (std::is_same<OutT, f16_t>::value)
                                    o[e] = f32_to_f16_rne(v[2 * e]) | (f32_to_f16_rne(v[2 * e + 1]) << 16);
                                else
                                    o[e] = pack_bf16_rne(v[2 * e], v[2 * e + 1]);
                            }
                            *reinterpret_cast<u32x4*>(d) = o;
                        }
                    }
                }
                asm volatile("" ::: "memory");
#pragma unroll
                for (int s = 0; s < G::SPP; ++s) {
                    const int sr = s * RPS + srow;
                    const u32x4 val = *reinterpret_cast<const u32x4*>(slab + sr * G::SROW + rc * 16);
                    const int row = rowb + FM * (p * G::SR + sr) + i;
                    if (row < g.M) {
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
        return rowb + WR <= g.M && colw + 64 <= g.N;
    };

    // prologue: DMA steps 0 to NS - 1; step 0's first fragments
    dprep();
    for (int i = 0; i < NS; ++i) {
        for (int k = 0; k < ND; ++k) dissue_one(k);
        dadvance();
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_vm_lgkm0((NS - 1) * ND));
    __builtin_amdgcn_s_barrier();

    using Y = std::true_type;
    using N = std::false_type;
    if constexpr (E8 && !WIDE) rd_scales(0, sa, sb);
    // A unit's bias is loaded at its start, for the wave's columns, one a lane: by
    // its end the load has long landed, and waits for no DMA under way.
    auto bias_of = [&](const Unit& u) {
        const int c = u.n0 + wn * 64 + lane;
        return g.bias && c < g.N ? bias_at(g.bias, g.bias_dtype, c) : 0.0f;
    };
    auto finish = [&](const Unit& u, float b) __attribute__((always_inline)) {
        if constexpr (!E8) {
#pragma unroll
            for (int i = 0; i < FM; ++i) fold(c_g - 1, i);
        }
        if (g.bias) wbias[lane] = b;
        asm volatile("" ::: "memory");
        after_epi = store_unit(u) ? 1 : 2;
    };
    auto start = [&](const Unit& u) __attribute__((always_inline)) {
        if constexpr (!E8) {
#pragma unroll
            for (int i = 0; i < FM; ++i) rows_in[i] = __builtin_amdgcn_ballot_w64(u.m0 + wm * WR + FM * fr + i < g.M);
            cols_in = __builtin_amdgcn_ballot_w64(u.n0 + wn * 64 + lane < g.N);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = v16f{};
        }
    };
    if constexpr (WIDE) {
        u32x4 r0[NF], r1[NF];
        for (int f = 0; f < NF; ++f) r0[f] = rd(0, f, 0, 0);
        using Q0 = std::integral_constant<int, 0>;
        using Q1 = std::integral_constant<int, 1>;
        using Q2 = std::integral_constant<int, 2>;
        using Q3 = std::integral_constant<int, 3>;
        for (int r = 0; r < my_units; ++r) {
            const Unit u = unit_of(r);
            const float b = bias_of(u);
            start(u);
            quarter(Y{}, Q0{}, r0, r1);
            quarter(N{}, Q1{}, r1, r0);
            quarter(N{}, Q2{}, r0, r1);
            quarter(N{}, Q3{}, r1, r0);
            for (int k = 1; k < steps; ++k) {
                quarter(N{}, Q0{}, r0, r1);
                quarter(N{}, Q1{}, r1, r0);
                quarter(N{}, Q2{}, r0, r1);
                quarter(N{}, Q3{}, r1, r0);
            }
            finish(u, b);
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
            const float b = bias_of(u);
            start(u);
            half(Y{}, N{}, fa0, fb0, fa1, fb1);
            half(N{}, Y{}, fa1, fb1, fa0, fb0);
            for (int k = 1; k < steps; ++k) {
                half(N{}, N{}, fa0, fb0, fa1, fb1);
                half(N{}, Y{}, fa1, fb1, fa0, fb0);
            }
            finish(u, b);
        }
    }
    __builtin_amdgcn_s_waitcnt(0);  // every DMA has landed before the block's LDS is released
}

template <int FA, bool E8, int FM> void launch(int c_dtype, const BlocksArgs& g, int ea, int eb, int grid, hipStream_t st) {
    if (c_dtype == DF_DTYPE_FLOAT32) blocks_tile_kernel<FA, float, E8, FM><<<grid, 512, 0, st>>>(g, ea, eb);
    else if (c_dtype == DF_DTYPE_HALF) blocks_tile_kernel<FA, f16_t, E8, FM><<<grid, 512, 0, st>>>(g, ea, eb);
    else blocks_tile_kernel<FA, uint16_t, E8, FM><<<grid, 512, 0, st>>>(g, ea, eb);
}

template <int FA>
void launch_as(bool e8, int fm, int c_dtype, const BlocksArgs& g, int ea, int eb, int grid, hipStream_t st) {
    if (e8) {
        if (fm == 1) launch<FA, true, 1>(c_dtype, g, ea, eb, grid, st);
        else if (fm == 2) launch<FA, true, 2>(c_dtype, g, ea, eb, grid, st);
        else launch<FA, true, 4>(c_dtype, g, ea, eb, grid, st);
    } else {
        if (fm == 1) launch<FA, false, 1>(c_dtype, g, ea, eb, grid, st);
        else launch<FA, false, 2>(c_dtype, g, ea, eb, grid, st);
    }
}

}  // namespace

void launch_block_tiles(int fmt_a, bool e8, int fm, int c_dtype, const BlocksArgs& g, int ea, int eb, int grid,
                        hipStream_t st) {
    if (fmt_a == E4M3) launch_as<E4M3>(e8, fm, c_dtype, g, ea, eb, grid, st);
    else launch_as<E5M2>(e8, fm, c_dtype, g, ea, eb, grid, st);
}

}  // namespace dfk
