// Gate/up and fc1 of large batches with both operands in MX formats (gfx950): MXFP8
// rows (e4m3) times MXFP4 weights (e2m1) on v_mfma_scale_f32_32x32x64_f8f6f4, which
// takes the codes and the scale bytes as they are: nothing is converted, and a
// MFMA does 64 k in the time the 16-bit one does 32.
//
// A product's 64 terms are exact, but aligned to the largest of them before they
// are added (terms 2^-19 or so below it lose bits: 2e-5 of the sum of magnitudes
// on average over scales spread by 2^14, nothing over the values of one row and
// column); the sums across K are f32. The intermediate's rounding to 16 bits, right
// after, is larger.
//
// Qwen3 T=16384 gate/up: 436 us (1.89 PFLOP/s; a library product of 8192^3 in fp8
// 3.0), on 16-bit copies of the rows 728 us. Per K tile and CU 50 KB come into LDS
// and 160 KB of fragments go out, some 1650 cycles of its port under the 2048 of the
// MFMAs: the two do not overlap fully.
//
// Tile 256 x 256, K tiles of 128, 8 waves (2 x 4), three LDS stages filled by DMA:
// 32 KB of row codes, 16 KB of weight codes, a dword of scales per row and column
// (the tile's four 32 k). Lane (h, r) (h = lane / 32) of a 64-k step holds, of the
// first operand (column r of the weights), k 32 h .. +31 in one 16-byte chunk, of
// the second (row r) k 16 h .. +15 and 32 + 16 h .. +15 in two; the scale of 32 k
// block h comes from the lanes of half h (checked on the hardware).
// Rows are gathered by pair and the epilogue is the 16-bit kernels'
// (moe_gemm_lds.hip), as is the split of the last round's tiles along K.
#include "cm_lds.hpp"

namespace cm {

using namespace lds;

namespace {

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

// opsel S: byte of the scale registers (0: first 64 k of the tile, 2: second)
template <int S>
__device__ __forceinline__ f32x16 mfma_mx(const u32x4& w, const u32x4& x0, const u32x4& x1, const f32x16& c, uint32_t sw,
                                          uint32_t sx) {
    const i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    const i32x8 b = {(int)x0[0], (int)x0[1], (int)x0[2], (int)x0[3], (int)x1[0], (int)x1[1], (int)x1[2], (int)x1[3]};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 4, 0, S, (int)sw, S, (int)sx);
}

template <int MODE>
__global__ __launch_bounds__(512, 1) void mx8_gemm_k(GemmArgs a) {
    constexpr bool DUAL = (MODE == kGateUp);
    constexpr int BM = 256, BN = 256, BK = 128, NW = 8, NST = 3, WM = 128, WN = 64, MB = 4, NB = 2;
    constexpr int SUBN = DUAL ? BN / 2 : BN;  // columns of a tensor
    constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK / 2, S_BYTES = 4 * (BM + BN);
    constexpr int STAGE = A_BYTES + B_BYTES + S_BYTES;
    constexpr int A_INS = A_BYTES / (1024 * NW), B_INS = B_BYTES / (1024 * NW), LOADS = A_INS + B_INS + 1;
    static_assert(S_BYTES == 256 * NW, "one scale instruction per wave");
    static_assert(NST * STAGE >= BM * SUBN * 2, "output tile fits the stages");
    __shared__ __attribute__((aligned(1024))) char smem[NST * STAGE];
    __shared__ int32_t s_dst[BM];

    const int nk_all = a.K / BK;
    int tile, ks, nsplit, fix_slot0, fix_ctr;
    if (a.tail_cus > 0) {
        if (!tail_item(*a.num_tiles * a.n_tiles, a.tail_cus, nk_all, tile, ks, nsplit, fix_slot0, fix_ctr)) return;
    } else {
        tile = xcd_logical(*a.num_tiles * a.n_tiles);
        if (tile < 0) return;
        ks = fix_slot0 = fix_ctr = 0;
        nsplit = 1;
    }
    const int mt = tile / a.n_tiles, nt = tile - mt * a.n_tiles;
    const int r0 = a.tile_row[mt], e = a.tile_exp[mt];
    const int m_valid = min(BM, a.offsets[e + 1] - r0);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3, lr = lane & 31, lh = lane >> 5;
    const int K = a.K, N = a.N, kb = K / 32;

    // (rows past the group's end: some pair's, never stored)
    auto row_of = [&](int r) { return (uint32_t)(a.sorted_pair[min(r0 + r, a.sorted_n - 1)] / a.k_top); };
    const i32x4 rA = make_rsrc(a.A, a.a_bytes), rX = make_rsrc(a.xs, a.a_bytes / 32);
    const long long wb = a.strideB / 2, sb = a.strideB / 32;
    const i32x4 rB0 = make_rsrc(reinterpret_cast<const char*>(a.B0) + (long long)e * wb, wb);
    const i32x4 rS0 = make_rsrc(a.mx0 + (long long)e * sb, sb);
    i32x4 rB1 = rB0, rS1 = rS0;
    if constexpr (DUAL) {
        rB1 = make_rsrc(reinterpret_cast<const char*>(a.B1) + (long long)e * wb, wb);
        rS1 = make_rsrc(a.mx1 + (long long)e * sb, sb);
    }
    const uint32_t smem_base = __builtin_amdgcn_readfirstlane(lds_addr(smem));
    uint32_t a_off[A_INS], b_off[B_INS], s_off;
#pragma unroll
    for (int i = 0; i < A_INS; ++i) {
        const int r = 8 * (NW * i + wave) + lane / 8;
        a_off[i] = row_of(r) * (uint32_t)K + (uint32_t)(a_swz<8>(r, lane % 8) * 16);
    }
#pragma unroll
    for (int i = 0; i < B_INS; ++i) {
        const int r = 16 * (NW * i + wave) + lane / 4, n = nt * SUBN + r % SUBN;
        b_off[i] = n < N ? (uint32_t)n * (uint32_t)(K / 2) + (uint32_t)(w4_swz<4>(r, lane % 4) * 16) : kOob;
    }
    // waves 0 .. 3 fetch the rows' scales, 4 .. 7 the columns'
    const int sr = 64 * (wave & 3) + lane;
    const bool s_up = DUAL && wave >= 4 && 64 * (wave & 3) >= SUBN;
    if (wave < 4) {
        s_off = row_of(sr) * (uint32_t)kb;
    } else {
        const int n = nt * SUBN + sr % SUBN;
        s_off = n < N ? (uint32_t)n * (uint32_t)kb : kOob;
    }
    const i32x4 rSc = wave < 4 ? rX : s_up ? rS1 : rS0;
    auto issue = [&](int stage, int kt) {
        const uint32_t sA = smem_base + stage * STAGE, sB = sA + A_BYTES;
#pragma unroll
        for (int i = 0; i < A_INS; ++i) dma16s(rA, sA + (NW * i + wave) * 1024, a_off[i], (uint32_t)kt * BK);
#pragma unroll
        for (int i = 0; i < B_INS; ++i) {
            const int q = NW * i + wave;
            dma16s(DUAL && 16 * q >= SUBN ? rB1 : rB0, sB + q * 1024, b_off[i], (uint32_t)kt * (BK / 2));
        }
        dma4(rSc, sB + B_BYTES + wave * 256, s_off == kOob ? kOob : s_off + 4u * (uint32_t)kt);
    };

    f32x16 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    int b_row[NB];  // this lane's column in each block (gate and up of the same columns for DUAL)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) b_row[nb] = (DUAL ? nb * SUBN + wn * 32 : wn * WN + nb * 32) + lr;

    const bool rows_live = wm * WM < m_valid;
    auto compute = [&](int stage) {
        const char* sA = smem + stage * STAGE;
        const char* sB = sA + A_BYTES;
        const uint32_t* sSA = reinterpret_cast<const uint32_t*>(sB + B_BYTES);
        const uint32_t* sSB = sSA + BM;
        uint32_t xs[MB], ws[NB];
        u32x4 x0[2][MB], x1[2][MB], w[2][NB];
        auto load = [&](int s) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                w[s][nb] = *reinterpret_cast<const u32x4*>(sB + b_row[nb] * (BK / 2) + w4_swz<4>(b_row[nb], 2 * s + lh) * 16);
#pragma unroll
            for (int mb = 0; mb < MB; ++mb) {
                const int r = wm * WM + mb * 32 + lr;
                x0[s][mb] = *reinterpret_cast<const u32x4*>(sA + r * BK + a_swz<8>(r, 4 * s + lh) * 16);
                x1[s][mb] = *reinterpret_cast<const u32x4*>(sA + r * BK + a_swz<8>(r, 4 * s + 2 + lh) * 16);
            }
        };
        load(0);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) ws[nb] = sSB[b_row[nb]] >> (8 * lh);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) xs[mb] = sSA[wm * WM + mb * 32 + lr] >> (8 * lh);
        __builtin_amdgcn_sched_barrier(0);
        load(1);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                acc[mb][nb] = mfma_mx<0>(w[0][nb], x0[0][mb], x1[0][mb], acc[mb][nb], ws[nb], xs[mb]);
        // one MFMA, then a read or two of the second half's operands
#pragma unroll
        for (int i = 0; i < MB * NB; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                acc[mb][nb] = mfma_mx<2>(w[1][nb], x0[1][mb], x1[1][mb], acc[mb][nb], ws[nb], xs[mb]);
        __builtin_amdgcn_sched_barrier(0);
    };

    int pre_dst[MB];
    float pre_w[MB];
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) {
        const int ml = wm * WM + mb * 32 + lr;
        const int r = r0 + (ml < m_valid ? ml : 0);
        const int p = a.sorted_pair[r];
        pre_dst[mb] = a.pair_dest ? a.pair_dest[p] : r;
        pre_w[mb] = a.fold_w ? a.routing_w[p] : 1.0f;
    }
    const int per = (nk_all + nsplit - 1) / nsplit, kt0 = min(nk_all, ks * per), nk = min(nk_all, kt0 + per) - kt0;
#pragma unroll
    for (int s = 0; s < NST - 1; ++s)
        if (s < nk) issue(s, kt0 + s);
    for (int kt = 0; kt < nk; ++kt) {
        wait_stage<LOADS, NST - 2>(min(NST - 2, nk - 1 - kt));
        wait_lgkm0();
        block_barrier();
        if (kt + NST - 1 < nk) issue((kt + NST - 1) % NST, kt0 + kt + NST - 1);
        if (rows_live) compute(kt % NST);
    }
    if (nsplit > 1 && !splitk_fixup<MB, NB, NW, 8>(a, acc, fix_slot0, fix_ctr, ks, nsplit, wave, lane)) return;
    if (wn == 0 && lane < 32) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) s_dst[wm * WM + mb * 32 + lane] = pre_dst[mb];
    }
    __syncthreads();  // every wave is done with the stages
    f32x16 none[1];
    staged_epilogue<kBF16, MODE, BM, BN, WM, WN, MB, NB, NW, false, 0, NST * STAGE, 1>(
        a, acc, smem, s_dst, m_valid, nt, wm, wn, lane, pre_w, nullptr, nullptr, none, nullptr);
}

}  // namespace

hipError_t launch_moe_gemm_mx8(int mode, const GemmArgs& a, hipStream_t stream) {
    if ((mode != kGateUp && mode != kFc1) || a.xs == nullptr || a.mx0 == nullptr ||
        (mode == kGateUp && a.mx1 == nullptr) || a.K % 128 || a.N % 32 || ((uintptr_t)a.xs & 3))
        return hipErrorInvalidValue;
    const long long tiles = (long long)a.m_tiles_max * a.n_tiles;
    const long long nwg = a.tail_cus > 0 ? 8 * ((tiles + 7) / 8 + a.tail_cus) : tiles;
    if (nwg > 0x7fffffffLL) return hipErrorInvalidValue;
    if (nwg <= 0) return hipSuccess;
    const dim3 g((unsigned)nwg);
    if (mode == kGateUp) hipLaunchKernelGGL(mx8_gemm_k<kGateUp>, g, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL(mx8_gemm_k<kFc1>, g, dim3(512), 0, stream, a);
    return hipGetLastError();
}

}  // namespace cm
