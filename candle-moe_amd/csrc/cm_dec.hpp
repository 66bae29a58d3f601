// Device helpers of the decode GEMMs (moe_gemv_dec.hip, moe_gemv_mx.hip): the
// 16x16x32 MFMA and how a workgroup finds its item and its expert's pairs.
#pragma once

#include "cm_lds.hpp"

namespace cm {
namespace dec {

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
    if constexpr (DT == kBF16) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
    }
}

// The touched-expert bitmap (LDS; the expert ids are kept in s_idx, -1:
// dropped) and this workgroup's item. With U touched experts and nblk column
// blocks, K is split into ks = min(cap / (U * nblk), ks_lim) slices (at least
// 1), so that the U * nblk * ks items fill one round of cap workgroups;
// workgroup w takes item w: the u-th touched expert (u = w / (nblk * ks)), a
// column block and a slice. [K,N] weights: the column blocks vary fastest,
// so that workgroups running side by side read neighbouring runs of the same
// k-rows; [N,K]: the slices, for neighbouring K runs of the same columns.
// s_misc[0..3] = expert (-1: no item), column block, slice, ks. Workgroup 0
// also stores ks to meta[slot] for the finishing launch.
template <int NT, bool TRANS>
__device__ __forceinline__ void dec_assign(const DecArgs& a, int slot, uint32_t* s_bm, int32_t* s_idx,
                                           int* s_misc) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nwords = (a.E + 31) >> 5;
    for (int w = tid; w < nwords; w += NT) s_bm[w] = 0u;
    __syncthreads();
    for (int p = tid; p < a.P; p += NT) {
        const uint32_t e = a.idx[p];
        const bool ok = e < (uint32_t)a.E;
        s_idx[p] = ok ? (int)e : -1;
        if (ok) atomicOr(&s_bm[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
    // wave 0: touched experts U, the slices, the item and its expert (the
    // u-th set bit; each lane two words: E <= 4096)
    if (wave == 0) {
        const uint32_t w0 = 2 * lane < nwords ? s_bm[2 * lane] : 0u;
        const uint32_t w1 = 2 * lane + 1 < nwords ? s_bm[2 * lane + 1] : 0u;
        const int c = __popc(w0) + __popc(w1);
        int incl = c;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int v = __shfl_up(incl, off);
            if (lane >= off) incl += v;
        }
        const int excl = incl - c;
        const int U = __shfl(incl, 63);
        const long long un = (long long)U * a.nblk;
        const int ks = un > 0 ? (int)max(1LL, min((long long)a.cap / un, (long long)a.ks_lim)) : 1;
        const long long w = blockIdx.x;
        const int per_u = a.nblk * ks;
        const int u = (int)(w / per_u);
        const int r_u = (int)(w - (long long)u * per_u);
        const int sl = TRANS ? r_u / a.nblk : r_u % ks;
        const int cb = TRANS ? r_u - sl * a.nblk : r_u / ks;
        if (lane == 0) {
            s_misc[0] = -1;
            s_misc[1] = cb;
            s_misc[2] = sl;
            s_misc[3] = ks;
            if (blockIdx.x == 0) a.meta[slot] = ks;
        }
        __builtin_amdgcn_wave_barrier();
        if (u < U && u >= excl && u < incl) {
            int need = u - excl;  // set bits to skip in this lane's words
            uint32_t wd = w0;
            int base = 64 * lane;
            if (need >= __popc(w0)) {
                need -= __popc(w0);
                wd = w1;
                base += 32;
            }
            for (int q = 0; q < need; ++q) wd &= wd - 1u;  // drop the lowest set bits
            s_misc[0] = base + __builtin_ctz(wd);
        }
    }
    __syncthreads();
}

// Expert e's pairs, ascending (a stable compaction of s_idx over NT-pair
// chunks), into s_rows; returns their number.
template <int NT>
__device__ __forceinline__ int dec_rows(const DecArgs& a, int e, const int32_t* s_idx, int32_t* s_rows,
                                        int* s_misc) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int run = 0;
    for (int p0 = 0; p0 < a.P; p0 += NT) {
        const int p = p0 + tid;
        const bool hit = p < a.P && s_idx[p] == e;
        const uint64_t m = __ballot(hit);
        if (lane == 0) s_misc[8 + wave] = __popcll(m);
        __syncthreads();
        int before = run;
        for (int w = 0; w < wave; ++w) before += s_misc[8 + w];
        int total = run;
        for (int w = 0; w < NT / 64; ++w) total += s_misc[8 + w];
        if (hit) s_rows[before + __popcll(m & ((1ull << lane) - 1ull))] = p;
        run = total;
        __syncthreads();
    }
    return run;
}

// The same without barriers where at most 64 pairs and no K slices leave little
// to sort: every wave finds the item by itself, one lane per pair. Experts in the
// order of their first pair. Returns the number of the expert's pairs (0: no item).
// (The bitmap's three barriers and LDS round trips are 0.7 us of a launch of 6.)
__device__ __forceinline__ int dec_assign64(const DecArgs& a, int slot, int32_t* s_rows, int& e, int& cb) {
    const int lane = threadIdx.x & 63;
    const uint32_t mine = lane < a.P ? a.idx[lane] : 0xffffffffu;
    if (blockIdx.x == 0 && threadIdx.x == 0) a.meta[slot] = 1;
    int u = (int)(blockIdx.x / (unsigned)a.nblk);
    cb = (int)(blockIdx.x - (unsigned)u * (unsigned)a.nblk);
    e = -1;
    uint64_t left = __ballot(mine < (uint32_t)a.E);
    while (left) {
        const uint32_t x = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
        const uint64_t m = __ballot(mine == x);
        if (u-- == 0) {
            e = (int)x;
            // (all waves write the same pairs; each reads its own writes)
            if ((m >> lane) & 1ull) s_rows[__popcll(m & ((1ull << lane) - 1ull))] = lane;
            __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
            __builtin_amdgcn_wave_barrier();
            return __popcll(m);
        }
        left &= ~m;
    }
    return 0;
}

}  // namespace dec
}  // namespace cm
