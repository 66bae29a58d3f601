// Decode GEMMs over MXFP4 expert weights (gfx950): few rows per touched expert, so
// the time is the weight stream (4.25 bits a weight) and the latency around it.
// Qwen3 T=16: gate/up 13.9 us (53.5 MB, 3.8 TB/s), down 8.9 (26.7 MB, 3.0 TB/s);
// from 8-bit rows T=8 13.5 / 8.4; Qwen3-30B-A3B T=1 gate/up 7.2 us (13.4 MB).
//
// As in moe_gemv_dec.hip a workgroup finds its item (touched expert, block of
// 16 * CPL columns) and the expert's pairs itself, its 4 waves split K (gate/up:
// two waves per tensor), weights go straight into registers and the parts meet
// through LDS once, in a fixed order. What differs:
//  * A step is 128 k: lane (g, i) (g = lane / 16, i = lane % 16) loads the 16
//    bytes that hold k0 + 32 g .. +31 of its column, which share one scale byte. The
//    gfx950 scaled conversions turn 8 codes and the scale into an operand of
//    v_mfma_f32_16x16x32, exactly in bf16: no weight is rounded, no sum rescaled.
//  * The block's scale bytes are one contiguous piece of memory and come through
//    LDS. (A byte load per lane beside every code load cost more than the codes:
//    loads alone, Qwen3 T=16 gate/up 16.5 against 12.0 us, Qwen3-30B-A3B T=1 7.4
//    against 5.8.)
//  * The expert's rows go through LDS (DMA, once per workgroup), so that a wave's
//    registers hold weights only and a whole K part of up to RING steps is in
//    flight at once. With the rows in the same registers, in flight next to the
//    weights, a step took twice the registers and the ring was half as long: Qwen3
//    T=16 gate/up 19.2, Qwen3-30B-A3B T=1 8.5 us (one wave per SIMD and item: the
//    time of a launch is its trips to memory).
//  * Rows are 16-bit or MXFP8 (X8: e4m3 codes and their scale bytes through LDS),
//    converted the same way.
// Rows of a tile are padded by 16 bytes in LDS: 16 lanes reading 16 rows at one k
// land in different banks. K chunks (DecArgs::kc) bound the LDS of long rows.
#include <algorithm>

#include "cm_dec.hpp"

namespace cm {

using namespace lds;
using namespace dec;

namespace {

constexpr int kMxWaves = 4;

// Weight steps in flight per wave: about 120 registers of them, so that two
// workgroups share a CU where their LDS lets them.
template <int CPL>
constexpr int mx_ring() { return CPL <= 3 ? 8 : CPL == 4 ? 6 : CPL == 6 ? 4 : 3; }

template <int DT, int MODE, int RB, int CPL, bool X8>
__global__ __launch_bounds__(64 * kMxWaves, 2) void mx_dec_k(DecArgs a) {
    constexpr bool DUAL = (MODE == kGateUp);
    constexpr bool GATHER = (MODE == kGateUp || MODE == kFc1);
    static_assert(GATHER || !X8, "8-bit rows: gate/up and fc1");
    constexpr int NT = 64 * kMxWaves, KP = DUAL ? kMxWaves / 2 : kMxWaves, RING = mx_ring<CPL>();
    constexpr int WGC = 16 * CPL, SPW = WGC + 4, AB = X8 ? 1 : 2;

    __shared__ uint32_t s_bm[kDecMaxE / 32];
    __shared__ int32_t s_idx[kDecMaxPairs];
    __shared__ int32_t s_rows[kDecMaxPairs];
    __shared__ int s_misc[8 + kMxWaves];
    // scale bytes of the block's columns (of both tensors), those of the rows (X8);
    // from a.lds_rows on the expert's rows, after the K loop the waves' parts
    // [wave][row][SPW]
    extern __shared__ __attribute__((aligned(16))) char s_dyn[];
    char* s_a = s_dyn + a.lds_rows;
    float* s_part = reinterpret_cast<float*>(s_a);

    int e, cb, cnt = 0;
    const bool few = a.P <= 64;
    if (few) {
        cnt = dec_assign64(a, GATHER ? 0 : 1, s_rows, e, cb);
    } else {
        dec_assign<NT, false>(a, GATHER ? 0 : 1, s_bm, s_idx, s_misc);
        e = s_misc[0];
        cb = s_misc[1];
    }
    if (e < 0) return;
    if (!few) cnt = dec_rows<NT>(a, e, s_idx, s_rows, s_misc);

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, li = lane & 15;
    const int tensor = DUAL ? wave / KP : 0;
    const int kpart = DUAL ? wave - tensor * KP : wave;
    const int K = a.K, N = a.N, col0 = cb * WGC;

    // codes and scale bytes of expert e (in-range loads only, zeros past), the rows
    const long long wbytes = a.strideB / 2, sbytes = a.strideB / 32;
    const int kb = K / 32, sblock = WGC * kb;  // scale bytes of a column, of the block
    const int sround = (sblock + 1023) & ~1023;
    const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(reinterpret_cast<const char*>(tensor ? a.B1 : a.B0)) + (long long)e * wbytes, 0, (int)wbytes,
        0x00020000);
    const i32x4 rA = make_rsrc(a.A, a.a_bytes);
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(s_dyn));

    // the block's scales, 1 KB per instruction, the waves of a tensor in turn (past
    // the expert's matrix: zeros)
    {
        const long long se = (long long)e * sbytes;
        const i32x4 rs = make_rsrc((tensor ? a.mx1 : a.mx0) + se, sbytes);
        for (int q = kpart; q < sround >> 10; q += KP)
            dma16(rs, lds0 + (uint32_t)(tensor * sround + q * 1024),
                  (uint32_t)col0 * (uint32_t)kb + (uint32_t)q * 1024u + 16u * (uint32_t)lane);
    }
    const uint8_t* s_sc = reinterpret_cast<const uint8_t*>(s_dyn) + tensor * sround + li * kb + g;
    const int xp = (kb + 255) & ~255;  // (X8) LDS pitch of a row's scale bytes
    uint8_t* s_xs = reinterpret_cast<uint8_t*>(s_dyn) + (DUAL ? 2 : 1) * sround;

    // first byte of this lane's codes in each column block; past N: out of range
    uint32_t wlane[CPL];
#pragma unroll
    for (int b = 0; b < CPL; ++b) {
        const int n = col0 + 16 * b + li;
        wlane[b] = n < N ? (uint32_t)n * (uint32_t)(K / 2) + 16u * (uint32_t)g : kOob;
    }

    for (int c0 = 0; c0 < cnt; c0 += RB * 16) {
        const int m_valid = min(RB * 16, cnt - c0);
        f32x4 acc[RB][CPL];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int b = 0; b < CPL; ++b) acc[rb][b] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < K; k0 += a.kc) {
            const int kn = min(a.kc, K - k0);  // k of this chunk
            const int segs = (kn * AB + 1023) >> 10;
            const int pitch = segs * 1024 + 16;
            if (k0 > 0 || c0 > 0) __syncthreads();  // (the LDS is read no more)
            if constexpr (X8) {
                if (k0 == 0 && kb % 4 == 0 && (reinterpret_cast<uintptr_t>(a.xs) & 3) == 0) {
                    // 256 bytes per instruction
                    const i32x4 rx = make_rsrc(a.xs, a.a_bytes / 32);
                    const int xsegs = xp >> 8;
                    for (int q = wave; q < m_valid * xsegs; q += kMxWaves) {
                        const int r = q / xsegs, at = (q - r * xsegs) * 256;
                        const uint32_t row = (uint32_t)(__builtin_amdgcn_readfirstlane(s_rows[c0 + r]) / a.k_top) * (uint32_t)kb;
                        dma4(rx, lds0 + (uint32_t)((DUAL ? 2 : 1) * sround + r * xp + at),
                             at + 4 * lane < kb ? row + (uint32_t)(at + 4 * lane) : kOob);
                    }
                } else if (k0 == 0) {
                    for (int q = tid; q < m_valid * kb; q += NT) {
                        const int r = q / kb;
                        s_xs[r * xp + (q - r * kb)] = a.xs[(long long)(s_rows[c0 + r] / a.k_top) * kb + (q - r * kb)];
                    }
                }
            }
            // rows to LDS: one instruction per 1 KB, the waves in turn
            for (int q = wave; q < m_valid * segs; q += kMxWaves) {
                const int r = q / segs, sg = q - r * segs;
                const int p = __builtin_amdgcn_readfirstlane(s_rows[c0 + r]);
                const uint32_t row = (uint32_t)(GATHER ? p / a.k_top : p) * (uint32_t)(K * AB) + (uint32_t)(k0 * AB);
                const uint32_t at = (uint32_t)sg * 1024u + 16u * (uint32_t)lane;
                dma16(rA, lds0 + (uint32_t)(a.lds_rows + r * pitch + sg * 1024), at < (uint32_t)(kn * AB) ? row + at : kOob);
            }

            // this wave's steps of the chunk
            const int nks = (kn + 127) / 128, per = (nks + KP - 1) / KP;
            const int s_lo = kpart * per, n = min(per, nks - s_lo);
            u32x4 wv[RING][CPL];
            auto load = [&](int i, int st) {
                const int k = k0 + (s_lo + st) * 128;
                const bool in = (st < n) & (k + 32 * g < k0 + kn);  // (K is a multiple of 32: whole chunks)
#pragma unroll
                for (int b = 0; b < CPL; ++b)
                    wv[i][b] = __builtin_amdgcn_raw_buffer_load_b128(rw, in ? wlane[b] + (uint32_t)(k / 2) : kOob, 0, 0);
            };
#pragma unroll
            for (int i = 0; i < RING; ++i) load(i, i);
            // the rows and scales are older than the RING steps' loads
            constexpr int LOADS = RING * CPL;
            static_assert(LOADS < 63, "vmcnt range");
            wait_vm<LOADS>();
            wait_lgkm0();
            block_barrier();

            uint32_t arow[RB];  // byte of this lane's k in its rows (rows past the last: the last)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
                arow[rb] = (uint32_t)(min(rb * 16 + li, m_valid - 1) * pitch + 32 * AB * g);
            auto compute = [&](int i, int st) {
                u32x4 ao[RB][4];
                const uint32_t ka = (uint32_t)((s_lo + st) * 128 * AB);
                const int kq = k0 / 32 + (s_lo + st) * 4;  // (its lane group's 32 k: + g)
                // past K the codes are zeros, and a foreign scale could be a NaN
                const bool in = kq + g < kb;
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const u32x4* src = reinterpret_cast<const u32x4*>(s_a + arow[rb] + ka);
                    if constexpr (X8) {
                        const u32x4 v0 = src[0], v1 = src[1];
                        const uint32_t xb = s_xs[min(rb * 16 + li, m_valid - 1) * xp + min(kq + g, kb - 1)];
                        const float sc = __uint_as_float(xb << 23);
                        ao[rb][0] = mx8x8_to<DT>(u32x2{v0[0], v0[1]}, sc);
                        ao[rb][1] = mx8x8_to<DT>(u32x2{v0[2], v0[3]}, sc);
                        ao[rb][2] = mx8x8_to<DT>(u32x2{v1[0], v1[1]}, sc);
                        ao[rb][3] = mx8x8_to<DT>(u32x2{v1[2], v1[3]}, sc);
                    } else {
#pragma unroll
                        for (int m = 0; m < 4; ++m) ao[rb][m] = src[m];
                    }
                }
#pragma unroll
                for (int b = 0; b < CPL; ++b) {
                    const uint32_t sb = s_sc[b * 16 * kb + kq];
                    const float sc = __uint_as_float((in ? sb : 127u) << 23);
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const u32x4 wo = mx4x8_to<DT>(wv[i][b][m], sc);
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) acc[rb][b] = mfma16<DT>(ao[rb][m], wo, acc[rb][b]);
                    }
                }
            };
            // full rounds, each step's slot refilled behind it; then what is left,
            // one branch inside the other (a join would wait for every load)
            int st = 0;
            for (; st + RING < n; st += RING) {
#pragma unroll
                for (int i = 0; i < RING; ++i) {
                    compute(i, st + i);
                    __builtin_amdgcn_sched_barrier(0);
                    load(i, st + i + RING);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            auto rest = [&](auto self, auto ic) -> void {
                constexpr int i = decltype(ic)::value;
                if constexpr (i < RING) {
                    if (st + i < n) {
                        compute(i, st + i);
                        __builtin_amdgcn_sched_barrier(0);
                        self(self, std::integral_constant<int, i + 1>{});
                    }
                }
            };
            rest(rest, std::integral_constant<int, 0>{});
        }

        // parts to LDS: lane (g, li) holds rows 4g .. 4g+3 of each row block at
        // column 16b + li
        __syncthreads();
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int v = 0; v < 4; ++v)
#pragma unroll
                for (int b = 0; b < CPL; ++b)
                    s_part[(wave * RB * 16 + rb * 16 + 4 * g + v) * SPW + 16 * b + li] = acc[rb][b][v];
        __syncthreads();
        // every thread: 8 consecutive columns of one row, the parts in wave order
        auto part_sums = [&](int m, int c8, int tn, float (&y)[8]) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                f32x4 v = *reinterpret_cast<const f32x4*>(s_part + (tn * KP * RB * 16 + m) * SPW + c8 + 4 * half);
#pragma unroll
                for (int pt = 1; pt < KP; ++pt) {
                    const f32x4 w =
                        *reinterpret_cast<const f32x4*>(s_part + ((tn * KP + pt) * RB * 16 + m) * SPW + c8 + 4 * half);
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] += w[j];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) y[4 * half + j] = v[j];
            }
        };
        constexpr int CH = WGC / 8;
        // (N is a multiple of 32: 8 columns lie wholly inside or outside)
        if constexpr (GATHER) {
            with_act(a.act, [&](auto act_c) {
                constexpr int ACT = decltype(act_c)::value;
                for (int q = tid; q < m_valid * CH; q += NT) {
                    const int m = q / CH, c8 = (q - m * CH) * 8;
                    if (col0 + c8 >= N) continue;
                    float y0[8], y1[8], h[8];
                    part_sums(m, c8, 0, y0);
                    if constexpr (DUAL) part_sums(m, c8, 1, y1);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[j] = DUAL ? act_t<ACT>(y0[j]) * y1[j] : act_t<ACT>(y0[j]);
                    u32x4 o;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = pack2<DT>(h[2 * j], h[2 * j + 1]);
                    *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(a.C) + (long long)s_rows[c0 + m] * N + col0 + c8) = o;
                }
            });
        } else {
            for (int q = tid; q < m_valid * CH; q += NT) {
                const int m = q / CH, c8 = (q - m * CH) * 8;
                if (col0 + c8 >= N) continue;
                float y[8];
                part_sums(m, c8, 0, y);
                float* dst = a.part + (long long)s_rows[c0 + m] * N + col0 + c8;
                *reinterpret_cast<f32x4*>(dst) = f32x4{y[0], y[1], y[2], y[3]};
                *reinterpret_cast<f32x4*>(dst + 4) = f32x4{y[4], y[5], y[6], y[7]};
            }
        }
    }
}

// Down / fc2 of a few tokens with the sum over a token's experts in the same launch:
// a workgroup has 16 columns of one token, its 8 waves the token's slots (and K
// parts of them where the slots are few). A wave streams its expert's 16 columns
// like the kernel above, rows and scales through its own LDS (it waits for its own
// DMA only); the MFMA's 16 rows are the one row. Then out = sum_j w_j y_j in slot
// order, each y_j its K parts in order. No partial rows in memory and no finishing
// launch; tokens of one expert read its weights each. T=1 down:
// Qwen3-30B-A3B 6.4 us (two launches 5.5 + 2.8), Qwen3 5.5: trips to cold memory.
constexpr int kSumWaves = 8;

template <int DT>
__global__ __launch_bounds__(64 * kSumWaves) void mx_dec_sum_k(DecArgs a, MxDecSum f) {
    constexpr int RING = 8;
    __shared__ float s_part[kMxSumSlots][16];
    __shared__ __attribute__((aligned(16))) char s_zero[kSumWaves][256];
    extern __shared__ __attribute__((aligned(16))) char s_dyn[];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, li = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int t = blockIdx.y, col0 = blockIdx.x * 16;
    const int K = a.K, kb = K / 32;
    const int rowb = (2 * K + 1023) & ~1023, scb = (16 * kb + 1023) & ~1023;
    char* s_row = s_dyn + wave * (rowb + scb);
    reinterpret_cast<uint32_t*>(s_zero[wave])[lane] = 0u;  // (read by this wave alone, in order)
    const uint8_t* s_sc = reinterpret_cast<const uint8_t*>(s_row + rowb) + li * kb + g;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_addr(s_row));
    const int slot0 = wave / f.parts, part = wave - slot0 * f.parts, step = kSumWaves / f.parts;
    const int nst = (K + 127) / 128, per = (nst + f.parts - 1) / f.parts;
    const int lo = part * per, n = min(per, nst - lo);
    const long long wbytes = a.strideB / 2, sbytes = a.strideB / 32;
    const i32x4 rA = make_rsrc(a.A, a.a_bytes);
    const uint32_t wlane = (uint32_t)(col0 + li) * (uint32_t)(K / 2) + 16u * (uint32_t)g;

    for (int j = slot0; j < f.k; j += step) {
        const int p = t * f.k + j;
        const uint32_t e = __builtin_amdgcn_readfirstlane(a.idx[p]);
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if (e < (uint32_t)a.E && n > 0) {
            for (int q = 0; q < rowb >> 10; ++q) {
                const uint32_t at = (uint32_t)q * 1024u + 16u * (uint32_t)lane;
                dma16(rA, lds0 + (uint32_t)(q * 1024), at < 2u * (uint32_t)K ? (uint32_t)p * 2u * (uint32_t)K + at : kOob);
            }
            const i32x4 rs = make_rsrc(a.mx0 + e * sbytes, sbytes);
            for (int q = 0; q < scb >> 10; ++q)
                dma16(rs, lds0 + (uint32_t)(rowb + q * 1024),
                      (uint32_t)col0 * (uint32_t)kb + (uint32_t)q * 1024u + 16u * (uint32_t)lane);
            const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<char*>(reinterpret_cast<const char*>(a.B0)) + e * wbytes, 0, (int)wbytes, 0x00020000);
            u32x4 wv[RING];
            auto load = [&](int i, int st) {
                const int k = (lo + st) * 128;
                const bool in = (st < n) & (k + 32 * g < K);
                wv[i] = __builtin_amdgcn_raw_buffer_load_b128(rw, in ? wlane + (uint32_t)(k / 2) : kOob, 0, 0);
            };
#pragma unroll
            for (int i = 0; i < RING; ++i) load(i, i);
            wait_vm<RING>();  // the row and the scales
            for (int st0 = 0; st0 < n; st0 += RING) {
#pragma unroll
                for (int i = 0; i < RING; ++i) {
                    // Steps past the last multiply zeros by zero codes (the row itself may
                    // hold an infinity, and zero times that is a NaN). Branches around
                    // them, one in the other, keep a step's reads from moving up:
                    // Qwen3-30B-A3B T=6 33.1 against 29.7 us.
                    const bool in = st0 + i < n;
                    const int k = (lo + min(st0 + i, n - 1)) * 128, kq = k / 32;
                    const u32x4* src = reinterpret_cast<const u32x4*>((in ? s_row + 2 * k : s_zero[wave]) + 64 * g);
                    const uint32_t sb = s_sc[kq];
                    const float sc = __uint_as_float((in && kq + g < kb ? sb : 127u) << 23);
#pragma unroll
                    for (int m = 0; m < 4; ++m) acc = mfma16<DT>(src[m], mx4x8_to<DT>(wv[i][m], sc), acc);
                    if (st0 + RING < n) load(i, st0 + i + RING);
                }
            }
            asm volatile("" ::: "memory");  // (the LDS of the next slot: after these reads)
        }
        if (g == 0) s_part[j * f.parts + part][li] = acc[0];
    }
    __syncthreads();
    if (tid < 16) {
        const long long at = (long long)t * a.N + col0 + tid;
        uint16_t* out = reinterpret_cast<uint16_t*>(f.out);
        float s = f.overwrite ? 0.f : Elem<DT>::to_f32(out[at]);
        for (int j = 0; j < f.k; ++j) {
            if (a.idx[t * f.k + j] >= (uint32_t)a.E) continue;  // (a dropped pair)
            float y = s_part[j * f.parts][tid];
            for (int q = 1; q < f.parts; ++q) y += s_part[j * f.parts + q][tid];
            s = fmaf(f.w[t * f.k + j], y, s);
        }
        out[at] = Elem<DT>::from_f32(s);
    }
}

template <int DT, int MODE, int RB, int CPL, bool X8>
hipError_t launch_one(const DecArgs& a, hipStream_t stream) {
    const long long nwg = (long long)a.max_groups * a.nblk;
    if (nwg > 0x7fffffffLL) return hipErrorInvalidValue;
    if (nwg <= 0) return hipSuccess;
    // LDS: scales, then the rows of one chunk or the waves' parts. (A token may name
    // one expert in several slots: up to P rows.)
    constexpr int AB = X8 ? 1 : 2, PART = kMxWaves * RB * 16 * (16 * CPL + 4) * 4;
    const long long rows = std::min(a.P, 16 * RB), kb = a.K / 32;
    const long long scales = (MODE == kGateUp ? 2 : 1) * ((16 * CPL * kb + 1023) / 1024 * 1024);
    const long long first = scales + (X8 ? rows * ((kb + 255) / 256 * 256) : 0);
    const long long most = ((kMxDecLds - first) / rows - 16) / 1024 * 1024 / AB;  // k of the rows that fit
    if (first + PART > kMxDecLds || most < 512) return hipErrorInvalidValue;
    DecArgs b = a;
    b.lds_rows = (int)first;
    const long long chunks = (a.K + most - 1) / most;
    b.kc = (int)(((a.K + chunks - 1) / chunks + 511) / 512 * 512);
    const long long pitch = ((long long)std::min(b.kc, a.K) * AB + 1023) / 1024 * 1024 + 16;
    const long long lds = first + std::max<long long>(rows * pitch, PART);
    if (lds > kMxDecLds) return hipErrorInvalidValue;
    hipLaunchKernelGGL((mx_dec_k<DT, MODE, RB, CPL, X8>), dim3((unsigned)nwg), dim3(64 * kMxWaves), (unsigned)lds, stream, b);
    return hipGetLastError();
}
template <int DT, int MODE, int RB, bool X8>
hipError_t launch_cols(const DecArgs& a, hipStream_t stream) {
    switch (a.cpl) {
        case 2: return launch_one<DT, MODE, RB, 2, X8>(a, stream);
        case 3: return launch_one<DT, MODE, RB, 3, X8>(a, stream);
        case 4: return launch_one<DT, MODE, RB, 4, X8>(a, stream);
        case 6: return launch_one<DT, MODE, RB, 6, X8>(a, stream);
        case 8:
            if constexpr (RB == 1) return launch_one<DT, MODE, RB, 8, X8>(a, stream);
            return hipErrorInvalidValue;
        default: return hipErrorInvalidValue;
    }
}
template <int DT, int MODE>
hipError_t launch_mode(const DecArgs& a, hipStream_t stream) {
    if constexpr (MODE != kDownRows) {
        if (a.xs) return a.rows_max > 16 ? launch_cols<DT, MODE, 2, true>(a, stream) : launch_cols<DT, MODE, 1, true>(a, stream);
    }
    return a.rows_max > 16 ? launch_cols<DT, MODE, 2, false>(a, stream) : launch_cols<DT, MODE, 1, false>(a, stream);
}
template <int DT>
hipError_t launch_dt(int mode, const DecArgs& a, hipStream_t stream) {
    switch (mode) {
        case kGateUp: return launch_mode<DT, kGateUp>(a, stream);
        case kFc1: return launch_mode<DT, kFc1>(a, stream);
        case kDownRows:
        case kFc2Rows: return launch_mode<DT, kDownRows>(a, stream);  // ([N,K] either way)
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

int mx_dec_cols(int mode, int rows_max, int K) {
    // (two row blocks of 8 columns do not fit 256 registers; scales at most 32 KB)
    const int most = (mode == kGateUp ? 1 : 2) * 32768 / K;
    return std::min(rows_max > 16 ? 6 : 8, most);
}

hipError_t launch_mx_dec_sum(int dtype, const DecArgs& a, const MxDecSum& s, hipStream_t stream) {
    MxDecSum f = s;
    f.parts = f.k > 4 ? 1 : f.k > 2 ? 2 : f.k > 1 ? 4 : 8;
    const int lds = kSumWaves * ((2 * a.K + 1023) / 1024 * 1024 + (a.K / 2 + 1023) / 1024 * 1024);
    if (f.k < 1 || f.k * f.parts > kMxSumSlots || a.mx0 == nullptr || a.K % 32 || a.N % 32 || a.K > kMxSumMaxK ||
        f.T < 1 || f.T > 65535)
        return hipErrorInvalidValue;
    const dim3 grid((unsigned)(a.N / 16), (unsigned)f.T), block(64 * kSumWaves);
    if (dtype == kBF16) hipLaunchKernelGGL(mx_dec_sum_k<kBF16>, grid, block, (unsigned)lds, stream, a, f);
    else if (dtype == kF16) hipLaunchKernelGGL(mx_dec_sum_k<kF16>, grid, block, (unsigned)lds, stream, a, f);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_mx_dec(int mode, int dtype, const DecArgs& a, hipStream_t stream) {
    if (a.P > kDecMaxPairs || a.E > kDecMaxE || a.ks_lim != 1 || a.meta == nullptr || a.mx0 == nullptr ||
        (mode == kGateUp && a.mx1 == nullptr) || a.K % 32 || a.N % 32)
        return hipErrorInvalidValue;
    if (dtype == kBF16) return launch_dt<kBF16>(mode, a, stream);
    if (dtype == kF16) return launch_dt<kF16>(mode, a, stream);
    return hipErrorInvalidValue;
}

}  // namespace cm
