// 4-bit weights: OCP MXFP4. A weight is e2m1 (one sign, two exponent and one
// mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) times a power of
// two that 32 weights in a row along K share, held as the byte e + 127 (E8M0; 255:
// NaN). Codes [E][N][K/2] bytes, K-contiguous, even k in the low half of a byte;
// scales [E][N][K/32] bytes: 4.25 bits per weight.
//
// quantize: e is the least with max|w| <= 6 * 2^e over the 32 (no value is cut
// off), 0 as the byte for 32 zeros, 255 where a weight is not finite; w / 2^e, an
// exact division, goes to the nearest e2m1, ties to the even code.
// dequantize: value * 2^e, exact in f32 and bf16 (an infinity from 2^128 on, to
// which weights past 3.5 * 2^126 go); in f16 it is rounded where it leaves that type's
// range.
// MXFP8 rows (e4m3 codes, the same scales): rows8_to dequantizes those.
// All bound by their bytes. quantize (once per weight tensor) bf16 128 x 2048 x 768:
// [K,N] 181 us (2.8 TB/s; neighbouring threads read neighbouring columns but write
// 16 bytes apart), [N,K] 382 us (each thread its own 64 bytes); dequantize 123 us
// (4.1 TB/s).
#include <algorithm>

#include "cm_common.hpp"
#include "cm_internal.hpp"

namespace cm {

namespace {

// 2^(s - 127); NaN for 255
__device__ __forceinline__ float e8m0_to_f32(uint32_t s) {
    return __uint_as_float(s == 255u ? 0x7fc00000u : s == 0u ? 0x00400000u : s << 23);
}
__device__ __forceinline__ float e2m1_to_f32(uint32_t c) {
    // exponent 0: mantissa * 0.5; else 2^(exponent - 1) * (1 + mantissa / 2)
    const uint32_t e = (c >> 1) & 3u, m = c & 1u;
    const float v = e == 0u ? 0.5f * (float)m : __uint_as_float(((126u + e) << 23) | (m << 22));
    return (c & 8u) ? -v : v;
}
__device__ __forceinline__ uint32_t f32_to_e2m1(float v) {
    const float a = fabsf(v);
    uint32_t c = a > 0.25f;
    c += a >= 0.75f;
    c += a > 1.25f;
    c += a >= 1.75f;
    c += a > 2.5f;
    c += a >= 3.5f;
    c += a > 5.0f;
    return c | (v < 0.f ? 8u : 0u);
}

// One thread per 32 weights of a column (kn: neighbouring threads read
// neighbouring columns).
template <int DT>
__global__ __launch_bounds__(256) void quantize_mxfp4_k(const void* __restrict__ w, int E, int K, int N, int kn,
                                                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    typedef typename Elem<DT>::storage S;
    const long long nb = K / 32, total = (long long)E * N * nb;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        long long e, n, b;
        if (kn) {
            n = i % N;
            b = i / N % nb;
            e = i / N / nb;
        } else {
            b = i % nb;
            n = i / nb % N;
            e = i / nb / N;
        }
        const S* src = reinterpret_cast<const S*>(w) + e * K * (long long)N + (kn ? b * 32 * N + n : n * K + b * 32);
        const long long step = kn ? N : 1;
        float v[32];
        uint32_t m = 0;
#pragma unroll
        for (int q = 0; q < 32; ++q) {
            v[q] = Elem<DT>::to_f32(src[q * step]);
            m = max(m, __float_as_uint(v[q]) & 0x7fffffffu);
        }
        // 6 = 1.5 * 2^2: the exponent is one more where the mantissa is above 1.5
        const int ex = (int)((m + 0x3fffffu) >> 23) - 2;
        const uint32_t s = m >= 0x7f800000u ? 255u : (uint32_t)max(ex, 0);
        const float inv = s == 255u ? 0.f : __uint_as_float(s >= 254u ? 0x00400000u : (254u - s) << 23);
        u32x4 o;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t x = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) x |= f32_to_e2m1(s == 255u ? 0.f : v[8 * d + q] * inv) << (4 * q);
            o[d] = x;
        }
        const long long blk = (e * N + n) * nb + b;
        *reinterpret_cast<u32x4*>(codes + blk * 16) = o;
        scales[blk] = (uint8_t)s;
    }
}

// One thread per 8 weights (a u32 of codes).
template <int DT>
__global__ __launch_bounds__(256) void dequantize_mxfp4_k(const uint32_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, long long total,
                                                          typename Elem<DT>::storage* __restrict__ out) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const uint32_t c = codes[i];
        const float s = e8m0_to_f32(scales[i >> 2]);
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = e2m1_to_f32((c >> (4 * q)) & 15u) * s;
        if constexpr (DT == kF32) {
            f32x4* p = reinterpret_cast<f32x4*>(out + i * 8);
            p[0] = f32x4{v[0], v[1], v[2], v[3]};
            p[1] = f32x4{v[4], v[5], v[6], v[7]};
        } else {
            u32x4 o;
#pragma unroll
            for (int q = 0; q < 4; ++q) o[q] = pack2<DT>(v[2 * q], v[2 * q + 1]);
            *reinterpret_cast<u32x4*>(out + i * 8) = o;
        }
    }
}

// One thread per 8 values of MXFP8 rows.
template <int DT>
__global__ __launch_bounds__(256) void rows8_to_k(const u32x2* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                  long long total, uint16_t* __restrict__ out) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const u32x2 c = codes[i];
        const float s = e8m0_to_f32(scales[i >> 2]);
        u32x4 o;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[q], false);
            const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[q], true);
            o[2 * q] = pack2<DT>(a[0] * s, a[1] * s);
            o[2 * q + 1] = pack2<DT>(b[0] * s, b[1] * s);
        }
        *reinterpret_cast<u32x4*>(out + i * 8) = o;
    }
}

unsigned blocks_for(long long n) { return (unsigned)std::min<long long>((n + 255) / 256, 1 << 20); }

}  // namespace

hipError_t launch_quantize_mxfp4(const void* w, int dtype, int E, int K, int N, int kn, uint8_t* codes,
                                 uint8_t* scales, hipStream_t stream) {
    const long long total = (long long)E * N * (K / 32);
    if (total <= 0) return hipSuccess;
    const dim3 g(blocks_for(total)), b(256);
    if (dtype == kBF16) hipLaunchKernelGGL(quantize_mxfp4_k<kBF16>, g, b, 0, stream, w, E, K, N, kn, codes, scales);
    else if (dtype == kF16) hipLaunchKernelGGL(quantize_mxfp4_k<kF16>, g, b, 0, stream, w, E, K, N, kn, codes, scales);
    else hipLaunchKernelGGL(quantize_mxfp4_k<kF32>, g, b, 0, stream, w, E, K, N, kn, codes, scales);
    return hipGetLastError();
}

hipError_t launch_dequantize_mxfp4(const void* codes, const void* scales, int E, int N, int K, void* out, int dtype,
                                   hipStream_t stream) {
    const long long total = (long long)E * N * (K / 8);
    if (total <= 0) return hipSuccess;
    const dim3 g(blocks_for(total)), b(256);
    const uint32_t* c = reinterpret_cast<const uint32_t*>(codes);
    const uint8_t* s = reinterpret_cast<const uint8_t*>(scales);
    if (dtype == kBF16)
        hipLaunchKernelGGL(dequantize_mxfp4_k<kBF16>, g, b, 0, stream, c, s, total, reinterpret_cast<uint16_t*>(out));
    else if (dtype == kF16)
        hipLaunchKernelGGL(dequantize_mxfp4_k<kF16>, g, b, 0, stream, c, s, total, reinterpret_cast<uint16_t*>(out));
    else
        hipLaunchKernelGGL(dequantize_mxfp4_k<kF32>, g, b, 0, stream, c, s, total, reinterpret_cast<float*>(out));
    return hipGetLastError();
}

hipError_t launch_rows8_to(const void* codes, const void* scales, long long T, int H, void* out, int dtype,
                           hipStream_t stream) {
    const long long total = T * (H / 8);
    if (total <= 0) return hipSuccess;
    const dim3 g(blocks_for(total)), b(256);
    const u32x2* c = reinterpret_cast<const u32x2*>(codes);
    const uint8_t* s = reinterpret_cast<const uint8_t*>(scales);
    if (dtype == kBF16) hipLaunchKernelGGL(rows8_to_k<kBF16>, g, b, 0, stream, c, s, total, reinterpret_cast<uint16_t*>(out));
    else hipLaunchKernelGGL(rows8_to_k<kF16>, g, b, 0, stream, c, s, total, reinterpret_cast<uint16_t*>(out));
    return hipGetLastError();
}

}  // namespace cm
