// The residual's addition and the root-mean-square norm of token rows, with an
// 8-bit form of the result:
//
//   z = x + r                       (f32; x where there is no residual)
//   r' = dtype(z)
//   y = z * 1/sqrt(mean(z^2) + eps) * w     (of z before its rounding)
//   output = dtype(y)
//   codes, scales: per 32 values along the row the least power of two 2^e with
//     max|y| <= 448 * 2^e, as the byte e + 127 (0 for 32 zeros, 255 with every
//     code NaN where a value is not finite), and e4m3(y / 2^e), ties to even
//     (MXFP8 of y before any rounding)
//
// Bound by its bytes: every element of x and r is read once and held in f32
// registers between the sum of squares (in f64) and the outputs. NT threads share a
// row, each holding CH chunks of 8 consecutive elements (16-byte loads of 16-bit
// rows); 4 neighbouring lanes hold a block of 32. bf16, all outputs: T=8191 H 4096
// 60 us (5.1 TB/s, what a copy reaches), f16 T=1000 H 2880 without codes 6.4 us with
// its launch, T=1 H 2048 2.7 us on the GPU (loads, two barriers' worth of
// reduction, stores).
#include "cm_common.hpp"
#include "cm_internal.hpp"

namespace cm {

namespace {

template <int DT>
__device__ __forceinline__ void load8(const void* base, long long at, float (&v)[8]) {
    if constexpr (DT == kF32) {
        const f32x4* p = reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(base) + at);
        const f32x4 a = p[0], b = p[1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = a[j];
            v[4 + j] = b[j];
        }
    } else {
        const u32x4 q = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(base) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = Elem<DT>::to_f32((uint16_t)(q[j] & 0xffffu));
            v[2 * j + 1] = Elem<DT>::to_f32((uint16_t)(q[j] >> 16));
        }
    }
}
template <int DT>
__device__ __forceinline__ void store8(void* base, long long at, const float (&v)[8]) {
    if constexpr (DT == kF32) {
        f32x4* p = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(base) + at);
        p[0] = f32x4{v[0], v[1], v[2], v[3]};
        p[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        u32x4 q;
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = pack2<DT>(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(base) + at) = q;
    }
}

// Codes of this lane's 8 values of a block of 32 (4 neighbouring lanes), and
// the block's scale byte.
__device__ __forceinline__ u32x2 mxfp8_codes(const float (&y)[8], uint32_t& scale) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(y[j]) & 0x7fffffffu);
    m = max(m, (uint32_t)xor_lane_i32<1>((int)m));
    m = max(m, (uint32_t)xor_lane_i32<2>((int)m));
    // 448 = 1.75 * 2^8: the exponent is one more where the mantissa is above 1.75
    const int e = (int)((m + 0x1fffffu) >> 23) - 8;
    scale = m >= 0x7f800000u ? 255u : (uint32_t)max(e, 0);
    // 2^(127 - scale) (scale 254: 2^-127, below the normal range)
    const float inv = scale == 255u ? __uint_as_float(0x7fc00000u)
                                    : __uint_as_float(scale >= 254u ? 0x00400000u : (254u - scale) << 23);
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * inv, y[5] * inv, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * inv, y[7] * inv, hi, true);
    return u32x2{(uint32_t)lo, (uint32_t)hi};
}

// 1/sqrt(mean + eps) as a sum of two f32. With it y = z * inv * w comes as a sum of
// two as well, within 2^-40 of its value (a y in f32's normal range). A y rounded to f32 can fall on the middle
// between two 8-bit codes, or on the border of two scales, and then goes the wrong
// way (some 20 of 33 million values); rounded to odd (cut off, the last bit set
// where anything was) it stays on its side. Where 1/sqrt(mean + eps) or its second
// part leaves f32's normal range (rows near the ends of it), the two hold it times
// 2^-sh, and z goes in times 2^sh.
struct InvNorm {
    float hi, lo;
    int sh = 0;
    __device__ __forceinline__ InvNorm(double sq, int H, float eps) {
        const double m = sq * (1.0 / (double)H) + (double)eps;
        double v;
        if (m > 1e-30 && m < 1e30) {  // (one Newton step on the f32 value: 2^-42)
            v = (double)__builtin_amdgcn_rsqf((float)m);
            v = fma(0.5 * v, fma(-m * v, v, 1.0), v);
        } else {
            v = 1.0 / sqrt(m);
            if (v > 0.0 && v < (double)INFINITY) v = frexp(v, &sh);
        }
        hi = (float)v;
        lo = hi < INFINITY ? (float)(v - (double)hi) : 0.f;
    }
    // y to the nearest f32; rest: what that left out
    __device__ __forceinline__ float times(float z, float w, float& rest) const {
        z = ldexpf(z, sh);
        const float p = z * hi;
        const float e = fmaf(z, lo, fmaf(z, hi, -p));  // (|z| hi <= sqrt(H): no overflow)
        float t = e * w;
        t = fabsf(t) < INFINITY ? t : 0.f;
        const float y = fmaf(p, w, t);
        rest = fmaf(p, w, -y) + t;
        return y;
    }
};
__device__ __forceinline__ float to_odd(float y, float rest) {
    uint32_t u = __float_as_uint(y);
    const bool below = (__float_as_uint(rest) ^ u) >> 31;  // (nearer to zero than y)
    if (fabsf(rest) > 0.f && fabsf(y) < INFINITY && y != 0.f) u = (u - (below ? 1u : 0u)) | 1u;
    return __uint_as_float(u);
}

template <int NT>
__device__ __forceinline__ double row_sum(double v, double* s_part) {
    constexpr int IN = NT < 64 ? NT : 64;
#pragma unroll
    for (int m = 1; m < IN; m <<= 1) v += __shfl_xor(v, m);
    if constexpr (NT > 64) {
        if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) v += s_part[w];
    }
    return v;
}

template <int DT, int NT, int CH>
__global__ __launch_bounds__(NT > kNormThreads ? NT : kNormThreads) void rms_norm_k(NormArgs a) {
    constexpr int RPW = NT > kNormThreads ? 1 : kNormThreads / NT;  // rows per workgroup (of 256 threads)
    __shared__ double s_part[NT > 64 ? NT / 64 : 1];
    const int t = threadIdx.x % NT;
    const long long row = (long long)blockIdx.x * RPW + threadIdx.x / NT;
    if (row >= a.T) return;  // (NT > 64: one row per workgroup, all its threads stay)
    const long long base = row * (long long)a.H;
    float z[CH][8], w[CH][8];  // (the weights before the reduction, not behind it)
    double sq = 0.0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int h = (c * NT + t) * 8;
        if (h >= a.H) continue;
        load8<DT>(a.x, base + h, z[c]);
        if (a.residual) {
            float r[8];
            load8<DT>(a.residual, base + h, r);
            load8<DT>(a.weight, h, w[c]);
#pragma unroll
            for (int j = 0; j < 8; ++j) z[c][j] += r[j];
        } else {
            load8<DT>(a.weight, h, w[c]);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sq = fma((double)z[c][j], (double)z[c][j], sq);
    }
    sq = row_sum<NT>(sq, s_part);
    const InvNorm inv(sq, a.H, a.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int h = (c * NT + t) * 8;
        if (h >= a.H) continue;
        if (a.residual_out) store8<DT>(a.residual_out, base + h, z[c]);
        float y[8], rest[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = inv.times(z[c][j], w[c][j], rest[j]);
        if (a.out) store8<DT>(a.out, base + h, y);
        if (a.codes) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = to_odd(y[j], rest[j]);
            // (hidden sizes of 8-bit calls are multiples of 32: a block's four
            // lanes are all here)
            uint32_t s;
            const u32x2 q = mxfp8_codes(y, s);
            *reinterpret_cast<u32x2*>(a.codes + base + h) = q;
            if ((t & 3) == 0) a.scales[(base + h) >> 5] = (uint8_t)s;
        }
    }
}

// Any size and alignment, no 8-bit form: one workgroup per row, elements one by
// one, read a second time for the outputs.
template <int DT>
__global__ __launch_bounds__(kNormThreads) void rms_norm_any_k(NormArgs a) {
    typedef typename Elem<DT>::storage S;
    __shared__ double s_part[kNormThreads / 64];
    const long long base = (long long)blockIdx.x * a.H;
    const S* x = reinterpret_cast<const S*>(a.x) + base;
    const S* r = a.residual ? reinterpret_cast<const S*>(a.residual) + base : nullptr;
    auto at = [&](int h) { return Elem<DT>::to_f32(x[h]) + (r ? Elem<DT>::to_f32(r[h]) : 0.f); };
    double sq = 0.0;
    for (int h = threadIdx.x; h < a.H; h += kNormThreads) {
        const float z = at(h);
        sq = fma((double)z, (double)z, sq);
    }
    sq = row_sum<kNormThreads>(sq, s_part);
    const InvNorm inv(sq, a.H, a.eps);
    for (int h = threadIdx.x; h < a.H; h += kNormThreads) {
        const float z = at(h);
        if (a.residual_out) reinterpret_cast<S*>(a.residual_out)[base + h] = Elem<DT>::from_f32(z);
        float rest;
        if (a.out)
            reinterpret_cast<S*>(a.out)[base + h] =
                Elem<DT>::from_f32(inv.times(z, Elem<DT>::to_f32(reinterpret_cast<const S*>(a.weight)[h]), rest));
    }
}

template <int DT, int NT, int CH>
hipError_t launch_rows(const NormArgs& a, hipStream_t stream) {
    constexpr int RPW = NT > kNormThreads ? 1 : kNormThreads / NT;
    hipLaunchKernelGGL((rms_norm_k<DT, NT, CH>), dim3((unsigned)((a.T + RPW - 1) / RPW)),
                       dim3(NT > kNormThreads ? NT : kNormThreads), 0, stream, a);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_dt(const NormArgs& a, hipStream_t stream) {
    if (!a.vec || a.H > 32768) {
        if (a.codes) return hipErrorInvalidValue;
        hipLaunchKernelGGL(rms_norm_any_k<DT>, dim3((unsigned)a.T), dim3(kNormThreads), 0, stream, a);
        return hipGetLastError();
    }
    if (a.H <= 512) return launch_rows<DT, 64, 1>(a, stream);
    if (a.H <= 1024) return launch_rows<DT, 64, 2>(a, stream);
    if (a.H <= 2048) return launch_rows<DT, 256, 1>(a, stream);
    if (a.H <= 4096) return launch_rows<DT, 256, 2>(a, stream);
    if (a.H <= 8192) return launch_rows<DT, 256, 4>(a, stream);
    return launch_rows<DT, 1024, 4>(a, stream);
}

}  // namespace

hipError_t launch_add_rms_norm(const NormArgs& a, int dtype, hipStream_t stream) {
    if (a.T <= 0) return hipSuccess;
    if (dtype == kF32) return launch_dt<kF32>(a, stream);
    if (dtype == kBF16) return launch_dt<kBF16>(a, stream);
    return launch_dt<kF16>(a, stream);
}

}  // namespace cm
