// Routing with groups: scores, a bias for the choice, a choice of groups, the
// top k and their weights, for one token per row of logits.
//
//   s_e = softmax(l)_e  or  1 / (1 + exp(-l_e))
//   c_e = s_e + b_e                                  (what the choice goes by)
//   group score = the sum of the group's `group_top` largest c
//   the `topk_groups` best groups, then the k best c in them, ties to the lower index
//   w_j = s at the chosen, / their sum (renormalize), * scale
//
// Scores are 64-bit: the choice is the one the definition makes in exact
// arithmetic unless two c differ by less than 1e-15, whatever the biases. A NaN
// counts as -infinity in the choice; logits of -infinity have score 0, also
// where a row has no others (then every weight is 0).
//
// One wave per row; lane g owns the VPT experts from g * VPT on.
#include <limits.h>
#include <math.h>

#include "cm_common.hpp"
#include "cm_internal.hpp"

namespace cm {

namespace {

constexpr int kRouteWaves = 4;

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// (value, index) of the best of the wave: the larger value, then the lower
// index; index INT_MAX: none
__device__ __forceinline__ void wave_best(double& v, int& i) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const double ov = __shfl_xor(v, m);
        const int oi = __shfl_xor(i, m);
        const bool take = oi != INT_MAX && (i == INT_MAX || ov > v || (ov == v && oi < i));
        v = take ? ov : v;
        i = take ? oi : i;
    }
}

template <int VPT, int DT>
__global__ __launch_bounds__(64 * kRouteWaves) void route_k(RouteArgs a) {
    typedef typename Elem<DT>::storage S;
    __shared__ double s_buf[kRouteWaves][64 * VPT];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long row = (long long)blockIdx.x * kRouteWaves + wave;
    const bool live = row < a.T;
    const S* src = reinterpret_cast<const S*>(a.logits) + (live ? row : 0) * (long long)a.E;
    double* buf = s_buf[wave];

    double s[VPT], c[VPT];
    uint32_t alive = 0;
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int e = lane * VPT + j;
        if (e < a.E) alive |= 1u << j;
        s[j] = e < a.E ? (double)Elem<DT>::to_f32(src[e]) : -(double)INFINITY;
    }
    if (a.score == kRouteSoftmax) {
        double m = -(double)INFINITY;
#pragma unroll
        for (int j = 0; j < VPT; ++j) m = fmax(m, s[j]);
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) m = fmax(m, __shfl_xor(m, x));
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            s[j] = s[j] == -(double)INFINITY ? 0.0 : exp(s[j] - m);
            sum += s[j];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int j = 0; j < VPT; ++j) s[j] = sum == 0.0 ? 0.0 : s[j] / sum;
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j) s[j] = 1.0 / (1.0 + exp(-s[j]));
    }
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int e = lane * VPT + j;
        c[j] = s[j] + (a.bias && e < a.E ? (double)a.bias[e] : 0.0);
        if (!(c[j] == c[j])) c[j] = -(double)INFINITY;
    }

    if (a.topk_groups < a.groups) {
        const int per = a.E / a.groups;
#pragma unroll
        for (int j = 0; j < VPT; ++j) buf[lane * VPT + j] = c[j];
        __syncthreads();
        double b1 = -(double)INFINITY, b2 = -(double)INFINITY;
        if (lane < a.groups) {
            for (int q = 0; q < per; ++q) {
                const double v = buf[lane * per + q];
                b2 = fmax(b2, fmin(b1, v));
                b1 = fmax(b1, v);
            }
        }
        double gs = a.group_top == 1 ? b1 : b1 + b2;
        if (!(gs == gs)) gs = -(double)INFINITY;
        int gi = lane < a.groups ? lane : INT_MAX;
        uint64_t keep = 0;
        for (int q = 0; q < a.topk_groups; ++q) {
            double v = gs;
            int i = gi;
            wave_best(v, i);
            keep |= 1ull << i;
            if (gi == i) gi = INT_MAX;
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            if (!((keep >> ((lane * VPT + j) / per)) & 1ull)) alive &= ~(1u << j);
        __syncthreads();
    }

    double total = 0.0;
    for (int q = 0; q < a.k; ++q) {
        double v = -(double)INFINITY;
        int i = INT_MAX;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            if (((alive >> j) & 1u) && (i == INT_MAX || c[j] > v)) {
                v = c[j];
                i = lane * VPT + j;
            }
        }
        wave_best(v, i);
        double w = 0.0;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            if (i == lane * VPT + j) {
                w = s[j];
                alive &= ~(1u << j);
            }
        }
        w = __shfl(w, i / VPT);
        total += w;
        if (lane == 0) {
            buf[q] = w;
            if (live) a.idx[row * a.k + q] = (uint32_t)i;
        }
    }
    __syncthreads();
    if (!live) return;
    for (int q = lane; q < a.k; q += 64) {
        double w = buf[q];
        if (a.renorm) w = total == 0.0 ? 0.0 : w / total;
        a.w[row * a.k + q] = (float)(w * (double)a.scale);
        a.ei[row * a.k + q] = (uint32_t)((long long)q * a.T + row);
    }
}

template <int VPT>
hipError_t launch_vpt(const RouteArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)((a.T + kRouteWaves - 1) / kRouteWaves)), block(64 * kRouteWaves);
    if (a.dtype == kF32) hipLaunchKernelGGL((route_k<VPT, kF32>), grid, block, 0, stream, a);
    else if (a.dtype == kBF16) hipLaunchKernelGGL((route_k<VPT, kBF16>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((route_k<VPT, kF16>), grid, block, 0, stream, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_route(const RouteArgs& a, hipStream_t stream) {
    if (a.T <= 0) return hipSuccess;
    if (a.E <= 64) return launch_vpt<1>(a, stream);
    if (a.E <= 128) return launch_vpt<2>(a, stream);
    if (a.E <= 256) return launch_vpt<4>(a, stream);
    if (a.E <= 512) return launch_vpt<8>(a, stream);
    return launch_vpt<16>(a, stream);
}

}  // namespace cm
