// Routing with groups: scores, a bias for the choice, a choice of groups, the
// top k and their weights, for one token per row of logits.
//
//   s_e = softmax(l)_e  or  1 / (1 + exp(-l_e))
//   c_e = s_e + b_e                                  (what the choice goes by)
//   group score = the sum of the group's `group_top` largest c
//   the `topk_groups` best groups, then the k best c in them, ties to the lower index
//   w_j = s at the chosen, / their sum (renormalize), * scale
//
// Scores are 64-bit and c is rounded to 64 bits once: the choice is the one of exact
// arithmetic where two c differ by more than a few of their roundings, 2^-52 *
// max(1, |c|) (with a bias of 100 scores closer than 1.4e-14 tie). A NaN
// counts as -infinity in the choice; logits of -infinity have score 0, also
// where a row has no others (then every weight is 0). Weights are 64-bit values
// rounded to f32 once, in both forms of a row.
//
// Two forms of a row:
//
//  exact: one wave per row, all scores and the choice in f64. Every shape; and
//    every row the fast form is not sure of. f32 logits of 256 experts in 8 groups,
//    sigmoid and bias: T = 4099 / 32768 22 / 108 us, bound by f64 exponentials and
//    64-bit exchanges.
//  fast: LPR lanes per row, VPT experts each, scores in f32 within a known
//    distance tau of the exact ones. A group's lanes are its own (padded), so
//    its two best c meet in log2(lanes) exchanges, and its place among the groups
//    is counted from their scores. The choice runs on 32-bit keys: c on a grid
//    between the row's largest c and a bound the k + 1 best lie above, over the
//    slot number: one v_max_u32 per exchange finds value and expert together.
//    k + 2 rounds give the k best and the next two. Where two neighbours in that
//    order (or a group at the border of the choice) are closer than 2 tau and the
//    grid, and not an exact tie (equal logits and biases), or a value is not
//    finite, the row goes the exact way: about one in 15000 of normal f32 logits
//    (groups closer than 2.4e-6). The k weights come from f64 exponentials of the
//    chosen logits, one lane each; where a softmax is not renormalised they are
//    divided by the row's sum of f64 exponentials (T = 32768: bf16 logits of 128
//    experts 15.4 -> 18.0 us, f32 of 256 13.4 -> 20).
//    T = 4099 6.1 us, up to 11.8 where a row goes the exact way, T = 32768 16 to 22
//    (none to four such rows), where reading the logits takes 0.9 / 7: bound by such
//    a row's dependent steps and the VALU (T = 32768: 8 waves per SIMD
//    of 989 vector instructions each, 15 us: exponentials, keys, the lanes' sorted
//    lists, k + 2 rounds of exchanges). T = 1 of 128 experts 3.4 us. bf16 logits of
//    128 experts, softmax, T = 4099 / 32768 10 / 15 us, where reading takes 0.3 / 2.2.
//    Rows whose experts tie at the border of the choice, like a batch's padding rows of
//    equal logits without a bias, all go the exact way, one after the other in their
//    wave: T = 32768, 256 experts in 8 groups, the last eighth of the rows 47 us, every
//    row 99; 128 experts, softmax, 33 / 68.
#include <limits.h>
#include <math.h>

#include "cm_common.hpp"
#include "cm_internal.hpp"
#include "cm_select.hpp"

namespace cm {

namespace {

constexpr int kRouteWaves = 4;

__device__ __forceinline__ double wave_sum(double v) { return group_sum<64>(v); }

// (value, index) of the best of the wave: the larger value, then the lower
// index; index INT_MAX: none
template <int M>
__device__ __forceinline__ void best_step(double& v, int& i) {
    const uint64_t u = __double_as_longlong(v);
    uint32_t al, bl, ah, bh, ai, bi;
    lane_pair<M>((uint32_t)u, al, bl);
    lane_pair<M>((uint32_t)(u >> 32), ah, bh);
    lane_pair<M>((uint32_t)i, ai, bi);
    const double x = __longlong_as_double(((uint64_t)ah << 32) | al), y = __longlong_as_double(((uint64_t)bh << 32) | bl);
    const bool take = (int)bi != INT_MAX && ((int)ai == INT_MAX || y > x || (y == x && (int)bi < (int)ai));
    v = take ? y : x;
    i = (int)(take ? bi : ai);
}
__device__ __forceinline__ void wave_best(double& v, int& i) {
    best_step<1>(v, i);
    best_step<2>(v, i);
    best_step<4>(v, i);
    best_step<8>(v, i);
    best_step<16>(v, i);
    best_step<32>(v, i);
}
// LDS written by some lanes of the wave is read by others (LDS operations of a
// wave stay in order; this keeps the compiler's in order too)
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One row on one wave; buf: 64 * VPT doubles of this wave.
template <int VPT, int DT>
__device__ __forceinline__ void route_exact_row(const RouteArgs& a, long long row, double* buf) {
    typedef typename Elem<DT>::storage S;
    const int lane = threadIdx.x & 63;
    const S* src = reinterpret_cast<const S*>(a.logits) + row * (long long)a.E;
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
        wave_lds_fence();
        double b1 = -(double)INFINITY, b2 = -(double)INFINITY;
        // the lanes of a group (a power of two of them) share its experts
        const int lanes = 64 >> (32 - __builtin_clz((unsigned)(a.groups - 1)));
        const int g = lane / lanes, first = lane - g * lanes;
        if (g < a.groups) {
            for (int q = first; q < per; q += lanes) {
                const double v = buf[g * per + q];
                b2 = fmax(b2, fmin(b1, v));
                b1 = fmax(b1, v);
            }
        }
        for (int x = 1; x < lanes; x <<= 1) {
            const double o1 = __shfl_xor(b1, x), o2 = __shfl_xor(b2, x);
            b2 = fmax(fmin(b1, o1), fmax(b2, o2));
            b1 = fmax(b1, o1);
        }
        double gs = a.group_top == 1 ? b1 : b1 + b2;
        if (!(gs == gs)) gs = -(double)INFINITY;
        // its place among the groups, ties to the lower one
        int place = 0;
        for (int q = 0; q < a.groups; ++q) {
            const double v = __shfl(gs, q * lanes);
            place += v > gs || (v == gs && q < g);
        }
        const uint64_t keep = __ballot(g < a.groups && first == 0 && place < a.topk_groups);
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            if (lane * VPT + j < a.E && !((keep >> ((lane * VPT + j) / per * lanes)) & 1ull)) alive &= ~(1u << j);
        wave_lds_fence();
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
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            if (i == lane * VPT + j) {
                buf[q] = s[j];
                alive &= ~(1u << j);
            }
        }
        if (lane == 0) a.idx[row * a.k + q] = (uint32_t)i;
    }
    wave_lds_fence();
    if (a.renorm)
        for (int q = 0; q < a.k; ++q) total += buf[q];
    for (int q = lane; q < a.k; q += 64) {
        double w = buf[q];
        if (a.renorm) w = total == 0.0 ? 0.0 : w / total;
        a.w[row * a.k + q] = (float)(w * (double)a.scale);
        a.ei[row * a.k + q] = (uint32_t)((long long)q * a.T + row);
    }
    wave_lds_fence();
}

template <int VPT, int DT>
__global__ __launch_bounds__(64 * kRouteWaves) void route_exact_k(RouteArgs a) {
    __shared__ double s_buf[kRouteWaves][64 * VPT];
    const int wave = threadIdx.x >> 6;
    const long long row = (long long)blockIdx.x * kRouteWaves + wave;
    if (row < a.T) route_exact_row<VPT, DT>(a, row, s_buf[wave]);
}

// Sorted descending by Batcher's odd-even merges.
template <int N>
__device__ __forceinline__ void sort_desc(uint32_t* k) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int q = p; q >= 1; q /= 2)
#pragma unroll
            for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
                for (int i = 0; i < q; ++i)
                    if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const uint32_t x = k[i + j], y = k[i + j + q];
                        k[i + j] = max(x, y);
                        k[i + j + q] = min(x, y);
                    }
}

// v of the lane's partner over a step of 2M lanes, in f32 (both values to both lanes)
template <int M>
__device__ __forceinline__ void pair_f32(float v, float& x, float& y) {
    uint32_t a, b;
    lane_pair<M>(__float_as_uint(v), a, b);
    x = __uint_as_float(a);
    y = __uint_as_float(b);
}
// (b1, b2): the two largest of a group of lanes
template <int M>
__device__ __forceinline__ void top2_step(float& b1, float& b2) {
    float p1, q1, p2, q2;
    pair_f32<M>(b1, p1, q1);
    pair_f32<M>(b2, p2, q2);
    b1 = fmaxf(p1, q1);
    b2 = fmaxf(fminf(p1, q1), fmaxf(p2, q2));
}

// lanes_log2: lanes of a group (all LPR with one group); cells: experts of a
// group; many: the chosen groups have at least k + 2 lanes with experts.
struct RouteFast {
    int lanes_log2, cells, many;
};

// WHOLE: every lane holds VPT experts or none, and logits and biases are read 16
// bytes at a time.
template <int LPR, int VPT, int DT, bool WHOLE>
__global__ __launch_bounds__(64 * kRouteWaves, LPR * VPT <= 256 ? 5 : 4) void route_fast_k(RouteArgs a, RouteFast f) {
    typedef typename Elem<DT>::storage S;
    constexpr int RPW = 64 / LPR, SLOTS = LPR * VPT, VS = SLOTS > 64 ? SLOTS / 64 : 1;
    constexpr int IB = SLOTS == 64 ? 6 : SLOTS == 128 ? 7 : SLOTS == 256 ? 8 : SLOTS == 512 ? 9 : 10;
    constexpr int QB = 32 - IB;
    static_assert((1 << IB) == SLOTS, "slot bits");
    __shared__ double s_buf[kRouteWaves][64 * VS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sub = lane % LPR;
    const long long row0 = ((long long)blockIdx.x * kRouteWaves + wave) * RPW;
    if (row0 >= a.T) return;
    const long long row = min(row0 + lane / LPR, (long long)a.T - 1);
    const bool live = row0 + lane / LPR < a.T;
    const int grp = sub >> f.lanes_log2;
    const int cell = (sub - (grp << f.lanes_log2)) * VPT;  // first expert of this lane in its group
    const int groups = a.topk_groups < a.groups ? a.groups : 1;
    const int nval = grp < groups ? max(0, min(f.cells - cell, VPT)) : 0;
    const int e0 = grp * f.cells + cell;
    const S* src = reinterpret_cast<const S*>(a.logits) + row * (long long)a.E;
    // (WHOLE: a lane without experts computes on zeros and is left out lane by lane)
    auto ours = [&](int j) { return WHOLE || j < nval; };

    // scores and what the choice goes by
    float l[VPT], c[VPT], b[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) l[j] = b[j] = 0.f;
    if constexpr (WHOLE) {
        if (nval) {
#pragma unroll
            for (int v = 0; v < VPT * (int)sizeof(S) / 16; ++v) {
                const u32x4 q = reinterpret_cast<const u32x4*>(src + e0)[v];
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    if constexpr (DT == kF32) {
                        l[(4 * v + d) % VPT] = __uint_as_float(q[d]);
                    } else {
                        l[(8 * v + 2 * d) % VPT] = Elem<DT>::to_f32((uint16_t)(q[d] & 0xffffu));
                        l[(8 * v + 2 * d + 1) % VPT] = Elem<DT>::to_f32((uint16_t)(q[d] >> 16));
                    }
                }
            }
            if (a.bias) {
#pragma unroll
                for (int v = 0; v < VPT / 4; ++v) {
                    const f32x4 q = reinterpret_cast<const f32x4*>(a.bias + e0)[v];
#pragma unroll
                    for (int d = 0; d < 4; ++d) b[(4 * v + d) % VPT] = q[d];
                }
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j)
            if (j < nval) {
                l[j] = Elem<DT>::to_f32(src[e0 + j]);
                if (a.bias) b[j] = a.bias[e0 + j];
            }
    }
    // 2^(x log2 e) by v_exp_f32: the product's rounding is |x| 2^-24 of the value,
    // at most 0.23 * 2^-24 of a sigmoid (s (1 - s) |x|) and 0.37 * 2^-24 of the
    // largest exponential of a softmax (|x| e^-|x|)
    constexpr float kLog2e = 1.44269504088896341f;
    float m = 0.f, tau = 3.5e-7f;
    double total = 1.0;
    if (a.score == kRouteSoftmax) {
        m = -INFINITY;
#pragma unroll
        for (int j = 0; j < VPT; ++j) m = ours(j) ? fmaxf(m, l[j]) : m;
        m = group_max<LPR>(nval > 0 ? m : -INFINITY);
        float part[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            c[j] = ours(j) ? __builtin_amdgcn_exp2f((l[j] - m) * kLog2e) : 0.f;
            part[j] = c[j];
        }
#pragma unroll
        for (int q = VPT / 2; q >= 1; q /= 2)
#pragma unroll
            for (int j = 0; j < q; ++j) part[j] += part[j + q];
        const double near = group_sum<LPR>(nval > 0 ? (double)part[0] : 0.0);
        const float inv = __builtin_amdgcn_rcpf((float)near);
        if (!a.renorm) {
            // weights are divided by the sum: of 64-bit exponentials, as in the exact form
            double sum = 0.0;
#pragma unroll
            for (int j = 0; j < VPT; ++j) sum += ours(j) ? exp((double)l[j] - (double)m) : 0.0;
            total = group_sum<LPR>(nval > 0 ? sum : 0.0);
        }
        tau = 9e-7f * inv;
#pragma unroll
        for (int j = 0; j < VPT; ++j) c[j] = fmaf(c[j], inv, b[j]);
    } else {
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const float t = __builtin_amdgcn_exp2f(fabsf(l[j]) * -kLog2e);
            c[j] = fmaf(l[j] < 0.f ? t : 1.f, __builtin_amdgcn_rcpf(1.f + t), b[j]);  // (a NaN through t)
        }
    }
    float zero = 0.f;  // NaN where a value is not finite
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        zero = ours(j) ? fmaf(c[j], 0.f, zero) : zero;
        c[j] = ours(j) ? c[j] : -INFINITY;
    }
    bool unsure = nval > 0 && !(zero == 0.f);

    bool kept = nval > 0;
    if (groups > 1) {
        float b1 = -INFINITY, b2 = -INFINITY;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            b2 = fmaxf(b2, fminf(b1, c[j]));
            b1 = fmaxf(b1, c[j]);
        }
        if (WHOLE && nval == 0) b1 = b2 = -INFINITY;
        if (f.lanes_log2 > 0) top2_step<1>(b1, b2);
        if (f.lanes_log2 > 1) top2_step<2>(b1, b2);
        if (f.lanes_log2 > 2) top2_step<4>(b1, b2);
        if (f.lanes_log2 > 3) top2_step<8>(b1, b2);
        if (f.lanes_log2 > 4) top2_step<16>(b1, b2);
        const float gs = a.group_top == 1 ? b1 : b1 + b2;
        // two scores of one or two c, each within tau and its rounding, and the sum's
        const float most = a.group_top == 1 ? fabsf(b1) : fmaxf(fabsf(b1), fabsf(b2));
        const float far = 5.f * (tau + 1.2e-7f * (grp < groups ? most : 0.f));
        const int base = lane - sub;
        int above = 0, level = 0;
        for (int q = 0; q < groups; ++q) {
            const float v = __shfl(gs, base + (q << f.lanes_log2));
            above += v > gs + far;
            level += v >= gs - far;  // (itself among them)
        }
        unsure |= nval > 0 && level > a.topk_groups && above < a.topk_groups;
        kept = kept && level <= a.topk_groups;
    }

    // the grid: [lo, hi] of what can be among the k + 2 best
    float top = -INFINITY, low = INFINITY;
#pragma unroll
    for (int j = 0; j < VPT; ++j) top = fmaxf(top, c[j]);
    low = top;
    if (!f.many) {
#pragma unroll
        for (int j = 0; j < VPT; ++j) low = ours(j) ? fminf(low, c[j]) : low;
    }
    const float hi = group_max<LPR>(kept ? top : -INFINITY);
    // (with many lanes each holds a value >= the least of their largest)
    const float lo = -group_max<LPR>(kept ? -low : -INFINITY);
    const float span = hi - lo;
    const float unit = span > 0.f ? (float)((1u << QB) - 16u) * __builtin_amdgcn_rcpf(span) : 0.f;
    const float first = fmaf(-lo, unit, 4.f);
    tau += 3.6e-7f * fmaxf(fabsf(hi), fabsf(lo));  // roundings of c, of first and of the product
    // (f32 holds 24 bits of a grid of more)
    const uint32_t apart = (uint32_t)fminf(2.f * tau * unit, 1e9f) + (16u << (QB > 24 ? QB - 24 : 0));
    // Experts in question lie at 1 (what is below the grid) and above, those of lanes
    // that are not kept at 0 (v_med3 takes a NaN to the lower bound): keys below kNone
    // are nobody's.
    constexpr uint32_t kNone = 1u << IB;
    // the grid's last place that f32 holds (2^QB - 1 rounds to 2^QB where QB > 24, which
    // the shift would take out of the key): roundings of unit and first carry the
    // largest c past it
    constexpr float kLast = (float)((1u << QB) - (QB > 24 ? 1u << (QB - 24) : 1u));
    static_assert((uint32_t)kLast < (1u << QB), "the largest key fits 32 bits");
    const float lane_unit = kept ? unit : 0.f, lane_first = kept ? first : 0.f, lane_low = kept ? 1.f : 0.f;
    uint32_t key[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const uint32_t q =
            (uint32_t)__builtin_amdgcn_fmed3f(fmaf(c[j], lane_unit, lane_first), lane_low, kLast);
        key[j] = ours(j) ? (q << IB) | (uint32_t)(SLOTS - 1 - (sub * VPT + j)) : 0u;
    }
    constexpr int NL = VPT > 8 ? VPT / 8 : 1, LEN = VPT / NL;  // sorted lists per lane
#pragma unroll
    for (int n = 0; n < NL; ++n) sort_desc<LEN>(key + n * LEN);
    uint32_t mine = 0;  // lane r of the row: the key of place r
    for (int r = 0; r <= a.k + 1; ++r) {
        uint32_t h = key[0];
        if constexpr (NL == 2) h = max(h, key[LEN]);
        const uint32_t best = group_key32_max<LPR>(h);
        mine = sub == r ? best : mine;
#pragma unroll
        for (int n = 0; n < NL; ++n) {
            const uint64_t pop = __ballot(key[n * LEN] == best);
#pragma unroll
            for (int q = 0; q < LEN; ++q)
                key[n * LEN + q] = key_take32(key[n * LEN + q], q + 1 < LEN ? key[n * LEN + (q + 1) % LEN] : 0u, pop);
        }
    }

    // places 0 .. k + 1, one lane each, and their scores in 64 bits
    const int slot = SLOTS - 1 - (int)(mine & (SLOTS - 1));
    const int sg = (slot / VPT) >> f.lanes_log2;
    const bool has = sub <= a.k + 1 && mine >= kNone;
    int e = has ? sg * f.cells + slot - (sg << f.lanes_log2) * VPT : INT_MAX;
    const float le = has ? Elem<DT>::to_f32(src[e]) : -INFINITY;
    const double be = has && a.bias ? (double)a.bias[e] : 0.0;
    const bool soft = a.score == kRouteSoftmax;
    double w = 0.0;
    if (has) {
        const double x = exp(soft ? (double)le - (double)m : -(double)le);
        w = soft ? (le == -INFINITY ? 0.0 : x) : 1.0 / (1.0 + x);
    }
    // No other expert can be among the k best if place k + 1 is clear of place
    // k - 1; the order of places 0 .. k goes by their exact c (those of a softmax
    // with a bias would need the exact sum: those rows need clear places).
    const uint32_t k1 = __shfl_down(mine, 1), k2 = __shfl_down(mine, 2);
    unsure |= sub < a.k && mine < kNone;
    unsure |= sub == a.k - 1 && k2 >= kNone && (mine >> IB) - (k2 >> IB) <= apart;
    if (soft && a.bias) {
        const float nl = __shfl_down(le, 1);
        const double nb = __shfl_down(be, 1);
        unsure |= sub < a.k && k1 >= kNone && (mine >> IB) - (k1 >> IB) <= apart && !(le == nl && be == nb);
    } else {
        const double ce = w + be;
        const double nc = __shfl_down(ce, 1);
        const int ne = __shfl_down(e, 1);
        const bool wrong = sub < a.k && ne != INT_MAX && (nc > ce || (nc == ce && ne < e));
        if (__any(wrong)) {
            const int base = lane - sub;
            int place = 0;
            for (int q = 0; q <= a.k; ++q) {
                const double vc = __shfl(ce, base + q);
                const int ve = __shfl(e, base + q);
                place += ve != INT_MAX && (vc > ce || (vc == ce && ve < e));
            }
            const int to = 4 * (sub <= a.k && e != INT_MAX ? base + place : lane);
            const uint64_t u = __double_as_longlong(w);
            e = __builtin_amdgcn_ds_permute(to, e);
            const uint32_t wl = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)(uint32_t)u);
            const uint32_t wh = (uint32_t)__builtin_amdgcn_ds_permute(to, (int)(uint32_t)(u >> 32));
            w = __longlong_as_double(((uint64_t)wh << 32) | wl);
        }
    }
    w = sub < a.k ? w : 0.0;
    if (soft && !a.renorm) w /= total;
    if (a.renorm) {
        const double sum = group_sum<LPR>(w);
        w = sum == 0.0 ? 0.0 : w / sum;
    }
    uint64_t redo = __ballot(unsure && live);
    const uint64_t own = (LPR == 64 ? ~0ull : ((1ull << (LPR % 64)) - 1ull) << (lane - sub));
    if (live && sub < a.k && !(redo & own)) {
        const long long at = row * a.k + sub;
        a.w[at] = (float)(w * (double)a.scale);
        a.idx[at] = (uint32_t)e;
        a.ei[at] = (uint32_t)((long long)sub * a.T + row);
    }
    while (redo) {
        const int r = __builtin_ctzll(redo) / LPR;
        route_exact_row<VS, DT>(a, row0 + r, s_buf[wave]);
        redo &= ~(LPR == 64 ? ~0ull : ((1ull << (LPR % 64)) - 1ull) << (r * LPR));
    }
}

template <int VPT>
hipError_t launch_exact(const RouteArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)((a.T + kRouteWaves - 1) / kRouteWaves)), block(64 * kRouteWaves);
    if (a.dtype == kF32) hipLaunchKernelGGL((route_exact_k<VPT, kF32>), grid, block, 0, stream, a);
    else if (a.dtype == kBF16) hipLaunchKernelGGL((route_exact_k<VPT, kBF16>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((route_exact_k<VPT, kF16>), grid, block, 0, stream, a);
    return hipGetLastError();
}

int next_pow2(int n) {
    int p = 1;
    while (p < n) p *= 2;
    return p;
}

// f for LPR lanes of VPT experts, if the row fits them (a place per lane for the
// k best and the next two).
template <int LPR, int VPT>
bool fits(const RouteArgs& a, RouteFast& f, bool& whole) {
    const int groups = a.topk_groups < a.groups ? a.groups : 1;
    f.cells = a.E / groups;
    const int full = (f.cells + VPT - 1) / VPT;  // lanes with experts in a group
    const int lanes = groups == 1 ? LPR : next_pow2(full);
    if (full > lanes || next_pow2(groups) * lanes > LPR || a.k + 2 > LPR) return false;
    f.lanes_log2 = __builtin_ctz(lanes);
    f.many = (groups == 1 ? 1 : a.topk_groups) * full >= a.k + 2;
    const int es = a.dtype == kF32 ? 4 : 2;
    whole = f.cells % VPT == 0 && VPT * es % 16 == 0 && (long long)a.E * es % 16 == 0 &&
            (((uintptr_t)a.logits | (uintptr_t)a.bias) & 15) == 0;
    return true;
}

template <int LPR, int VPT, int DT>
void launch_form(const RouteArgs& a, const RouteFast& f, bool whole, const dim3& grid, hipStream_t stream) {
    const dim3 block(64 * kRouteWaves);
    if constexpr (VPT * (DT == kF32 ? 4 : 2) % 16 == 0) {
        if (whole) {
            hipLaunchKernelGGL((route_fast_k<LPR, VPT, DT, true>), grid, block, 0, stream, a, f);
            return;
        }
    }
    hipLaunchKernelGGL((route_fast_k<LPR, VPT, DT, false>), grid, block, 0, stream, a, f);
}
template <int LPR, int VPT>
bool launch_fast(const RouteArgs& a, hipStream_t stream, hipError_t& e) {
    RouteFast f;
    bool whole;
    if (!fits<LPR, VPT>(a, f, whole)) return false;
    const int rows = kRouteWaves * (64 / LPR);
    const dim3 grid((unsigned)(((long long)a.T + rows - 1) / rows));
    if (a.dtype == kF32) launch_form<LPR, VPT, kF32>(a, f, whole, grid, stream);
    else if (a.dtype == kBF16) launch_form<LPR, VPT, kBF16>(a, f, whole, grid, stream);
    else launch_form<LPR, VPT, kF16>(a, f, whole, grid, stream);
    e = hipGetLastError();
    return true;
}

// Rows a launch needs before fewer lanes per row pay: with fewer the device is
// not full either way and the shorter chains of 64 lanes are ahead.
constexpr int kRouteManyRows = 2048;

}  // namespace

hipError_t launch_route(const RouteArgs& a, hipStream_t stream) {
    if (a.T <= 0) return hipSuccess;
    hipError_t e;
    if (a.T >= kRouteManyRows &&
        (launch_fast<16, 4>(a, stream, e) || launch_fast<16, 8>(a, stream, e) || launch_fast<16, 16>(a, stream, e) ||
         launch_fast<32, 8>(a, stream, e) || launch_fast<32, 16>(a, stream, e)))
        return e;
    if (launch_fast<64, 2>(a, stream, e) || launch_fast<64, 4>(a, stream, e) || launch_fast<64, 8>(a, stream, e) ||
        launch_fast<64, 16>(a, stream, e))
        return e;
    if (a.E <= 64) return launch_exact<1>(a, stream);
    if (a.E <= 128) return launch_exact<2>(a, stream);
    if (a.E <= 256) return launch_exact<4>(a, stream);
    if (a.E <= 512) return launch_exact<8>(a, stream);
    return launch_exact<16>(a, stream);
}

}  // namespace cm
