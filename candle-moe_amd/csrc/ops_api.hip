// C entry points of the operators around the expert products: routing with
// groups, the residual's addition with the root-mean-square norm, 4-bit weights
// and the MoE over them.
#include <algorithm>

#include "../../include/candle_moe.h"
#include "cm_common.hpp"
#include "cm_internal.hpp"

namespace cm {

static bool aligned(const void* p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

// ------------------------------------------------- MoE over 4-bit weights
struct MxCall {
    const void* x;
    const void* x_scale;  // null: 16-bit rows
    const void *gate, *up, *down;
    const void *gate_s, *up_s, *down_s;
    const void *rw, *idx;
    void* out;
    int T, H, I, E, k, act;
    uint32_t moe_type, dtype;
    bool accumulate;
};

static int run_mx(const MxCall& c, hipStream_t s) {
    if (c.T < 0) return set_error(CANDLE_MOE_ERR_INVALID, "fused_moe_mxfp4: num_tokens must be >= 0 (got %d)", c.T);
    if (c.E < 1 || c.E > 4096)
        return set_error(CANDLE_MOE_ERR_INVALID, "fused_moe_mxfp4: num_experts must be in [1, 4096] (got %d)", c.E);
    if (c.k < 1)
        return set_error(CANDLE_MOE_ERR_INVALID, "fused_moe_mxfp4: num_selected_experts must be >= 1 (got %d)", c.k);
    if (c.act < 0 || c.act > 2)
        return set_error(CANDLE_MOE_ERR_INVALID, "fused_moe_mxfp4: activation_type must be 0, 1 or 2 (got %d)", c.act);
    if (c.moe_type > 1)
        return set_error(CANDLE_MOE_ERR_INVALID, "fused_moe_mxfp4: moe_type must be one of 0 or 1 (got %u)", c.moe_type);
    if (c.dtype > 1)
        return set_error(CANDLE_MOE_ERR_UNSUPPORTED, "fused_moe_mxfp4: dtype must be 0 (f16) or 1 (bf16) (got %u)",
                         c.dtype);
    if (c.H < 1 || c.I < 1 || c.H % 32 || c.I % 32)
        return set_error(CANDLE_MOE_ERR_UNSUPPORTED,
                         "fused_moe_mxfp4: hidden_dim and intermediate_dim must be positive multiples of 32 (got %d, %d)",
                         c.H, c.I);
    const long long P = (long long)c.T * c.k, lim = 0x7fffff00LL;
    if (P > 0x7fffffffLL)
        return set_error(CANDLE_MOE_ERR_INVALID,
                         "fused_moe_mxfp4: num_tokens * num_selected_experts exceeds 2^31-1");
    if (c.T == 0) return CANDLE_MOE_OK;
    const bool qwen3 = c.moe_type == 0;
    if (!c.x || !c.gate || !c.up || !c.gate_s || !c.up_s || !c.rw || !c.idx || !c.out)
        return set_error(CANDLE_MOE_ERR_INVALID, "fused_moe_mxfp4: null tensor pointer");
    if (qwen3 && (!c.down || !c.down_s))
        return set_error(CANDLE_MOE_ERR_INVALID, "fused_moe_mxfp4: down_q and down_scale are required for moe_type 0 (Qwen3)");
    if (!aligned(c.x, 16) || !aligned(c.gate, 16) || !aligned(c.up, 16) || (qwen3 && !aligned(c.down, 16)) ||
        !aligned(c.out, 16))
        return set_error(CANDLE_MOE_ERR_UNSUPPORTED,
                         "fused_moe_mxfp4: input, weights and output must be 16-byte aligned");
    if ((long long)c.T * c.H * 2 >= lim || P * c.I * 2 >= lim || (long long)c.H * c.I * 2 >= lim)
        return set_error(CANDLE_MOE_ERR_UNSUPPORTED, "fused_moe_mxfp4: operands beyond 2 GiB");
    if (!aligned(c.gate_s, 16) || !aligned(c.up_s, 16) || (qwen3 && !aligned(c.down_s, 16)))
        return set_error(CANDLE_MOE_ERR_UNSUPPORTED, "fused_moe_mxfp4: weight scales must be 16-byte aligned");
    const MxWeights mx = {reinterpret_cast<const uint8_t*>(c.gate_s), reinterpret_cast<const uint8_t*>(c.up_s),
                          reinterpret_cast<const uint8_t*>(c.down_s), reinterpret_cast<const uint8_t*>(c.x_scale)};
    return fused_moe_impl(c.x, c.gate, c.up, c.down, c.rw, c.idx, c.out, c.T, c.H, c.I, c.E, c.k, c.act, c.moe_type,
                          c.dtype, nullptr, 0, true, !c.accumulate, s, nullptr, false, &mx);
}

}  // namespace cm

extern "C" {

int candle_moe_topk_route(const void* logits, uint32_t logits_dtype, const float* bias, float* topk_weight,
                          void* topk_indices, void* token_expert_indices, int num_experts, int num_tokens, int topk,
                          int score, int num_groups, int topk_groups, int group_top, int renormalize, float scale,
                          void* stream) {
    cm::clear_error();
    const int E = num_experts, T = num_tokens, G = num_groups;
    if (T < 0) return cm::set_error(CANDLE_MOE_ERR_INVALID, "topk_route: num_tokens must be >= 0 (got %d)", T);
    if (E < 1 || E > 1024)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "topk_route: num_experts must be in [1, 1024] (got %d)", E);
    if (logits_dtype > 2)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "topk_route: dtype must be 0, 1 or 2 (got %u)", logits_dtype);
    if (score != cm::kRouteSoftmax && score != cm::kRouteSigmoid)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "topk_route: score must be 0 (softmax) or 1 (sigmoid) (got %d)",
                             score);
    if (G < 1 || G > cm::kRouteMaxGroups || E % G)
        return cm::set_error(CANDLE_MOE_ERR_INVALID,
                             "topk_route: num_groups must be in [1, %d] and divide num_experts=%d (got %d)",
                             cm::kRouteMaxGroups, E, G);
    if (topk_groups < 1 || topk_groups > G)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "topk_route: topk_groups must be in [1, num_groups=%d] (got %d)", G,
                             topk_groups);
    if (group_top < 1 || group_top > 2 || group_top > E / G)
        return cm::set_error(CANDLE_MOE_ERR_INVALID,
                             "topk_route: group_top must be 1 or 2 and at most the %d experts of a group (got %d)", E / G,
                             group_top);
    if (topk < 1 || topk > topk_groups * (E / G))
        return cm::set_error(CANDLE_MOE_ERR_INVALID,
                             "topk_route: topk must be in [1, %d], the experts of the chosen groups (got %d)",
                             topk_groups * (E / G), topk);
    if ((long long)T * topk > 0x7fffffffLL || T > cm::kRouteMaxRows)
        return cm::set_error(CANDLE_MOE_ERR_INVALID,
                             "topk_route: at most %d tokens and 2^31-1 pairs of them and their experts (got %d x %d)",
                             cm::kRouteMaxRows, T, topk);
    if (T == 0) return CANDLE_MOE_OK;
    if (!logits || !topk_weight || !topk_indices || !token_expert_indices)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "topk_route: null tensor pointer");
    cm::RouteArgs a = {};
    a.logits = logits;
    a.bias = bias;
    a.w = topk_weight;
    a.idx = reinterpret_cast<uint32_t*>(topk_indices);
    a.ei = reinterpret_cast<uint32_t*>(token_expert_indices);
    a.T = T;
    a.E = E;
    a.k = topk;
    a.dtype = (int)logits_dtype;
    a.score = score;
    a.groups = G;
    a.topk_groups = topk_groups;
    a.group_top = group_top;
    a.renorm = renormalize ? 1 : 0;
    a.scale = scale;
    const hipError_t e = cm::launch_route(a, reinterpret_cast<hipStream_t>(stream));
    return e == hipSuccess ? CANDLE_MOE_OK : cm::hip_fail(e, "topk_route launch");
}

int candle_moe_add_rms_norm(const void* input, const void* residual, const void* weight, void* residual_output,
                            void* output, void* codes, void* scales, int num_tokens, int hidden_dim, float eps,
                            uint32_t dtype, void* stream) {
    cm::clear_error();
    const int T = num_tokens, H = hidden_dim;
    if (T < 0) return cm::set_error(CANDLE_MOE_ERR_INVALID, "add_rms_norm: num_tokens must be >= 0 (got %d)", T);
    if (H < 1 || H > cm::kNormMaxHidden)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "add_rms_norm: hidden_dim must be in [1, %d] (got %d)",
                             cm::kNormMaxHidden, H);
    if (dtype > 2) return cm::set_error(CANDLE_MOE_ERR_INVALID, "add_rms_norm: dtype must be 0, 1 or 2 (got %u)", dtype);
    if (!(eps >= 0.0f)) return cm::set_error(CANDLE_MOE_ERR_INVALID, "add_rms_norm: eps must be >= 0 (got %g)", (double)eps);
    if (!codes != !scales)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "add_rms_norm: codes and scales go together");
    if (codes && (H % 32 || H > 32768))
        return cm::set_error(CANDLE_MOE_ERR_UNSUPPORTED,
                             "add_rms_norm: the 8-bit form needs a hidden_dim that is a multiple of 32, at most 32768 (got %d)",
                             H);
    if (T == 0) return CANDLE_MOE_OK;
    if (!input || !weight) return cm::set_error(CANDLE_MOE_ERR_INVALID, "add_rms_norm: null tensor pointer");
    if (!output && !codes)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "add_rms_norm: output or codes and scales must be given");
    cm::NormArgs a = {};
    a.x = input;
    a.residual = residual;
    a.weight = weight;
    a.residual_out = residual_output;
    a.out = output;
    a.codes = reinterpret_cast<uint8_t*>(codes);
    a.scales = reinterpret_cast<uint8_t*>(scales);
    a.T = T;
    a.H = H;
    a.eps = eps;
    a.vec = H % 8 == 0 && cm::aligned(input, 16) && cm::aligned(residual, 16) && cm::aligned(weight, 16) &&
            cm::aligned(residual_output, 16) && cm::aligned(output, 16) && cm::aligned(codes, 8);
    if (codes && !a.vec)
        return cm::set_error(CANDLE_MOE_ERR_UNSUPPORTED, "add_rms_norm: the 8-bit form needs 16-byte aligned tensors");
    hipError_t e = hipSuccess;
    const long long es = dtype == 2 ? 4 : 2;
    for (long long t = 0; t < T && e == hipSuccess; t += cm::kNormMaxRows) {
        cm::NormArgs b = a;
        auto from = [&](const void* p, long long row) {
            return p ? reinterpret_cast<const char*>(p) + t * row : nullptr;
        };
        b.x = from(a.x, H * es);
        b.residual = from(a.residual, H * es);
        b.residual_out = const_cast<char*>(from(a.residual_out, H * es));
        b.out = const_cast<char*>(from(a.out, H * es));
        if (codes) {
            b.codes = a.codes + t * H;
            b.scales = a.scales + t * (H / 32);
        }
        b.T = (int)std::min<long long>(T - t, cm::kNormMaxRows);
        e = cm::launch_add_rms_norm(b, (int)dtype, reinterpret_cast<hipStream_t>(stream));
    }
    return e == hipSuccess ? CANDLE_MOE_OK : cm::hip_fail(e, "add_rms_norm launch");
}

int candle_moe_quantize_mxfp4(const void* weights, uint32_t dtype, int num_experts, int k_dim, int n_dim, int input_kn,
                              void* codes, void* scales, void* stream) {
    cm::clear_error();
    if (dtype > 2) return cm::set_error(CANDLE_MOE_ERR_INVALID, "quantize_mxfp4: dtype must be 0, 1 or 2 (got %u)", dtype);
    if (num_experts < 0 || k_dim < 0 || n_dim < 0)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "quantize_mxfp4: sizes must be >= 0");
    if (k_dim % 32)
        return cm::set_error(CANDLE_MOE_ERR_UNSUPPORTED, "quantize_mxfp4: k_dim must be a multiple of 32 (got %d)", k_dim);
    if ((long long)num_experts * k_dim * n_dim == 0) return CANDLE_MOE_OK;
    if (!weights || !codes || !scales)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "quantize_mxfp4: null tensor pointer");
    if (!cm::aligned(codes, 16))
        return cm::set_error(CANDLE_MOE_ERR_UNSUPPORTED, "quantize_mxfp4: codes must be 16-byte aligned");
    const hipError_t e = cm::launch_quantize_mxfp4(weights, (int)dtype, num_experts, k_dim, n_dim, input_kn ? 1 : 0,
                                                   reinterpret_cast<uint8_t*>(codes),
                                                   reinterpret_cast<uint8_t*>(scales),
                                                   reinterpret_cast<hipStream_t>(stream));
    return e == hipSuccess ? CANDLE_MOE_OK : cm::hip_fail(e, "quantize_mxfp4 launch");
}

int candle_moe_dequantize_mxfp4(const void* codes, const void* scales, int num_experts, int n_dim, int k_dim, void* out,
                                uint32_t dtype, void* stream) {
    cm::clear_error();
    if (dtype > 2)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "dequantize_mxfp4: dtype must be 0, 1 or 2 (got %u)", dtype);
    if (num_experts < 0 || k_dim < 0 || n_dim < 0)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "dequantize_mxfp4: sizes must be >= 0");
    if (k_dim % 32)
        return cm::set_error(CANDLE_MOE_ERR_UNSUPPORTED, "dequantize_mxfp4: k_dim must be a multiple of 32 (got %d)", k_dim);
    if ((long long)num_experts * k_dim * n_dim == 0) return CANDLE_MOE_OK;
    if (!codes || !scales || !out)
        return cm::set_error(CANDLE_MOE_ERR_INVALID, "dequantize_mxfp4: null tensor pointer");
    if (!cm::aligned(codes, 16) || !cm::aligned(out, 16))
        return cm::set_error(CANDLE_MOE_ERR_UNSUPPORTED, "dequantize_mxfp4: codes and out must be 16-byte aligned");
    const hipError_t e = cm::launch_dequantize_mxfp4(codes, scales, num_experts, n_dim, k_dim, out, (int)dtype,
                                                     reinterpret_cast<hipStream_t>(stream));
    return e == hipSuccess ? CANDLE_MOE_OK : cm::hip_fail(e, "dequantize_mxfp4 launch");
}

int candle_moe_fused_moe_mxfp4(const void* input, const void* input_scale, const void* gate_q, const void* up_q,
                               const void* down_q, const void* gate_scale, const void* up_scale, const void* down_scale,
                               const void* routing_weights, const void* expert_indices, void* output, int num_tokens,
                               int hidden_dim, int intermediate_dim, int num_experts, int num_selected_experts,
                               int activation_type, uint32_t moe_type, uint32_t dtype, int accumulate, void* stream) {
    cm::clear_error();
    cm::MxCall c = {};
    c.x = input;
    c.x_scale = input_scale;
    c.gate = gate_q;
    c.up = up_q;
    c.down = down_q;
    c.gate_s = gate_scale;
    c.up_s = up_scale;
    c.down_s = down_scale;
    c.rw = routing_weights;
    c.idx = expert_indices;
    c.out = output;
    c.T = num_tokens;
    c.H = hidden_dim;
    c.I = intermediate_dim;
    c.E = num_experts;
    c.k = num_selected_experts;
    c.act = activation_type;
    c.moe_type = moe_type;
    c.dtype = dtype;
    c.accumulate = accumulate != 0;
    return cm::run_mx(c, reinterpret_cast<hipStream_t>(stream));
}

}  // extern "C"
