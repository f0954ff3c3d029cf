// The gradient of the routing weights on the logits.
//
//   softmax: w_j = f e^{l_j} / sum over the selected of e^{l_i}, since their sum of probabilities is at least topk / experts >= 1 / 4096, above the clamp at 2^-14; with v = w / f
//     dl_j = w_j sum_i v_i (g_j - g_i)          which differences keep exact where a weight is nearly one, g_j - sum_i v_i g_i would not
//   sigmoid, normalised: dl_j = (1 - p_j) w_j sum_i v_i (g_j - g_i), or (1 - p_j) w_j g_j where the sum is clamped;  not normalised: (1 - p_j) w_j g_j
//   the other columns are zero;  shared expert: dl = g w (1 - w)
//
// A warp takes a token: zeros over its row, then the selected columns. Bound by writing the rows.
#include <algorithm>

#include "common.cuh"

namespace b2 {
namespace {

struct RouteGradArgs {
    const float * logits;
    const int * ids;
    const float * w, * g, * sw, * gs;            // weights and their gradients, the shared expert's (null: none)
    float * out;
    long long ld, ldg;
    int experts, topk, n, sigmoid, norm, add, together;
    float scale;
};

constexpr int GRAD_WARPS = 4;
__global__ void __launch_bounds__(32 * GRAD_WARPS) route_grad_k(const RouteGradArgs p) {
    grid_release();
    grid_wait();
    const int t = blockIdx.x * GRAD_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    // rows one behind the other: the block's four begin on 16 bytes and are zeroed together
    if (p.together) {
        float * const rows = p.out + size_t(blockIdx.x) * GRAD_WARPS * p.ldg;
        const int count = int(min((long long)GRAD_WARPS, (long long)p.n - (long long)blockIdx.x * GRAD_WARPS) * p.ldg);
        for (int c = 4 * threadIdx.x; c < count; c += 4 * 32 * GRAD_WARPS) {
            if (c + 4 <= count) *reinterpret_cast<float4 *>(rows + c) = make_float4(0.f, 0.f, 0.f, 0.f);
            else for (int l = c; l < count; ++l) rows[l] = 0.f;
        }
        __syncthreads();
    }
    if (t >= p.n) return;
    const int * ids = p.ids + size_t(t) * p.topk;
    const float * w = p.w + size_t(t) * p.topk, * g = p.g + size_t(t) * p.topk, * logits = p.logits + size_t(t) * p.ld;
    float * out = p.out + size_t(t) * p.ldg;
    if (!p.add && !p.together)
        for (int c = lane; c < p.experts; c += 32) out[c] = 0.f;
    // sigmoid: is the selected ones' sum above the clamp. Without the logits of ids outside of the experts, the weights tell: they add up to the scale where it was, and to less of it where the clamp was divided by
    bool coupled = p.norm;
    if (p.sigmoid && p.norm) {
        float sum = 0.f;
        bool all = true;
        for (int s = lane; s < p.topk; s += 32) {
            const int id = ids[s];
            if (unsigned(id) < unsigned(p.experts)) sum += 1.f / (1.f + expf(-logits[id]));
            else all = false;
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        coupled = sum > 6.103515625e-5f;
        if (!coupled && !__all_sync(0xffffffffu, all)) {
            float total = 0.f;
            for (int s = lane; s < p.topk; s += 32) total += w[s];
#pragma unroll
            for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
            // (weights of three roundings each, added up in 128 steps and five at most: 2^-16)
            coupled = total / p.scale > 1.f - 0x1p-16f;
        }
    }
    __syncwarp();                                                      // the zeros come before the values
    for (int s0 = 0; s0 < p.topk; s0 += 32) {
        const int s = s0 + lane;
        const bool in = s < p.topk;
        const int id = in ? ids[s] : -1;
        const bool live = unsigned(id) < unsigned(p.experts);
        const float wj = in ? w[s] : 0.f, gj = in ? g[s] : 0.f;
        float d = gj;
        if (coupled) {
            d = 0.f;
            for (int b = 0; b < p.topk; b += 32) {
                const float wi = b == s0 ? wj : b + lane < p.topk ? w[b + lane] : 0.f, gi = b == s0 ? gj : b + lane < p.topk ? g[b + lane] : 0.f;
                const int most = min(32, p.topk - b);
                for (int i = 0; i < most; ++i) d = fmaf(__shfl_sync(0xffffffffu, wi, i), gj - __shfl_sync(0xffffffffu, gi, i), d);
            }
            d /= p.scale;
        }
        d *= wj;
        if (p.sigmoid && live) d /= 1.f + expf(logits[id]);
        // an expert that a token names more than once (no routing does): the first lane takes them all
        const unsigned same = __match_any_sync(0xffffffffu, live ? id : -1 - lane);
        float sum = d;
        if (__any_sync(0xffffffffu, same != 1u << lane)) {
            sum = 0.f;
            for (int i = 0; i < 32; ++i) {
                const float o = __shfl_sync(0xffffffffu, d, i);
                if (same >> i & 1) sum += o;
            }
        }
        if (live && __ffs(same) - 1 == lane) out[id] = p.add || s0 ? out[id] + sum : sum;
        __syncwarp();
    }
    if (p.gs && lane == 0) {
        const float v = p.sw[t], d = p.gs[t] * v * (1.f - v);
        out[p.experts] = p.add ? out[p.experts] + d : d;
    }
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" B2MOE_API int32_t b2moe_route_backward(int32_t gating, const float * logits, int32_t ld, const int32_t * ids, const float * weights, const float * grad_weights, const float * shared_weights,
                                                  const float * grad_shared, int32_t experts, int32_t topk, int32_t norm, float scale, int32_t n, float * grad_logits, int32_t ldg, int32_t accumulate,
                                                  b2moe_stream stream) {
    if ((gating != B2MOE_SOFTMAX && gating != B2MOE_SIGMOID) || experts <= 0 || experts > 4096 || topk <= 0 || topk > experts || n <= 0) return B2MOE_ERR_SHAPE;
    if (ldg < experts + (grad_shared ? 1 : 0) || (gating == B2MOE_SIGMOID && ld < experts) || !(scale - scale == 0.f)) return B2MOE_ERR_SHAPE;
    if (!ids || !weights || !grad_weights || !grad_logits || (gating == B2MOE_SIGMOID && !logits) || (grad_shared && !shared_weights)) return B2MOE_ERR_NULL;
    for (const void * p : {static_cast<const void *>(logits), static_cast<const void *>(ids), static_cast<const void *>(weights), static_cast<const void *>(grad_weights),
                           static_cast<const void *>(shared_weights), static_cast<const void *>(grad_shared), static_cast<const void *>(grad_logits)})
        if (!aligned_to(p, 4)) return B2MOE_ERR_ALIGN;
    const RouteGradArgs a{logits, ids, weights, grad_weights, shared_weights, grad_shared, grad_logits, ld, ldg, experts, topk, n, gating == B2MOE_SIGMOID, gating == B2MOE_SOFTMAX || norm, accumulate,
                          !accumulate && ldg == experts + (grad_shared ? 1 : 0) && aligned16(grad_logits), scale == 0.f ? 1.f : scale};
    launch_overlapped(route_grad_k, dim3(ceil_div(n, GRAD_WARPS)), dim3(32 * GRAD_WARPS), 0, as_stream(stream), a);
    return launch_status();
}
