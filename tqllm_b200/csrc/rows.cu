// Rows of tokens sorted by expert, and rows of slots back to their tokens with the routing weights, with the gradients of both.
//
//   slot(a): the place of assignment a in the plan's permutation
//   there:   rows[slot(t topk + s)] = x[t]                                    gradient: dx[t] = sum_s drows[slot(t topk + s)]
//   back:    out[t] = r[t] + sum_s w[t][s] y[slot(t topk + s)] + ws[t] y[slot(shared t)]
//            gradient: dy[slot] = w[t][s] dout[t],  dw[t][s] = dout[t] . y[slot]
//
// A block takes a token: its row is read once and written to all its slots, or gathered from them. Nothing is summed in an order that changes, so there are no atomics. Bound by memory.
#include <algorithm>

#include "common.cuh"

namespace b2 {
namespace {

constexpr int MAX_ASSIGNMENTS = 0x3fffffff;      // as b2moe_dispatch

struct ThereArgs {
    const uint4 * x;
    uint4 * rows;
    const int * ids, * plan;
    int * slots;
    long long ldx, ldr;                          // in pieces of 16 bytes, as `pieces`
    int pieces, n, topk, experts, shared;        // shared: tokens of the always-on expert in the plan
};

// The slot of assignment a by a warp: the list of its expert holds it in ascending order, so 32 places are looked at at a time. Lists of another order (b2moe_plan_from_groups) are gone through.
// -1 where the plan does not hold it. What is read is inside the permutation whatever the ids are
__device__ __forceinline__ int find_slot(const ThereArgs & p, int a, int e) {
    if (e < 0 || e > p.experts) return -1;
    const int lane = threadIdx.x & 31, e1 = p.experts + 1, total = p.n * p.topk + p.shared;
    const int * offsets = p.plan + PLAN_HDR + e1, * perm = p.plan + PLAN_HDR + 3 * e1 + 1;
    const int first = max(0, offsets[e]), end = min(total, offsets[e + 1]);
    int lo = first, hi = end;
    while (hi - lo > 32) {
        // the last entry of each of 32 parts: the first one that is not below a ends the part that may hold it
        const int part = (hi - lo + 31) >> 5, at = min(hi, lo + (lane + 1) * part) - 1;
        const unsigned not_below = __ballot_sync(0xffffffffu, perm[at] >= a);
        if (!not_below) { lo = hi; break; }
        const int which = __ffs(not_below) - 1;
        lo += which * part;
        hi = min(hi, lo + part);
    }
    unsigned hit = __ballot_sync(0xffffffffu, lo + lane < hi && perm[lo + lane] == a);
    if (hit) return lo + __ffs(hit) - 1;
    for (int b = first; b < end; b += 32) {
        hit = __ballot_sync(0xffffffffu, b + lane < end && perm[b + lane] == a);
        if (hit) return b + __ffs(hit) - 1;
    }
    return -1;
}

constexpr int THERE_LIST = 32;                   // slots of a token that are looked for before they are written
template <int P>
__global__ void __launch_bounds__(256) there_k(const ThereArgs p) {
    __shared__ int list[THERE_LIST];
    grid_release();
    grid_wait();
    const int t = blockIdx.x, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, lane = threadIdx.x & 31, A = p.n * p.topk;
    const int step = gridDim.y * blockDim.x * P, all = p.topk + (p.shared ? 1 : 0);
    const uint4 * x = p.x + size_t(t) * p.ldx;
    for (int j0 = blockIdx.y * blockDim.x * P; j0 < p.pieces; j0 += step) {
        uint4 v[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = j0 + i * blockDim.x + threadIdx.x;
            if (j < p.pieces) v[i] = x[j];
        }
        for (int s0 = 0; s0 < all; s0 += THERE_LIST) {
            const bool again = j0 == int(blockIdx.y * blockDim.x * P) || all > THERE_LIST;      // the list of a token with few slots stays from its first pieces on
            if (again) {
                __syncthreads();
                for (int s = s0 + warp; s < min(all, s0 + THERE_LIST); s += warps) {
                    const bool shared = s == p.topk;
                    const int a = shared ? A + t : t * p.topk + s, e = shared ? p.experts : p.ids[a], slot = shared || e < p.experts ? find_slot(p, a, e) : -1;
                    if (lane == 0) {
                        list[s - s0] = slot;
                        if (p.slots && j0 == 0) p.slots[a] = slot;
                    }
                }
                __syncthreads();
            }
            for (int s = s0; s < min(all, s0 + THERE_LIST); ++s) {
                const int slot = list[s - s0];
                if (slot < 0) continue;
                uint4 * row = p.rows + size_t(slot) * p.ldr;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int j = j0 + i * blockDim.x + threadIdx.x;
                    if (j < p.pieces) row[j] = v[i];
                }
            }
        }
    }
}

// 16 bytes of a row as 32-bit values
template <int DT> struct Vec {
    static constexpr int N = DT == B2MOE_F32 ? 4 : 8;
    static __device__ __forceinline__ void open(const uint4 & w, float (&f)[N]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int l = 0; l < 4; ++l) {
            if constexpr (DT == B2MOE_F32) {
                f[l] = __uint_as_float(u[l]);
            } else if constexpr (DT == B2MOE_BF16) {
                f[2 * l] = __uint_as_float(u[l] << 16);
                f[2 * l + 1] = __uint_as_float(u[l] & 0xffff0000u);
            } else {
                const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&u[l]));
                f[2 * l] = v.x;
                f[2 * l + 1] = v.y;
            }
        }
    }
    static __device__ __forceinline__ uint4 close(const float (&f)[N]) {
        uint32_t u[4];
#pragma unroll
        for (int l = 0; l < 4; ++l) {
            if constexpr (DT == B2MOE_F32) {
                u[l] = __float_as_uint(f[l]);
            } else if constexpr (DT == B2MOE_BF16) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * l], f[2 * l + 1]);
                u[l] = *reinterpret_cast<const uint32_t *>(&b);
            } else {
                const __half2 b = __floats2half2_rn(f[2 * l], f[2 * l + 1]);
                u[l] = *reinterpret_cast<const uint32_t *>(&b);
            }
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
};

struct BackArgs {
    const uint4 * y, * residual;
    uint4 * out;
    const int * slots;
    const float * w, * sw;                       // null: one
    long long ldy, ldr, ldo;
    int pieces, n, topk, shared, rows;           // shared: the slots of the always-on expert follow the routed ones; rows: of y, nothing is read behind them
};

constexpr int BACK_SLOTS = 5;                    // slots whose rows are asked for at once
template <int DT>
__global__ void __launch_bounds__(256) back_k(const BackArgs p) {
    constexpr int N = Vec<DT>::N;
    grid_release();
    grid_wait();
    const int t = blockIdx.x, j = blockIdx.y * blockDim.x + threadIdx.x;
    if (j >= p.pieces) return;
    float acc[N], f[N];
    if (p.residual) Vec<DT>::open(p.residual[size_t(t) * p.ldr + j], acc);
    else
#pragma unroll
        for (int l = 0; l < N; ++l) acc[l] = 0.f;
    const int all = p.topk + (p.shared ? 1 : 0);
    for (int s0 = 0; s0 < all; s0 += BACK_SLOTS) {
        uint4 v[BACK_SLOTS];
        float w[BACK_SLOTS];
        bool live[BACK_SLOTS];
#pragma unroll
        for (int i = 0; i < BACK_SLOTS; ++i) {
            const int s = s0 + i;
            live[i] = false;
            if (s >= all) continue;
            const size_t a = s < p.topk ? size_t(t) * p.topk + s : size_t(p.n) * p.topk + t;
            const int slot = p.slots[a];
            live[i] = unsigned(slot) < unsigned(p.rows);
            w[i] = s < p.topk ? (p.w ? p.w[a] : 1.f) : p.sw ? p.sw[t] : 1.f;
            if (live[i]) v[i] = p.y[size_t(slot) * p.ldy + j];
        }
#pragma unroll
        for (int i = 0; i < BACK_SLOTS; ++i)
            if (live[i]) {
                Vec<DT>::open(v[i], f);
#pragma unroll
                for (int l = 0; l < N; ++l) acc[l] = fmaf(w[i], f[l], acc[l]);
            }
    }
    p.out[size_t(t) * p.ldo + j] = Vec<DT>::close(acc);
}

struct BackGradArgs {
    const uint4 * dout, * y;
    uint4 * dy;
    const int * slots;
    const float * w, * sw;
    float * dw, * dsw;                           // null: not wanted
    long long ldo, ldy, ldd;
    int pieces, n, topk, shared, rows;
};

// a block takes an assignment: its part of the token's gradient, its row, and the product of the two
template <int DT>
__global__ void __launch_bounds__(256) back_grad_k(const BackGradArgs p) {
    constexpr int N = Vec<DT>::N;
    __shared__ float red[8];
    grid_release();
    grid_wait();
    const int all = p.topk + (p.shared ? 1 : 0), t = blockIdx.x / all, s = blockIdx.x % all;
    const size_t a = s < p.topk ? size_t(t) * p.topk + s : size_t(p.n) * p.topk + t;
    const int slot = p.slots[a];
    const bool live = unsigned(slot) < unsigned(p.rows);
    float dot = 0.f;
    if (live) {
        const float w = s < p.topk ? (p.w ? p.w[a] : 1.f) : p.sw ? p.sw[t] : 1.f;
        const uint4 * d = p.dout + size_t(t) * p.ldo, * y = p.y + size_t(slot) * p.ldy;
        uint4 * dy = p.dy + size_t(slot) * p.ldd;
        for (int j = threadIdx.x; j < p.pieces; j += blockDim.x) {
            float g[N], f[N];
            Vec<DT>::open(d[j], g);
            if (p.y) {
                Vec<DT>::open(y[j], f);
#pragma unroll
                for (int l = 0; l < N; ++l) dot = fmaf(g[l], f[l], dot);
            }
            if (p.dy) {
#pragma unroll
                for (int l = 0; l < N; ++l) g[l] *= w;
                dy[j] = Vec<DT>::close(g);
            }
        }
    }
    float * out = s < p.topk ? (p.dw ? p.dw + a : nullptr) : p.dsw ? p.dsw + t : nullptr;
    if (!out) return;
#pragma unroll
    for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = dot;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < int(blockDim.x >> 5); ++w) dot += red[w];
    *out = dot;
}

// what the calls have in common; pieces of 16 bytes
bool batch(int n, int topk, int hidden, int dtype) { return n > 0 && topk > 0 && (long long)n * topk <= MAX_ASSIGNMENTS && hidden > 0 && valid_dtype(dtype) && hidden % (16 / int(dtype_bytes(dtype))) == 0; }
bool stride(const void * p, long long ld, int hidden, int dtype) { return !p || (ld >= hidden && ld % (16 / (long long)dtype_bytes(dtype)) == 0); }
int threads_for(int pieces) { return std::min(256, ceil_div(pieces, 32) * 32); }

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" B2MOE_API int32_t b2moe_dispatch_rows(const void * x, int32_t dtype, int64_t ldx, const int32_t * ids, const int32_t * plan, int32_t n, int32_t topk, int32_t hidden, int32_t experts,
                                                 int32_t shared_tokens, void * rows, int64_t ldr, int32_t * slots, b2moe_stream stream) {
    if (!batch(n, topk, hidden, dtype) || experts <= 0 || shared_tokens < 0 || shared_tokens > n || !stride(x, ldx, hidden, dtype) || !stride(rows, ldr, hidden, dtype)) return B2MOE_ERR_SHAPE;
    if (!x || !ids || !plan || !rows) return B2MOE_ERR_NULL;
    if (!aligned16(x) || !aligned16(rows) || !aligned_to(ids, 4) || !aligned_to(plan, 4) || !aligned_to(slots, 4)) return B2MOE_ERR_ALIGN;
    const int per = 16 / int(dtype_bytes(dtype)), pieces = hidden / per, threads = threads_for(pieces);
    const ThereArgs a{static_cast<const uint4 *>(x), static_cast<uint4 *>(rows), ids, plan, slots, ldx / per, ldr / per, pieces, n, topk, experts, shared_tokens};
    launch_overlapped(there_k<2>, dim3(n), dim3(threads), 0, as_stream(stream), a);
    return launch_status();
}

extern "C" B2MOE_API int32_t b2moe_combine_rows(const void * y, int32_t dtype, int64_t ldy, int32_t rows, const int32_t * slots, const float * weights, const float * shared_weights,
                                                const void * residual, int64_t ldr, int32_t n, int32_t topk, int32_t hidden, int32_t shared_tokens, void * out, int64_t ldo, b2moe_stream stream) {
    if (!batch(n, topk, hidden, dtype) || rows <= 0 || (shared_tokens != 0 && shared_tokens != n)) return B2MOE_ERR_SHAPE;
    if (!stride(y, ldy, hidden, dtype) || !stride(residual, ldr, hidden, dtype) || !stride(out, ldo, hidden, dtype)) return B2MOE_ERR_SHAPE;
    if (!y || !slots || !out) return B2MOE_ERR_NULL;
    if (!aligned16(y) || !aligned16(residual) || !aligned16(out) || !aligned_to(slots, 4) || !aligned_to(weights, 4) || !aligned_to(shared_weights, 4)) return B2MOE_ERR_ALIGN;
    const int per = 16 / int(dtype_bytes(dtype)), pieces = hidden / per, threads = threads_for(pieces);
    const BackArgs a{static_cast<const uint4 *>(y), static_cast<const uint4 *>(residual), static_cast<uint4 *>(out), slots, weights, shared_weights, ldy / per, ldr / per, ldo / per, pieces, n, topk, shared_tokens ? 1 : 0, rows};
    const dim3 grid(n, ceil_div(pieces, threads));
    cudaStream_t s = as_stream(stream);
    if (dtype == B2MOE_F32) launch_overlapped(back_k<B2MOE_F32>, grid, dim3(threads), 0, s, a);
    else if (dtype == B2MOE_F16) launch_overlapped(back_k<B2MOE_F16>, grid, dim3(threads), 0, s, a);
    else launch_overlapped(back_k<B2MOE_BF16>, grid, dim3(threads), 0, s, a);
    return launch_status();
}

extern "C" B2MOE_API int32_t b2moe_combine_rows_backward(const void * grad_out, int32_t dtype, int64_t ldgo, const void * y, int64_t ldy, int32_t rows, const int32_t * slots, const float * weights,
                                                         const float * shared_weights, int32_t n, int32_t topk, int32_t hidden, int32_t shared_tokens, void * grad_y, int64_t ldgy, float * grad_weights,
                                                         float * grad_shared, b2moe_stream stream) {
    if (!batch(n, topk, hidden, dtype) || rows <= 0 || (shared_tokens != 0 && shared_tokens != n) || (grad_shared && !shared_tokens) || (long long)n * (topk + 1) > 0x7fffffffLL) return B2MOE_ERR_SHAPE;
    if (!stride(grad_out, ldgo, hidden, dtype) || !stride(y, ldy, hidden, dtype) || !stride(grad_y, ldgy, hidden, dtype)) return B2MOE_ERR_SHAPE;
    if (!grad_out || !slots || (!grad_y && !grad_weights && !grad_shared) || ((grad_weights || grad_shared) && !y)) return B2MOE_ERR_NULL;
    if (!aligned16(grad_out) || !aligned16(y) || !aligned16(grad_y) || !aligned_to(slots, 4) || !aligned_to(weights, 4) || !aligned_to(shared_weights, 4) || !aligned_to(grad_weights, 4) ||
        !aligned_to(grad_shared, 4)) return B2MOE_ERR_ALIGN;
    const int per = 16 / int(dtype_bytes(dtype)), pieces = hidden / per, threads = threads_for(pieces);
    const bool dots = grad_weights || grad_shared;
    const BackGradArgs a{static_cast<const uint4 *>(grad_out), dots ? static_cast<const uint4 *>(y) : nullptr, static_cast<uint4 *>(grad_y), slots, weights, shared_weights, grad_weights, grad_shared,
                         ldgo / per, ldy / per, ldgy / per, pieces, n, topk, shared_tokens ? 1 : 0, rows};
    const dim3 grid(unsigned(n) * unsigned(topk + (shared_tokens ? 1 : 0)));
    cudaStream_t s = as_stream(stream);
    if (dtype == B2MOE_F32) launch_overlapped(back_grad_k<B2MOE_F32>, grid, dim3(threads), 0, s, a);
    else if (dtype == B2MOE_F16) launch_overlapped(back_grad_k<B2MOE_F16>, grid, dim3(threads), 0, s, a);
    else launch_overlapped(back_grad_k<B2MOE_BF16>, grid, dim3(threads), 0, s, a);
    return launch_status();
}
