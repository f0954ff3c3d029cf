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

// A warp takes an assignment, or (grid.y) a part of its row: the row of its token, whose first pieces are on their way while the slot is looked for, to its slot. (The other warps of the token find the row in the L1.)
constexpr int THERE_PIECES = 8;
__global__ void __launch_bounds__(256) there_k(const ThereArgs p) {
    grid_release();
    grid_wait();
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, A = p.n * p.topk;
    const bool shared = i >= A;
    if (i >= A + (p.shared ? p.n : 0)) return;
    const int t = shared ? i - A : i / p.topk, e = shared ? p.experts : p.ids[i];
    const uint4 * x = p.x + size_t(t) * p.ldx;
    const int share = (p.pieces + 32 * gridDim.y - 1) / (32 * gridDim.y) * 32, begin = blockIdx.y * share, end = min(p.pieces, begin + share);
    uint4 v[THERE_PIECES];
    auto load = [&](int j0) {
#pragma unroll
        for (int c = 0; c < THERE_PIECES; ++c)
            if (j0 + 32 * c + lane < end) v[c] = x[j0 + 32 * c + lane];
    };
    load(begin);
    const int slot = shared || e < p.experts ? find_slot(p, i, e) : -1;
    if (p.slots && lane == 0 && blockIdx.y == 0) p.slots[i] = slot;
    if (slot < 0) return;
    uint4 * row = p.rows + size_t(slot) * p.ldr;
    for (int j0 = begin; j0 < end; j0 += 32 * THERE_PIECES) {
        if (j0 > begin) load(j0);
#pragma unroll
        for (int c = 0; c < THERE_PIECES; ++c)
            if (j0 + 32 * c + lane < end) row[j0 + 32 * c + lane] = v[c];
    }
}

// The slot of every assignment of the plan, for launches of many tokens. Words of assignments that the plan does not hold stay as they are: whoever reads one looks whether the plan leads back
__global__ void __launch_bounds__(256) slots_k(const ThereArgs p) {
    grid_release();
    grid_wait();
    const int i = blockIdx.x * 256 + threadIdx.x, e1 = p.experts + 1, A = p.n * p.topk;
    if (i >= min(p.plan[PLAN_NGROUPED], A + p.shared)) return;
    const int a = p.plan[PLAN_HDR + 3 * e1 + 1 + i];
    if (unsigned(a) < unsigned(A + (p.shared ? p.n : 0))) p.slots[a] = i;
}
// A warp (short rows) or a block takes a token: its row is read once, P pieces a thread at a time, and written to all its slots
template <int P, bool WARP>
__global__ void __launch_bounds__(256) there_token_k(const ThereArgs p) {
    __shared__ int list[32];
    grid_release();
    grid_wait();
    const int lane = threadIdx.x & 31, nt = WARP ? 32 : blockDim.x, tid = WARP ? lane : threadIdx.x, t = WARP ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (t >= p.n) return;
    const int A = p.n * p.topk, e1 = p.experts + 1, all = p.topk + (p.shared ? 1 : 0), * perm = p.plan + PLAN_HDR + 3 * e1 + 1, total = max(0, min(p.plan[PLAN_NGROUPED], A + p.shared));
    const uint4 * x = p.x + size_t(t) * p.ldx;
    for (int first = 0; first < p.pieces; first += P * nt) {
        const int j0 = first + tid;
        uint4 v[P];
#pragma unroll
        for (int c = 0; c < P; ++c)
            if (j0 + nt * c < p.pieces) v[c] = x[j0 + nt * c];
        for (int s0 = 0; s0 < all; s0 += 32) {
            int slot = -1;
            if (s0 + lane < all && tid < 32) {
                const int a = s0 + lane < p.topk ? t * p.topk + s0 + lane : A + t;
                slot = p.slots[a];
                if (unsigned(slot) >= unsigned(total) || perm[slot] != a) {
                    slot = -1;
                    p.slots[a] = -1;
                }
            }
            if (!WARP) {
                if (first + s0) __syncthreads();                       // the slots before have been read
                if (tid < 32) list[lane] = slot;
                __syncthreads();
            }
            for (int s = 0; s < min(32, all - s0); ++s) {
                const int at = WARP ? __shfl_sync(0xffffffffu, slot, s) : list[s];
                if (at < 0) continue;
                uint4 * row = p.rows + size_t(at) * p.ldr;
#pragma unroll
                for (int c = 0; c < P; ++c)
                    if (j0 + nt * c < p.pieces) row[j0 + nt * c] = v[c];
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

// S: slots whose rows are asked for at once, with the registers that let eight blocks or five of an SM run; twelve where there is a block or two an SM (64 tokens of 2048 from eleven slots: 3.9 us with five, 2.9 with twelve). us with 5 slots (five blocks) / 3 (eight) / 2 (eight):
//   4096 tokens of 2048 from ten slots 34.3 / 50.3 / 37.7, 4093 of 4096 from nine 63.8 / 87.1 / 65.5, 8192 of 4096 from two 57.2 / 56.7 / 45.0
// A thread takes a piece of a token, and the blocks of a token lie next to one another. (A warp that goes over a token's pieces with the slots in its lanes takes 58 us where this takes 33: 4096 tokens of 2048 from ten slots.)
template <int DT, int S>
__global__ void __launch_bounds__(256, S <= 2 ? 8 : S <= 5 ? 5 : 2) back_k(const BackArgs p) {
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
    for (int s0 = 0; s0 < all; s0 += S) {
        uint4 v[S];
        float w[S];
        int slot[S];
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const int s = s0 + i;
            slot[i] = -1;
            if (s >= all) continue;
            const size_t a = s < p.topk ? size_t(t) * p.topk + s : size_t(p.n) * p.topk + t;
            slot[i] = p.slots[a];
            w[i] = s < p.topk ? (p.w ? p.w[a] : 1.f) : p.sw ? p.sw[t] : 1.f;
        }
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (unsigned(slot[i]) < unsigned(p.rows)) v[i] = p.y[size_t(slot[i]) * p.ldy + j];
#pragma unroll
        for (int i = 0; i < S; ++i)
            if (unsigned(slot[i]) < unsigned(p.rows)) {
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

// A warp takes W assignments at a time (two of short rows), or (W = 0, launches of few assignments) a block takes one: the token's gradient, the row, and the product of the two
template <int DT, int W>
__global__ void __launch_bounds__(256) back_grad_k(const BackGradArgs p) {
    constexpr int N = Vec<DT>::N, M = W ? W : 1, P = 4 / M;            // pieces of an assignment in flight
    __shared__ float red[8];
    grid_release();
    grid_wait();
    const int nt = W ? 32 : blockDim.x, tid = W ? threadIdx.x & 31 : threadIdx.x, i0 = W ? (blockIdx.x * 8 + (threadIdx.x >> 5)) * M : blockIdx.x;
    const int A = p.n * p.topk, all = A + (p.shared ? p.n : 0);
    if (i0 >= all) return;
    int t[M], slot[M];
    float w[M], dot[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        const int i = i0 + m;
        t[m] = i < A ? i / p.topk : i - A;
        slot[m] = i < all ? p.slots[i] : -1;
        w[m] = i >= all ? 0.f : i >= A ? (p.sw ? p.sw[t[m]] : 1.f) : p.w ? p.w[i] : 1.f;
        dot[m] = 0.f;
    }
    for (int j0 = tid; j0 < p.pieces; j0 += P * nt) {
        uint4 g[M][P], v[M][P];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int c = 0; c < P; ++c)
                if (unsigned(slot[m]) < unsigned(p.rows) && j0 + c * nt < p.pieces) {
                    if (p.y) v[m][c] = p.y[size_t(slot[m]) * p.ldy + j0 + c * nt];
                    g[m][c] = p.dout[size_t(t[m]) * p.ldo + j0 + c * nt];
                }
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int c = 0; c < P; ++c)
                if (unsigned(slot[m]) < unsigned(p.rows) && j0 + c * nt < p.pieces) {
                    float a[N], f[N];
                    Vec<DT>::open(g[m][c], a);
                    if (p.y) {
                        Vec<DT>::open(v[m][c], f);
#pragma unroll
                        for (int l = 0; l < N; ++l) dot[m] = fmaf(a[l], f[l], dot[m]);
                    }
                    if (p.dy) {
#pragma unroll
                        for (int l = 0; l < N; ++l) a[l] *= w[m];
                        p.dy[size_t(slot[m]) * p.ldd + j0 + c * nt] = Vec<DT>::close(a);
                    }
                }
    }
    if (!p.dw && !p.dsw) return;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int d = 16; d; d >>= 1) dot[m] += __shfl_xor_sync(0xffffffffu, dot[m], d);
    if (!W) {
        if ((tid & 31) == 0) red[tid >> 5] = dot[0];
        __syncthreads();
        for (int u = 1; u < int(blockDim.x >> 5) && tid == 0; ++u) dot[0] += red[u];
    }
    if (tid) return;
#pragma unroll
    for (int m = 0; m < M; ++m) {
        const int i = i0 + m;
        if (i < A) {
            if (p.dw) p.dw[i] = dot[m];
        } else if (i < all && p.dsw) {
            p.dsw[t[m]] = dot[m];
        }
    }
}

// what the calls have in common; pieces of 16 bytes
// n * (topk + 1) stays inside 32 bits: topk >= 1 and n topk < 2^30
bool batch(int n, int topk, int hidden, int dtype) { return n > 0 && topk > 0 && (long long)n * topk <= MAX_ASSIGNMENTS && hidden > 0 && valid_dtype(dtype) && hidden % (16 / int(dtype_bytes(dtype))) == 0; }
bool stride(const void * p, long long ld, int hidden, int dtype) { return !p || (ld >= hidden && ld % (16 / (long long)dtype_bytes(dtype)) == 0); }
// From how many tokens on a launch looks the slots up first; parts of rows that the launches of fewer have at most. us, there: 64 tokens of 2048 to eleven slots whole / in parts 3.1 / 2.3, 140 of 4096 to eight 5.7 / 4.1; 1000 of 2048 to four
// in parts beyond this number 5.5 instead of 4.5
constexpr int MANY_TOKENS = 148 * 8, THERE_WARPS = 148 * 16;
// From how many assignments on a warp takes one in the gradient. us, block / warp: 640 of 2048 4.2 / 3.4, 2240 of 2048 8.2 / 4.6, 1120 of 4096 5.3 / 6.9, 41,000 of 2048 82 / 56
inline int grad_many(int pieces) { return 148 * (pieces <= 256 ? 4 : 8); }
// Up to how many pieces a row has two assignments go to a warp there. us, one / two / four a warp, bf16: 8192 tokens of 128 to four 9.7 / 8.0 / 9.0, of 512 12.3 / 10.5 / 13.5, of 1024 26.2 / 24.7 / 32.2, of 2048 46.5 / 48.0 / 58.3; 40,000 of
// 256 to two 35.3 / 23.3 / 26.1; 1000 of 256 to two 2.1 / 2.7 / 2.8, of 1024 3.1 / 4.6 / 5.1
constexpr int GRAD_ONE = 64;
int threads_for(int pieces) { return std::min(256, ceil_div(pieces, 32) * 32); }

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" B2MOE_API int32_t b2moe_dispatch_rows(const void * x, int32_t dtype, int64_t ldx, const int32_t * ids, const int32_t * plan, int32_t n, int32_t topk, int32_t hidden, int32_t experts,
                                                 int32_t shared_tokens, void * rows, int64_t ldr, int32_t * slots, b2moe_stream stream) {
    if (!batch(n, topk, hidden, dtype) || experts <= 0 || shared_tokens < 0 || shared_tokens > n || !stride(x, ldx, hidden, dtype) || !stride(rows, ldr, hidden, dtype)) return B2MOE_ERR_SHAPE;
    if (!x || !ids || !plan || !rows) return B2MOE_ERR_NULL;
    if (!aligned16(x) || !aligned16(rows) || !aligned_to(ids, 4) || !aligned_to(plan, 4) || !aligned_to(slots, 4)) return B2MOE_ERR_ALIGN;
    const int per = 16 / int(dtype_bytes(dtype)), pieces = hidden / per;
    const ThereArgs a{static_cast<const uint4 *>(x), static_cast<uint4 *>(rows), ids, plan, slots, ldx / per, ldr / per, pieces, n, topk, experts, shared_tokens};
    const long long all = n * (long long)topk + (shared_tokens ? n : 0);
    cudaStream_t s = as_stream(stream);
    if (!slots || n < MANY_TOKENS) {
        const int parts = int(std::max(1LL, std::min<long long>(ceil_div(pieces, 64), THERE_WARPS / all)));      // of a row, while that makes no more warps than run at once
        launch_overlapped(there_k, dim3(unsigned((all + 7) / 8), parts), dim3(256), 0, s, a);
        return launch_status();
    }
    launch_overlapped(slots_k, dim3(unsigned((all + 255) / 256)), dim3(256), 0, s, a);
    if (int32_t rc = launch_status()) return rc;
    if (pieces <= 64) launch_overlapped(there_token_k<2, true>, dim3(ceil_div(n, 8)), dim3(256), 0, s, a);
    else launch_overlapped(there_token_k<2, false>, dim3(n), dim3(std::min(256, ceil_div(pieces, 64) * 32)), 0, s, a);
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
    cudaStream_t s = as_stream(stream);
    const dim3 grid(n, ceil_div(pieces, threads));
    const int all = topk + (shared_tokens ? 1 : 0);
    const bool few = (long long)n * grid.y <= 2 * 148;
    auto go = [&](auto two, auto five, auto twelve) { launch_overlapped(all <= 2 ? two : few && all > 5 ? twelve : five, grid, dim3(threads), 0, s, a); };
    if (dtype == B2MOE_F32) go(back_k<B2MOE_F32, 2>, back_k<B2MOE_F32, 5>, back_k<B2MOE_F32, 12>);
    else if (dtype == B2MOE_F16) go(back_k<B2MOE_F16, 2>, back_k<B2MOE_F16, 5>, back_k<B2MOE_F16, 12>);
    else go(back_k<B2MOE_BF16, 2>, back_k<B2MOE_BF16, 5>, back_k<B2MOE_BF16, 12>);
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
    const long long all = (long long)n * topk + (shared_tokens ? n : 0);
    cudaStream_t s = as_stream(stream);
    auto go = [&](auto block, auto one, auto two) {
        if (all < grad_many(pieces)) return launch_overlapped(block, dim3(unsigned(all)), dim3(threads), 0, s, a);
        const int each = pieces > GRAD_ONE ? 1 : 2;
        launch_overlapped(each == 1 ? one : two, dim3(unsigned((all + 8 * each - 1) / (8 * each))), dim3(256), 0, s, a);
    };
    if (dtype == B2MOE_F32) go(back_grad_k<B2MOE_F32, 0>, back_grad_k<B2MOE_F32, 1>, back_grad_k<B2MOE_F32, 2>);
    else if (dtype == B2MOE_F16) go(back_grad_k<B2MOE_F16, 0>, back_grad_k<B2MOE_F16, 1>, back_grad_k<B2MOE_F16, 2>);
    else go(back_grad_k<B2MOE_BF16, 0>, back_grad_k<B2MOE_BF16, 1>, back_grad_k<B2MOE_BF16, 2>);
    return launch_status();
}
