// Products of 8-bit integers with a scale for each activation row and each weight row: dense (b2moe_linear_i8) and grouped by expert, the expert
// products over a plan on banks of type B2MOE_I8.
//
//   sum_tr = sum_j q_tj w_rj   exactly, in 32-bit integers (so K may be split in any way and the order does not show in the result)
//   y_tr = sum_tr * (s_t v_r);   gate/up: act_tr = silu(g_tr) u_tr
//
// The sum is exact, y has three roundings (the sum to fp32, the product of the scales, their product) and the one to its own type.
#include <type_traits>

#include "int8.cuh"

namespace b2 {
int32_t check_bank(const b2moe_bank * b);
int harness_family();
namespace {

__device__ __forceinline__ void mma_i8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// weights are read once: past the L1
__device__ __forceinline__ uint4 load_stream(const int8_t * p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(__cvta_generic_to_global(p)));
    return r;
}

// A few tokens per expert: bound by streaming the weights. A block takes 16 weight rows of one expert (of both matrices with MATS = 2) and all the
// expert's tokens, 8 NT at a time; its warps share the columns in pieces of 64, 16 bytes a lane and row, straight from memory into the fragments of the tensor
// core: lane (g, t) holds bytes 16 t.. of rows g and g + 8, so word i of both operands stands for the same four columns, which is all that a sum over columns needs.
// UNROLL: steps that a warp asks for at once. EPI: a dense call with an epilogue.
template <int MATS, int NT, int UNROLL, bool EPI>
__global__ void __launch_bounds__(512) i8_stream_k(const I8Args p) {
    extern __shared__ int red[];                                       // [warps][MATS][NT][16 rows][8 tokens]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, g = lane >> 2, t = lane & 3, r0 = blockIdx.x * 16;
    // a dense call's weights are asked into the L2 while the launch in front of this one runs (they are not read before it is through): 4096 x 4096, one row, 5.0 -> 4.6 us
    if (!p.plan && threadIdx.x < 16 && r0 + int(threadIdx.x) < p.rows)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(__cvta_generic_to_global(p.w[0] + size_t(r0 + threadIdx.x) * p.cols)), "r"(uint32_t(p.cols)) : "memory");
    grid_wait();
    grid_release();                                                    // after the wait: a down product behind this launch may read the plan above its own
    int e = 0, count = p.n, first = 0;
    const int * perm = nullptr;
    if (p.plan) {
        const int e1 = p.experts + 1;
        if (int(blockIdx.y) >= p.plan[PLAN_NACTIVE]) return;
        e = p.plan[PLAN_HDR + 2 * e1 + 1 + blockIdx.y];
        count = p.plan[PLAN_HDR + e];
        first = p.plan[PLAN_HDR + e1 + e];
        perm = p.plan + PLAN_HDR + 3 * e1 + 1 + first;
    }
    const bool shared = p.plan && e == p.experts;
    if (shared && !p.shared_w[0]) return;                              // a plan with a shared expert, a call without one
    const int rg = min(r0 + g, p.rows - 1), rh = min(r0 + g + 8, p.rows - 1);
    const int8_t * wg[MATS], * wh[MATS];
    const float * v[MATS];
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
        const int8_t * w = shared ? p.shared_w[m] : p.w[m] + size_t(e) * p.rows * p.cols;
        wg[m] = w + size_t(rg) * p.cols + 16 * t;
        wh[m] = w + size_t(rh) * p.cols + 16 * t;
        v[m] = shared ? p.shared_v[m] : p.v[m] + size_t(e) * p.rows;
    }
    const int steps = (p.cols + 63) / 64;
#pragma unroll 1
    for (int j0 = 0; j0 < count; j0 += 8 * NT) {
        const int8_t * b[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int j = min(j0 + 8 * i + g, count - 1);
            b[i] = p.q + size_t(p.plan ? source_row(p, first + j, perm[j]) : j) * p.ldq + 16 * t;
        }
        int acc[MATS][NT][4] = {};
#pragma unroll 1
        for (int s0 = warp; s0 < steps; s0 += UNROLL * warps) {
            uint4 x[UNROLL][NT], ag[UNROLL][MATS], ah[UNROLL][MATS];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int k = 64 * (s0 + u * warps);
                const bool in = k + 16 * t < p.cols;
#pragma unroll
                for (int m = 0; m < MATS; ++m) {
                    ag[u][m] = in ? load_stream(wg[m] + k) : make_uint4(0, 0, 0, 0);
                    ah[u][m] = in ? load_stream(wh[m] + k) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) x[u][i] = in ? *reinterpret_cast<const uint4 *>(b[i] + k) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                for (int m = 0; m < MATS; ++m)
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        mma_i8(acc[m][i], ag[u][m].x, ah[u][m].x, ag[u][m].y, ah[u][m].y, x[u][i].x, x[u][i].y);
                        mma_i8(acc[m][i], ag[u][m].z, ah[u][m].z, ag[u][m].w, ah[u][m].w, x[u][i].z, x[u][i].w);
                    }
        }
        if (j0) __syncthreads();                                       // the sums of the tokens before have been read
#pragma unroll
        for (int m = 0; m < MATS; ++m)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                int2 * d = reinterpret_cast<int2 *>(red + ((warp * MATS + m) * NT + i) * 128);
                d[g * 4 + t] = make_int2(acc[m][i][0], acc[m][i][1]);
                d[(g + 8) * 4 + t] = make_int2(acc[m][i][2], acc[m][i][3]);
            }
        __syncthreads();
        for (int x = threadIdx.x; x < 128 * NT; x += blockDim.x) {
            const int r = x & 15, jj = x >> 4, j = j0 + jj, row = r0 + r;
            if (row >= p.rows || j >= count) continue;
            int sum[MATS];
#pragma unroll
            for (int m = 0; m < MATS; ++m) {
                sum[m] = 0;
                for (int w = 0; w < warps; ++w) sum[m] += red[((w * MATS + m) * NT + (jj >> 3)) * 128 + r * 8 + (jj & 7)];
            }
            const int a = p.plan ? perm[j] : j;
            const float s = p.s[p.plan ? source_row(p, first + j, a) : j];
            float out = float(sum[0]) * (s * v[0][row]);
            if (MATS == 2) {
                const float u = float(sum[MATS - 1]) * (s * v[MATS - 1][row]);
                out = out / (1.f + expf(-out)) * u;
            }
            if (EPI) out = finish_one(p, sum[0], s * v[0][row], p.bias ? p.bias[row] : 0.f, p.residual ? load_act(p.residual, p.y_dtype, size_t(j) * p.ldr + row) : 0.f);
            store_act(p.y, p.y_dtype, size_t(a) * p.ldy + row, out);
        }
    }
}

// Warps that share a block's columns: eight where a launch has few blocks, else four; sixteen for long rows of a dense call whose blocks are all on the SMs at once. us with 4 / 8 / 16, one row:
//   4096 x 4096 10.0 / 6.5 / 4.6      2048 x 8192 15.7 / 9.3 / 6.2      1411 x 2560 5.1 / 3.6 / 2.9      1024 x 2048 4.2 / 3.0 / 2.7
//   512 x 1024   2.4 / 2.2 / 2.4      8192 x 1024  3.7 / 3.4 / 5.5      gate/up of one token of ten experts 11.3 / 9.0 / 12.1
// Eight steps at once where a warp has as many (before / with): 8192 x 8192 16.1 / 15.3, 2048 x 8192 6.1 / 5.7; down of 64 experts of 4096 x 4096 at three each 181.6 / 171.8, of eight of
// 2048 x 4096 17.9 / 17.0; where it has fewer it loses: 4096 x 4096 4.5 / 4.8
template <int MATS, int NT, bool EPI>
int32_t launch_stream(const I8Args & a, int groups, cudaStream_t s) {
    const int blocks = ceil_div(a.rows, 16), steps = ceil_div(a.cols, 64);
    const int warps = !a.plan && blocks <= 148 * 2 && steps >= 32 ? 16 : (long long)blocks * groups < 148 * 4 ? 8 : 4;
    auto kernel = i8_stream_k<MATS, NT, (NT > 2 ? 2 : 4), EPI>;
    if constexpr (MATS == 1 && NT == 1)
        if (steps >= 8 * warps) kernel = i8_stream_k<1, 1, 8, EPI>;
    launch_overlapped(kernel, dim3(blocks, groups), dim3(32 * warps), size_t(warps) * MATS * NT * 128 * sizeof(int), s, a);
    return launch_status();
}
template <int MATS, bool EPI = false>
int32_t i8_stream(const I8Args & a, int groups, long long tokens, cudaStream_t s) {
    if (groups > 65535) return B2MOE_ERR_SHAPE;                        // the grid's second extent
    // rows that a pass over the weights serves: a second pass of some experts (from the L2) costs less than the registers of 16 rows (512 experts at five each: 184 and 222 us)
    if (tokens <= 8LL * groups) return launch_stream<MATS, 1, EPI>(a, groups, s);
    if (tokens <= 16LL * groups) return launch_stream<MATS, 2, EPI>(a, groups, s);
    return launch_stream<MATS, 4, EPI>(a, groups, s);
}
int groups_of(int experts, int n, int topk, int shared_tokens) { return int(std::min((long long)n * topk, (long long)experts)) + (shared_tokens ? 1 : 0); }

I8Args grouped(const b2moe_bank * a, const b2moe_bank * b, const b2moe_bank * sa, const b2moe_bank * sb, const int * plan, int n, int topk, int shared_tokens, void * y, int y_dtype) {
    I8Args p{};
    const b2moe_bank * m[2] = {a, b}, * sm[2] = {sa, sb};
    for (int i = 0; i < 2; ++i) {
        if (m[i]) { p.w[i] = static_cast<const int8_t *>(m[i]->data); p.v[i] = static_cast<const float *>(m[i]->aux); }
        if (shared_tokens && sm[i]) { p.shared_w[i] = static_cast<const int8_t *>(sm[i]->data); p.shared_v[i] = static_cast<const float *>(sm[i]->aux); }
    }
    p.experts = a->experts; p.rows = a->rows; p.cols = a->cols;
    p.plan = plan; p.n = n; p.assignments = n * topk; p.topk = topk;
    p.y = y; p.y_dtype = y_dtype; p.ldy = a->rows;
    return p;
}

}  // namespace

size_t i8_workspace_bytes(int rows_x, int k) { return i8_rows_bytes(rows_x, k); }
// rows in slot order, and the slot of every assignment
size_t i8_slot_bytes(int slot_rows, int k) { return i8_rows_bytes(slot_rows, k) + align_up(size_t(slot_rows) * sizeof(int), 256); }

// The form of a product: the streaming kernel for a few rows, the tensor-core GEMM (int8_gemm.cu) for more. us, streamed / GEMM:
//   dense, from 17 rows on
//     4096 x 4096   16 rows 5.5 / 8.0, 24 7.9 / 8.0, 48 13.1 / 8.2          2048 x 8192   16 6.9 / 8.8, 17 10.4 / 8.9
//     1411 x 2560   16 3.6 / 5.9, 32 5.7 / 6.0                              8192 x 8192   16 17.3 / 15.5, 17 22.4 / 15.3
//   gate/up, from seven rows per expert on (the GEMM's times have a launch more in them, since its rows lie in slot order)
//     128 experts of 1408 x 4096   at 4 each 221 / 233, at 8 307 / 245      512 of 512 x 2048   at 2.5 155 / 168, at 5 184 / 187
//     32 of 512 x 1024   at 4 8.9 / 14.2, at 16 17.1 / 15.3
//   down, where they are in slot order anyway, also where the SMs get eight items each, and for short rows from three per expert or four items an SM on
//     128 of 4096 x 1408   at 0.5 63 / 60, at 1 95 / 80, at 4 138 / 120     512 of 2048 x 512   two tokens of ten 9.5 / 9.7, four 14.8 / 11.9, 64 110 / 67
//     32 of 1024 x 512   at 2 7.8 / 7.7, at 4 9.6 / 7.6
constexpr int I8_DENSE_ROWS = 16, I8_GEMM_MIN_PER = 7, I8_SHORT_MIN_PER = 3, I8_MANY_ITEMS = 148 * 8, I8_SHORT_ITEMS = 148 * 4;
bool i8_takes_gemm(int experts, bool worth) {
    const int family = harness_family();
    if (!i8_gemm_supported(experts) || family == B2MOE_FAMILY_GENERIC || family == B2MOE_FAMILY_DECODE || family == B2MOE_FAMILY_DECODE_KERNELS) return false;
    return family == B2MOE_FAMILY_GEMM || worth;
}
int per_group(int experts, long long rows) { return int(std::min<long long>(1 << 20, (rows + experts - 1) / experts)); }

// x [n][cols]; the workspace holds the rows of the n tokens
int32_t i8_gateup(const b2moe_bank * gate, const b2moe_bank * up, const b2moe_bank * shared_gate, const b2moe_bank * shared_up, const void * x, int x_dtype, const int * plan, int n,
                  int topk, int shared_tokens, long long live, void * act, int act_dtype, void * ws, void * rows_buf, size_t rows_buf_bytes, cudaStream_t s) {
    if ((long long)n * topk + shared_tokens > I8_MAX_ROWS) return B2MOE_ERR_SHAPE;
    I8Args p = grouped(gate, up, shared_gate, shared_up, plan, n, topk, shared_tokens, act, act_dtype);
    const int total = n * topk + shared_tokens;
    if (i8_takes_gemm(gate->experts, live >= (long long)I8_GEMM_MIN_PER * gate->experts) && rows_buf_bytes >= i8_slot_bytes(total, gate->cols)) {
        const I8Rows rows = i8_rows(rows_buf, total);
        int * inverse = reinterpret_cast<int *>(static_cast<char *>(rows_buf) + i8_rows_bytes(total, gate->cols));
        if (int32_t rc = i8_quantize_scatter(x, x_dtype, n, gate->cols, rows, inverse, plan, gate->experts, topk, shared_tokens, s)) return rc;
        p.q = rows.q; p.ldq = gate->cols; p.s = rows.scale; p.slots = 1;
        return i8_gemm<2>(p, total, per_group(gate->experts, live), const_cast<int *>(plan) + PLAN_STATUS, s);
    }
    const I8Rows rows = i8_rows(ws, n);
    if (int32_t rc = i8_quantize(x, x_dtype, gate->cols, n, gate->cols, rows.q, gate->cols, rows.scale, s)) return rc;
    p.q = rows.q; p.ldq = gate->cols; p.s = rows.scale; p.per_token = 1;
    return i8_stream<2>(p, groups_of(gate->experts, n, topk, shared_tokens), live + shared_tokens, s);
}
// x [assignments][cols] (per_token: [n][cols]); the workspace holds a row per assignment, in slot order
int32_t i8_down(const b2moe_bank * down, const b2moe_bank * shared_down, const void * x, int x_dtype, bool per_token, const int * plan, int n, int topk, int shared_tokens, long long live,
                void * y, int y_dtype, void * ws, cudaStream_t s) {
    if ((long long)n * topk + shared_tokens > I8_MAX_ROWS) return B2MOE_ERR_SHAPE;
    I8Args p = grouped(down, nullptr, shared_down, nullptr, plan, n, topk, shared_tokens, y, y_dtype);
    const int total = n * topk + shared_tokens;
    const I8Rows rows = i8_rows(ws, total);
    if (int32_t rc = i8_quantize_slots(x, x_dtype, per_token, n, down->cols, rows, plan, down->experts, topk, shared_tokens, s)) return rc;
    p.q = rows.q; p.ldq = down->cols; p.s = rows.scale; p.slots = 1;
    const bool short_rows = down->cols <= I8_SHORT_COLS, all = live == (long long)n * topk;
    const long long items = (long long)groups_of(down->experts, n, topk, shared_tokens) * ceil_div(down->rows, 128);
    if (i8_takes_gemm(down->experts, live >= (long long)(short_rows ? I8_SHORT_MIN_PER : I8_GEMM_MIN_PER) * down->experts || (all && items >= (short_rows ? I8_SHORT_ITEMS : I8_MANY_ITEMS))))
        return i8_gemm<1>(p, total, per_group(down->experts, live), const_cast<int *>(plan) + PLAN_STATUS, s);
    return i8_stream<1>(p, groups_of(down->experts, n, topk, shared_tokens), live + shared_tokens, s);
}

namespace {
__global__ void i8_dump_k(const int8_t * w, const float * v, int rows, int cols, float * out) {
    const size_t row = blockIdx.x;
    for (int j = threadIdx.x; j < cols; j += blockDim.x) out[row * cols + j] = float(w[row * cols + j]) * v[row];
}
}  // namespace
int32_t i8_dump(const b2moe_bank & b, float * out, cudaStream_t s) {
    const long long rows = (long long)b.experts * b.rows;
    if (rows > 0x7fffffffLL) return B2MOE_ERR_SHAPE;
    i8_dump_k<<<unsigned(rows), 128, 0, s>>>(static_cast<const int8_t *>(b.data), static_cast<const float *>(b.aux), b.rows, b.cols, out);
    return launch_status();
}

}  // namespace b2

using namespace b2;

static int32_t linear_any(const int8_t * q, int64_t ldq, const float * scale, const b2moe_bank * w, int32_t n, const float * bias, int32_t act, const void * residual, int64_t ldr, void * y,
                          int32_t y_dtype, int64_t ldy, int32_t * status, b2moe_stream stream) {
    if (int32_t rc = check_bank(w)) return rc;
    if (w->type != B2MOE_I8) return B2MOE_ERR_FORMAT;
    if (n <= 0 || n > I8_MAX_ROWS || w->experts != 1 || !valid_dtype(y_dtype) || ldq < w->cols || ldq % 16 || ldy < w->rows) return B2MOE_ERR_SHAPE;
    if (act < B2MOE_ACT_NONE || act > B2MOE_ACT_GELU_TANH || (residual && ldr < w->rows)) return B2MOE_ERR_SHAPE;
    if (!q || !scale || !y) return B2MOE_ERR_NULL;
    if (!aligned16(q) || !aligned_to(y, dtype_bytes(y_dtype)) || !aligned_to(scale, 4) || !aligned_to(status, 4)) return B2MOE_ERR_ALIGN;
    if (!aligned_to(bias, 4) || !aligned_to(residual, dtype_bytes(y_dtype))) return B2MOE_ERR_ALIGN;
    I8Args p{};
    p.w[0] = static_cast<const int8_t *>(w->data); p.v[0] = static_cast<const float *>(w->aux);
    p.experts = 1; p.rows = w->rows; p.cols = w->cols;
    p.q = q; p.ldq = ldq; p.s = scale; p.n = n;
    p.y = y; p.y_dtype = y_dtype; p.ldy = ldy;
    p.bias = bias; p.residual = residual; p.ldr = ldr; p.act = act;
    if (i8_takes_gemm(1, n > I8_DENSE_ROWS)) return i8_gemm<1>(p, n, n, status, as_stream(stream));
    return has_epilogue(p) ? i8_stream<1, true>(p, 1, n, as_stream(stream)) : i8_stream<1>(p, 1, n, as_stream(stream));
}

extern "C" B2MOE_API int32_t b2moe_linear_i8(const int8_t * q, int64_t ldq, const float * scale, const b2moe_bank * w, int32_t n, void * y, int32_t y_dtype, int64_t ldy, int32_t * status,
                                             b2moe_stream stream) {
    return linear_any(q, ldq, scale, w, n, nullptr, B2MOE_ACT_NONE, nullptr, 0, y, y_dtype, ldy, status, stream);
}
extern "C" B2MOE_API int32_t b2moe_linear_i8_epilogue(const int8_t * q, int64_t ldq, const float * scale, const b2moe_bank * w, int32_t n, const float * bias, int32_t act, const void * residual,
                                                      int64_t ldr, void * y, int32_t y_dtype, int64_t ldy, int32_t * status, b2moe_stream stream) {
    return linear_any(q, ldq, scale, w, n, bias, act, residual, ldr, y, y_dtype, ldy, status, stream);
}
