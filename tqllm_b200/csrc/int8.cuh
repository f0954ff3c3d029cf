// What the kernels of 8-bit banks (B2MOE_I8) share: the operand form of activation rows and the entry points between the files.
#pragma once
#include <algorithm>

#include "common.cuh"
#include "two.cuh"

namespace b2 {

// |q w| <= 2^14 each: sums of fewer than 2^17 products stay inside 32 bits
constexpr int I8_MAX_COLS = (1 << 17) - 16;
// rows up to here are short: the tensor-core form runs two blocks an SM
constexpr int I8_SHORT_COLS = 1024;
// rows of a call or of an expert, assignments: tile arithmetic stays inside 32 bits
constexpr int I8_MAX_ROWS = (1 << 30) - 1;
inline bool i8_cols(int cols) { return cols > 0 && cols % 16 == 0 && cols <= I8_MAX_COLS; }

// Operand form of activation rows inside a workspace: `rows` 8-bit rows of k values, a scale each
struct I8Rows { int8_t * q; float * scale; };
inline size_t i8_rows_bytes(int rows, int k) { return align_up(size_t(rows) * sizeof(float), 256) + align_up(size_t(rows) * k, 256); }
inline I8Rows i8_rows(void * ws, int rows) {
    return {reinterpret_cast<int8_t *>(ws) + align_up(size_t(rows) * sizeof(float), 256), static_cast<float *>(ws)};
}

// One product, or gate and up together
struct I8Args {
    const int8_t * w[2], * shared_w[2];          // gate and up, or one matrix: [experts][rows][cols]
    const float * v[2], * shared_v[2];           // their scales, [experts][rows]
    int experts, rows, cols;
    const int8_t * q;                            // rows in operand form
    long long ldq;
    const float * s;
    const int * plan;                            // null: one matrix, rows 0..n of q
    int n, assignments, topk, per_token, slots;  // slots: row i of q belongs to slot i of the plan; else to its token (per_token) or assignment
    void * y;
    int y_dtype;
    long long ldy;
    // what follows a dense product (null, null, B2MOE_ACT_NONE: nothing): y = act(product + bias) + residual, residual of y's type
    const float * bias;
    const void * residual;
    long long ldr;
    int act;
};

inline bool has_epilogue(const I8Args & a) { return a.bias || a.residual || a.act != B2MOE_ACT_NONE; }

__device__ __forceinline__ Two reciprocal(Two a) {                     // off by one step; 1 / inf = 0
    float2 f = apart(a);
    asm("rcp.approx.f32 %0, %0;" : "+f"(f.x));
    asm("rcp.approx.f32 %0, %0;" : "+f"(f.y));
    return two(f.x, f.y);
}
__device__ __forceinline__ Two exp2_near(Two a) {                      // off by two steps
    float2 f = apart(a);
    asm("ex2.approx.f32 %0, %0;" : "+f"(f.x));
    asm("ex2.approx.f32 %0, %0;" : "+f"(f.y));
    return two(f.x, f.y);
}
__device__ __forceinline__ float exp2_normal(float a) {                // off by two steps; zero below 2^-126
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
    return a;
}
// erfc(x / sqrt 2), x >= 0, as e^(-x^2 / 2) t Q(t) with t = 1 / (1 + 0.265 x): Q was fitted to erfcx on (0, 14.5] for the least largest relative error (1.4e-8). With its roundings 12 + 2 x^2 steps
// of 2^-24 at most, and no branch
__device__ __forceinline__ Two normal_tail(Two x) {
    const Two t = reciprocal(fma2(two(0.265f), x, two(1.f)));
    Two q = two(0.061249539f);
    q = fma2(q, t, two(-0.28660402f));
    q = fma2(q, t, two(0.43190601f));
    q = fma2(q, t, two(-0.22857844f));
    q = fma2(q, t, two(0.27311337f));
    q = fma2(q, t, two(0.12178868f));
    q = fma2(q, t, two(0.20511049f));
    q = fma2(q, t, two(0.21053351f));
    q = fma2(q, t, two(0.2114808f));
    return exp2_near(two(-0.72134752f) * x * x) * (t * q);
}
// 2 N values at a time under one switch, so that they are in flight together. What is small stays exact to its own size: the negative tail of GELU is a complementary error function,
// (1 + tanh z) / 2 = 1 / (1 + e^-2z), or e^z e^z / (1 + e^2z) below zero, and where e^-v passes 32 bits before v / (1 + e^-v) leaves them, that is v e^(v / 2) e^(v / 2). A NaN stays one
constexpr float FAR_SILU = -80.f;                // (selects instead of the branch: 4096 rows of 4096 x 512 36.6 us instead of 35.3)
template <int N>
__device__ __forceinline__ void activate(int act, Two (&f)[N]) {
    if (act == B2MOE_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 v = apart(f[i]);
            f[i] = two(v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y);
        }
    } else if (act == B2MOE_ACT_SILU) {
        float least = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) least = fminf(least, fminf(apart(f[i]).x, apart(f[i]).y));
        if (least >= FAR_SILU) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 v = apart(f[i]);
                f[i] = f[i] * reciprocal(two(expf(-v.x), expf(-v.y)) + two(1.f));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float2 v = apart(f[i]);
                const bool x = v.x < FAR_SILU, y = v.y < FAR_SILU;
                const Two e = two(expf(x ? 0.5f * v.x : -v.x), expf(y ? 0.5f * v.y : -v.y));
                const float2 near = apart(f[i] * reciprocal(e + two(1.f))), far = apart(f[i] * e * e);
                f[i] = two(x ? far.x : near.x, y ? far.y : near.y);
            }
        }
    } else if (act == B2MOE_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float2 v = apart(f[i]);
            const Two x = two(fminf(fabsf(v.x), 1e30f), fminf(fabsf(v.y), 1e30f));
            f[i] = fma2(two(-0.5f) * x, normal_tail(x), two(v.x < 0.f ? 0.f : v.x, v.y < 0.f ? 0.f : v.y));
        }
    } else if (act == B2MOE_ACT_GELU_TANH) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const Two z = two(1.1511041f) * fma2(two(0.044715f) * f[i] * f[i], f[i], f[i]);        // log2(e) z. (Without the root, an exponential below the normal numbers: 4096 x 512 34.1 us instead of 32.5)
            const float2 v = apart(z);
            const float ex = exp2_normal(-fabsf(v.x)), ey = exp2_normal(-fabsf(v.y));              // e^-|z|: a normal number as long as the output is one
            const Two e = two(ex, ey), low = two(v.x < 0.f ? ex : 1.f, v.y < 0.f ? ey : 1.f);
            f[i] = f[i] * low * low * reciprocal(fma2(e, e, two(1.f)));
        }
    }
}
// outputs of one weight row with what follows the product (scale: of the row times of the weight row); every rounding is written out, so that all forms give the same bits
template <int N>
__device__ __forceinline__ void finish(const I8Args & p, const int (&sum)[N], const Two (&scale)[N / 2], float bias, const float (&residual)[N], Two (&f)[N / 2]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) f[i] = two(float(sum[2 * i]), float(sum[2 * i + 1])) * scale[i] + two(bias);
    activate(p.act, f);
    if (p.residual)
#pragma unroll
        for (int i = 0; i < N / 2; ++i) f[i] = f[i] + two(residual[2 * i], residual[2 * i + 1]);
}
__device__ __forceinline__ float finish_one(const I8Args & p, int sum, float scale, float bias, float residual) {
    Two f[1];
    finish<2>(p, {sum, 0}, {two(scale, 0.f)}, bias, {residual, 0.f}, f);
    return apart(f[0]).x;
}

__device__ __forceinline__ int source_row(const I8Args & p, int slot, int a) {
    return p.slots ? slot : !p.per_token ? a : a < p.assignments ? a / p.topk : a - p.assignments;
}

// rows x[0..n) of ldx elements -> q (stride ldq), scale
int32_t i8_quantize(const void * x, int x_dtype, long long ldx, int n, int k, int8_t * q, long long ldq, float * scale, cudaStream_t s);
// the rows of the grouped assignments in slot order: slot i holds assignment perm[i], whose row is its token's (per_token) or its own
int32_t i8_quantize_slots(const void * x, int x_dtype, bool per_token, int n, int k, const I8Rows & rows, const int * plan, int experts, int topk, int shared_tokens, cudaStream_t s);
// the same for rows of tokens, each quantised once and written to all its slots; inverse: scratch, a word per assignment
int32_t i8_quantize_scatter(const void * x, int x_dtype, int n, int k, const I8Rows & rows, int * inverse, const int * plan, int experts, int topk, int shared_tokens, cudaStream_t s);

// the tensor-core form for many rows (int8_gemm.cu): true when it takes banks of this many experts; status: where a wait that runs out is noted (may be null);
// per_group: expected rows per expert. Rows of grouped calls lie in slot order
bool i8_gemm_supported(int experts);
template <int MATS> int32_t i8_gemm(const I8Args & a, long long q_rows, int per_group, int * status, cudaStream_t s);

}  // namespace b2
