// What the kernels of 8-bit banks (B2MOE_I8) share: the operand form of activation rows and the entry points between the files.
#pragma once
#include <algorithm>

#include "common.cuh"

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
};

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
