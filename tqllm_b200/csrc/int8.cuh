// What the kernels of 8-bit banks (B2MOE_I8) share: the operand form of activation rows and the entry points between the files.
#pragma once
#include <algorithm>

#include "common.cuh"

namespace b2 {

// |q w| <= 2^14 each: sums of fewer than 2^17 products stay inside 32 bits
constexpr int I8_MAX_COLS = (1 << 17) - 16;
inline bool i8_cols(int cols) { return cols > 0 && cols % 16 == 0 && cols <= I8_MAX_COLS; }

// Operand form of activation rows inside a workspace: `rows` 8-bit rows of k values, a scale each
struct I8Rows { int8_t * q; float * scale; };
inline size_t i8_rows_bytes(int rows, int k) { return align_up(size_t(rows) * sizeof(float), 256) + align_up(size_t(rows) * k, 256); }
inline I8Rows i8_rows(void * ws, int rows) {
    return {reinterpret_cast<int8_t *>(ws) + align_up(size_t(rows) * sizeof(float), 256), static_cast<float *>(ws)};
}

// rows x[0..n) of ldx elements -> q (stride ldq), scale. plan: the rows of the grouped assignments in slot order instead (slot i holds assignment
// perm[i], whose row is its token's with per_token and its own otherwise), at most n of them
int32_t i8_quantize(const void * x, int x_dtype, long long ldx, int n, int k, int8_t * q, long long ldq, float * scale, const int * plan, int experts,
                    int assignments, int topk, bool per_token, cudaStream_t s);

}  // namespace b2
