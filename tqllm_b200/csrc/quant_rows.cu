// Rows of floating-point values -> 8-bit integers and a scale for each row: s = max|x| / 127, q = the integer nearest to 127 x / max|x|.
//
// One pass: a block holds its row in registers between the maximum and the rounding (rows of more than 16,384 values are read again, from the L2).
// Bound by memory: two or four bytes a value are read, one is written.
#include "int8.cuh"

namespace b2 {
namespace {

struct QuantArgs {
    const void * x;
    long long ldx, ldq;
    int k;
    int8_t * q;
    float * scale;
    const int * plan;                // null: row i of x; else slot i of the plan
    int experts, assignments, topk, per_token;
};

// The nearest integer to 127 x / top, halves to even, exactly: t = x * (127 / top) is off by less than 127 * 2^-22, so only values that close to a half
// need the comparison of 127 x with (m + 1/2) top, whose sides have 31 and 32 bits and are exact in 64-bit floats.
__device__ __forceinline__ int nearest(float x, float top, float inv) {
    const float t = x * inv, r = rintf(t);
    int q = int(r);
    if (fabsf(fabsf(t - r) - 0.5f) < 4e-5f) {
        const float m = floorf(t);
        const double a = 127.0 * double(x), h = (double(m) + 0.5) * double(top);
        const int lo = int(m);
        q = a > h ? lo + 1 : a < h ? lo : lo + (lo & 1);
    }
    return q;
}

// 16 neighbouring values of a row
template <int DT>
__device__ __forceinline__ void load16(const void * x, size_t i, float (&v)[16]) {
    if (DT == B2MOE_F32) {
        const float4 * p = reinterpret_cast<const float4 *>(static_cast<const float *>(x) + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4 f = p[j];
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        }
    } else {
        using T = typename Elem<DT == B2MOE_F32 ? B2MOE_F16 : DT>::type;
        const uint4 * p = reinterpret_cast<const uint4 *>(static_cast<const T *>(x) + i);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint4 w = p[j];
            const T * h = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int l = 0; l < 8; ++l) v[8 * j + l] = Elem<DT == B2MOE_F32 ? B2MOE_F16 : DT>::to_f(h[l]);
        }
    }
}

// C: pieces of 16 values that a thread holds; 0: more than that, the row is read twice
template <int DT, int C>
__global__ void __launch_bounds__(256) quant_rows_k(const QuantArgs p) {
    __shared__ float red[8];
    grid_release();
    grid_wait();
    long long src = blockIdx.x;
    if (p.plan) {
        if (int(blockIdx.x) >= p.plan[PLAN_NGROUPED]) return;
        const int * perm = p.plan + PLAN_HDR + 3 * (p.experts + 1) + 1;
        const int a = perm[blockIdx.x];
        src = !p.per_token ? a : a < p.assignments ? a / p.topk : a - p.assignments;
    }
    const size_t row = size_t(src) * p.ldx;
    const int pieces = p.k / 16, nt = blockDim.x;
    constexpr int H = C ? C : 1;
    float v[H][16];
    float top = 0.f;
    bool bad = false;                                                  // an infinity or a NaN in the row
    auto look = [&](const float (&w)[16]) {
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, fabsf(w[j]));
#pragma unroll
        for (int j = 0; j < 16; ++j) bad |= !(fabsf(w[j]) < INFINITY);
    };
    if (C) {
#pragma unroll
        for (int c = 0; c < H; ++c) {
            const int i = c * nt + threadIdx.x;
            if (i < pieces) load16<DT>(p.x, row + size_t(i) * 16, v[c]);
        }
#pragma unroll
        for (int c = 0; c < H; ++c)
            if (c * nt + int(threadIdx.x) < pieces) look(v[c]);
    } else {
        for (int i = threadIdx.x; i < pieces; i += nt) {
            load16<DT>(p.x, row + size_t(i) * 16, v[0]);
            look(v[0]);
        }
    }
    if (bad) top = INFINITY;
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (nt > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
        __syncthreads();
        top = red[0];
        for (int w = 1; w < nt / 32; ++w) top = fmaxf(top, red[w]);
    }
    if (threadIdx.x == 0) p.scale[blockIdx.x] = top < INFINITY ? __fdiv_rn(top, 127.f) : __int_as_float(0x7fc00000);
    const bool zero = top == 0.f || top == INFINITY;
    const float up = top < 0x1p-100f ? 0x1p100f : 1.f, t = top * up, inv = zero ? 0.f : __fdiv_rn(127.f, t);      // 127 / top would overflow below 2^-121
    int8_t * q = p.q + size_t(blockIdx.x) * p.ldq;
    auto put = [&](int i, const float (&w)[16]) {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] = 0;
#pragma unroll
            for (int l = 0; l < 4; ++l) o[j] |= (zero ? 0u : uint32_t(nearest(w[4 * j + l] * up, t, inv)) & 0xffu) << (8 * l);
        }
        *reinterpret_cast<uint4 *>(q + size_t(i) * 16) = make_uint4(o[0], o[1], o[2], o[3]);
    };
    if (C) {
#pragma unroll
        for (int c = 0; c < H; ++c) {
            const int i = c * nt + threadIdx.x;
            if (i < pieces) put(i, v[c]);
        }
    } else {
        for (int i = threadIdx.x; i < pieces; i += nt) {
            load16<DT>(p.x, row + size_t(i) * 16, v[0]);
            put(i, v[0]);
        }
    }
}

template <int DT>
void launch_quant(const QuantArgs & a, int n, cudaStream_t s) {
    // as many threads as the row has pieces, up to 256; the pieces a thread takes stay in registers up to four
    const int pieces = a.k / 16, threads = std::min(256, (pieces + 31) / 32 * 32), per = ceil_div(pieces, threads);
    auto go = [&](auto kernel) { launch_overlapped(kernel, dim3(n), dim3(threads), 0, s, a); };
    if (per == 1) go(quant_rows_k<DT, 1>);
    else if (per == 2) go(quant_rows_k<DT, 2>);
    else if (per <= 4) go(quant_rows_k<DT, 4>);
    else go(quant_rows_k<DT, 0>);
}

}  // namespace

int32_t i8_quantize(const void * x, int x_dtype, long long ldx, int n, int k, int8_t * q, long long ldq, float * scale, const int * plan, int experts,
                    int assignments, int topk, bool per_token, cudaStream_t s) {
    const QuantArgs a{x, ldx, ldq, k, q, scale, plan, experts, assignments, topk, per_token};
    if (x_dtype == B2MOE_F32) launch_quant<B2MOE_F32>(a, n, s);
    else if (x_dtype == B2MOE_F16) launch_quant<B2MOE_F16>(a, n, s);
    else launch_quant<B2MOE_BF16>(a, n, s);
    return launch_status();
}

}  // namespace b2

using namespace b2;

extern "C" B2MOE_API int32_t b2moe_quantize_rows(const void * x, int32_t x_dtype, int64_t ldx, int32_t n, int32_t k, int8_t * q, int64_t ldq, float * scale,
                                                 b2moe_stream stream) {
    if (n <= 0 || !i8_cols(k) || !valid_dtype(x_dtype) || ldx < k || ldx % (x_dtype == B2MOE_F32 ? 4 : 8) || ldq < k || ldq % 16) return B2MOE_ERR_SHAPE;
    if (!x || !q || !scale) return B2MOE_ERR_NULL;
    if (!aligned16(x) || !aligned16(q)) return B2MOE_ERR_ALIGN;
    return i8_quantize(x, x_dtype, ldx, n, k, q, ldq, scale, nullptr, 0, 0, 1, false, as_stream(stream));
}
