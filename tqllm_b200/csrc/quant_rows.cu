// Rows of floating-point values -> 8-bit integers and a scale for each row: s = max|x| / 127, q = the integer nearest to 127 x / max|x|.
//
// One pass: the row stays in registers between the maximum and the rounding (rows of more than 16,384 values are read again, from the L2).
// Bound by memory: two or four bytes a value are read, one is written. 8192 x 4096 bf16 take 15.9 us (6.3 TB/s, 0.97 of measured; 33 us with a rounding, a conversion and
// an exactness test of its own for each value), 40960 x 512 fp32 17.9 us (0.90).
#include <cstring>
#include <type_traits>

#include "int8.cuh"

namespace b2 {
namespace {

struct QuantArgs {
    const void * x;
    long long ldx, ldq;
    int n, k;
    int8_t * q;
    float * scale;
    const int * plan;                // null: row i of x; else slot i of the plan
    int experts, assignments, topk, per_token;
    int shared;
    const int * inverse;             // SCATTER: row i is quantised once and written to the slots of its assignments
};

// The nearest integer to 127 x / top, halves to even, exactly: 127 x and (m + 1/2) top have 31 and 32 bits and are compared in 64-bit floats
__device__ __noinline__ uint32_t nearest_exact(float x, float top) {
    const double a = 127.0 * double(x), m = floor(a / double(top)), h = (m + 0.5) * double(top);
    const int lo = int(m);
    return uint32_t(a > h ? lo + 1 : a < h ? lo : lo + (lo & 1)) & 0xffu;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 16 neighbouring values of a row as they lie in memory
template <int DT> struct Piece {
    static constexpr int W = DT == B2MOE_F32 ? 4 : 2;                 // 16-byte words
    uint4 w[W];
    __device__ __forceinline__ void load(const void * x, size_t i) {
        const uint4 * p = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(x) + i * (DT == B2MOE_F32 ? 4 : 2));
#pragma unroll
        for (int j = 0; j < W; ++j) w[j] = p[j];
    }
    __device__ __forceinline__ uint32_t word(int j) const { return j % 4 == 0 ? w[j / 4].x : j % 4 == 1 ? w[j / 4].y : j % 4 == 2 ? w[j / 4].z : w[j / 4].w; }
    __device__ __forceinline__ float value(int i) const {
        if (DT == B2MOE_F32) return __uint_as_float(word(i));
        const uint32_t u = word(i / 2);
        if (DT == B2MOE_BF16) return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
        return __half2float(__ushort_as_half((unsigned short)(i & 1 ? u >> 16 : u & 0xffffu)));
    }
    // the largest magnitude; a NaN where there is one
    __device__ __forceinline__ float top() const {
        if (DT == B2MOE_F32) {
            float m = fabsf(value(0));
#pragma unroll
            for (int i = 1; i < 16; ++i) m = max_nan(m, fabsf(value(i)));
            return m;
        }
        using V = typename std::conditional<DT == B2MOE_BF16, __nv_bfloat162, __half2>::type;
        auto at = [&](int j) { const uint32_t u = word(j); return __habs2(*reinterpret_cast<const V *>(&u)); };
        V m = at(0);
#pragma unroll
        for (int j = 1; j < 8; ++j) m = __hmax2_nan(m, at(j));
        uint32_t u;
        memcpy(&u, &m, 4);
        Piece q;
        q.w[0].x = u;
        return max_nan(q.value(0), q.value(1));
    }
    // the piece once more, values close to a half exactly (a function of its own: the registers of what is rare do not count in the kernel)
    static __device__ __noinline__ uint4 again(const Piece w, float top, float inv, float near) {
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[j] = 0;
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const float x = w.value(4 * j + l), f = __fmaf_rn(x, inv, 12582912.f);
                o[j] |= (fabsf(__fmaf_rn(x, inv, 12582912.f - f)) > near ? nearest_exact(x, top) : __float_as_uint(f) & 0xffu) << (8 * l);
            }
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
    // x * inv + 1.5 * 2^23 is the nearest integer in the low bits of a float. With CHECK, values whose quotient lies further than `near` from an integer are done
    // again, exactly
    template <bool CHECK>
    __device__ __forceinline__ uint4 quantized(float top, float inv, float near) const {
        constexpr float MAGIC = 12582912.f;
        uint32_t o[4];
        float off = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t b[4];
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                const float x = value(4 * j + l), f = __fmaf_rn(x, inv, MAGIC);
                b[l] = __float_as_uint(f);
                if (CHECK) off = fmaxf(off, fabsf(__fmaf_rn(x, inv, MAGIC - f)));
            }
            o[j] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
        }
        if (CHECK && off > near) return again(*this, top, inv, near);
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
};

// a piece of 16-bit values, exactly: 127 x and (m + 1/2) top have 18 and 19 bits and are compared as they are
template <int DT>
__device__ __noinline__ uint4 exact_piece(const Piece<DT> w, float top) {
    const float up = top < 0x1p-100f ? 0x1p100f : 1.f, t = top * up, inv = __fdiv_rn(127.f, t);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        o[j] = 0;
#pragma unroll
        for (int l = 0; l < 4; ++l) {
            const float x = w.value(4 * j + l) * up, m = floorf(x * inv), a = 127.f * x, h = (m + 0.5f) * t;
            const int lo = int(m);
            o[j] |= (uint32_t(a > h ? lo + 1 : a < h ? lo : lo + (lo & 1)) & 0xffu) << (8 * l);
        }
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

// How a row is rounded: q = the integer nearest to x * inv, and what has to be done exactly.
//   fp32: inv = 127 / top rounded, x * inv is off by 127 * 2^-24 at most: values that close to a half are done again.
//   16 bits: a quotient t = 127 x / top of two such values is a half or at least t * 2^-19 away from one, and x * inv with inv rounded up is off by less than
//   t * 2^-22: only halves are in question. 127 divides 2 m + 1 at the half m + 1/2 unless it divides the mantissa of top, so the half is 63.5 (x = top / 2: one value in a thousand),
//   and the rounding of inv moves it away from zero, to 64, the even side. Where it does divide the mantissa, inv is exact (and halves go to the even side by themselves) or
//   the row is done exactly (seven of 1,024 mantissas of fp16).
// tests/test_int8_host.py goes through all pairs of mantissas. Where 127 / top would overflow, all values of the row are done exactly.
struct Rule { float inv, near; bool check; };
template <int DT>
__device__ __forceinline__ Rule rule_of(float top) {
    if (!(top < INFINITY) || top == 0.f) return {0.f, 1.f, false};
    if (top < 0x1p-120f) return {0.f, -1.f, true};
    if (DT == B2MOE_F32) return {__fdiv_rn(127.f, top), 0.5f - 1e-5f, true};
    const float inv = __fdiv_ru(127.f, top);
    return {inv, 1.f, ((__float_as_uint(top) & 0x7fffffu) | 0x800000u) % 127u == 0u && __fmaf_rn(inv, top, -127.f) != 0.f};
}

// C: pieces that a thread holds; 0: more than that, the row is read twice. WARP: a warp takes a row (launches of many rows: no barrier, eight rows a block);
// otherwise the block does
template <int DT, int C, bool WARP, bool SCATTER>
__global__ void __launch_bounds__(256) quant_rows_k(const QuantArgs p) {
    __shared__ float red[8];
    grid_release();
    grid_wait();
    const int nt = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int i = WARP ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    long long src = i;
    const int * perm = p.plan + PLAN_HDR + 3 * (p.experts + 1) + 1;
    if (!SCATTER && p.plan) {
        if (i >= p.plan[PLAN_NGROUPED]) return;
        const int a = perm[i];
        if (a >= p.assignments && !p.shared) return;                   // a plan with a shared expert, a call without one
        src = !p.per_token ? a : a < p.assignments ? a / p.topk : a - p.assignments;
    } else if (i >= p.n) {
        return;
    }
    const size_t row = size_t(src) * p.ldx;
    const int pieces = p.k / 16;
    constexpr int H = C ? C : 1;
    Piece<DT> v[H];
    float top = 0.f;
    if (C) {
#pragma unroll
        for (int c = 0; c < H; ++c)
            if (c * nt + tid < pieces) v[c].load(p.x, row + size_t(c * nt + tid) * 16);
#pragma unroll
        for (int c = 0; c < H; ++c)
            if (c * nt + tid < pieces) top = max_nan(top, v[c].top());
    } else {
        for (int j = tid; j < pieces; j += nt) {
            v[0].load(p.x, row + size_t(j) * 16);
            top = max_nan(top, v[0].top());
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (!WARP && nt > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
        __syncthreads();
        top = red[0];
        for (int w = 1; w < nt / 32; ++w) top = max_nan(top, red[w]);
    }
    const bool fine = top < INFINITY;                                  // no infinity, no NaN
    const float scale = fine ? __fdiv_rn(top, 127.f) : __int_as_float(0x7fc00000);
    const Rule r = rule_of<DT>(top);
    auto round = [&](const Piece<DT> & w) {
        return !fine ? make_uint4(0, 0, 0, 0) : !r.check ? w.template quantized<false>(top, r.inv, 1.f) : DT == B2MOE_F32 ? w.template quantized<true>(top, r.inv, r.near) : exact_piece<DT>(w, top);
    };
    // place(f): f(row of q) for every place that the row goes to
    auto place = [&](auto f) {
        if (!SCATTER) return f(size_t(i));
        const int grouped = p.plan[PLAN_NGROUPED];
        for (int s = 0; s <= p.topk; ++s) {
            // an assignment that was skipped has no entry: whatever its word holds, the plan does not lead back from there
            const int a = s < p.topk ? i * p.topk + s : p.assignments + i, slot = s < p.topk || p.shared ? p.inverse[a] : -1;
            if (slot >= 0 && slot < grouped && perm[slot] == a) f(size_t(slot));
        }
    };
    if (tid == 0) place([&](size_t at) { p.scale[at] = scale; });
    if (C) {
        uint4 o[H];
#pragma unroll
        for (int c = 0; c < H; ++c)
            if (c * nt + tid < pieces) o[c] = round(v[c]);
        place([&](size_t at) {
#pragma unroll
            for (int c = 0; c < H; ++c)
                if (c * nt + tid < pieces) *reinterpret_cast<uint4 *>(p.q + at * p.ldq + size_t(c * nt + tid) * 16) = o[c];
        });
    } else {
        for (int j = tid; j < pieces; j += nt) {
            v[0].load(p.x, row + size_t(j) * 16);
            const uint4 o = round(v[0]);
            place([&](size_t at) { *reinterpret_cast<uint4 *>(p.q + at * p.ldq + size_t(j) * 16) = o; });
        }
    }
}

// Slot of every grouped assignment below `words`, what the array has room for: a plan with a shared expert holds assignments behind the routed ones, which a call without one
// has no words for
__global__ void __launch_bounds__(256) inverse_k(const int * plan, int experts, int words, int * inverse) {
    grid_release();
    grid_wait();
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= plan[PLAN_NGROUPED]) return;
    const int a = plan[PLAN_HDR + 3 * (experts + 1) + 1 + i];
    if (a < words) inverse[a] = i;
}

template <int DT, bool SCATTER>
void launch_quant(const QuantArgs & a, cudaStream_t s) {
    auto go = [&](auto kernel, int blocks, int threads) { launch_overlapped(kernel, dim3(blocks), dim3(threads), 0, s, a); };
    const int pieces = a.k / 16, by_warp = ceil_div(pieces, 32);
    // Many rows (they fill the SMs with 16 warps each): four pieces a thread, a warp a row where that does. 8192 x 4096 bf16 with 256 / 128 / 64 threads a row 28.6 / 22.2 / 18.5 us,
    // 40960 x 512 fp32 with a warp a block / eight warps of a row each 43.4 / 19.2. Rows that are written to several slots have more stores than loads and take the other shape (4096 x 2048 to ten slots
    // each 26 / 18)
    if constexpr (!SCATTER)
        if (a.n >= 148 * 16) {
            const int blocks = ceil_div(a.n, 8);
            if (by_warp == 1) return go(quant_rows_k<DT, 1, true, false>, blocks, 256);
            if (by_warp == 2) return go(quant_rows_k<DT, 2, true, false>, blocks, 256);
            if (by_warp <= 4) return go(quant_rows_k<DT, 4, true, false>, blocks, 256);
            if (by_warp <= 32) return go(quant_rows_k<DT, 4, false, false>, a.n, ceil_div(by_warp, 4) * 32);
        }
    // a few: as many threads as the row has pieces, up to 256
    const int threads = std::min(256, by_warp * 32), per = ceil_div(pieces, threads);
    if (per == 1) go(quant_rows_k<DT, 1, false, SCATTER>, a.n, threads);
    else if (per == 2) go(quant_rows_k<DT, 2, false, SCATTER>, a.n, threads);
    else if (per <= 4) go(quant_rows_k<DT, 4, false, SCATTER>, a.n, threads);
    else go(quant_rows_k<DT, 0, false, SCATTER>, a.n, threads);
}

}  // namespace

namespace {
template <bool SCATTER>
int32_t quantize(const QuantArgs & a, int x_dtype, cudaStream_t s) {
    if (x_dtype == B2MOE_F32) launch_quant<B2MOE_F32, SCATTER>(a, s);
    else if (x_dtype == B2MOE_F16) launch_quant<B2MOE_F16, SCATTER>(a, s);
    else launch_quant<B2MOE_BF16, SCATTER>(a, s);
    return launch_status();
}
}  // namespace

int32_t i8_quantize(const void * x, int x_dtype, long long ldx, int n, int k, int8_t * q, long long ldq, float * scale, cudaStream_t s) {
    return quantize<false>(QuantArgs{x, ldx, ldq, n, k, q, scale}, x_dtype, s);
}
int32_t i8_quantize_slots(const void * x, int x_dtype, bool per_token, int n, int k, const I8Rows & rows, const int * plan, int experts, int topk, int shared_tokens, cudaStream_t s) {
    const int A = n * topk;
    return quantize<false>(QuantArgs{x, k, k, A + shared_tokens, k, rows.q, rows.scale, plan, experts, A, topk, per_token, shared_tokens ? 1 : 0}, x_dtype, s);
}
int32_t i8_quantize_scatter(const void * x, int x_dtype, int n, int k, const I8Rows & rows, int * inverse, const int * plan, int experts, int topk, int shared_tokens, cudaStream_t s) {
    const int words = n * topk + shared_tokens;
    launch_overlapped(inverse_k, dim3(ceil_div(words, 256)), dim3(256), 0, s, plan, experts, words, inverse);
    if (int32_t rc = launch_status()) return rc;
    return quantize<true>(QuantArgs{x, k, k, n, k, rows.q, rows.scale, plan, experts, n * topk, topk, 1, shared_tokens ? 1 : 0, inverse}, x_dtype, s);
}

}  // namespace b2

using namespace b2;

extern "C" B2MOE_API int32_t b2moe_quantize_rows(const void * x, int32_t x_dtype, int64_t ldx, int32_t n, int32_t k, int8_t * q, int64_t ldq, float * scale,
                                                 b2moe_stream stream) {
    if (n <= 0 || n > I8_MAX_ROWS || !i8_cols(k) || !valid_dtype(x_dtype) || ldx < k || ldx % (x_dtype == B2MOE_F32 ? 4 : 8) || ldq < k || ldq % 16) return B2MOE_ERR_SHAPE;
    if (!x || !q || !scale) return B2MOE_ERR_NULL;
    if (!aligned16(x) || !aligned16(q) || !aligned_to(scale, 4)) return B2MOE_ERR_ALIGN;
    return i8_quantize(x, x_dtype, ldx, n, k, q, ldq, scale, as_stream(stream));
}
