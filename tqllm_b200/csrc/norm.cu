// Root-mean-square norm of rows with the skip connection's addition, out as rows of the input's type and as 8-bit integers with a scale a row; its gradient.
//
//   h = x + r (32 bits)      rho = 1 / sqrt(mean h^2 + eps)      y = h rho w
//   8 bits: u = h w, q = the integer nearest to 127 u / max|u|, scale = max|u| rho / 127: rho cancels in q, so maximum and squares come from one pass over registers
//   gradient: a = dy w, c = mean(a h);  dx = rho (a - h rho^2 c) + dsum;  dw = sum over rows of dy h rho
//
// One pass: the row stays in registers between its sums and its outputs. Bound by memory.
#include <algorithm>

#include "int8.cuh"

namespace b2 {
namespace {

constexpr int NORM_MAX_COLS = 16384;             // 512 threads of 32 values
constexpr int SMS = 148;

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// V neighbouring values as they lie in memory: 16 bytes where rows allow it (V > 1), else one. 16-bit values are unpacked where they are used and take half a register each until then
template <int DT, int V> struct Piece {
    using T = typename Elem<DT>::type;
    static constexpr int PER = 16 / int(sizeof(T)), WORDS = V > PER ? V / PER : 1;
    uint4 w[WORDS];
    __device__ __forceinline__ void load(const void * p, size_t i) {
        const uint4 * at = reinterpret_cast<const uint4 *>(static_cast<const T *>(p) + i);
#pragma unroll
        for (int j = 0; j < WORDS; ++j) w[j] = at[j];
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int j = 0; j < WORDS; ++j) w[j] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ uint32_t word(int j) const { return j % 4 == 0 ? w[j / 4].x : j % 4 == 1 ? w[j / 4].y : j % 4 == 2 ? w[j / 4].z : w[j / 4].w; }
    __device__ __forceinline__ float operator[](int i) const {
        if (DT == B2MOE_F32) return __uint_as_float(word(i));
        const uint32_t u = word(i / 2);
        if (DT == B2MOE_BF16) return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
        return __half2float(__ushort_as_half((unsigned short)(i & 1 ? u >> 16 : u & 0xffffu)));
    }
};
template <int DT> struct Piece<DT, 1> {
    float v;
    __device__ __forceinline__ void load(const void * p, size_t i) { v = load_act(p, DT, i); }
    __device__ __forceinline__ void zero() { v = 0.f; }
    __device__ __forceinline__ float operator[](int) const { return v; }
};
template <int DT, int V> __device__ __forceinline__ void store_piece(void * p, size_t i, const float (&v)[V]) {
    using T = typename Elem<DT>::type;
    T * at = static_cast<T *>(p) + i;
    if constexpr (V == 1) {
        store_act(at, DT, 0, v[0]);
    } else {
        constexpr int PER = 16 / int(sizeof(T));
#pragma unroll
        for (int j = 0; j < V / PER; ++j) {
            uint32_t u[4];
#pragma unroll
            for (int l = 0; l < 4; ++l) {
                if (DT == B2MOE_F32) {
                    u[l] = __float_as_uint(v[j * PER + l]);
                } else if (DT == B2MOE_BF16) {
                    const __nv_bfloat162 b = __floats2bfloat162_rn(v[j * PER + 2 * l], v[j * PER + 2 * l + 1]);
                    u[l] = *reinterpret_cast<const uint32_t *>(&b);
                } else {
                    const __half2 b = __floats2half2_rn(v[j * PER + 2 * l], v[j * PER + 2 * l + 1]);
                    u[l] = *reinterpret_cast<const uint32_t *>(&b);
                }
            }
            reinterpret_cast<uint4 *>(at)[j] = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
}

struct NormArgs {
    const void * x, * r, * w;
    long long ldx, ldr, lds, ldy, ldq;
    float eps;
    int n, k;
    void * sum, * y;
    int8_t * q;
    float * scale;
};

__device__ __forceinline__ float2 shuffled(float2 v, int d) { return make_float2(__shfl_xor_sync(0xffffffffu, v.x, d), __shfl_xor_sync(0xffffffffu, v.y, d)); }
template <class T> __device__ __forceinline__ T shuffled(T v, int d) { return __shfl_xor_sync(0xffffffffu, v, d); }
// sums and maxima over the threads of a row, the same bits in all of them: a warp's, or the block's (red: a word for each warp, which no reduction has used since the last barrier but one)
template <bool WARP, class T, class F>
__device__ __forceinline__ T over_row(T v, T none, T * red, F join) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = join(v, shuffled(v, d));
    if (WARP) return v;
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (warps == 1) return v;
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? red[lane] : none;
#pragma unroll
    for (int d = 16; d; d >>= 1) v = join(v, shuffled(v, d));
    return v;
}
struct Add { __device__ float operator()(float a, float b) const { return a + b; } };
struct Add2 { __device__ float2 operator()(float2 a, float2 b) const { return make_float2(a.x + b.x, a.y + b.y); } };
struct AddMax { __device__ float2 operator()(float2 a, float2 b) const { return make_float2(a.x + b.x, max_nan(a.y, b.y)); } };
struct Max { __device__ double operator()(double a, double b) const { return fmax(a, b); } };

// The integer nearest to 127 u / top for products u = h w that 64 bits hold exactly, halves to even, exactly: 127 u and (m + 1/2) top are compared through what rounding
// the latter leaves over
__device__ __noinline__ int nearest_product(float h, float w, double top) {
    const double u = double(h) * double(w), a = fabs(u), m = floor(127.0 * a / top), half = m + 0.5;
    const double p = half * top, over = fma(127.0, a, -p), rest = fma(half, top, -p);
    const int lo = int(m), q = over > rest ? lo + 1 : over < rest ? lo : lo + (lo & 1);
    return u < 0.0 ? -q : q;
}

// Squares that pass the range of 32 bits: the row is taken once more in this unit, in which they do not (16384 squares of 2^48 at most), nor does what is small count there
constexpr float UNIT = 0x1p-80f;

// P pieces of V values a thread; WARP: a warp a row, eight rows a block; otherwise the block takes a row. WDT: the weight's type; Q: 8-bit rows are wanted
template <int DT, int WDT, int V, int P, bool WARP, bool Q>
__global__ void __launch_bounds__(WARP ? 256 : 512) norm_k(const NormArgs p) {
    __shared__ float2 red[32], red_again[32];
    __shared__ double red_exact[32];
    grid_release();
    grid_wait();
    const int nt = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int row = WARP ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && row >= p.n) return;                                    // no barrier follows in this form
    float h[P][V];
    Piece<WDT, V> w[P];
    {
        Piece<DT, V> x[P], r[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = (i * nt + tid) * V;
            x[i].zero();
            r[i].zero();
            w[i].zero();
            if (j >= p.k) continue;
            x[i].load(p.x, size_t(row) * p.ldx + j);
            if (p.r) r[i].load(p.r, size_t(row) * p.ldr + j);
            w[i].load(p.w, j);
        }
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int l = 0; l < V; ++l) h[i][l] = p.r ? x[i][l] + r[i][l] : x[i][l];
    }
    auto sums = [&]() {                                                // squares, the largest product
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int l = 0; l < V; ++l) {
                v.x = fmaf(h[i][l], h[i][l], v.x);
                if (Q) v.y = max_nan(v.y, fabsf(h[i][l] * w[i][l]));
            }
        return v;
    };
    auto join = [&](float2 v, float2 * red) {
        if constexpr (Q) return over_row<WARP>(v, make_float2(0.f, 0.f), red, AddMax());
        else return make_float2(over_row<WARP>(v.x, 0.f, reinterpret_cast<float *>(red), Add()), 0.f);
    };
    float2 mine = sums();
    if (p.sum) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = (i * nt + tid) * V;
            if (j < p.k) store_piece<DT, V>(p.sum, size_t(row) * p.lds + j, h[i]);
        }
    }
    float2 all = join(mine, red);
    const bool fine = all.y < INFINITY;                                // no infinity, no NaN, no product beyond 32 bits
    float unit = 1.f;
    if (!(all.x < INFINITY)) {
        unit = UNIT;
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int l = 0; l < V; ++l) h[i][l] *= UNIT;
        mine = sums();
        all = join(mine, red_again);
    }
    const float rho = 1.f / sqrtf(all.x / float(p.k) + p.eps * unit * unit);
    if (p.y) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = (i * nt + tid) * V;
            if (j >= p.k) continue;
            float y[V];
#pragma unroll
            for (int l = 0; l < V; ++l) y[l] = h[i][l] * rho * w[i][l];
            store_piece<DT, V>(p.y, size_t(row) * p.ldy + j, y);
        }
    }
    if constexpr (Q) {
        const float top = all.y;
        // the largest product exactly: among those that round to the largest
        double exact = 0.0;
        if (mine.y == top) {
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int l = 0; l < V; ++l)
                    if (fabsf(h[i][l] * w[i][l]) == top) exact = fmax(exact, fabs(double(h[i][l]) * double(w[i][l])));
        }
        exact = over_row<WARP>(exact, 0.0, red_exact, Max());
        if (tid == 0) p.scale[row] = fine ? top * rho / 127.f : __int_as_float(0x7fc00000);
        const bool tiny = top < 0x1p-100f;                             // products have lost bits there
        const float inv = tiny || !fine ? 0.f : __fdiv_rn(127.f, top);
        // u, top and inv are off by 2^-24 each, their quotient by 127 times the sum: those that close to a half are done again
        const float near = !fine || top == 0.f ? 1.f : tiny ? -1.f : 0.5f - 5e-5f;
        constexpr float MAGIC = 12582912.f;                            // u * inv + 1.5 * 2^23: the nearest integer in the low bits
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = (i * nt + tid) * V;
            if (j >= p.k) continue;
            uint32_t b[V];
            float off = 0.f;
#pragma unroll
            for (int l = 0; l < V; ++l) {
                const float u = fine ? h[i][l] * w[i][l] : 0.f, f = __fmaf_rn(u, inv, MAGIC);
                b[l] = __float_as_uint(f);
                off = fmaxf(off, fabsf(__fmaf_rn(u, inv, MAGIC - f)));
            }
            if (off > near) {
#pragma unroll
                for (int l = 0; l < V; ++l) {
                    const float u = h[i][l] * w[i][l], f = __uint_as_float(b[l]);
                    if (fabsf(__fmaf_rn(u, inv, MAGIC - f)) > near) b[l] = uint32_t(nearest_product(h[i][l], w[i][l], exact));
                }
            }
            uint32_t o[V / 4];
#pragma unroll
            for (int l = 0; l < V / 4; ++l) o[l] = __byte_perm(__byte_perm(b[4 * l], b[4 * l + 1], 0x0040), __byte_perm(b[4 * l + 2], b[4 * l + 3], 0x0040), 0x5410);
            int8_t * at = p.q + size_t(row) * p.ldq + j;
            if constexpr (V == 8) *reinterpret_cast<uint2 *>(at) = make_uint2(o[0], o[1]);
            else *reinterpret_cast<uint32_t *>(at) = o[0];
        }
    }
}

template <int DT, int WDT, bool Q>
void launch_norm_wide(const NormArgs & a, cudaStream_t s) {
    constexpr int V = DT == B2MOE_F32 ? 4 : 8, MOST = NORM_MAX_COLS / V / 512;
    const int by_warp = ceil_div(a.k / V, 32);
    auto go = [&](auto kernel, int blocks, int threads) { launch_overlapped(kernel, dim3(blocks), dim3(threads), 0, s, a); };
    if (by_warp <= 4 && a.n >= SMS * 16) go(norm_k<DT, WDT, V, 4, true, Q>, ceil_div(a.n, 8), 256);
    else if (by_warp <= 16 && a.n < SMS * 16) go(norm_k<DT, WDT, V, 1, false, Q>, a.n, by_warp * 32);
    else if (by_warp <= 64) go(norm_k<DT, WDT, V, 4, false, Q>, a.n, ceil_div(by_warp, 4) * 32);
    else go(norm_k<DT, WDT, V, MOST, false, Q>, a.n, ceil_div(by_warp, MOST) * 32);
}
template <int DT, int WDT>
int32_t launch_norm(const NormArgs & a, bool wide, cudaStream_t s) {
    if (wide && a.q) launch_norm_wide<DT, WDT, true>(a, s);
    else if (wide) launch_norm_wide<DT, WDT, false>(a, s);
    else if (a.k <= 2048) launch_overlapped(norm_k<DT, WDT, 1, 4, false, false>, dim3(a.n), dim3(ceil_div(a.k, 128) * 32), 0, s, a);
    else launch_overlapped(norm_k<DT, WDT, 1, 32, false, false>, dim3(a.n), dim3(ceil_div(a.k, 1024) * 32), 0, s, a);
    return launch_status();
}

struct NormGradArgs {
    const void * h, * w, * dy, * ds;
    long long ldh, ldy, lds, ldx;
    float eps;
    int n, k;
    void * dx;
    float * parts;                     // [blocks][k]: each block's sums for the weight's gradient (null: not wanted)
};

template <int DT, int WDT, int V, int P>
__global__ void __launch_bounds__(512) norm_grad_k(const NormGradArgs p) {
    __shared__ float2 red[2][32], red_again[2][32];
    grid_release();
    grid_wait();
    const int nt = blockDim.x, tid = threadIdx.x;
    Piece<WDT, V> w[P];
    float dw[P][V];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int j = (i * nt + tid) * V;
        w[i].zero();
        if (j < p.k) w[i].load(p.w, j);
#pragma unroll
        for (int l = 0; l < V; ++l) dw[i][l] = 0.f;
    }
    int turn = 0;                                                      // two sets of words in turn: one barrier a row
    for (int row = blockIdx.x; row < p.n; row += gridDim.x, turn ^= 1) {
        Piece<DT, V> h[P], g[P], s[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = (i * nt + tid) * V;
            h[i].zero();
            g[i].zero();
            s[i].zero();
            if (j >= p.k) continue;
            h[i].load(p.h, size_t(row) * p.ldh + j);
            g[i].load(p.dy, size_t(row) * p.ldy + j);
            if (p.ds) s[i].load(p.ds, size_t(row) * p.lds + j);
        }
        float unit = 1.f;
        auto sums = [&]() {
            float2 v = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int l = 0; l < V; ++l) {
                    const float f = h[i][l] * unit;
                    v.x = fmaf(f, f, v.x);
                    v.y = fmaf(g[i][l] * w[i][l], f, v.y);
                }
            return v;
        };
        float2 v = over_row<false>(sums(), make_float2(0.f, 0.f), red[turn], Add2());
        if (!(v.x < INFINITY)) {
            unit = UNIT;
            v = over_row<false>(sums(), make_float2(0.f, 0.f), red_again[turn], Add2());
        }
        // in the unit: rho h as it is, rho the unit times as large
        const float m = v.x / float(p.k) + p.eps * unit * unit, rho = 1.f / sqrtf(m), t = v.y / float(p.k) / m, out = rho * unit;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = (i * nt + tid) * V;
            if (j >= p.k) continue;
            float d[V];
#pragma unroll
            for (int l = 0; l < V; ++l) {
                const float f = h[i][l] * unit;
                d[l] = fmaf(out, fmaf(-f, t, g[i][l] * w[i][l]), s[i][l]);
                dw[i][l] = fmaf(g[i][l], f * rho, dw[i][l]);
            }
            store_piece<DT, V>(p.dx, size_t(row) * p.ldx + j, d);
        }
    }
    if (p.parts) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = (i * nt + tid) * V;
            if (j >= p.k) continue;
#pragma unroll
            for (int l = 0; l < V; ++l) p.parts[size_t(blockIdx.x) * p.k + j + l] = dw[i][l];
        }
    }
}

// dw[j] = (accumulate: +) the sum over the blocks' parts, in a fixed order: 32 columns a block, eight threads a column
__global__ void __launch_bounds__(256) norm_weight_grad_k(const float * parts, int blocks, int k, float * dw, int accumulate) {
    __shared__ float part[8][32];
    grid_release();
    grid_wait();
    const int j = blockIdx.x * 32 + (threadIdx.x & 31), y = threadIdx.x >> 5;
    float s = 0.f;
    if (j < k)
#pragma unroll 8
        for (int b = y; b < blocks; b += 8) s += parts[size_t(b) * k + j];
    part[y][threadIdx.x & 31] = s;
    __syncthreads();
    if (y || j >= k) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
    dw[j] = accumulate ? dw[j] + s : s;
}

int grad_blocks(int n, int k) { return std::min(n, SMS * std::max(1, std::min(16, 8192 / k))); }

template <int DT, int WDT>
void launch_norm_grad(const NormGradArgs & a, bool wide, cudaStream_t s) {
    constexpr int V = DT == B2MOE_F32 ? 4 : 8, MOST = NORM_MAX_COLS / V / 512;
    auto go = [&](auto kernel, int threads) { launch_overlapped(kernel, dim3(a.parts ? grad_blocks(a.n, a.k) : a.n), dim3(threads), 0, s, a); };
    if (!wide) return a.k <= 2048 ? go(norm_grad_k<DT, WDT, 1, 4>, ceil_div(a.k, 128) * 32) : go(norm_grad_k<DT, WDT, 1, 32>, ceil_div(a.k, 1024) * 32);
    const int by_warp = ceil_div(a.k / V, 32);
    if (by_warp <= 8) go(norm_grad_k<DT, WDT, V, 1>, by_warp * 32);
    else if (by_warp <= 32) go(norm_grad_k<DT, WDT, V, 2>, ceil_div(by_warp, 2) * 32);
    else go(norm_grad_k<DT, WDT, V, MOST>, ceil_div(by_warp, MOST) * 32);
}

// rows of 16-byte pieces: the columns, every row's first value and the strides
struct Rows { const void * p; long long ld; int dtype; };
bool in_pieces(int k, std::initializer_list<Rows> rows) {
    for (const Rows & r : rows) {
        const int per = 16 / int(dtype_bytes(r.dtype));
        if (r.p && (k % per || r.ld % per || !aligned16(r.p))) return false;
    }
    return true;
}
bool weight_type(int dtype, int weight_dtype) { return weight_dtype == B2MOE_F32 || weight_dtype == dtype; }

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" B2MOE_API int32_t b2moe_rms_norm(const void * x, int32_t dtype, int64_t ldx, const void * residual, int64_t ldr, const void * weight, int32_t weight_dtype, float eps, int32_t n,
                                            int32_t k, void * sum, int64_t lds, void * y, int64_t ldy, int8_t * q, int64_t ldq, float * scale, b2moe_stream stream) {
    if (n <= 0 || n > I8_MAX_ROWS || k <= 0 || k > NORM_MAX_COLS || !valid_dtype(dtype) || !weight_type(dtype, weight_dtype) || !(eps >= 0.f) || !(eps < INFINITY)) return B2MOE_ERR_SHAPE;
    if (ldx < k || (residual && ldr < k) || (sum && lds < k) || (y && ldy < k) || (q && (k % 16 || ldq < k || ldq % 16))) return B2MOE_ERR_SHAPE;
    if (!x || !weight || (!y && !q) || (q && !scale) || (sum && !residual)) return B2MOE_ERR_NULL;
    const size_t e = dtype_bytes(dtype);
    if (!aligned_to(x, e) || !aligned_to(residual, e) || !aligned_to(sum, e) || !aligned_to(y, e) || !aligned_to(weight, dtype_bytes(weight_dtype)) || !aligned16(q) || !aligned_to(scale, 4)) return B2MOE_ERR_ALIGN;
    const bool wide = in_pieces(k, {{x, ldx, dtype}, {residual, ldr, dtype}, {sum, lds, dtype}, {y, ldy, dtype}, {weight, 0, weight_dtype}});
    if (q && !wide) return B2MOE_ERR_ALIGN;                            // rows in 8 bits come from rows in pieces of 16 bytes
    const NormArgs a{x, residual, weight, ldx, ldr, lds, ldy, ldq, eps, n, k, sum, y, q, scale};
    cudaStream_t s = as_stream(stream);
    if (dtype == B2MOE_F32) return launch_norm<B2MOE_F32, B2MOE_F32>(a, wide, s);
    if (dtype == B2MOE_F16) return weight_dtype == B2MOE_F32 ? launch_norm<B2MOE_F16, B2MOE_F32>(a, wide, s) : launch_norm<B2MOE_F16, B2MOE_F16>(a, wide, s);
    return weight_dtype == B2MOE_F32 ? launch_norm<B2MOE_BF16, B2MOE_F32>(a, wide, s) : launch_norm<B2MOE_BF16, B2MOE_BF16>(a, wide, s);
}

extern "C" B2MOE_API size_t b2moe_rms_norm_backward_workspace_bytes(int32_t n, int32_t k) {
    if (n <= 0 || n > I8_MAX_ROWS || k <= 0 || k > NORM_MAX_COLS) return 0;
    return align_up(size_t(grad_blocks(n, k)) * k * sizeof(float), 16);
}

extern "C" B2MOE_API int32_t b2moe_rms_norm_backward(const void * h, int32_t dtype, int64_t ldh, const void * weight, int32_t weight_dtype, const void * grad_y, int64_t ldgy,
                                                     const void * grad_sum, int64_t ldgs, float eps, int32_t n, int32_t k, void * grad_x, int64_t ldgx, float * grad_weight,
                                                     int32_t accumulate, void * workspace, size_t workspace_bytes, b2moe_stream stream) {
    if (n <= 0 || n > I8_MAX_ROWS || k <= 0 || k > NORM_MAX_COLS || !valid_dtype(dtype) || !weight_type(dtype, weight_dtype) || !(eps >= 0.f) || !(eps < INFINITY)) return B2MOE_ERR_SHAPE;
    if (ldh < k || ldgy < k || ldgx < k || (grad_sum && ldgs < k)) return B2MOE_ERR_SHAPE;
    if (!h || !weight || !grad_y || !grad_x || (grad_weight && !workspace)) return B2MOE_ERR_NULL;
    const size_t e = dtype_bytes(dtype);
    if (!aligned_to(h, e) || !aligned_to(grad_y, e) || !aligned_to(grad_sum, e) || !aligned_to(grad_x, e) || !aligned_to(weight, dtype_bytes(weight_dtype)) || !aligned_to(grad_weight, 4) ||
        (grad_weight && !aligned16(workspace))) return B2MOE_ERR_ALIGN;
    if (grad_weight && workspace_bytes < b2moe_rms_norm_backward_workspace_bytes(n, k)) return B2MOE_ERR_WORKSPACE;
    const bool wide = in_pieces(k, {{h, ldh, dtype}, {grad_y, ldgy, dtype}, {grad_sum, ldgs, dtype}, {grad_x, ldgx, dtype}, {weight, 0, weight_dtype}});
    const NormGradArgs a{h, weight, grad_y, grad_sum, ldh, ldgy, ldgs, ldgx, eps, n, k, grad_x, grad_weight ? static_cast<float *>(workspace) : nullptr};
    cudaStream_t s = as_stream(stream);
    if (dtype == B2MOE_F32) launch_norm_grad<B2MOE_F32, B2MOE_F32>(a, wide, s);
    else if (dtype == B2MOE_F16 && weight_dtype == B2MOE_F32) launch_norm_grad<B2MOE_F16, B2MOE_F32>(a, wide, s);
    else if (dtype == B2MOE_F16) launch_norm_grad<B2MOE_F16, B2MOE_F16>(a, wide, s);
    else if (weight_dtype == B2MOE_F32) launch_norm_grad<B2MOE_BF16, B2MOE_F32>(a, wide, s);
    else launch_norm_grad<B2MOE_BF16, B2MOE_BF16>(a, wide, s);
    if (int32_t rc = launch_status()) return rc;
    if (!grad_weight) return B2MOE_OK;
    launch_overlapped(norm_weight_grad_k, dim3(ceil_div(k, 32)), dim3(256), 0, s, static_cast<const float *>(workspace), grad_blocks(n, k), k, grad_weight, accumulate);
    return launch_status();
}
