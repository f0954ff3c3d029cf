// Root-mean-square norm of rows with the skip connection's addition, out as rows of the input's type and as 8-bit integers with a scale a row; its gradient.
//
//   h = x + r (32 bits)      rho = 1 / sqrt(mean h^2 + eps)      y = h rho w
//   8 bits: u = h w, q = the integer nearest to 127 u / max|u|, scale = max|u| rho / 127: rho cancels in q, so maximum and squares come from one pass over registers
//   gradient: a = dy w, c = mean(a h);  dx = rho (a - h rho^2 c) + dsum;  dw = sum over rows of dy h rho
//
// One pass: the row stays in registers between its sums and its outputs. Bound by memory.
#include <algorithm>
#include <type_traits>

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
__device__ __forceinline__ float largest(float a, Two b) {             // of three magnitudes; a NaN where there is one
    const float2 f = apart(b);
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(f.x)), "f"(fabsf(f.y)));
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
    __device__ __forceinline__ uint32_t & word(int j) { return j % 4 == 0 ? w[j / 4].x : j % 4 == 1 ? w[j / 4].y : j % 4 == 2 ? w[j / 4].z : w[j / 4].w; }
    __device__ __forceinline__ uint32_t word(int j) const { return j % 4 == 0 ? w[j / 4].x : j % 4 == 1 ? w[j / 4].y : j % 4 == 2 ? w[j / 4].z : w[j / 4].w; }
    // those of the values i .. i + V - 1 of a row that lie in [0, k), one by one; the piece is zero before
    __device__ __forceinline__ void load_some(const void * row, int i, int k) {
#pragma unroll
        for (int l = 0; l < V; ++l)
            if (unsigned(i + l) < unsigned(k)) {
                if constexpr (DT == B2MOE_F32) word(l) = static_cast<const uint32_t *>(row)[i + l];
                else word(l / 2) |= uint32_t(static_cast<const uint16_t *>(row)[i + l]) << (16 * (l & 1));
            }
    }
    // values outside of [0, k) become zero
    __device__ __forceinline__ void trim(int i, int k) {
#pragma unroll
        for (int l = 0; l < V; ++l)
            if (unsigned(i + l) >= unsigned(k)) {
                if constexpr (DT == B2MOE_F32) word(l) = 0u;
                else word(l / 2) &= l & 1 ? 0x0000ffffu : 0xffff0000u;
            }
    }
    __device__ __forceinline__ Two pair(int l) const { return two((*this)[2 * l], (*this)[2 * l + 1]); }
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
    __device__ __forceinline__ void load_some(const void * row, int i, int k) { if (unsigned(i) < unsigned(k)) load(row, i); }
    __device__ __forceinline__ void zero() { v = 0.f; }
    __device__ __forceinline__ float operator[](int) const { return v; }
    __device__ __forceinline__ Two pair(int) const { return two(v, 0.f); }
};
template <int DT, int V> __device__ __forceinline__ void store_some(void * row, int i, int k, const float (&v)[V]) {
#pragma unroll
    for (int l = 0; l < V; ++l)
        if (unsigned(i + l) < unsigned(k)) store_act(row, DT, size_t(i + l), v[l]);
}
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

// The pieces of a row. As it is: piece c holds the values from c V on, every row begins on 16 bytes and ends with a whole piece. SHIFT: rows begin `phase` values behind 16 bytes, in all matrices alike (odd k, a
// view of a wider matrix): piece c holds the values from c V - phase on, the first and the last are not whole and go value by value
template <int V, bool SHIFT> struct Grid {
    int k, phase;
    __device__ __forceinline__ int first(int c) const { return c * V - (SHIFT ? phase : 0); }
    __device__ __forceinline__ bool any(int j) const { return j < k && (!SHIFT || j + V > 0); }
    __device__ __forceinline__ bool whole(int j) const { return !SHIFT || (j >= 0 && j + V <= k); }
    __device__ __forceinline__ int some_whole() const { const int j = phase ? V - phase : 0; return j + V <= k ? j : -1; }      // where there is one
};
template <int V> __device__ __forceinline__ int phase_of(const void * row, int size) { return V == 1 ? 0 : int(reinterpret_cast<uintptr_t>(row) / size % V); }
template <int DT, int V, bool SHIFT>
__device__ __forceinline__ void put(void * base, size_t row, int j, const Grid<V, SHIFT> & grid, const float (&v)[V]) {
    void * at = static_cast<typename Elem<DT>::type *>(base) + row;
    if (grid.whole(j)) store_piece<DT, V>(at, j, v);
    else store_some<DT, V>(at, j, grid.k, v);
}
template <int DT, int V, bool SHIFT>
__device__ __forceinline__ void put(void * base, size_t row, int j, const Grid<V, SHIFT> & grid, const Two (&v)[(V + 1) / 2]) {
    float f[V];
#pragma unroll
    for (int l = 0; l < V; ++l) f[l] = l & 1 ? apart(v[l / 2]).y : apart(v[l / 2]).x;
    put<DT>(base, row, j, grid, f);
}
// the norm's weight begins on 16 bytes where the rows do, and is read value by value where they do not
template <int WDT, int V, bool SHIFT>
__device__ __forceinline__ void get_weight(Piece<WDT, V> & w, const void * base, int j, const Grid<V, SHIFT> & grid) {
    if (SHIFT) w.load_some(base, j, grid.k);
    else w.load(base, j);
}

struct NormArgs {
    const void * x, * r, * w;
    long long ldx, ldr, lds, ldy, ldq;
    float eps, inv_k;
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
    if (warps <= 4) {
        v = red[0];
        for (int i = 1; i < warps; ++i) v = join(v, red[i]);
        return v;
    }
    v = lane < warps ? red[lane] : none;
#pragma unroll
    for (int d = 16; d; d >>= 1) v = join(v, shuffled(v, d));
    return v;
}
struct Add { __device__ float operator()(float a, float b) const { return a + b; } };
struct Max { __device__ float operator()(float a, float b) const { return fmaxf(a, b); } };
struct Max2 { __device__ float2 operator()(float2 a, float2 b) const { return make_float2(fmaxf(a.x, b.x), fmaxf(a.y, b.y)); } };
struct Add2 { __device__ float2 operator()(float2 a, float2 b) const { return make_float2(a.x + b.x, a.y + b.y); } };
struct AddMax { __device__ float2 operator()(float2 a, float2 b) const { return make_float2(a.x + b.x, max_nan(a.y, b.y)); } };

// The integer nearest to 127 u / top for a product u = h w, which 64 bits hold exactly, halves to even, where it is `low` or the next: 127 |u| and (low + 1/2) top are compared through what rounding the
// latter leaves over
__device__ __forceinline__ int decide(float h, float w, double low, double top) {
    const double u = double(h) * double(w), half = low + 0.5, p = half * top, diff = fma(127.0, fabs(u), -p) - fma(half, top, -p);
    const int lo = int(low), q = diff > 0.0 ? lo + 1 : diff < 0.0 ? lo : lo + (lo & 1);
    return u < 0.0 ? -q : q;
}

// 1 / sqrt(v): the approximation and a step of Newton's, off by 1.5 steps of 2^-24. (Root and reciprocal by their own rounded instructions, done by every thread of a row: 8192 x 4096 to 8 bits 35.3 us instead of 34.6)
__device__ __forceinline__ float inverse_root(float v) {
    float r;
    asm("rsqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
    const float half = fmaf(-v * r, r, 1.f) * 0.5f;
    return v > 0x1p-126f && v < INFINITY ? fmaf(r, half, r) : r;       // 0, infinities and NaN as they come
}

constexpr float MAGIC = 12582912.f, OFF = 3.2f * 0x1p-24f;
__device__ __forceinline__ bool near_half(float u, float inv) {
    const float m = MAGIC - __fmaf_rn(u, inv, MAGIC);
    return fmaf(fabsf(m), OFF, fabsf(__fmaf_rn(u, inv, m))) > 0.5f - OFF;
}
// Rows whose mean square (with eps) lies outside of this range: squares have passed 32 bits, or lost bits below their normal numbers. They are taken once more in a unit of their own
constexpr float LEAST = 0x1p-64f;
__device__ __forceinline__ int exponent_of(float power) { return int(__float_as_uint(power) >> 23) - 127; }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }
__device__ __forceinline__ bool ordinary(float m) { return m >= LEAST && m < INFINITY; }
// A power of two that brings a row's largest value to 2^48: 16384 squares stay inside of 32 bits, and only what is 2^-111 of the largest square loses bits. 2^90 at most (values below the normal numbers become
// 2^-59 at least), and at most what takes eps to 2^100, beside which smaller squares do not count
__device__ __forceinline__ float unit_of(float largest, float eps) {
    return power_of_two(min(min(90, 175 - int(__float_as_uint(largest) >> 23)), (100 - exponent_of(eps)) / 2));
}

// P pieces of V values a thread, in pairs (V = 1: a value and a zero); WARP: a warp a row, eight rows a block; otherwise the block, of MOST threads at most, takes a row. WDT: the weight's type; Q: 8-bit
// rows are wanted. Registers are held to what this many blocks of an SM have: left alone, the second look at rows that are not ordinary takes up to 38 more than the rest needs (8192 x 256 bf16: 4.4 us
// instead of 3.5, 512 x 4096 2.9 instead of 2.6)
template <int DT, int WDT, int V, int P, bool WARP, bool Q, bool SHIFT, int MOST>
constexpr int norm_blocks() {
    constexpr bool narrow = V == 8 && WDT == DT && !Q;
    if (SHIFT) return P == 1 ? 10 : 1;
    if (WARP) return narrow ? 3 : 2;
    if (V > 1 && MOST == 128) return Q ? 5 : 6;
    return P == 1 && narrow ? 4 : 1;
}
template <int DT, int WDT, int V, int P, bool WARP, bool Q, bool SHIFT, int MOST>
__global__ void __launch_bounds__(MOST, norm_blocks<DT, WDT, V, P, WARP, Q, SHIFT, MOST>()) norm_k(const NormArgs p) {
    __shared__ float2 red[SHIFT ? 2 : 1][32];
    __shared__ float red_again[32];
    __shared__ unsigned long long exact_top[WARP ? 8 : 1];
    grid_release();
    grid_wait();
    const int nt = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    unsigned long long * const exact = exact_top + (WARP ? threadIdx.x >> 5 : 0);
    if (Q && tid == 0) *exact = 0;
    const int row0 = WARP ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if ((WARP || SHIFT) && row0 >= p.n) return;                        // no barrier follows, or none for the whole block
    using T = typename Elem<DT>::type;
    constexpr int H = (V + 1) / 2;
    const Grid<V, SHIFT> grid{p.k, SHIFT ? phase_of<V>(static_cast<const T *>(p.x) + size_t(row0) * p.ldx, sizeof(T)) : 0};
    Piece<WDT, V> w[P];
    if (SHIFT)
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = grid.first(i * nt + tid);
            w[i].zero();
            if (grid.any(j)) get_weight(w[i], p.w, j, grid);
        }
    // SHIFT: the block walks rows, a multiple of V apart, so that their phase stays and its weights, which come value by value, are read once
    int turn = 0;
#pragma unroll 1
    for (int row = row0; row < p.n; row += SHIFT ? int(gridDim.x) : p.n, turn ^= SHIFT) {
        const size_t x0 = size_t(row) * p.ldx;
        Two h[P][H];
        {
            Piece<DT, V> x[P], r[P];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int j = grid.first(i * nt + tid);
                x[i].zero();
                r[i].zero();
                if (!SHIFT) w[i].zero();
                if (!grid.any(j)) continue;
                const int from = grid.whole(j) ? j : grid.some_whole();
                if (SHIFT && from < 0) continue;
                x[i].load(p.x, x0 + from);
                if (p.r) r[i].load(p.r, size_t(row) * p.ldr + from);
                if (!SHIFT) get_weight(w[i], p.w, j, grid);
            }
            // pieces that are not whole have asked for another one (a branch around each load would wait for it), and come now
            if (SHIFT)
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int j = grid.first(i * nt + tid);
                    if (!grid.any(j) || grid.whole(j)) continue;
                    x[i].zero();
                    x[i].load_some(static_cast<const T *>(p.x) + x0, j, p.k);
                    if (!p.r) continue;
                    r[i].zero();
                    r[i].load_some(static_cast<const T *>(p.r) + size_t(row) * p.ldr, j, p.k);
                }
            if (p.r) {
#pragma unroll
                for (int i = 0; i < P; ++i)
#pragma unroll
                    for (int l = 0; l < H; ++l) h[i][l] = x[i].pair(l) + r[i].pair(l);
            } else {
#pragma unroll
                for (int i = 0; i < P; ++i)
#pragma unroll
                    for (int l = 0; l < H; ++l) h[i][l] = x[i].pair(l);
            }
        }
        float tops[Q ? P : 1];                                             // of the pieces
        Two squares = two(0.f);
        float2 mine = make_float2(0.f, 0.f);                               // squares, the largest product
#pragma unroll
        for (int i = 0; i < P; ++i) {
            if (Q) tops[i] = 0.f;
#pragma unroll
            for (int l = 0; l < H; ++l) {
                squares = fma2(h[i][l], h[i][l], squares);
                if (Q) tops[i] = largest(tops[i], h[i][l] * w[i].pair(l));
            }
            if (Q) mine.y = max_nan(mine.y, tops[i]);
        }
        mine.x = apart(squares).x + apart(squares).y;
        if (p.sum) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int j = grid.first(i * nt + tid);
                if (grid.any(j)) put<DT>(p.sum, size_t(row) * p.lds, j, grid, h[i]);
            }
        }
        float2 all;
        if constexpr (Q) all = over_row<WARP>(mine, make_float2(0.f, 0.f), red[turn], AddMax());
        else all = make_float2(over_row<WARP>(mine.x, 0.f, reinterpret_cast<float *>(red[turn]), Add()), 0.f);
        const bool fine = all.y < INFINITY;                                // no infinity, no NaN, no product beyond 32 bits
        float unit = 1.f, m = fmaf(all.x, p.inv_k, p.eps);
        if (!ordinary(m)) {
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int l = 0; l < H; ++l) most = fmaxf(most, fmaxf(fabsf(apart(h[i][l]).x), fabsf(apart(h[i][l]).y)));
            unit = unit_of(over_row<WARP>(most, 0.f, red_again, Max()), p.eps);
            squares = two(0.f);
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int l = 0; l < H; ++l) {
                    const Two f = h[i][l] * two(unit);
                    squares = fma2(f, f, squares);
                    if (!Q) h[i][l] = f;                                   // with 8-bit rows the products stay those of the values as they came
                }
            if (!WARP) __syncthreads();                                    // the maxima have been read
            m = fmaf(over_row<WARP>(apart(squares).x + apart(squares).y, 0.f, red_again, Add()), p.inv_k, p.eps * unit * unit);
        }
        const float rho = inverse_root(m);                                 // in the unit
        if (p.y) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int j = grid.first(i * nt + tid);
                if (!grid.any(j)) continue;
                Two y[H];
#pragma unroll
                for (int l = 0; l < H; ++l) y[l] = (Q ? h[i][l] * two(unit) : h[i][l]) * two(rho) * w[i].pair(l);
                put<DT>(p.y, size_t(row) * p.ldy, j, grid, y);
            }
        }
        if constexpr (Q) {
            // the products are worked out again below: kept since the sums they would take 32 registers (and spill)
#pragma unroll
            for (int i = 0; i < P; ++i)
#pragma unroll
                for (int l = 0; l < H; ++l) asm("" : "+l"(h[i][l].v));
            const float top = all.y;
            if (tid == 0) p.scale[row] = !fine ? __int_as_float(0x7fc00000) : !(top > 0.f) ? 0.f : unit == 1.f ? top * rho / 127.f : float(double(top) * rho * unit / 127.0);
            if (WARP || blockDim.x == 32) __syncwarp();
            // the largest product exactly, from the pieces of those that round to the largest (numbers above zero are ordered as their bits are)
            if (mine.y == top && top > 0.f) {
                double most = 0.0;
#pragma unroll
                for (int i = 0; i < P; ++i)
                    if (tops[i] == top)
#pragma unroll
                        for (int l = 0; l < V; ++l) {
                            const float hl = l & 1 ? apart(h[i][l / 2]).y : apart(h[i][l / 2]).x;
                            if (fabsf(hl * w[i][l]) == top) most = fmax(most, fabs(double(hl) * double(w[i][l])));
                        }
                atomicMax(exact, (unsigned long long)__double_as_longlong(most));
            }
            const bool tiny = top < 0x1p-100f;                             // products have lost bits there, or all of theirs
            const float inv = tiny || !fine ? 0.f : __fdiv_rn(127.f, top);
            // (OFF) u, top and inv are off by 2^-24 of themselves each, the quotient t by 3 |t| 2^-24: those that close to a half are done again, exactly. The nearest integer m comes from t + 1.5 * 2^23;
            // |t| <= |m| + 1/2. A piece is looked at by its largest m and its largest distance from an integer (one row of 4096 in fifteen has such a piece)
            uint32_t some = 0;                                             // pieces with such a value
            int8_t * const q = p.q + size_t(row) * p.ldq;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                uint32_t b[V], o[V / 4];
                float far = 0.f, big = 0.f;
#pragma unroll
                for (int l = 0; l < H; ++l) {
                    const Two u = h[i][l] * w[i].pair(l), f = fma2(u, two(inv), two(MAGIC)), m = fma2(f, two(-1.f), two(MAGIC));
                    const float2 g = apart(f);
                    b[2 * l] = __float_as_uint(g.x);
                    b[2 * l + 1] = __float_as_uint(g.y);
                    big = largest(big, m);
                    far = largest(far, fma2(u, two(inv), m));
                }
#pragma unroll
                for (int l = 0; l < V / 4; ++l) o[l] = fine ? __byte_perm(__byte_perm(b[4 * l], b[4 * l + 1], 0x0040), __byte_perm(b[4 * l + 2], b[4 * l + 3], 0x0040), 0x5410) : 0u;
                const int j = grid.first(i * nt + tid);
                if (j >= p.k) continue;
                if constexpr (V == 8) *reinterpret_cast<uint2 *>(q + j) = make_uint2(o[0], o[1]);
                else *reinterpret_cast<uint32_t *>(q + j) = o[0];
                if (fmaf(big, OFF, far) > 0.5f - OFF) some |= 1u << i;
            }
            if (WARP || blockDim.x == 32) __syncwarp();
            else __syncthreads();                                          // the exact top is there
            if (tiny) {
                // all products exactly, then the largest, the scale and every integer from it
                double most = 0.0;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    unsigned long long bits = 0;
#pragma unroll
                    for (int l = 0; l < H; ++l) bits |= h[i][l].v;
                    if (bits & 0x7fffffff7fffffffull)                      // rows of zeros have nothing to work out
#pragma unroll
                        for (int l = 0; l < V; ++l) most = fmax(most, fabs(double(l & 1 ? apart(h[i][l / 2]).y : apart(h[i][l / 2]).x) * double(w[i][l])));
                }
                if (most > 0.0) atomicMax(exact, (unsigned long long)__double_as_longlong(most));
                if (WARP || blockDim.x == 32) __syncwarp();
                else __syncthreads();
                most = __longlong_as_double((long long)*exact);
                if (most == 0.0) return;
                if (tid == 0) p.scale[row] = float(most * rho * unit / 127.0);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const int j = grid.first(i * nt + tid);
                    if (j < p.k)
#pragma unroll
                        for (int l = 0; l < V; ++l) {
                            const float hl = l & 1 ? apart(h[i][l / 2]).y : apart(h[i][l / 2]).x;
                            q[j + l] = int8_t(decide(hl, w[i][l], floor(127.0 * fabs(double(hl) * double(w[i][l])) / most), most));
                        }
                }
                return;
            }
            if (!some || !fine) return;
            const double largest_product = __longlong_as_double((long long)*exact);
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (some >> i & 1u)
#pragma unroll
                    for (int l = 0; l < V; ++l) {
                        const float hl = l & 1 ? apart(h[i][l / 2]).y : apart(h[i][l / 2]).x, u = hl * w[i][l];
                        if (near_half(u, inv)) q[grid.first(i * nt + tid) + l] = int8_t(decide(hl, w[i][l], double(floorf(fabsf(u * inv))), largest_product));
                    }
        }
    }
}

// how the rows of a call lie
enum Form { WHOLE, SHIFTED, SINGLE };            // whole pieces of 16 bytes; pieces behind a phase that all matrices share; value by value

// us, a warp a row / a piece a thread / 128 threads (bf16): 1024 x 256 1.8 / 1.6 / 1.8, 2368 x 256 1.8 / 2.8 / 2.8, 2368 x 1024 2.6 / 3.4 / 2.8, 8192 x 256 3.5 / 8.9 / 9.1, 8192 x 1024 5.0 / 9.0 / 9.0, 512 x 4096 - / 2.5 / 2.8,
// 2368 x 4096 - / 7.5 / 6.0, 8192 x 4096 - / 30.0 / 24.3; to 8 bits 1024 x 1024 4.0 / 3.2 / 4.3, 8192 x 1024 11.3 / 12.9 / 11.4, 512 x 4096 - / 4.8 / 4.4, 2368 x 4096 - / 16.5 / 11.3, 512 x 2048 fp32 - / 4.0 / 3.0
template <int DT, int WDT, bool Q>
void launch_norm_whole(const NormArgs & a, cudaStream_t s) {
    constexpr int V = DT == B2MOE_F32 ? 4 : 8, MOST = NORM_MAX_COLS / V / 512;
    const int by_warp = ceil_div(a.k / V, 32);
    auto go = [&](auto kernel, int blocks, int threads) { launch_overlapped(kernel, dim3(blocks), dim3(threads), 0, s, a); };
    if (by_warp <= 4 && a.n >= SMS * 16) go(norm_k<DT, WDT, V, 4, true, Q, false, 256>, ceil_div(a.n, 8), 256);
    else if (by_warp <= 16 && a.n < SMS * 16) go(norm_k<DT, WDT, V, 1, false, Q, false, 512>, a.n, by_warp * 32);
    else if (by_warp <= 16) go(norm_k<DT, WDT, V, 4, false, Q, false, 128>, a.n, ceil_div(by_warp, 4) * 32);
    else go(norm_k<DT, WDT, V, MOST, false, Q, false, 512>, a.n, ceil_div(by_warp, MOST) * 32);
}
template <int DT, int WDT>
int32_t launch_norm(const NormArgs & a, Form form, cudaStream_t s) {
    constexpr int V = DT == B2MOE_F32 ? 4 : 8, MOST = NORM_MAX_COLS / V / 512;
    auto go = [&](auto kernel, int threads) { launch_overlapped(kernel, dim3(a.n), dim3(threads), 0, s, a); };
    const int by_warp = ceil_div(a.k + V - 1, 32 * V);                 // SHIFTED: a phase of V - 1 at most
    if (form == WHOLE && a.q) launch_norm_whole<DT, WDT, true>(a, s);
    else if (form == WHOLE) launch_norm_whole<DT, WDT, false>(a, s);
    else if (form == SHIFTED && by_warp <= 16 * MOST) {
        // blocks that walk rows, a multiple of eight: 1024 threads an SM, of short rows 2048 (8192 x 333: 13.2 and 9.7 us)
        const int threads = by_warp <= 4 ? by_warp * 32 : ceil_div(by_warp, MOST) * 32;
        const dim3 blocks(std::min((a.n + 7) / 8 * 8, SMS * std::max(1, (by_warp <= 4 ? 2048 : 1024) / threads) / 8 * 8));
        if (by_warp <= 4) launch_overlapped(norm_k<DT, WDT, V, 1, false, false, true, 128>, blocks, dim3(threads), 0, s, a);
        else launch_overlapped(norm_k<DT, WDT, V, MOST, false, false, true, 512>, blocks, dim3(threads), 0, s, a);
    }
    else if (a.k <= 2048) go(norm_k<DT, WDT, 1, 4, false, false, false, 512>, ceil_div(a.k, 128) * 32);
    else go(norm_k<DT, WDT, 1, 32, false, false, false, 512>, ceil_div(a.k, 1024) * 32);
    return launch_status();
}

struct NormGradArgs {
    const void * h, * w, * dy, * ds;
    long long ldh, ldy, lds, ldx;
    float eps, inv_k;
    int n, k, stages;
    void * dx;
    float * parts;                     // [blocks][k]: each block's sums for the weight's gradient (null: not wanted)
};

__device__ __forceinline__ void copy16(void * shared, const void * global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(shared))), "l"(__cvta_generic_to_global(global)) : "memory");
}

// A block walks rows, the weight's gradient in registers. V > 1: the pieces of the rows to come are on their way into shared memory (`stages` rows of them), each thread's own, so that no barrier is needed for them;
// V = 1: one row after the other. SHIFT: the grid is a multiple of V, so that all rows of a block have the same phase and a thread its columns
// WARP (short rows): a warp a row, eight rows a block at a time and no barrier; the warps' sums for the weight's gradient meet at the end
template <int DT, int WDT, int V, int P, bool SHIFT, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512, (WARP ? 2 : 1) * (P <= 2 ? 2 : 1)) norm_grad_k(const NormGradArgs p) {
    extern __shared__ __align__(16) uint4 ahead[];                     // [stages][h, dy, ds][P][threads]
    __shared__ float2 red[2][32], red_again[32];
    grid_release();
    grid_wait();
    const int nt = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x, warp = threadIdx.x >> 5;
    const int row0 = WARP ? blockIdx.x * 8 + warp : blockIdx.x, step = WARP ? gridDim.x * 8 : gridDim.x;
    constexpr bool COPIES = V > 1;
    uint4 * const ring = ahead + (WARP ? size_t(warp) * p.stages * 3 * P * 32 : 0);
    using T = typename Elem<DT>::type;
    const Grid<V, SHIFT> grid{p.k, SHIFT ? phase_of<V>(static_cast<const T *>(p.h) + size_t(row0) * p.ldh, sizeof(T)) : 0};
    Piece<WDT, V> w[P];
    float dw[P][V];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int j = grid.first(i * nt + tid);
        w[i].zero();
        if (grid.any(j)) get_weight(w[i], p.w, j, grid);
#pragma unroll
        for (int l = 0; l < V; ++l) dw[i][l] = 0.f;
    }
    // A piece that is not whole comes with its neighbours in the matrix, which `trim` drops; in front of the matrix and behind it there may be nothing to read
    auto bring = [&](uint4 * to, const void * base, int row, long long ld, int j) {
        const T * at = static_cast<const T *>(base) + size_t(row) * ld;
        if (grid.whole(j) || (row * ld + j >= 0 && row * ld + j + V <= (p.n - 1) * ld + p.k)) return copy16(to, at + j);
        Piece<DT, V> some;
        some.zero();
        some.load_some(at, j, p.k);
        if constexpr (COPIES) *to = some.w[0];
    };
    auto copy = [&](int row, int stage) {
        if (row < p.n) {
            uint4 * at = ring + size_t(stage) * 3 * P * nt + tid;
#pragma unroll
            for (int i = 0; i < P; ++i, at += nt) {
                const int j = grid.first(i * nt + tid);
                if (!grid.any(j)) continue;
                bring(at, p.h, row, p.ldh, j);
                bring(at + P * nt, p.dy, row, p.ldy, j);
                if (p.ds) bring(at + 2 * P * nt, p.ds, row, p.lds, j);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");           // an empty one behind the last row: the count stays
    };
    if (COPIES)
        for (int s = 0; s < p.stages; ++s) copy(row0 + s * step, s);
    int turn = 0, stage = 0;                                           // two sets of words in turn: one barrier a row
    for (int row = row0; row < p.n; row += step, turn ^= 1) {
        if (COPIES) {
            if (p.stages == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
            else if (p.stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
            else asm volatile("cp.async.wait_group 2;" ::: "memory");
        }
        // piece i of the row's matrix m (h, dy, ds), read where it is wanted: the row is not held in registers across the barrier (that took twice as many, and half of the blocks)
        auto piece = [&](int m, int i, int j) {
            Piece<DT, V> v;
            if constexpr (COPIES) {
                v.w[0] = ring[(size_t(stage) * 3 + m) * P * nt + i * nt + tid];
                if (SHIFT && !grid.whole(j)) v.trim(j, p.k);
            } else {
                v.load(m == 0 ? p.h : m == 1 ? p.dy : p.ds, size_t(row) * (m == 0 ? p.ldh : m == 1 ? p.ldy : p.lds) + j);
            }
            return v;
        };
        // FAR: the row and a = dy w are taken in units of their own
        float unit = 1.f, unit_a = 1.f;
        // what(h, a, so far) over the row's values. Value by value a second look takes the weight once more, so that it needs no registers beside the first one's
        auto look = [&](auto what, auto again) {
            float2 v = make_float2(0.f, 0.f);
            auto add = [&](int i, const Piece<WDT, V> & w) {
                const int j = grid.first(i * nt + tid);
                if (!grid.any(j)) return;
                const Piece<DT, V> h = piece(0, i, j), g = piece(1, i, j);
#pragma unroll
                for (int l = 0; l < V; ++l) v = what(h[l], g[l] * w[l], v);
            };
            if constexpr (again && !COPIES) {
#pragma unroll 2
                for (int i = 0; i < P; ++i) {
                    const int j = grid.first(i * nt + tid);
                    Piece<WDT, V> once;
                    once.zero();
                    if (grid.any(j)) get_weight(once, p.w, j, grid);
                    add(i, once);
                }
            } else {
#pragma unroll
                for (int i = 0; i < P; ++i) add(i, w[i]);
            }
            return v;
        };
        auto sums = [](float h, float a, float2 v) { return make_float2(fmaf(h, h, v.x), fmaf(a, h, v.y)); };
        auto finish = [&](auto FAR, float rho, float t) {
            // a product of the units that may pass 32 bits by itself, in two halves
            const int e = exponent_of(unit) - exponent_of(unit_a);
            const float half = power_of_two(e / 2), rest = power_of_two(e - e / 2);
            const bool far = FAR && (COPIES || unit != 1.f || unit_a != 1.f);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int j = grid.first(i * nt + tid);
                if (!grid.any(j)) continue;
                const Piece<DT, V> h = piece(0, i, j), g = piece(1, i, j);
                Piece<DT, V> s;
                s.zero();
                if (p.ds) s = piece(2, i, j);
                float d[V];
#pragma unroll
                for (int l = 0; l < V; ++l) {
                    const float f = FAR ? h[l] * unit : h[l], a = fmaf(-f, t, FAR ? g[l] * w[i][l] * unit_a : g[l] * w[i][l]);
                    d[l] = far ? fmaf(rho * a * half, rest, s[l]) : fmaf(rho, a, s[l]);
                    dw[i][l] = fmaf(g[l], f * rho, dw[i][l]);
                }
                put<DT>(p.dx, size_t(row) * p.ldx, j, grid, d);
            }
        };
        float2 v = over_row<WARP>(look(sums, std::false_type{}), make_float2(0.f, 0.f), red[turn], Add2());
        float m = fmaf(v.x, p.inv_k, p.eps), rho = inverse_root(m), t = v.y * p.inv_k * rho * rho;
        if (!ordinary(m) || !(fabsf(t) < INFINITY)) {
            const float2 largest = over_row<WARP>(look([&](float h, float a, float2 v) { return make_float2(fmaxf(v.x, fabsf(h)), fmaxf(v.y, fabsf(a))); }, std::true_type{}), make_float2(0.f, 0.f), red_again, Max2());
            unit = unit_of(largest.x, p.eps);
            unit_a = unit_of(largest.y, 0.f);
            if (!WARP) __syncthreads();                                // the maxima have been read
            v = over_row<WARP>(look([&](float h, float a, float2 v) { return sums(h * unit, a * unit_a, v); }, std::true_type{}), make_float2(0.f, 0.f), red_again, Add2());
            m = fmaf(v.x, p.inv_k, p.eps * unit * unit);
            // in the units: rho h as it is, rho and t h in theirs
            rho = inverse_root(m);
            t = v.y * p.inv_k * rho * rho;
        }
        // (value by value there is one form: two of 32 values a thread spill, 2048 x 4097 62 us instead of 55)
        if (COPIES && unit == 1.f && unit_a == 1.f) finish(std::false_type{}, rho, t);
        else finish(std::true_type{}, rho, t);
        if (COPIES) {                                                  // this row's pieces have been read
            copy(row + p.stages * step, stage);
            if (++stage == p.stages) stage = 0;
        }
    }
    if (p.parts) {
        if (WARP) __syncthreads();                                     // the ring is free: a row of sums a warp
        float * const at = WARP ? reinterpret_cast<float *>(ahead) + warp * (32 * P * V) : p.parts + size_t(blockIdx.x) * p.k;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int j = grid.first(i * nt + tid);
            if (!grid.any(j)) continue;
            if constexpr (COPIES && !SHIFT) {
#pragma unroll
                for (int l = 0; l < V; l += 4) *reinterpret_cast<float4 *>(at + j + l) = make_float4(dw[i][l], dw[i][l + 1], dw[i][l + 2], dw[i][l + 3]);
            } else {
#pragma unroll
                for (int l = 0; l < V; ++l)
                    if (unsigned(j + l) < unsigned(p.k)) at[j + l] = dw[i][l];
            }
        }
        if (WARP) {
            __syncthreads();
            for (int j = threadIdx.x; j < p.k; j += 256) {
                const float * from = reinterpret_cast<const float *>(ahead) + j;
                float sum = from[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) sum += from[i * (32 * P * V)];
                p.parts[size_t(blockIdx.x) * p.k + j] = sum;
            }
        }
    }
}

// dw[j] = (accumulate: +) the sum over the blocks' parts, in a fixed order: 32 columns a block; a warp takes one part, or (WIDE: rows of whole 16 bytes) four with 16 bytes a lane, and all parts are on their way
// at once. (30000 x 256: 14.1 us a value a lane, 12.5 with 16 bytes; with eight warps four more)
template <bool WIDE>
__global__ void __launch_bounds__(1024) norm_weight_grad_k(const float * parts, int blocks, int k, float * dw, int accumulate) {
    __shared__ float part[32][33];
    grid_release();
    grid_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float s = 0.f;
    if (WIDE) {
        const int j = blockIdx.x * 32 + (lane & 7) * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j < k)
#pragma unroll 5
            for (int b = warp * 4 + (lane >> 3); b < blocks; b += 128) {
                const float4 a = *reinterpret_cast<const float4 *>(parts + size_t(b) * k + j);
                v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
            }
#pragma unroll
        for (int d = 8; d <= 16; d <<= 1) {
            v.x += __shfl_xor_sync(0xffffffffu, v.x, d); v.y += __shfl_xor_sync(0xffffffffu, v.y, d);
            v.z += __shfl_xor_sync(0xffffffffu, v.z, d); v.w += __shfl_xor_sync(0xffffffffu, v.w, d);
        }
        if (lane < 8) { part[warp][4 * lane] = v.x; part[warp][4 * lane + 1] = v.y; part[warp][4 * lane + 2] = v.z; part[warp][4 * lane + 3] = v.w; }
    } else {
        const int j = blockIdx.x * 32 + lane;
        if (j < k)
#pragma unroll 10
            for (int b = warp; b < blocks; b += 32) s += parts[size_t(b) * k + j];
        part[warp][lane] = s;
    }
    __syncthreads();
    // the 32 sums of a column by a warp
    s = part[lane][warp];
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const int c = blockIdx.x * 32 + warp;
    if (lane || c >= k) return;
    dw[c] = accumulate ? dw[c] + s : s;
}

// Blocks that walk the rows, and so the parts of the weight's gradient. Long rows: as many of an SM as 32 KB of 16-bit values in a row each make, eight at most; a multiple of eight, the most phases that rows
// have. Short ones, a warp each: four blocks an SM, or two where a row takes four pieces a lane. us, half of these / these / twice as many blocks, bf16: 8192 x 4096 48.8 / 50.9 / 53.1, 8192 x 2048 27.6 / 30.1 / 30.1,
// 4096 x 8192 51.5 / 49.1 / 55.1, 2048 x 16384 50.4 / 50.4 / 63.5, 600 x 4096 8.7 / 8.8 / 9.9; a warp each: 30000 x 256 13.0 / 12.8 / 14.4, 30000 x 512 24.9 / 25.8 / 26.2, 8192 x 1024 13.2 / 12.6 / 14.7, 16000 x 128 8.8 / 8.9 / 10.5
constexpr int GRAD_NUM = 16384;
int grad_blocks_most(int n, int k) { return std::min((n + 7) / 8 * 8, SMS * std::max(4, std::min(8, GRAD_NUM / k)) / 8 * 8); }

template <int DT, int WDT>
int32_t launch_norm_grad(NormGradArgs a, Form form, cudaStream_t s, int & blocks) {
    constexpr int V = DT == B2MOE_F32 ? 4 : 8, MOST = NORM_MAX_COLS / V / 512;
    // per_sm blocks fill an SM's shared memory, so that a launch that becomes resident while the one before it runs spreads over all SMs (69 us instead of 49 for 8192 x 4096, with more than two of an SM)
    auto go = [&](auto kernel, bool by_row, int threads, int pieces, int per_sm) -> int32_t {
        const size_t row = size_t(3) * pieces * threads * 16, room = 228 * 1024 / per_sm - 2048;      // of a stage; of a block (an SM's 228 KB, less a block's own 1 KB and its static words)
        a.stages = int(std::min<size_t>(3, std::max<size_t>(1, row ? room / row : 1)));
        if (room > 48 * 1024 && !allow_smem(kernel, 226 * 1024)) return B2MOE_ERR_CUDA;
        blocks = by_row ? std::min(ceil_div(a.n, 8), SMS * per_sm) : std::min((a.n + 7) / 8 * 8, SMS * per_sm / 8 * 8);
        launch_overlapped(kernel, dim3(blocks), dim3(threads), row ? std::max(a.stages * row, room) : 0, s, a);
        return launch_status();
    };
    const int by_warp = ceil_div(form == SHIFTED ? a.k + V - 1 : a.k, 32 * V), per_sm = std::max(1, std::min(8, GRAD_NUM / a.k));      // a warp's pieces
    if (form == SINGLE || by_warp > 16 * MOST) {
        if (a.k <= 2048) return go(norm_grad_k<DT, WDT, 1, 4, false, false>, false, ceil_div(a.k, 128) * 32, 0, per_sm);
        return go(norm_grad_k<DT, WDT, 1, 32, false, false>, false, ceil_div(a.k, 1024) * 32, 0, per_sm);
    }
    auto with = [&](auto shift) -> int32_t {
        constexpr bool SHIFT = decltype(shift)::value;
        if (by_warp <= 1) return go(norm_grad_k<DT, WDT, V, 1, SHIFT, true>, true, 256, 1, 4);
        if (by_warp <= 2) return go(norm_grad_k<DT, WDT, V, 2, SHIFT, true>, true, 256, 2, 4);
        if (by_warp <= 4) return go(norm_grad_k<DT, WDT, V, 4, SHIFT, true>, true, 256, 4, 2);
        if (by_warp <= 32) return go(norm_grad_k<DT, WDT, V, 2, SHIFT, false>, false, ceil_div(by_warp, 2) * 32, 2, per_sm);
        return go(norm_grad_k<DT, WDT, V, MOST, SHIFT, false>, false, ceil_div(by_warp, MOST) * 32, MOST, per_sm);
    };
    return form == SHIFTED ? with(std::true_type{}) : with(std::false_type{});
}

struct Rows { const void * p; long long ld; };
Form form_of(int k, int dtype, const void * weight, std::initializer_list<Rows> rows) {
    const int size = int(dtype_bytes(dtype)), per = 16 / size, phase = int(reinterpret_cast<uintptr_t>(rows.begin()->p) / size % per), ld = int(rows.begin()->ld % per);
    bool whole = k % per == 0 && phase == 0 && ld == 0 && aligned16(weight), shared = true;
    for (const Rows & r : rows)
        if (r.p) shared = shared && int(reinterpret_cast<uintptr_t>(r.p) / size % per) == phase && int(r.ld % per) == ld;
    return shared ? (whole ? WHOLE : SHIFTED) : SINGLE;
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
    const Form form = form_of(k, dtype, weight, {{x, ldx}, {residual, ldr}, {sum, lds}, {y, ldy}});
    if (q && form != WHOLE) return B2MOE_ERR_ALIGN;                            // rows in 8 bits come from rows in pieces of 16 bytes
    const NormArgs a{x, residual, weight, ldx, ldr, lds, ldy, ldq, eps, 1.f / float(k), n, k, sum, y, q, scale};
    cudaStream_t s = as_stream(stream);
    if (dtype == B2MOE_F32) return launch_norm<B2MOE_F32, B2MOE_F32>(a, form, s);
    if (dtype == B2MOE_F16) return weight_dtype == B2MOE_F32 ? launch_norm<B2MOE_F16, B2MOE_F32>(a, form, s) : launch_norm<B2MOE_F16, B2MOE_F16>(a, form, s);
    return weight_dtype == B2MOE_F32 ? launch_norm<B2MOE_BF16, B2MOE_F32>(a, form, s) : launch_norm<B2MOE_BF16, B2MOE_BF16>(a, form, s);
}

extern "C" B2MOE_API size_t b2moe_rms_norm_backward_workspace_bytes(int32_t n, int32_t k) {
    if (n <= 0 || n > I8_MAX_ROWS || k <= 0 || k > NORM_MAX_COLS) return 0;
    return align_up(size_t(grad_blocks_most(n, k)) * k * sizeof(float), 16);
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
    const Form form = form_of(k, dtype, weight, {{h, ldh}, {grad_y, ldgy}, {grad_sum, ldgs}, {grad_x, ldgx}});
    const NormGradArgs a{h, weight, grad_y, grad_sum, ldh, ldgy, ldgs, ldgx, eps, 1.f / float(k), n, k, 1, grad_x, grad_weight ? static_cast<float *>(workspace) : nullptr};
    cudaStream_t s = as_stream(stream);
    int32_t rc, blocks = 0;
    if (dtype == B2MOE_F32) rc = launch_norm_grad<B2MOE_F32, B2MOE_F32>(a, form, s, blocks);
    else if (dtype == B2MOE_F16) rc = weight_dtype == B2MOE_F32 ? launch_norm_grad<B2MOE_F16, B2MOE_F32>(a, form, s, blocks) : launch_norm_grad<B2MOE_F16, B2MOE_F16>(a, form, s, blocks);
    else rc = weight_dtype == B2MOE_F32 ? launch_norm_grad<B2MOE_BF16, B2MOE_F32>(a, form, s, blocks) : launch_norm_grad<B2MOE_BF16, B2MOE_BF16>(a, form, s, blocks);
    if (rc) return rc;
    if (!grad_weight) return B2MOE_OK;
    // in plain stream order: as an early resident it takes the registers of the rows' last blocks (8192 x 4096: 52.4 us, 49.8 so)
    const dim3 grid(ceil_div(k, 32)), block(1024);
    const float * parts = static_cast<const float *>(workspace);
    if (k % 4) norm_weight_grad_k<false><<<grid, block, 0, s>>>(parts, blocks, k, grad_weight, accumulate);
    else norm_weight_grad_k<true><<<grid, block, 0, s>>>(parts, blocks, k, grad_weight, accumulate);
    return launch_status();
}
