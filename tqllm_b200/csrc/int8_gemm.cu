// Products of 8-bit integers for many rows: tcgen05.mma kind::i8, 32-bit sums in tensor memory. See int8_products.cu for the arithmetic.
//
// D [128 weight rows x N activation rows] = W Q^T: both operands are rows of K bytes as they lie in memory, brought 128 columns at a time by TMA into
// 128-byte swizzled tiles, so nothing is converted on the way. The weight rows are the M side: an item of N = 16 to 256 activation rows wastes little where an
// expert has few, and a warp of the epilogue stores neighbouring outputs of one activation row. Gate and up share a tile, 16 rows of each in turn, so that lanes l and
// l + 16 of the epilogue hold both sums of an output.
//
// One block per SM walks the items (tile of activation rows, block of weight rows): one thread issues the copies into a ring, one the products, eight warps
// empty one accumulator while the next one fills.
#include <cuda.h>

#include <cstring>

#include "int8.cuh"
#include "tc_ptx.cuh"
#include "tensor_map.cuh"

namespace b2 {
namespace {
using namespace tc;

constexpr int TC_THREADS = 384, TC_EPI_WARP0 = 4, TC_EPI_WARPS = 8, TC_EPI_THREADS = 32 * TC_EPI_WARPS, TC_MAX_STAGES = 12, TC_MAX_EXPERTS = 4096;
constexpr int TC_A_BYTES = 128 * 128, TC_SMEM = 227 * 1024;

struct TcMaps { CUtensorMap a[2], shared[2], b; };
struct TcArgs {
    int nt, box, stages, row_blocks, tiles;     // activation rows of an item, of a copy; ring; blocks of weight rows; items of a dense call in the row direction
    uint32_t tmem_cols;
    int * status;
};

// kind::i8: A and B signed 8-bit, D signed 32-bit, both K-major
__device__ __forceinline__ uint32_t idesc_i8(uint32_t m, uint32_t n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24); }
__device__ __forceinline__ void mma_i8(bool lead, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t id, uint32_t acc) {
    asm volatile("{\n .reg .pred p, q;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %6, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
                 " @q tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, p;\n}" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(id), "r"(acc), "r"(SW128_DESC_HI), "r"(uint32_t(lead)) : "memory");
}
__device__ __forceinline__ void epi_sync() { asm volatile("bar.sync 1, %0;" ::"n"(TC_EPI_THREADS) : "memory"); }

struct TcItem { int e, first, count, rb; };      // expert, first row (slot), rows, block of weight rows

// this lane's weight row of an item
template <int MATS>
__device__ __forceinline__ int weight_row(const TcItem & im, int quarter, int lane) {
    return MATS == 2 ? im.rb * 64 + 16 * quarter + (lane & 15) : im.rb * 128 + 32 * quarter + lane;
}
// the item's outputs from tensor memory; t: (output row, scale) of its activation rows, v: the scales of the lane's weight row
template <int MATS, class T>
__device__ __forceinline__ void store_item(const I8Args & p, const TcItem & im, uint32_t taddr, const int2 * t, const float (&v)[MATS], int quarter, int half, int lane) {
    const bool upper = MATS == 2 && lane >= 16;
    const int row = weight_row<MATS>(im, quarter, lane);
    const bool in = row < p.rows;
    T * const y = static_cast<T *>(p.y) + row;
    auto put = [&](int at, float f) {
        T * d = y + size_t(uint32_t(at)) * p.ldy;
        if constexpr (std::is_same<T, float>::value) *d = f;
        else if constexpr (std::is_same<T, __half>::value) *d = __float2half_rn(f);
        else *d = __float2bfloat16_rn(f);
    };
#pragma unroll 1
    for (int c = 16 * half; c < im.count; c += 32) {
        uint32_t d[16];
        tmem_ld16(taddr + c, d);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
            const int4 two = *reinterpret_cast<const int4 *>(t + c + j);      // activation rows c + j and the next: (output row, scale) each
            const float s0 = __int_as_float(two.y), s1 = __int_as_float(two.w);
            if (MATS == 2) {
                // lanes l and l + 16 hold gate and up of the same output: they swap, and l finishes the even row, l + 16 the odd one
                const uint32_t other = __shfl_xor_sync(0xffffffffu, upper ? d[j] : d[j + 1], 16);
                const int gs = int(upper ? other : d[j]), us = int(upper ? d[j + 1] : other);
                const float s = upper ? s1 : s0, g = float(gs) * (s * v[0]), u = float(us) * (s * v[MATS - 1]);
                if (in && c + j + int(upper) < im.count) put(upper ? two.z : two.x, g / (1.f + expf(-g)) * u);
            } else {
                if (in && c + j < im.count) put(two.x, float(int(d[j])) * (s0 * v[0]));
                if (in && c + j + 1 < im.count) put(two.z, float(int(d[j + 1])) * (s1 * v[0]));
            }
        }
    }
}

template <int MATS>
__global__ void __launch_bounds__(TC_THREADS, 1) i8_gemm_k(const I8Args p, const TcArgs c, const __grid_constant__ TcMaps maps) {
    extern __shared__ __align__(1024) uint8_t tc_mem[];
    __shared__ __align__(16) int2 table[2][256];
    __shared__ __align__(8) uint64_t bars[2 * TC_MAX_STAGES + 5];
    __shared__ int scan[TC_THREADS / 32];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t stage_bytes = TC_A_BYTES + c.nt * 128;
    uint8_t * const ring = tc_mem + (1024u - (saddr(tc_mem) & 1023u)) % 1024u;
    const int e1 = p.experts + 1;
    int * const ends = reinterpret_cast<int *>(ring + size_t(c.stages) * stage_bytes), * const offs = ends + e1;      // tiles up to and with expert e, its first slot
    const uint32_t full = saddr(bars), empty = full + 8 * TC_MAX_STAGES, acc_full = empty + 8 * TC_MAX_STAGES, acc_empty = acc_full + 16, drain = acc_empty + 16;
    if (threadIdx.x == 0) {
        for (int i = 0; i < c.stages; ++i) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) { bar_init(acc_full + 8 * i, 1); bar_init(acc_empty + 8 * i, TC_EPI_WARPS); }
        bar_init(drain, 1);
        bar_init_fence();
        abort_flag = 0;
        for (int m = 0; m < MATS; ++m) { prefetch_map(maps.a + m); if (p.plan) prefetch_map(maps.shared + m); }
        prefetch_map(&maps.b);
    }
    if (warp == 1) tmem_alloc(saddr(&tmem_slot), c.tmem_cols);
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    grid_wait();
    grid_release();                                                    // after the wait: a down product behind this launch may read the plan above its own
    const int * counts = p.plan + PLAN_HDR, * offsets = counts + e1, * perm = offsets + e1 + 1 + e1;
    int tiles = c.tiles;
    if (p.plan) {
        // inclusive prefix sums of the experts' tiles: a span of experts a thread
        const int span = (e1 + TC_THREADS - 1) / TC_THREADS, lo = min(e1, int(threadIdx.x) * span), hi = min(e1, lo + span);
        int mine = 0;
        for (int e = lo; e < hi; ++e) mine += (counts[e] + c.nt - 1) / c.nt;
        int run = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, run, d);
            if (lane >= d) run += o;
        }
        if (lane == 31) scan[warp] = run;
        __syncthreads();
        run -= mine;
        for (int w = 0; w < warp; ++w) run += scan[w];
        for (int e = lo; e < hi; ++e) {
            run += (counts[e] + c.nt - 1) / c.nt;
            ends[e] = run;
            offs[e] = offsets[e];
        }
        if (threadIdx.x == 0) offs[e1] = offsets[e1];
        __syncthreads();
        tiles = ends[e1 - 1];
    }
    const int items = tiles * c.row_blocks, steps = (p.cols + 127) / 128;
    auto locate = [&](int it) {
        TcItem im;
        const int tile = it / c.row_blocks;
        im.rb = it - tile * c.row_blocks;
        im.e = 0;
        int t = tile;
        im.first = 0;
        im.count = p.n;
        if (p.plan) {
            int lo = 0, hi = e1 - 1;                                   // the first expert whose tiles end behind this one
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (ends[mid] > tile) hi = mid;
                else lo = mid + 1;
            }
            im.e = lo;
            t = tile - (lo ? ends[lo - 1] : 0);
            im.first = offs[lo];
            im.count = offs[lo + 1] - offs[lo];
        }
        im.first += t * c.nt;
        im.count = min(c.nt, im.count - t * c.nt);
        return im;
    };
    auto give_up = [&]() {
        abort_flag = 1;
        if (c.status) atomicExch(c.status, 2);
    };

    if (warp == 0) {
        // ---- copies ----
        uint32_t issued = 0, slot = 0, phase = 1;                      // phase: of the empty barrier's wait (none in the first round)
        bool ok = true;
        const bool lead = elect_one();
#pragma unroll 1
        for (int it = blockIdx.x; it < items && ok && !abort_flag; it += gridDim.x) {
            const TcItem im = locate(it);
            const bool shared = p.plan && im.e == p.experts;
            const CUtensorMap * a = shared ? maps.shared : maps.a;
            const int e = shared ? 0 : im.e, boxes = (im.count + c.box - 1) / c.box;
#pragma unroll 1
            for (int k = 0; k < steps; ++k) {
                if (issued >= uint32_t(c.stages) && !warp_wait(empty + 8 * slot, phase)) { ok = false; break; }
                if (lead) {
                    const uint32_t bar = full + 8 * slot, dst = saddr(ring) + slot * stage_bytes;
                    bar_expect_tx(bar, TC_A_BYTES + uint32_t(boxes * c.box) * 128);
                    if (MATS == 2) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            tma_load_3d(dst + 4096 * i, a, 128 * k, 64 * im.rb + 16 * i, e, bar);
                            tma_load_3d(dst + 4096 * i + 2048, a + 1, 128 * k, 64 * im.rb + 16 * i, e, bar);
                        }
                    } else {
                        tma_load_3d(dst, a, 128 * k, 128 * im.rb, e, bar);
                    }
                    for (int i = 0; i < boxes; ++i) tma_load_2d(dst + TC_A_BYTES + i * c.box * 128, &maps.b, 128 * k, im.first + i * c.box, bar);
                }
                __syncwarp();
                ++issued;
                if (++slot == uint32_t(c.stages)) { slot = 0; phase ^= 1u; }
            }
        }
        if (!ok && lane == 0) give_up();
        // before leaving, every copy must have landed (after a clean run these waits return at once)
#pragma unroll 1
        for (uint32_t i = issued > uint32_t(c.stages) ? issued - c.stages : 0; i < issued; ++i) bar_wait(full + 8 * (i % c.stages), (i / c.stages) & 1u);
    } else if (warp == 1) {
        // ---- products: the whole warp walks the loop, one lane issues ----
        const bool lead = elect_one();
        const uint32_t a0 = sw128_desc_lo(saddr(ring)), step = stage_bytes >> 4;
        uint32_t slot = 0, phase = 0, done = 0;
        bool ok = true;
#pragma unroll 1
        for (int it = blockIdx.x; it < items && ok && !abort_flag; it += gridDim.x, ++done) {
            const uint32_t h = done & 1u, d = tmem + h * c.nt, id = idesc_i8(128, uint32_t(__shfl_sync(0xffffffffu, locate(it).count, 0) + 15) & ~15u);
            if (done >= 2 && !warp_wait(acc_empty + 8 * h, ((done >> 1) - 1) & 1u)) { ok = false; break; }
            fence_after();
#pragma unroll 1
            for (int k = 0; k < steps; ++k) {
                if (!warp_wait(full + 8 * slot, phase)) { ok = false; break; }
                fence_after();
                const uint32_t a = a0 + slot * step, b = a + (TC_A_BYTES >> 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) mma_i8(lead, d, a + 2 * i, b + 2 * i, id, k > 0 || i > 0);
                mma_commit(lead, empty + 8 * slot);
                if (++slot == uint32_t(c.stages)) { slot = 0; phase ^= 1u; }
            }
            if (ok) mma_commit(lead, acc_full + 8 * h);
        }
        if (!ok && lane == 0) give_up();
        // nothing may be in flight when the tensor memory is freed
        mma_commit(lead, drain);
        warp_wait(drain, 0);
    } else if (warp >= TC_EPI_WARP0) {
        // ---- results: warp q of either half reads the lanes 32 (q mod 4) of tensor memory, the halves take 16 columns in turn ----
        const int tid = threadIdx.x - 32 * TC_EPI_WARP0, quarter = warp & 3, half = (warp - TC_EPI_WARP0) >> 2;
        // what the stores of an item need to know (its rows' places and scales, the weight row's scales) is asked for an item ahead
        int2 mine = make_int2(0, 0);
        float v[MATS];
        auto fetch = [&](const TcItem & im) {
            if (tid < im.count) mine = make_int2(p.plan ? perm[im.first + tid] : im.first + tid, __float_as_int(p.s[im.first + tid]));
            const int row = weight_row<MATS>(im, quarter, lane);
#pragma unroll
            for (int m = 0; m < MATS; ++m) v[m] = row < p.rows ? (p.plan && im.e == p.experts ? p.shared_v[m] : p.v[m] + size_t(im.e) * p.rows)[row] : 0.f;
        };
        uint32_t done = 0;
        bool ok = true;
        TcItem im{}, next{};
        if (int(blockIdx.x) < items) {
            next = locate(blockIdx.x);
            fetch(next);
        }
#pragma unroll 1
        for (int it = blockIdx.x; it < items; it += gridDim.x, ++done) {
            const uint32_t h = done & 1u;
            im = next;
            if (tid < im.count) table[h][tid] = mine;
            float scale[MATS];
#pragma unroll
            for (int m = 0; m < MATS; ++m) scale[m] = v[m];
            epi_sync();                                                // the table is there; the other one's item has been read by every warp
            if (it + int(gridDim.x) < items) {
                next = locate(it + gridDim.x);
                fetch(next);
            }
            ok = ok && !abort_flag && warp_wait(acc_full + 8 * h, (done >> 1) & 1u);
            fence_after();
            if (ok) {
                const uint32_t taddr = tmem + h * c.nt + (uint32_t(32 * quarter) << 16);
                if (p.y_dtype == B2MOE_F32) store_item<MATS, float>(p, im, taddr, table[h], scale, quarter, half, lane);
                else if (p.y_dtype == B2MOE_F16) store_item<MATS, __half>(p, im, taddr, table[h], scale, quarter, half, lane);
                else store_item<MATS, __nv_bfloat16>(p, im, taddr, table[h], scale, quarter, half, lane);
            } else if (lane == 0) {
                give_up();
            }
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(acc_empty + 8 * h);
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == 1) tmem_free(tmem, c.tmem_cols);
}

int sm_count() {
    static const int count = [] {                                      // the library runs on one kind of GPU
        int dev = 0, n = 0;
        return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
    }();
    return count;
}
bool map_rows(CUtensorMap & m, const int8_t * base, int cols, long long rows, long long stride, int experts, int box) {
    if (experts) {
        const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(experts)}, strides[2] = {cuuint64_t(stride), cuuint64_t(stride) * rows};
        const cuuint32_t b[3] = {128, cuuint32_t(box), 1};
        return encode_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, b, CU_TENSOR_MAP_SWIZZLE_128B);
    }
    const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)}, strides[1] = {cuuint64_t(stride)};
    const cuuint32_t b[2] = {128, cuuint32_t(box)};
    return encode_map(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, b, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace

bool i8_gemm_supported(int experts) { return experts <= TC_MAX_EXPERTS; }

template <int MATS>
int32_t i8_gemm(const I8Args & p, long long q_rows, int per_group, int * status, cudaStream_t s) {
    TcArgs c{};
    c.row_blocks = ceil_div(p.rows, MATS == 2 ? 64 : 128);
    // Items of 256 rows halve what the weights cost in copies and products (8192 x 4096 x 4096: 96 us, with 128 rows 153), items of 128 leave room for six ring
    // stages instead of four and waste less where an expert has fewer (512 experts at 80 each, gate/up 211 against 225 us; 128 experts at 16 each 242 and 263, at 128 each with a
    // skewed load 385 and 333); below that nothing is gained (64 rows, 16 each: 248). A dense call takes the large ones where they fill the SMs
    c.nt = per_group > 96 && (p.plan || (long long)ceil_div(p.n, 256) * c.row_blocks >= sm_count()) ? 256 : 128;
    c.box = 64;                                                        // rows of a copy: an item takes as many copies as it has rows for
    c.tiles = p.plan ? 0 : ceil_div(p.n, c.nt);
    c.tmem_cols = std::max(32, 2 * c.nt);
    c.status = status;
    const size_t table = p.plan ? size_t(2 * (p.experts + 1) + 1) * sizeof(int) : 0, fixed = 8 * 1024;      // static arrays and the alignment of the ring
    c.stages = int(std::min<size_t>(TC_MAX_STAGES, (TC_SMEM - fixed - table) / (TC_A_BYTES + size_t(c.nt) * 128)));
    TcMaps maps;
    std::memset(&maps, 0, sizeof(maps));
    const int box = MATS == 2 ? 16 : 128;
    bool ok = map_rows(maps.b, p.q, p.cols, q_rows, p.ldq, 0, c.box);
    for (int m = 0; m < MATS; ++m) {
        ok = ok && map_rows(maps.a[m], p.w[m], p.cols, p.rows, p.cols, p.experts, box);
        if (p.shared_w[m]) ok = ok && map_rows(maps.shared[m], p.shared_w[m], p.cols, p.rows, p.cols, 1, box);
        else maps.shared[m] = maps.a[m];
    }
    if (!ok) return B2MOE_ERR_CUDA;
    const size_t smem = 1024 + size_t(c.stages) * (TC_A_BYTES + size_t(c.nt) * 128) + table;
    if (cudaFuncSetAttribute(i8_gemm_k<MATS>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)) != cudaSuccess) return B2MOE_ERR_CUDA;
    const long long most = p.plan ? (long long)sm_count() : (long long)c.tiles * c.row_blocks;
    launch_overlapped(i8_gemm_k<MATS>, dim3(unsigned(std::min<long long>(sm_count(), most))), dim3(TC_THREADS), smem, s, p, c, maps);
    return launch_status();
}
template int32_t i8_gemm<1>(const I8Args &, long long, int, int *, cudaStream_t);
template int32_t i8_gemm<2>(const I8Args &, long long, int, int *, cudaStream_t);

}  // namespace b2
