// Products of 8-bit integers for many rows: tcgen05.mma kind::i8, 32-bit sums in tensor memory. See int8_products.cu for the arithmetic.
//
// D [128 weight rows x N activation rows] = W Q^T: both operands are rows of K bytes as they lie in memory, brought 128 columns at a time by TMA into
// 128-byte swizzled tiles, so nothing is converted on the way. The weight rows are the M side: an item of N = 16 to 256 activation rows wastes little where an
// expert has few, and a warp of the epilogue stores neighbouring outputs of one activation row. Gate and up share a tile, 16 rows of each in turn, so that lanes l and
// l + 16 of the epilogue hold both sums of an output.
//
// One block per SM (two for short rows) walks the items (tile of activation rows, block of weight rows): one thread issues the copies into a ring, one the products, eight warps
// empty one accumulator while the next one fills.
//   8192 rows of 4096 x 4096: 86 to 90 us by card, 3.2e15 operations a second (1.93 of the measured bf16 rate); 96 without pairs, 150 with items of 128 rows. Bound by the tensor pipe.
//   gate/up of 128 experts of 1408 x 4096 at 16 rows each: 241 us, 6.1 TB/s (0.94 of measured); down of 512 of 2048 x 512 at 1.2 rows each: 62 us, 5.9 TB/s. Bound by reading the weights.
#include <cooperative_groups.h>
#include <cuda.h>

#include <array>
#include <cstring>

#include "int8.cuh"
#include "tc_ptx.cuh"
#include "tensor_map.cuh"

namespace b2 {
namespace {
using namespace tc;

constexpr int TC_THREADS = 384, TC_EPI_WARP0 = 4, TC_EPI_WARPS = 8, TC_EPI_THREADS = 32 * TC_EPI_WARPS, TC_MAX_STAGES = 12, TC_MAX_EXPERTS = 4096;
constexpr int TC_A_BYTES = 128 * 128, TC_SMEM = 227 * 1024, TC_MAX_SPLIT = 8;
// static arrays and the alignment of the ring; what a launch asks for at most
constexpr int TC_FIXED = 8 * 1024, TC_ALIGN = 1024, TC_SMEM_MOST = TC_SMEM - TC_FIXED + TC_ALIGN;

struct TcMaps { CUtensorMap a[2], shared[2], b; };
struct TcArgs {
    int nt, box, stages, row_blocks, tiles;     // activation rows of an item, of a copy; ring; blocks of weight rows; items of a dense call in the row direction
    int half;                                   // columns of an accumulator
    int b_rows;                                 // a block's copies of an item's rows
    uint32_t tmem_cols;
    int * status;
    int drop;                                   // test hook: the copies of this step of every block are left out (-1: none)
};
int g_drop_step = -1;

// kind::i8: A and B signed 8-bit, D signed 32-bit, both K-major
__device__ __forceinline__ uint32_t idesc_i8(uint32_t m, uint32_t n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24); }
__device__ __forceinline__ void mma_i8(bool lead, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t id, uint32_t acc) {
    asm volatile("{\n .reg .pred p, q;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %6, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
                 " @q tcgen05.mma.cta_group::1.kind::i8 [%0], da, db, %3, p;\n}" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(id), "r"(acc), "r"(SW128_DESC_HI), "r"(uint32_t(lead)) : "memory");
}
// The same across a pair of blocks (the even one of a cluster issues): 256 rows of D, 128 in either block's tensor memory; A and B lie half in either block's shared memory
__device__ __forceinline__ void mma_i8_pair(bool lead, uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t id, uint32_t acc) {
    asm volatile("{\n .reg .pred p, q;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %6, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
                 " @q tcgen05.mma.cta_group::2.kind::i8 [%0], da, db, %3, p;\n}" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(id), "r"(acc), "r"(SW128_DESC_HI), "r"(uint32_t(lead)) : "memory");
}
// one arrival at the barrier of this place in both blocks
__device__ __forceinline__ void mma_commit_pair(bool lead, uint32_t bar) {
    asm volatile("{\n .reg .pred q;\n .reg .b16 m;\n setp.ne.b32 q, %1, 0;\n mov.b16 m, 3;\n"
                 " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n}" ::"r"(bar), "r"(uint32_t(lead)) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t slot_saddr, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot_saddr), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t base, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols) : "memory");
}
// copies into this block's shared memory whose completion goes to a barrier of either block of the pair
__device__ __forceinline__ void pair_load_3d(uint32_t dst, const void * map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void pair_load_2d(uint32_t dst, const void * map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, int rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
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

// The outputs of an item that was left unfinished by a wait that ran out: NaN, since the call may have no status word to tell. One weight row; of the item's activation rows this half's 16 of every 32.
// Not inlined, so that it takes no registers from what happens
__device__ __noinline__ void spoil_rows(void * y, int dtype, long long ldy, int row, const int2 * t, int count, int half) {
    for (int c = 16 * half; c < count; c += 32)
        for (int j = c; j < min(c + 16, count); ++j) store_act(y, dtype, size_t(uint32_t(t[j].x)) * ldy + row, __int_as_float(0x7fc00000));
}

// SPLIT (dense calls with few items): the blocks of a cluster take parts of an item's columns each, and then a share of its activation rows each, whose parts they
// read from one another's shared memory: whole numbers, so the sum is the same
// PAIR (long rows): two blocks take neighbouring blocks of weight rows of the same activation rows, of which each brings a half: the copies from the L2, which set the pace of
// large calls, are a third fewer. The even block issues the products of both and has the barriers of the operands and of the sums that have been read.
enum { TC_SPLIT = 1, TC_PAIR = 2 };
template <int MATS, int MODE>
__global__ void __launch_bounds__(TC_THREADS, MODE ? 1 : 2) i8_gemm_k(const I8Args p, const TcArgs c, const __grid_constant__ TcMaps maps) {
    extern __shared__ __align__(1024) uint8_t tc_mem[];
    __shared__ __align__(16) int2 table[2][256];
    __shared__ __align__(8) uint64_t bars[2 * TC_MAX_STAGES + 5];
    __shared__ int scan[TC_THREADS / 32];
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int abort_flag;
    constexpr bool SPLIT = MODE == TC_SPLIT, PAIR = MODE == TC_PAIR;
    namespace cg = cooperative_groups;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = PAIR ? blockIdx.x & 1 : 0;
    const uint32_t stage_bytes = TC_A_BYTES + c.b_rows * 128;
    uint8_t * const ring = tc_mem + (1024u - (saddr(tc_mem) & 1023u)) % 1024u;
    const int e1 = p.experts + 1;
    int * const ends = reinterpret_cast<int *>(ring + size_t(c.stages) * stage_bytes), * const offs = ends + e1;      // tiles up to and with expert e, its first slot
    const uint32_t full = saddr(bars), empty = full + 8 * TC_MAX_STAGES, acc_full = empty + 8 * TC_MAX_STAGES, acc_empty = acc_full + 16, drain = acc_empty + 16;
    if (threadIdx.x == 0) {
        for (int i = 0; i < c.stages; ++i) { bar_init(full + 8 * i, 1); bar_init(empty + 8 * i, 1); }
        for (int i = 0; i < 2; ++i) { bar_init(acc_full + 8 * i, 1); bar_init(acc_empty + 8 * i, (PAIR ? 2 : 1) * TC_EPI_WARPS); }
        bar_init(drain, 1);
        bar_init_fence();
        abort_flag = 0;
        for (int m = 0; m < MATS; ++m) { prefetch_map(maps.a + m); if (p.plan) prefetch_map(maps.shared + m); }
        prefetch_map(&maps.b);
    }
    if (warp == 1) {
        if (PAIR) tmem_alloc_pair(saddr(&tmem_slot), c.tmem_cols);
        else tmem_alloc(saddr(&tmem_slot), c.tmem_cols);
    }
    fence_before();
    if (PAIR) cg::this_cluster().sync();                               // the other block's barriers are there
    else __syncthreads();
    fence_after();
    const uint32_t tmem = tmem_slot;
    grid_wait();
    grid_release();                                                    // after the wait: a down product behind this launch may read the plan above its own
    const int * counts = p.plan + PLAN_HDR, * offsets = counts + e1, * perm = offsets + e1 + 1 + e1;
    const int ne = p.shared_w[0] ? e1 : p.experts;
    int tiles = c.tiles;
    if (p.plan) {
        // inclusive prefix sums of the experts' tiles: a span of experts a thread (a call without a shared expert leaves that of the plan out)
        const int span = (ne + TC_THREADS - 1) / TC_THREADS, lo = min(ne, int(threadIdx.x) * span), hi = min(ne, lo + span);
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
        if (threadIdx.x == 0) offs[ne] = offsets[ne];
        __syncthreads();
        tiles = ends[ne - 1];
    }
    // an item: a tile of activation rows and a block (PAIR: two) of weight rows; the blocks of a pair walk the same items
    const int item_blocks = PAIR ? (c.row_blocks + 1) / 2 : c.row_blocks, it0 = PAIR ? blockIdx.x >> 1 : blockIdx.x, it_step = PAIR ? gridDim.x >> 1 : gridDim.x;
    const int items = tiles * item_blocks, all_steps = (p.cols + 127) / 128;
    const int k0 = SPLIT ? all_steps * int(blockIdx.z) / int(gridDim.z) : 0, k1 = SPLIT ? all_steps * (int(blockIdx.z) + 1) / int(gridDim.z) : all_steps;
    auto locate = [&](int it) {
        TcItem im;
        const int tile = it / item_blocks;
        im.rb = PAIR ? 2 * (it - tile * item_blocks) + rank : it - tile * item_blocks;
        im.e = 0;
        int t = tile;
        im.first = 0;
        im.count = p.n;
        if (p.plan) {
            int lo = 0, hi = ne - 1;                                   // the first expert whose tiles end behind this one
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
        const uint32_t full0 = PAIR ? at_rank(full, 0) : full;
#pragma unroll 1
        for (int it = it0; it < items && ok && !abort_flag; it += it_step) {
            const TcItem im = locate(it);
            const bool shared = p.plan && im.e == p.experts;
            const CUtensorMap * a = shared ? maps.shared : maps.a;
            const int e = shared ? 0 : im.e, boxes = PAIR ? (im.count + 2 * c.box - 1) / (2 * c.box) : (im.count + c.box - 1) / c.box;      // PAIR: of this block's half
            const int first = im.first + (PAIR ? rank * boxes * c.box : 0);
#pragma unroll 1
            for (int k = k0; k < k1; ++k) {
                if (issued >= uint32_t(c.stages) && !warp_wait(empty + 8 * slot, phase)) { ok = false; break; }
                if (lead && int(issued) != c.drop) {
                    const uint32_t bar = PAIR ? full0 + 8 * slot : full + 8 * slot, dst = saddr(ring) + slot * stage_bytes;
                    if (!PAIR || rank == 0) bar_expect_tx(full + 8 * slot, (PAIR ? 2 : 1) * (TC_A_BYTES + uint32_t(boxes * c.box) * 128));
                    if (PAIR) {
                        if (MATS == 2) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                pair_load_3d(dst + 4096 * i, a, 128 * k, 64 * im.rb + 16 * i, e, bar);
                                pair_load_3d(dst + 4096 * i + 2048, a + 1, 128 * k, 64 * im.rb + 16 * i, e, bar);
                            }
                        } else {
                            pair_load_3d(dst, a, 128 * k, 128 * im.rb, e, bar);
                        }
                        for (int i = 0; i < boxes; ++i) pair_load_2d(dst + TC_A_BYTES + i * c.box * 128, &maps.b, 128 * k, first + i * c.box, bar);
                    } else if (MATS == 2) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            tma_load_3d(dst + 4096 * i, a, 128 * k, 64 * im.rb + 16 * i, e, bar);
                            tma_load_3d(dst + 4096 * i + 2048, a + 1, 128 * k, 64 * im.rb + 16 * i, e, bar);
                        }
                    } else {
                        tma_load_3d(dst, a, 128 * k, 128 * im.rb, e, bar);
                    }
                    if (!PAIR) for (int i = 0; i < boxes; ++i) tma_load_2d(dst + TC_A_BYTES + i * c.box * 128, &maps.b, 128 * k, first + i * c.box, bar);
                }
                __syncwarp();
                ++issued;
                if (++slot == uint32_t(c.stages)) { slot = 0; phase ^= 1u; }
            }
        }
        if (!ok && lane == 0) give_up();
        // Before leaving, every copy must have landed (after a clean run these waits return at once). The barriers of a pair's copies are the even block's, which waits for those that it has
        // announced. The odd block knows that its copies have landed, and that the arrivals which the products send to its own barriers are here, when the last product of every stage has reported to
        // it; where that does not come, it leaves its copies a tenth of a second (by the SM's clock, 2 GHz at most), a thousand times what one takes.
        if (PAIR && rank == 1) {
#pragma unroll 1
            for (uint32_t i = issued > uint32_t(c.stages) ? issued - c.stages : 0; ok && i < issued; ++i) ok = warp_wait(empty + 8 * (i % c.stages), (i / c.stages) & 1u);
            if (!ok) {
                const long long begin = clock64();
                while (clock64() - begin < 200000000LL) __nanosleep(1000);
            }
        } else
#pragma unroll 1
        for (uint32_t i = issued > uint32_t(c.stages) ? issued - c.stages : 0; i < issued; ++i)
            if (int(i) != c.drop) bar_wait(full + 8 * (i % c.stages), (i / c.stages) & 1u);
    } else if (warp == 1 && rank == 0) {
        // ---- products: the whole warp walks the loop, one lane issues ----
        const bool lead = elect_one();
        const uint32_t a0 = sw128_desc_lo(saddr(ring)), step = stage_bytes >> 4;
        uint32_t slot = 0, phase = 0, done = 0;
        bool ok = true;
#pragma unroll 1
        for (int it = it0; it < items && ok && !abort_flag; it += it_step, ++done) {
            const uint32_t h = done & 1u, d = tmem + h * c.half, count = __shfl_sync(0xffffffffu, locate(it).count, 0);
            const uint32_t id = PAIR ? idesc_i8(256, (count + 2 * c.box - 1) / (2 * c.box) * (2 * c.box)) : idesc_i8(128, (count + 15) & ~15u);
            if (done >= 2 && !warp_wait(acc_empty + 8 * h, ((done >> 1) - 1) & 1u)) { ok = false; break; }
            fence_after();
#pragma unroll 1
            for (int k = k0; k < k1; ++k) {
                if (!warp_wait(full + 8 * slot, phase)) { ok = false; break; }
                fence_after();
                const uint32_t a = a0 + slot * step, b = a + (TC_A_BYTES >> 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (PAIR) mma_i8_pair(lead, d, a + 2 * i, b + 2 * i, id, k > k0 || i > 0);
                    else mma_i8(lead, d, a + 2 * i, b + 2 * i, id, k > k0 || i > 0);
                }
                if (PAIR) mma_commit_pair(lead, empty + 8 * slot);
                else mma_commit(lead, empty + 8 * slot);
                if (++slot == uint32_t(c.stages)) { slot = 0; phase ^= 1u; }
            }
            if (ok) {
                if (PAIR) mma_commit_pair(lead, acc_full + 8 * h);
                else mma_commit(lead, acc_full + 8 * h);
            }
        }
        if (!ok && lane == 0) give_up();
        // nothing may be in flight when the tensor memory is freed
        if (PAIR) mma_commit_pair(lead, drain);
        else mma_commit(lead, drain);
        warp_wait(drain, 0);
    } else if (PAIR && warp == 1) {
        warp_wait(drain, 0);                                           // the even block's last word to this one: it arrives whether or not a wait of its own ran out
    } else if (SPLIT && warp >= TC_EPI_WARP0) {
        // ---- this block's part: from tensor memory to the ring, which nothing uses any more, 128 weight rows for each activation row ----
        const int quarter = warp & 3, half = (warp - TC_EPI_WARP0) >> 2;
        const TcItem im = locate(blockIdx.x);
        if (warp_wait(acc_full, 0)) {
            fence_after();
#pragma unroll 1
            for (int col = 16 * half; col < im.count; col += 32) {
                uint32_t d[16];
                tmem_ld16(tmem + (uint32_t(32 * quarter) << 16) + col, d);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) reinterpret_cast<uint32_t *>(ring)[(col + j) * 128 + 32 * quarter + lane] = d[j];
            }
        } else if (lane == 0) {
            give_up();
        }
    } else if (!SPLIT && warp >= TC_EPI_WARP0) {
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
        const uint32_t acc_empty0 = PAIR ? at_rank(acc_empty, 0) : acc_empty;
        uint32_t done = 0;
        bool ok = true;
        TcItem im{}, next{};
        if (it0 < items) {
            next = locate(it0);
            fetch(next);
        }
#pragma unroll 1
        for (int it = it0; it < items; it += it_step, ++done) {
            const uint32_t h = done & 1u;
            im = next;
            if (tid < im.count) table[h][tid] = mine;
            float scale[MATS];
#pragma unroll
            for (int m = 0; m < MATS; ++m) scale[m] = v[m];
            epi_sync();                                                // the table is there; the other one's item has been read by every warp
            if (it + it_step < items) {
                next = locate(it + it_step);
                fetch(next);
            }
            ok = ok && !abort_flag && warp_wait(acc_full + 8 * h, (done >> 1) & 1u);
            fence_after();
            if (ok) {
                const uint32_t taddr = tmem + h * c.half + (uint32_t(32 * quarter) << 16);
                if (p.y_dtype == B2MOE_F32) store_item<MATS, float>(p, im, taddr, table[h], scale, quarter, half, lane);
                else if (p.y_dtype == B2MOE_F16) store_item<MATS, __half>(p, im, taddr, table[h], scale, quarter, half, lane);
                else store_item<MATS, __nv_bfloat16>(p, im, taddr, table[h], scale, quarter, half, lane);
            } else {
                if (lane == 0) give_up();
                const int row = weight_row<MATS>(im, quarter, lane);
                if (row < p.rows) spoil_rows(p.y, p.y_dtype, p.ldy, row, table[h], im.count, half);
            }
            fence_before();
            __syncwarp();
            if (lane == 0) {
                if (PAIR) bar_arrive_cluster(acc_empty0 + 8 * h);
                else bar_arrive(acc_empty + 8 * h);
            }
        }
    }
    fence_before();
    if (PAIR) cg::this_cluster().sync();                               // what either block sends to the other has arrived: each waited for what it was sent (above), arrivals of threads come before this
    else __syncthreads();
    fence_after();
    if (warp == 1) {
        if (PAIR) tmem_free_pair(tmem, c.tmem_cols);
        else tmem_free(tmem, c.tmem_cols);
    }
    if constexpr (SPLIT) {
        cg::cluster_group cluster = cg::this_cluster();
        const TcItem im = locate(blockIdx.x);
        const int parts = gridDim.z, lo = im.count * int(blockIdx.z) / parts, hi = im.count * (int(blockIdx.z) + 1) / parts, r = threadIdx.x & 127, row = 128 * im.rb + r;
        const bool in = row < p.rows;
        const float v = in ? p.v[0][row] : 0.f;
        uint32_t place[TC_MAX_SPLIT];
#pragma unroll
        for (int z = 0; z < TC_MAX_SPLIT; ++z) asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(place[z]) : "r"(saddr(ring) + 4 * r), "r"(z < parts ? z : 0));
        cluster.sync();
        // four activation rows of a thread at a time: a read of another block's memory takes several hundred cycles
        constexpr int STEP = TC_THREADS / 128;
        for (int col = lo + (threadIdx.x >> 7); col < hi && in; col += 4 * STEP) {
            int part[4][TC_MAX_SPLIT];
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int at = min(col + i * STEP, hi - 1);
                s[i] = p.s[im.first + at];
#pragma unroll
                for (int z = 0; z < TC_MAX_SPLIT; ++z)
                    if (z < parts) asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(part[i][z]) : "r"(place[z] + uint32_t(at) * 512u) : "memory");
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int sum = 0;
#pragma unroll
                for (int z = 0; z < TC_MAX_SPLIT; ++z)
                    if (z < parts) sum += part[i][z];
                if (col + i * STEP < hi) store_act(p.y, p.y_dtype, size_t(im.first + col + i * STEP) * p.ldy + row, float(sum) * (s[i] * v));
            }
        }
        cluster.sync();                                                // the parts stay until every block has read them
        if (abort_flag && in)                                          // and where this block has no part, what the cluster stored of the item is none
            for (int col = threadIdx.x >> 7; col < im.count; col += STEP) store_act(p.y, p.y_dtype, size_t(im.first + col) * p.ldy + row, __int_as_float(0x7fc00000));
    }
}

int sm_count() {
    static const int count = [] {                                      // the library runs on one kind of GPU
        int dev = 0, n = 0;
        return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
    }();
    return count;
}
template <class K>
int32_t launch_cluster(K kernel, dim3 grid, dim3 cluster, size_t smem, cudaStream_t s, const I8Args & p, const TcArgs & c, const TcMaps & maps) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(TC_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster.x; at[0].val.clusterDim.y = cluster.y; at[0].val.clusterDim.z = cluster.z;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = g_overlap ? 2 : 1;
    if (cudaLaunchKernelEx(&cfg, kernel, p, c, maps) != cudaSuccess) return B2MOE_ERR_CUDA;
    return launch_status();
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

// the most clusters of this many blocks that run at once (a cluster stays inside a GPC: 148 SMs hold fewer than 148 / 8 of eight)
int clusters_at_once(int size) {
    static const std::array<int, TC_MAX_SPLIT + 1> most = [] {
        std::array<int, TC_MAX_SPLIT + 1> m{};
        if (!allow_smem(i8_gemm_k<1, TC_SPLIT>, TC_SMEM_MOST)) return m;
        for (int size = 2; size <= TC_MAX_SPLIT; ++size) {
            cudaLaunchConfig_t cfg{};
            cfg.gridDim = dim3(1, 1, size); cfg.blockDim = dim3(TC_THREADS); cfg.dynamicSmemBytes = TC_SMEM_MOST;
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = 1; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = size;
            cfg.attrs = at; cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&m[size], i8_gemm_k<1, TC_SPLIT>, &cfg) != cudaSuccess) m[size] = 0;
        }
        cudaGetLastError();
        return m;
    }();
    return most[size];
}
// Blocks that share an item's columns: as many as one round of clusters has room for, with four steps of 128 columns each at least, and none where an item has fewer than 16: a step takes such a
// block 0.3 us, the meeting at the end 1.5 to 2 us and more with many rows. us, one block / this:
//              4096 x 4096    1411 x 2560    2048 x 8192    8192 x 1024 (with two)
//    16 rows   11.2 / 7.9      7.6 / 5.7     19.3 / 8.3      4.9 / 6.4
//   128 rows   13.8 / 10.0    10.1 / 7.5     22.6 / 10.3     7.1 / 9.9
int split_of(long long items, int steps) {
    int split = 1;
    for (int s = 2; s <= TC_MAX_SPLIT; ++s)
        if (steps >= 16 && s * 4 <= steps && items <= clusters_at_once(s)) split = s;
    return split;
}

// Activation rows of an item of a dense call: the rows are cut alike into the number of tiles that is expected to cost least. In steps of an item of 256 rows: a round of items takes its steps
// in proportion to 128 + rows (its weights, its rows), those that share columns meet for six of 128 rows. us, with items of 128 or 256 rows / cut alike:
//   rows of 4096 x 4096: 515 21.9 / 15.4, 1000 24.7 / 18.3, 1500 27.3 / 25.7
//   2100 rows of 1411 x 2560 17.6 / 13.0, 1500 of 4096 x 1408 17.6 / 15.0, 515 of 4096 x 512 6.4 / 5.6
int dense_rows(int n, int row_blocks, int steps, bool longer, bool two, int sms) {
    const int most = two ? 128 : 256, least = two ? 32 : 96, first = ceil_div(n, most);
    int best = most;
    float cost = 1e30f;
    for (int r = most; r >= least; r -= 16) {                          // multiples of 16, made as small as their number of tiles allows
        const int tiles = ceil_div(n, r), rows = (ceil_div(n, tiles) + 15) / 16 * 16;
        if (rows < least && tiles > first) break;
        const bool pair = longer && rows > 128;
        const long long items = (long long)ceil_div(n, rows) * (pair ? ceil_div(row_blocks, 2) : row_blocks), at_once = pair ? sms / 2 : two ? 2 * sms : sms;
        const int split = split_of((long long)ceil_div(n, rows) * row_blocks, steps);
        const float each = float(128 + (pair ? (rows + 63) / 64 * 64 : rows)) / 384.f;
        const float c = split > 1 ? float(steps) / split * each + 6.f * rows / 128.f : float((items + at_once - 1) / at_once) * steps * each;
        if (c < cost) { cost = c; best = rows; }
    }
    return best;
}

}  // namespace

void i8_drop_step(int step) { g_drop_step = step; }
bool i8_gemm_supported(int experts) { return experts <= TC_MAX_EXPERTS; }

template <int MATS>
int32_t i8_gemm(const I8Args & p, long long q_rows, int per_group, int * status, cudaStream_t s) {
    TcArgs c{};
    c.row_blocks = ceil_div(p.rows, MATS == 2 ? 64 : 128);
    // The shape of a launch, by the columns and the rows that an item will have. Times in us.
    // Items of 256 rows halve what the weights cost in copies and products; items of 128 leave room for six ring stages instead of four and waste less where an expert has fewer. 256 / 128:
    //   dense 8192 rows of 4096 x 4096                96 / 150
    //   gate/up, 512 experts at 80 rows each         225 / 211
    //   gate/up, 128 experts at 128 each, skewed     333 / 385
    // (64 rows gain nothing further: 248 against 242 with 128, at 16 each.)
    // Pairs pay from long rows on, where the products of an item outlast what its blocks tell each other. Single / pair:
    //   dense 8192 rows of 4096 x 4096              96.5 / 87.1      of 4096 x 2048    59.6 / 60.3      of 4096 x 1024    49.1 / 53.6      of 8192 x 8192    378.6 / 353.0
    //   gate/up, 128 experts of 4096 columns, at 16 each 248.5 (items of 128) / 246.2, at 160 344.9 / 326.2, at 320 613 / 584
    //   gate/up, 512 experts of 2048 columns, at 160 each 304 / 318      down, 512 of 512 columns at 80 each 193 / 242
    // Short rows: two blocks an SM with half the ring each. An item of a few steps takes longer from its first copy to its last store than its copies alone, and one block's items hide behind the
    // other's. One / two:
    //   down, 512 experts of 512 columns, at one row each 76 / 60, at 80 192 / 178, at 320 650 / 498; of 768 columns at 40 64 / 67
    //   gate/up of 512 columns at 8 each 107 / 78, of 2048 columns at 80 242 / 258
    //   dense 8192 rows of 4096 x 512 44 / 36, of 4096 x 1024 49 / 42
    const int sms = sm_count();
    const bool longer = p.cols > 2560, two = p.cols <= I8_SHORT_COLS;
    if (p.plan) c.nt = two ? 128 : per_group > 96 || longer ? 256 : 128;
    else c.nt = dense_rows(p.n, c.row_blocks, ceil_div(p.cols, 128), longer, two, sms);
    c.tiles = p.plan ? 0 : ceil_div(p.n, c.nt);
    // A dense call with few items: as many blocks an item as run at once
    const int split = MATS == 1 && !p.plan ? split_of((long long)c.tiles * c.row_blocks, ceil_div(p.cols, 128)) : 1;
    const bool pair = split == 1 && longer && c.nt > 128;
    c.box = pair || two ? 32 : 64;                                     // rows of a copy: an item takes as many copies as it has rows for
    c.tmem_cols = 32;
    while (c.tmem_cols < 2 * uint32_t(c.nt)) c.tmem_cols *= 2;
    c.b_rows = (pair ? ceil_div(c.nt, 2 * c.box) : ceil_div(c.nt, c.box)) * c.box;
    const size_t stage_bytes = TC_A_BYTES + size_t(c.b_rows) * 128;
    c.half = c.tmem_cols / 2;
    c.status = status;
    c.drop = g_drop_step;
    const size_t table = p.plan ? size_t(2 * (p.experts + 1) + 1) * sizeof(int) : 0;
    c.stages = int(std::min<size_t>(TC_MAX_STAGES, ((two ? TC_SMEM / 2 : TC_SMEM) - TC_FIXED - table) / stage_bytes));
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
    const size_t smem = TC_ALIGN + size_t(c.stages) * stage_bytes + table;
    const long long items = (long long)c.tiles * c.row_blocks;
    if constexpr (MATS == 1)
        if (split > 1) {
            if (!allow_smem(i8_gemm_k<1, TC_SPLIT>, TC_SMEM_MOST)) return B2MOE_ERR_CUDA;
            return launch_cluster(i8_gemm_k<1, TC_SPLIT>, dim3(unsigned(items), 1, split), dim3(1, 1, split), smem, s, p, c, maps);
        }
    if (pair) {
        if (!allow_smem(i8_gemm_k<MATS, TC_PAIR>, TC_SMEM_MOST)) return B2MOE_ERR_CUDA;
        const long long pairs = (long long)c.tiles * ceil_div(c.row_blocks, 2);
        return launch_cluster(i8_gemm_k<MATS, TC_PAIR>, dim3(unsigned(2 * (p.plan ? sms / 2 : std::min<long long>(sms / 2, pairs)))), dim3(2), smem, s, p, c, maps);
    }
    if (!allow_smem(i8_gemm_k<MATS, 0>, TC_SMEM_MOST)) return B2MOE_ERR_CUDA;
    const int blocks = two ? 2 * sms : sms;
    launch_overlapped(i8_gemm_k<MATS, 0>, dim3(unsigned(p.plan ? blocks : std::min<long long>(blocks, items))), dim3(TC_THREADS), smem, s, p, c, maps);
    return launch_status();
}
template int32_t i8_gemm<1>(const I8Args &, long long, int, int *, cudaStream_t);
template int32_t i8_gemm<2>(const I8Args &, long long, int, int *, cudaStream_t);

}  // namespace b2
