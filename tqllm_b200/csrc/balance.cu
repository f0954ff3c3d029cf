// The balance loss of a routed batch, the counts per expert and sequence that it is made of, and its gradient on the logits.
//
//   p_te = softmax over experts of u_te,  u = the logit (softmax gating) or log sigmoid of it (sigmoid gating: the scores divided by their sum)
//   c_se = assignments of sequence s to expert e,  T_s = its unmasked tokens,  P_se = sum_t p_te / T_s
//   L = coef / S+ * sum_s E / (k T_s) * sum_e c_se P_se                       (S+: sequences with T_s > 0)
//   dL/dl_tj = g coef / S+ * E / (k T_s^2) * p_tj (c_sj - sum_e p_te c_se) * (1 | 1 - sigmoid(l_tj))
// The p_te of a token add up to one, so any number may be taken off the c_se. The gradient takes off their least: what is left stays positive and no larger than it was, an even load
// has a gradient of zero instead of the rounding of the sum, and a nearly even one, which the loss makes for, loses fewer bits to the difference.
//
// The batch is cut into chunks of tokens that lie in one sequence each. Chunk j of sequence s has the number offsets[s] / chunk + s + j: the
// numbers of two sequences never meet (a sequence of len tokens has at most ceil(len / chunk) <= floor((offsets[s] + len) / chunk) - floor(offsets[s] / chunk) + 1
// chunks), so a block finds its chunk from the offsets alone, without a scan and without the host knowing them. Each chunk leaves the sums of its
// rows of probabilities and its counts in the workspace; a second launch adds them up in a fixed order, so that a batch gives the same bits every time.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "common.cuh"

namespace b2 {
namespace {

constexpr int ALONE_THREADS = 512, BAL_THREADS = 256, BAL_WARPS = BAL_THREADS / 32, BAL_MAX_EXPERTS = 4096, SUM_COLS = 32, SUM_ROWS = 16, SUM_ASK = 8;

struct BalArgs {
    const float * logits;
    int ld;
    const int * ids;
    int topk;
    const uint8_t * mask;
    const int * offsets;             // [sequences + 1], or null: one sequence of all n tokens
    int sequences, experts, n, chunk, chunks;
    float coef;
    float * part_prob;               // [chunks][experts]
    int * part_count;                // [chunks][experts]
    int * part_tokens;               // [chunks]
    float * dots;                    // [sequences][slices of SUM_COLS experts]
    int * ticket;
    float * loss, * prob;
    int * counts, * tokens;          // tokens: [sequences + 1], the last one S+
};

// the tokens [lo, hi) of sequence s: inside the batch whatever the offsets hold
__device__ __forceinline__ int2 span_of(const int * offsets, int s, int n) {
    if (!offsets) return make_int2(0, n);
    const int lo = min(max(offsets[s], 0), n);
    return make_int2(lo, max(lo, min(offsets[s + 1], n)));
}
// the block's chunk: (sequence, first token, end), sequence -1 where the number belongs to none
__device__ __forceinline__ int3 find_chunk(const int * offsets, int sequences, int n, int chunk, int at) {
    __shared__ int3 found;
    if (threadIdx.x == 0) found = make_int3(-1, 0, 0);
    __syncthreads();
    for (int s = threadIdx.x; s < sequences; s += blockDim.x) {
        const int2 w = span_of(offsets, s, n);
        const int j = at - (w.x / chunk + s), t0 = w.x + j * chunk;
        if (j >= 0 && t0 < w.y) found = make_int3(s, t0, min(w.y, t0 + chunk));
    }
    __syncthreads();
    return found;
}

// One row of scores in registers: V values a lane, G warps a row (value i of lane l of the row's warp w is expert 32 G i + 32 w + l).
template <int V, int G>
struct Row {
    float v[V];                                                        // probabilities (after scores())
    float * red;                                                       // G > 1: the block's reduction words
    int first;

    __device__ __forceinline__ float all(float x, bool largest) {
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            const float y = __shfl_xor_sync(0xffffffffu, x, d);
            x = largest ? fmaxf(x, y) : x + y;
        }
        if (G > 1) {
            const int w = threadIdx.x >> 5;
            __syncthreads();                                           // the words of the reduction before have been read
            if ((threadIdx.x & 31) == 0) red[w] = x;
            __syncthreads();
            x = red[w / G * G];
#pragma unroll
            for (int i = 1; i < G; ++i) x = largest ? fmaxf(x, red[w / G * G + i]) : x + red[w / G * G + i];
        }
        return x;
    }
    // the least of whole numbers, as all()
    __device__ __forceinline__ int least(int x) {
        x = __reduce_min_sync(0xffffffffu, x);
        if (G > 1) {
            const int w = threadIdx.x >> 5;
            int * words = reinterpret_cast<int *>(red);
            __syncthreads();
            if ((threadIdx.x & 31) == 0) words[w] = x;
            __syncthreads();
            x = words[w / G * G];
#pragma unroll
            for (int i = 1; i < G; ++i) x = min(x, words[w / G * G + i]);
        }
        return x;
    }
    // logits -> p; slope[i] = 1 - sigmoid(l) where the gating is the sigmoid one. A row without a finite score (all -inf) gives zeros.
    template <bool SIGMOID, bool SLOPE>
    __device__ __forceinline__ void scores(const float * logits, int experts, float (&slope)[SLOPE ? V : 1]) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = first + 32 * G * i;
            v[i] = e < experts ? logits[e] : -INFINITY;
            top = fmaxf(top, v[i]);
        }
        top = all(top, true);
        // below -60 a sigmoid is the exponential to 26 digits, and quotients of exponentials do not underflow with their largest taken out
        const bool exponential = !SIGMOID || top < -60.f;
        const float shift = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float l = v[i];
            if (SIGMOID) {
                const float a = expf(-fabsf(l)), r = 1.f / (1.f + a);
                if (SLOPE) slope[SLOPE ? i : 0] = l >= 0.f ? a * r : r;
                v[i] = exponential ? expf(l - shift) : l >= 0.f ? r : a * r;
            } else {
                v[i] = expf(l - shift);
            }
            sum += v[i];
        }
        sum = all(sum, false);
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] *= inv;
    }
};

// Bound by reading the logits once. A warp (four from 513 experts on) holds a row in registers: one read, the softmax's maximum and sum by shuffles, and the
// column sums of a warp's rows stay in registers until the chunk is through.
// ALONE: a batch of one sequence and a few tokens is one block's, which writes the results itself.
template <int V, int G, bool SIGMOID, bool ALONE>
__global__ void __launch_bounds__(ALONE ? ALONE_THREADS : BAL_THREADS) balance_rows_k(const BalArgs p) {
    extern __shared__ float cols[];                                    // [WARPS / G][experts], then the counters; ALONE: the counters behind them
    constexpr int THREADS = ALONE ? ALONE_THREADS : BAL_THREADS, WARPS = THREADS / 32;
    __shared__ float red[WARPS];
    grid_release();
    grid_wait();
    int3 c;
    if (ALONE) {
        const int2 w = span_of(p.offsets, 0, p.n);
        c = make_int3(0, w.x, w.y);
    } else {
        c = find_chunk(p.offsets, p.sequences, p.n, p.chunk, blockIdx.x);
        if (blockIdx.x == 0 && threadIdx.x == 0) *p.ticket = 0;
        if (c.x < 0) return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / G;
    constexpr int ROWS = WARPS / G;
    Row<V, G> row;
    row.red = red;
    row.first = (warp % G) * 32 + lane;
    float acc[V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 1
    for (int t0 = c.y; t0 < c.z; t0 += ROWS) {                         // every warp walks the same number of steps: with G > 1 they hold barriers
        const int t = t0 + group;
        const bool live = t < c.z && !(p.mask && !p.mask[t]);
        if (G == 1 && !live) continue;
        float none[1];
        row.template scores<SIGMOID, false>(p.logits + size_t(live ? t : c.y) * p.ld, p.experts, none);
        if (live) {
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] += row.v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (row.first + 32 * G * i < p.experts) cols[size_t(group) * p.experts + row.first + 32 * G * i] = acc[i];
    __syncthreads();
    if (!ALONE) {
        for (int e = threadIdx.x; e < p.experts; e += THREADS) {
            float sum = cols[e];
#pragma unroll
            for (int i = 1; i < ROWS; ++i) sum += cols[size_t(i) * p.experts + e];
            p.part_prob[size_t(blockIdx.x) * p.experts + e] = sum;
        }
        __syncthreads();
    }
    int * hist = reinterpret_cast<int *>(cols) + (ALONE ? ROWS * p.experts : 0);
    for (int e = threadIdx.x; e < p.experts; e += THREADS) hist[e] = 0;
    __syncthreads();
    for (long long i = (long long)c.y * p.topk + threadIdx.x; i < (long long)c.z * p.topk; i += THREADS) {
        const int id = p.ids[i];
        if (id >= 0 && id < p.experts && !(p.mask && !p.mask[i / p.topk])) atomicAdd(&hist[id], 1);      // whole numbers: any order gives the same
    }
    const int mine = c.y + int(threadIdx.x);                           // a chunk has fewer tokens than the block threads
    const int tokens = __syncthreads_count(mine < c.z && !(p.mask && !p.mask[mine]));
    if (ALONE) {
        float dot = 0.f;
        for (int e = threadIdx.x; e < p.experts; e += THREADS) {
            float sum = cols[e];
#pragma unroll
            for (int i = 1; i < ROWS; ++i) sum += cols[size_t(i) * p.experts + e];
            const float mean = tokens ? sum / float(tokens) : 0.f;
            p.prob[e] = mean;
            p.counts[e] = hist[e];
            dot += float(hist[e]) * mean;
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (lane == 0) red[warp] = dot;
        __syncthreads();
        if (threadIdx.x == 0) {
            dot = 0.f;
            for (int w = 0; w < WARPS; ++w) dot += red[w];
            p.tokens[0] = tokens;
            p.tokens[1] = tokens > 0;
            *p.loss = tokens ? float(double(p.coef) * p.experts / p.topk * (double(dot) / double(tokens))) : 0.f;
        }
        return;
    }
    if (threadIdx.x == 0) p.part_tokens[blockIdx.x] = tokens;
    for (int e = threadIdx.x; e < p.experts; e += THREADS) p.part_count[size_t(blockIdx.x) * p.experts + e] = hist[e];
}

// One block per sequence and SUM_COLS experts adds the chunks up; the last block of all adds the sequences.
__global__ void __launch_bounds__(SUM_COLS * SUM_ROWS) balance_sum_k(const BalArgs p) {
    __shared__ float sp[SUM_ROWS][SUM_COLS];
    __shared__ int sc[SUM_ROWS][SUM_COLS], st[SUM_ROWS];
    __shared__ bool last;
    grid_release();
    grid_wait();
    const int s = blockIdx.y, lane = threadIdx.x & 31, r = threadIdx.x >> 5, e = blockIdx.x * SUM_COLS + lane;
    const int2 w = span_of(p.offsets, s, p.n);
    const int first = w.x / p.chunk + s, count = (w.y - w.x + p.chunk - 1) / p.chunk;
    float prob = 0.f;
    int c = 0, tokens = 0;
    const bool in = e < p.experts;
    const float * pp = p.part_prob + size_t(first) * p.experts + e;
    const int * pc = p.part_count + size_t(first) * p.experts + e;
    for (int j0 = r; j0 < count; j0 += SUM_ROWS * SUM_ASK) {           // the loads of several chunks together
        float f[SUM_ASK];
        int n[SUM_ASK], k[SUM_ASK];
#pragma unroll
        for (int i = 0; i < SUM_ASK; ++i) {
            const int j = j0 + i * SUM_ROWS;
            f[i] = in && j < count ? pp[size_t(j) * p.experts] : 0.f;
            n[i] = in && j < count ? pc[size_t(j) * p.experts] : 0;
            k[i] = j < count ? p.part_tokens[first + j] : 0;
        }
#pragma unroll
        for (int i = 0; i < SUM_ASK; ++i) { prob += f[i]; c += n[i]; tokens += k[i]; }
    }
    sp[r][lane] = prob;
    sc[r][lane] = c;
    if (lane == 0) st[r] = tokens;
    __syncthreads();
    if (r == 0) {
        tokens = 0;
        prob = 0.f;
        c = 0;
#pragma unroll
        for (int i = 0; i < SUM_ROWS; ++i) { prob += sp[i][lane]; c += sc[i][lane]; tokens += st[i]; }
        const float mean = tokens ? prob / float(tokens) : 0.f;
        if (e < p.experts) {
            p.prob[size_t(s) * p.experts + e] = mean;
            p.counts[size_t(s) * p.experts + e] = c;
        }
        float dot = e < p.experts ? float(c) * mean : 0.f;
#pragma unroll
        for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (lane == 0) {
            p.dots[size_t(s) * gridDim.x + blockIdx.x] = dot;
            if (blockIdx.x == 0) p.tokens[s] = tokens;
            __threadfence();
            last = atomicAdd(p.ticket, 1) == int(gridDim.x * gridDim.y) - 1;
        }
    }
    __syncthreads();
    if (!last) return;
    __threadfence();
    // sequences in a fixed order: lane i of the first warp takes i, i + 32, ...; then a tree over the lanes
    if (threadIdx.x >= 32) return;
    double sum = 0.0;
    int filled = 0;
    for (int q = lane; q < p.sequences; q += 32) {
        const int t = __ldcg(p.tokens + q);
        if (t == 0) continue;
        ++filled;
        float dot = 0.f;
        for (int x = 0; x < int(gridDim.x); ++x) dot += __ldcg(p.dots + size_t(q) * gridDim.x + x);
        sum += double(dot) / double(t);
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, d);
        filled += __shfl_xor_sync(0xffffffffu, filled, d);
    }
    if (lane == 0) {
        p.tokens[p.sequences] = filled;
        *p.loss = filled ? float(double(p.coef) * p.experts / p.topk / filled * sum) : 0.f;
    }
}

struct BalBackArgs {
    const float * logits;
    int ld, topk;
    const uint8_t * mask;
    const int * offsets;
    int sequences, experts, n, chunk;
    float coef;
    const int * counts, * tokens;
    const float * grad_loss;
    float * grad;
    int ldg, accumulate;
};
// The logits once more (the loss keeps no probabilities: n x experts of them would be written and read in their place), and the gradient.
template <int V, int G, bool SIGMOID>
__global__ void __launch_bounds__(BAL_THREADS) balance_backward_k(const BalBackArgs p) {
    __shared__ float red[BAL_WARPS];
    grid_release();
    grid_wait();
    if (p.offsets && !p.accumulate) {                                  // rows in front of the first sequence and behind the last have no part in the loss
        const int lo = min(max(p.offsets[0], 0), p.n), hi = min(max(p.offsets[p.sequences], lo), p.n);
        for (int t = blockIdx.x; t < p.n - (hi - lo); t += gridDim.x)
            for (int e = threadIdx.x; e < p.experts; e += BAL_THREADS) p.grad[size_t(t < lo ? t : t + hi - lo) * p.ldg + e] = 0.f;
    }
    const int3 c = find_chunk(p.offsets, p.sequences, p.n, p.chunk, blockIdx.x);
    if (c.x < 0) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp / G;
    constexpr int ROWS = BAL_WARPS / G;
    Row<V, G> row;
    row.red = red;
    row.first = (warp % G) * 32 + lane;
    const float tokens = float(p.tokens[c.x]);
    const float factor = (p.grad_loss ? *p.grad_loss : 1.f) * p.coef / float(max(p.tokens[p.sequences], 1)) * float(p.experts) / (float(p.topk) * tokens * tokens);
    // what the counts have more than the least, from whole numbers: 32-bit floats do not hold counts from 2^24 on
    int count[V], least = INT_MAX;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = row.first + 32 * G * i;
        count[i] = e < p.experts ? p.counts[size_t(c.x) * p.experts + e] : INT_MAX;
        least = min(least, count[i]);
    }
    least = row.least(least);
    float weight[V];
#pragma unroll
    for (int i = 0; i < V; ++i) weight[i] = row.first + 32 * G * i < p.experts ? float(count[i] - least) : 0.f;
#pragma unroll 1
    for (int t0 = c.y; t0 < c.z; t0 += ROWS) {
        const int t = t0 + group;
        const bool inside = t < c.z, live = inside && !(p.mask && !p.mask[t]);
        if (G == 1 && !inside) break;
        float * out = p.grad + size_t(inside ? t : c.y) * p.ldg;
        if (G == 1 && !live) {
            if (!p.accumulate)
                for (int e = lane; e < p.experts; e += 32) out[e] = 0.f;
            continue;
        }
        float slope[SIGMOID ? V : 1];
        row.template scores<SIGMOID, SIGMOID>(p.logits + size_t(live ? t : c.y) * p.ld, p.experts, slope);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) dot += row.v[i] * weight[i];
        dot = row.all(dot, false);
        if (!inside) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = row.first + 32 * G * i;
            if (e >= p.experts) break;
            float g = live ? row.v[i] * (weight[i] - dot) * factor : 0.f;
            if (SIGMOID && live) g *= slope[SIGMOID ? i : 0];
            if (p.accumulate) { if (live) out[e] += g; }
            else out[e] = g;
        }
    }
}

// Tokens per chunk: eight (one a warp) while that makes at most two blocks an SM, then what two blocks an SM leave, up to 128: the second launch
// reads a row of the workspace for each chunk.
inline int bal_chunk(int n) { return 8 * std::min(16, std::max(1, ceil_div(n, 148 * 2 * 8))); }
inline long long bal_chunks(int n, int sequences) { return n / bal_chunk(n) + (long long)sequences; }

template <template <int, int, bool> class K, class Args>
int32_t launch_rows(const Args & a, int gating, long long chunks, int threads, size_t (*smem)(int, int), cudaStream_t s) {
    auto go = [&](auto v, auto g) {
        constexpr int V = decltype(v)::value, G = decltype(g)::value;
        const size_t bytes = smem(a.experts, G);
        if (gating == B2MOE_SIGMOID) launch_overlapped(K<V, G, true>::fn(), dim3(unsigned(chunks)), dim3(threads), bytes, s, a);
        else launch_overlapped(K<V, G, false>::fn(), dim3(unsigned(chunks)), dim3(threads), bytes, s, a);
        return launch_status();
    };
    using std::integral_constant;
    const int e = a.experts;
    if (e <= 32) return go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    if (e <= 64) return go(integral_constant<int, 2>{}, integral_constant<int, 1>{});
    if (e <= 128) return go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    if (e <= 256) return go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    if (e <= 512) return go(integral_constant<int, 16>{}, integral_constant<int, 1>{});
    if (e <= 1024) return go(integral_constant<int, 8>{}, integral_constant<int, 4>{});
    if (e <= 2048) return go(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    return go(integral_constant<int, 32>{}, integral_constant<int, 4>{});
}
template <int V, int G, bool S> struct RowsKernel { static auto fn() { return balance_rows_k<V, G, S, false>; } };
template <int V, int G, bool S> struct AloneKernel { static auto fn() { return balance_rows_k<V, G, S, true>; } };
template <int V, int G, bool S> struct BackKernel { static auto fn() { return balance_backward_k<V, G, S>; } };

struct BalSpace { size_t prob, count, tokens, dots, ticket, total; };
BalSpace bal_space(int experts, int n, int sequences) {
    BalSpace w{};
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at = align_up(at + bytes, 256); return o; };
    // room for the chunks of eight tokens, whatever the chunk is: the size grows with n (the number of chunks does not)
    const size_t chunks = std::min<size_t>(size_t(n) / 8, 148 * 2 + size_t(n) / 128) + sequences + 1;
    w.prob = take(chunks * experts * sizeof(float));
    w.count = take(chunks * experts * sizeof(int));
    w.tokens = take(chunks * sizeof(int));
    w.dots = take(size_t(sequences) * ceil_div(experts, SUM_COLS) * sizeof(float));
    w.ticket = take(sizeof(int));
    w.total = at;
    return w;
}
int32_t bal_check(int gating, int ld, int topk, const int32_t * offsets, int sequences, int experts, int n) {
    if (gating != B2MOE_SOFTMAX && gating != B2MOE_SIGMOID) return B2MOE_ERR_SHAPE;
    if (n <= 0 || experts <= 0 || experts > BAL_MAX_EXPERTS || topk <= 0 || topk > experts || ld < experts) return B2MOE_ERR_SHAPE;
    if (sequences <= 0 || sequences > 65535 || (!offsets && sequences != 1) || (long long)n * topk > 0x3fffffffLL) return B2MOE_ERR_SHAPE;
    return B2MOE_OK;
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" B2MOE_API size_t b2moe_balance_workspace_bytes(int32_t experts, int32_t n, int32_t sequences) {
    if (experts <= 0 || experts > BAL_MAX_EXPERTS || n <= 0 || sequences <= 0 || sequences > 65535) return 0;
    return bal_space(experts, n, sequences).total;
}

extern "C" B2MOE_API int32_t b2moe_balance_loss(int32_t gating, const float * logits, int32_t ld, const int32_t * ids, int32_t topk, const uint8_t * mask,
                                                const int32_t * offsets, int32_t sequences, int32_t experts, int32_t n, float coef, float * loss,
                                                int32_t * counts, float * prob, int32_t * tokens, void * workspace, size_t workspace_bytes,
                                                b2moe_stream stream) {
    if (int32_t rc = bal_check(gating, ld, topk, offsets, sequences, experts, n)) return rc;
    if (!logits || !ids || !loss || !counts || !prob || !tokens || !workspace) return B2MOE_ERR_NULL;
    if (!aligned16(workspace) || !aligned_to(logits, 4) || !aligned_to(ids, 4) || !aligned_to(offsets, 4) || !aligned_to(loss, 4) || !aligned_to(counts, 4) || !aligned_to(prob, 4) ||
        !aligned_to(tokens, 4)) return B2MOE_ERR_ALIGN;
    const BalSpace w = bal_space(experts, n, sequences);
    if (workspace_bytes < w.total) return B2MOE_ERR_WORKSPACE;
    char * base = static_cast<char *>(workspace);
    const long long chunks = bal_chunks(n, sequences);
    const BalArgs a{logits, ld, ids, topk, mask, offsets, sequences, experts, n, bal_chunk(n), int(chunks), coef,
                    reinterpret_cast<float *>(base + w.prob), reinterpret_cast<int *>(base + w.count), reinterpret_cast<int *>(base + w.tokens),
                    reinterpret_cast<float *>(base + w.dots), reinterpret_cast<int *>(base + w.ticket), loss, prob, counts, tokens};
    cudaStream_t s = as_stream(stream);
    // one launch in place of two: 48 tokens of 32 experts, loss and gradient 12.4 -> 8.3 us (the launch alone 4.6 us with eight warps, 3.6 with sixteen). Four rows a warp at most; the counters fit behind the sums up to 2048 experts
    if (sequences == 1 && n <= 64 && experts <= 2048)
        return launch_rows<AloneKernel>(a, gating, 1, ALONE_THREADS, [](int e, int g) { return size_t(ALONE_THREADS / 32 / g + 1) * e * sizeof(float); }, s);
    if (int32_t rc = launch_rows<RowsKernel>(a, gating, chunks, BAL_THREADS, [](int e, int g) { return size_t(BAL_WARPS / g) * e * sizeof(float); }, s)) return rc;
    launch_overlapped(balance_sum_k, dim3(ceil_div(experts, SUM_COLS), sequences), dim3(SUM_COLS * SUM_ROWS), 0, s, a);
    return launch_status();
}

extern "C" B2MOE_API int32_t b2moe_balance_loss_backward(int32_t gating, const float * logits, int32_t ld, int32_t topk, const uint8_t * mask,
                                                         const int32_t * offsets, int32_t sequences, int32_t experts, int32_t n, float coef,
                                                         const int32_t * counts, const int32_t * tokens, const float * grad_loss, float * grad_logits,
                                                         int32_t ldg, int32_t accumulate, b2moe_stream stream) {
    if (int32_t rc = bal_check(gating, ld, topk, offsets, sequences, experts, n)) return rc;
    if (ldg < experts) return B2MOE_ERR_SHAPE;
    if (!logits || !counts || !tokens || !grad_logits) return B2MOE_ERR_NULL;
    if (!aligned_to(logits, 4) || !aligned_to(offsets, 4) || !aligned_to(counts, 4) || !aligned_to(tokens, 4) || !aligned_to(grad_loss, 4) || !aligned_to(grad_logits, 4)) return B2MOE_ERR_ALIGN;
    const BalBackArgs a{logits, ld, topk, mask, offsets, sequences, experts, n, bal_chunk(n), coef, counts, tokens, grad_loss, grad_logits, ldg, accumulate};
    return launch_rows<BackKernel>(a, gating, bal_chunks(n, sequences), BAL_THREADS, [](int, int) { return size_t(0); }, as_stream(stream));
}
