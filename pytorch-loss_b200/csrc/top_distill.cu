// Distillation from a teacher's best alternatives: a row of the student's logits against a short list of tokens with
// log probabilities q.
//     w = softmax of q over the list      loss = sum_k w_k (log w_k - log p_k)      dloss/dx_j = (p_j - w_j) / T
// (w_j: the sum over the list's entries with token j).  Entries with a negative token do not exist; a row without
// any mass is not read, costs nothing and counts for nothing in a mean.
//
// distill_lists_kernel turns the lists into weights once (one warp per row), the other kernels take these.  The
// training step ('mean' / 'sum') reads the logits from memory once; without it the statistics kernel and the gradient
// kernel of token_stats.cuh read them once each.
#include "token_stats.cuh"

namespace b200 {
namespace {

constexpr int kListWarps = 16;              // rows of a block of the list kernel
constexpr int kListSlots = 512;             // blocks of the list kernel, at most: each counts its rows
constexpr size_t kStepHeld = 72 * 1024;     // longest row that a block holds: three blocks on an SM
constexpr int kStepPieces = 16;             // of 8 KB (128 threads) or 16 KB (256)

// Scratch: the blocks' row counts, then per row statistics, sum of w log w, loss and weights.
struct DistillScratch {
    int *counts;
    float4 *stats;
    float *base, *losses, *weight;
};
constexpr size_t kScratchHead = kListSlots * 4;
inline DistillScratch carve(void *scratch, int64_t rows) {
    char *at = static_cast<char *>(scratch);
    DistillScratch d;
    d.counts = reinterpret_cast<int *>(at);
    d.stats = reinterpret_cast<float4 *>(at + kScratchHead);
    d.base = reinterpret_cast<float *>(d.stats + rows);
    d.losses = d.base + rows;
    d.weight = d.losses + rows;
    return d;
}

__global__ void __launch_bounds__(32 * kListWarps) distill_lists_kernel(const int64_t *tokens, const float *q, float *weight,
                                                            float *base, int *counts, int64_t rows, int K, int V) {
    static_assert(kMaxList == 128, "four entries a lane");
    __shared__ __align__(16) int ids[kListWarps][kMaxList];
    __shared__ float ws[kListWarps][kMaxList];
    __shared__ int valid_rows[kListWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();                                // (the kernel behind takes its place on the SMs meanwhile)
    int valid = 0;
    for (int64_t r = int64_t(blockIdx.x) * kListWarps + warp; r < rows; r += int64_t(gridDim.x) * kListWarps) {
        float x[kMaxList / 32], w[kMaxList / 32];
        int own[kMaxList / 32];
        float best = -INFINITY;
        bool bad = false;
#pragma unroll
        for (int e = 0; e < kMaxList / 32; ++e) {
            const int i = lane + 32 * e;
            int64_t id = -1;
            x[e] = -INFINITY;
            if (i < K) {
                id = tokens[r * K + i];
                if (id >= 0) x[e] = q[r * K + i];
                bad = bad || id >= V;
            }
            own[e] = id >= 0 && id < V ? int(id) : -1;
            ids[warp][i] = own[e];
            best = max_nan(best, x[e]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max_nan(best, __shfl_xor_sync(0xffffffffu, best, o));
        bad = __any_sync(0xffffffffu, bad);
        const bool nothing = best == -INFINITY && !bad;
        float total = 0.f;
#pragma unroll
        for (int e = 0; e < kMaxList / 32; ++e) {
            if (32 * e >= K) break;
            x[e] = x[e] == -INFINITY ? -INFINITY : x[e] - best;
            w[e] = x[e] == -INFINITY ? 0.f : expf(x[e]);
            total += w[e];
        }
        total = warp_sum(total);
        const float log_total = logf(total);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < kMaxList / 32; ++e) {
            if (32 * e >= K) break;
            w[e] /= total;
            if (w[e] > 0.f || w[e] != w[e]) sum += w[e] * (x[e] - log_total);
            ws[warp][lane + 32 * e] = own[e] < 0 ? 0.f : w[e];
        }
        sum = warp_sum(sum);
        __syncwarp();
        // the same token twice?  Rare: only looked for here
        int meets[kMaxList / 32] = {};
        for (int j = 0; j < K; j += 4) {
            const int4 four = *reinterpret_cast<const int4 *>(&ids[warp][j]);
#pragma unroll
            for (int e = 0; e < kMaxList / 32; ++e) {
                if (32 * e >= K) break;
                meets[e] += (four.x == own[e]) + (four.y == own[e]) + (four.z == own[e]) + (four.w == own[e]);
            }
        }
        int twins = 0;                                      // (every entry meets itself)
#pragma unroll
        for (int e = 0; e < kMaxList / 32; ++e) twins += own[e] >= 0 && meets[e] > 1 ? 1 : 0;
        const bool merge = __any_sync(0xffffffffu, twins > 0);
        for (int e = 0; e * 32 < K; ++e) {
            const int i = lane + 32 * e;
            if (i >= K) break;
            float sum_w = ws[warp][i];
            if (merge) {                                    // the first of such entries carries the weight of all
                const int id = ids[warp][i];
                bool first = id >= 0;
                sum_w = 0.f;
                for (int j = 0; j < K; ++j)
                    if (ids[warp][j] == id) {
                        first = first && j >= i;
                        sum_w += ws[warp][j];
                    }
                if (!first) sum_w = 0.f;
            }
            weight[r * K + i] = sum_w;
        }
        if (lane == 0) base[r] = bad ? __int_as_float(0x7fc00000) : nothing ? INFINITY : sum;
        valid += nothing ? 0 : 1;
        __syncwarp();
    }
    if (lane == 0) valid_rows[warp] = valid;
    __syncthreads();
    if (threadIdx.x == 0) {
        int n = 0;
        for (int w = 0; w < kListWarps; ++w) n += valid_rows[w];
        counts[blockIdx.x] = n;
    }
    if (blockIdx.x == 0)
        for (int i = int(gridDim.x) + int(threadIdx.x); i < kListSlots; i += 32 * kListWarps) counts[i] = 0;
}

// record = {sum of the losses, number of rows that have one, mean, sum}: one block, so the order is always the same.
__global__ void __launch_bounds__(1024) distill_finish_kernel(const float *losses, const int *counts, int64_t rows,
                                                              ReduceRecord *out) {
    __shared__ double sh[64];
    pdl_wait();
    double sum = 0.0, count = threadIdx.x < kListSlots ? double(counts[threadIdx.x]) : 0.0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) sum += double(losses[i]);
    block_sum2(sum, count, sh);
    if (threadIdx.x == 0) {
        out->sum = sum;
        out->count = count;
        out->mean = float(sum / count);
        out->sum32 = float(sum);
        out->pad[0] = 0.f;
        out->pad[1] = 0.f;
    }
}

struct StepParams {
    const void *x;
    void *grad;
    int64_t stride, rows;
    int V, K, part_shift;       // 2^part_shift blocks of a cluster share a row
    float c, inv_t;
    const int64_t *ids;
    const float *weight, *base;
    const int *counts;          // the rows of a mean, in kListSlots parts; null: a sum
    float *losses;
    float4 *stats;              // what the gradient needs if it has to be written again
};

// One row per block (HELD: copied to shared memory once, in pieces, and read twice there) or per cluster of up to two
// blocks (read twice, the second time from L2).  The gradient leaves as 16-byte stores, and what the list changes is
// written once more behind them.
// Bound: HBM, 2 x the logits' bytes; two exponentials an element and the joins between the blocks come next.
template <typename T, int THREADS, bool HELD>
__global__ void __launch_bounds__(THREADS) distill_step_kernel(const StepParams p) {
    namespace cg = cooperative_groups;
    constexpr int N = TokenVec<T>::N, WARPS = THREADS / 32;
    extern __shared__ __align__(16) uint4 held[];
    __shared__ uint64_t full[kStepPieces];
    __shared__ float wm[WARPS], wsum[WARPS], wloss[WARPS], joined[3], of_row[2];
    __shared__ int wcount[WARPS];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int parts = 1 << p.part_shift, rank = int(blockIdx.x) & (parts - 1);
    const int64_t r = int64_t(blockIdx.x >> p.part_shift);
    const T *row = static_cast<const T *>(p.x) + r * p.stride;
    T *g = static_cast<T *>(p.grad) + r * int64_t(p.V);
    const RowPart part = row_part(row, p.V, rank, p.part_shift);
    pdl_wait();                                             // (the lists' kernel)
    const float base = p.base[r];
    ListShare<T, THREADS> list;
    list.load(p.ids + r * p.K, p.weight + r * p.K, p.K, t);
    int count = 0;
    if (p.counts && t < kListSlots / 4) {
        const int4 four = reinterpret_cast<const int4 *>(p.counts)[t];
        count = (four.x + four.y) + (four.z + four.w);
    }
    if (base == INFINITY) {                                 // (all blocks of the cluster)
        for (int i = part.body + t * N; i < part.body_end; i += THREADS * N)
            st_stream16(g + i, make_uint4(0u, 0u, 0u, 0u));
        if (t < ragged_count(part)) g[ragged_index(part, t)] = from_f32<T>(0.f);
        if (rank == 0 && t == 0) p.losses[r] = 0.f;
        return;
    }
    // (pieces of as many vectors as a step of all threads takes: work begins with the first)
    constexpr int PIECE = kTokenUnroll * THREADS * N;
    if (HELD) {
        if (t == 0) {
            for (int i = 0; i < kStepPieces; ++i) mbar_init(&full[i], 1);
            fence_mbar_init();
            for (int i = 0; part.body + i * PIECE < part.body_end; ++i) {
                const int n = min(PIECE, part.body_end - part.body - i * PIECE);
                mbar_expect_tx(&full[i], uint32_t(n) * uint32_t(sizeof(T)));
                bulk_load_1d(held + i * (PIECE / N), row + part.body + i * PIECE, uint32_t(n) * uint32_t(sizeof(T)), &full[i]);
            }
        }
        __syncthreads();
    }
    list.fetch(part, row);

    RowStat<false> st;
    st.init();
    bool arrived = true;
    auto load = [&](int i) { return HELD ? held[(i - part.body) / N] : *reinterpret_cast<const uint4 *>(row + i); };
    scan_part<T, THREADS>(row, part, t, p.c, st, load, [](int, float) {}, [&](int k) {
        if (HELD && arrived) arrived = mbar_wait_bounded(&full[k / kTokenUnroll], 0, nullptr);
    });
    if (!arrived) st.m = __int_as_float(0x7fc00000);        // (a copy that never came shows as NaN)
    st.join_warp(p.c);
    count = __reduce_add_sync(0xffffffffu, count);
    if (lane == 0) {
        wm[warp] = st.m;
        wsum[warp] = st.s;
        wcount[warp] = count;
    }
    __syncthreads();
    st.init();
    count = 0;
    if (lane < WARPS) {
        st.m = wm[lane];
        st.s = wsum[lane];
        count = wcount[lane];
    }
    st.join_warp(p.c);
    count = __reduce_add_sync(0xffffffffu, count);
    cg::cluster_group cluster = cg::this_cluster();
    if (parts > 1) {
        if (t == 0) {
            joined[0] = st.m;
            joined[1] = st.s;
        }
        cluster.sync();
        st.init();
        if (lane < parts) {
            const float *other = cluster.map_shared_rank(&joined[0], lane);
            st.m = other[0];
            st.s = other[1];
        }
        st.join_warp(p.c);
    }

    const float m = reference_of(st.m), log2s = log2f(st.s);
    const bool nothing = st.s == 0.f;
    if (t == 0) {                                           // (out of the registers that the loop below wants)
        of_row[0] = m;
        of_row[1] = st.s;
    }
    float scale = p.inv_t;
    if (p.counts) scale /= float(count);
    if (base != base) scale = base;
    const float A = nothing ? 0.f : scale / st.s;
    auto one = [&](float v) { return ex2f((v - m) * p.c) * A; };
    const pk_t negm = psplat(-m), cc = psplat(p.c), aa = psplat(A);
    const int vectors = (part.body_end - part.body) / N;
    const uint4 *src = (HELD ? held : reinterpret_cast<const uint4 *>(row + part.body)) + t;
    T *dst = g + part.body + t * N;
    auto gradient = [&](const uint4 &v, T *to) {
        float2 d[N / 2];
#pragma unroll
        for (int h = 0; h < N / 2; ++h)
            d[h] = upk2(pmul(pex2(pmul(padd(pk2(TokenVec<T>::pair(v, h)), negm), cc)), aa));
        st_stream16(to, TokenVec<T>::pack(d));
    };
    int i = t;
    for (; i + 3 * THREADS < vectors; i += 4 * THREADS, src += 4 * THREADS, dst += 4 * THREADS * N) {
        uint4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = src[k * THREADS];
#pragma unroll
        for (int k = 0; k < 4; ++k) gradient(v[k], dst + k * THREADS * N);
    }
    for (; i < vectors; i += THREADS, src += THREADS, dst += THREADS * N) gradient(*src, dst);
    if (t < ragged_count(part)) {
        const int j = ragged_index(part, t);
        g[j] = from_f32<T>(one(to_f32(row[j])));
    }
    // each block's part of the loss: sum over its part of the list
    float loss = 0.f;
#pragma unroll
    for (int i = 0; i < list.N; ++i)
        if (list.w[i] > 0.f) loss = fmaf(-list.w[i], nothing ? -INFINITY : log_prob(list.x[i], m, p.inv_t, log2s), loss);
    loss = warp_sum(loss);
    if (lane == 0) wloss[warp] = loss;
    __syncthreads();                                        // (what the list changes has been written, too)
#pragma unroll
    for (int i = 0; i < list.N; ++i)
        if (list.w[i] > 0.f && !nothing) g[list.id[i]] = from_f32<T>(fmaf(-scale, list.w[i], one(list.x[i])));
    if (t == 0) {
        loss = 0.f;
        for (int i = 0; i < WARPS; ++i) loss += wloss[i];
        joined[2] = loss;
    }
    if (parts > 1) {
        cluster.sync();
        if (rank == 0 && t == 0) {
            for (int i = 1; i < parts; ++i) loss += cluster.map_shared_rank(&joined[0], i)[2];
        }
        cluster.sync();                                     // (nobody leaves while its memory is read)
    }
    if (rank == 0 && t == 0) {
        const float s = of_row[1];
        p.losses[r] = base + loss;
        p.stats[r] = make_float4(of_row[0], s == 0.f ? 0.f : 1.f / s, 0.f, log2f(s));
    }
}

// Behind a bfloat16 step: its gradient for an upstream gradient other than 1, from the logits and what the step left.  As
// many bytes as scaling the written gradient would move, but one rounding.  A grid of what runs at once goes through the
// chunks, so that it costs 2 us to find that the upstream gradient is 1.
__global__ void __launch_bounds__(256) distill_again_kernel(const TokenGradParams p, unsigned chunks) {
    if (*p.d_out == 1.f) return;
    for (unsigned i = blockIdx.x; i < chunks; i += gridDim.x) {
        token_grad_chunk<__nv_bfloat16, 256, kList, true>(p, i);
        __syncthreads();                                    // (the chunk's list is in shared memory)
    }
}

// How a step treats a row.  Measured (us, lists of 20; two passes: statistics, then gradient):
//   [16384, 4096] bfloat16 (8 KB)     held by 128 threads 73, by 256 104     two passes 99     from L2 169
//   [16384, 16384] bfloat16 (32 KB)   185, 185                               261               247
//   [16384, 32768] bfloat16 (64 KB)   404, 367                               501               391
//   [8192, 24000] float32 (96 KB)     (two blocks on an SM) 322              357               257
//   [8192, 65536] bfloat16 (128 KB)                                          487               408, by two blocks 462
//   [3000, 50001] float32 (200 KB)                                           281               274, by two blocks 240
//   [4096, 131072] bfloat16 (256 KB)                                         479               488, by two blocks 408
//   [2048, 81920] float32 (320 KB)                                           312               311, by two blocks 287
//   [2048, 131072] float32 (512 KB)                                          478               532, by two blocks 529
// With few rows a step leaves SMs idle where two passes split the rows, but both are short of what the host needs for the
// call: [8, 80000] bfloat16 11 against 8, [148, 80000] 14 against 21, [8, 32768] 8 against 8.
// Rows off the gradient's place within 16 bytes have no step: [8192, 50257] bfloat16 with rows of 50304 482 against 302.
// From L2 works while the rows under way fit there (three blocks of 512 threads an SM: 57 MB at 128 KB, where 12 % of
// the rows are read from memory twice).  What the step loses there it loses to its phases: a block reads, joins, writes.
enum StepWay { kNoStep, kHeld128, kHeld256, kFromL2, kFromL2Pair };
inline StepWay step_way(int64_t V, int dtype) {
    const int64_t bytes = V * int64_t(dtype_size(dtype));
    return bytes <= 4096                ? kNoStep
           : bytes <= 16 * 1024         ? kHeld128
           : bytes <= int64_t(kStepHeld) ? kHeld256
           : bytes <= 160 * 1024        ? kFromL2
           : bytes <= 320 * 1024        ? kFromL2Pair
                                        : kNoStep;
}

template <typename T, int THREADS> int launch_held(const StepParams &p, const char *what, cudaStream_t stream) {
    const size_t bytes = size_t(p.V) * sizeof(T) / 16 * 16;
    if (const int rc = set_smem(distill_step_kernel<T, THREADS, true>, bytes)) return rc;
    return launch_cluster(distill_step_kernel<T, THREADS, true>, p.rows, THREADS, bytes, 1, true, stream, what, p);
}
template <typename T> int launch_step(StepParams p, int dtype, cudaStream_t stream) {
    const char *what = "distillation step kernel launch";
    const StepWay way = step_way(p.V, dtype);
    if (way == kHeld128) return launch_held<T, 128>(p, what, stream);
    if (way == kHeld256) return launch_held<T, 256>(p, what, stream);
    p.part_shift = way == kFromL2Pair ? 1 : 0;
    return launch_cluster(distill_step_kernel<T, 512, false>, p.rows << p.part_shift, 512, 0, 1 << p.part_shift, true,
                          stream, what, p);
}

int launch_finish(const float *losses, const int *counts, int64_t rows, void *out, cudaStream_t stream) {
    return launch_cluster(distill_finish_kernel, 1, 1024, 0, 1, true, stream, "distillation sum kernel launch", losses, counts,
                          rows, static_cast<ReduceRecord *>(out));
}

int launch_lists(const int64_t *tokens, const float *q, const DistillScratch &d, int64_t rows, int K, int V,
                 cudaStream_t stream) {
    int64_t grid = (rows + kListWarps - 1) / kListWarps;
    grid = grid < 1 ? 1 : grid > kListSlots ? kListSlots : grid;
    distill_lists_kernel<<<unsigned(grid), 32 * kListWarps, 0, stream>>>(tokens, q, d.weight, d.base, d.counts, rows, K, V);
    return launch_status("distillation list kernel launch");
}

int check_distill(const char *who, const void *x, const int64_t *tokens, const void *scratch, size_t scratch_bytes,
                  int64_t rows, int64_t V, int64_t stride, int dtype, int K, float temperature) {
    if (const int rc = check_rows(who, x, rows, V, stride, dtype, temperature)) return rc;
    if (K < 1 || K > kMaxList) {
        set_error("%s: lists of 1 to %d tokens", who, kMaxList);
        return B200_ERR_ARG;
    }
    if (rows > 0 && (!tokens || !lies_on(tokens, 8))) {
        set_error("%s: null or misaligned pointer", who);
        return B200_ERR_ARG;
    }
    if (!scratch || !lies_on(scratch, 16) || scratch_bytes < b200_top_distill_scratch_bytes(rows, K)) {
        set_error("%s: scratch of %zu bytes on a 16-byte address required", who, b200_top_distill_scratch_bytes(rows, K));
        return B200_ERR_WORKSPACE;
    }
    return B200_OK;
}

TokenGradParams grad_params(const void *logits, const int64_t *top_tokens, const void *scratch, const float *d_loss, int per_row,
                            const void *count, void *grad, int64_t rows, int64_t V, int64_t stride, int K, float temperature) {
    const DistillScratch d = carve(const_cast<void *>(scratch), rows);
    TokenGradParams p{};
    p.x = logits;
    p.grad = grad;
    p.stride = stride;
    p.rows = rows;
    p.V = int(V);
    p.inv_t = 1.f / temperature;
    p.c = float(1.4426950408889634 / double(temperature));
    p.ids = top_tokens;
    p.weight = d.weight;
    p.base = d.base;
    p.stats = d.stats;
    p.d_out = d_loss;
    p.d_out_step = per_row ? 1 : 0;
    p.count = static_cast<const double *>(count);
    p.K = K;
    return p;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" size_t b200_top_distill_scratch_bytes(int64_t rows, int K) {
    if (rows < 0 || K < 0) return 0;
    return kScratchHead + size_t(rows) * (16 + 4 + 4 + 4 * size_t(K));
}

extern "C" int b200_top_distill_forward(const void *logits, const int64_t *top_tokens, const float *top_logprobs,
                                        float *losses, void *out, void *scratch, size_t scratch_bytes, int64_t rows,
                                        int64_t V, int64_t stride, int dtype, int K, float temperature, void *stream) {
    const char *who = "b200_top_distill_forward";
    if (const int rc = check_distill(who, logits, top_tokens, scratch, scratch_bytes, rows, V, stride, dtype, K, temperature))
        return rc;
    if ((rows > 0 && (!top_logprobs || (!losses && !out))) || !lies_on(top_logprobs, 4) || !lies_on(losses, 4) ||
        !lies_on(out, 8)) {
        set_error("%s: null or misaligned pointer", who);
        return B200_ERR_ARG;
    }
    if (rows == 0 && !out) return B200_OK;                  // (no rows' losses: an empty tensor has no address)
    const DistillScratch d = carve(scratch, rows);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (const int rc = launch_lists(top_tokens, top_logprobs, d, rows, K, int(V), s)) return rc;
    TokenParams p{};
    p.x = logits;
    p.stride = stride;
    p.rows = rows;
    p.V = int(V);
    p.inv_t = 1.f / temperature;
    p.c = float(1.4426950408889634 / double(temperature));
    p.ids = top_tokens;
    p.weight = d.weight;
    p.base = d.base;
    p.K = K;
    p.out = losses ? losses : d.losses;
    p.stats = d.stats;
    const int rc = dtype == B200_F32   ? launch_stats<float, kList, false>(p, dtype, s)
                   : dtype == B200_F16 ? launch_stats<__half, kList, false>(p, dtype, s)
                                       : launch_stats<__nv_bfloat16, kList, false>(p, dtype, s);
    if (rc || !out) return rc;
    return launch_finish(p.out, d.counts, rows, out, s);
}

extern "C" int b200_top_distill_backward(const void *logits, const int64_t *top_tokens, const void *scratch,
                                         size_t scratch_bytes, const float *d_loss, int per_row, const void *count,
                                         void *grad_logits, int64_t rows, int64_t V, int64_t stride, int dtype, int K,
                                         float temperature, void *stream) {
    const char *who = "b200_top_distill_backward";
    if (const int rc = check_distill(who, logits, top_tokens, scratch, scratch_bytes, rows, V, stride, dtype, K, temperature))
        return rc;
    if ((rows > 0 && (!d_loss || !grad_logits)) || !lies_on(count, 8) || !lies_on(d_loss, 4) ||
        !lies_on(grad_logits, dtype_size(dtype))) {
        set_error("%s: null or misaligned pointer", who);
        return B200_ERR_ARG;
    }
    const TokenGradParams p = grad_params(logits, top_tokens, scratch, d_loss, per_row, count, grad_logits, rows, V, stride, K,
                                          temperature);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return dtype == B200_F32   ? launch_grad<float, kList>(p, dtype, s)
           : dtype == B200_F16 ? launch_grad<__half, kList>(p, dtype, s)
                               : launch_grad<__nv_bfloat16, kList>(p, dtype, s);
}

extern "C" int b200_top_distill_step_path(const void *logits, const void *grad_logits, int64_t rows, int64_t V,
                                          int64_t stride, int dtype) {
    if (rows < 1 || rows > 0x0fffffff || V < 1 || V > (int64_t(1) << 30) || (dtype != B200_F32 && dtype != B200_BF16))
        return 0;
    if (((reinterpret_cast<uintptr_t>(logits) - reinterpret_cast<uintptr_t>(grad_logits)) & 15) != 0) return 0;
    if (rows > 1 && ((stride - V) * int64_t(dtype_size(dtype))) % 16 != 0) return 0;
    return step_way(V, dtype) != kNoStep;
}

extern "C" int b200_top_distill_step(const void *logits, const int64_t *top_tokens, const float *top_logprobs,
                                     void *grad_logits, void *out, void *scratch, size_t scratch_bytes, int64_t rows,
                                     int64_t V, int64_t stride, int dtype, int K, float temperature, int mean,
                                     void *stream) {
    const char *who = "b200_top_distill_step";
    if (const int rc = check_distill(who, logits, top_tokens, scratch, scratch_bytes, rows, V, stride, dtype, K, temperature))
        return rc;
    if (!lies_on(top_logprobs, 4) || !lies_on(out, 8)) {
        set_error("%s: misaligned pointer", who);
        return B200_ERR_ARG;
    }
    if (!top_logprobs || !grad_logits || !out || !b200_top_distill_step_path(logits, grad_logits, rows, V, stride, dtype)) {
        set_error("%s: these logits have no one-pass step", who);
        return B200_ERR_UNSUPPORTED;
    }
    const DistillScratch d = carve(scratch, rows);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (const int rc = launch_lists(top_tokens, top_logprobs, d, rows, K, int(V), s)) return rc;
    StepParams p{};
    p.x = logits;
    p.grad = grad_logits;
    p.stride = stride;
    p.rows = rows;
    p.V = int(V);
    p.K = K;
    p.c = float(1.4426950408889634 / double(temperature));
    p.inv_t = 1.f / temperature;
    p.ids = top_tokens;
    p.weight = d.weight;
    p.base = d.base;
    p.counts = mean ? d.counts : nullptr;
    p.losses = d.losses;
    p.stats = d.stats;
    const int rc = dtype == B200_F32 ? launch_step<float>(p, dtype, s) : launch_step<__nv_bfloat16>(p, dtype, s);
    if (rc) return rc;
    return launch_finish(d.losses, d.counts, rows, out, s);
}

extern "C" int b200_top_distill_step_backward(const void *logits, const int64_t *top_tokens, const void *scratch,
                                              size_t scratch_bytes, const float *d_loss, const void *count,
                                              void *grad_logits, int64_t rows, int64_t V, int64_t stride, int dtype, int K,
                                              float temperature, void *stream) {
    const char *who = "b200_top_distill_step_backward";
    if (const int rc = check_distill(who, logits, top_tokens, scratch, scratch_bytes, rows, V, stride, dtype, K, temperature))
        return rc;
    if (!d_loss || !lies_on(d_loss, 4) || !lies_on(count, 8)) {
        set_error("%s: null or misaligned pointer", who);
        return B200_ERR_ARG;
    }
    if (dtype != B200_BF16 || !grad_logits || !b200_top_distill_step_path(logits, grad_logits, rows, V, stride, dtype)) {
        set_error("%s: need bfloat16 logits that have a one-pass step", who);
        return B200_ERR_UNSUPPORTED;
    }
    TokenGradParams p = grad_params(logits, top_tokens, scratch, d_loss, 0, count, grad_logits, rows, V, stride, K, temperature);
    p.chunks = grad_chunks(row_vectors(V, dtype));
    const int64_t chunks = rows * p.chunks, most = int64_t(sm_count()) * 6;
    if (chunks > 0x7fffffff) {
        set_error("%s: %lld rows of %d logits are more than one launch covers", who, (long long)rows, p.V);
        return B200_ERR_UNSUPPORTED;
    }
    return launch_cluster(distill_again_kernel, chunks < most ? chunks : most, 256, 0, 1, false,
                          static_cast<cudaStream_t>(stream), "distillation gradient kernel launch", p, unsigned(chunks));
}
