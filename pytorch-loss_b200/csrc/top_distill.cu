// Distillation from a teacher's best alternatives: a row of the student's logits against a short list of tokens with
// log probabilities q.
//     w = softmax of q over the list      loss = sum_k w_k (log w_k - log p_k)      dloss/dx_j = (p_j - w_j) / T
// (w_j: the sum over the list's entries with token j).  Entries with a negative token do not exist; a row without
// any mass is not read, costs nothing and counts for nothing in a mean.
//
// distill_lists_kernel turns the lists into weights once (one warp per row), the other kernels take these.  The
// training step ('mean' / 'sum') holds the row in shared memory -- split over the blocks of a cluster where it is
// longer than one block's share -- and reads the logits once; without it the statistics kernel and the gradient
// kernel of token_stats.cuh read them once each.
#include "token_stats.cuh"

namespace b200 {
namespace {

constexpr int kListSlots = 512;             // blocks of the list kernel, at most: each counts its rows
constexpr int kStepThreads = 512;
constexpr size_t kStepShare = 64 * 1024;    // bytes of a row per block where eight blocks suffice
constexpr size_t kStepMost = 200 * 1024;    // beyond: two passes

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

__global__ void __launch_bounds__(256) distill_lists_kernel(const int64_t *tokens, const float *q, float *weight,
                                                            float *base, int *counts, int64_t rows, int K, int V) {
    __shared__ int ids[8][kMaxList];
    __shared__ float ws[8][kMaxList];
    __shared__ int valid_rows[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int valid = 0;
    for (int64_t r = int64_t(blockIdx.x) * 8 + warp; r < rows; r += int64_t(gridDim.x) * 8) {
        float x[kMaxList / 32];
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
            ids[warp][i] = id >= 0 && id < V ? int(id) : -1;
            best = max_nan(best, x[e]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max_nan(best, __shfl_xor_sync(0xffffffffu, best, o));
        bad = __any_sync(0xffffffffu, bad);
        const bool nothing = best == -INFINITY && !bad;
        float total = 0.f;
#pragma unroll
        for (int e = 0; e < kMaxList / 32; ++e) total += x[e] == -INFINITY ? 0.f : expf(x[e] - best);
        total = warp_sum(total);
        const float log_total = logf(total);
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < kMaxList / 32; ++e) {
            const float lw = x[e] - best - log_total;
            const float w = x[e] == -INFINITY ? 0.f : expf(x[e] - best) / total;
            if (w > 0.f || w != w) sum += w * lw;
            ws[warp][lane + 32 * e] = ids[warp][lane + 32 * e] < 0 ? 0.f : w;
        }
        sum = warp_sum(sum);
        __syncwarp();
        // entries with the same token: the first one carries the weight of all
        for (int e = 0; e * 32 < K; ++e) {
            const int i = lane + 32 * e;
            if (i >= K) break;
            const int id = ids[warp][i];
            float w = 0.f;
            bool first = id >= 0;
            for (int j = 0; j < K; ++j)
                if (ids[warp][j] == id) {
                    first = first && j >= i;
                    w += ws[warp][j];
                }
            weight[r * K + i] = first ? w : 0.f;
        }
        if (lane == 0) base[r] = bad ? __int_as_float(0x7fc00000) : nothing ? INFINITY : sum;
        valid += nothing ? 0 : 1;
        __syncwarp();
    }
    if (lane == 0) valid_rows[warp] = valid;
    __syncthreads();
    if (threadIdx.x == 0) {
        int n = 0;
        for (int w = 0; w < 8; ++w) n += valid_rows[w];
        counts[blockIdx.x] = n;
    }
    if (blockIdx.x == 0)
        for (int i = int(gridDim.x) + int(threadIdx.x); i < kListSlots; i += 256) counts[i] = 0;
}

// record = {sum of the losses, number of rows that have one, mean, sum}: one block, so the order is always the same.
__global__ void __launch_bounds__(1024) distill_finish_kernel(const float *losses, const int *counts, int64_t rows,
                                                              ReduceRecord *out) {
    __shared__ double sh[64];
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
    int V, K, parts;
    float c, inv_t;
    const int64_t *ids;
    const float *weight, *base;
    const int *counts;          // the rows of a mean, in kListSlots parts; null: a sum
    float *losses;
};

// One row per cluster of `parts` blocks; each block's part of it is copied to shared memory once (bulk copy), read
// twice there (statistics, gradient), and the gradient leaves as 16-byte stores.
// Bound: HBM, 2 x the logits' bytes; two exponentials an element and the joins between the blocks come next.
template <typename T>
__global__ void __launch_bounds__(kStepThreads) distill_step_kernel(const StepParams p) {
    namespace cg = cooperative_groups;
    constexpr int N = TokenVec<T>::N, WARPS = kStepThreads / 32;
    extern __shared__ __align__(16) uint4 held[];
    __shared__ uint64_t full;
    __shared__ float wm[WARPS], wsum[WARPS], joined[2];
    __shared__ int wcount[WARPS];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int rank = int(blockIdx.x % unsigned(p.parts));
    const int64_t r = int64_t(blockIdx.x / unsigned(p.parts));
    const T *row = static_cast<const T *>(p.x) + r * p.stride;
    T *g = static_cast<T *>(p.grad) + r * int64_t(p.V);
    const RowPart part = row_part(row, p.V, rank, p.parts);
    const float base = p.base[r];
    if (base == INFINITY) {                                 // (all blocks of the cluster)
        for (int i = part.body + t * N; i < part.body_end; i += kStepThreads * N)
            st_stream16(g + i, make_uint4(0u, 0u, 0u, 0u));
        if (t < ragged_count(part)) g[ragged_index(part, t)] = from_f32<T>(0.f);
        if (rank == 0 && t == 0) p.losses[r] = 0.f;
        return;
    }
    const int n = part.body_end - part.body;
    if (t == 0) {
        mbar_init(&full, 1);
        fence_mbar_init();
        if (n > 0) {
            const uint32_t bytes = uint32_t(n) * uint32_t(sizeof(T));
            mbar_expect_tx(&full, bytes);
            bulk_load_1d(held, row + part.body, bytes, &full);
        }
    }
    __syncthreads();
    int count = p.counts && t < kListSlots ? p.counts[t] : 0;
    count = __reduce_add_sync(0xffffffffu, count);
    const bool arrived = n == 0 || mbar_wait_bounded(&full, 0, nullptr);

    RowStat<false> st;
    st.init();
    auto load = [&](int i) { return held[(i - part.body) / N]; };
    if (arrived) scan_part<T, kStepThreads>(row, part, t, p.c, st, load);
    else st.m = __int_as_float(0x7fc00000);                 // (a copy that never came shows as NaN)
    st.join_warp(p.c);
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
    if (p.parts > 1) {
        if (t == 0) {
            joined[0] = st.m;
            joined[1] = st.s;
        }
        cluster.sync();
        st.init();
        if (lane < p.parts) {
            const float *other = cluster.map_shared_rank(&joined[0], lane);
            st.m = other[0];
            st.s = other[1];
        }
        st.join_warp(p.c);
        cluster.barrier_arrive();                           // (this block has read what it needs)
    }

    const float m = reference_of(st.m);
    const bool nothing = st.s == 0.f;
    float scale = p.inv_t;
    if (p.counts) scale /= float(count);
    if (base != base) scale = base;
    const float A = nothing ? 0.f : scale / st.s;
    auto one = [&](float v) { return ex2f(max_nan((v - m) * p.c, kTokenFloor)) * A; };
    const pk_t negm = psplat(-m), cc = psplat(p.c), aa = psplat(A);
    for (int i = part.body + t * N; i < part.body_end; i += kStepThreads * N) {
        const uint4 v = load(i);
        float2 d[N / 2];
#pragma unroll
        for (int h = 0; h < N / 2; ++h) {
            float2 z = upk2(pmul(padd(pk2(TokenVec<T>::pair(v, h)), negm), cc));
            z.x = max_nan(z.x, kTokenFloor);
            z.y = max_nan(z.y, kTokenFloor);
            d[h] = upk2(pmul(pex2(pk2(z)), aa));
        }
        st_stream16(g + i, TokenVec<T>::pack(d));
    }
    if (t < ragged_count(part)) {
        const int j = ragged_index(part, t);
        g[j] = from_f32<T>(one(to_f32(row[j])));
    }
    __syncthreads();                                        // (what the list changes has been written)
    float loss = 0.f;
    for (int i = t; i < p.K; i += kStepThreads) {
        const float w = p.weight[r * p.K + i];
        if (w > 0.f) {
            const int64_t j = p.ids[r * p.K + i];
            const float x = to_f32(row[j]);
            if (j >= part.first && j < part.last && !nothing) g[j] = from_f32<T>(fmaf(-scale, w, one(x)));
            loss = fmaf(-w, nothing ? -INFINITY : log_prob(x, m, p.inv_t, log2f(st.s)), loss);
        }
    }
    if (rank == 0) {                                        // (the list lies in the first four warps)
        loss = warp_sum(loss);
        if (lane == 0) wm[warp] = loss;
        __syncthreads();
        if (t == 0) p.losses[r] = base + (wm[0] + wm[1]) + (wm[2] + wm[3]);
    }
    if (p.parts > 1) cluster.barrier_wait();                // (nobody leaves while its memory is read)
}

inline int step_parts(int64_t V, int dtype) {
    const size_t bytes = size_t(V) * dtype_size(dtype);
    int parts = 1;
    while (parts < kMaxCluster && bytes > kStepShare * parts) parts *= 2;
    return bytes <= kStepMost * parts ? parts : 0;
}

template <typename T> int launch_step(const StepParams &p, cudaStream_t stream) {
    const size_t vectors = (size_t(p.V) * sizeof(T) / 16 + p.parts - 1) / p.parts;
    const size_t bytes = vectors * 16 + 16;
    if (const int rc = set_smem(distill_step_kernel<T>, bytes)) return rc;
    return launch_cluster(distill_step_kernel<T>, p.rows * p.parts, kStepThreads, bytes, p.parts, false, stream,
                          "distillation step kernel launch", p);
}

int launch_lists(const int64_t *tokens, const float *q, const DistillScratch &d, int64_t rows, int K, int V,
                 cudaStream_t stream) {
    int64_t grid = (rows + 7) / 8;
    grid = grid < 1 ? 1 : grid > kListSlots ? kListSlots : grid;
    distill_lists_kernel<<<unsigned(grid), 256, 0, stream>>>(tokens, q, d.weight, d.base, d.counts, rows, K, V);
    return launch_status("distillation list kernel launch");
}

int check_distill(const char *who, const void *x, const int64_t *tokens, const void *scratch, size_t scratch_bytes,
                  int64_t rows, int64_t V, int64_t stride, int dtype, int K, float temperature) {
    if (const int rc = check_rows(who, x, rows, V, stride, dtype, temperature)) return rc;
    if (K < 1 || K > kMaxList) {
        set_error("%s: lists of 1 to %d tokens", who, kMaxList);
        return B200_ERR_ARG;
    }
    if (rows > 0 && !tokens) {
        set_error("%s: null pointer", who);
        return B200_ERR_ARG;
    }
    if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15) || scratch_bytes < b200_top_distill_scratch_bytes(rows, K)) {
        set_error("%s: scratch of %zu bytes on a 16-byte address required", who, b200_top_distill_scratch_bytes(rows, K));
        return B200_ERR_WORKSPACE;
    }
    return B200_OK;
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
    if ((rows > 0 && !top_logprobs) || (!losses && !out)) {
        set_error("%s: null pointer", who);
        return B200_ERR_ARG;
    }
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
    distill_finish_kernel<<<1, 1024, 0, s>>>(p.out, d.counts, rows, static_cast<ReduceRecord *>(out));
    return launch_status("distillation sum kernel launch");
}

extern "C" int b200_top_distill_backward(const void *logits, const int64_t *top_tokens, const void *scratch,
                                         size_t scratch_bytes, const float *d_loss, int per_row, const void *count,
                                         void *grad_logits, int64_t rows, int64_t V, int64_t stride, int dtype, int K,
                                         float temperature, void *stream) {
    const char *who = "b200_top_distill_backward";
    if (const int rc = check_distill(who, logits, top_tokens, scratch, scratch_bytes, rows, V, stride, dtype, K, temperature))
        return rc;
    if ((rows > 0 && (!d_loss || !grad_logits)) || (reinterpret_cast<uintptr_t>(count) & 7) ||
        (reinterpret_cast<uintptr_t>(grad_logits) & (dtype_size(dtype) - 1))) {
        set_error("%s: null or misaligned pointer", who);
        return B200_ERR_ARG;
    }
    const DistillScratch d = carve(const_cast<void *>(scratch), rows);
    TokenGradParams p{};
    p.x = logits;
    p.grad = grad_logits;
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
    return step_parts(V, dtype) > 0;
}

extern "C" int b200_top_distill_step(const void *logits, const int64_t *top_tokens, const float *top_logprobs,
                                     void *grad_logits, void *out, void *scratch, size_t scratch_bytes, int64_t rows,
                                     int64_t V, int64_t stride, int dtype, int K, float temperature, int mean,
                                     void *stream) {
    const char *who = "b200_top_distill_step";
    if (const int rc = check_distill(who, logits, top_tokens, scratch, scratch_bytes, rows, V, stride, dtype, K, temperature))
        return rc;
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
    p.parts = step_parts(V, dtype);
    p.c = float(1.4426950408889634 / double(temperature));
    p.inv_t = 1.f / temperature;
    p.ids = top_tokens;
    p.weight = d.weight;
    p.base = d.base;
    p.counts = mean ? d.counts : nullptr;
    p.losses = d.losses;
    const int rc = dtype == B200_F32 ? launch_step<float>(p, s) : launch_step<__nv_bfloat16>(p, s);
    if (rc) return rc;
    distill_finish_kernel<<<1, 1024, 0, s>>>(d.losses, d.counts, rows, static_cast<ReduceRecord *>(out));
    return launch_status("distillation sum kernel launch");
}
