// Layer norm over rows of D contiguous elements, forward and backward.
//     mean, var of the row      r = 1 / sqrt(var + eps)      h = (x - mean) r      y = h w + b
//     g = dy w     dx = r (g - mean(g) - h mean(g h))     dw = sum over rows of dy h     db = sum over rows of dy
// Statistics, h and all sums are float32; a result is rounded once.
//
// The variance is the mean square of x - mean, taken from registers after the mean is known: no difference of large
// squares.  Backward recomputes h from x and the row's {mean, r} (8 bytes a row).  dw and db: a thread keeps the same
// columns for all its rows, in registers; each block leaves one partial row, which norm_columns_kernel adds up in
// block order, so results repeat bit for bit.
//
// Bound: HBM (2 s D per row forward, 3 s D backward, s the element's bytes).  Measured, us and share of the 6.55 TB/s of
// a copy:  [16384, 4096] bfloat16, float32 weights   50 (0.82) + 80 (0.77)     [16384, 8192] float16   90 (0.91) + 151 (0.81)
//          [32768, 2048] float32                     81 (1.01) + 137 (0.90)    [16384, 4001] float32   92 (0.87) + 150 (0.80)
//          [4096, 12288] bfloat16                    39 (0.78) + 113 (0.41)    [8192, 16384] float32  226 (0.73) + 309 (0.80)
// Beyond 8192 columns backward waits for a cluster's barrier in every row (2 us).  16-bit rows that are not whole vectors
// go element by element ([16384, 4001] float16 89 (0.45) + 139 (0.43)), forward rows beyond 64 KB in three sweeps
// ([1024, 40000] bfloat16 84, 0.30).
#include <algorithm>

#include "token_rows.cuh"

namespace b200 {
namespace {

struct NormParams {
    const void *x, *w, *b, *dy;
    void *y, *dx;
    float2 *stats;              // {mean, r} per row
    float *partial;             // [blocks][2][D]
    int64_t x_stride, dy_stride, rows;
    int D, stages;
    int blocks, share;          // blocks of a cluster that share a row, and columns of each (the last one: what is left)
    float eps;
};
constexpr int kMaxSlots = 8;
constexpr size_t kRingBytes = 200 * 1024;     // of an SM's shared memory

// V elements of T as floats.
template <typename T, int V> __device__ __forceinline__ void load_pack(const T *p, float (&f)[V]) {
    if constexpr (V * sizeof(T) >= 16) {
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < V / E; ++i) {
            const Vec16<T> t = *reinterpret_cast<const Vec16<T> *>(p + i * E);
#pragma unroll
            for (int k = 0; k < E; ++k) f[i * E + k] = to_f32(t.v[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) f[k] = to_f32(p[k]);
    }
}
template <typename T, int V> __device__ __forceinline__ void store_pack(T *p, const float (&f)[V]) {
    if constexpr (V * sizeof(T) == 16) {
        Vec16<T> t;
#pragma unroll
        for (int k = 0; k < V; ++k) t.v[k] = from_f32<T>(f[k]);
        st_stream16(p, t);
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) p[k] = from_f32<T>(f[k]);
    }
}

// Sum over the G threads of a row; every thread gets it.  `sh`: G / 32 floats for this call alone.
template <int G> __device__ __forceinline__ float row_sum(float v, float *sh) {
    v = warp_sum(v);
    if (G == 32) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(lane < G / 32 ? sh[lane] : 0.f);
}

template <typename T> constexpr int wide = 16 / int(sizeof(T));
template <typename T> constexpr int kRowElements = 4 * wide<T>;      // forward: 64 bytes of a row a thread

// Two elements side by side, as floats.
template <typename T> __device__ __forceinline__ pk_t pair_of(const T *p) { return ld_pk(p); }
template <> __device__ __forceinline__ pk_t pair_of(const __nv_bfloat16 *p) {
    const unsigned w = *reinterpret_cast<const unsigned *>(p);
    return pk2(make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)));
}

// A vector of 16 or 8 bytes of a row, as words.
template <int W> struct RowWords {
    unsigned w[W];
};
template <int W> __device__ __forceinline__ RowWords<W> load_words(const void *p) {
    RowWords<W> r;
    if constexpr (W == 4) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                     : "l"(p));
    } else {
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
    }
    return r;
}
template <int W> __device__ __forceinline__ void store_words(void *p, const RowWords<W> &r) {
    if constexpr (W == 4)
        asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]), "r"(r.w[3]) : "memory");
    else
        asm volatile("st.global.cs.v2.u32 [%0], {%1,%2};" ::"l"(p), "r"(r.w[0]), "r"(r.w[1]) : "memory");
}
// The words themselves are what lives on from here: without this the compiler keeps the floats made of them, twice as
// many registers for 16-bit types (72 against 52 a thread).
template <int N, int W> __device__ __forceinline__ void keep_words(RowWords<W> (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < W; ++k) asm volatile("" : "+r"(v[i].w[k]));
}
// Elements of a vector: 16 bytes; 8 bytes for 16-bit rows with float32 weight and bias, whose vectors are then 16
// bytes that lie side by side in a warp (with 32 bytes a thread every access is spread over twice the cache lines:
// [16384, 4096] bfloat16 62 against 50 us when it was chosen).
template <typename T, typename P> constexpr int row_vector = sizeof(P) > sizeof(T) ? 4 : wide<T>;
template <typename T, typename P> constexpr int row_vectors_held = kRowElements<T> / row_vector<T, P>;

// Rows of whole vectors: a row stays in the registers of its G threads (a warp, or a block) as the words it was read as,
// 64 bytes a thread, so that many of them are on their way at once.
template <typename T, typename P, int G>
__global__ void __launch_bounds__(G == 32 ? 256 : G) norm_forward_kernel(const NormParams p) {
    constexpr int V = row_vector<T, P>, N = row_vectors_held<T, P>, W = V * int(sizeof(T)) / 4;
    __shared__ float sh[2][32];
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t r = G == 32 ? int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5) : int64_t(blockIdx.x);
    if (r >= p.rows) return;
    const T *x = static_cast<const T *>(p.x) + r * p.x_stride;
    T *y = static_cast<T *>(p.y) + r * int64_t(p.D);
    RowWords<W> v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int j = (i * G + t) * V;
        if (j < p.D) v[i] = load_words<W>(x + j);
        else
#pragma unroll
            for (int k = 0; k < W; ++k) v[i].w[k] = 0u;
    }
    auto pair = [&](int i, int h) { return pair_of(reinterpret_cast<const T *>(v[i].w) + 2 * h); };
    pk_t sum = psplat(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int h = 0; h < V / 2; ++h) sum = padd(sum, pair(i, h));
    const float inv_d = 1.f / float(p.D);
    float2 s = upk2(sum);
    const float mean = row_sum<G>(s.x + s.y, sh[0]) * inv_d;
    keep_words(v);
    const pk_t negm = psplat(-mean);
    sum = psplat(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if ((i * G + t) * V < p.D) {
#pragma unroll
            for (int h = 0; h < V / 2; ++h) {
                const pk_t d = padd(pair(i, h), negm);
                sum = pfma(d, d, sum);
            }
        }
    }
    s = upk2(sum);
    const float rstd = rsqrtf(row_sum<G>(s.x + s.y, sh[1]) * inv_d + p.eps);
    keep_words(v);
    if (t == 0 && p.stats) p.stats[r] = make_float2(mean, rstd);
    const P *w = static_cast<const P *>(p.w), *b = static_cast<const P *>(p.b);
    const pk_t rr = psplat(rstd);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int j = (i * G + t) * V;
        if (j < p.D) {
            static_assert(V * sizeof(P) == 16, "a vector of weights is one access");
            uint4 a, c;
            if (w) a = __ldg(reinterpret_cast<const uint4 *>(w + j));
            if (b) c = __ldg(reinterpret_cast<const uint4 *>(b + j));
            RowWords<W> out;
#pragma unroll
            for (int h = 0; h < V / 2; ++h) {
                const pk_t u = pmul(padd(pair(i, h), negm), rr);
                const pk_t aw = w ? pair_of(reinterpret_cast<const P *>(&a) + 2 * h) : psplat(1.f);
                const pk_t cb = b ? pair_of(reinterpret_cast<const P *>(&c) + 2 * h) : psplat(0.f);
                st_pk(reinterpret_cast<T *>(out.w) + 2 * h, pfma(u, aw, cb));
            }
            store_words(y + j, out);
        }
    }
}

// Any row length: three sweeps over the row, the later ones from L2.
template <typename T, typename P> __global__ void __launch_bounds__(1024) norm_forward_any_kernel(const NormParams p) {
    __shared__ float sh[2][32];
    const int64_t r = blockIdx.x;
    const T *x = static_cast<const T *>(p.x) + r * p.x_stride;
    T *y = static_cast<T *>(p.y) + r * int64_t(p.D);
    const P *w = static_cast<const P *>(p.w), *b = static_cast<const P *>(p.b);
    float sum = 0.f;
    for (int64_t j = threadIdx.x; j < p.D; j += 1024) sum += to_f32(x[j]);
    const float inv_d = 1.f / float(p.D);
    const float mean = row_sum<1024>(sum, sh[0]) * inv_d;
    sum = 0.f;
    for (int64_t j = threadIdx.x; j < p.D; j += 1024) {
        const float d = to_f32(x[j]) - mean;
        sum = fmaf(d, d, sum);
    }
    const float rstd = rsqrtf(row_sum<1024>(sum, sh[1]) * inv_d + p.eps);
    if (threadIdx.x == 0 && p.stats) p.stats[r] = make_float2(mean, rstd);
    for (int64_t j = threadIdx.x; j < p.D; j += 1024) {
        float v = (to_f32(x[j]) - mean) * rstd;
        if (w) v *= to_f32(w[j]);
        if (b) v += to_f32(b[j]);
        y[j] = from_f32<T>(v);
    }
}

// ---- rows through shared memory
//
// A group of G threads owns every (blocks x groups)-th row.  Its rows arrive by bulk copies in a ring of `stages` slots,
// so that the next rows are on their way while one is worked on.  A thread owns the same kColumns columns in every
// row: weight, bias and the sums for their gradients stay in its registers, as pairs for the packed arithmetic.  There
// is one barrier per row, behind which everybody has read the row's slot, so that it can be filled again.
// Rows of more than 8192 columns are split over the blocks of a cluster: the warps' sums go to all blocks' shared
// memory, and the row's barrier is the cluster's.
constexpr int kColumns = 16, kPairs = kColumns / 2;         // of a thread
constexpr int kTeamThreads = 512, kTeamColumns = kTeamThreads * kColumns;      // blocks that share a row
constexpr int kMaxRowBlocks = 8;
template <int G> constexpr int ring_block = G < 256 ? 256 : G;
// Blocks per SM that the registers are laid out for (forward, backward).
template <int G> constexpr int forward_blocks = G <= 256 ? 3 : 1;
template <int G> constexpr int backward_blocks = G <= 256 ? 2 : 1;

// Barrier of a group: the warp, some warps of the block (one named barrier each), or the block.
template <int G> __device__ __forceinline__ void group_barrier(int group) {
    if (G == 32) __syncwarp();
    else if (G == ring_block<G>) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(G) : "memory");
}

// Element j of a row whose first element lies `off` elements behind a 16-byte boundary stands at slot + off + j: what
// lies between two boundaries is copied in bulk (one thread), the ragged elements (V == 1 only) one by one.
template <typename T> __device__ __forceinline__ int row_offset(const T *row) {
    return int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}
struct RowBody {
    int body, n;                                            // first element and number of elements of the bulk copy
};
template <typename T, int V> __device__ __forceinline__ RowBody row_body(const T *row, int D) {
    constexpr int E = 16 / int(sizeof(T));
    if (V > 1) return RowBody{0, D};
    const int off = row_offset(row);
    RowBody r;
    r.body = min(D, off ? E - off : 0);
    r.n = (D - r.body) / E * E;
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void fill_slot(T *slot, const T *row, int D, int t, uint64_t *bar) {
    const RowBody r = row_body<T, V>(row, D);
    const int off = V == 1 ? row_offset(row) : 0;
    if (t == 0 && r.n > 0) bulk_load_1d(slot + off + r.body, row + r.body, uint32_t(r.n) * uint32_t(sizeof(T)), bar);
    if (V == 1) {
        const int tail = r.body + r.n;
        if (t < r.body) slot[off + t] = row[t];
        if (t < D - tail) slot[off + tail + t] = row[tail + t];
        // The bulk copy that refills the slot may cover these bytes (its row starts elsewhere within 16 bytes): the
        // threads that wrote them order their stores before it, the barrier in front of the refill does the rest.
        if (t < r.body || t < D - tail) fence_proxy_async_smem();
    }
}
// Bytes of a slot: the row and the place of its first element in 16 bytes.
__host__ __device__ inline size_t slot_bytes(int D, size_t s) { return (size_t(D) * s + 31) / 16 * 16; }

// A thread's columns: packs of V, pack i starts at column (i * G + t) * V.  Columns behind the row's end read as 0.
template <int V, int G> __device__ __forceinline__ int column_of(int t, int e) { return ((e / V) * G + t) * V + e % V; }
template <typename T, int V, int G, int PAIRS>
__device__ __forceinline__ void load_columns(const T *row, int D, int t, pk_t (&v)[PAIRS]) {
    row += t * V;                                           // (the packs lie constant distances behind)
    D -= t * V;
    if constexpr (V > 1) {
#pragma unroll
        for (int i = 0; i < 2 * PAIRS / V; ++i) {
            uint4 raw[V * sizeof(T) / 16];
#pragma unroll
            for (int q = 0; q < int(V * sizeof(T) / 16); ++q)
                raw[q] = i * G * V < D ? reinterpret_cast<const uint4 *>(row + i * G * V)[q] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int h = 0; h < V / 2; ++h) v[i * (V / 2) + h] = pair_of(reinterpret_cast<const T *>(raw) + 2 * h);
        }
    } else {
#pragma unroll
        for (int h = 0; h < PAIRS; ++h) {
            const int j = 2 * h * G;
            v[h] = pk2(make_float2(j < D ? to_f32(row[j]) : 0.f, j + G < D ? to_f32(row[j + G]) : 0.f));
        }
    }
}
template <typename T, int V, int G, int PAIRS>
__device__ __forceinline__ void store_columns(T *row, int D, int t, const pk_t (&v)[PAIRS]) {
    row += t * V;
    D -= t * V;
    if constexpr (V > 1) {
#pragma unroll
        for (int i = 0; i < 2 * PAIRS / V; ++i) {
            const int j = i * G * V;
            if (j < D) {
                uint4 raw[V * sizeof(T) / 16];
#pragma unroll
                for (int h = 0; h < V / 2; ++h) st_pk(reinterpret_cast<T *>(raw) + 2 * h, v[i * (V / 2) + h]);
#pragma unroll
                for (int q = 0; q < int(V * sizeof(T) / 16); ++q)
                    st_stream16(reinterpret_cast<char *>(row + j) + 16 * q, raw[q]);
            }
        }
    } else {
#pragma unroll
        for (int h = 0; h < PAIRS; ++h) {
            const int j = 2 * h * G;
            const float2 f = upk2(v[h]);
            if (j < D) row[j] = from_f32<T>(f.x);
            if (j + G < D) row[j + G] = from_f32<T>(f.y);
        }
    }
}
// The group's ring; a slot holds x, or x and dy, of a row.
template <typename T, int V, int G> struct Ring {
    uint64_t *full;
    char *slots;
    size_t slot;
    int stages, t;
    __device__ __forceinline__ void init(uint64_t *bars, char *memory, size_t slot_size, int n, int thread, int group) {
        full = bars;
        slots = memory;
        slot = slot_size;
        stages = n;
        t = thread;
        if (t == 0) {
            for (int i = 0; i < n; ++i) mbar_init(&full[i], 1);
            fence_mbar_init();
        }
        group_barrier<G>(group);
    }
    __device__ __forceinline__ void fill(int stage, const T *x, int D) {
        if (t == 0) mbar_expect_tx(&full[stage], uint32_t(row_body<T, V>(x, D).n) * uint32_t(sizeof(T)));
        fill_slot<T, V>(reinterpret_cast<T *>(slots + size_t(stage) * slot), x, D, t, &full[stage]);
    }
    __device__ __forceinline__ void fill(int stage, const T *x, const T *dy, int D) {
        if (t == 0)
            mbar_expect_tx(&full[stage], uint32_t(row_body<T, V>(x, D).n + row_body<T, V>(dy, D).n) * uint32_t(sizeof(T)));
        char *at = slots + size_t(stage) * 2 * slot;
        fill_slot<T, V>(reinterpret_cast<T *>(at), x, D, t, &full[stage]);
        fill_slot<T, V>(reinterpret_cast<T *>(at + slot), dy, D, t, &full[stage]);
    }
};
__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fc00000); }

// Rows that are not whole vectors at 16-byte addresses (V == 1).
template <typename T, typename P, int G>
__global__ void __launch_bounds__(ring_block<G>, forward_blocks<G>) norm_forward_ragged_kernel(const NormParams p) {
    constexpr int GROUPS = ring_block<G> / G, WARPS = G / 32;
    extern __shared__ __align__(16) char slots[];
    __shared__ uint64_t full[GROUPS][kMaxSlots];
    __shared__ float2 moments[GROUPS][2][WARPS];            // {mean, sum of squares around it} of each warp's columns
    __shared__ int lost[GROUPS];
    const int t = threadIdx.x % G, group = threadIdx.x / G, lane = threadIdx.x & 31, warp = t >> 5;
    const int64_t first = int64_t(blockIdx.x) * GROUPS + group, step = int64_t(gridDim.x) * GROUPS;
    const size_t slot = slot_bytes(p.D, sizeof(T));
    const T *xs = static_cast<const T *>(p.x);
    const float inv_d = 1.f / float(p.D);

    Ring<T, 1, G> ring;
    if (t == 0) lost[group] = 0;
    ring.init(full[group], slots + size_t(group) * p.stages * slot, slot, p.stages, t, group);
    for (int i = 0; i < p.stages && first + i * step < p.rows; ++i) ring.fill(i, xs + (first + i * step) * p.x_stride, p.D);
    pk_t w[kPairs], b[kPairs];
#pragma unroll
    for (int h = 0; h < kPairs; ++h) {
        w[h] = psplat(1.f);
        b[h] = psplat(0.f);
    }
    if (p.w) load_columns<P, 1, G>(static_cast<const P *>(p.w), p.D, t, w);
    if (p.b) load_columns<P, 1, G>(static_cast<const P *>(p.b), p.D, t, b);
    // columns of warp `of`
    auto columns_of = [&](int of) {
        int n = 0;
        for (int i = 0; i < kColumns; ++i) n += min(max(p.D - (i * G + of * 32), 0), 32);
        return float(n);
    };
    const float n_own = columns_of(warp), n_lane = lane < WARPS ? columns_of(lane) : 0.f;
    const float inv_own = n_own > 0.f ? 1.f / n_own : 0.f;
    group_barrier<G>(group);

    int stage = 0, turn = 0;
    uint32_t parity = 0;
    bool dead = false;                                      // a copy never came: the group's rows become NaN
    for (int64_t r = first; r < p.rows; r += step) {
        if (!dead && !mbar_wait_bounded(&full[group][stage], parity, nullptr)) lost[group] = 1;
        const T *row = reinterpret_cast<const T *>(ring.slots + size_t(stage) * slot) + row_offset(xs + r * p.x_stride);
        pk_t v[kPairs];
        load_columns<T, 1, G>(row, p.D, t, v);
        pk_t sum2 = v[0];
#pragma unroll
        for (int h = 1; h < kPairs; ++h) sum2 = padd(sum2, v[h]);
        const float2 s2 = upk2(sum2);
        float mean = warp_sum(s2.x + s2.y) * inv_own;
        const pk_t around = psplat(-mean);
        pk_t sq2 = psplat(0.f);
#pragma unroll
        for (int h = 0; h < kPairs; ++h) {
            float2 f = upk2(padd(v[h], around));
            if (column_of<1, G>(t, 2 * h) >= p.D) f.x = 0.f;
            if (column_of<1, G>(t, 2 * h + 1) >= p.D) f.y = 0.f;
            sq2 = pfma(pk2(f), pk2(f), sq2);
        }
        const float2 q2 = upk2(sq2);
        float square = warp_sum(q2.x + q2.y);
        if (G > 32) {
            if (lane == 0) moments[group][turn][warp] = make_float2(mean, square);
            group_barrier<G>(group);
            // the mean of the means, and the squares around it
            const float2 m = moments[group][turn][lane < WARPS ? lane : 0];
            mean = warp_sum(n_lane * m.x) * inv_d;
            const float d = m.x - mean;
            square = warp_sum(lane < WARPS ? fmaf(n_lane * d, d, m.y) : 0.f);
        } else {
            __syncwarp();
        }
        if (lost[group]) dead = true;
        const int64_t ahead = r + int64_t(p.stages) * step;
        if (!dead && ahead < p.rows) ring.fill(stage, xs + ahead * p.x_stride, p.D);
        const float rstd = dead ? nan_f() : rsqrtf(square * inv_d + p.eps);
        if (t == 0 && p.stats) p.stats[r] = make_float2(mean, rstd);
        const pk_t negm = psplat(-mean), rr = psplat(rstd);
#pragma unroll
        for (int h = 0; h < kPairs; ++h) v[h] = pfma(pmul(padd(v[h], negm), rr), w[h], b[h]);
        store_columns<T, 1, G>(static_cast<T *>(p.y) + r * int64_t(p.D), p.D, t, v);
        turn ^= 1;
        if (++stage == p.stages) {
            stage = 0;
            parity ^= 1;
        }
    }
}

// The part of a row that this block owns, and where it starts.
struct RowShare {
    int first, n;
};
__device__ __forceinline__ RowShare row_share(const NormParams &p, int rank) {
    return RowShare{rank * p.share, min(p.share, p.D - rank * p.share)};
}
// Leaves a warp's two numbers where all of the row's warps find them (every block's shared memory), and waits for
// everybody's.
template <int G>
__device__ __forceinline__ void exchange(float2 *slots, int warp, int rank, int blocks, float2 v, int group) {
    namespace cg = cooperative_groups;
    if (G == kTeamThreads && blocks > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        const int lane = threadIdx.x & 31;
        if (lane < blocks) cluster.map_shared_rank(slots, lane)[rank * (G / 32) + warp] = v;
        cluster.sync();
    } else {
        if ((threadIdx.x & 31) == 0) slots[warp] = v;
        group_barrier<G>(group);
    }
}
template <int G> constexpr int sum_slots = G == kTeamThreads ? G / 32 * kMaxRowBlocks : G / 32;

template <typename T, typename P, int V, int G>
__global__ void __launch_bounds__(ring_block<G>, backward_blocks<G>) norm_backward_kernel(const NormParams p) {
    constexpr int GROUPS = ring_block<G> / G, WARPS = G / 32;
    extern __shared__ __align__(16) char slots[];
    __shared__ uint64_t full[GROUPS][kMaxSlots];
    __shared__ float2 sums[GROUPS][2][sum_slots<G>];
    __shared__ int lost[GROUPS];
    const int t = threadIdx.x % G, group = threadIdx.x / G, lane = threadIdx.x & 31, warp = t >> 5;
    const int rank = G == kTeamThreads ? int(blockIdx.x % unsigned(p.blocks)) : 0;
    const int64_t team = G == kTeamThreads ? blockIdx.x / unsigned(p.blocks) : blockIdx.x;
    const int64_t teams = G == kTeamThreads ? gridDim.x / unsigned(p.blocks) : gridDim.x;
    const int64_t first = team * GROUPS + group, step = teams * GROUPS;
    const RowShare own = row_share(p, rank);
    const size_t slot = slot_bytes(p.share, sizeof(T));
    const T *xs = static_cast<const T *>(p.x) + own.first, *ys = static_cast<const T *>(p.dy) + own.first;
    const float inv_d = 1.f / float(p.D);

    Ring<T, V, G> ring;
    if (t == 0) lost[group] = 0;
    ring.init(full[group], slots + size_t(group) * p.stages * 2 * slot, slot, p.stages, t, group);
    for (int i = 0; i < p.stages && first + i * step < p.rows; ++i)
        ring.fill(i, xs + (first + i * step) * p.x_stride, ys + (first + i * step) * p.dy_stride, own.n);
    pk_t dw[kPairs], db[kPairs], w[kPairs];
#pragma unroll
    for (int h = 0; h < kPairs; ++h) {
        dw[h] = db[h] = psplat(0.f);
        w[h] = psplat(1.f);
    }
    if (p.w) load_columns<P, V, G>(static_cast<const P *>(p.w) + own.first, own.n, t, w);
    float2 next = first < p.rows ? p.stats[first] : make_float2(0.f, 0.f);
    if (G == kTeamThreads && p.blocks > 1) cooperative_groups::this_cluster().sync();
    else group_barrier<G>(group);

    int stage = 0, turn = 0;
    uint32_t parity = 0;
    bool dead = false;                                      // a copy never came: the group's rows become NaN
    for (int64_t r = first; r < p.rows; r += step) {
        float2 st = next;
        if (r + step < p.rows) next = p.stats[r + step];
        if (!dead && !mbar_wait_bounded(&full[group][stage], parity, nullptr)) {
            lost[group] = 1;
            st.y = nan_f();
        }
        const T *x = reinterpret_cast<const T *>(ring.slots + size_t(stage) * 2 * slot);
        const T *dy = reinterpret_cast<const T *>(reinterpret_cast<const char *>(x) + slot);
        if (V == 1) {
            x += row_offset(xs + r * p.x_stride);
            dy += row_offset(ys + r * p.dy_stride);
        }
        pk_t h[kPairs], g[kPairs];
        pk_t sg2 = psplat(0.f), sgh2 = psplat(0.f);
        load_columns<T, V, G>(x, own.n, t, h);
        load_columns<T, V, G>(dy, own.n, t, g);
        {
            // (the difference first, as forward forms it: x r - mean r would be off by 2^-24 |mean| r in every column)
            const pk_t negm = psplat(-st.x), rr = psplat(st.y);
#pragma unroll
            for (int i = 0; i < kPairs; ++i) {
                h[i] = pmul(padd(h[i], negm), rr);
                dw[i] = pfma(g[i], h[i], dw[i]);
                db[i] = padd(db[i], g[i]);
                g[i] = pmul(g[i], w[i]);
                sg2 = padd(sg2, g[i]);
                sgh2 = pfma(g[i], h[i], sgh2);
            }
        }
        const float2 a = upk2(sg2), c = upk2(sgh2);
        float sg = warp_sum(a.x + a.y), sgh = warp_sum(c.x + c.y);
        if (G > 32) {
            const float2 *all = sums[group][turn];
            exchange<G>(sums[group][turn], warp, rank, p.blocks, make_float2(sg, sgh), group);
            if (G == kTeamThreads && p.blocks > 1) {
                sg = sgh = 0.f;
                for (int i = lane; i < WARPS * p.blocks; i += 32) {
                    sg += all[i].x;
                    sgh += all[i].y;
                }
                sg = warp_sum(sg);
                sgh = warp_sum(sgh);
            } else {                                        // (each lane starts with one of the WARPS numbers)
                const float2 one = all[lane & (WARPS - 1)];
                sg = one.x;
                sgh = one.y;
#pragma unroll
                for (int o = WARPS / 2; o > 0; o >>= 1) {
                    sg += __shfl_xor_sync(0xffffffffu, sg, o);
                    sgh += __shfl_xor_sync(0xffffffffu, sgh, o);
                }
            }
        } else {
            __syncwarp();
        }
        if (lost[group]) dead = true;
        const int64_t ahead = r + int64_t(p.stages) * step;
        if (!dead && ahead < p.rows) ring.fill(stage, xs + ahead * p.x_stride, ys + ahead * p.dy_stride, own.n);
        // dx = r g - r mean(g) - h r mean(g h)
        const float r0 = dead ? nan_f() : st.y;
        const pk_t rr = psplat(r0), c0 = psplat(-sg * inv_d * r0), c1 = psplat(-sgh * inv_d * r0);
#pragma unroll
        for (int i = 0; i < kPairs; ++i) g[i] = pfma(g[i], rr, pfma(h[i], c1, c0));
        store_columns<T, V, G>(static_cast<T *>(p.dx) + r * int64_t(p.D) + own.first, own.n, t, g);
        turn ^= 1;
        if (++stage == p.stages) {
            stage = 0;
            parity ^= 1;
        }
    }
    if (G == kTeamThreads && p.blocks > 1) cooperative_groups::this_cluster().sync();    // (nobody leaves while it is written to)
    if (!p.partial) return;
    float *out = p.partial + team * 2 * p.D + own.first;
    if (dead) dw[0] = db[0] = psplat(nan_f());
    if (GROUPS > 1) {                                       // the groups' columns, one group after the other
        float *columns = reinterpret_cast<float *>(slots);  // (every copy has been waited for)
        for (int turns = 0; turns < GROUPS; ++turns) {
            __syncthreads();
            if (group == turns) {
#pragma unroll
                for (int e = 0; e < kColumns; ++e) {
                    const int j = column_of<V, G>(t, e);
                    const float2 a = upk2(dw[e / 2]), c = upk2(db[e / 2]);
                    if (j < own.n) {
                        columns[j] = (turns ? columns[j] : 0.f) + (e % 2 ? a.y : a.x);
                        columns[own.n + j] = (turns ? columns[own.n + j] : 0.f) + (e % 2 ? c.y : c.x);
                    }
                }
            }
        }
        __syncthreads();
        for (int j = threadIdx.x; j < 2 * own.n; j += ring_block<G>) out[j] = columns[j];
    } else {
#pragma unroll
        for (int e = 0; e < kColumns; ++e) {
            const int j = column_of<V, G>(t, e);
            const float2 a = upk2(dw[e / 2]), c = upk2(db[e / 2]);
            if (j < own.n) {
                out[j] = e % 2 ? a.y : a.x;
                out[p.D + j] = e % 2 ? c.y : c.x;
            }
        }
    }
}

// Any row length: dx of a row per block ...
template <typename T, typename P> __global__ void __launch_bounds__(1024) norm_backward_any_kernel(const NormParams p) {
    __shared__ float sh[2][32];
    const int64_t r = blockIdx.x;
    const T *x = static_cast<const T *>(p.x) + r * p.x_stride, *dy = static_cast<const T *>(p.dy) + r * p.dy_stride;
    T *dx = static_cast<T *>(p.dx) + r * int64_t(p.D);
    const P *w = static_cast<const P *>(p.w);
    const float2 st = p.stats[r];
    float sg = 0.f, sgh = 0.f;
    for (int64_t j = threadIdx.x; j < p.D; j += 1024) {
        const float g = to_f32(dy[j]) * (w ? to_f32(w[j]) : 1.f);
        sg += g;
        sgh = fmaf(g, (to_f32(x[j]) - st.x) * st.y, sgh);
    }
    const float inv_d = 1.f / float(p.D);
    sg = row_sum<1024>(sg, sh[0]) * inv_d;
    sgh = row_sum<1024>(sgh, sh[1]) * inv_d;
    for (int64_t j = threadIdx.x; j < p.D; j += 1024) {
        const float g = to_f32(dy[j]) * (w ? to_f32(w[j]) : 1.f);
        dx[j] = from_f32<T>(st.y * (g - sg - (to_f32(x[j]) - st.x) * st.y * sgh));
    }
}
// ... and the columns' sums of a share of the rows (blockIdx.y of gridDim.y) per block of 256 columns.
template <typename T> __global__ void __launch_bounds__(256) norm_columns_any_kernel(const NormParams p) {
    const int64_t j = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (j >= p.D) return;
    const T *x = static_cast<const T *>(p.x) + j, *dy = static_cast<const T *>(p.dy) + j;
    float dw = 0.f, db = 0.f;
    for (int64_t r = blockIdx.y; r < p.rows; r += gridDim.y) {
        const float2 st = p.stats[r];
        const float g = to_f32(dy[r * p.dy_stride]);
        dw = fmaf(g, (to_f32(x[r * p.x_stride]) - st.x) * st.y, dw);
        db += g;
    }
    float *out = p.partial + int64_t(blockIdx.y) * 2 * p.D;
    out[j] = dw;
    out[p.D + j] = db;
}

// dw and db from the blocks' partial rows: 32 columns by 16 shares of the blocks to a block.
template <typename P>
__global__ void __launch_bounds__(512) norm_columns_kernel(const float *partial, int blocks, int D, P *dw, P *db) {
    __shared__ float sh[16][33];
    pdl_wait();
    const int lane = threadIdx.x & 31, share = threadIdx.x >> 5;
    const int64_t width = 2 * int64_t(D);
    const int64_t j = int64_t(blockIdx.x) * 32 + lane;
    float sum = 0.f;
    if (j < width)
        for (int i = share; i < blocks; i += 16) sum += partial[i * width + j];
    sh[share][lane] = sum;
    __syncthreads();
    if (share == 0 && j < width) {
#pragma unroll
        for (int i = 1; i < 16; ++i) sum += sh[i][lane];
        if (j < D) {
            if (dw) dw[j] = from_f32<P>(sum);
        } else if (db) {
            db[j - D] = from_f32<P>(sum);
        }
    }
}

// How rows go through shared memory: threads to a row (of one block), blocks to a row, blocks per SM, slots;
// threads == 0: not at all (longer than a cluster's columns).
struct RingPlan {
    int threads, blocks, share, per_sm, stages;
    int groups() const { return threads && threads < 256 ? 256 / threads : 1; }
};
inline RingPlan ring_plan(int D, size_t s, bool backward) {
    RingPlan r{0, 1, D, 1, 0};
    for (int g : {512, 256, 128, 64, 32})
        if (g * kColumns >= D) r.threads = g;
    if (r.threads == 0) {
        r.blocks = (D + kTeamColumns - 1) / kTeamColumns;
        if (r.blocks > kMaxRowBlocks) return r;
        r.threads = kTeamThreads;
        r.share = ((D + r.blocks - 1) / r.blocks + 63) / 64 * 64;
    }
    if (r.threads <= 256) r.per_sm = backward ? 2 : 3;
    // (at least two slots: 8192 columns of x and dy in float32 are 64 KB)
    r.stages = int(kRingBytes / r.per_sm / (slot_bytes(r.share, s) * (backward ? 2 : 1) * r.groups()));
    if (r.stages > kMaxSlots) r.stages = kMaxSlots;
    return r;
}
// Teams of blocks that share a row.
inline int ring_teams(int64_t rows, const RingPlan &plan) {
    const int64_t most = plan.threads == 0 ? 64 : std::max<int64_t>(int64_t(sm_count()) * plan.per_sm / plan.blocks, 1);
    const int64_t want = (rows + plan.groups() - 1) / plan.groups();
    return int(want < 1 ? 1 : want > most ? most : want);
}
template <typename K> int launch_ring(K kernel, NormParams p, const RingPlan &plan, int block, size_t smem, const char *what, cudaStream_t s) {
    p.stages = plan.stages;
    p.blocks = plan.blocks;
    p.share = plan.share;
    if (const int rc = set_smem(kernel, smem)) return rc;
    return launch_cluster(kernel, int64_t(ring_teams(p.rows, plan)) * plan.blocks, block, smem, plan.blocks, false, s, what, p);
}
inline bool on16(const void *p) { return lies_on(p, 16); }

template <typename T, typename P> struct NormLaunch {
    template <int G> static int forward_rows(const NormParams &p, cudaStream_t s) {
        const int64_t grid = G == 32 ? (p.rows + 7) / 8 : p.rows;
        norm_forward_kernel<T, P, G><<<unsigned(grid), G == 32 ? 256 : G, 0, s>>>(p);
        return launch_status("layer norm kernel launch");
    }
    template <int G> static int forward_ragged(const NormParams &p, const RingPlan &plan, cudaStream_t s) {
        const size_t smem = size_t(plan.stages) * slot_bytes(p.D, sizeof(T)) * plan.groups();
        return launch_ring(norm_forward_ragged_kernel<T, P, G>, p, plan, ring_block<G>, smem, "layer norm kernel launch", s);
    }
    static int forward(const NormParams &p, cudaStream_t s) {
        constexpr int V = wide<T>;
        const bool vec = p.D % V == 0 && on16(p.x) && on16(p.y) && (p.rows < 2 || p.x_stride % V == 0) && on16(p.w) && on16(p.b);
        const int64_t threads = vec ? (p.D + kRowElements<T> - 1) / kRowElements<T> : INT64_MAX;
        if (threads <= 32) return forward_rows<32>(p, s);
        if (threads <= 64) return forward_rows<64>(p, s);
        if (threads <= 128) return forward_rows<128>(p, s);
        if (threads <= 256) return forward_rows<256>(p, s);
        if (threads <= 512) return forward_rows<512>(p, s);
        if (threads <= 1024) return forward_rows<1024>(p, s);
        const RingPlan plan = ring_plan(p.D, sizeof(T), false);
        if (!vec && plan.blocks == 1) {
            switch (plan.threads) {
                case 32: return forward_ragged<32>(p, plan, s);
                case 64: return forward_ragged<64>(p, plan, s);
                case 128: return forward_ragged<128>(p, plan, s);
                case 256: return forward_ragged<256>(p, plan, s);
                case 512: return forward_ragged<512>(p, plan, s);
            }
        }
        norm_forward_any_kernel<T, P><<<unsigned(p.rows), 1024, 0, s>>>(p);
        return launch_status("layer norm kernel launch");
    }
    template <int V, int G> static int backward(const NormParams &p, const RingPlan &plan, cudaStream_t s) {
        const size_t ring = size_t(plan.stages) * 2 * slot_bytes(plan.share, sizeof(T)) * plan.groups();
        const size_t columns = G < 256 ? size_t(p.D) * 8 : 0;
        return launch_ring(norm_backward_kernel<T, P, V, G>, p, plan, ring_block<G>, ring > columns ? ring : columns,
                           "layer norm gradient kernel launch", s);
    }
    template <int V> static int backward_of(const NormParams &p, const RingPlan &plan, cudaStream_t s) {
        switch (plan.threads) {
            case 32: return backward<V, 32>(p, plan, s);
            case 64: return backward<V, 64>(p, plan, s);
            case 128: return backward<V, 128>(p, plan, s);
            case 256: return backward<V, 256>(p, plan, s);
            case 512: return backward<V, 512>(p, plan, s);
        }
        norm_backward_any_kernel<T, P><<<unsigned(p.rows), 1024, 0, s>>>(p);
        if (const int rc = launch_status("layer norm gradient kernel launch")) return rc;
        if (!p.partial) return B200_OK;
        norm_columns_any_kernel<T><<<dim3(unsigned((p.D + 255) / 256), unsigned(ring_teams(p.rows, plan))), 256, 0, s>>>(p);
        return launch_status("layer norm column kernel launch");
    }
    static int backward(const NormParams &p, void *dw, void *db, cudaStream_t s) {
        constexpr int V = wide<T>;
        const bool vec = p.D % V == 0 && on16(p.x) && on16(p.dx) && on16(p.dy) && on16(p.w) &&
                         (p.rows < 2 || (p.x_stride % V == 0 && p.dy_stride % V == 0));
        const RingPlan plan = ring_plan(p.D, sizeof(T), true);
        if (p.rows > 0) {
            const int rc = vec ? backward_of<V>(p, plan, s) : backward_of<1>(p, plan, s);
            if (rc) return rc;
        }
        if (!p.partial) return B200_OK;
        return launch_cluster(norm_columns_kernel<P>, (2 * int64_t(p.D) + 31) / 32, 512, 0, 1, true, s,
                              "layer norm column kernel launch", static_cast<const float *>(p.partial),
                              p.rows > 0 ? ring_teams(p.rows, plan) : 0, p.D, static_cast<P *>(dw), static_cast<P *>(db));
    }
};

int check_norm(const char *who, int64_t rows, int64_t D, int dtype, int param_dtype) {
    if (rows < 0 || D < 1) {
        set_error("%s: need rows >= 0 and D >= 1", who);
        return B200_ERR_ARG;
    }
    if (rows > 0x7fffffff || D > (int64_t(1) << 30)) {
        set_error("%s: at most 2^31 - 1 rows of 2^30 elements", who);
        return B200_ERR_UNSUPPORTED;
    }
    if (!dtype_known(dtype) || (param_dtype != dtype && param_dtype != B200_F32)) {
        set_error("%s: weight and bias are float32 or have the rows' type", who);
        return B200_ERR_ARG;
    }
    return B200_OK;
}

template <typename F> int by_type(int dtype, int param_dtype, F f) {
    if (dtype == B200_F32) return f(NormLaunch<float, float>());
    if (dtype == B200_F16)
        return param_dtype == B200_F32 ? f(NormLaunch<__half, float>()) : f(NormLaunch<__half, __half>());
    return param_dtype == B200_F32 ? f(NormLaunch<__nv_bfloat16, float>()) : f(NormLaunch<__nv_bfloat16, __nv_bfloat16>());
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" int b200_layer_norm(const void *x, const void *weight, const void *bias, void *y, void *stats, int64_t rows,
                               int64_t D, int64_t stride, int dtype, int param_dtype, float eps, void *stream) {
    const char *who = "b200_layer_norm";
    if (const int rc = check_norm(who, rows, D, dtype, param_dtype)) return rc;
    const size_t e = dtype_size(dtype), pe = dtype_size(param_dtype);
    if (!(eps >= 0.f) || stride < 0 || (rows > 0 && (!x || !y)) || !lies_on(stats, 8) || !lies_on(x, e) || !lies_on(y, e) ||
        !lies_on(weight, pe) || !lies_on(bias, pe)) {
        set_error("%s: null or misaligned pointer, or eps < 0", who);
        return B200_ERR_ARG;
    }
    if (rows == 0) return B200_OK;
    NormParams p{};
    p.x = x;
    p.w = weight;
    p.b = bias;
    p.y = y;
    p.stats = static_cast<float2 *>(stats);
    p.x_stride = stride;
    p.rows = rows;
    p.D = int(D);
    p.eps = eps;
    return by_type(dtype, param_dtype, [&](auto l) { return l.forward(p, static_cast<cudaStream_t>(stream)); });
}

extern "C" size_t b200_layer_norm_scratch_bytes(int64_t rows, int64_t D) {
    if (rows < 0 || D < 1) return 0;
    const int64_t most = int64_t(sm_count()) * 2 < 64 ? 64 : int64_t(sm_count()) * 2;
    return size_t(rows < 1 ? 1 : rows < most ? rows : most) * size_t(D) * 8;
}

extern "C" int b200_layer_norm_backward(const void *x, const void *weight, const void *stats, const void *dy, void *dx,
                                        void *dweight, void *dbias, void *scratch, size_t scratch_bytes, int64_t rows,
                                        int64_t D, int64_t stride, int64_t dy_stride, int dtype, int param_dtype,
                                        void *stream) {
    const char *who = "b200_layer_norm_backward";
    if (const int rc = check_norm(who, rows, D, dtype, param_dtype)) return rc;
    const size_t e = dtype_size(dtype), pe = dtype_size(param_dtype);
    if (stride < 0 || dy_stride < 0 || (rows > 0 && (!x || !dy || !dx || !stats)) || !lies_on(stats, 8) || !lies_on(x, e) ||
        !lies_on(dy, e) || !lies_on(dx, e) || !lies_on(weight, pe) || !lies_on(dweight, pe) || !lies_on(dbias, pe)) {
        set_error("%s: null or misaligned pointer", who);
        return B200_ERR_ARG;
    }
    if ((dweight || dbias) && (!scratch || !on16(scratch) || scratch_bytes < b200_layer_norm_scratch_bytes(rows, D))) {
        set_error("%s: scratch of %zu bytes on a 16-byte address required", who, b200_layer_norm_scratch_bytes(rows, D));
        return B200_ERR_WORKSPACE;
    }
    NormParams p{};
    p.x = x;
    p.w = weight;
    p.dy = dy;
    p.dx = dx;
    p.stats = const_cast<float2 *>(static_cast<const float2 *>(stats));
    p.partial = dweight || dbias ? static_cast<float *>(scratch) : nullptr;
    p.x_stride = stride;
    p.dy_stride = dy_stride;
    p.rows = rows;
    p.D = int(D);
    return by_type(dtype, param_dtype,
                   [&](auto l) { return l.backward(p, dweight, dbias, static_cast<cudaStream_t>(stream)); });
}
