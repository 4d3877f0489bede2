// Rows of a language model's logits (one row per token, V contiguous logits): what the log-probability and the
// distillation kernels share.
//
// With z_j = (x_j - m) * c in units of log2 (c = log2(e) / temperature, m the row's maximum), e_j = 2^z_j,
// s = sum e_j and u = sum e_j z_j:
//     p_j = e_j / s      log p_j = ln2 (z_j - log2 s)      entropy = ln2 (log2 s - u / s)
// m, s and u come from ONE pass: every thread keeps its own running maximum and rescales its sums where the maximum
// rises (once per 4 vectors at most), threads, warps and the blocks of a cluster are joined afterwards.
//
// The difference x_j - m is formed before the scaling, so rows of the type's lowest value (a mask that left nothing)
// stay finite.  Where z_j itself enters a sum it is held at -200 or more (2^-200 is 0 here), so that a masked logit
// (-inf) adds 0 * -200 and not 0 * inf to u.  Maxima hand NaN on: a NaN logit gives NaN results, never a hidden one.  A row of -inf alone has
// s = 0; each kernel says what it returns there.
//
// A row starts wherever its tensor puts it: the elements in front of the first 16-byte boundary and behind the last
// one are read one by one, all others as 16-byte vectors.
#pragma once
#include <cooperative_groups.h>

#include "pipeline.cuh"

namespace b200 {
namespace {

constexpr float kTokenLn2 = 0.6931471805599453f;
constexpr float kTokenFloor = -200.f;       // smallest z: 2^-200 = 0 in float32
constexpr int kTokenUnroll = 4;             // vectors of a thread in flight
constexpr int kMaxList = 128;               // alternatives per row
constexpr int kMaxCluster = 8;              // blocks that share a row

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Whether a maximum rises (or is NaN).  Not a plain comparison: the library is built with denormals flushed, and the
// maxima keep them apart.
__device__ __forceinline__ bool rises(float to, float m) {
    unsigned r;
    asm("{\n\t.reg .pred p;\n\tsetp.gtu.f32 p, %1, %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "f"(to), "f"(m));
    return r != 0u;
}
// The reference that a maximum stands for: 0 where there is nothing but -inf, so that differences exist.
__device__ __forceinline__ float reference_of(float m) { return m == -INFINITY ? 0.f : m; }

// log p in nats; not by way of z, which the type's lowest value would take past float32's range.
__device__ __forceinline__ float log_prob(float x, float m, float inv_t, float log2s) {
    return (x - m) * inv_t - kTokenLn2 * log2s;
}

// ---- 16-byte vectors of logits as pairs of floats

template <typename T> struct TokenVec;
__device__ __forceinline__ unsigned word_of(const uint4 &v, int i) {
    return i & 2 ? (i & 1 ? v.w : v.z) : (i & 1 ? v.y : v.x);
}
template <> struct TokenVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ float element(const uint4 &v, int i) { return __uint_as_float(word_of(v, i)); }
    static constexpr unsigned kMasked = 0xff800000u;              // -inf
    static __device__ __forceinline__ float2 pair(const uint4 &v, int i) {
        return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                      : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
    }
    static __device__ __forceinline__ float largest(const uint4 &v) {
        return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    template <int COUNT> static __device__ __forceinline__ float largest(const uint4 (&v)[COUNT]) {
        float m = largest(v[0]);
#pragma unroll
        for (int k = 1; k < COUNT; ++k) m = max_nan(m, largest(v[k]));
        return m;
    }
    static __device__ __forceinline__ uint4 pack(const float2 (&g)[2]) {
        return make_uint4(__float_as_uint(g[0].x), __float_as_uint(g[0].y), __float_as_uint(g[1].x),
                          __float_as_uint(g[1].y));
    }
};
template <> struct TokenVec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float element(const uint4 &v, int i) {
        const unsigned w = word_of(v, i >> 1);
        return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w >> 16 : w)));
    }
    static constexpr unsigned kMasked = 0xfc00fc00u;
    static __device__ __forceinline__ __half2 word(unsigned w) { return *reinterpret_cast<__half2 *>(&w); }
    static __device__ __forceinline__ float2 pair(const uint4 &v, int i) {
        return __half22float2(word(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w));
    }
    static __device__ __forceinline__ __half2 largest2(const uint4 &v) {
        return __hmax2_nan(__hmax2_nan(word(v.x), word(v.y)), __hmax2_nan(word(v.z), word(v.w)));
    }
    static __device__ __forceinline__ float largest(const uint4 &v) {
        const __half2 m = largest2(v);
        return max_nan(__low2float(m), __high2float(m));
    }
    template <int COUNT> static __device__ __forceinline__ float largest(const uint4 (&v)[COUNT]) {
        __half2 m = largest2(v[0]);
#pragma unroll
        for (int k = 1; k < COUNT; ++k) m = __hmax2_nan(m, largest2(v[k]));
        return max_nan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ uint4 pack(const float2 (&g)[4]) {
        uint4 r;
        __half2 a = __float22half2_rn(g[0]), b = __float22half2_rn(g[1]), c = __float22half2_rn(g[2]),
                d = __float22half2_rn(g[3]);
        r.x = *reinterpret_cast<unsigned *>(&a);
        r.y = *reinterpret_cast<unsigned *>(&b);
        r.z = *reinterpret_cast<unsigned *>(&c);
        r.w = *reinterpret_cast<unsigned *>(&d);
        return r;
    }
};
template <> struct TokenVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float element(const uint4 &v, int i) {
        const unsigned w = word_of(v, i >> 1);
        return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    }
    static constexpr unsigned kMasked = 0xff80ff80u;
    static __device__ __forceinline__ __nv_bfloat162 word(unsigned w) { return *reinterpret_cast<__nv_bfloat162 *>(&w); }
    static __device__ __forceinline__ float2 pair(const uint4 &v, int i) {
        const unsigned w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    static __device__ __forceinline__ __nv_bfloat162 largest2(const uint4 &v) {
        return __hmax2_nan(__hmax2_nan(word(v.x), word(v.y)), __hmax2_nan(word(v.z), word(v.w)));
    }
    static __device__ __forceinline__ float largest(const uint4 &v) {
        const __nv_bfloat162 m = largest2(v);
        return max_nan(__low2float(m), __high2float(m));
    }
    template <int COUNT> static __device__ __forceinline__ float largest(const uint4 (&v)[COUNT]) {
        __nv_bfloat162 m = largest2(v[0]);
#pragma unroll
        for (int k = 1; k < COUNT; ++k) m = __hmax2_nan(m, largest2(v[k]));
        return max_nan(__low2float(m), __high2float(m));
    }
    static __device__ __forceinline__ uint4 pack(const float2 (&g)[4]) {
        uint4 r;
        __nv_bfloat162 a = __float22bfloat162_rn(g[0]), b = __float22bfloat162_rn(g[1]),
                       c = __float22bfloat162_rn(g[2]), d = __float22bfloat162_rn(g[3]);
        r.x = *reinterpret_cast<unsigned *>(&a);
        r.y = *reinterpret_cast<unsigned *>(&b);
        r.z = *reinterpret_cast<unsigned *>(&c);
        r.w = *reinterpret_cast<unsigned *>(&d);
        return r;
    }
};

template <typename T> __device__ __forceinline__ uint4 masked_vec() {
    constexpr unsigned w = TokenVec<T>::kMasked;
    return make_uint4(w, w, w, w);
}

// ---- which part of a row a block reads

// Elements [first, last) of a row; [body, body_end) of them are whole 16-byte vectors at 16-byte addresses.  The ragged
// ends belong to the first and the last part.
struct RowPart {
    int first, body, body_end, last;
};
template <typename T> __device__ __forceinline__ int ragged_head(const T *row, int V) {
    const int off = int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    return min(V, off ? TokenVec<T>::N - off : 0);
}
// Part `rank` of 2^shift parts of a row (no division: it would cost a thread as much as 20 elements).
template <typename T>
__device__ __forceinline__ RowPart row_part(const T *row, int V, int rank, int shift) {
    constexpr int N = TokenVec<T>::N;
    const int head = ragged_head(row, V);
    const int64_t nvec = (V - head) / N;
    RowPart r;
    r.body = head + int(nvec * rank >> shift) * N;
    r.body_end = head + int(nvec * (rank + 1) >> shift) * N;
    r.first = rank == 0 ? 0 : r.body;
    r.last = rank + 1 == 1 << shift ? V : r.body_end;
    return r;
}
// Chunk `index` of `chunks` chunks of `vectors` vectors (the last one: what is left).
template <typename T>
__device__ __forceinline__ RowPart row_chunk(const T *row, int V, int index, int chunks, int vectors) {
    constexpr int N = TokenVec<T>::N;
    const int head = ragged_head(row, V), nvec = (V - head) / N;
    RowPart r;
    r.body = head + min(nvec, index * vectors) * N;
    r.body_end = head + min(nvec, (index + 1) * vectors) * N;
    r.first = index == 0 ? 0 : r.body;
    r.last = index == chunks - 1 ? V : r.body_end;
    return r;
}
// The i-th element of a part that no vector covers (i < ragged_count), as an index into the row.
__device__ __forceinline__ int ragged_count(const RowPart &r) { return (r.body - r.first) + (r.last - r.body_end); }
__device__ __forceinline__ int ragged_index(const RowPart &r, int i) {
    const int head = r.body - r.first;
    return i < head ? r.first + i : r.body_end + (i - head);
}

// ---- statistics

template <bool ENTROPY> struct RowStat {
    float m, s, u;
    __device__ __forceinline__ void init() {
        m = -INFINITY;
        s = 0.f;
        u = 0.f;
    }
    // Sums relative to `to` >= m from here on.
    __device__ __forceinline__ void raise(float to, float c) {
        float w = 0.f, d = 0.f;
        if (m != -INFINITY) {
            d = max_nan((m - reference_of(to)) * c, kTokenFloor);
            w = ex2f(d);
        }
        if (ENTROPY) u = w * fmaf(d, s, u);
        s *= w;
        m = to;
    }
    __device__ __forceinline__ void add(float x, float c) {          // one element
        const float to = max_nan(m, x);
        if (rises(to, m)) raise(to, c);
        const float z = max_nan((x - reference_of(m)) * c, kTokenFloor), e = ex2f(z);
        s += e;
        if (ENTROPY) u = fmaf(e, z, u);
    }
    // Some vectors; returns the largest logit among them.
    template <typename T, int COUNT> __device__ __forceinline__ float add(const uint4 (&v)[COUNT], float c) {
        const float own = TokenVec<T>::largest(v), to = max_nan(m, own);
        if (rises(to, m)) raise(to, c);
        const pk_t negm = psplat(-reference_of(m)), cc = psplat(c);
        pk_t s2 = psplat(0.f), u2 = psplat(0.f);
#pragma unroll
        for (int k = 0; k < COUNT; ++k) {
#pragma unroll
            for (int i = 0; i < TokenVec<T>::N / 2; ++i) {
                float2 z = upk2(pmul(padd(pk2(TokenVec<T>::pair(v[k], i)), negm), cc));
                if (ENTROPY) {
                    z.x = max_nan(z.x, kTokenFloor);
                    z.y = max_nan(z.y, kTokenFloor);
                }
                const pk_t zz = pk2(z), e = pex2(zz);
                s2 = padd(s2, e);
                if (ENTROPY) u2 = pfma(e, zz, u2);
            }
        }
        const float2 a = upk2(s2);
        s += a.x + a.y;
        if (ENTROPY) {
            const float2 b = upk2(u2);
            u += b.x + b.y;
        }
        return own;
    }
    // All lanes of a warp: the warp's statistics in every lane.
    __device__ __forceinline__ void join_warp(float c) {
        float to = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) to = max_nan(to, __shfl_xor_sync(0xffffffffu, to, o));
        raise(to, c);
        s = warp_sum(s);
        if (ENTROPY) u = warp_sum(u);
    }
};

// The statistics of a part of a row, the vectors dealt out to G threads in turn; `load(i)` gives the vector that
// starts at element i.  Every thread returns its own share.  `seen(k, m)`: m is the largest logit among the thread's
// vectors from its k-th on that were just taken in (up to kTokenUnroll of them).  `ready(k)` is called before the
// thread's vectors from its k-th on, up to kTokenUnroll of them, are loaded (k a multiple of that).
template <typename T, int G, bool ENTROPY, typename Load, typename Seen, typename Ready>
__device__ __forceinline__ void scan_part(const T *row, const RowPart &part, int t, float c, RowStat<ENTROPY> &st,
                                          Load load, Seen seen, Ready ready) {
    constexpr int N = TokenVec<T>::N, U = kTokenUnroll;
    const int last_lane = (31 - (t & 31)) * N;              // (a warp takes its steps together)
    int i = part.body + t * N, k = 0;
    for (; int64_t(i) + last_lane + (U - 1) * (G * N) < part.body_end; i += U * G * N, k += U) {
        uint4 v[U];
        ready(k);
#pragma unroll
        for (int h = 0; h < U; ++h) v[h] = load(i + h * (G * N));
        seen(k, st.template add<T>(v, c));
    }
    // what is left, up to four vectors, some of them not in every lane: all on their way before the first is worked on;
    // three or four are a batch again, with masked vectors where there are none (one look at the maximum)
    uint4 v[U];
    if (i < part.body_end) ready(k);
#pragma unroll
    for (int h = 0; h < U; ++h) v[h] = int64_t(i) + h * (G * N) < part.body_end ? load(i + h * (G * N)) : masked_vec<T>();
    if (__any_sync(0xffffffffu, int64_t(i) + 2 * (G * N) < part.body_end)) {
        const float most = st.template add<T>(v, c);
        if (i < part.body_end) seen(k, most);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (int64_t(i) + h * (G * N) < part.body_end) seen(k + h, st.template add<T>(reinterpret_cast<const uint4 (&)[1]>(v[h]), c));
    }
    if (t < ragged_count(part)) st.add(to_f32(row[ragged_index(part, t)]), c);
}
template <typename T, int G, bool ENTROPY, typename Load>
__device__ __forceinline__ void scan_part(const T *row, const RowPart &part, int t, float c, RowStat<ENTROPY> &st,
                                          Load load) {
    scan_part<T, G>(row, part, t, c, st, load, [](int, float) {}, [](int) {});
}

// ---- host side: launches of clusters of blocks

template <typename... KArgs, typename... Args>
inline int launch_cluster(void (*kernel)(KArgs...), int64_t grid, int block, size_t smem, int cluster, bool dependent,
                          cudaStream_t stream, const char *what, Args &&...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(grid));
    cfg.blockDim = dim3(unsigned(block));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = unsigned(cluster);
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (dependent) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
    const int rc = launch_status(what);
    if (rc == B200_OK && e != cudaSuccess) {
        set_error("%s: %s", what, cudaGetErrorString(e));
        return B200_ERR_LAUNCH;
    }
    return rc;
}

// Whether a pointer (null included) lies on a multiple of `bytes`, a power of two.
inline bool lies_on(const void *p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// 16-byte vectors of a row, at most.
inline int64_t row_vectors(int64_t V, int dtype) { return V * int64_t(dtype_size(dtype)) / 16; }

}  // namespace
}  // namespace b200
