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
// Bound: HBM (2 s D per row forward, 3 s D backward, s the element's bytes).
#include "common.cuh"

namespace b200 {
namespace {

struct NormParams {
    const void *x, *w, *b, *dy;
    void *y, *dx;
    float2 *stats;              // {mean, r} per row
    float *partial;             // [blocks][2][D]
    int64_t x_stride, dy_stride, rows;
    int D;
    float eps;
};

// V elements of T as floats.
template <typename T, int V> struct Pack {
    T v[V];
};
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

// Sum over the G threads of a row; every thread gets it.  `sh`: G / 32 floats of its own for each call.
template <int G> __device__ __forceinline__ float row_sum(float v, float *sh) {
    v = warp_sum(v);
    if (G == 32) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(lane < G / 32 ? sh[lane] : 0.f);
}

// A thread holds N packs of V elements of its row: pack i starts at column (i * G + t) * V.
template <typename T> constexpr int wide = 16 / int(sizeof(T));
template <int V> constexpr int packs = V == 1 ? 16 : 4;

template <typename T, typename P, int V, int G>
__global__ void __launch_bounds__(G == 32 ? 256 : G) norm_forward_kernel(const NormParams p) {
    constexpr int N = packs<V>;
    __shared__ float sh[2][32];
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t r = G == 32 ? int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5) : int64_t(blockIdx.x);
    if (r >= p.rows) return;
    const T *x = static_cast<const T *>(p.x) + r * p.x_stride;
    T *y = static_cast<T *>(p.y) + r * int64_t(p.D);
    float v[N][V];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int j = (i * G + t) * V;
        if (j < p.D) {
            load_pack<T, V>(x + j, v[i]);
#pragma unroll
            for (int k = 0; k < V; ++k) sum += v[i][k];
        }
    }
    const float inv_d = 1.f / float(p.D);
    const float mean = row_sum<G>(sum, sh[0]) * inv_d;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if ((i * G + t) * V < p.D) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                v[i][k] -= mean;
                sum = fmaf(v[i][k], v[i][k], sum);
            }
        }
    }
    const float rstd = rsqrtf(row_sum<G>(sum, sh[1]) * inv_d + p.eps);
    if (t == 0 && p.stats) p.stats[r] = make_float2(mean, rstd);
    const P *w = static_cast<const P *>(p.w), *b = static_cast<const P *>(p.b);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int j = (i * G + t) * V;
        if (j < p.D) {
            float a[V];
#pragma unroll
            for (int k = 0; k < V; ++k) v[i][k] *= rstd;
            if (w) {
                load_pack<P, V>(w + j, a);
#pragma unroll
                for (int k = 0; k < V; ++k) v[i][k] *= a[k];
            }
            if (b) {
                load_pack<P, V>(b + j, a);
#pragma unroll
                for (int k = 0; k < V; ++k) v[i][k] += a[k];
            }
            store_pack<T, V>(y + j, v[i]);
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

template <typename T, typename P, int V, int G>
__global__ void __launch_bounds__(G == 32 ? 256 : G) norm_backward_kernel(const NormParams p) {
    constexpr int N = packs<V>;
    __shared__ float sh[4][32];
    extern __shared__ float columns[];                      // G == 32: [2][D]
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int64_t first = G == 32 ? int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5) : int64_t(blockIdx.x);
    const int64_t step = G == 32 ? int64_t(gridDim.x) * 8 : int64_t(gridDim.x);
    const P *w = static_cast<const P *>(p.w);
    const float inv_d = 1.f / float(p.D);
    float dw[N][V], db[N][V];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) dw[i][k] = db[i][k] = 0.f;
    int turn = 0;                                           // (the sums of two rows in a row do not share memory)
    for (int64_t r = first; r < p.rows; r += step, turn ^= 2) {
        const T *x = static_cast<const T *>(p.x) + r * p.x_stride, *dy = static_cast<const T *>(p.dy) + r * p.dy_stride;
        T *dx = static_cast<T *>(p.dx) + r * int64_t(p.D);
        const float2 st = p.stats[r];
        float h[N][V], g[N][V];
        float sg = 0.f, sgh = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (i * G + t) * V;
            if (j < p.D) {
                load_pack<T, V>(x + j, h[i]);
                load_pack<T, V>(dy + j, g[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (i * G + t) * V;
            if (j < p.D) {
                float a[V];
                if (w) load_pack<P, V>(w + j, a);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    h[i][k] = (h[i][k] - st.x) * st.y;
                    dw[i][k] = fmaf(g[i][k], h[i][k], dw[i][k]);
                    db[i][k] += g[i][k];
                    if (w) g[i][k] *= a[k];
                    sg += g[i][k];
                    sgh = fmaf(g[i][k], h[i][k], sgh);
                }
            }
        }
        sg = warp_sum(sg);
        sgh = warp_sum(sgh);
        if (G > 32) {
            const int lane = threadIdx.x & 31;
            if (lane == 0) {
                sh[turn][threadIdx.x >> 5] = sg;
                sh[turn + 1][threadIdx.x >> 5] = sgh;
            }
            __syncthreads();
            sg = warp_sum(lane < G / 32 ? sh[turn][lane] : 0.f);
            sgh = warp_sum(lane < G / 32 ? sh[turn + 1][lane] : 0.f);
        }
        sg *= inv_d;
        sgh *= inv_d;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int j = (i * G + t) * V;
            if (j < p.D) {
#pragma unroll
                for (int k = 0; k < V; ++k) g[i][k] = st.y * (g[i][k] - sg - h[i][k] * sgh);
                store_pack<T, V>(dx + j, g[i]);
            }
        }
    }
    if (!p.partial) return;
    float *out = p.partial + int64_t(blockIdx.x) * 2 * p.D;
    if (G == 32) {                                          // the eight warps' columns, one warp after the other
        for (int j = threadIdx.x; j < 2 * p.D; j += 256) columns[j] = 0.f;
        for (int warp = 0; warp < 8; ++warp) {
            __syncthreads();
            if (int(threadIdx.x >> 5) == warp) {
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const int j = (i * G + t) * V + k;
                        if (j < p.D) {
                            columns[j] += dw[i][k];
                            columns[p.D + j] += db[i][k];
                        }
                    }
            }
        }
        __syncthreads();
        for (int j = threadIdx.x; j < 2 * p.D; j += 256) out[j] = columns[j];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int j = (i * G + t) * V + k;
                if (j < p.D) {
                    out[j] = dw[i][k];
                    out[p.D + j] = db[i][k];
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

// Threads to a row: the fewest of 32, 128, 256, 512, 1024 that hold it, 0 if none does.
inline int row_threads(int D, int v) {
    const int per = v == 1 ? 16 : 4 * v;
    for (int g : {32, 128, 256, 512, 1024})
        if (int64_t(g) * per >= D) return g;
    return 0;
}
// Backward holds two rows and two sums a column in registers: up to 512 threads' worth.
inline int backward_threads(int D, int v) {
    const int g = row_threads(D, v);
    return g <= 512 ? g : 0;
}
inline int backward_blocks(int64_t rows, int g) {
    const int64_t per_block = g == 32 ? 8 : 1, most = g == 0 ? 64 : int64_t(sm_count()) * (g <= 128 ? 2 : 1);
    const int64_t want = (rows + per_block - 1) / per_block;
    return int(want < 1 ? 1 : want > most ? most : want);
}
inline bool on16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, typename P> struct NormLaunch {
    template <int V, int G> static int forward(const NormParams &p, cudaStream_t s) {
        const int64_t grid = G == 32 ? (p.rows + 7) / 8 : p.rows;
        norm_forward_kernel<T, P, V, G><<<unsigned(grid), G == 32 ? 256 : G, 0, s>>>(p);
        return launch_status("layer norm kernel launch");
    }
    template <int V> static int forward_of(const NormParams &p, cudaStream_t s) {
        switch (row_threads(p.D, V)) {
            case 32: return forward<V, 32>(p, s);
            case 128: return forward<V, 128>(p, s);
            case 256: return forward<V, 256>(p, s);
            case 512: return forward<V, 512>(p, s);
            case 1024: return forward<V, 1024>(p, s);
        }
        norm_forward_any_kernel<T, P><<<unsigned(p.rows), 1024, 0, s>>>(p);
        return launch_status("layer norm kernel launch");
    }
    static int forward(const NormParams &p, cudaStream_t s) {
        constexpr int V = wide<T>;
        const bool vec = p.D % V == 0 && on16(p.x) && on16(p.y) && (p.rows < 2 || p.x_stride % V == 0) && on16(p.w) && on16(p.b);
        return vec ? forward_of<V>(p, s) : forward_of<1>(p, s);
    }
    template <int V, int G> static int backward(const NormParams &p, int blocks, cudaStream_t s) {
        const size_t smem = G == 32 ? size_t(p.D) * 8 : 0;
        norm_backward_kernel<T, P, V, G><<<unsigned(blocks), G == 32 ? 256 : G, smem, s>>>(p);
        return launch_status("layer norm gradient kernel launch");
    }
    template <int V> static int backward_of(const NormParams &p, int g, int blocks, cudaStream_t s) {
        switch (g) {
            case 32: return backward<V, 32>(p, blocks, s);
            case 128: return backward<V, 128>(p, blocks, s);
            case 256: return backward<V, 256>(p, blocks, s);
            case 512: return backward<V, 512>(p, blocks, s);
        }
        norm_backward_any_kernel<T, P><<<unsigned(p.rows), 1024, 0, s>>>(p);
        if (const int rc = launch_status("layer norm gradient kernel launch")) return rc;
        if (!p.partial) return B200_OK;
        norm_columns_any_kernel<T><<<dim3(unsigned((p.D + 255) / 256), unsigned(blocks)), 256, 0, s>>>(p);
        return launch_status("layer norm column kernel launch");
    }
    static int backward(const NormParams &p, void *dw, void *db, cudaStream_t s) {
        constexpr int V = wide<T>;
        const bool vec = p.D % V == 0 && on16(p.x) && on16(p.dx) && on16(p.dy) && on16(p.w) &&
                         (p.rows < 2 || (p.x_stride % V == 0 && p.dy_stride % V == 0));
        const int g = vec ? backward_threads(p.D, V) : backward_threads(p.D, 1);
        const int blocks = backward_blocks(p.rows, g);
        if (p.rows > 0) {
            const int rc = vec ? backward_of<V>(p, g, blocks, s) : backward_of<1>(p, g, blocks, s);
            if (rc) return rc;
        }
        if (!p.partial) return B200_OK;
        norm_columns_kernel<P><<<unsigned((2 * int64_t(p.D) + 31) / 32), 512, 0, s>>>(
            p.partial, p.rows > 0 ? blocks : 0, p.D, static_cast<P *>(dw), static_cast<P *>(db));
        return launch_status("layer norm column kernel launch");
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
    if (!(eps >= 0.f) || stride < 0 || (rows > 0 && (!x || !y)) || (reinterpret_cast<uintptr_t>(stats) & 7)) {
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
    const int64_t most = int64_t(sm_count()) * 2;
    return size_t(rows < 1 ? 1 : rows < most ? rows : most) * size_t(D) * 8;
}

extern "C" int b200_layer_norm_backward(const void *x, const void *weight, const void *stats, const void *dy, void *dx,
                                        void *dweight, void *dbias, void *scratch, size_t scratch_bytes, int64_t rows,
                                        int64_t D, int64_t stride, int64_t dy_stride, int dtype, int param_dtype,
                                        void *stream) {
    const char *who = "b200_layer_norm_backward";
    if (const int rc = check_norm(who, rows, D, dtype, param_dtype)) return rc;
    if (stride < 0 || dy_stride < 0 || (rows > 0 && (!x || !dy || !dx || !stats)) || (reinterpret_cast<uintptr_t>(stats) & 7)) {
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
