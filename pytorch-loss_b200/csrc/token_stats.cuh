// The forward kernel of the log-probability and distillation operators (token_logprobs.cu, top_distill.cu) and the
// kernel that writes a gradient from a row's statistics.  Formulas: token_rows.cuh.
#pragma once
#include "token_rows.cuh"

namespace b200 {
namespace {

// kTokens: one given token per row, entropy, best alternatives.  kList: a list of tokens with weights per row.
enum TokenMode { kTokens = 0, kList = 1 };

struct TokenParams {
    const void *x;              // logits: row r starts at element r * stride
    int64_t stride, rows;
    int V;
    float c, inv_t;             // log2(e) / temperature, 1 / temperature
    const int64_t *ids;         // kTokens: [rows]; kList: [rows, K]
    const float *weight;        // kList: [rows, K], a row sums to 1, 0 where nothing is asked
    const float *base;          // kList: [rows], sum of w log w; +inf: nothing is asked of the row, NaN: a bad token
    int64_t ignore;
    int K;                      // kTokens: alternatives; kList: length of the lists
    float *out, *entropy;       // log probabilities and entropies, or losses
    float4 *stats;              // {m, 1 / s, u / s, log2 s} for the gradient (may be null)
    float *top_logprobs;
    int64_t *top_tokens;
    int part_shift;             // 2^part_shift blocks of a cluster share a row
};

// ---- alternatives
// Order: larger logits first, the lower index first among equals (-0 = +0), NaN in front of everything.  A key holds
// that order in one unsigned number: the value's bits made monotone, above the inverted index.
__device__ __forceinline__ unsigned value_key(float x) {
    unsigned b = __float_as_uint(x);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
    if ((b << 1) == 0u) b = 0u;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(unsigned k) {
    return k == 0xffffffffu ? __uint_as_float(0x7fc00000u)
                            : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long top_key(float x, int j) {
    return (static_cast<unsigned long long>(value_key(x)) << 32) | unsigned(~j);
}

template <int G> __device__ __forceinline__ void group_sync() {
    if (G == 32) __syncwarp();
    else __syncthreads();
}

// Candidates that a group of G threads keeps.  32 lanes: their lists are at most 32 long (largest() below).
template <int G> constexpr int kCandidates = G == 32 ? 256 : 1024;

// A thread's vectors fall into up to kSegments segments of 2^shift vectors (4 at least), whose maxima are kept.
constexpr int kSegments = 8;
template <int N, int G> __device__ __forceinline__ int segment_shift(const RowPart &part) {
    const int per = ((part.body_end - part.body) / N + G - 1) / G;      // vectors of thread 0
    const int least = (per + kSegments - 1) / kSegments;
    return least <= 4 ? 2 : 32 - __clz(least - 1);
}

template <int G, bool TOP> struct TokenShared {
    float m[G / 32], s[G / 32], u[G / 32];
    float joined[3];                                     // this block's share of the row, for the cluster
    int count, member_count;
    unsigned bound;
    unsigned short keys[TOP ? G : 1];                    // upper halves of the keys of the threads' maxima ...
    unsigned short segment[TOP ? kSegments : 1][TOP ? G : 1];   // ... and of those of their segments
    unsigned short members[TOP ? kSegments * G : 1];     // segments that reach the bound: thread + G * segment
    unsigned hist[TOP ? 256 : 1];
    alignas(16) unsigned long long cand[TOP ? kCandidates<G> : 1];
    unsigned long long best[TOP ? kMaxList : 1];
};

// The smallest key among the `want` largest of the part (0 if the part has no more than that): eight passes over the
// part, one digit of the 64-bit keys each.  Only for parts whose candidates do not fit: logits that agree at
// thousands of places (a mask that leaves fewer than `want` is such a row), or lie so that a few threads see all the large
// ones.  Element by element, so a row costs 50 times what it does otherwise: [4096, 32768] float16 with 10 live logits and
// 20 alternatives 3610 us against 72, one row of 131072 142 against 10.
template <typename T, int G, bool TOP>
__device__ __noinline__ unsigned long long exact_bound(const T *row, RowPart part, int t, int want,
                                                       TokenShared<G, TOP> &sh) {
    if (part.last - part.first <= want) return 0ull;
    unsigned long long prefix = 0ull;
    for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = t; i < 256; i += G) sh.hist[i] = 0u;
        group_sync<G>();
        for (int base = part.first; base < part.last; base += G) {
            const int j = base + t;
            const unsigned long long key = j < part.last ? top_key(to_f32(row[j]), j) : 0ull;
            const bool in = j < part.last && (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8)));
            const unsigned digit = unsigned(key >> shift) & 255u;
            const unsigned live = __ballot_sync(0xffffffffu, in);
            if (live == 0u) continue;
            const unsigned first = __shfl_sync(0xffffffffu, digit, __ffs(live) - 1);
            if (__all_sync(0xffffffffu, !in || digit == first)) {       // (equal logits: one addition for all lanes)
                if ((t & 31) == 0) atomicAdd(&sh.hist[first], unsigned(__popc(live)));
            } else if (in) {
                atomicAdd(&sh.hist[digit], 1u);
            }
        }
        group_sync<G>();
        // from the largest digit down: the one at which `want` is reached (every warp finds the same)
        unsigned mine = 0u;
        const int lane = t & 31;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine += sh.hist[255 - lane * 8 - i];
        unsigned upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        const int owner = __ffs(__ballot_sync(0xffffffffu, upto >= unsigned(want))) - 1;
        int digit = 0, left = 0;
        if (lane == owner) {
            left = want - int(upto - mine);
            digit = 255 - lane * 8;
            while (int(sh.hist[digit]) < left) left -= int(sh.hist[digit--]);
        }
        want = __shfl_sync(0xffffffffu, left, owner);
        prefix |= static_cast<unsigned long long>(__shfl_sync(0xffffffffu, digit, owner)) << shift;
        group_sync<G>();
    }
    return prefix;
}

// How many of n keys are larger than k.
__device__ __forceinline__ int larger_keys(const unsigned long long *keys, int n, unsigned long long k) {
    int a = 0, b = 0;
    int j = 0;
#pragma unroll 4
    for (; j + 1 < n; j += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(keys + j);
        a += two.x > k ? 1 : 0;
        b += two.y > k ? 1 : 0;
    }
    if (j < n) a += keys[j] > k ? 1 : 0;
    return a + b;
}

// Of n candidates (0: none) those that reach the K-th largest of their upper 16 bits; returns how many these are.
template <int G, bool TOP> __device__ __forceinline__ int narrow(int n, int t, int K, TokenShared<G, TOP> &sh) {
    constexpr int PER = kCandidates<G> / G, WARPS = G / 32;
    unsigned long long own[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) own[i] = t + i * G < n ? sh.cand[t + i * G] : 0ull;
    unsigned bound = 0u;
#pragma unroll 1
    for (int bit = 15; bit >= 0; --bit) {
        const unsigned trial = bound | (1u << bit);
        unsigned of = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) of += unsigned(own[i] >> 48) >= trial ? 1u : 0u;
        of = __reduce_add_sync(0xffffffffu, of);
        if (G > 32) {
            if ((t & 31) == 0) sh.hist[bit * WARPS + (t >> 5)] = of;
            __syncthreads();
            of = 0u;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) of += sh.hist[bit * WARPS + i];
        }
        if (of >= unsigned(K)) bound = trial;
    }
    group_sync<G>();                                        // (everybody has read the candidates and their number)
    if (t == 0) sh.count = 0;
    group_sync<G>();
#pragma unroll
    for (int i = 0; i < PER; ++i)
        if (own[i] && unsigned(own[i] >> 48) >= bound) sh.cand[atomicAdd(&sh.count, 1)] = own[i];
    group_sync<G>();
    return sh.count;
}

// sh.best[0..K) = the K largest keys of the part in order, 0 behind its end.  `m`: the largest logit of each thread.
//
// The K-th largest of the threads' maxima is a lower bound of the K-th largest logit, so only the few segments whose
// maximum reaches it are read again (from L2, by all threads at once), and what is kept of them is little more than K.
// The bound is taken to the upper 16 bits of the keys: a warp finds it in 16 steps.  The order among the kept is a count
// of larger keys.
template <typename T, int G, bool TOP, typename Load>
__device__ __forceinline__ void largest(const T *row, const RowPart &part, int t, float m, int K,
                                        TokenShared<G, TOP> &sh, Load load) {
    constexpr int N = TokenVec<T>::N, PER = G / 32, CAP = kCandidates<G>;
    const unsigned key = value_key(m) >> 16;
    sh.keys[t] = static_cast<unsigned short>(key);
    if (t == 0) sh.count = sh.member_count = 0;
    group_sync<G>();
    if (t < 32) {
        unsigned k[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) k[i] = sh.keys[t + 32 * i];
        unsigned bound = 0u;
        if (PER > 1 && K <= 24) {                           // (32 maxima say enough)
#pragma unroll
            for (int i = 1; i < PER; ++i) k[0] = max(k[0], k[i]);
#pragma unroll 1
            for (int bit = 15; bit >= 0; --bit) {
                const unsigned trial = bound | (1u << bit);
                if (__popc(__ballot_sync(0xffffffffu, k[0] >= trial)) >= K) bound = trial;
            }
        } else {
#pragma unroll 1
            for (int bit = 15; bit >= 0; --bit) {
                const unsigned trial = bound | (1u << bit);
                unsigned n = 0u;
#pragma unroll
                for (int i = 0; i < PER; ++i) n += k[i] >= trial ? 1u : 0u;
                if (__reduce_add_sync(0xffffffffu, n) >= unsigned(K)) bound = trial;
            }
        }
        if (t == 0) sh.bound = bound;
    }
    group_sync<G>();
    const unsigned bound = sh.bound;
    // (the bound as a logit: the smallest value with these upper 16 bits; NaN and "everything" pass every comparison)
    const float least = bound >= 0xffffu ? INFINITY : bound == 0u ? -INFINITY : key_value(bound << 16);
    auto keep = [&](float x, int j) {
        if (x < least) return;
        const unsigned long long k = top_key(x, j);
        if (unsigned(k >> 48) >= bound) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < CAP) sh.cand[at] = k;
        }
    };
    const int shift = segment_shift<N, G>(part);
    if (key >= bound) {
        const int per = ((part.body_end - part.body) / N - t + G - 1) / G;          // this thread's vectors
        for (int i = 0; i << shift < per; ++i)
            if (sh.segment[i][t] >= bound) sh.members[atomicAdd(&sh.member_count, 1)] = static_cast<unsigned short>(t + G * i);
        if (t < ragged_count(part)) {
            const int j = ragged_index(part, t);
            keep(to_f32(row[j]), j);
        }
    }
    group_sync<G>();
    // the vectors of these segments, dealt out to all threads: `lanes` threads to each
    const int members = sh.member_count, lane_shift = min(shift, 5), lanes = 1 << lane_shift;
    for (int i = t >> lane_shift; i < members; i += G >> lane_shift) {
        const int owner = sh.members[i] % G, first = sh.members[i] / G << shift;
        for (int k = t & (lanes - 1); k < 1 << shift; k += lanes) {
            const int64_t at = part.body + (owner + int64_t(first + k) * G) * N;
            if (at >= part.body_end) break;
            const uint4 v = load(int(at));
            // (which elements first: a warp then goes once or twice through what it costs to keep one, not N times)
            unsigned wanted = 0u;
#pragma unroll
            for (int h = 0; h < N / 2; ++h) {
                const float2 x = TokenVec<T>::pair(v, h);
                wanted |= (x.x < least ? 0u : 1u << (2 * h)) | (x.y < least ? 0u : 2u << (2 * h));
            }
            while (wanted) {
                const int e = __ffs(wanted) - 1;
                wanted &= wanted - 1u;
                keep(TokenVec<T>::element(v, e), int(at) + e);
            }
        }
    }
    group_sync<G>();
    int n = sh.count;
    if (n > CAP) {
        const unsigned long long least = exact_bound<T, G, TOP>(row, part, t, K, sh);
        if (t == 0) sh.count = 0;
        group_sync<G>();
        for (int j = part.first + t; j < part.last; j += G) {
            const unsigned long long k = top_key(to_f32(row[j]), j);
            if (k >= least) sh.cand[atomicAdd(&sh.count, 1)] = k;       // (at most K <= kMaxList of them)
        }
        group_sync<G>();
        n = sh.count;
    } else if (n > 2 * K + 32) {
        n = narrow<G>(n, t, K, sh);                         // (short rows and long lists: the threads' maxima say little)
    }
    for (int i = t; i < K; i += G)
        if (i >= n) sh.best[i] = 0ull;
    for (int i = t; i < n; i += G) {
        const unsigned long long k = sh.cand[i];
        const int rank = larger_keys(sh.cand, n, k);
        if (rank < K) sh.best[rank] = k;
    }
    group_sync<G>();
}

// G threads to a row (32: eight rows to a block), or the G threads of each of `parts` blocks.
// Bound: HBM, the logits once; instruction issue and the 16 exponentials a clock of an SM are next (16-bit logits
// take 11.6 of them at HBM speed).
template <typename T, int G, int MODE, bool TOP>
__global__ void __launch_bounds__(G == 32 ? 256 : G, G == 32 ? 5 : 1536 / G) token_stats_kernel(const TokenParams p) {
    constexpr bool ENTROPY = MODE == kTokens;
    constexpr int WARPS = G / 32, GROUPS = G == 32 ? 8 : 1;
    __shared__ TokenShared<G, TOP> shared[GROUPS];
    const int t = G == 32 ? threadIdx.x & 31 : threadIdx.x, lane = threadIdx.x & 31;
    TokenShared<G, TOP> &sh = shared[G == 32 ? threadIdx.x >> 5 : 0];
    const int parts = 1 << (G == 32 ? 0 : p.part_shift);
    const int rank = G == 32 ? 0 : int(blockIdx.x) & (parts - 1);
    const int64_t r = G == 32 ? int64_t(blockIdx.x) * GROUPS + (threadIdx.x >> 5) : int64_t(blockIdx.x >> p.part_shift);
    if (r >= p.rows) return;
    const T *row = static_cast<const T *>(p.x) + r * p.stride;

    // rows that are not asked for are not read (the blocks of a cluster leave together)
    int64_t token = 0;
    float given = 0.f;
    bool bad = false;
    if (MODE == kTokens) {
        token = p.ids[r];
        if (token == p.ignore) {
            if (rank == 0) {
                if (t == 0) {
                    p.out[r] = 0.f;
                    p.entropy[r] = 0.f;
                }
                if (TOP)
                    for (int i = t; i < p.K; i += G) {
                        p.top_logprobs[r * p.K + i] = 0.f;
                        p.top_tokens[r * p.K + i] = -1;
                    }
            }
            return;
        }
        bad = token < 0 || token >= p.V;
        if (rank == 0 && t == 0 && !bad) given = to_f32(row[token]);
    } else {
        pdl_wait();                                         // (the lists' kernel)
        given = p.base[r];
        if (given == INFINITY) {
            if (rank == 0 && t == 0) p.out[r] = 0.f;
            return;
        }
    }

    const RowPart part = row_part(row, p.V, rank, G == 32 ? 0 : p.part_shift);
    auto load = [row](int i) { return ld_stream16<uint4>(row + i); };
    RowStat<ENTROPY> st;
    st.init();
    if constexpr (TOP) {
        const int shift = segment_shift<TokenVec<T>::N, G>(part);
        int current = 0;
        float most = -INFINITY;
        scan_part<T, G>(row, part, t, p.c, st, load, [&](int k, float m) {
            if (k >> shift != current) {
                sh.segment[current][t] = static_cast<unsigned short>(value_key(most) >> 16);
                current = k >> shift;
                most = -INFINITY;
            }
            most = max_nan(most, m);
        }, [](int) {});
        sh.segment[current][t] = static_cast<unsigned short>(value_key(most) >> 16);
    } else {
        scan_part<T, G>(row, part, t, p.c, st, load);
    }
    const float own_max = st.m;
    st.join_warp(p.c);
    if (G > 32) {
        if (lane == 0) {
            sh.m[t >> 5] = st.m;
            sh.s[t >> 5] = st.s;
            if (ENTROPY) sh.u[t >> 5] = st.u;
        }
        __syncthreads();
        if (t < 32) {                                       // the block's statistics: the first warp's business
            st.init();
            if (lane < WARPS) {
                st.m = sh.m[lane];
                st.s = sh.s[lane];
                if (ENTROPY) st.u = sh.u[lane];
            }
            st.join_warp(p.c);
        }
    }
    if constexpr (TOP) largest<T, G, TOP>(row, part, t, own_max, p.K, sh, load);

    int found = TOP ? p.K : 0;
    if (G > 32 && parts > 1) {
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        if (t == 0) {
            sh.joined[0] = st.m;
            sh.joined[1] = st.s;
            sh.joined[2] = ENTROPY ? st.u : 0.f;
        }
        cluster.sync();
        if (rank == 0) {
            if (t < 32) {
                st.init();
                if (lane < parts) {
                    const float *other = cluster.map_shared_rank(&sh.joined[0], lane);
                    st.m = other[0];
                    st.s = other[1];
                    if (ENTROPY) st.u = other[2];
                }
                st.join_warp(p.c);
            }
            if constexpr (TOP) {
                found = parts * p.K;                        // (0 where a part has fewer logits)
                for (int i = t; i < found; i += G)
                    sh.cand[i] = cluster.map_shared_rank(&sh.best[0], i / p.K)[i % p.K];
            }
        }
        cluster.sync();                                     // (nobody leaves while its memory is read)
        if (rank != 0) return;
        if constexpr (TOP) {
            if (found > 2 * p.K + 32) found = narrow<G, TOP>(found, t, p.K, sh);
        }
    }
    if constexpr (TOP) {
        // the first warp's statistics for all
        if (t == 0) {
            sh.joined[0] = reference_of(st.m);
            sh.joined[1] = st.s == 0.f ? INFINITY : log2f(st.s);    // (a row of -inf: every log probability is -inf)
        }
        group_sync<G>();
        const float m = sh.joined[0], log2s = sh.joined[1];
        for (int i = t; i < found; i += G) {
            const unsigned long long k = parts > 1 ? sh.cand[i] : sh.best[i];
            const int place = parts > 1 ? larger_keys(sh.cand, found, k) : i;
            if (k == 0ull || place >= p.K) continue;
            const float x = key_value(unsigned(k >> 32));
            p.top_logprobs[r * p.K + place] = log2s == INFINITY ? -INFINITY : log_prob(x, m, p.inv_t, log2s);
            p.top_tokens[r * p.K + place] = int64_t(~unsigned(k));
        }
    }
    if (t >= 32) return;

    const float m = reference_of(st.m), log2s = log2f(st.s);
    const bool nothing = st.s == 0.f;                       // a row of -inf
    if (MODE == kTokens) {
        if (t == 0) {
            const float mean = nothing ? 0.f : st.u / st.s;
            p.out[r] = bad ? __int_as_float(0x7fc00000) : nothing ? -INFINITY
                                                                  : log_prob(given, m, p.inv_t, log2s);
            p.entropy[r] = nothing ? 0.f : max_nan(kTokenLn2 * (log2s - mean), 0.f);
            if (p.stats) p.stats[r] = make_float4(m, nothing ? 0.f : 1.f / st.s, mean, log2s);
        }
    } else {
        // sum of w (log w - log p) over the list; `given` holds the sum of w log w
        float part_loss = 0.f;
        for (int i = lane; i < p.K; i += 32) {
            const float w = p.weight[r * p.K + i];
            if (w > 0.f) {                                  // (0 for tokens that do not exist)
                const float x = to_f32(row[p.ids[r * p.K + i]]);
                part_loss = fmaf(-w, nothing ? -INFINITY : log_prob(x, m, p.inv_t, log2s), part_loss);
            }
        }
        part_loss = warp_sum(part_loss);
        if (lane == 0) {
            p.out[r] = given + part_loss;
            if (p.stats) p.stats[r] = make_float4(m, nothing ? 0.f : 1.f / st.s, 0.f, log2s);
        }
    }
}

// A thread's entries of a row's list that lie in a part of the row: weight (0: none), token and logit.  Loaded under the
// row's own loads, so that the accesses one after the other cost nothing behind them.
template <typename T, int G> struct ListShare {
    static constexpr int N = kMaxList > G ? kMaxList / G : 1;
    float w[N], x[N];
    int64_t id[N];
    // What the list says ...
    __device__ __forceinline__ void load(const int64_t *ids, const float *weight, int K, int t) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool there = t + i * G < K;
            w[i] = there ? weight[t + i * G] : 0.f;
            id[i] = there ? ids[t + i * G] : -1;
            x[i] = 0.f;
        }
    }
    // ... and the logits it asks for: weight 0 for what is not in this part.
    __device__ __forceinline__ void fetch(const RowPart &part, const T *row) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (w[i] > 0.f && id[i] >= part.first && id[i] < part.last) x[i] = to_f32(row[id[i]]);
            else w[i] = 0.f;
        }
    }
};

// Which entries of a row's list each thread meets among the elements it writes: the thread that owns an element is
// handed its entry, so that the element leaves complete (a second, 2-byte store to lines on their way to memory cost
// the gradient kernel 15 %: [16384, 32768] bfloat16 with lists of 20 391 against 341 us; 317 now).
template <int G> struct ListChain {
    int head[G];
    int next[kMaxList], at[kMaxList];
    float w[kMaxList];
};
// All threads of the group; returns this thread's first entry (-1: none).
template <typename T, int G>
__device__ __forceinline__ int deal_list(const ListShare<T, G> &list, const RowPart &part, int t, ListChain<G> &chain) {
    chain.head[t] = -1;
    group_sync<G>();
#pragma unroll
    for (int k = 0; k < list.N; ++k) {
        if (list.w[k] > 0.f && list.id[k] >= part.first && list.id[k] < part.last) {
            const int i = t + k * G, j = int(list.id[k]);
            const int owner = j < part.body       ? j - part.first
                              : j < part.body_end ? (j - part.body) / TokenVec<T>::N % G
                                                  : part.body - part.first + j - part.body_end;
            chain.at[i] = j;
            chain.w[i] = list.w[k];
            chain.next[i] = atomicExch(&chain.head[owner], i);
        }
    }
    group_sync<G>();
    return chain.head[t];
}
// Adds scale * w to what the list asks for among the 2 * PAIRS elements from `first` on.
template <int G, int PAIRS>
__device__ __forceinline__ void add_entries(float2 (&d)[PAIRS], int first, int entry, const ListChain<G> &chain, float scale) {
    for (; entry >= 0; entry = chain.next[entry]) {
        const int at = chain.at[entry] - first;
        const float w = chain.w[entry];
        if (unsigned(at) < unsigned(2 * PAIRS)) {
#pragma unroll
            for (int h = 0; h < PAIRS; ++h) {
                if (at == 2 * h) d[h].x = fmaf(scale, w, d[h].x);
                if (at == 2 * h + 1) d[h].y = fmaf(scale, w, d[h].y);
            }
        }
    }
}

// ---- gradient from the statistics
// kTokens: g_j = e_j (A + B z_j) + dl [j = token] / T,  A = -(dl - dh ln2 u / s) / (s T),  B = -dh ln2 / (s T)
// kList:   g_j = scale (p_j - w_j) / T
// where e_j = 2^z_j; elementwise: reads the logits once, writes the gradient once, no barrier before the last list
// step.  A row of -inf alone gets zeros, one that is not asked for too (without being read).
struct TokenGradParams {
    const void *x;
    void *grad;                 // [rows, V], contiguous
    int64_t stride, rows;
    int V;
    float c, inv_t;
    const int64_t *ids;
    const float *weight, *base;
    const float4 *stats;
    const float *d_out;         // upstream gradient of the log probabilities or losses: [rows] or one value
    int d_out_step;             // 1: one per row, 0: one for all
    const float *d_entropy;     // [rows] or null
    const double *count;        // kList: divisor (null: none)
    int64_t ignore;
    int K;
    int chunks;                 // blocks per row
};

// G threads to a chunk of G * kTokenUnroll vectors.  ALIGNED: logits and gradient rows start at the same place within
// 16 bytes, so that whole vectors of one are whole vectors of the other; else the logits are read one by one (a padded
// head with an odd vocabulary: [16384, 50257] bfloat16 with rows of 50304 628 against 501 us, [8192, 50257] float32 486
// against 485).
template <typename T, int G, int MODE, bool ALIGNED>
__device__ __forceinline__ void token_grad_chunk(const TokenGradParams &p, unsigned unit) {
    constexpr int N = TokenVec<T>::N;
    constexpr int GROUPS = 256 / G;
    const int t = threadIdx.x % G;
    const int64_t r = G == 32 ? unit : unit / unsigned(p.chunks);
    const int chunk = G == 32 ? 0 : int(unit % unsigned(p.chunks));
    if (r >= p.rows) return;
    const T *x = static_cast<const T *>(p.x) + r * p.stride;
    T *g = static_cast<T *>(p.grad) + r * int64_t(p.V);

    // everything that hangs on nothing first
    const int64_t id = MODE == kTokens ? p.ids[r] : 0;
    const float base = MODE == kList ? p.base[r] : 0.f;
    const float4 st = p.stats[r];                           // (not written for rows that are not asked for: not used then)
    float dl = p.d_out ? p.d_out[r * p.d_out_step] : 0.f;
    const float dh = MODE == kTokens && p.d_entropy ? p.d_entropy[r] : 0.f;
    ListShare<T, G> list;
    if (MODE == kList) list.load(p.ids + r * p.K, p.weight + r * p.K, p.K, t);

    float A = 0.f, B = 0.f, at_token = 0.f;
    int token = -1;
    const float m = st.x;
    bool zero = MODE == kTokens ? id == p.ignore : base == INFINITY;
    if (!zero) {
        if (MODE == kTokens) {
            const bool bad = id < 0 || id >= p.V;
            if (bad) dl = __int_as_float(0x7fc00000);
            B = -dh * kTokenLn2 * st.y * p.inv_t;
            A = -(dl - dh * kTokenLn2 * st.z) * st.y * p.inv_t;
            token = bad ? -1 : int(id);
            at_token = dl * p.inv_t;
            zero = st.y == 0.f && !bad;
        } else {
            float scale = dl * p.inv_t;
            if (p.count) scale = float(double(scale) / *p.count);
            if (base != base) scale = base;
            A = scale * st.y;
            at_token = -scale;
            zero = st.y == 0.f;
        }
    }

    const RowPart part = row_chunk(static_cast<const T *>(g), p.V, chunk, p.chunks, G * kTokenUnroll);
    const pk_t negm = psplat(-m), cc = psplat(p.c), aa = psplat(A), bb = psplat(B);
    auto one = [&](float v) {                               // without what a given token adds
        const float z = max_nan((v - m) * p.c, kTokenFloor), e = ex2f(z);
        return e * fmaf(B, z, A);
    };
    // (a chunk is one step: its vectors are all on their way before the first is worked on)
    const int i = part.body + t * N;
    uint4 v[kTokenUnroll];
#pragma unroll
    for (int k = 0; k < kTokenUnroll; ++k) {
        const int64_t at = i + int64_t(k) * (G * N);
        v[k] = make_uint4(0u, 0u, 0u, 0u);
        if (!zero && at < part.body_end) {
            if (ALIGNED) {
                v[k] = ld_stream16<uint4>(x + at);
            } else {
                T e[N];
#pragma unroll
                for (int h = 0; h < N; ++h) e[h] = x[at + h];
                memcpy(&v[k], e, 16);
            }
        }
    }
    __shared__ ListChain<G> chains[MODE == kList ? GROUPS : 1];
    ListChain<G> &chain = chains[MODE == kList ? threadIdx.x / G : 0];
    const int entry = MODE == kList && !zero ? deal_list(list, part, t, chain) : -1;
#pragma unroll
    for (int k = 0; k < kTokenUnroll; ++k) {
        const int64_t at = i + int64_t(k) * (G * N);
        if (at >= part.body_end) break;
        if (!zero) {
            float2 d[N / 2];
#pragma unroll
            for (int h = 0; h < N / 2; ++h) {
                float2 z = upk2(pmul(padd(pk2(TokenVec<T>::pair(v[k], h)), negm), cc));
                if (MODE == kTokens) {
                    z.x = max_nan(z.x, kTokenFloor);
                    z.y = max_nan(z.y, kTokenFloor);
                }
                const pk_t zz = pk2(z);
                const pk_t e = pex2(zz);
                d[h] = upk2(MODE == kTokens ? pmul(e, pfma(bb, zz, aa)) : pmul(e, aa));
            }
            if (MODE == kTokens && unsigned(token - int(at)) < unsigned(N)) {
                const int w = token - int(at);
#pragma unroll
                for (int h = 0; h < N / 2; ++h) {
                    if (w == 2 * h) d[h].x += at_token;
                    if (w == 2 * h + 1) d[h].y += at_token;
                }
            }
            if (MODE == kList) add_entries(d, int(at), entry, chain, at_token);
            v[k] = TokenVec<T>::pack(d);
        }
        st_stream16(g + at, v[k]);
    }
    if (t < ragged_count(part)) {
        const int j = ragged_index(part, t);
        float2 d[1] = {make_float2(zero ? 0.f : one(to_f32(x[j])), 0.f)};
        if (MODE == kTokens && !zero && j == token) d[0].x += at_token;
        if (MODE == kList) add_entries(d, j, entry, chain, at_token);
        g[j] = from_f32<T>(d[0].x);
    }
}
template <typename T, int G, int MODE, bool ALIGNED>
__global__ void __launch_bounds__(256) token_grad_kernel(const TokenGradParams p) {
    token_grad_chunk<T, G, MODE, ALIGNED>(p, blockIdx.x * (256 / G) + threadIdx.x / G);
}

// ---- launches

// Over how many blocks of a cluster a row is split: with few rows, as long as all blocks run at once and every thread
// still has a vector.
inline int row_part_shift(int64_t rows, int64_t V, int dtype) {
    const int64_t vectors = row_vectors(V, dtype), room = int64_t(sm_count()) * 8;
    int shift = 0;
    while (2 << shift <= kMaxCluster && rows << (shift + 1) <= room && vectors >> (shift + 1) >= 256) ++shift;
    return shift;
}

// How many threads share a row.  What a row costs besides its elements (joins, barriers, finding the alternatives) is
// paid per thread, so few threads are better -- as long as there are rows enough to fill the SMs several times over,
// and a list of alternatives is short against the number of threads.  Measured, us at 32 / 128 / 256 threads:
//   [32768, 4000] bfloat16 (8 KB)     log probabilities 50 / 67 / 107    with 20 alternatives 106 / 146 / 244
//   [16384, 8192] float32 (32 KB)     79 / 80 / 85                       169 / 119 / 149
//   [16384, 32768] bfloat16 (64 KB)   170 / 167 / 171                    349 / 220 / 252
//   [2047, 100003] float16 (200 KB)   105 / 80 / 71                      333 / 104 / 88    (one wave of 128 threads)
// More than 32 alternatives take 256 threads: [16384, 32768] bfloat16 64 of them 301, 128 of them 396 (20: 224, 32: 236 at
// 128 threads; the bytes 164).
template <typename T, int MODE, bool TOP> int launch_stats(const TokenParams &prm, int dtype, cudaStream_t stream) {
    TokenParams p = prm;
    const char *what = "token statistics kernel launch";
    if (p.rows == 0) return B200_OK;
    const int64_t bytes = p.V * int64_t(sizeof(T)), sms = sm_count();
    const bool shortlist = !TOP || p.K <= 32;
    p.part_shift = 0;
    if (shortlist && (bytes <= 4096 || (p.rows >= 32 * sms && bytes <= (TOP ? 16384 : 32768))))
        return launch_cluster(token_stats_kernel<T, 32, MODE, TOP>, (p.rows + 7) / 8, 256, 0, 1, MODE == kList, stream, what, p);
    p.part_shift = row_part_shift(p.rows, p.V, dtype);
    if (p.part_shift == 0 && shortlist && (p.rows >= 32 * sms || bytes <= 131072))
        return launch_cluster(token_stats_kernel<T, 128, MODE, TOP>, p.rows, 128, 0, 1, MODE == kList, stream, what, p);
    return launch_cluster(token_stats_kernel<T, 256, MODE, TOP>, p.rows << p.part_shift, 256, 0, 1 << p.part_shift, MODE == kList, stream, what,
                          p);
}

// Chunks of a row of so many vectors, 256 threads to a chunk.
inline int grad_chunks(int64_t vectors) { return int((vectors + 256 * kTokenUnroll - 1) / (256 * kTokenUnroll)); }

template <typename T, int MODE> int launch_grad(const TokenGradParams &prm, int dtype, cudaStream_t stream) {
    TokenGradParams p = prm;
    const char *what = "token gradient kernel launch";
    if (p.rows == 0) return B200_OK;
    const int64_t vectors = row_vectors(p.V, dtype);
    const int64_t shift = int64_t((reinterpret_cast<uintptr_t>(p.x) - reinterpret_cast<uintptr_t>(p.grad)) & 15);
    const bool aligned = shift == 0 && (p.rows == 1 || ((p.stride - p.V) * int64_t(sizeof(T))) % 16 == 0);
    if (vectors <= 32 * kTokenUnroll) {
        p.chunks = 1;
        const int64_t grid = (p.rows + 7) / 8;
        return aligned ? launch_cluster(token_grad_kernel<T, 32, MODE, true>, grid, 256, 0, 1, false, stream, what, p)
                       : launch_cluster(token_grad_kernel<T, 32, MODE, false>, grid, 256, 0, 1, false, stream, what, p);
    }
    p.chunks = grad_chunks(vectors);
    const int64_t grid = p.rows * p.chunks;
    if (grid > 0x7fffffff) {
        set_error("%s: %lld rows of %d logits are more than one launch covers", what, (long long)p.rows, p.V);
        return B200_ERR_UNSUPPORTED;
    }
    return aligned ? launch_cluster(token_grad_kernel<T, 256, MODE, true>, grid, 256, 0, 1, false, stream, what, p)
                   : launch_cluster(token_grad_kernel<T, 256, MODE, false>, grid, 256, 0, 1, false, stream, what, p);
}

// What every entry point of the family refuses.
inline int check_rows(const char *who, const void *x, int64_t rows, int64_t V, int64_t stride, int dtype, float temperature) {
    if (rows < 0 || V < 1 || (rows > 1 && stride < 0)) {
        set_error("%s: need rows >= 0, V >= 1 and stride >= 0", who);
        return B200_ERR_ARG;
    }
    if (rows > 0x0fffffff || V > (int64_t(1) << 30)) {
        set_error("%s: at most 2^28 - 1 rows and 2^30 logits per row", who);
        return B200_ERR_UNSUPPORTED;
    }
    if (!dtype_known(dtype)) {
        set_error("%s: unknown dtype code %d", who, dtype);
        return B200_ERR_ARG;
    }
    if (!(temperature >= 1e-4f && temperature <= 1e4f)) {
        set_error("%s: the temperature must lie between 1e-4 and 1e4", who);
        return B200_ERR_ARG;
    }
    if (rows > 0 && (!x || !lies_on(x, dtype_size(dtype)))) {
        set_error("%s: the logits are null or not aligned to their type", who);
        return B200_ERR_ARG;
    }
    return B200_OK;
}

}  // namespace
}  // namespace b200
