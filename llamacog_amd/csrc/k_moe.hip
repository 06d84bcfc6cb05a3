// k_moe.hip — expert routing: the stable sort of (token, slot) pairs by expert, rows copied into
// that order, and the weighted rows back in token order with their gradient.
//
//   pair      p = token * used + slot with expert id ids[p]; an id outside 0 .. n_expert - 1 (a
//             padded token) belongs to no expert
//   sort      order: the pairs by expert, by pair within one, -1 behind the last; rank: each
//             pair's place, -1 without an expert; offsets[e]: the first place of expert e
//   gather    xs[rank[t][j]] = x[t]; rows behind offsets[n_expert] are zero
//   combine   y[t] = sum over j of w[t][j] ys[rank[t][j]], float32, slots in order (the gather's
//             gradient is the combine without weights)
//   back      dys[rank[t][j]] = w[t][j] dy[t], dw[t][j] = dy[t] . ys[rank[t][j]] in float32
#include "devops.h"

namespace mi355x_ops {

static inline unsigned ceil_div(int64_t a, int64_t b) { return (unsigned) ((a + b - 1) / b); }

// ---- sort ------------------------------------------------------------------------------------
// A counting sort without atomics, so that places never depend on timing.  A workgroup takes a
// chunk of pairs, each of its waves one run of it, 64 pairs at a time: lanes with the same expert
// find each other by one ballot per bit of the id, the lowest of them keeps the wave's count.
// One chunk is one launch; more are two: the chunks' counts, then their places, where every
// workgroup sums the counts in front of its own (at most SORT_CHUNKS of them).
constexpr int SORT_WAVES = 16;
constexpr int SORT_CHUNK = 4096;    // least pairs of a chunk
constexpr int SORT_CHUNKS = 128;

static int64_t sort_chunk(int64_t pairs) {   // pairs per chunk, a multiple of 64 per wave
    int64_t c = SORT_CHUNK;
    while ((pairs + c - 1) / c > SORT_CHUNKS) c *= 2;
    return c;
}

template <class I> __device__ __forceinline__ int expert_of(const I * ids, int64_t p, int64_t end, int n_expert) {
    if (p >= end) return -1;
    const I v = ids[p];
    return v >= 0 && v < (I) n_expert ? (int) v : -1;
}

// the lanes of the wave whose id is this lane's
__device__ __forceinline__ unsigned long long same_lanes(int id, int bits) {
    unsigned long long m = ~0ull;
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((id >> b) & 1);
        m &= ((id >> b) & 1) ? set : ~set;
    }
    return m & __ballot(id >= 0);
}

template <class I>
__device__ __forceinline__ void count_run(const I * ids, int64_t p0, int64_t p1, int n_expert, int bits, int * cnt) {
    const int lane = threadIdx.x & 63;
    for (int64_t p = p0; p < p1; p += 64) {
        const int id = expert_of(ids, p + lane, p1, n_expert);
        const unsigned long long m = same_lanes(id, bits);
        if (id >= 0 && __builtin_ctzll(m) == lane) cnt[id] += __popcll(m);
    }
}

// exclusive prefix over the workgroup's 1024 threads; `total` gets the sum
__device__ __forceinline__ int block_prefix(int v, int * part, int & total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int upto = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 63) part[wave] = upto;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
        const int s = part[w];
        before += w < wave ? s : 0;
        all += s;
    }
    total = all;
    return before + upto - v;
}

template <class I, bool COUNT_ONLY>
static __global__ void __launch_bounds__(64 * SORT_WAVES) k_moe_sort(const I * __restrict__ ids, int64_t pairs, int64_t chunk,
                                                              int n_expert, int bits, int32_t * __restrict__ counts,
                                                              int32_t * __restrict__ order, int32_t * __restrict__ rank,
                                                              int32_t * __restrict__ offsets) {
    extern __shared__ int cnt[];   // [SORT_WAVES][n_expert]
    __shared__ int part[SORT_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = threadIdx.x;
    const int64_t c0 = (int64_t) blockIdx.x * chunk, c1 = min(c0 + chunk, pairs);
    const int64_t run = chunk / SORT_WAVES;
    const int64_t p0 = min(c0 + wave * run, c1), p1 = min(p0 + run, c1);
    for (int i = threadIdx.x; i < SORT_WAVES * n_expert; i += 64 * SORT_WAVES) cnt[i] = 0;
    __syncthreads();
    count_run(ids, p0, p1, n_expert, bits, cnt + wave * n_expert);
    __syncthreads();
    if (COUNT_ONLY) {
        if (e < n_expert) {
            int s = 0;
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) s += cnt[w * n_expert + e];
            counts[(int64_t) blockIdx.x * n_expert + e] = s;
        }
        return;
    }
    // expert e's pairs in all chunks, and in those before this one
    int all = 0, before = 0;
    if (e < n_expert) {
        if (gridDim.x == 1) {
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) all += cnt[w * n_expert + e];
        } else {
            for (int c = 0; c < (int) gridDim.x; ++c) {
                const int s = counts[(int64_t) c * n_expert + e];
                before += c < (int) blockIdx.x ? s : 0;
                all += s;
            }
        }
    }
    int held;
    const int first = block_prefix(all, part, held);
    if (e < n_expert) {
        if (blockIdx.x == 0) offsets[e] = first;
        int at = first + before;
#pragma unroll
        for (int w = 0; w < SORT_WAVES; ++w) {
            const int s = cnt[w * n_expert + e];
            cnt[w * n_expert + e] = at;
            at += s;
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[n_expert] = held;
    __syncthreads();
    int * mine = cnt + wave * n_expert;
    for (int64_t p = p0; p < p1; p += 64) {
        const int id = expert_of(ids, p + lane, p1, n_expert);
        const unsigned long long m = same_lanes(id, bits);
        int place = -1;
        if (id >= 0) {
            place = mine[id] + __popcll(m & ((1ull << lane) - 1));
            order[place] = (int32_t) (p + lane);
        }
        if (p + lane < p1) {
            rank[p + lane] = place;
            if (p + lane >= held) order[p + lane] = -1;
        }
        // the places above are read before the count moves on: one wave, in order
        if (id >= 0 && __builtin_ctzll(m) == lane) mine[id] += __popcll(m);
    }
}

size_t moe_sort_workspace(int64_t pairs, int n_expert) {
    const int64_t chunk = sort_chunk(pairs), n = (pairs + chunk - 1) / chunk;
    return n > 1 ? (size_t) n * n_expert * sizeof(int32_t) : 0;
}

hipError_t moe_sort(const void * ids, int id_bytes, int64_t pairs, int n_expert, int32_t * order, int32_t * rank,
                    int32_t * offsets, void * work, hipStream_t st) {
    int bits = 1;
    while ((1 << bits) < n_expert) ++bits;
    const int64_t chunk = sort_chunk(pairs);
    const unsigned n = pairs ? ceil_div(pairs, chunk) : 1;
    const size_t lds = (size_t) SORT_WAVES * n_expert * sizeof(int);
    auto go = [&](auto i) {
        using I = decltype(i);
        if (n > 1)
            k_moe_sort<I, true><<<n, 64 * SORT_WAVES, lds, st>>>((const I *) ids, pairs, chunk, n_expert, bits,
                                                                 (int32_t *) work, order, rank, offsets);
        k_moe_sort<I, false><<<n, 64 * SORT_WAVES, lds, st>>>((const I *) ids, pairs, chunk, n_expert, bits, (int32_t *) work,
                                                              order, rank, offsets);
        return hipGetLastError();
    };
    return id_bytes == 8 ? go(int64_t{}) : go(int32_t{});
}

// ---- rows ------------------------------------------------------------------------------------
// All three are bound by memory: every row is read once and written once, a token's row once for
// all of its slots (the gather goes by rank, not by order, for that).  A lane owns N columns of a
// token; lanes are laid over the columns in a power of two.
struct row_args {
    int64_t T, D, pairs;
    int used, lsh;   // slots; log2 of the lanes over a row
};

__device__ __forceinline__ bool my_columns(const row_args & a, int N, int64_t & t, int64_t & col) {
    col = ((int64_t) blockIdx.y << a.lsh | (threadIdx.x & ((1 << a.lsh) - 1))) * N;
    t = (int64_t) blockIdx.x * (256 >> a.lsh) + (threadIdx.x >> a.lsh);
    return t < a.T && col < a.D;
}

template <class T, int N>
static __global__ void __launch_bounds__(256) k_moe_gather(row_args a, const T * __restrict__ x, int64_t ldx,
                                                    const int32_t * __restrict__ order, const int32_t * __restrict__ rank,
                                                    T * __restrict__ xs) {
    using V = pack<T, N>;
    int64_t t, col;
    if (!my_columns(a, N, t, col)) return;
    const V v = *(const V *) (x + t * ldx + col);
    for (int j = 0; j < a.used; ++j) {
        const int64_t p = t * a.used + j, r = rank[p];
        if (r >= 0 && r < a.pairs) *(V *) (xs + r * a.D + col) = v;
        if (order[p] < 0) *(V *) (xs + p * a.D + col) = V{};
    }
}

template <class T, int N, bool WEIGHTED>
static __global__ void __launch_bounds__(256) k_moe_combine(row_args a, const T * __restrict__ ys, int64_t ldys,
                                                     const int32_t * __restrict__ rank, const float * __restrict__ w,
                                                     T * __restrict__ y) {
    using V = pack<T, N>;
    int64_t t, col;
    if (!my_columns(a, N, t, col)) return;
    float s[N] = {};
    for (int j = 0; j < a.used; ++j) {
        const int64_t p = t * a.used + j, r = rank[p];
        if (r < 0 || r >= a.pairs) continue;   // whatever the weight and the row behind it hold
        const V v = *(const V *) (ys + r * ldys + col);
        const float f = WEIGHTED ? w[p] : 1.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = fmaf(f, to_f32(v.v[i]), s[i]);
    }
    V o;
#pragma unroll
    for (int i = 0; i < N; ++i) o.v[i] = from_f32<T>(s[i]);
    *(V *) (y + t * a.D + col) = o;
}

// one workgroup per token: its dy row once, each slot's row read and its gradient written, the dot
// products joined in shared memory in a fixed order.  A lane's columns are 16 bytes wide whatever the
// access width A, so that the sums do not depend on alignment.
template <class T, int A>
static __global__ void __launch_bounds__(256) k_moe_combine_back(row_args a, const T * __restrict__ dy, int64_t lddy,
                                                                 const T * __restrict__ ys, int64_t ldys,
                                                                 const int32_t * __restrict__ order,
                                                                 const int32_t * __restrict__ rank,
                                                                 const float * __restrict__ w, T * __restrict__ dys,
                                                                 float * __restrict__ dw) {
    using V = pack<T, A>;
    constexpr int N = 16 / sizeof(T);
    __shared__ float part[MOE_MAX_USED][4];
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int j = 0; j < a.used; ++j) {
        const int64_t p = t * a.used + j, r = rank[p];
        const bool held = r >= 0 && r < a.pairs, empty = order[p] < 0;
        const float f = w[p];
        float dot = 0.0f;
        for (int64_t col = (int64_t) threadIdx.x * N; col < a.D; col += 256 * N) {
#pragma unroll
            for (int i = 0; i < N; i += A) {
                if (col + i >= a.D) break;   // D is a multiple of A
                if (held) {
                    const V g = *(const V *) (dy + t * lddy + col + i), v = *(const V *) (ys + r * ldys + col + i);
                    V o;
#pragma unroll
                    for (int k = 0; k < A; ++k) {
                        dot = fmaf(to_f32(g.v[k]), to_f32(v.v[k]), dot);
                        o.v[k] = from_f32<T>(f * to_f32(g.v[k]));
                    }
                    *(V *) (dys + r * a.D + col + i) = o;
                }
                if (empty) *(V *) (dys + p * a.D + col + i) = V{};
            }
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) dot += __shfl_xor(dot, d);
        if (lane == 0) part[j][wave] = held ? dot : 0.0f;
    }
    __syncthreads();
    if ((int) threadIdx.x < a.used) {
        const float * q = part[threadIdx.x];
        dw[t * a.used + threadIdx.x] = (q[0] + q[1]) + (q[2] + q[3]);
    }
}

// the widest access that every row and base allows: f(type, columns per lane)
template <class F> static hipError_t with_columns(int type, int64_t D, uintptr_t bases, int64_t lds, F && f) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int W = 16 / sizeof(T);
        const int64_t step = D | lds;
        auto fits = [&](int n) { return step % n == 0 && bases % (n * sizeof(T)) == 0; };
        if (fits(W)) return f(t, std::integral_constant<int, W>{});
        if (fits(W / 2)) return f(t, std::integral_constant<int, W / 2>{});
        if (W > 4 && fits(2)) return f(t, std::integral_constant<int, 2>{});
        return f(t, std::integral_constant<int, 1>{});
    });
}

static row_args row_layout(int64_t T, int64_t D, int used, int N, dim3 & grid) {
    row_args a{T, D, T * used, used, 0};
    const int64_t cols = (D + N - 1) / N;
    while (a.lsh < 8 && (1 << a.lsh) < cols) ++a.lsh;
    grid = dim3(ceil_div(T, 256 >> a.lsh), ceil_div(cols, (int64_t) 1 << a.lsh));
    return a;
}

hipError_t moe_gather(int type, const void * x, int64_t ldx, int64_t T, int64_t D, int used, const int32_t * order,
                      const int32_t * rank, void * xs, hipStream_t st) {
    return with_columns(type, D, (uintptr_t) x | (uintptr_t) xs, ldx, [&](auto t, auto n) {
        using E = decltype(t);
        dim3 grid;
        const row_args a = row_layout(T, D, used, n, grid);
        k_moe_gather<E, n><<<grid, 256, 0, st>>>(a, (const E *) x, ldx, order, rank, (E *) xs);
        return hipGetLastError();
    });
}

hipError_t moe_combine(int type, const void * ys, int64_t ldys, int64_t T, int64_t D, int used, const int32_t * rank,
                       const float * w, void * y, hipStream_t st) {
    return with_columns(type, D, (uintptr_t) ys | (uintptr_t) y, ldys, [&](auto t, auto n) {
        using E = decltype(t);
        dim3 grid;
        const row_args a = row_layout(T, D, used, n, grid);
        if (w) k_moe_combine<E, n, true><<<grid, 256, 0, st>>>(a, (const E *) ys, ldys, rank, w, (E *) y);
        else k_moe_combine<E, n, false><<<grid, 256, 0, st>>>(a, (const E *) ys, ldys, rank, w, (E *) y);
        return hipGetLastError();
    });
}

hipError_t moe_combine_back(int type, const void * dy, int64_t lddy, const void * ys, int64_t ldys, int64_t T, int64_t D,
                            int used, const int32_t * order, const int32_t * rank, const float * w, void * dys, float * dw,
                            hipStream_t st) {
    return with_columns(type, D, (uintptr_t) dy | (uintptr_t) ys | (uintptr_t) dys, lddy | ldys, [&](auto t, auto n) {
        using E = decltype(t);
        const row_args a{T, D, T * used, used, 0};
        k_moe_combine_back<E, n><<<(unsigned) T, 256, 0, st>>>(a, (const E *) dy, lddy, (const E *) ys, ldys, order, rank, w,
                                                                (E *) dys, dw);
        return hipGetLastError();
    });
}

}  // namespace mi355x_ops
