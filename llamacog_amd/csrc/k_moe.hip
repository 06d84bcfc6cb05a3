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
// workgroup sums the counts in front of its own (at most SORT_CHUNKS of them).  Bound by latency:
// ids are loaded SORT_LOADS at a time, the chunks' counts are summed by all threads.  2 pairs 3.2 us,
// 131072 by 128 experts 15.5 (4.8 and 10.7).  Whole calls with chunks of 1024 / 2048 / 4096 pairs: 4000 by 8 experts
// 8.1 / 9.0 / 6.4 us, 4000 by 128 7.5 / 9.3 / 8.4, 16384 by 64 8.0 / 9.2 / 12.5, 131072 by 128 9.9 / 10.8 / 14.8,
// 524288 by 256 19.7 / 18.6 / 18.9; with chunks of 8192 4000 took 8.3.
constexpr int SORT_WAVES = 16;
constexpr int SORT_LOADS = 4;
constexpr int SORT_CHUNK = SORT_WAVES * SORT_LOADS * 64;    // least pairs of a chunk
constexpr int SORT_CHUNKS = 128;

static int64_t sort_chunk(int64_t pairs) {   // pairs per chunk
    int64_t c = SORT_CHUNK;
    while ((pairs + c - 1) / c > SORT_CHUNKS) c *= 2;
    return c;
}

// what lanes of this wave wrote to shared memory is read by its other lanes behind this: its accesses are
// done in order anyway, this keeps the compiler to it
static __device__ __forceinline__ void in_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// the lanes of the wave whose id is this lane's
static __device__ __forceinline__ unsigned long long same_lanes(int id, int bits) {
    unsigned long long m = ~0ull;
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((id >> b) & 1);
        m &= ((id >> b) & 1) ? set : ~set;
    }
    return m & __ballot(id >= 0);
}

// f(pair of this lane, its expert or -1, the lanes with the same one) for a wave's run of pairs
template <class I, class F>
static __device__ __forceinline__ void for_run(const I * ids, int64_t p0, int64_t p1, int n_expert, int bits, F && f) {
    const int lane = threadIdx.x & 63;
    for (int64_t p = p0; p < p1; p += 64 * SORT_LOADS) {
        I v[SORT_LOADS];
#pragma unroll
        for (int i = 0; i < SORT_LOADS; ++i) v[i] = p + 64 * i + lane < p1 ? ids[p + 64 * i + lane] : (I) -1;
#pragma unroll
        for (int i = 0; i < SORT_LOADS; ++i) {
            if (p + 64 * i >= p1) break;
            const int id = v[i] >= 0 && v[i] < (I) n_expert ? (int) v[i] : -1;
            f(p + 64 * i + lane, id, same_lanes(id, bits));
            in_order();   // the next 64 count on from what these wrote
        }
    }
}

// exclusive prefix over the workgroup's 1024 threads; `total` gets the sum
static __device__ __forceinline__ int block_prefix(int v, int * part, int & total) {
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
    __shared__ int part[SORT_WAVES], sums[2][64 * SORT_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = threadIdx.x;
    const int64_t c0 = (int64_t) blockIdx.x * chunk, c1 = min(c0 + chunk, pairs);
    const int64_t run = chunk / SORT_WAVES;
    const int64_t p0 = min(c0 + wave * run, c1), p1 = min(p0 + run, c1);
    int * mine = cnt + wave * n_expert;
    for (int i = lane; i < n_expert; i += 64) mine[i] = 0;
    in_order();
    for_run(ids, p0, p1, n_expert, bits, [&](int64_t, int id, unsigned long long m) {
        if (id >= 0 && __builtin_ctzll(m) == lane) mine[id] += __popcll(m);
    });
    if (COUNT_ONLY) {
        __syncthreads();
        if (e < n_expert) {
            int s = 0;
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) s += cnt[w * n_expert + e];
            counts[(int64_t) blockIdx.x * n_expert + e] = s;
        }
        return;
    }
    // expert e's pairs in all chunks, and in those before this one: `share` threads for each expert
    if (gridDim.x > 1) {
        const int share = 64 * SORT_WAVES / n_expert;
        const int ex = threadIdx.x % n_expert, first = threadIdx.x / n_expert;
        int all = 0, before = 0;
        if (first < share) {
#pragma unroll 8
            for (int c = first; c < (int) gridDim.x; c += share) {
                const int s = counts[(int64_t) c * n_expert + ex];
                before += c < (int) blockIdx.x ? s : 0;
                all += s;
            }
        }
        sums[0][threadIdx.x] = all;
        sums[1][threadIdx.x] = before;
    }
    __syncthreads();
    int all = 0, before = 0;
    if (e < n_expert) {
        if (gridDim.x == 1) {
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) all += cnt[w * n_expert + e];
        } else {
            for (int k = 0; k < 64 * SORT_WAVES / n_expert; ++k) {
                all += sums[0][k * n_expert + e];
                before += sums[1][k * n_expert + e];
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
    for_run(ids, p0, p1, n_expert, bits, [&](int64_t p, int id, unsigned long long m) {
        int place = -1;
        if (id >= 0) {
            place = mine[id] + __popcll(m & ((1ull << lane) - 1));
            order[place] = (int32_t) p;
        }
        if (p < p1) {
            rank[p] = place;
            if (p >= held) order[p] = -1;
        }
        // the places above are read before the count moves on: one wave, in order
        if (id >= 0 && __builtin_ctzll(m) == lane) mine[id] += __popcll(m);
    });
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
        auto pass = [&](auto kernel) {
            return launch(kernel, n, 64 * SORT_WAVES, lds, st, (const I *) ids, pairs, chunk, n_expert, bits, (int32_t *) work, order, rank,
                          offsets);
        };
        const hipError_t e = n > 1 ? pass(k_moe_sort<I, true>) : hipSuccess;
        return e == hipSuccess ? pass(k_moe_sort<I, false>) : e;
    };
    return id_bytes == 8 ? go(int64_t{}) : go(int32_t{});
}

// ---- rows ------------------------------------------------------------------------------------
// All three are bound by memory: every row is read once and written once, a token's row once for
// all of its slots (the gather goes by rank, not by order, for that).  A lane owns 16 bytes of a
// token's columns, the last one what is left; lanes are laid over the columns in a power of two.
// Rows lie on any address.  16384 tokens, 8 slots, 2048 bf16 columns: gather 103 us (5.9 TB/s, nearly all
// writes, past the caches: 112 through them), combine 127 - 132 (4.7 TB/s), back 230 (5.0 TB/s).  With 2047 columns
// 148, 143 and 316, with 2046 142, 137 and 288: rows begin anywhere in a cache line, and most 16-byte accesses are
// not aligned to their size.
struct row_args {
    int64_t T, D, pairs;
    int used, lsh;   // slots; log2 of the lanes over a row
};

template <class T> constexpr int COLS = 16 / sizeof(T);

static __device__ __forceinline__ bool my_columns(const row_args & a, int N, int64_t & t, int64_t & col) {
    col = ((int64_t) blockIdx.y << a.lsh | (threadIdx.x & ((1 << a.lsh) - 1))) * N;
    t = group_id() * (256 >> a.lsh) + (threadIdx.x >> a.lsh);
    return t < a.T && col < a.D;
}

// n elements of a row from `p` on, in one access if it is all N, zeros behind them; WHOLE: it always is
template <bool WHOLE, class T, int N> static __device__ __forceinline__ pack<T, N> take(const T * p, int64_t n) {
    if (WHOLE || n >= N) return get<T, N>(p);
    pack<T, N> v = {};
    for (int i = 0; i < N; ++i)
        if (i < n) v.v[i] = p[i];
    return v;
}
template <bool WHOLE, bool STREAM, class T, int N> static __device__ __forceinline__ void give(T * p, int64_t n, const pack<T, N> & v) {
    if (WHOLE || n >= N) return put<STREAM>(p, v);
    for (int i = 0; i < N; ++i)
        if (i < n) p[i] = v.v[i];
}

template <class T, bool WHOLE, bool STREAM>
static __global__ void __launch_bounds__(256) k_moe_gather(row_args a, const T * __restrict__ x, int64_t ldx,
                                                           const int32_t * __restrict__ order,
                                                           const int32_t * __restrict__ rank, T * __restrict__ xs) {
    int64_t t, col;
    if (!my_columns(a, COLS<T>, t, col)) return;
    const int64_t n = a.D - col;
    const pack<T, COLS<T>> v = take<WHOLE, T, COLS<T>>(x + t * ldx + col, n);
    for (int j = 0; j < a.used; ++j) {
        const int64_t p = t * a.used + j, r = rank[p];
        if (r >= 0 && r < a.pairs) give<WHOLE, STREAM>(xs + r * a.D + col, n, v);
        if (order[p] < 0) give<WHOLE, STREAM>(xs + p * a.D + col, n, pack<T, COLS<T>>{});
    }
}

template <class T, bool WHOLE, bool WEIGHTED>
static __global__ void __launch_bounds__(256) k_moe_combine(row_args a, const T * __restrict__ ys, int64_t ldys,
                                                            const int32_t * __restrict__ rank, const float * __restrict__ w,
                                                            T * __restrict__ y) {
    constexpr int N = COLS<T>;
    int64_t t, col;
    if (!my_columns(a, N, t, col)) return;
    float s[N] = {};
    constexpr int BATCH = 4;   // rows on their way at a time
    for (int j0 = 0; j0 < a.used; j0 += BATCH) {
        pack<T, N> v[BATCH];
        float f[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
            const int64_t p = t * a.used + j0 + k, r = j0 + k < a.used ? rank[p] : -1;
            // a slot without an expert adds zero, whatever the weight and the row behind it hold
            const bool held = r >= 0 && r < a.pairs;
            v[k] = held ? take<WHOLE, T, N>(ys + r * ldys + col, a.D - col) : pack<T, N>{};
            f[k] = !held ? 0.0f : WEIGHTED ? w[p] : 1.0f;
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
#pragma unroll
            for (int i = 0; i < N; ++i) s[i] = fmaf(f[k], to_f32(v[k].v[i]), s[i]);
    }
    pack<T, N> o;
#pragma unroll
    for (int i = 0; i < N; ++i) o.v[i] = from_f32<T>(s[i]);
    give<WHOLE, false>(y + t * a.D + col, a.D - col, o);
}

// Each slot's row read and its gradient written; a token's lanes (up to a workgroup) go through its
// columns and join their dot products, in a wave by exchanges, over waves in shared memory, always
// in the same order.  A token's slots follow one another, so that its dy row comes from memory once;
// where the tokens are too few to fill the card, every slot has lanes of its own (gridDim.y).
template <class T, bool WHOLE, bool STREAM>
static __global__ void __launch_bounds__(256) k_moe_combine_back(row_args a, const T * __restrict__ dy, int64_t lddy,
                                                                 const T * __restrict__ ys, int64_t ldys,
                                                                 const int32_t * __restrict__ order,
                                                                 const int32_t * __restrict__ rank,
                                                                 const float * __restrict__ w, T * __restrict__ dys,
                                                                 float * __restrict__ dw) {
    constexpr int N = COLS<T>;
    __shared__ float part[4][MOE_MAX_USED];
    const int lanes = 1 << a.lsh, mine = threadIdx.x & (lanes - 1);
    const int64_t t = group_id() * (256 >> a.lsh) + (threadIdx.x >> a.lsh);
    const bool here = t < a.T;
    for (int j = blockIdx.y; j < a.used; j += gridDim.y) {
        float dot = 0.0f;
        if (here) {
            const int64_t p = t * a.used + j, r = rank[p];
            const bool held = r >= 0 && r < a.pairs, empty = order[p] < 0;
            const float f = w[p];
            for (int64_t col = (int64_t) mine * N; col < a.D; col += lanes * N) {
                const int64_t n = a.D - col;
                if (held) {
                    const pack<T, N> g = take<WHOLE, T, N>(dy + t * lddy + col, n), v = take<WHOLE, T, N>(ys + r * ldys + col, n);
                    pack<T, N> o;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        dot = fmaf(to_f32(g.v[i]), to_f32(v.v[i]), dot);
                        o.v[i] = from_f32<T>(f * to_f32(g.v[i]));
                    }
                    give<WHOLE, STREAM>(dys + r * a.D + col, n, o);
                }
                if (empty) give<WHOLE, STREAM>(dys + p * a.D + col, n, pack<T, N>{});
            }
        }
        for (int d = min(lanes, 64) / 2; d; d >>= 1) dot += __shfl_xor(dot, d);
        if (lanes <= 64) {
            if (here && mine == 0) dw[t * a.used + j] = dot;
        } else if ((threadIdx.x & 63) == 0) {
            part[threadIdx.x >> 6][j] = dot;
        }
    }
    if (lanes <= 64) return;
    __syncthreads();
    if (here && mine < a.used && mine % gridDim.y == blockIdx.y) {
        const int wave = threadIdx.x >> 6;
        float s = part[wave][mine] + part[wave + 1][mine];
        if (lanes == 256) s += part[2][mine] + part[3][mine];
        dw[t * a.used + mine] = s;
    }
}

// f(element type, WHOLE, a flag) as template arguments, the layout of the rows and the groups of tokens and columns
template <class F> static hipError_t with_rows(int type, int64_t T, int64_t D, int used, bool flag, F && f) {
    return with_type(type, [&](auto t) {
        using E = decltype(t);
        row_args a{T, D, T * used, used, 0};
        const int64_t cols = (D + COLS<E> - 1) / COLS<E>;
        while (a.lsh < 8 && (1 << a.lsh) < cols) ++a.lsh;
        const dim3 grid = row_groups(ceil_div(T, 256 >> a.lsh), ceil_div(cols, (int64_t) 1 << a.lsh));
        auto with_flag = [&](auto whole) { return flag ? f(t, whole, std::true_type{}, a, grid) : f(t, whole, std::false_type{}, a, grid); };
        return D % COLS<E> == 0 ? with_flag(std::true_type{}) : with_flag(std::false_type{});
    });
}

hipError_t moe_gather(int type, const void * x, int64_t ldx, int64_t T, int64_t D, int used, const int32_t * order,
                      const int32_t * rank, void * xs, hipStream_t st) {
    const bool stream = T * used * D * (type == ELEM_F32 ? 4 : 2) > STREAM_BYTES;
    return with_rows(type, T, D, used, stream, [&](auto t, auto whole, auto flag, const row_args & a, dim3 grid) {
        using E = decltype(t);
        return launch(k_moe_gather<E, whole, flag>, grid, 256, 0, st, a, (const E *) x, ldx, order, rank, (E *) xs);
    });
}

hipError_t moe_combine(int type, const void * ys, int64_t ldys, int64_t T, int64_t D, int used, const int32_t * rank,
                       const float * w, void * y, hipStream_t st) {
    return with_rows(type, T, D, used, w != nullptr, [&](auto t, auto whole, auto flag, const row_args & a, dim3 grid) {
        using E = decltype(t);
        return launch(k_moe_combine<E, whole, flag>, grid, 256, 0, st, a, (const E *) ys, ldys, rank, w, (E *) y);
    });
}

hipError_t moe_combine_back(int type, const void * dy, int64_t lddy, const void * ys, int64_t ldys, int64_t T, int64_t D,
                            int used, const int32_t * order, const int32_t * rank, const float * w, void * dys, float * dw,
                            hipStream_t st) {
    const bool stream = T * used * D * (type == ELEM_F32 ? 4 : 2) > STREAM_BYTES;
    return with_rows(type, T, D, used, stream, [&](auto t, auto whole, auto flag, row_args a, dim3) {
        using E = decltype(t);
        // here a lane may have several columns: no more lanes than columns, so that none is idle for long
        if (a.lsh > 0 && ((int64_t) COLS<E> << a.lsh) > D + COLS<E> - 1) --a.lsh;
        const int64_t n = ceil_div(T, 256 >> a.lsh);
        // slots side by side or one after the other: 512 tokens of 8 x 2048 bf16 9.8 us and 16.0, 1024 15.7 and 18.7,
        // 2000 28.3 both, 4096 62.0 and 59.6
        const dim3 groups = row_groups(n, n < 2048 ? used : 1);
        return launch(k_moe_combine_back<E, whole, flag>, groups, 256, 0, st, a, (const E *) dy, lddy, (const E *) ys, ldys, order, rank, w,
                      (E *) dys, dw);
    });
}

}  // namespace mi355x_ops
