// k_mx4.hip — MXFP4 (OCP microscaling: E2M1 elements, one E8M0 exponent per 32): quantisation,
// dequantisation and the product for few rows on gfx950's scaled matrix instructions.
//
//   quantise  a = max |x| over a block; s = clamp(floor(log2 a) - 2, -127, 127) (a = 0: -127); the
//             code is x * 2^-s rounded to E2M1, to nearest with ties to even, at most 6.  Every
//             step but that rounding is exact.  A block with an infinity or a NaN gets exponent
//             byte 255 and stands for NaN throughout.
//   product   y[t][m] = sum over blocks of 2^(sw + sx) * sum of 32 w * x, float32 sums.
#include "mx4.h"

namespace mi355x_ops {

static inline unsigned ceil_div(int64_t a, int64_t b) { return (unsigned) ((a + b - 1) / b); }

// ---- quantisation ----------------------------------------------------------------------------
// Bound by memory: 2 or 4 B read and 17/32 B written per element.  A lane takes 8 elements (a
// 16-B load of the 16-bit types), four lanes a block: their maximum is two DPP steps, and the
// conversion is the hardware's (v_cvt_scalef32_pk_fp4: one rounding, saturating).  Lanes are laid
// over a row's columns in a power of two so that no division is needed; a workgroup takes QROWS
// times as many rows as its lanes hold, loads first, to keep bytes in flight.  28672 x 8192: 120 us from
// bf16, 5.0 TB/s, the rate of a copy; 234 us from float32, 4.5 TB/s.  Right behind a kernel that has written 470 MB
// the first takes 143 (median; 122 at least).
constexpr int QROWS = 4;

template <class T>
static __global__ void __launch_bounds__(256) k_mx4_quantize(const T * __restrict__ x, int64_t ldx, int64_t rows, int64_t K, int lsh,
                                                      uint8_t * __restrict__ codes, uint8_t * __restrict__ scales) {
    const int64_t c = (int64_t) blockIdx.y << lsh | (threadIdx.x & ((1 << lsh) - 1));
    if (c >= K / 8) return;   // K / 8 is a multiple of four: the four lanes of a block stay together
    const int rp = 256 >> lsh;
    const int64_t row0 = group_id() * rp * QROWS + (threadIdx.x >> lsh);
    float v[QROWS][8];
#pragma unroll
    for (int i = 0; i < QROWS; ++i) {
        const int64_t row = min(row0 + (int64_t) i * rp, rows - 1);
        load8(x + row * ldx + c * 8, v[i]);
    }
#pragma unroll
    for (int i = 0; i < QROWS; ++i) {
        const int64_t row = row0 + (int64_t) i * rp;
        if (row >= rows) break;
        const unsigned e = mx4_block_exponent(v[i]);
        *(uint32_t *) (codes + row * (K / 2) + c * 4) = mx4_pack8(v[i], e);
        if ((c & 3) == 0) {
            uint8_t * sp = scales + ((c >> 5) * rows + row) * 8;
            int b = (c >> 2) & 7;
            sp[b] = (uint8_t) e;
            if (c + 4 == K / 8)
                while (++b < 8) sp[b] = 0;   // past K
        }
    }
}

static int row_shift(int64_t cols) {   // log2 of the lanes laid over a row of `cols` columns, 4 to 256
    int s = 2;
    while (s < 8 && (1 << s) < cols) ++s;
    return s;
}

hipError_t mx4_quantize(int type, const void * x, int64_t ldx, int64_t rows, int64_t K, uint8_t * codes, uint8_t * scales,
                        hipStream_t st) {
    const int lsh = row_shift(K / 8);
    const dim3 grid = row_groups(ceil_div(rows, (int64_t) (256 >> lsh) * QROWS), ceil_div(K / 8, 1 << lsh));
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return launch(k_mx4_quantize<T>, grid, 256, 0, st, (const T *) x, ldx, rows, K, lsh, codes, scales);
    });
}

// ---- values back -----------------------------------------------------------------------------
// Bound by memory, laid out as the quantisation is: 28672 x 8192 to bf16 119 us, 5.0 TB/s.
template <class T>
static __global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t * __restrict__ codes, const uint8_t * __restrict__ scales,
                                                        int64_t rows, int64_t K, int lsh, T * __restrict__ y) {
    const int64_t c = (int64_t) blockIdx.y << lsh | (threadIdx.x & ((1 << lsh) - 1));
    if (c >= K / 8) return;
    const int rp = 256 >> lsh;
    const int64_t row0 = group_id() * rp * QROWS + (threadIdx.x >> lsh);
    uint32_t q[QROWS];
    unsigned e[QROWS];
#pragma unroll
    for (int i = 0; i < QROWS; ++i) {
        const int64_t row = min(row0 + (int64_t) i * rp, rows - 1);
        q[i] = *(const uint32_t *) (codes + row * (K / 2) + c * 4);
        e[i] = scales[((c >> 5) * rows + row) * 8 + ((c >> 2) & 7)];
    }
#pragma unroll
    for (int i = 0; i < QROWS; ++i) {
        const int64_t row = row0 + (int64_t) i * rp;
        if (row >= rows) break;
        float v[8];
        mx4_unpack8(q[i], e[i], v);
        store8(y + row * K + c * 8, v);
    }
}

hipError_t mx4_dequantize(const mx4_mat & m, int type, void * y, hipStream_t st) {
    const int lsh = row_shift(m.K / 8);
    const dim3 grid = row_groups(ceil_div(m.rows, (int64_t) (256 >> lsh) * QROWS), ceil_div(m.K / 8, 1 << lsh));
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return launch(k_mx4_dequantize<T>, grid, 256, 0, st, m.codes, m.scales, m.rows, m.K, lsh, (T *) y);
    });
}

// ---- product, few rows -----------------------------------------------------------------------
// Bound by the weights' bytes.  Weight rows are the matrix instruction's first operand (16x16x128:
// lane l holds row l % 16 and the 32-block l / 16, one 16-B load; four lanes read 64 B of a row side
// by side), x rows the second, so a lane's four results are four neighbouring outputs of an x row.
//
// A workgroup keeps the 16 NT x rows of a tile in shared memory and goes through groups of 16 weight
// rows.  KS of its MV_WAVES waves share a group, each taking every KS-th 256-element plane of K, and
// join their sums in shared memory; with KS = 1 there is nothing to join and no wave waits for
// another.  KS is raised only where the groups alone are too few waves for the memory (mv_split).
// A wave's next planes are always on their way while it multiplies the present ones.
//
// The x rows come as MXFP4, or as floats that every workgroup quantises for itself behind its first
// weight loads: that costs a little arithmetic in each and saves a launch.
//
// One row, weights that no cache holds: 4096 x 14336 10.7 us, 28672 x 4096 14.4 (4.3 TB/s), two experts of 28672 x
// 4096 26 (4.8 TB/s): about 3 us until the first weights have come, then the memory's rate.  The same weights call
// after call, which the 256-MB cache then holds in part: 9.7, 13.7 and 25.

// U planes of a row group
template <int U> struct mv_weights {
    int4 w[U][2];
    uint2 e[U];
    __device__ __forceinline__ void load(const mx4_args & a, const uint8_t * wc, const uint8_t * ws, int64_t row, int s0, int step, int q) {
        const int S = (a.KB + 7) / 8;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * step;
            if (s >= S) break;
            e[u] = *(const uint2 *) (ws + ((int64_t) s * a.M + row) * 8);
#pragma unroll
            for (int j = 0; j < 2; ++j) w[u][j] = *(const int4 *) (wc + (row * a.KB + min(s * 8 + 4 * j + q, a.KB - 1)) * 16);
        }
    }
};

struct mxfp4 {};   // the type of x rows that are quantised already

template <int NT, int KS, class X, class Y, bool IDS>
static __global__ void __launch_bounds__(64 * MV_WAVES, 4) k_mx4_mv(mx4_args a, const X * __restrict__ x, int64_t ldx, int per_tile) {
    constexpr int U = 2, GW = MV_WAVES / KS;   // planes at a time; groups at a time
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // x rows, then sums to join
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, q = lane >> 4, part = wave % KS;
    const int64_t tile = blockIdx.x / per_tile;
    const tile_rows tr = IDS ? tile_scan(a, 16 * NT).tile(a, tile)
                             : tile_rows{0, tile * 16 * NT, min((int64_t) 16 * NT, a.T - tile * 16 * NT)};
    if (tr.n <= 0) return;
    Y * y = (Y *) a.y + tr.first * a.M;
    const int64_t g0 = blockIdx.x % per_tile * GW;
    if (IDS && tr.expert < 0) {   // pairs that no expert takes
        for (int64_t g = g0; g * 16 < a.M; g += (int64_t) per_tile * GW)
            for (int i = threadIdx.x; i < 16 * GW * tr.n; i += 64 * MV_WAVES) {
                const int64_t m = g * 16 + i % (16 * GW);
                if (m < a.M) y[i / (16 * GW) * a.M + m] = from_f32<Y>(0.0f);
            }
        return;
    }
    const uint8_t * wc = a.w_codes + tr.expert * a.w_codes_stride;
    const uint8_t * ws = a.w_scales + tr.expert * a.w_scales_stride;
    const int S = (a.KB + 7) / 8;
    mv_weights<U> now, next;
    auto row_of = [&](int64_t g) { return min((g + wave / KS) * 16 + r, a.M - 1); };
    now.load(a, wc, ws, row_of(g0), part, KS, q);

    const int row_bytes = mv_row_bytes(a.KB);
    if constexpr (std::is_same_v<X, mxfp4>) {
        for (int t = wave; t < tr.n; t += MV_WAVES) {
            const int64_t row = x_row<IDS>(a, tr.first + t);
            for (int c = lane; c < a.KB; c += 64) {
                *(int4 *) (lds + t * row_bytes + c * 16) = *(const int4 *) (a.x_codes + (row * a.KB + c) * 16);
                lds[t * row_bytes + a.KB * 16 + c] = a.x_scales[((c >> 3) * a.x_rows + row) * 8 + (c & 7)];
            }
        }
    } else {
        for (int t = 0; t < tr.n; ++t) {
            const X * row = x + x_row<IDS>(a, tr.first + t) * ldx;
            for (int c = threadIdx.x; c < a.KB * 4; c += 64 * MV_WAVES) {
                float v[8];
                load8(row + (int64_t) c * 8, v);
                const unsigned e = mx4_block_exponent(v);
                *(uint32_t *) (lds + t * row_bytes + c * 4) = mx4_pack8(v, e);
                if ((c & 3) == 0) lds[t * row_bytes + a.KB * 16 + (c >> 2)] = (uint8_t) e;
            }
        }
    }
    __syncthreads();
    const uint8_t * xl[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xl[n] = lds + min(16 * n + r, (int) tr.n - 1) * row_bytes;
    float * red = (float *) (lds + min((int64_t) 16 * NT, a.T) * row_bytes);   // [GW][KS][16][16]

    for (int64_t g = g0; g * 16 < a.M; g += (int64_t) per_tile * GW) {
        v4f acc[NT] = {};
        for (int s0 = part; s0 < S; s0 += KS * U) {
            const bool more = s0 + KS * U < S;
            next.load(a, wc, ws, row_of(more ? g : g + (int64_t) per_tile * GW), more ? s0 + KS * U : part, KS, q);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u * KS;
                if (s >= S) break;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int b = s * 8 + 4 * j + q, bc = min(b, a.KB - 1);
                    const bool in = b < a.KB;   // past K: zero codes, finite exponents
                    const int4 w = in ? now.w[u][j] : int4{0, 0, 0, 0};
                    const int sw = in ? (int) ((j ? now.e[u].y : now.e[u].x) >> (8 * q)) : 0;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        acc[n] = mfma_mx4_16(w, *(const int4 *) (xl[n] + bc * 16), acc[n], sw, in ? xl[n][a.KB * 16 + bc] : 0);
                }
            }
            now = next;
        }
        const int64_t m0 = (g + wave / KS) * 16;
        if constexpr (KS == 1) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (16 * n + r < tr.n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (m0 + 4 * q + i < a.M) y[(16 * n + r) * a.M + m0 + 4 * q + i] = from_f32<Y>(acc[n][i]);
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) {   // 16 x rows at a time, to leave shared memory for another workgroup
                __syncthreads();             // the sums before have been taken
                *(v4f *) &red[(wave * 16 + r) * 16 + 4 * q] = acc[n];
                __syncthreads();
                for (int i = threadIdx.x; i < GW * 256; i += 64 * MV_WAVES) {
                    const int k = i / 256, t = 16 * n + i / 16 % 16;
                    const int64_t m = (g + k) * 16 + i % 16;
                    if (t >= tr.n || m >= a.M) continue;
                    float sum = 0.0f;
#pragma unroll
                    for (int p = 0; p < KS; ++p) sum += red[(k * KS + p) * 256 + i % 256];
                    y[t * a.M + m] = from_f32<Y>(sum);
                }
            }
        }
    }
}

template <int NT, class X, bool IDS>
static hipError_t run_mv(const mx4_args & a, const X * x, int64_t ldx, int ytype, hipStream_t st) {
    const int64_t tiles = IDS ? id_tiles(a, 16 * NT) : (a.T + 16 * NT - 1) / (16 * NT);
    const int64_t busy = mv_busy(a, NT);
    const int ks = mv_split(a, NT);
    return with_type(ytype, [&](auto t) {
        using Y = decltype(t);
        auto go = [&](auto split) {
            constexpr int KS = split;
            const int64_t rounds = ((a.M + 15) / 16 + MV_WAVES / KS - 1) / (MV_WAVES / KS);
            const int64_t fair = (MV_GROUPS + busy - 1) / busy;   // each with its turn of the groups
            const int per_tile = (int) (rounds < fair ? rounds : fair);
            if (per_tile * tiles > MAX_WAVES / MV_WAVES) return hipErrorInvalidConfiguration;
            return launch(k_mx4_mv<NT, KS, X, Y, IDS>, (unsigned) (per_tile * tiles), 64 * MV_WAVES, mv_lds(a, NT, KS), st, a, x, ldx,
                          per_tile);
        };
        switch (ks) {
            case 1: return go(std::integral_constant<int, 1>{});
            case 2: return go(std::integral_constant<int, 2>{});
            case 4: return go(std::integral_constant<int, 4>{});
            default: return go(std::integral_constant<int, 8>{});
        }
    });
}

static mx4_args product_args(const mx4_mat & w, const mx4_mat & x, const moe_view * v, void * y) {
    mx4_args a{};
    a.w_codes = w.codes;
    a.w_scales = w.scales;
    a.M = w.rows;
    a.KB = (int) (w.K / MX4_BLOCK);
    a.w_codes_stride = w.rows * (w.K / 2);
    a.w_scales_stride = (w.K + MX4_PLANE - 1) / MX4_PLANE * w.rows * 8;
    a.x_codes = x.codes;
    a.x_scales = x.scales;
    a.x_rows = x.rows;
    a.T = v ? v->pairs : x.rows;
    a.y = y;
    if (v) {
        a.order = v->order;
        a.offsets = v->offsets;
        a.n_expert = v->n_expert;
        a.used = v->used;
    }
    return a;
}

mx4_needs mx4_product_needs(const mx4_mat & w, int64_t x_rows, const moe_view * v) {
    const mx4_args a = product_args(w, {nullptr, nullptr, x_rows, w.K}, v, nullptr);
    return {!float_rows(a), few_rows(a) ? 0 : mx4_tile_workspace(a)};
}

hipError_t mx4_product(const mx4_mat & w, const mx4_mat & x, const moe_view * v, int ytype, void * y, void * part, hipStream_t st) {
    const mx4_args a = product_args(w, x, v, y);
    const mxfp4 * in = nullptr;
    if (!few_rows(a)) return mx4_product_tile(a, (float *) part, ytype, st);
    if (v) return run_mv<1, mxfp4, true>(a, in, 0, ytype, st);
    return mv_tiles(a) == 2 ? run_mv<2, mxfp4, false>(a, in, 0, ytype, st) : run_mv<1, mxfp4, false>(a, in, 0, ytype, st);
}

hipError_t mx4_product_float(const mx4_mat & w, int xtype, const void * x, int64_t ldx, int64_t x_rows, const moe_view * v,
                             int ytype, void * y, hipStream_t st) {
    const mx4_args a = product_args(w, {nullptr, nullptr, x_rows, w.K}, v, y);
    return with_type(xtype, [&](auto t) {
        using X = decltype(t);
        return v ? run_mv<1, X, true>(a, (const X *) x, ldx, ytype, st) : run_mv<1, X, false>(a, (const X *) x, ldx, ytype, st);
    });
}

}  // namespace mi355x_ops
