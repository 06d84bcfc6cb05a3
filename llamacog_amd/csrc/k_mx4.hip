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
// times as many rows as its lanes hold, loads first, to keep bytes in flight.
constexpr int QROWS = 4;

template <class T, bool VEC>
static __global__ void __launch_bounds__(256) k_mx4_quantize(const T * __restrict__ x, int64_t ldx, int64_t rows, int64_t K, int lsh,
                                                      uint8_t * __restrict__ codes, uint8_t * __restrict__ scales) {
    const int64_t c = (int64_t) blockIdx.y << lsh | (threadIdx.x & ((1 << lsh) - 1));
    if (c >= K / 8) return;   // K / 8 is a multiple of four: the four lanes of a block stay together
    const int rp = 256 >> lsh;
    const int64_t row0 = (int64_t) blockIdx.x * rp * QROWS + (threadIdx.x >> lsh);
    float v[QROWS][8];
#pragma unroll
    for (int i = 0; i < QROWS; ++i) {
        const int64_t row = min(row0 + (int64_t) i * rp, rows - 1);
        load8<T, VEC>(x + row * ldx + c * 8, v[i]);
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
    const dim3 grid(ceil_div(rows, (int64_t) (256 >> lsh) * QROWS), ceil_div(K / 8, 1 << lsh));
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        // a lane's 8 elements are read with 16-B accesses where every row starts on 16 B
        const bool vec = ((uintptr_t) x % 16 == 0) && (ldx * (int64_t) sizeof(T) % 16 == 0);
        if (vec) k_mx4_quantize<T, true><<<grid, 256, 0, st>>>((const T *) x, ldx, rows, K, lsh, codes, scales);
        else k_mx4_quantize<T, false><<<grid, 256, 0, st>>>((const T *) x, ldx, rows, K, lsh, codes, scales);
        return hipGetLastError();
    });
}

// ---- values back -----------------------------------------------------------------------------
template <class T>
static __global__ void __launch_bounds__(256) k_mx4_dequantize(const uint8_t * __restrict__ codes, const uint8_t * __restrict__ scales,
                                                        int64_t rows, int64_t K, int lsh, T * __restrict__ y) {
    const int64_t c = (int64_t) blockIdx.y << lsh | (threadIdx.x & ((1 << lsh) - 1));
    if (c >= K / 8) return;
    const int rp = 256 >> lsh;
    const int64_t row0 = (int64_t) blockIdx.x * rp * QROWS + (threadIdx.x >> lsh);
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
    const dim3 grid(ceil_div(m.rows, (int64_t) (256 >> lsh) * QROWS), ceil_div(m.K / 8, 1 << lsh));
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        k_mx4_dequantize<T><<<grid, 256, 0, st>>>(m.codes, m.scales, m.rows, m.K, lsh, (T *) y);
        return hipGetLastError();
    });
}

// ---- product, few rows -----------------------------------------------------------------------
// A workgroup takes 16 weight rows and 16 NT x rows; its waves take the 256-element planes of K
// in turn and their sums are joined in shared memory.  Weight rows are the matrix instruction's
// first operand (16x16x128: lane l holds row l % 16 and the 32-block l / 16, one 16-B load), x rows
// the second, so a lane's four results are four neighbouring outputs of one x row.
template <int NT, int W, class Y, bool IDS>
static __global__ void __launch_bounds__(64 * W) k_mx4_mv(mx4_args a) {
    constexpr int U = NT == 1 ? 4 : 2;   // planes whose loads are issued together
    __shared__ float red[W][NT][16][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r = lane & 15, q = lane >> 4;
    const int64_t groups = (a.M + 15) / 16;
    const int64_t m0 = (blockIdx.x % groups) * 16;
    const int64_t tile = blockIdx.x / groups;
    tile_rows tr = IDS ? find_tile(a, tile, 16 * NT) : tile_rows{0, tile * 16 * NT, min((int64_t) 16 * NT, a.T - tile * 16 * NT)};
    if (tr.n <= 0) return;
    Y * y = (Y *) a.y;
    if (IDS && tr.expert < 0) {   // pairs that no expert takes
        for (int i = threadIdx.x; i < 16 * tr.n; i += 64 * W)
            if (m0 + (i & 15) < a.M) y[(tr.first + (i >> 4)) * a.M + m0 + (i & 15)] = from_f32<Y>(0.0f);
        return;
    }
    const uint8_t * wc = a.w_codes + tr.expert * a.w_codes_stride;
    const uint8_t * ws = a.w_scales + tr.expert * a.w_scales_stride;
    const int64_t row = min(m0 + r, a.M - 1);
    const uint8_t * wrow = wc + row * (int64_t) a.KB * 16;
    int64_t xr[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xr[n] = x_row<IDS>(a, tr.first + min((int64_t) 16 * n + r, tr.n - 1));
    const int S = (a.KB + 7) / 8;
    v4f acc[NT] = {};
    for (int s0 = wave; s0 < S; s0 += W * U) {
        int4 w[U][2], x[U][NT][2];
        uint32_t sw[U][2], sx[U][NT][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min(s0 + u * W, S - 1);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int64_t b = min(s * 8 + 4 * j + q, a.KB - 1);
                w[u][j] = *(const int4 *) (wrow + b * 16);
                sw[u][j] = *(const uint32_t *) (ws + ((int64_t) s * a.M + row) * 8 + 4 * j);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    x[u][n][j] = *(const int4 *) (a.x_codes + (xr[n] * a.KB + b) * 16);
                    sx[u][n][j] = *(const uint32_t *) (a.x_scales + (s * a.x_rows + xr[n]) * 8 + 4 * j);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                // past K: zero codes and a finite exponent
                const bool in = (s0 + u * W) * 8 + 4 * j + q < a.KB;
                const int4 wv = in ? w[u][j] : int4{0, 0, 0, 0};
                const int wsc = in ? (int) (sw[u][j] >> (8 * q)) : 0;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int xsc = in ? (int) (sx[u][n][j] >> (8 * q)) : 0;
                    acc[n] = mfma_mx4_16(wv, x[u][n][j], acc[n], wsc, xsc);
                }
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) *(v4f *) &red[wave][n][r][4 * q] = acc[n];
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 256; i += 64 * W) {
        const int t = i >> 4, m = i & 15;
        if (t >= tr.n || m0 + m >= a.M) continue;
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) s += red[k][t >> 4][t & 15][m];
        y[(tr.first + t) * a.M + m0 + m] = from_f32<Y>(s);
    }
}

template <bool IDS> static hipError_t product_mv(const mx4_args & a, int64_t tokens, int ytype, hipStream_t st) {
    return with_type(ytype, [&](auto t) {
        using Y = decltype(t);
        const int64_t groups = (a.M + 15) / 16;
        const int64_t tiles = IDS ? id_tiles(a, 16) : (tokens + 15) / 16;
        k_mx4_mv<1, 4, Y, IDS><<<(unsigned) (groups * tiles), 256, 0, st>>>(a);
        return hipGetLastError();
    });
}

static mx4_args product_args(const mx4_mat & w, const mx4_mat & x, void * y) {
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
    a.T = x.rows;
    a.y = y;
    return a;
}

hipError_t mx4_product(const mx4_mat & w, const mx4_mat & x, int ytype, void * y, hipStream_t st) {
    const mx4_args a = product_args(w, x, y);
    if (x.rows > 64) return mx4_product_tile(a, ytype, st);
    return product_mv<false>(a, x.rows, ytype, st);
}

hipError_t mx4_product_id(const mx4_mat & w, const mx4_mat & x, const moe_view & v, int ytype, void * y, hipStream_t st) {
    mx4_args a = product_args(w, x, y);
    a.order = v.order;
    a.offsets = v.offsets;
    a.n_expert = v.n_expert;
    a.used = v.used;
    a.T = v.pairs;
    if (v.pairs > 64 * v.n_expert) return mx4_product_tile(a, ytype, st);
    return product_mv<true>(a, v.pairs, ytype, st);
}

}  // namespace mi355x_ops
