// mx4.h — device helpers of the MXFP4 kernels: the block format, the scaled matrix instructions
// and the search for a tile of sorted pairs.
#pragma once

#include "devops.h"
#include "mx4_rules.h"

namespace mi355x_ops {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

// ---- elements --------------------------------------------------------------------------------
template <class T> __device__ __forceinline__ void load8(const T * p, float (&v)[8]) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += N) {
        const pack<T, N> q = get<T, N>(p + i);
#pragma unroll
        for (int j = 0; j < N; ++j) v[i + j] = to_f32(q.v[j]);
    }
}

template <class T> __device__ __forceinline__ void store8(T * p, const float (&v)[8]) {
    constexpr int N = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 8; i += N) {
        pack<T, N> q;
#pragma unroll
        for (int j = 0; j < N; ++j) q.v[j] = from_f32<T>(v[i + j]);
        put<false>(p + i, q);
    }
}

template <int CTRL> __device__ __forceinline__ unsigned dpp_mov(unsigned v) {
    return (unsigned) __builtin_amdgcn_update_dpp(0, (int) v, CTRL, 0xf, 0xf, true);
}

// the exponent byte of the block that four neighbouring lanes hold, 8 elements each.  The maximum
// is taken over the magnitude's bits: they order as the numbers do, infinities and NaNs last.
__device__ __forceinline__ unsigned mx4_block_exponent(const float (&v)[8]) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    m = max(m, dpp_mov<0xB1>(m));   // quad_perm 1 0 3 2
    m = max(m, dpp_mov<0x4E>(m));   // quad_perm 2 3 0 1
    const unsigned e = m >> 23;     // 0 below 2^-126, where the exponent is at its least anyway
    return e == 255 ? 255u : e > 2 ? e - 2 : 0u;
}

// 2^(byte - 127); byte 0 is a number under the normal range
__device__ __forceinline__ float mx4_scale(unsigned e) { return __uint_as_float(e ? e << 23 : 1u << 22); }

// eight elements to codes, element i in bits 4 i: the conversion divides by the scale, rounds to
// nearest even and stops at 6
__device__ __forceinline__ uint32_t mx4_pack8(const float (&v)[8], unsigned e) {
    const float s = mx4_scale(e);
    unsigned q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], s, 3);
    return e == 255 ? 0u : q;
}

__device__ __forceinline__ void mx4_unpack8(uint32_t q, unsigned e, float (&v)[8]) {
    const float s = e == 255 ? __uint_as_float(0x7fc00000u) : mx4_scale(e);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const unsigned c = q >> (4 * i);
        // E2M1: (1 + m / 2) 2^(x - 1), m / 2 for x = 0
        const unsigned x = (c >> 1) & 3, m = c & 1;
        const unsigned bits = x ? (x + 126) << 23 | m << 22 : m ? 0x3f000000u : 0u;
        v[i] = __uint_as_float(bits | (c & 8) << 28) * s;   // exact: two bits times a power of two
    }
}

// ---- matrix instructions ---------------------------------------------------------------------
// 16x16x128, both operands FP4.  Lane l: row l % 16 of each operand, its elements 32 (l / 16) to
// 32 (l / 16) + 31 in 16 bytes, their exponent in byte 0 of the scale register; results: column
// l % 16 (second operand's row), rows 4 (l / 16) + i.
__device__ __forceinline__ v4f mfma_mx4_16(const int4 & a, const int4 & b, v4f c, int sa, int sb) {
    const v8i va = {a.x, a.y, a.z, a.w, 0, 0, 0, 0}, vb = {b.x, b.y, b.z, b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, 0, sa, 0, sb);
}

// ---- arguments of the products ---------------------------------------------------------------
struct mx4_args : product_size {
    const uint8_t * w_codes;
    const uint8_t * w_scales;
    int64_t w_codes_stride, w_scales_stride;   // from one expert's matrix to the next
    const uint8_t * x_codes;
    const uint8_t * x_scales;
    int64_t x_rows;                            // rows of the x matrix (its scale planes' stride)
    const int32_t * order;
    const int32_t * offsets;
    int used;                                  // 0: x rows are in sorted order
    void * y;
};

// k_mx4_gemm.hip; by experts where a.n_expert is not 0.  part: mx4_tile_workspace(a) bytes
int64_t mx4_tile_workspace(const mx4_args & a);
hipError_t mx4_product_tile(const mx4_args & a, float * part, int ytype, hipStream_t st);

// ---- tiles of sorted pairs -------------------------------------------------------------------
struct tile_rows {
    int64_t expert;   // -1: rows behind the last expert's
    int64_t first;    // first sorted row
    int64_t n;        // rows, 0: no such tile
};

// most tiles of `rows` sorted rows that any routing of a.T pairs can need, the rows behind the last
// expert's included: sum of ceil(n_e / rows) over at most min(T, n_expert) experts and one rest
static inline int64_t id_tiles(const mx4_args & a, int rows) {
    const int64_t used = a.T < a.n_expert ? a.T : a.n_expert;
    return a.T / rows + used + 1;
}

// The tiles of `rows` sorted rows: experts in order, then the rows that no expert takes.  Every wave
// counts them by itself, lane l those of its ceil(n_expert / 64) experts.
struct tile_scan {
    int e0, e1, mine, upto;   // this lane's experts and tiles, and the tiles up to them
    int total, held;          // all experts' tiles, their rows
    int rows;

    __device__ __forceinline__ tile_scan(const mx4_args & a, int rows) : rows(rows) {
        const int lane = threadIdx.x & 63;
        const int per = (a.n_expert + 63) / 64;
        e0 = min(lane * per, a.n_expert);
        e1 = min(e0 + per, a.n_expert);
        mine = 0;
        for (int e = e0; e < e1; ++e) mine += tiles_of(a.offsets[e + 1] - a.offsets[e], rows);
        upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(upto, d);
            if (lane >= d) upto += o;
        }
        total = max(0, __builtin_amdgcn_readlane(upto, 63));
        held = max(0, __builtin_amdgcn_readfirstlane(a.offsets[a.n_expert]));
    }
    // with the rest's
    __device__ __forceinline__ int64_t tiles(const mx4_args & a) const { return total + max((int64_t) 0, (a.T - held + rows - 1) / rows); }

    __device__ __forceinline__ tile_rows tile(const mx4_args & a, int64_t i) const {
        tile_rows tr;
        if (i >= total) {
            tr.expert = -1;
            tr.first = held + (i - total) * rows;
            tr.n = max((int64_t) 0, min((int64_t) rows, a.T - tr.first));
            return tr;
        }
        const unsigned long long hit = __ballot(upto > (int) i);
        const int owner = (int) __builtin_ctzll(hit);
        int e = e0, first = 0, n = 0;
        if ((int) (threadIdx.x & 63) == owner) {
            int left = (int) i - (upto - mine);
            for (;; ++e) {
                n = a.offsets[e + 1] - a.offsets[e];
                const int t = tiles_of(n, rows);
                if (left < t || e + 1 >= e1) break;
                left -= t;
            }
            first = a.offsets[e] + left * rows;
            n = min(rows, n - left * rows);
        }
        tr.expert = __builtin_amdgcn_readlane(e, owner);
        tr.first = max(0, __builtin_amdgcn_readlane(first, owner));
        tr.n = min((int64_t) __builtin_amdgcn_readlane(n, owner), a.T - tr.first);   // whatever the offsets hold
        return tr;
    }
};

// the x row of y row p, inside the matrix whatever the order holds
template <bool IDS> __device__ __forceinline__ int64_t x_row(const mx4_args & a, int64_t p) {
    if (!IDS || a.used == 0) return p;
    return min((int64_t) max(0, a.order[p] / a.used), a.x_rows - 1);
}

}  // namespace mi355x_ops
