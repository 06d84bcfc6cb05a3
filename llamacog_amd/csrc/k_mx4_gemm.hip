// k_mx4_gemm.hip — the MXFP4 product for many rows, dense and by experts: tiles on
// v_mfma_scale_f32_32x32x64 (both operands FP4).
//
// A workgroup of WM x WN waves computes TM = 32 FM WM weight rows by TN = 32 FN WN x rows, a plane
// of 256 elements of K at a time.  Both operands' codes (128 B of a row) and exponents (8 B) go
// from memory to shared memory without registers, one plane ahead of the arithmetic in a second
// buffer.
//   - The 32x32x64 instruction wants from lane l 32 consecutive elements of row l % 32, and their
//     exponent in a byte of a register that the instruction names.  Which 32-blocks of K meet in an
//     instruction is free as long as both operands agree: step j takes block j from lanes 0-31 and
//     block 4 + j from lanes 32-63, so that a lane's four exponents of a plane are one aligned word.
//   - Row r's 16-B block b lies in slot b ^ (r % 8): eight neighbouring lanes of a fragment read hit
//     eight different 16-B columns.  The copies to shared memory can only write lane after lane, so
//     the order is made on the reading side: a lane fetches block (l % 8) ^ (l / 8) of its row.
//   - Past K both exponents are 0, so that the product of two codes vanishes (2^-254 of it).
//   - Past M and T rows repeat the last one; their results are not stored.
#include "mx4.h"

namespace mi355x_ops {

typedef __attribute__((address_space(3))) char lds_char;

// 16 or 4 B per lane from memory to shared memory at `to` + lane * size, in flight until vmcnt says
static __device__ __forceinline__ void dma16(const uint8_t * from, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}
static __device__ __forceinline__ void dma4(const uint8_t * from, unsigned to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(from) : "memory");
}

// 32x32x64, both operands FP4, exponents in byte J of the scale registers.  Lane l: row l % 32 of each
// operand, 32 elements in 16 bytes; results: column l % 32 (second operand's row), rows
// 8 (i / 4) + 4 (l / 32) + i % 4.
template <int J> static __device__ __forceinline__ v16f mfma_mx4_32(const int4 & a, const int4 & b, v16f c, int sa, int sb) {
    const v8i va = {a.x, a.y, a.z, a.w, 0, 0, 0, 0}, vb = {b.x, b.y, b.z, b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, c, 4, 4, J, sa, J, sb);
}

template <int FM, int FN, int WM, int WN> struct tile_shape {
    static constexpr int TM = 32 * FM * WM, TN = 32 * FN * WN, NW = WM * WN;
    static constexpr int CODES = (TM + TN) * 128, STAGE = CODES + (TM + TN) * 8;
    static constexpr int CI = (TM + TN) / 8;    // 1-KiB copies of a plane's codes: 8 rows each
    static constexpr int SI = (TM + TN) / 32;   // 256-B copies of its exponents: 32 rows each
    static_assert(CI % NW == 0 && SI % NW == 0 && TM % 32 == 0, "every wave issues the same copies");
};

template <int J, int FM, int FN>
static __device__ __forceinline__ void mma_step(v16f (&acc)[FM][FN], const char * ca, const char * cb, int lane, const int (&sa)[FM],
                                                const int (&sb)[FN]) {
    const int slot = ((J + 4 * (lane >> 5)) ^ (lane & 7)) * 16;
    int4 a[FM], b[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) a[i] = *(const int4 *) (ca + i * 32 * 128 + slot);
#pragma unroll
    for (int i = 0; i < FN; ++i) b[i] = *(const int4 *) (cb + i * 32 * 128 + slot);
#pragma unroll
    for (int n = 0; n < FN; ++n)
#pragma unroll
        for (int m = 0; m < FM; ++m) acc[m][n] = mfma_mx4_32<J>(a[m], b[n], acc[m][n], sa[m], sb[n]);
}

template <class Y, int N> static __device__ __forceinline__ void store_out(Y * y, const float * v, int64_t left) {
    if (left >= N) {
        pack<Y, N> q;
#pragma unroll
        for (int i = 0; i < N; ++i) q.v[i] = from_f32<Y>(v[i]);
        *(pack<Y, N> *) y = q;
    } else {
        for (int i = 0; i < left; ++i) y[i] = from_f32<Y>(v[i]);
    }
}

template <int FM, int FN, int WM, int WN, class Y, bool IDS>
static __global__ void __launch_bounds__(64 * WM * WN) k_mx4_tile(mx4_args a, int64_t tiles_m, int64_t tiles_n) {
    using S = tile_shape<FM, FN, WM, WN>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t id = blockIdx.x;
    const int64_t m0 = id / tiles_n * S::TM;
    const tile_rows tr = IDS ? find_tile(a, id % tiles_n, S::TN)
                             : tile_rows{0, id % tiles_n * S::TN, min((int64_t) S::TN, a.T - id % tiles_n * S::TN)};
    if (tr.n <= 0) return;
    Y * y = (Y *) a.y;
    if (IDS && tr.expert < 0) {   // pairs that no expert takes
        const int64_t cols = min((int64_t) S::TM, a.M - m0);
        for (int64_t i = threadIdx.x; i < S::TM * tr.n; i += 64 * S::NW)
            if (i % S::TM < cols) y[(tr.first + i / S::TM) * a.M + m0 + i % S::TM] = from_f32<Y>(0.0f);
        return;
    }
    const int planes = (a.KB + 7) / 8;

    // this wave's copies: rows of the weights first, then of x
    const uint8_t * code_row[S::CI / S::NW];
    const uint8_t * exp_row[S::SI / S::NW];
    int64_t exp_step[S::SI / S::NW];
    const uint8_t * wc = a.w_codes + tr.expert * a.w_codes_stride;
    const uint8_t * ws = a.w_scales + tr.expert * a.w_scales_stride;
#pragma unroll
    for (int k = 0; k < S::CI / S::NW; ++k) {
        const int r = (wave + k * S::NW) * 8 + (lane >> 3);
        const int64_t row = r < S::TM ? min(m0 + r, a.M - 1) : x_row<IDS>(a, tr.first + min((int64_t) r - S::TM, tr.n - 1));
        code_row[k] = (r < S::TM ? wc : a.x_codes) + row * a.KB * 16;
    }
#pragma unroll
    for (int k = 0; k < S::SI / S::NW; ++k) {
        const int r = (wave + k * S::NW) * 32 + (lane >> 1);
        const int64_t row = r < S::TM ? min(m0 + r, a.M - 1) : x_row<IDS>(a, tr.first + min((int64_t) r - S::TM, tr.n - 1));
        exp_row[k] = (r < S::TM ? ws : a.x_scales) + row * 8 + (lane & 1) * 4;
        exp_step[k] = (r < S::TM ? a.M : a.x_rows) * 8;
    }
    const unsigned lds0 = (unsigned) (uintptr_t) (lds_char *) lds;
    const int blk = (lane & 7) ^ (lane >> 3);
    auto copy_plane = [&](int s) {
        const unsigned to = lds0 + (s & 1) * S::STAGE;
        const int64_t at = (int64_t) min(s * 8 + blk, a.KB - 1) * 16;
#pragma unroll
        for (int k = 0; k < S::CI / S::NW; ++k) dma16(code_row[k] + at, to + (wave + k * S::NW) * 1024);
#pragma unroll
        for (int k = 0; k < S::SI / S::NW; ++k)
            dma4(exp_row[k] + s * exp_step[k], to + S::CODES + (wave + k * S::NW) * 256);
    };

    const int wm = wave % WM * 32 * FM, wn = S::TM + wave / WM * 32 * FN;
    v16f acc[FM][FN] = {};
    copy_plane(0);
    for (int s = 0; s < planes; ++s) {
        // this plane has come, and no wave still reads the other buffer
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        if (s + 1 < planes) copy_plane(s + 1);
        const char * buf = lds + (s & 1) * S::STAGE;
        const char * ca = buf + (wm + (lane & 31)) * 128, * cb = buf + (wn + (lane & 31)) * 128;
        const char * ea = buf + S::CODES + (wm + (lane & 31)) * 8 + (lane >> 5) * 4;
        const char * eb = buf + S::CODES + (wn + (lane & 31)) * 8 + (lane >> 5) * 4;
        const int left = min(max(a.KB - s * 8 - 4 * (lane >> 5), 0), 4);   // blocks of this lane within K
        const unsigned mask = left == 4 ? ~0u : (1u << (8 * left)) - 1;
        int sa[FM], sb[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) sa[i] = (int) (*(const unsigned *) (ea + i * 32 * 8) & mask);
#pragma unroll
        for (int i = 0; i < FN; ++i) sb[i] = (int) (*(const unsigned *) (eb + i * 32 * 8) & mask);
        mma_step<0>(acc, ca, cb, lane, sa, sb);
        mma_step<1>(acc, ca, cb, lane, sa, sb);
        mma_step<2>(acc, ca, cb, lane, sa, sb);
        mma_step<3>(acc, ca, cb, lane, sa, sb);
    }
    const bool wide = a.M % 4 == 0;
#pragma unroll
    for (int n = 0; n < FN; ++n) {
        const int64_t t = wn - S::TM + n * 32 + (lane & 31);
        if (t >= tr.n) continue;
#pragma unroll
        for (int m = 0; m < FM; ++m)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int64_t row = m0 + wm + m * 32 + 2 * i + 4 * (lane >> 5);
                float v[4] = {acc[m][n][i], acc[m][n][i + 1], acc[m][n][i + 2], acc[m][n][i + 3]};
                Y * to = y + (tr.first + t) * a.M + row;
                if (wide) {
                    if (row < a.M) store_out<Y, 4>(to, v, 4);
                } else {
                    for (int k = 0; k < 4; ++k)
                        if (row + k < a.M) to[k] = from_f32<Y>(v[k]);
                }
            }
    }
}

template <int FM, int FN, int WM, int WN, bool IDS>
static hipError_t run_tile(const mx4_args & a, int ytype, hipStream_t st) {
    using S = tile_shape<FM, FN, WM, WN>;
    const int64_t tm = (a.M + S::TM - 1) / S::TM, tn = IDS ? id_tiles(a, S::TN) : (a.T + S::TN - 1) / S::TN;
    return with_type(ytype, [&](auto t) {
        using Y = decltype(t);
        auto * k = k_mx4_tile<FM, FN, WM, WN, Y, IDS>;
        const hipError_t e = hipFuncSetAttribute((const void *) k, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * S::STAGE);
        if (e != hipSuccess) return e;
        k<<<(unsigned) (tm * tn), 64 * S::NW, 2 * S::STAGE, st>>>(a, tm, tn);
        return hipGetLastError();
    });
}

hipError_t mx4_product_tile(const mx4_args & a, int ytype, hipStream_t st) {
    return a.offsets ? run_tile<4, 4, 2, 2, true>(a, ytype, st) : run_tile<4, 4, 2, 2, false>(a, ytype, st);
}

}  // namespace mi355x_ops
