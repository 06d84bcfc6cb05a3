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
//   - Row r's 16-B block b lies in slot b ^ (r / 2 % 8): the 64 banks hold two rows, so that any 16
//     rows that differ mod 16 are read without a conflict.  The copies to shared memory can only
//     write lane after lane, so the order is made on the reading side: each lane fetches the block
//     that belongs in its slot.
//   - Past K both exponents are 0, so that the product of two codes vanishes (2^-254 of it).
//   - Past M and T rows repeat the last one; their results are not stored.
#include "mx4.h"

#include <utility>

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
    static_assert(CI % NW == 0 && SI % NW == 0 && NW % 2 == 0, "every wave issues the same copies");
};

// the fragments of one step: FM of the weights, FN of x
template <int FM, int FN> struct frags {
    int4 a[FM], b[FN];
    // one of the FM + FN reads; the first instructions want a[0] and b[0]
    template <int I> __device__ __forceinline__ void load(const char * ca, const char * cb) {
        if constexpr (I == 0) a[0] = *(const int4 *) ca;
        else if constexpr (I <= FN) b[I - 1] = *(const int4 *) (cb + (I - 1) * 32 * 128);
        else a[I - FN] = *(const int4 *) (ca + (I - FN) * 32 * 128);
    }
};

template <int N, class F> static __device__ __forceinline__ void unroll(F && f) {
    [&]<int... I>(std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }(std::make_integer_sequence<int, N>{});
}

// step J's instructions, with between(i) in front of the i-th: a wave issues in order, and a queue
// that is full of its memory instructions would hold up the next matrix instruction behind them
template <int J, int FM, int FN, class F>
static __device__ __forceinline__ void mma_step(v16f (&acc)[FM][FN], const frags<FM, FN> & f, const int (&sa)[FM],
                                                const int (&sb)[FN], F && between) {
    unroll<FM * FN>([&](auto i) {
        constexpr int m = i / FN, n = i % FN;
        between(i);
        __builtin_amdgcn_sched_barrier(0);
        acc[m][n] = mfma_mx4_32<J>(f.a[m], f.b[n], acc[m][n], sa[m], sb[n]);
        __builtin_amdgcn_sched_barrier(0);
    });
}

// Workgroup -> tile.  Consecutive workgroups go round the eight XCDs: each XCD gets one run of the
// tiles, so that what its workgroups share meets in its L2.  A run goes along GROUP x tiles, then
// to the next weight tile: the 32 that an XCD has at a time are about 4 by 8.
static __device__ __forceinline__ void tile_of(unsigned id, unsigned tiles_m, unsigned tiles_n, unsigned & tm, unsigned & tn) {
    constexpr unsigned GROUP = 8;
    const unsigned n = tiles_m * tiles_n, xcd = id & 7;
    id = xcd * (n >> 3) + min(xcd, n & 7) + (id >> 3);
    const unsigned g = id / (GROUP * tiles_m), wide = min(GROUP, tiles_n - g * GROUP);
    id -= g * GROUP * tiles_m;
    tm = id / wide;
    tn = g * GROUP + id % wide;
}

template <int FM, int FN, int WM, int WN, class Y, bool IDS>
static __global__ void __launch_bounds__(64 * WM * WN) k_mx4_tile(mx4_args a, unsigned tiles_m, unsigned tiles_n) {
    using S = tile_shape<FM, FN, WM, WN>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int64_t m0 = (int64_t) tm * S::TM;
    const tile_rows tr = IDS ? find_tile(a, tn, S::TN) : tile_rows{0, (int64_t) tn * S::TN, min((int64_t) S::TN, a.T - (int64_t) tn * S::TN)};
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
    // the block that this lane copies: its rows are 8 (wave + k NW) + lane / 8, NW even
    const int blk = (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4));
    // copy k of plane s into buffer `into`: codes, then exponents
    constexpr int CK = S::CI / S::NW, COPIES = CK + S::SI / S::NW;
    auto copy = [&](int s, int64_t at, int into, auto kc) {
        constexpr int k = kc;
        const unsigned to = lds0 + into * S::STAGE;
        if constexpr (k < CK) dma16(code_row[k] + at, to + (wave + k * S::NW) * 1024);
        else dma4(exp_row[k - CK] + s * exp_step[k - CK], to + S::CODES + (wave + (k - CK) * S::NW) * 256);
    };
    auto code_at = [&](int s) { return (int64_t) min(s * 8 + blk, a.KB - 1) * 16; };

    const int wm = wave % WM * 32 * FM, wn = S::TM + wave / WM * 32 * FN;
    const int r31 = lane & 31, half = lane >> 5;
    const char * ca = lds + (wm + r31) * 128, * cb = lds + (wn + r31) * 128;
    const char * ea = lds + S::CODES + (wm + r31) * 8 + half * 4, * eb = lds + S::CODES + (wn + r31) * 8 + half * 4;
    int slot[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) slot[j] = ((j + 4 * half) ^ (r31 >> 1 & 7)) * 16;
    auto load_exps = [&](int s, int (&na)[FM], int (&nb)[FN]) {
        const int at = (s & 1) * S::STAGE;
#pragma unroll
        for (int i = 0; i < FM; ++i) na[i] = *(const int *) (ea + at + i * 32 * 8);
#pragma unroll
        for (int i = 0; i < FN; ++i) nb[i] = *(const int *) (eb + at + i * 32 * 8);
    };
    auto take_exps = [&](int s, int (&sa)[FM], int (&sb)[FN], const int (&na)[FM], const int (&nb)[FN]) {
        const int left = min(max(a.KB - s * 8 - 4 * half, 0), 4);   // this lane's blocks within K
        const int mask = left == 4 ? ~0 : (1 << (8 * left)) - 1;
#pragma unroll
        for (int i = 0; i < FM; ++i) sa[i] = na[i] & mask;
#pragma unroll
        for (int i = 0; i < FN; ++i) sb[i] = nb[i] & mask;
    };

    // A step's fragments are read between the instructions of the one before.  Before a plane's last
    // step all waves have read its buffer and the next plane has come: the barrier stands there.
    // Then the next plane's first fragments are read, and the plane after it is copied during this
    // step (part 0) and the next plane's first two (parts 1 and 2).
    constexpr int INS = FM * FN, FR = FM + FN, EVERY = INS / FR > 0 ? INS / FR : 1;
    constexpr int SLOTS = INS / 2, PER = (COPIES + 3 * SLOTS - 1) / (3 * SLOTS);   // copies in front of every second one
    v16f acc[FM][FN] = {};
    frags<FM, FN> f0, f1;
    int sa[FM], sb[FN], na[FM], nb[FN];
    const int last = planes - 1;
    auto reads = [&](frags<FM, FN> & f, int at, int j, auto i) {
        if constexpr (i % EVERY == 0 && i / EVERY < FR) f.template load<i / EVERY>(ca + at + slot[j], cb + at + slot[j]);
    };
    auto copies = [&](int s, int64_t at, int into, auto part, auto i) {
        if constexpr (i % 2 == 1)
            unroll<PER>([&](auto k) {
                constexpr int c = (part * SLOTS + i / 2) * PER + k;
                if constexpr (c < COPIES) copy(s, at, into, std::integral_constant<int, c>{});
            });
    };
    constexpr std::integral_constant<int, 0> P0{};
    constexpr std::integral_constant<int, 1> P1{};
    constexpr std::integral_constant<int, 2> P2{};
    unroll<COPIES>([&](auto k) { copy(0, code_at(0), 0, k); });
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    unroll<INS>([&](auto i) { copies(min(1, last), code_at(min(1, last)), 1, P0, i); });
    unroll<FR>([&](auto i) { f0.template load<i>(ca + slot[0], cb + slot[0]); });
    load_exps(0, na, nb);
    take_exps(0, sa, sb, na, nb);
    for (int s = 0; s < last; ++s) {
        const int at = (s & 1) * S::STAGE, to = (s + 1) & 1;
        const int64_t from = code_at(s + 1);
        mma_step<0>(acc, f0, sa, sb, [&](auto i) { reads(f1, at, 1, i); copies(s + 1, from, to, P1, i); });
        mma_step<1>(acc, f1, sa, sb, [&](auto i) { reads(f0, at, 2, i); copies(s + 1, from, to, P2, i); });
        mma_step<2>(acc, f0, sa, sb, [&](auto i) { reads(f1, at, 3, i); });
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        load_exps(s + 1, na, nb);
        // behind the last plane the last one comes again, into a buffer that nothing reads any more
        const int next = min(s + 2, last);
        const int64_t next_from = code_at(next);
        mma_step<3>(acc, f1, sa, sb, [&](auto i) { reads(f0, S::STAGE - at, 0, i); copies(next, next_from, s & 1, P0, i); });
        take_exps(s + 1, sa, sb, na, nb);
    }
    const int at = (last & 1) * S::STAGE;
    mma_step<0>(acc, f0, sa, sb, [&](auto i) { reads(f1, at, 1, i); });
    mma_step<1>(acc, f1, sa, sb, [&](auto i) { reads(f0, at, 2, i); });
    mma_step<2>(acc, f0, sa, sb, [&](auto i) { reads(f1, at, 3, i); });
    mma_step<3>(acc, f1, sa, sb, [](auto) {});
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no copy is left when the shared memory is given back

    // The results go out through shared memory: straight from the registers a store would touch 32 x
    // rows with 16 bytes each.  Rows of TM outputs lie 16 B past a multiple of the 64 banks apart, so
    // that 16 x rows times four neighbouring outputs cover them.
    constexpr int ROW = S::TM * (int) sizeof(Y) + 16;
    constexpr int PASSES = (S::TN * ROW + 2 * S::STAGE - 1) / (2 * S::STAGE), PT = S::TN / PASSES;
    static_assert(PT % 32 == 0 && PT * ROW <= 2 * S::STAGE, "whole fragments in a pass");
    const int cols = (int) min((int64_t) S::TM, a.M - m0);
    const bool wide = a.M * (int64_t) sizeof(Y) % 16 == 0;
    Y * out = y + tr.first * a.M + m0;
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
        __syncthreads();
#pragma unroll
        for (int n = 0; n < FN; ++n) {
            const int t = wn - S::TM + n * 32 - pass * PT;
            if (t < 0 || t >= PT) continue;
#pragma unroll
            for (int m = 0; m < FM; ++m)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    pack<Y, 4> q;
#pragma unroll
                    for (int k = 0; k < 4; ++k) q.v[k] = from_f32<Y>(acc[m][n][i + k]);
                    *(pack<Y, 4> *) (lds + (t + r31) * ROW + (wm + m * 32 + 2 * i + 4 * half) * sizeof(Y)) = q;
                }
        }
        __syncthreads();
        const int rows = (int) min((int64_t) PT, tr.n - pass * PT);
        if (wide) {
            constexpr int V = 16 / sizeof(Y), PER = S::TM / V;
            for (int i = threadIdx.x; i < rows * PER; i += 64 * S::NW)
                if (i % PER * V < cols)
                    *(pack<Y, V> *) (out + (int64_t) (pass * PT + i / PER) * a.M + i % PER * V) =
                        *(const pack<Y, V> *) (lds + i / PER * ROW + i % PER * 16);
        } else {
            for (int i = threadIdx.x; i < rows * S::TM; i += 64 * S::NW)
                if (i % S::TM < cols)
                    out[(int64_t) (pass * PT + i / S::TM) * a.M + i % S::TM] =
                        *(const Y *) (lds + i / S::TM * ROW + i % S::TM * (int) sizeof(Y));
        }
    }
}

template <int FM, int FN, int WM, int WN, bool IDS>
static hipError_t run_tile(const mx4_args & a, int ytype, hipStream_t st) {
    using S = tile_shape<FM, FN, WM, WN>;
    const int64_t tm = (a.M + S::TM - 1) / S::TM, tn = IDS ? id_tiles(a, S::TN) : (a.T + S::TN - 1) / S::TN;
    if (tm * tn > MAX_WAVES / S::NW) return hipErrorInvalidConfiguration;
    return with_type(ytype, [&](auto t) {
        using Y = decltype(t);
        auto * k = k_mx4_tile<FM, FN, WM, WN, Y, IDS>;
        const hipError_t e = hipFuncSetAttribute((const void *) k, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * S::STAGE);
        if (e != hipSuccess) return e;
        k<<<(unsigned) (tm * tn), 64 * S::NW, 2 * S::STAGE, st>>>(a, (unsigned) tm, (unsigned) tn);
        return hipGetLastError();
    });
}

hipError_t mx4_product_tile(const mx4_args & a, int ytype, hipStream_t st) {
    return a.offsets ? run_tile<4, 4, 2, 2, true>(a, ytype, st) : run_tile<4, 4, 2, 2, false>(a, ytype, st);
}

}  // namespace mi355x_ops
