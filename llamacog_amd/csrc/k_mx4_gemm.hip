// k_mx4_gemm.hip — the MXFP4 product for many rows, dense and by experts: tiles on
// v_mfma_scale_f32_32x32x64 (both operands FP4).
//
// A workgroup of WM x WN waves computes TM = 32 FM WM weight rows by TN = 32 FN WN x rows, a plane of
// 256 elements of K at a time.  Both operands' codes (128 B of a row, a cache line) and exponents
// (8 B) go from memory to shared memory without registers, into a ring of STAGES planes.
//   - The 32x32x64 instruction wants from lane l 32 consecutive elements of row l % 32, and their
//     exponent in a byte of a register that the instruction names.  Which 32-blocks of K meet in an
//     instruction is free as long as both operands agree: step j of a plane takes block j from lanes
//     0-31 and block 4 + j from lanes 32-63, so that a lane's four exponents are one aligned word.
//   - Row r's 16-B block b lies in slot b ^ (r / 2 % 8): the 64 banks hold two rows, so that any 16
//     rows that differ mod 16 are read without a conflict.  The copies to shared memory can only
//     write lane after lane, so the order is made on the reading side: each lane fetches the block
//     that belongs in its slot.
//   - Past K both exponents are 0, so that the product of two codes vanishes (2^-254 of it).
//   - Past M and T rows repeat the last one; their results are not stored.
// Bound by cycles: 2048 x 28672 x 8192 takes 432 thousand of them on random codes and 436 on zeros (251 and 193 us:
// the clock is 1.72 and 2.27 GHz), and the matrix cores are busy for 229 thousand, 53 %.  An eighth is the last round of
// tiles, half full; of a plane's about 3000 cycles in a 256 x 256 tile the matrix cores have 2048.  251 us are 3.8
// PFLOP/s, 4096 x 4096 x 28672 in 217 us 4.4; the instruction alone reaches 6.15 on random codes.  A row's 128 B of
// a plane are a whole cache line: planes of half that, in a ring of four, took 9 % longer.
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

template <int FM, int FN, int WM, int WN, int STAGES> struct tile_shape {
    static constexpr int TM = 32 * FM * WM, TN = 32 * FN * WN, NW = WM * WN;
    static constexpr int CODES = (TM + TN) * 128, STAGE = CODES + (TM + TN) * 8, LDS = STAGES * STAGE;
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
// to the next weight tile: the 32 that an XCD has at a time are about 4 by 8.  With GROUP 1 / 4 / 8 / 16,
// 2048 x 28672 x 8192 took 275 / 274 / 272 / 271 us, 4096 x 4096 x 28672 218 / 217 / 217 / 227, 2048 x 14336 x 4096
// 76 / 74 / 73 / 77.
static __device__ __forceinline__ void tile_of(unsigned id, unsigned tiles_m, unsigned tiles_n, unsigned & tm, unsigned & tn) {
    constexpr unsigned GROUP = 8;
    const unsigned n = tiles_m * tiles_n, xcd = id & 7;
    id = xcd * (n >> 3) + min(xcd, n & 7) + (id >> 3);
    const unsigned g = id / (GROUP * tiles_m), wide = min(GROUP, tiles_n - g * GROUP);
    id -= g * GROUP * tiles_m;
    tm = id / wide;
    tn = g * GROUP + id % wide;
}

template <int FM, int FN, int WM, int WN, int STAGES, class Y, bool IDS>
static __global__ void __launch_bounds__(64 * WM * WN) k_mx4_tile(mx4_args a, unsigned tiles_m, unsigned tiles_n) {
    using S = tile_shape<FM, FN, WM, WN, STAGES>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned id = (unsigned) group_id();
    unsigned tm, tn;
    tile_rows tr;
    if constexpr (IDS) {
        const tile_scan scan(a, S::TN);
        tiles_n = (unsigned) scan.tiles(a);   // the launch is for any routing
        if (id >= tiles_m * tiles_n) return;
        tile_of(id, tiles_m, tiles_n, tm, tn);
        tr = scan.tile(a, tn);
    } else {
        if (id >= tiles_m * tiles_n) return;
        tile_of(id, tiles_m, tiles_n, tm, tn);
        tr = {0, (int64_t) tn * S::TN, min((int64_t) S::TN, a.T - (int64_t) tn * S::TN)};
    }
    const int64_t m0 = (int64_t) tm * S::TM;
    if (tr.n <= 0) return;
    // with K in shares, each writes sums of its own
    Y * y = (Y *) a.y + (int64_t) blockIdx.y * a.T * a.M;
    if (IDS && tr.expert < 0) {   // pairs that no expert takes
        const int64_t cols = min((int64_t) S::TM, a.M - m0);
        for (int64_t i = threadIdx.x; i < S::TM * tr.n; i += 64 * S::NW)
            if (i % S::TM < cols) y[(tr.first + i / S::TM) * a.M + m0 + i % S::TM] = from_f32<Y>(0.0f);
        return;
    }

    // this wave's copies: rows of the weights first, then of x
    constexpr int CK = S::CI / S::NW, COPIES = CK + S::SI / S::NW;
    const uint8_t * code_row[CK];
    const uint8_t * exp_row[COPIES - CK];
    int64_t exp_step[COPIES - CK];
    const uint8_t * wc = a.w_codes + tr.expert * a.w_codes_stride;
    const uint8_t * ws = a.w_scales + tr.expert * a.w_scales_stride;
    auto source = [&](int r) {
        return r < S::TM ? min(m0 + r, a.M - 1) : x_row<IDS>(a, tr.first + min((int64_t) r - S::TM, tr.n - 1));
    };
#pragma unroll
    for (int k = 0; k < CK; ++k) {
        const int r = (wave + k * S::NW) * 8 + (lane >> 3);
        code_row[k] = (r < S::TM ? wc : a.x_codes) + source(r) * a.KB * 16;
    }
#pragma unroll
    for (int k = 0; k < COPIES - CK; ++k) {
        const int r = (wave + k * S::NW) * 32 + (lane >> 1);
        exp_row[k] = (r < S::TM ? ws : a.x_scales) + source(r) * 8 + (lane & 1) * 4;
        exp_step[k] = (r < S::TM ? a.M : a.x_rows) * 8;
    }
    const unsigned lds0 = (unsigned) (uintptr_t) (lds_char *) lds;
    // the block that this lane copies: its rows are 8 (wave + k NW) + lane / 8, NW even
    const int blk = (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4));
    const int planes = (a.KB + 7) / 8, share = (planes + gridDim.y - 1) / gridDim.y, first = blockIdx.y * share;
    const int last = min(share, planes - first) - 1;   // this workgroup's planes, from `first` on
    // copy c of plane h into its place in the ring; past the last plane that one comes again, into a
    // place that nothing reads any more, so that the number of copies on their way is always known
    auto copy = [&](int h, auto cc) {
        constexpr int c = cc;
        const unsigned to = lds0 + h % STAGES * S::STAGE;
        const int p = first + min(h, last);
        if constexpr (c < CK) dma16(code_row[c] + (int64_t) min(p * 8 + blk, a.KB - 1) * 16, to + (wave + c * S::NW) * 1024);
        else dma4(exp_row[c - CK] + p * exp_step[c - CK], to + S::CODES + (wave + (c - CK) * S::NW) * 256);
    };

    const int wm = wave % WM * 32 * FM, wn = S::TM + wave / WM * 32 * FN;
    const int r31 = lane & 31, half = lane >> 5;
    const char * ca = lds + (wm + r31) * 128, * cb = lds + (wn + r31) * 128;
    const char * ea = lds + S::CODES + (wm + r31) * 8 + half * 4, * eb = lds + S::CODES + (wn + r31) * 8 + half * 4;
    int slot[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) slot[j] = ((j + 4 * half) ^ (r31 >> 1 & 7)) * 16;
    int sa[FM], sb[FN], na[FM], nb[FN];
    auto load_exps = [&](int at) {
#pragma unroll
        for (int i = 0; i < FM; ++i) na[i] = *(const int *) (ea + at + i * 32 * 8);
#pragma unroll
        for (int i = 0; i < FN; ++i) nb[i] = *(const int *) (eb + at + i * 32 * 8);
    };
    auto take_exps = [&](int h) {   // this lane's four blocks', 0 past K
        const int left = min(max(a.KB - (first + h) * 8 - 4 * half, 0), 4);
        const int mask = left == 4 ? ~0 : (1 << (8 * left)) - 1;
#pragma unroll
        for (int i = 0; i < FM; ++i) sa[i] = na[i] & mask;
#pragma unroll
        for (int i = 0; i < FN; ++i) sb[i] = nb[i] & mask;
    };

    // A step's fragments are read between the instructions of the one before.  Before a plane's last
    // step all waves have read its place and the next plane has come: the barrier stands there.  Then
    // the next plane's first fragments are read, and plane h + STAGES is copied to the free place
    // during this step (part 0) and the next plane's first two (parts 1 and 2), spread over their
    // instructions: all at once they would hold up the wave that issues them.
    constexpr int INS = FM * FN, FR = FM + FN, PER = (FR + INS - 1) / INS, EVERY = INS / FR > 0 ? INS / FR : 1;
    constexpr int AHEAD = (STAGES - 2) * COPIES;   // copies of later planes on their way at the barrier
    v16f acc[FM][FN] = {};
    frags<FM, FN> f0, f1;
    auto reads = [&](frags<FM, FN> & f, int at, int j, auto i) {
        if constexpr (i % EVERY == 0)
            unroll<PER>([&](auto k) {
                constexpr int n = i / EVERY * PER + k;
                if constexpr (n < FR) f.template load<n>(ca + at + slot[j], cb + at + slot[j]);
            });
    };
    auto copies = [&](int h, auto part, auto i) {   // those in front of instruction i of part's step
        unroll<COPIES>([&](auto c) {
            if constexpr ((c * 2 + 1) * 3 * INS / (2 * COPIES) == part * INS + i) copy(h, c);
        });
    };
    constexpr std::integral_constant<int, 0> P0{};
    constexpr std::integral_constant<int, 1> P1{};
    constexpr std::integral_constant<int, 2> P2{};
    for (int h = 0; h < STAGES - 1; ++h) unroll<COPIES>([&](auto c) { copy(h, c); });
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(AHEAD) : "memory");
    unroll<INS>([&](auto i) { copies(STAGES - 1, P0, i); });
    // a wave whose part of the tile lies past M or the tile's rows only copies: its results are not
    // stored, and the others have the matrix cores to themselves
    if (m0 + wm >= a.M || wn - S::TM >= tr.n) {
        for (int h = 0; h < last; ++h) {
            unroll<INS>([&](auto i) { copies(h + STAGES - 1, P1, i); });
            unroll<INS>([&](auto i) { copies(h + STAGES - 1, P2, i); });
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(AHEAD) : "memory");
            unroll<INS>([&](auto i) { copies(h + STAGES, P0, i); });
        }
    } else {
        unroll<FR>([&](auto i) { f0.template load<i>(ca + slot[0], cb + slot[0]); });
        load_exps(0);
        take_exps(0);
        int at = 0;
        for (int h = 0; h < last; ++h) {
            mma_step<0>(acc, f0, sa, sb, [&](auto i) { reads(f1, at, 1, i); copies(h + STAGES - 1, P1, i); });
            mma_step<1>(acc, f1, sa, sb, [&](auto i) { reads(f0, at, 2, i); copies(h + STAGES - 1, P2, i); });
            mma_step<2>(acc, f0, sa, sb, [&](auto i) { reads(f1, at, 3, i); });
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(AHEAD) : "memory");
            at = at + S::STAGE == S::LDS ? 0 : at + S::STAGE;
            load_exps(at);
            mma_step<3>(acc, f1, sa, sb, [&](auto i) { reads(f0, at, 0, i); copies(h + STAGES, P0, i); });
            take_exps(h + 1);
        }
        mma_step<0>(acc, f0, sa, sb, [&](auto i) { reads(f1, at, 1, i); });
        mma_step<1>(acc, f1, sa, sb, [&](auto i) { reads(f0, at, 2, i); });
        mma_step<2>(acc, f0, sa, sb, [&](auto i) { reads(f1, at, 3, i); });
        mma_step<3>(acc, f1, sa, sb, [](auto) {});
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no copy is left when the shared memory gets another use

    // The results go out through shared memory: straight from the registers a store would touch 32 x
    // rows with 16 bytes each.  Rows of TM outputs lie 16 B past a multiple of the 64 banks apart, so
    // that 16 x rows times four neighbouring outputs cover them.
    constexpr int ROW = S::TM * (int) sizeof(Y) + 16;
    constexpr int PASSES = (S::TN * ROW + S::LDS - 1) / S::LDS, PT = S::TN / PASSES;
    static_assert(PT % 32 == 0 && PT * ROW <= S::LDS, "whole fragments in a pass");
    const int cols = (int) min((int64_t) S::TM, a.M - m0);
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
                    char * to = lds + (t + r31) * ROW + (wm + m * 32 + 2 * i + 4 * half) * (int) sizeof(Y);
                    __builtin_memcpy(__builtin_assume_aligned(to, sizeof(q)), &q, sizeof(q));
                }
        }
        __syncthreads();
        const int rows = (int) min((int64_t) PT, tr.n - pass * PT);
        constexpr int V = 16 / sizeof(Y), PER = S::TM / V;
        for (int i = threadIdx.x; i < rows * PER; i += 64 * S::NW) {
            const int c = i % PER * V;
            if (c >= cols) continue;
            pack<Y, V> q;
            __builtin_memcpy(&q, __builtin_assume_aligned(lds + i / PER * ROW + i % PER * 16, 16), 16);
            Y * to = out + (int64_t) (pass * PT + i / PER) * a.M + c;
            if (c + V <= cols) put<false>(to, q);
            else
                for (int k = 0; k < V; ++k)
                    if (c + k < cols) to[k] = q.v[k];
        }
    }
}

// y = the shares' sums, one after the other
template <class Y> static __global__ void __launch_bounds__(256) k_mx4_join(const float * __restrict__ part, int64_t n, int shares, Y * __restrict__ y) {
    const int64_t i = ((int64_t) blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
    if (i + 4 <= n) {
        float s[4] = {};
#pragma unroll 4
        for (int k = 0; k < shares; ++k) {
            const pack<float, 4> v = get<float, 4>(part + k * n + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += v.v[j];
        }
        for (int j = 0; j < 4; ++j) y[i + j] = from_f32<Y>(s[j]);
    } else {
        for (int64_t j = i; j < n; ++j) {
            float s = 0.0f;
            for (int k = 0; k < shares; ++k) s += part[k * n + j];
            y[j] = from_f32<Y>(s);
        }
    }
}

template <int FM, int FN, int WM, int WN, int STAGES, bool IDS>
static hipError_t run_tile(const mx4_args & a, int shares, float * part, int ytype, hipStream_t st) {
    using S = tile_shape<FM, FN, WM, WN, STAGES>;
    const int64_t tm = (a.M + S::TM - 1) / S::TM, tn = IDS ? id_tiles(a, S::TN) : (a.T + S::TN - 1) / S::TN;
    if (tm * tn >> 32) return hipErrorInvalidConfiguration;   // no card holds these results
    const dim3 grid = row_groups(tm * tn, shares, S::NW);
    auto go = [&](auto t, const mx4_args & a) {
        return launch(k_mx4_tile<FM, FN, WM, WN, STAGES, decltype(t), IDS>, grid, 64 * S::NW, S::LDS, st, a, (unsigned) tm, (unsigned) tn);
    };
    if (shares == 1) return with_type(ytype, [&](auto t) { return go(t, a); });
    mx4_args to_part = a;
    to_part.y = part;
    const hipError_t e = go(float{}, to_part);
    if (e != hipSuccess) return e;
    const int64_t n = a.T * a.M;
    return with_type(ytype, [&](auto t) {
        using Y = decltype(t);
        return launch(k_mx4_join<Y>, (unsigned) ((n + 1023) / 1024), 256, 0, st, part, n, shares, (Y *) a.y);
    });
}

int64_t mx4_tile_workspace(const mx4_args & a) {
    const tile_choice c = pick_tile(a);
    return c.shares > 1 ? c.shares * a.T * a.M * (int64_t) sizeof(float) : 0;
}

template <bool IDS> static hipError_t product_tile(const mx4_args & a, float * part, int ytype, hipStream_t st) {
    const tile_choice c = pick_tile(a);
    if (c.side == 256) return run_tile<4, 2, 2, 4, 2, IDS>(a, c.shares, part, ytype, st);
    if (c.side == 128 && c.stages == 4) return run_tile<2, 2, 2, 2, 4, IDS>(a, c.shares, part, ytype, st);
    if (c.side == 128) return run_tile<2, 2, 2, 2, 2, IDS>(a, c.shares, part, ytype, st);
    return run_tile<1, 2, 2, 1, IDS ? 2 : 4, IDS>(a, c.shares, part, ytype, st);
}

hipError_t mx4_product_tile(const mx4_args & a, float * part, int ytype, hipStream_t st) {
    return a.n_expert ? product_tile<true>(a, part, ytype, st) : product_tile<false>(a, part, ytype, st);
}

}  // namespace mi355x_ops
