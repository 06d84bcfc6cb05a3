// mx4_rules.h — which kernel an MXFP4 product takes: the rules on its sizes, without HIP, so that a test
// on the host sees their choice.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace mi355x_ops {

struct product_size {
    int64_t M;      // rows of the weights
    int KB;         // K / 32
    int64_t T;      // rows of y
    int n_expert;   // 0: dense
};

// tiles of `rows` rows that hold n, which may be close to 2^31
constexpr int tiles_of(int n, int rows) { return n / rows + (n % rows > 0); }

// ---- few rows (k_mx4.hip) --------------------------------------------------------------------
constexpr int MV_WAVES = 8;              // of a workgroup
constexpr int64_t MV_LDS = 144 * 1024;   // most shared memory of a workgroup, of a CU's 160 KiB

// bytes of an x row in shared memory: codes and exponents, an odd number of 16-B columns, so that the
// same column of 16 rows lies in 16 different ones of the banks
constexpr int mv_row_bytes(int KB) { return ((KB + (KB + 15) / 16) | 1) * 16; }

// NT tiles of 16 x rows, and sums to join where KS waves share a group
inline int64_t mv_lds(const product_size & a, int NT, int KS) {
    return mv_row_bytes(a.KB) * (a.T < 16 * NT ? a.T : 16 * NT) + (KS > 1 ? MV_WAVES * 1024 : 0);
}

// tiles of 16 NT x rows to reckon with: by experts as many as an even routing fills
inline int64_t mv_busy(const product_size & a, int NT) {
    return a.n_expert ? std::min(a.T, (int64_t) a.n_expert) : (a.T + 16 * NT - 1) / (16 * NT);
}

// Workgroups in all: three for a CU.  With 256 / 512 / 768 / 1024 / 1536, 28672 x 4096 by one row takes 16.1 / 14.5 /
// 14.5 / 14.5 / 14.5 us, 32001 x 4096 by 29 rows 23.1 / 21.4 / 21.3 / 21.6 / 21.4, 800 pairs by 128 experts of
// 1408 x 2048 66 / 54 / 51 / 58 / 46.
constexpr int64_t MV_GROUPS = 768;

// how many waves share a group of 16 weight rows: as few as give the tiles MV_FILL waves in all.  With
// 1024 / 2048 / 4096 / 8192, 4096 x 14336 by one row takes 13.5 / 10.9 / 10.8 / 10.8 us, by 16 rows (quantised
// before) 18.9 / 16.3 / 16.2 / 16.3, 32001 x 4096 by 29 rows 21.5 / 21.3 / 26.9 / 27.7.
constexpr int64_t MV_FILL = 2048;
inline int mv_split(const product_size & a, int NT) {
    const int64_t groups = (a.M + 15) / 16 * mv_busy(a, NT);
    int ks = 1;
    while (ks < MV_WAVES && groups * ks < MV_FILL && a.KB > 8 * ks) ks *= 2;
    return ks;
}

// The kernel for few rows: up to 32, by experts up to 16 each on average.  4096 x 4096 by 20 and 32 rows takes 6.1
// and 6.5 us here, 8.0 and 9.1 in the tiles below; 28672 x 4096 by 33 and 64 rows 25 and 26, there 16 and 17; 256 pairs
// by 256 experts of 1408 x 2048, evenly, 49 and 54.  It is not always the faster one: 28672 x 4096 by 32 rows 18.0
// and 15.8, 4096 x 14336 by 17 and 32 rows (the 32 in two tiles, each of which reads the weights) 15.3 and 15.8,
// there 12.7 and 12.2.  Nor does it look at the routing, which is on the device: those 256 pairs all on one expert take 25
// and 12, 2048 pairs by 128 experts 60 and 44 evenly, 56 and 41 with nine in ten on eight of them.
inline bool few_rows(const product_size & a) {
    return a.T <= (a.n_expert ? 16 * (int64_t) a.n_expert : 32) && mv_lds(a, 1, MV_WAVES) <= MV_LDS;
}

// Few enough that every workgroup may quantise those of its tile, which saves a launch.  4096 x 14336 by 1 / 2 / 3 /
// 4 / 8 float32 rows 10.9 / 12.2 / 13.6 / 14.8 / 20.7 us so, 13.3 / 13.6 / 13.8 / 13.9 / 14.1 with a launch for them;
// 28672 x 4096 by bf16 rows 14.6 / 15.9 / 16.0 / 16.2 / 18.2 and 17.4 / 17.3 / 17.3 / 17.4 / 17.7.  By experts a
// workgroup has only its own expert's: 16 pairs by 8 experts of 28672 x 4096 87 and 89, 12 by 64 of 1408 x 2048 9.2
// and 11.2, 48 of the latter 15.7 and 18.0.
inline bool float_rows(const product_size & a) { return few_rows(a) && a.T <= (a.n_expert ? 16 : 2); }

// how many tiles of 16 x rows a workgroup keeps: two where they fit (32 up to K = 8160), so that the weights are read once
inline int mv_tiles(const product_size & a) { return !a.n_expert && a.T > 16 && mv_lds(a, 2, MV_WAVES) <= MV_LDS ? 2 : 1; }

// ---- tiles (k_mx4_gemm.hip) ------------------------------------------------------------------
// Which tile: the one whose time, by what a CU was measured to take (us), comes out least.  A plane
// (256 of K) takes 2.1 in a 256 x 256 tile, 0.65 in a 128 x 128 tile alone on its CU and 0.8 in one of
// several, 0.33 and 0.26 in 64 x 64 tiles; beginning and end add 8, 4 and 4.  Tiles come in whole rounds
// of the CUs; experts' are counted as half full at their ends, a quarter of a tile each, since waves
// without rows cost little, and the routing's rounds as half one more.  Large tiles move the least
// bytes for their products, small ones give more CUs work: 512 x 28672 x 4096 takes 41 us in tiles of
// 256, 54 in tiles of 128 and 83 in tiles of 64, 1024 x 4096 x 4096 27, 15 and 25, 256 x 4096 x 4096 26, 12.5 and 10;
// 8192 pairs by 8 experts of 4096 x 14336 297, 333 and 509.
// Deep rings serve CUs that have one tile (1024 x 4096 x 4096 in tiles of 128: 15.0 us with four planes, 16.6
// with two), shallow ones let several share a CU (2048 x 4096 x 4096: 27.5 and 24.7; in tiles of 64, 600 pairs
// by 8 experts of 4096 x 4096 31 and 28, but 200 by 4 experts 12 and 17.5; dense 256 x 4096 x 14336 24 and 46).
// A long K over few tiles is cut into shares whose sums a second kernel joins: 128 x 4096 x 14336 23 us whole and
// 18 so, 64 x 4096 x 14336 23 and 13, 100 x 640 x 14336 22 and 10.
struct tile_choice {
    int side, stages, shares;
};

inline tile_choice pick_tile(const product_size & a) {
    const bool ids = a.n_expert != 0;
    constexpr double CUS = 256;
    const int planes = (a.KB + 7) / 8;
    auto rounds = [&](double n) { return ids ? std::max(n + 0.5, 1.0) : std::ceil(n); };
    tile_choice best = {};
    double least = 0;
    for (const int side : {256, 128, 64}) {
        const int64_t busy = std::min(a.T, (int64_t) a.n_expert);
        const double cols = ids ? (double) a.T / side + 0.25 * busy : (double) ((a.T + side - 1) / side);
        const double tiles = cols * ((a.M + side - 1) / side) / CUS;   // for each CU
        for (int shares = 1; shares <= 16 && (shares == 1 || planes >= 2 * shares); shares *= 2) {
            const double n = tiles * shares, p = (planes + shares - 1) / shares;
            double t;
            if (side == 256) t = rounds(n) * (p * 2.1 + 8);
            else if (side == 128) t = n <= 1 ? rounds(n) * (p * 0.65 + 4) : rounds(n) * p * 0.8 + rounds(n / 2) * 4;
            else t = n <= 1 ? rounds(n) * (p * 0.33 + 4) : rounds(n) * p * 0.26 + rounds(n / 4) * 4;
            // the join: a launch, and the sums written and read
            if (shares > 1) t += 3 + (double) shares * a.T * a.M * 8 / 4e6;
            if (least == 0 || t < least) {
                least = t;
                best = {side, side == 256 ? 2 : side == 128 ? (n <= 1 ? 4 : 2) : (ids ? 2 : 4), shares};
            }
        }
    }
    // every share has planes of its own
    while (best.shares > 1 && (planes + best.shares - 1) / best.shares * (best.shares - 1) >= planes) best.shares /= 2;
    return best;
}

}  // namespace mi355x_ops
