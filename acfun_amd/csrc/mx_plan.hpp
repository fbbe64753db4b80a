// mx_plan.hpp -- the sizes of MXFP4 operands, and which kernel, tile and number of
// launches a product or a layer takes; independent of HIP so that it can be
// exercised on the host.
#pragma once
#include <cstddef>

namespace acfun {

constexpr long long mx_row_tiles(int rows) { return ((long long)rows + 15) / 16; }
constexpr int mx_k_tiles(int K) { return (int)(((long long)K + 127) / 128); }
constexpr int mx_scale_tiles(int K) { return (int)(((long long)K + 511) / 512); }
constexpr size_t mx_code_bytes(int rows, int K) { return (size_t)mx_row_tiles(rows) * mx_k_tiles(K) * 1024; }
constexpr size_t mx_scale_bytes(int rows, int K) { return (size_t)mx_row_tiles(rows) * mx_scale_tiles(K) * 256; }

// A launch has fewer than 2^32 threads.
constexpr bool launch_fits(long long groups, int threads) { return groups < (1ll << 32) / threads; }

// ---------------------------------------------------------------- quantizer
constexpr int kMxThreads = 256;
constexpr long long mx_quant_groups(int rows, int K, int trans) {
    return (trans ? ((long long)rows + 63) / 64 * 4 : mx_row_tiles(rows)) * mx_scale_tiles(K);
}
constexpr bool mx_quant_fits(int rows, int K, int trans) {
    return launch_fits(mx_quant_groups(rows, K, trans), kMxThreads);
}

// ---------------------------------------------------------------- products
enum MmKind { FEW16, FEW32, FEW64, MANY128, MANY256, KINDS };
constexpr struct { int edge, threads; } kMmTile[KINDS] = {{16, 512}, {32, 256}, {64, 512}, {128, 256}, {256, 256}};

constexpr long long mm_tiles(int M, int N, int edge) {
    return (((long long)M + edge - 1) / edge) * (((long long)N + edge - 1) / edge);
}
// Workgroups of `tiles`: the same number for each of 8 XCDs.
constexpr long long xcd_groups(long long tiles) { return (tiles + 7) / 8 * 8; }

// Whether a product can run on a kind: its launch fits, and MANY's 32-bit offsets
// into a tile's operands reach.
constexpr bool mm_fits(int M, int N, int K, int kind) {
    return launch_fits(xcd_groups(mm_tiles(M, N, kMmTile[kind].edge)), kMmTile[kind].threads) &&
           (kind < MANY128 || (K > 0 && K <= (1 << 22)));
}
constexpr bool mm_fits(int M, int N, int K) {
    for (int i = 0; i < KINDS; ++i)
        if (mm_fits(M, N, K, i)) return true;
    return false;
}

// Times in us that choose a kernel and its tile, fitted to those of every tile over
// 300 sizes (bf16, replayed from a graph): a call takes `lat` while the CUs have less
// than a tile each, and `base` and `each` times the tiles of a CU from there.  Over 360
// sizes (M of 16 to 8192, N of 64 to 8192, K of 128 to 8192, three sets of operands in
// turn) the tile chosen is 0.8 % slower than the best of each in the mean, 25 % at most
// (64 x 2048 x 8192: 7.2 with tiles of 32, 5.7 with 16).  Measured, us: 128 x 8192 x 4096
// 10.0 with tiles of 32, 8.6 with 64, 11.1 with 128; 512 x 8192 x 1024 14.6 with 64, 6.8
// with 128; 8192 x 8192 x 4096 154 with 128, 132 with 256.
inline double tile_time(double lat, double base, double each, double tiles_per_cu) {
    const double t = base + each * tiles_per_cu;
    return t > lat ? t : lat;
}
constexpr double kNever = 1e30;

// The fastest kernel that a product fits, and its time; kNever if it fits none.
inline MmKind mm_choose(int M, int N, int K, double cus, double& us) {
    const double k = K;
    auto per_cu = [&](int b) { return (double)mm_tiles(M, N, b) / cus; };
    auto more = [](double a, double b) { return a > b ? a : b; };
    const double t[KINDS] = {
        tile_time(2.72 + 0.89e-4 * k, 2.18 + 0.64e-4 * k, more(0.42 + 1.12e-4 * k, 2.42e-4 * k), per_cu(16)),
        tile_time(2.73, 2.73 + 2.7e-4 * k, more(0.247 + 1.74e-4 * k, 3.8e-4 * k), per_cu(32)),
        tile_time(3.57 + 6.6e-4 * k, 1.91 + 2.65e-4 * k, 2.3 + 8.2e-4 * k, per_cu(64)),
        tile_time(3.87 + 17.6e-4 * k, 3.88 + 2.9e-4 * k, 1.39 + 18.8e-4 * k, per_cu(128)),
        tile_time(7.28 + 43.5e-4 * k, 4.37 + 1.6e-4 * k, 7.32 + 63.7e-4 * k, per_cu(256)),
    };
    int best = FEW16;
    us = kNever;
    for (int i = 0; i < KINDS; ++i)
        if (mm_fits(M, N, K, i) && t[i] < us) us = t[i], best = i;
    return (MmKind)best;
}

// ---------------------------------------------------------------- layers
// The LDS of k_mxmm_few: the partial sums of W waves, and quantized rows, for which
// there is room for 1, 2, 4, 8 or 16.
constexpr size_t kLds = 160 * 1024;
template <int TM, int TN, int W>
constexpr size_t kFewSums = (size_t)W * TM * TN * 68 * 16;
constexpr int few_rows(int M) { return M > 8 ? 16 : M > 4 ? 8 : M > 2 ? 4 : M; }
constexpr size_t few_rows_lds(int M, int K) { return (size_t)few_rows(M) * mx_scale_tiles(K) * (256 + 16); }

// A layer whose workgroups each quantize their 16 rows for tn tiles of 16 columns:
// whether LDS has room for the rows and the launch fits.
constexpr int kRowsWaves = 8;
constexpr long long rows_groups(int M, int N, int tn) {
    return xcd_groups(mx_row_tiles(M) * ((mx_row_tiles(N) + tn - 1) / tn));
}
constexpr bool rows_fits(int M, int N, int K, int tn) {
    return kFewSums<1, 1, kRowsWaves> * tn + few_rows_lds(M, K) <= kLds &&
           launch_fits(rows_groups(M, N, tn), 64 * kRowsWaves);
}
// Its time: `pieces` of a row and 512 k fall to each wave.
inline double rows_time(int M, int N, int K, double cus, int tn) {
    if (!rows_fits(M, N, K, tn)) return kNever;
    const double k = K, pieces = (double)(((M < 16 ? M : 16) * (long long)mx_scale_tiles(K) + 7) / 8);
    const double per_cu = (double)mx_row_tiles(M) * (double)((mx_row_tiles(N) + tn - 1) / tn) / cus;
    return tile_time(3.05 + 0.037 * tn + (0.94e-4 * tn - 0.77e-4) * k + 0.167 * pieces, 2.4 + 0.13 * pieces,
                     0.42 + 0.132 * tn + (1.32e-4 + 0.78e-4 * tn) * k + 0.074 * pieces, per_cu);
}
constexpr bool fc_fits(int M, int N, int K) {
    return (mx_quant_fits(M, K, 0) && mm_fits(M, N, K)) ||
           (K > 0 && (rows_fits(M, N, K, 1) || rows_fits(M, N, K, 2) || rows_fits(M, N, K, 4)));
}

// The rows up to which a layer is always one launch while its stream is captured into a
// graph, where LDS has room for 16 of them: two launches need a temporary, which a graph
// cannot keep, and programs that capture have to know beforehand what they may.  Measured
// in a graph, us, against two calls on the caller's buffers: 16 x 4096 x 4096 5.8 and 5.1,
// 128 x 4096 x 4096 10.0 and 8.9, 512 x 4096 x 4096 34 and 15, 512 x 8192 x 8192 196 and 27.
constexpr int kCapturedRows = 512;

struct FcPlan {
    int tn;                         // tiles of a workgroup that quantizes its rows; 0: LDS has no room for them
    bool one;                       // one launch of those is faster than two
    bool captured;                  // one launch is taken on a captured stream
};
// One launch, in which every workgroup quantizes its 16 rows, or two, of which the
// first takes 2.45 us and its traffic at 4.5 TB/s?  Measured, us: 16 x 2048 x 2048 4.4
// and 5.0, 16 x 2048 x 8192 9.0 and 6.1; 128 x 2048 x 1024 4.3 and 5.7, 333 x 2048 x
// 2048 10.1 and 8.2.
inline FcPlan fc_plan(int M, int N, int K, size_t elem, double cus) {
    double two, one = kNever;
    (void)mm_choose(M, N, K, cus, two);
    two = mx_quant_fits(M, K, 0) ? two + 2.45 + (double)M * K * (elem + 0.53) * 0.22e-6 : kNever;
    int tn = 0;
    for (int n = 1; n <= 4; n *= 2)
        if (const double t = rows_time(M, N, K, cus, n); t < one) one = t, tn = n;
    return {tn, one < two, one < two || (tn && M <= kCapturedRows)};
}

}  // namespace acfun
