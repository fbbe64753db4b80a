// q8_plan.hpp -- the sizes of Q8 operands, and which kernel, tile and number of
// launches a product or a layer takes; independent of HIP so that it can be
// exercised on the host.
#pragma once
#include "mx_plan.hpp"

namespace acfun {

constexpr long long q8_row_tiles(int rows) { return ((long long)rows + 15) / 16; }
constexpr int q8_k_tiles(int K) { return (int)(((long long)K + 63) / 64); }
constexpr size_t q8_code_bytes(int rows, int K) { return (size_t)q8_row_tiles(rows) * q8_k_tiles(K) * 1024; }
constexpr size_t q8_scale_bytes(int rows) { return (size_t)q8_row_tiles(rows) * 64; }

// A sum of K products of two codes, at most 127^2 each, is exact in 32 bits.
constexpr int kQ8MaxK = 131072;
static_assert(127ll * 127 * kQ8MaxK < (1ll << 31), "sums in 32 bits");

// ---------------------------------------------------------------- quantizer
// Rows along K: 8 waves to R rows, a wave 1024 / R k of each at once.
constexpr int kQ8RowThreads = 512;
constexpr long long q8_row_groups(int rows, int R) { return q8_row_tiles(rows) * (16 / R); }
// Two rows while a CU has one workgroup of them at most, four past that.  Measured, us, bf16,
// K of 4096: 16 rows 2.8 and 3.9 with four (8.7 with 16), 512 rows 3.6 and 4.4, 1024
// rows 5.8 and 4.9, 4096 rows 12.8 and 10.8 (15.1 with 16); the kernel's turns without values, of
// which two rows have twice as many, are in these.
constexpr int q8_rows_of(int rows, int cus) { return rows <= 2 * cus ? 2 : 4; }
// The steps that a wave keeps in LDS: a power of two, 64 KB at most.
constexpr int q8_row_steps(int K, int R, size_t elem) {
    const int steps = ((4 * q8_k_tiles(K) + 64 / R - 1) / (64 / R) + 7) / 8, most = elem == 4 ? 2 : 4;
    int n = 1;
    while (n < steps && n < most) n *= 2;
    return n;
}
// Rows across K: 64 bytes of rows to a workgroup.  Measured, us, fp32 [4096][8192]: 52 with
// 64 bytes and 1024 threads, 59 with 32 and 512; 72 with 32 and 1024, whose registers spill.
constexpr int kQ8ColThreads = 1024;
template <size_t elem>
constexpr int kQ8Cols = elem == 4 ? 16 : 32;
constexpr long long q8_col_groups(int rows, size_t elem) {
    return (q8_row_tiles(rows) * 16 * (long long)elem + 63) / 64;
}
// Back: 4 waves, each with some tiles.
constexpr int kQ8Threads = 256, kQ8BackTiles = 2;
constexpr long long q8_dequant_groups(int rows, int K) {
    return (q8_row_tiles(rows) * q8_k_tiles(K) + 4 * kQ8BackTiles - 1) / (4 * kQ8BackTiles);
}
constexpr bool q8_quant_fits(int rows, int trans) {
    return trans ? launch_fits(xcd_groups(q8_col_groups(rows, 4)), kQ8ColThreads)
                 : launch_fits(q8_row_groups(rows, 4), kQ8RowThreads);
}
constexpr bool q8_dequant_fits(int rows, int K) { return launch_fits(q8_dequant_groups(rows, K), kQ8Threads); }

// ---------------------------------------------------------------- products
// Tiles of rows x columns of C; with two projections (gated) all but the smallest have
// half the columns, of each.
enum Q8Kind { Q8_FEW16, Q8_FEW32, Q8_FEW64, Q8_MANY128, Q8_MANY256, Q8_KINDS };
constexpr struct { int edge, threads; } kQ8Tile[Q8_KINDS] = {{16, 512}, {32, 256}, {64, 512}, {128, 256}, {256, 256}};
constexpr int q8_columns(int kind, bool gated) { return kQ8Tile[kind].edge / (gated && kind != Q8_FEW16 ? 2 : 1); }
constexpr long long q8_tiles(int M, int N, int kind, bool gated) {
    const int e = kQ8Tile[kind].edge, c = q8_columns(kind, gated);
    return (((long long)M + e - 1) / e) * (((long long)N + c - 1) / c);
}
constexpr bool q8_mm_fits(int M, int N, int K, int kind, bool gated) {
    return launch_fits(xcd_groups(q8_tiles(M, N, kind, gated)), kQ8Tile[kind].threads) && (kind < Q8_MANY128 || K > 0);
}
constexpr bool q8_mm_fits(int M, int N, int K, bool gated) {
    for (int i = 0; i < Q8_KINDS; ++i)
        if (q8_mm_fits(M, N, K, i, gated)) return true;
    return false;
}

// Times in us that choose a tile, fitted to those of every tile over 220 sizes (bf16, from
// a graph, three sets of operands in turn): a call takes lat while the CUs have less than
// a tile each, base and each times the tiles of a CU from there, in whole turns up to four
// where a CU has room for one tile; all three grow with K.  The tile chosen is 0.5 % slower than
// the best in the mean, 21 % at most (19 x 1728 x 4608 gated: 5.9 with tiles of 16,
// 7.2 with 32).  Measured, us: 59 x 8128 x 4416 13.8, 9.4 and 10.9 with tiles of 16, 32
// and 64; 4877 x 2304 x 5888 158, 75 and 69 with 64, 128 and 256.
struct Q8Fit { double lat, lat_k, base, base_k, each, each_k; bool turns; };
constexpr Q8Fit kQ8Fit[2][Q8_KINDS] = {
    {{2.441, 1.549e-4, 2.059, 2.321e-4, 0.353, 2.682e-4, false},
     {2.391, 4.580e-4, 2.086, 4.557e-4, 0.279, 7.361e-4, false},
     {3.125, 10.39e-4, 1.870, 8.392e-4, 2.724, 14.00e-4, true},
     {3.756, 26.30e-4, 3.178, 19.59e-4, 2.176, 35.10e-4, false},
     {7.311, 74.40e-4, 7.970, 47.43e-4, 5.462, 99.93e-4, true}},
    {{2.722, 2.758e-4, 2.013, 4.313e-4, 0.610, 3.939e-4, false},
     {2.656, 4.436e-4, 2.450, 4.657e-4, 0.238, 5.718e-4, false},
     {3.490, 8.139e-4, 1.144, 10.28e-4, 2.576, 13.69e-4, true},
     {3.822, 27.28e-4, 3.804, 12.32e-4, 1.650, 39.17e-4, false},
     {6.317, 80.47e-4, 8.421, 28.47e-4, 5.272, 96.93e-4, true}}};
inline double q8_time(int M, int N, int K, int kind, bool gated, double cus) {
    const Q8Fit& f = kQ8Fit[gated][kind];
    double t = (double)q8_tiles(M, N, kind, gated) / cus;
    if (f.turns && t > 1 && t < 4) t = (double)(int)(t + 0.98);
    return tile_time(f.lat + f.lat_k * K, f.base + f.base_k * K, f.each + f.each_k * K, t);
}
// The fastest tile of those whose launch holds the product.
inline Q8Kind q8_choose(int M, int N, int K, bool gated, double cus) {
    int best = Q8_FEW16;
    double us = kNever;
    for (int i = 0; i < Q8_KINDS; ++i)
        if (q8_mm_fits(M, N, K, i, gated))
            if (const double t = q8_time(M, N, K, i, gated, cus); t < us) us = t, best = i;
    return (Q8Kind)best;
}

// ---------------------------------------------------------------- layers
// LDS of k_q8mm_few: the partial sums of its waves for each projection, and quantized rows,
// for which there is room for 1, 2, 4, 8 or 16, with their maxima and scales.
constexpr size_t q8_few_sums(int tm, int tn, int waves, int mats) { return (size_t)waves * tm * tn * mats * 68 * 16; }
constexpr size_t q8_rows_lds(int M, int K) { return (size_t)few_rows(M) * q8_k_tiles(K) * 64 + 192; }
// One launch, in which every workgroup quantizes its 16 rows: whether LDS has room.
constexpr bool q8_rows_fit(int M, int N, int K, bool gated) {
    return q8_few_sums(1, 1, 8, gated ? 2 : 1) + q8_rows_lds(M, K) <= kLds && q8_mm_fits(M, N, K, Q8_FEW16, gated);
}
// It is taken up to two pieces of a row and 512 k for each of its 8 waves, which take 0.6
// us and 0.8 for each; a launch of the quantizer takes 2.8, its turns without values among
// them.  Measured, us, K and N of 4096, in one and in two: 1 row 6.6 and 8.1, 2 rows 7.4 and
// 8.1, 4 rows 8.7 and 8.1, 16 rows 19 and 8.2.
constexpr bool q8_rows_one(int M, int K) { return M <= 16 && M * (((long long)K + 511) / 512) <= 16; }

// ---------------------------------------------------------------- sampling
// A workgroup of `threads` to a row, or `parts` of 1024 with `per` columns each (whole
// 1024s, which are two waves' loads).
constexpr int kSampleMaxCols = 1 << 24, kSampleParts = 32;
// A row's sum of weights is below 2^63 in steps of 2^-f.  With f for the most that `cols` weights can
// have, half a step for each is 2^-25 of the largest weight up to this many; wider rows have f for what
// theirs have.
constexpr int kSampleFrac = 48, kSampleEven = 1 << 19;
constexpr int sample_frac(int cols) {
    int bits = 0;
    while ((1 << bits) < cols) ++bits;
    return 62 - bits < kSampleFrac ? 62 - bits : kSampleFrac;
}
constexpr bool sample_fits(int rows) { return launch_fits(rows, 1024); }
struct SamplePlan { int parts, per, threads; };
// Parts from 24,576 columns on while a row has 2,048 columns for each row of the call.
// Measured, us, one workgroup (in a graph) and parts: mixed settings bf16 1 x 32768 18 and
// 20, 1 x 131072 36 and 20, 16 x 65536 45 and 31, 64 x 131072 101 and 61; a nucleus fp32 1 x 32768
// 28 and 23, 32 x 65536 47 and 41; all settings on fp32 1 x 32768 23 and 23, 1 x 131072 40 and 24,
// 32 x 65536 31 and 37, 64 x 65536 32 and 41, 128 x 131072 52 and 68.
inline SamplePlan sample_plan(int rows, int cols, int cus) {
    if (cols < 24576 || (long long)rows * 2048 > cols)
        return {1, cols, cols <= 1024 ? 256 : cols <= 8192 ? 512 : 1024};
    int parts = (cols + 4095) / 4096;
    if (parts > kSampleParts) parts = kSampleParts;
    while (parts > 2 && (long long)parts * rows > 2 * cus) --parts;
    const int per = (int)(((long long)cols + parts - 1) / parts + 1023) / 1024 * 1024;
    return {(cols + per - 1) / per, per, 1024};
}

}  // namespace acfun
