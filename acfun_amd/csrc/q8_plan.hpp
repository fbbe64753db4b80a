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
constexpr int kQ8Threads = 256;
constexpr long long q8_quant_groups(int rows, int trans) {
    return trans ? ((long long)rows + 63) / 64 : q8_row_tiles(rows) * 16;
}
constexpr long long q8_dequant_groups(int rows, int K) {
    return (q8_row_tiles(rows) * q8_k_tiles(K) * 64 + kQ8Threads - 1) / kQ8Threads;
}
constexpr bool q8_quant_fits(int rows, int trans) { return launch_fits(q8_quant_groups(rows, trans), kQ8Threads); }
constexpr bool q8_dequant_fits(int rows, int K) { return launch_fits(q8_dequant_groups(rows, K), kQ8Threads); }

// ---------------------------------------------------------------- products
// Workgroups of a product in tiles of 16 tm x 16 tn.
constexpr long long q8_groups(int M, int N, int tm, int tn) {
    return xcd_groups(((q8_row_tiles(M) + tm - 1) / tm) * ((q8_row_tiles(N) + tn - 1) / tn));
}
constexpr bool q8_mm_fits(int M, int N) { return launch_fits(q8_groups(M, N, 1, 1), 512); }

// LDS of k_q8mm_few: the partial sums of W waves for `mats` projections, and quantized
// rows, for which there is room for 1, 2, 4, 8 or 16, with their scales.
constexpr size_t q8_few_sums(int tm, int tn, int waves, int mats) { return (size_t)waves * tm * tn * mats * 68 * 16; }
constexpr size_t q8_rows_lds(int M, int K) { return (size_t)few_rows(M) * q8_k_tiles(K) * 64 + 64; }
constexpr bool q8_rows_fit(int M, int N, int K, bool gated) {
    return q8_few_sums(1, 1, 8, gated ? 2 : 1) + q8_rows_lds(M, K) <= kLds && q8_mm_fits(M, N);
}

}  // namespace acfun
