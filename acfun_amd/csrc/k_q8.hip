// k_q8.hip -- the Q8 quantizer and its inverse (layout and rounding: q8.hpp).
#include "q8.hpp"

namespace acfun {
namespace {

typedef int i4v __attribute__((ext_vector_type(4)));

// Rows along K: a workgroup to a row, which it reads twice.
template <class T>
__global__ __launch_bounds__(kQ8Threads) void k_q8_quant(const T* __restrict__ x, int rows, int K,
                                                         int8_t* __restrict__ codes, float* __restrict__ scales) {
    __shared__ unsigned top[kQ8Threads / 64];
    const unsigned row = blockIdx.x, t = threadIdx.x;
    const T* const xr = x + (size_t)row * K;
    const bool live = row < (unsigned)rows;
    unsigned m = 0;
    if (live)
        for (int k = 8 * t; k < K; k += 8 * kQ8Threads) {
            const auto v = load_vec<T, 8>(xr + k, K - k);
#pragma unroll
            for (int e = 0; e < 8; ++e) m = umax(m, bits_abs((float)v[e]));
        }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m = umax(m, __shfl_xor(m, d));
    if ((t & 63) == 0) top[t >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQ8Threads / 64; ++i) m = umax(m, top[i]);
    const Q8Scale sc(m);
    if (t == 0) scales[row] = sc.s;
    const int kt = q8_k_tiles(K);
    for (int p = t; p < 4 * kt; p += kQ8Threads) {              // 16 k each
        union { int8_t b[16]; i4v v; } c;
        const int left = live ? K - 16 * p : 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const auto v = load_vec<T, 8>(xr + 16 * p + 8 * h, left - 8 * h);
#pragma unroll
            for (int e = 0; e < 8; ++e) c.b[8 * h + e] = (int8_t)sc.code((float)v[e]);
        }
        *(i4v*)(codes + ((((size_t)(row >> 4) * kt + (p >> 2)) * 64 + 16 * (p & 3) + (row & 15)) << 4)) = c.v;
    }
}

// Rows across K (weights [K][rows]): a workgroup to 64 rows, a lane to a row, K split
// between the waves.
template <class T>
__global__ __launch_bounds__(kQ8Threads) void k_q8_quant_t(const T* __restrict__ x, int rows, int K,
                                                           int8_t* __restrict__ codes, float* __restrict__ scales) {
    constexpr int W = kQ8Threads / 64;
    __shared__ unsigned top[W][64];
    const unsigned l = threadIdx.x & 63, w = threadIdx.x >> 6, row = blockIdx.x * 64 + l;
    const bool live = row < (unsigned)rows;
    const T* const xr = x + row;
    unsigned m = 0;
    if (live)
        for (int k = w; k < K; k += W) m = umax(m, bits_abs((float)xr[(size_t)k * rows]));
    top[w][l] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) m = umax(m, top[i][l]);
    const Q8Scale sc(m);
    if (row >= (((unsigned)rows + 15) & ~15u)) return;
    if (w == 0) scales[row] = sc.s;
    const int kt = q8_k_tiles(K);
    for (int p = w; p < 4 * kt; p += W) {
        union { int8_t b[16]; i4v v; } c;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int k = 16 * p + e;
            c.b[e] = live && k < K ? (int8_t)sc.code((float)xr[(size_t)k * rows]) : (int8_t)0;
        }
        *(i4v*)(codes + ((((size_t)(row >> 4) * kt + (p >> 2)) * 64 + 16 * (p & 3) + (row & 15)) << 4)) = c.v;
    }
}

// The other way: 16 codes to a thread.  127 times a rounded scale may pass the largest
// value, which the row had then.
template <class T>
__global__ __launch_bounds__(kQ8Threads) void k_q8_dequant(const int8_t* __restrict__ codes,
                                                           const float* __restrict__ scales, int rows, int K,
                                                           T* __restrict__ x) {
    const size_t i = (size_t)blockIdx.x * kQ8Threads + threadIdx.x;
    const int kt = q8_k_tiles(K), lane = (int)(i & 63);
    const size_t tile = i >> 6, rt = tile / (unsigned)kt;
    const size_t row = rt * 16 + (lane & 15);
    const int k = (int)(tile - rt * (unsigned)kt) * 64 + 16 * (lane >> 4);
    if (row >= (size_t)rows || k >= K) return;
    union { int8_t b[16]; i4v v; } c;
    c.v = *(const i4v*)(codes + (i << 4));
    const float s = scales[row];
    const float most = sizeof(T) == 4 ? 0x1.fffffep+127f : __is_same(T, _Float16) ? 65504.f : 0x1.fep+127f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = (float)c.b[8 * h + e] * s;
            f[e] = v > most ? most : v < -most ? -most : v;
        }
        if (k + 8 * h < K) store_vec<T, 8>(x + row * K + k + 8 * h, K - k - 8 * h, f);
    }
}

}  // namespace

bool q8_quantize(const void* x, int type, int rows, int K, int trans, int8_t* codes, float* scales, hipStream_t s) {
    const unsigned grid = (unsigned)q8_quant_groups(rows, trans);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if (trans) {
            ACFUN_LAUNCH("k_q8_quant_t", (k_q8_quant_t<T>), dim3(grid), dim3(kQ8Threads), 0, s, (const T*)x, rows, K,
                         codes, scales);
            return check_launch("k_q8_quant_t");
        }
        ACFUN_LAUNCH("k_q8_quant", (k_q8_quant<T>), dim3(grid), dim3(kQ8Threads), 0, s, (const T*)x, rows, K, codes,
                     scales);
        return check_launch("k_q8_quant");
    });
}

bool q8_dequantize(const int8_t* codes, const float* scales, int rows, int K, void* x, int type, hipStream_t s) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        ACFUN_LAUNCH("k_q8_dequant", (k_q8_dequant<T>), dim3((unsigned)q8_dequant_groups(rows, K)), dim3(kQ8Threads), 0,
                     s, codes, scales, rows, K, (T*)x);
        return check_launch("k_q8_dequant");
    });
}

}  // namespace acfun
