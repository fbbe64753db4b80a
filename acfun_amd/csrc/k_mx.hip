// k_mx.hip -- the MXFP4 quantizer and its inverse (layout and rounding: mx.hpp).
#include "mx.hpp"

namespace acfun {
namespace {

typedef unsigned u4v __attribute__((ext_vector_type(4)));
typedef __bf16 b2v __attribute__((ext_vector_type(2)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));

// Four pairs of values -> eight codes.
__device__ __forceinline__ unsigned codes8(const float* v, float scale) {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
    return r;
}

// One thread: one block of 32 k of one row, padding included.
template <class T, bool TRANS>
__global__ __launch_bounds__(256) void k_mx_quant(const T* __restrict__ x, int rows, int K, long long blocks,
                                                  uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= blocks) return;
    const int kt = mx_k_tiles(K), st = mx_scale_tiles(K), kb = st * 16;
    const int r = (int)(i / kb), b = (int)(i - (long long)r * kb);
    float v[32];
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        const int k = 32 * b + e;
        v[e] = r < rows && k < K ? (float)x[TRANS ? (size_t)k * rows + r : (size_t)r * K + k] : 0.f;
        const unsigned u = __float_as_uint(v[e]) & 0x7fffffffu;
        top = u > top ? u : top;
    }
    const unsigned byte = mx_scale_byte(top);
    const float scale = mx_scale_float(byte == 255 ? 0 : byte);
    const long long t16 = r >> 4;
    const int lane = 16 * (b & 3) + (r & 15);
    scales[(t16 * st + (b >> 4)) * 256 + 4 * lane + ((b >> 2) & 3)] = (uint8_t)byte;
    if (b < 4 * kt) {
        u4v c;
#pragma unroll
        for (int q = 0; q < 4; ++q) c[q] = codes8(v + 8 * q, scale);
        *(u4v*)(codes + ((t16 * kt + (b >> 2)) * 64 + lane) * 16) = c;
    }
}

template <class T>
__global__ __launch_bounds__(256) void k_mx_dequant(const uint8_t* __restrict__ codes,
                                                    const uint8_t* __restrict__ scales, int rows, int K,
                                                    long long blocks, T* __restrict__ x) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= blocks) return;
    const int kt = mx_k_tiles(K), st = mx_scale_tiles(K), kb = (K + 31) / 32;
    const int r = (int)(i / kb), b = (int)(i - (long long)r * kb);
    const long long t16 = r >> 4;
    const int lane = 16 * (b & 3) + (r & 15);
    const unsigned byte = scales[(t16 * st + (b >> 4)) * 256 + 4 * lane + ((b >> 2) & 3)];
    const float scale = byte == 255 ? __uint_as_float(0x7fc00000u) : mx_scale_float(byte);
    const u4v c = *(const u4v*)(codes + ((t16 * kt + (b >> 2)) * 64 + lane) * 16);
    constexpr unsigned kTwice[2] = {0x03020100u, 0x0c080604u};   // twice the values of codes 0..7
#pragma unroll
    for (int e = 0; e < 32; ++e) {
        const unsigned q = (c[e >> 3] >> (4 * (e & 7))) & 15u;
        const float m = 0.5f * (float)((kTwice[(q >> 2) & 1] >> (8 * (q & 3))) & 255u);
        const int k = 32 * b + e;
        if (k < K) x[(size_t)r * K + k] = (T)((q & 8 ? -m : m) * scale);
    }
}

bool grid_ok(long long n, const char* what) {
    if (n < (1ll << 31)) return true;
    set_error("%s: too large", what);
    return false;
}

}  // namespace

bool mx_quantize(const void* x, int type, int rows, int K, int trans, uint8_t* codes, uint8_t* scales,
                 hipStream_t s) {
    const long long blocks = mx_row_tiles(rows) * 16 * mx_scale_tiles(K) * 16, grid = (blocks + 255) / 256;
    if (!grid_ok(grid, "acfun_dev_quantize_mxfp4")) return false;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if (trans)
            ACFUN_LAUNCH("k_mx_quant", (k_mx_quant<T, true>), dim3((unsigned)grid), dim3(256), 0, s, (const T*)x,
                         rows, K, blocks, codes, scales);
        else
            ACFUN_LAUNCH("k_mx_quant", (k_mx_quant<T, false>), dim3((unsigned)grid), dim3(256), 0, s, (const T*)x,
                         rows, K, blocks, codes, scales);
        return check_launch("k_mx_quant");
    });
}

bool mx_dequantize(const uint8_t* codes, const uint8_t* scales, int rows, int K, void* x, int type,
                   hipStream_t s) {
    const long long blocks = (long long)rows * ((K + 31) / 32), grid = (blocks + 255) / 256;
    if (!grid_ok(grid, "acfun_dev_dequantize_mxfp4")) return false;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        ACFUN_LAUNCH("k_mx_dequant", (k_mx_dequant<T>), dim3((unsigned)grid), dim3(256), 0, s, codes, scales, rows,
                     K, blocks, (T*)x);
        return check_launch("k_mx_dequant");
    });
}

}  // namespace acfun
