// k_mx.hip -- the MXFP4 quantizer and its inverse (layout and rounding: mx.hpp).
//
// Memory bounds them: max|x| of a block is found among the threads that hold it, so
// a value is read once.  Measured: 4096 x 4096 bf16 8.0 us and back 7.4 (42 MB each, 5.3 and
// 5.7 TB/s), fp32 weights [4096][8192] 23.2 (152 MB, 6.5 TB/s; operands that the caches held
// from the call before), there and back with others each time 56; with a thread to a
// block and its 32 values read one by one 166 and 749 there and back.
#include <type_traits>

#include "mx.hpp"

namespace acfun {
namespace {


// Rows along K.  A workgroup: one scale tile, 16 rows x 512 k.  Thread (r, j, p) has
// the values 8 p .. 8 p + 7 of block j of row r of each of the four 128 k, so 16
// threads read 128 consecutive k of a row, four of them share a block, and a wave
// writes 64 consecutive bytes of codes to each of four places.
template <class T>
__global__ __launch_bounds__(kMxThreads) void k_mx_quant(const T* __restrict__ x, int rows, int K, int st,
                                                  uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const int t = threadIdx.x, r = t >> 4, j = (t >> 2) & 3, p = t & 3;
    const int rt = (int)(blockIdx.x / (unsigned)st), b = (int)(blockIdx.x - (unsigned)rt * st);
    const int kt = mx_k_tiles(K), left = K - 512 * b;
    const unsigned row = rt * 16u + r;
    typename VecOf<T, 8>::type v[4];
    const T* xr = x + (size_t)row * K + 512 * b;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int k = 128 * s + 32 * j + 8 * p;
        v[s] = load_vec<T, 8>(xr + k, row < (unsigned)rows ? left - k : 0);
    }
    const size_t lane = 16 * j + r;
    unsigned bytes = 0;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        unsigned byte;
        const unsigned c = mx_codes_of4(v[s], byte);
        bytes |= byte << (8 * s);
        if (4 * b + s < kt)
            ((unsigned*)codes)[(((size_t)rt * kt + 4 * b + s) * 64 + lane) * 4 + p] = c;
    }
    if (p == 0) ((unsigned*)scales)[((size_t)rt * st + b) * 64 + lane] = bytes;
}

// Rows across K (weights [K][rows]).  A workgroup: 64 rows, block j of each 128 k
// of a scale tile; wave s has the s-th 128 k and lane r a row, so that a wave reads
// 64 neighbours of each k and writes 256 consecutive bytes of codes.
template <class T>
__global__ __launch_bounds__(kMxThreads) void k_mx_quant_t(const T* __restrict__ x, int rows, int K, int groups,
                                                    int st, uint8_t* __restrict__ codes,
                                                    uint8_t* __restrict__ scales) {
    __shared__ unsigned bytes[4][64];
    const int l = threadIdx.x & 63, s = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = (int)(blockIdx.x % (unsigned)groups), bj = (int)(blockIdx.x / (unsigned)groups);
    const int b = bj >> 2, j = bj & 3, kt = mx_k_tiles(K);
    const int k0 = 128 * s + 32 * j, left = K - 512 * b;
    const unsigned row = 64u * g + l;
    float v[32];
    unsigned top = 0;
    const T* xk = x + ((size_t)512 * b + k0) * rows + row;
#pragma unroll
    for (int e = 0; e < 32; ++e) v[e] = row < (unsigned)rows && k0 + e < left ? (float)xk[(size_t)e * rows] : 0.f;
#pragma unroll
    for (int e = 0; e < 32; ++e) top = umax(top, bits_abs(v[e]));
    float scale;
    const unsigned byte = mx_scale(top >> 23, scale);
    bytes[s][l] = byte;
    const size_t rt = row >> 4, lane = 16 * j + (row & 15);
    const bool tile = row < (((unsigned)rows + 15) & ~15u);
    if (tile && 4 * b + s < kt) {
        u4v c;
#pragma unroll
        for (int q = 0; q < 4; ++q) c[q] = mx_codes8(v + 8 * q, scale);
        *(u4v*)(codes + ((rt * kt + 4 * b + s) * 64 + lane) * 16) = c;
    }
    __syncthreads();
    if (s == 0 && tile)
        ((unsigned*)scales)[(rt * st + b) * 64 + lane] =
            bytes[0][l] | bytes[1][l] << 8 | bytes[2][l] << 16 | bytes[3][l] << 24;
}

// The other way.  A thread has V values (16 bytes) of each part of a row's 128 k, so
// that 16 threads store 256 consecutive bytes: eight bf16 or fp16 of one part, four fp32
// of each of two, for which the codes are read as halves of dwords.  Rows of whole
// cache lines are stored past the caches; of others the caches join the parts.
template <class T>
__global__ __launch_bounds__(kMxThreads) void k_mx_dequant(const uint8_t* __restrict__ codes,
                                                    const uint8_t* __restrict__ scales, int rows, int K, int st,
                                                    T* __restrict__ x) {
    constexpr int V = 16 / (int)sizeof(T), H = 8 / V;
    const int t = threadIdx.x, r = t >> 4, l = t & 15;
    const int rt = (int)(blockIdx.x / (unsigned)st), b = (int)(blockIdx.x - (unsigned)rt * st);
    const int kt = mx_k_tiles(K), left = K - 512 * b;
    const unsigned row = rt * 16u + r;
    if (row >= (unsigned)rows) return;
    unsigned bytes[H], c[4][H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        const int k = 16 * V * h + V * l;                       // of the 128
        const size_t lane = 16 * (k >> 5) + r;
        bytes[h] = ((const unsigned*)scales)[((size_t)rt * st + b) * 64 + lane];
#pragma unroll
        for (int s = 0; s < 4; ++s)
            c[s][h] = 4 * b + s < kt ? ((const unsigned*)codes)[(((size_t)rt * kt + 4 * b + s) * 64 + lane) * 4 +
                                                                (k >> 3 & 3)] >> 4 * (k & 7) : 0;
    }
    T* xr = x + (size_t)row * K + 512 * b;
    // ENDS: 0 rows of whole cache lines, 1 of whole 16 bytes, 2 others
    auto put = [&](auto ENDS) {
        constexpr int ends = decltype(ENDS)::value;
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int k = 128 * s + 16 * V * h + V * l;
                const unsigned byte = (bytes[h] >> (8 * s)) & 255u;
                const float scale = mx_scale_float(byte == 255 ? 0 : byte);
                float f[V];
                auto pair = [&](int e, auto v) {
                    f[e] = byte == 255 ? __uint_as_float(0x7fc00000u) : v[0];
                    f[e + 1] = byte == 255 ? __uint_as_float(0x7fc00000u) : v[1];
                };
                pair(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[s][h], scale, 0));
                pair(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[s][h], scale, 1));
                if constexpr (V == 8) {
                    pair(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[s][h], scale, 2));
                    pair(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[s][h], scale, 3));
                }
                if (k < left) store_vec<T, V, ends == 0>(xr + k, ends < 2 ? V : left - k, f);
            }
    };
    if (K % (8 * V) == 0) put(std::integral_constant<int, 0>{});
    else if (K % V == 0) put(std::integral_constant<int, 1>{});
    else put(std::integral_constant<int, 2>{});
}

}  // namespace

bool mx_quantize(const void* x, int type, int rows, int K, int trans, uint8_t* codes, uint8_t* scales,
                 hipStream_t s) {
    const long long st = mx_scale_tiles(K), groups = ((long long)rows + 63) / 64;
    const long long grid = mx_quant_groups(rows, K, trans);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if (trans) {
            ACFUN_LAUNCH("k_mx_quant_t", (k_mx_quant_t<T>), dim3((unsigned)grid), dim3(kMxThreads), 0, s, (const T*)x,
                         rows, K, (int)groups, (int)st, codes, scales);
            return check_launch("k_mx_quant_t");
        }
        ACFUN_LAUNCH("k_mx_quant", (k_mx_quant<T>), dim3((unsigned)grid), dim3(kMxThreads), 0, s, (const T*)x, rows, K,
                     (int)st, codes, scales);
        return check_launch("k_mx_quant");
    });
}

bool mx_dequantize(const uint8_t* codes, const uint8_t* scales, int rows, int K, void* x, int type,
                   hipStream_t s) {
    const long long st = mx_scale_tiles(K), grid = mx_quant_groups(rows, K, 0);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        ACFUN_LAUNCH("k_mx_dequant", (k_mx_dequant<T>), dim3((unsigned)grid), dim3(kMxThreads), 0, s, codes, scales, rows,
                     K, (int)st, (T*)x);
        return check_launch("k_mx_dequant");
    });
}

}  // namespace acfun
