// mx.hpp -- MXFP4 operands (microscaled 4-bit floating point) and the element
// types of the float tensors of the transformer-layer entry points.
//
// A block is 32 consecutive k of one row: 32 codes of 4 bits (e2m1: sign, then
// 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one scale byte (e8m0: 2^(byte - 127); 255 = NaN).
// With a = max|x| of the block, byte = max(floor(log2 a) - 2, -127) + 127, and a
// code is x / 2^(byte - 127) rounded to the nearest value, halves to the even
// code, at most 6.  A NaN or an infinity in a block gives byte 255.
//
// Both arrays are laid out as the scaled MFMA reads them.  Codes: tiles of 16
// rows x 128 k, 1024 bytes each, row tiles outermost; the 16 bytes of block j
// (of 4) and row r of a tile are its number 16 j + r, which is the lane that
// feeds them to v_mfma_scale_f32_16x16x128; k even is the low half of a byte.
// A tile is one contiguous kilobyte: one wave's 16-byte loads, and one
// contiguous read from LDS.  Scale bytes: tiles of 16 rows x 512 k, 256 bytes
// each; byte 4 (16 j + r) + s belongs to block j of the tile's s-th 128 k, so
// that a lane's dword holds its scales for four MFMAs and op_sel picks one.
// Rows are padded to 16, codes to 128 k and scales to 512 k; the quantizer
// writes zeros there.
#pragma once
#include "mx_plan.hpp"
#include "rt.hpp"

namespace acfun {

// Element types of float tensors (ACFUN_F32, ACFUN_BF16, ACFUN_F16).
inline bool type_ok(int t) { return t >= 0 && t <= 2; }
inline size_t type_size(int t) { return t == 0 ? 4 : 2; }
// Calls f with a value of the C++ type.
template <class F>
auto with_type(int t, F f) {
    return t == 0 ? f(0.f) : t == 1 ? f((__bf16)0.f) : f((_Float16)0.f);
}

// Eight values, or 16 bytes, of a tensor from any element boundary: global loads and
// stores need no more alignment than an element's.
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f8u __attribute__((ext_vector_type(8), aligned(4)));
typedef __bf16 b8u __attribute__((ext_vector_type(8), aligned(2)));
typedef _Float16 h8u __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 b4u __attribute__((ext_vector_type(4), aligned(2)));
typedef _Float16 h4u __attribute__((ext_vector_type(4), aligned(2)));
template <class T, int N> struct VecOf;
template <> struct VecOf<__bf16, 4> { typedef b4u type; };
template <> struct VecOf<_Float16, 4> { typedef h4u type; };
template <> struct VecOf<float, 4> { typedef f4u type; };
template <> struct VecOf<float, 8> { typedef f8u type; };
template <> struct VecOf<__bf16, 8> { typedef b8u type; };
template <> struct VecOf<_Float16, 8> { typedef h8u type; };
// The first `left` of N values from p; `fill` for the others, which are not read.
template <class T, int N>
__device__ __forceinline__ typename VecOf<T, N>::type load_vec(const T* p, int left, float fill = 0.f) {
    typename VecOf<T, N>::type v;
    if (left >= N) return *(const typename VecOf<T, N>::type*)p;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = e < left ? p[e] : (T)fill;
    return v;
}
// The first `left` of N values to p.  PAST: past the caches, for results that a kernel
// writes as whole lines and that would push out what others read.
template <class T, int N, bool PAST = false>
__device__ __forceinline__ void store_vec(T* p, int left, const float (&v)[N]) {
    if (left >= N) {
        typedef typename VecOf<T, N>::type V;
        V o;
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = (T)v[e];
        if constexpr (PAST) __builtin_nontemporal_store(o, (V*)p);
        else *(V*)p = o;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (e < left) p[e] = (T)v[e];
    }
}
// Lane permutations: xor 1 and xor 2 within four lanes, the mirror of eight and of sixteen.
template <int CTRL>
__device__ __forceinline__ unsigned lane_perm(unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140;

// Eight values -> eight codes.
__device__ __forceinline__ unsigned mx_codes8(const float* v, float scale) {
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
    return r;
}
__device__ __forceinline__ unsigned umax(unsigned a, unsigned b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned bits_abs(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A block's scale byte, and the scale for the hardware's conversions (which read its
// exponent), from the exponent field of max|x| as fp32.  255 (a NaN or an infinity is
// the largest of the values' bit patterns without sign) makes any codes do.
__device__ __forceinline__ unsigned mx_scale(unsigned e, float& scale) {
    const unsigned b = e > 2 ? e - 2 : 0;
    scale = __uint_as_float(b << 23 | 0x400000u);
    return e == 255 ? 255u : b;
}
// 2^(byte - 127)
__device__ __forceinline__ float mx_scale_float(unsigned byte) {
    return __uint_as_float(byte ? byte << 23 : 0x400000u);
}

// Eight values of a block that four neighbouring lanes hold: the block's scale byte
// and the lane's codes.  The 16-bit types find their maximum and are converted as
// pairs, with half the instructions.
__device__ __forceinline__ unsigned max_of4(unsigned top) {
    top = umax(top, lane_perm<kXor1>(top));
    return umax(top, lane_perm<kXor2>(top));
}
__device__ __forceinline__ unsigned mx_codes_of4(const f8u& v, unsigned& byte) {
    float f[8];
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = v[e], top = umax(top, bits_abs(f[e]));
    float scale;
    byte = mx_scale(max_of4(top) >> 23, scale);
    return mx_codes8(f, scale);
}
typedef unsigned u4v __attribute__((ext_vector_type(4)));
// (by value: a bit_cast of a vector's element itself would read element 0)
template <class P>
__device__ __forceinline__ P as_pair(unsigned u) { return __builtin_bit_cast(P, u); }
__device__ __forceinline__ unsigned max16_of4(const u4v& v) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    auto abs2 = [](unsigned u) { return as_pair<us2>(u & 0x7fff7fffu); };
    const us2 m = __builtin_elementwise_max(__builtin_elementwise_max(abs2(v[0]), abs2(v[1])),
                                            __builtin_elementwise_max(abs2(v[2]), abs2(v[3])));
    return max_of4(umax(m[0], m[1]));
}
__device__ __forceinline__ unsigned mx_codes_of4(const b8u& v, unsigned& byte) {
    typedef __bf16 b2v __attribute__((ext_vector_type(2)));
    const u4v u = __builtin_bit_cast(u4v, v);
    float scale;
    byte = mx_scale(max16_of4(u) >> 7, scale);
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_pair<b2v>(u[0]), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_pair<b2v>(u[1]), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_pair<b2v>(u[2]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, as_pair<b2v>(u[3]), scale, 3);
}
__device__ __forceinline__ unsigned mx_codes_of4(const h8u& v, unsigned& byte) {
    typedef _Float16 h2v __attribute__((ext_vector_type(2)));
    const u4v u = __builtin_bit_cast(u4v, v);
    const _Float16 top = __builtin_bit_cast(_Float16, (unsigned short)max16_of4(u));
    float scale;
    byte = mx_scale(__float_as_uint((float)top) >> 23, scale);
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, as_pair<h2v>(u[0]), scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, as_pair<h2v>(u[1]), scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, as_pair<h2v>(u[2]), scale, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, as_pair<h2v>(u[3]), scale, 3);
}

// k_mx.hip
bool mx_quantize(const void* x, int type, int rows, int K, int trans, uint8_t* codes, uint8_t* scales,
                 hipStream_t s);
bool mx_dequantize(const uint8_t* codes, const uint8_t* scales, int rows, int K, void* x, int type,
                   hipStream_t s);
// k_mxmm.hip: C[M,N] = act(A B^T + bias), A and B in 4 bits.
bool mx_gemm(int M, int N, int K, const uint8_t* A, const uint8_t* As, const uint8_t* B, const uint8_t* Bs,
             void* C, int type, const float* bias, int act, hipStream_t s);
// The same with float rows quantized in the call.
bool mx_fc(const void* x, int type, int M, int K, const uint8_t* B, const uint8_t* Bs, const float* bias,
           int N, void* C, int act, hipStream_t s);

// k_norm.hip
struct NormArgs {
    const void *y, *x;              // y: the block's output (null: h = norm(x) alone)
    int rows, cols, layer;          // layer: subtract the mean
    const float *post_w, *post_b;   // norm of y
    const void* gate;               // [ceil(rows / gate_group)][cols], null: 1
    int gate_group;
    float res_scale;
    const float *pre_w, *pre_b;     // norm of the sum
    float eps;
    void *x_out, *h;                // h null: no norm of the sum
    int step = 0;                   // rows from one to the next of a workgroup
};
bool norm_rows(const NormArgs& a, int type, hipStream_t s);
constexpr int kNormMaxCols = 32768;

}  // namespace acfun
