// q8.hpp -- Q8 operands (8-bit integers with a scale for each row).
//
// A row is codes q in -127..127 and one fp32 scale: with a = max|x| of the row,
// scale = a / 127 rounded to fp32, q = x / scale rounded to the nearest integer,
// halves to the even one.  A scale below 2^-126 is 0, and so are its codes; a row
// with a NaN or an infinity has scale NaN and codes 0.
//
// Codes lie as the int8 MFMA reads them: tiles of 16 rows x 64 k, 1024 bytes each, row
// tiles outermost; the 16 bytes number 16 j + r of a tile are k = 16 j .. 16 j + 15 of
// its row r, which is the lane that feeds them to v_mfma_i32_16x16x64_i8 (and, two
// tiles of rows and half of k at a time, to v_mfma_i32_32x32x32_i8).  A tile is one
// contiguous kilobyte: one wave's 16-byte loads, and one contiguous read from LDS.
// Rows are padded to 16 and K to 64 with zeros, scales to 16 rows with zeros.
#pragma once
#include "mx.hpp"
#include "q8_plan.hpp"

namespace acfun {

// The scale of a row from the bits of its max|x| (fp32, no sign), and what its
// codes are found with.
struct Q8Scale {
    float s, inv;                               // inv 0: codes are all 0
    Q8Scale() = default;
    __device__ __forceinline__ explicit Q8Scale(unsigned top) {
        s = __uint_as_float(top) / 127.f;
        const bool bad = top >= 0x7f800000u, live = s >= 0x1p-126f && !bad;
        s = bad ? __uint_as_float(0x7fc00000u) : live ? s : 0.f;
        inv = live ? __builtin_amdgcn_rcpf(s) : 0.f;    // (a step or two off, which the codes allow for)
    }
};
// N values' codes, of which the low byte of c holds each.  q is x / s rounded, from x times
// about 1 / s, in the low bits of a float that has no others below 1; it is off by less
// than one.  What is left over, r = x - q s, is a multiple of half of s's last place and no
// more than s, so the fused product has it exactly, and while it is less than half of s
// for every value the codes are right.  False where it is not: halves, and quotients that
// 1 / s brought to the wrong side of one, a few in a million.
constexpr float kQ8Round = 0x1.8p23f;
template <int N>
__device__ __forceinline__ bool q8_codes_near(const Q8Scale& sc, const float (&v)[N], unsigned (&c)[N]) {
    float most = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float z = __builtin_fmaf(v[e], sc.inv, kQ8Round);
        c[e] = __float_as_uint(z);
        most = __builtin_fmaxf(most, __builtin_fabsf(__builtin_fmaf(kQ8Round - z, sc.s, v[e])));
    }
    return 2.f * most < sc.s;
}
// The same for every value: where 2 |r| - s, exact too, is past 0, or is 0 and q odd, the
// code is the next one on r's side.
template <int N>
__device__ __forceinline__ void q8_codes_exact(const Q8Scale& sc, const float (&v)[N], unsigned (&c)[N]) {
    const unsigned mask = sc.inv == 0.f ? 0u : ~0u;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float z = __builtin_fmaf(v[e], sc.inv, kQ8Round), r = __builtin_fmaf(kQ8Round - z, sc.s, v[e]);
        const float over = __builtin_fmaf(2.f, __builtin_fabsf(r), -sc.s);
        const unsigned q = __float_as_uint(z);
        const bool next = (int)(__float_as_uint(over) + (q & 1)) > 0;
        c[e] = (q + (next ? (unsigned)((int)__float_as_uint(r) >> 31 | 1) : 0u)) & mask;
    }
}
template <int N>
__device__ __forceinline__ void q8_codes(const Q8Scale& sc, const float (&v)[N], unsigned (&c)[N]) {
    if (!q8_codes_near(sc, v, c)) q8_codes_exact(sc, v, c);
}
// The low bytes of four.
__device__ __forceinline__ int low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
    return (int)__builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u),
                                      0x05040100u);
}

// The largest over a wave's lanes, in every lane.
__device__ __forceinline__ unsigned wave_max(unsigned v) {
    v = umax(v, lane_perm<kXor1>(v));
    v = umax(v, lane_perm<kXor2>(v));
    v = umax(v, lane_perm<kMirror8>(v));
    v = umax(v, lane_perm<kMirror16>(v));
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = umax(p[0], p[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return umax(q[0], q[1]);
}
// max|x| of eight values as bits of fp32, by the type's own bits (whose order without
// sign is the values').
__device__ __forceinline__ unsigned abs_max8(const f8u& v) {
    unsigned m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = umax(m, bits_abs(v[e]));
    return m;
}
__device__ __forceinline__ unsigned abs_max8_16(const u4v& v) {
    typedef unsigned short us2 __attribute__((ext_vector_type(2)));
    auto abs2 = [](unsigned u) { return as_pair<us2>(u & 0x7fff7fffu); };
    const us2 m = __builtin_elementwise_max(__builtin_elementwise_max(abs2(v[0]), abs2(v[1])),
                                            __builtin_elementwise_max(abs2(v[2]), abs2(v[3])));
    return umax(m[0], m[1]);
}
__device__ __forceinline__ unsigned abs_max8(const b8u& v) { return abs_max8_16(__builtin_bit_cast(u4v, v)) << 16; }
__device__ __forceinline__ unsigned abs_max8(const h8u& v) {
    return __float_as_uint((float)__builtin_bit_cast(_Float16, (unsigned short)abs_max8_16(__builtin_bit_cast(u4v, v))));
}
// Eight values of a tensor of E as floats; eight codes as bytes.
template <class E>
__device__ __forceinline__ void floats8(const typename VecOf<E, 8>::type& v, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
}
__device__ __forceinline__ int2 bytes8(const unsigned (&c)[8]) {
    return {low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7])};
}

// Activations, as in the header.  exp by the hardware's 2^x, off by a step, 2^-23; half a
// step of its argument is |v| 2^-24 of the result, and the reciprocal is off by a step: 2^-17
// in all for |v| up to 88, beside half a step of bf16 and fp16, 2^-9 and 2^-12 of a value at
// least.  EXACT (fp32 results) adds what the argument's rounding lost, and divides.  NaN stays NaN.
template <bool EXACT>
__device__ __forceinline__ float exp_of(float v) {
    constexpr float L = 0x1.715476p+0f, l = 0x1.4ae0cp-26f, ln2 = 0x1.62e43p-1f;  // log2 e = L + l
    const float t = v * L, e = __builtin_amdgcn_exp2f(t);
    if constexpr (!EXACT) return e;
    const float d = __builtin_fmaf(v, L, -t) + v * l;
    return __builtin_fabsf(v) < 88.f ? __builtin_fmaf(e, d * ln2, e) : e;                // (past it e may be infinite)
}
constexpr int ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_GELU_TANH = 4;
template <bool EXACT>
__device__ __forceinline__ float act_value(float v, int act) {
    if (act == 0) return v;
    if (act == ACT_RELU) return __builtin_elementwise_maximum(v, 0.f);
    if (act == ACT_GELU) return 0.5f * v * erfcf(v * -0x1.6a09e6p-1f);
    float z = v;
    if (act == ACT_GELU_TANH) z = 0x1.988454p+0f * (v + 0.044715f * v * v * v);                // 2 sqrt(2 / pi)
    const float e = 1.f + exp_of<EXACT>(-z);
    if constexpr (EXACT) return v / e;
    return v * __builtin_amdgcn_rcpf(e);
}

struct Q8Product {
    int M, N, K;
    const void* A;                              // codes, or float rows of a layer
    const float* As;                            // (null: float rows)
    const int8_t* B[2];
    const float* Bs[2];
    const float* bias[2];
    void* C;
    int act;
    bool gated;                                 // two projections
};

// k_q8.hip
bool q8_quantize(const void* x, int type, int rows, int K, int trans, int8_t* codes, float* scales, hipStream_t s);
bool q8_dequantize(const int8_t* codes, const float* scales, int rows, int K, void* x, int type, hipStream_t s);
// k_q8mm.hip: C = act(A B0^T + bias0), times A B1^T + bias1 if there is a second.
bool q8_gemm(const Q8Product& p, int type, hipStream_t s);
// The same with float rows quantized in the call, which an error names.
bool q8_fc(const char* who, const Q8Product& p, int type, hipStream_t s);

// k_sample.hip
struct SampleArgs {
    const void* x;
    int rows, cols, ld;
    const float* temp;
    const int* top_k;
    const float *top_p, *min_p, *u;
    int* token;
    float* prob;
};
bool sample_rows(const SampleArgs& a, int type, hipStream_t s);

}  // namespace acfun
