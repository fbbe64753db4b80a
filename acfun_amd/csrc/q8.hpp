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
    float s, inv;
    bool codes;                                 // false: they are all 0
    __device__ __forceinline__ explicit Q8Scale(unsigned top) {
        s = __uint_as_float(top) / 127.f;
        codes = s >= 0x1p-126f && top < 0x7f800000u;
        if (top >= 0x7f800000u) s = __uint_as_float(0x7fc00000u);
        else if (!codes) s = 0.f;
        inv = 1.f / s;
    }
    // x / s rounded, halves to even.  x times 1 / s is off by less than one; what is left
    // over, x - q s, is a multiple of half of s's last place and no more than s, so the fused
    // product has it exactly, and it says which side of the half x is on.
    __device__ __forceinline__ int code(float x) const {
        const float q = __builtin_rintf(x * inv), r = __builtin_fmaf(-q, s, x), t = 2.f * __builtin_fabsf(r);
        const int i = (int)q, d = (int)(__float_as_uint(r) >> 31) * -2 + 1;
        return codes ? i + (t > s || (t == s && (i & 1)) ? d : 0) : 0;
    }
};

// Activations (ACFUN_RELU and the others of the header).  exp by the hardware's 2^x: one
// step of its argument is |v| / 2^24 of the result, which bf16 and fp16 do not show;
// EXACT (fp32 results) adds what the argument's rounding lost.  NaN stays NaN.
template <bool EXACT>
__device__ __forceinline__ float exp_of(float v) {
    constexpr float L = 0x1.715476p+0f, l = 0x1.4ae0cp-26f, ln2 = 0x1.62e43p-1f;  // log2 e = L + l
    const float t = v * L, e = __builtin_amdgcn_exp2f(t);
    if constexpr (!EXACT) return e;
    const float d = __builtin_fmaf(v, L, -t) + v * l;
    return __builtin_fabsf(v) < 88.f ? __builtin_fmaf(e, d * ln2, e) : e;                // (past it e may be infinite)
}
template <bool EXACT>
__device__ __forceinline__ float act_value(float v, int act) {
    if (act == 0) return v;
    if (act == 1) return __builtin_elementwise_maximum(v, 0.f);
    if (act == 3) return 0.5f * v * erfcf(v * -0x1.6a09e6p-1f);
    float z = v;
    if (act == 4) z = 0x1.988454p+0f * (v + 0.044715f * v * v * v);                // 2 sqrt(2 / pi)
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
constexpr int kSampleMaxCols = 1 << 24;
constexpr bool sample_fits(int rows) { return launch_fits(rows, 1024); }
bool sample_rows(const SampleArgs& a, int type, hipStream_t s);

}  // namespace acfun
