// k_mxmm.hip -- products of MXFP4 operands (mx.hpp) on the scaled MFMA.
#include "mx.hpp"

namespace acfun {
namespace {

typedef int i4v __attribute__((ext_vector_type(4)));
typedef int i8v __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ i8v wide(i4v v) { return i8v{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

// One wave: a 16 x 16 tile of C.  The weights are the MFMA's A operand, so a
// lane's four results are consecutive columns of one row of C.
template <class T>
__global__ __launch_bounds__(64) void k_mxmm16(int M, int N, int K, const uint8_t* __restrict__ A,
                                               const uint8_t* __restrict__ As, const uint8_t* __restrict__ B,
                                               const uint8_t* __restrict__ Bs, T* __restrict__ C,
                                               const float* __restrict__ bias, int act, long long nt) {
    const int lane = threadIdx.x;
    const long long tm = blockIdx.x / nt, tn = blockIdx.x - tm * nt;
    const int kt = mx_k_tiles(K), st = mx_scale_tiles(K);
    const i4v* a = (const i4v*)A + tm * kt * 64 + lane;
    const i4v* b = (const i4v*)B + tn * kt * 64 + lane;
    const unsigned* as = (const unsigned*)As + tm * st * 64 + lane;
    const unsigned* bs = (const unsigned*)Bs + tn * st * 64 + lane;
    f4v acc = {0.f, 0.f, 0.f, 0.f};
    for (int k = 0; k < kt; ++k) {
        const int sh = 8 * (k & 3);
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(b[k * 64]), wide(a[k * 64]), acc, 4, 4, 0,
                                                               bs[(k >> 2) * 64] >> sh, 0, as[(k >> 2) * 64] >> sh);
    }
    const int m = (int)tm * 16 + (lane & 15), n0 = (int)tn * 16 + 4 * (lane >> 4);
    if (m >= M) return;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (n0 + e < N) C[(size_t)m * N + n0 + e] = (T)act_apply(acc[e] + (bias ? bias[n0 + e] : 0.f), act);
}

}  // namespace

bool mx_gemm(int M, int N, int K, const uint8_t* A, const uint8_t* As, const uint8_t* B, const uint8_t* Bs,
             void* C, int type, const float* bias, int act, hipStream_t s) {
    const long long nt = mx_row_tiles(N), tiles = mx_row_tiles(M) * nt;
    if (tiles >= (1ll << 31)) {
        set_error("acfun_dev_gemm_mxfp4: too large");
        return false;
    }
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        ACFUN_LAUNCH("k_mxmm16", (k_mxmm16<T>), dim3((unsigned)tiles), dim3(64), 0, s, M, N, K, A, As, B, Bs,
                     (T*)C, bias, act, nt);
        return check_launch("k_mxmm16");
    });
}

bool mx_fc(const void* x, int type, int M, int K, const uint8_t* B, const uint8_t* Bs, const float* bias,
           int N, void* C, int act, hipStream_t s) {
    Scratch codes(mx_code_bytes(M, K), s), scales(mx_scale_bytes(M, K), s);
    if (K > 0 && (!codes.p || !scales.p)) return false;
    return (K == 0 || mx_quantize(x, type, M, K, 0, codes.as<uint8_t>(), scales.as<uint8_t>(), s)) &&
           mx_gemm(M, N, K, codes.as<uint8_t>(), scales.as<uint8_t>(), B, Bs, C, type, bias, act, s);
}

}  // namespace acfun
