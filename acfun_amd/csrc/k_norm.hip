// k_norm.hip -- the norms before and after a block, with the block's gate and
// the residual sum.
//
//   norm(v) = (v - mean) / sqrt(mean((v - mean)^2) + eps) * w + b   (layer)
//   norm(v) = v / sqrt(mean(v^2) + eps) * w + b                     (RMS)
//   x_out = res_scale * x + gate * norm(y),  h = norm(x_out)
//
// Everything is in fp32; x_out and h are rounded once, when they are stored (h
// is the norm of the sum before its rounding).
#include "mx.hpp"

namespace acfun {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_sum(float v, float* red) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();                                   // red may still be read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[0];
    for (int i = 1; i < kThreads / 64; ++i) t += red[i];
    return t;
}

// Mean (layer) and 1 / sqrt(variance + eps) of a row held as up to kPer values
// per thread.
template <int PER>
__device__ __forceinline__ void row_stats(const float (&v)[PER], int cols, int layer, float eps, float* red,
                                          float& mean, float& rs) {
    mean = 0.f;
    if (layer) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) s += v[i];       // 0 past the row's end
        mean = block_sum(s, red) / (float)cols;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const float d = i * kThreads + (int)threadIdx.x < cols ? v[i] - mean : 0.f;
        q = fmaf(d, d, q);
    }
    rs = 1.f / sqrtf(block_sum(q, red) / (float)cols + eps);
}

// One workgroup per row, the row in registers: every value is read once.
template <class T, int PER>
__global__ __launch_bounds__(kThreads) void k_norm_row(NormArgs a) {
    __shared__ float red[kThreads / 64];
    const size_t row = blockIdx.x, at = row * a.cols;
    const T *xr = (const T*)a.x + at, *yr = (const T*)a.y + at;
    float v[PER], mean, rs;
    if (a.y) {
        const T* gr = a.gate ? (const T*)a.gate + row / a.gate_group * a.cols : nullptr;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = i * kThreads + threadIdx.x;
            v[i] = c < a.cols ? (float)yr[c] : 0.f;
        }
        row_stats<PER>(v, a.cols, a.layer, a.eps, red, mean, rs);
        T* xo = (T*)a.x_out + at;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = i * kThreads + threadIdx.x;
            if (c >= a.cols) continue;
            float n = (v[i] - mean) * rs * (a.post_w ? a.post_w[c] : 1.f) + (a.post_b ? a.post_b[c] : 0.f);
            if (gr) n *= (float)gr[c];
            v[i] = a.res_scale * (float)xr[c] + n;
            xo[c] = (T)v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = i * kThreads + threadIdx.x;
            v[i] = c < a.cols ? (float)xr[c] : 0.f;
        }
    }
    if (!a.h) return;
    row_stats<PER>(v, a.cols, a.layer, a.eps, red, mean, rs);
    T* hr = (T*)a.h + at;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int c = i * kThreads + threadIdx.x;
        if (c < a.cols)
            hr[c] = (T)((v[i] - mean) * rs * (a.pre_w ? a.pre_w[c] : 1.f) + (a.pre_b ? a.pre_b[c] : 0.f));
    }
}

template <class T, int PER>
bool launch(const NormArgs& a, hipStream_t s) {
    ACFUN_LAUNCH("k_norm_row", (k_norm_row<T, PER>), dim3((unsigned)a.rows), dim3(kThreads), 0, s, a);
    return check_launch("k_norm_row");
}

}  // namespace

bool norm_rows(const NormArgs& a, int type, hipStream_t s) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        const int per = (a.cols + kThreads - 1) / kThreads;
        return per <= 4 ? launch<T, 4>(a, s) : per <= 16 ? launch<T, 16>(a, s) : per <= 32 ? launch<T, 32>(a, s)
             : launch<T, 128>(a, s);
    });
}

}  // namespace acfun
