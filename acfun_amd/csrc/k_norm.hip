// k_norm.hip -- the norms before and after a block, with the block's gate and
// the residual sum.
//
//   norm(v) = (v - mean) / sqrt(mean((v - mean)^2) + eps) * w + b   (layer)
//   norm(v) = v / sqrt(mean(v^2) + eps) * w + b                     (RMS)
//   x_out = res_scale * x + gate * norm(y),  h = norm(x_out)
//
// Everything is in fp32; x_out and h are rounded once, when they are stored (h
// is the norm of the sum before its rounding).
//
// Memory bounds it: a row is read and written once, whatever the statistics
// need, and results of whole lines are stored past the caches.  Measured: norm and
// residual of 8192 x 8192 bf16 97 us (537 MB, 5.5 TB/s, a copy's rate), the norm of
// 4096 x 4096 fp16 12.3 us; one token 2.1 and eight 3.9 us in a graph, 4.1 and 4.7 from
// the host, which is the cost of a launch.  Rows whose width is no whole chunk start
// off a dword's boundary in 16-bit types: 8192 x 8111 137 us (3.9 TB/s).  With a value per
// thread and step and parameters read for every row: 478, 26.1, 5.6 and 21.2.
// Wide rows, norm and residual, TB/s: 8192 x 16384 bf16 5.5, 4096 x 32768 bf16 4.7; fp32 4096
// x 16384 5.0, 4096 x 32768 4.5; the norm alone 5.3 to 5.8.  The least are widths just past
// a launch's step, which leave up to half of the threads without a chunk: 8192 x 8448 bf16
// 4.2, 4096 x 16388 fp32 3.8.
#include <type_traits>

#include "mx.hpp"

namespace acfun {
namespace {

// The sum over a wave's lanes, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
    v += __uint_as_float(lane_perm<kXor1>(__float_as_uint(v)));
    v += __uint_as_float(lane_perm<kXor2>(__float_as_uint(v)));
    v += __uint_as_float(lane_perm<kMirror8>(__float_as_uint(v)));
    v += __uint_as_float(lane_perm<kMirror16>(__float_as_uint(v)));
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// The sum over the NW waves of a row.  Two buffers in turn: a wave that writes
// one has passed the barrier that follows every wave's reads of it.
template <int NW>
struct RowSum {
    float (*red)[NW];
    int at = 0;
    __device__ __forceinline__ float operator()(float v) {
        v = wave_sum(v);
        if constexpr (NW > 1) {
            if ((threadIdx.x & 63) == 0) red[at][threadIdx.x >> 6] = v;
            __syncthreads();
            v = red[at][0];
#pragma unroll
            for (int i = 1; i < NW; ++i) v += red[at][i];
            at ^= 1;
        }
        return v;
    }
};

// TPR threads to a row (64: a wave, four rows to a workgroup), CH chunks of 16
// bytes to a thread.  The row stays in registers, so every value is read once;
// a workgroup takes rows in turn, `step` apart.  With one or two chunks it keeps the
// weights and the gate of its columns and has the next row's loads under way; biases
// are read where they are added.  128 registers, for four waves per SIMD, hold that
// but for some residuals past 8192 columns: 2 registers of a lane go to memory with
// 1024 threads and two chunks of 16-bit types, 2 with four chunks of fp16 in rows of no
// whole chunk, and 44 to 48 with the eight chunks of fp32 past 16384 columns.  WHOLE: rows
// are whole chunks, so a thread's chunk is all there or not at all, with half the code:
// one row's time is for a good part the fetching of it.
// (gridDim is not asked for: the hidden arguments that it comes with, and any more
// than 128 bytes of them, cost a launch 0.7 us on the host.)
template <class T, int TPR, int CH, bool RES, bool WHOLE>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR, 4) void k_norm_row(NormArgs a) {
    constexpr int VN = 16 / (int)sizeof(T), NW = TPR / 64, RPB = TPR == 64 ? 4 : 1;
    constexpr bool KEEP = CH <= 2;
    typedef typename VecOf<T, VN>::type V;
    typedef typename VecOf<float, VN>::type P;
    __shared__ float red[2][NW];
    RowSum<NW> sum{red};
    const int t = threadIdx.x & (TPR - 1), cols = a.cols;
    int row = (int)(blockIdx.x * RPB) + (RPB > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
    if (row >= a.rows) return;
    auto col = [&](int i) { return (i * TPR + t) * VN; };
    auto get = [&](const T* p, int i) {
        V v = {};
        if constexpr (!WHOLE) v = load_vec<T, VN>(p + col(i), cols - col(i));
        else if (col(i) < cols) v = *(const V*)(p + col(i));
        return v;
    };
    auto get_par = [&](const float* p, int i) {
        P v = {};
        if constexpr (!WHOLE) v = load_vec<float, VN>(p + col(i), cols - col(i));
        else if (col(i) < cols) v = *(const P*)(p + col(i));
        return v;
    };
    auto put = [&](T* p, int i, const float (&v)[VN]) {
        if constexpr (!WHOLE) store_vec<T, VN>(p + col(i), cols - col(i), v);
        else if (col(i) < cols) store_vec<T, VN, true>(p + col(i), VN, v);
    };
    V yv[CH], xv[CH], gv[KEEP ? CH : 1];           // a row of x beside y: KEEP only
    int group = -1;
    auto load = [&](int r) {
        const size_t at = (size_t)r * cols;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            if constexpr (RES) yv[i] = get((const T*)a.y + at, i);
            if constexpr (!RES || KEEP) xv[i] = get((const T*)a.x + at, i);
        }
    };
    auto gate_vec = [&](int i) { return get((const T*)a.gate + (size_t)group * cols, i); };
    auto load_gate = [&](int r) {
        if (!RES || !a.gate || r / a.gate_group == group) return;
        group = r / a.gate_group;
        if constexpr (KEEP) {
#pragma unroll
            for (int i = 0; i < CH; ++i) gv[i] = gate_vec(i);
        }
    };
    load(row);
    load_gate(row);
    P kept[2][KEEP ? CH : 1];
    if constexpr (KEEP) {
#pragma unroll
        for (int q = RES ? 0 : 1; q < 2; ++q)
            if (const float* const w = q ? a.pre_w : a.post_w) {
#pragma unroll
                for (int i = 0; i < CH; ++i) kept[q][i] = get_par(w, i);
            }
    }
    // (n * weight + bias) of chunk i, in place
    auto scale = [&](auto Q, int i, float (&n)[VN]) {
        constexpr int q = decltype(Q)::value;
        const float *const pw = q ? a.pre_w : a.post_w, *const pb = q ? a.pre_b : a.post_b;
        if (pw) {
            P w;
            if constexpr (KEEP) w = kept[q][i];
            else w = get_par(pw, i);
#pragma unroll
            for (int e = 0; e < VN; ++e) n[e] *= w[e];
        }
        if (pb) {
            const P b = get_par(pb, i);
#pragma unroll
            for (int e = 0; e < VN; ++e) n[e] += b[e];
        }
    };
    const float inv = 1.f / (float)cols;
    float v[CH][VN];
    auto in = [&](int i, int e) { return WHOLE ? col(i) < cols : col(i) + e < cols; };
    auto stats = [&](float& mean, float& rs) {
        mean = 0.f;
        float q = 0.f;
        if (a.layer) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int e = 0; e < VN; ++e) s += v[i][e];         // 0 past the row's end
            mean = sum(s) * inv;
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int e = 0; e < VN; ++e) {
                    const float d = in(i, e) ? v[i][e] - mean : 0.f;
                    q = fmaf(d, d, q);
                }
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int e = 0; e < VN; ++e) q = fmaf(v[i][e], v[i][e], q);
        }
        rs = 1.f / sqrtf(sum(q) * inv + a.eps);
    };
    using Post = std::integral_constant<int, 0>;
    using Pre = std::integral_constant<int, 1>;
    for (;;) {
        const size_t at = (size_t)row * cols;
        const bool more = a.step < a.rows - row;
        const int next = more ? row + a.step : row;
        float mean, rs;
        if constexpr (RES) {
            V x[CH];
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                if constexpr (KEEP) x[i] = xv[i];
#pragma unroll
                for (int e = 0; e < VN; ++e) v[i][e] = (float)yv[i][e];
            }
            if (KEEP && more) load(next);
            stats(mean, rs);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                float n[VN];
                if constexpr (!KEEP) x[i] = get((const T*)a.x + at, i);
#pragma unroll
                for (int e = 0; e < VN; ++e) n[e] = (v[i][e] - mean) * rs;
                scale(Post{}, i, n);
                if (a.gate) {
                    V g;
                    if constexpr (KEEP) g = gv[i];
                    else g = gate_vec(i);
#pragma unroll
                    for (int e = 0; e < VN; ++e) n[e] *= (float)g[e];
                }
#pragma unroll
                for (int e = 0; e < VN; ++e) v[i][e] = in(i, e) ? a.res_scale * (float)x[i][e] + n[e] : 0.f;
                put((T*)a.x_out + at, i, v[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (int e = 0; e < VN; ++e) v[i][e] = (float)xv[i][e];
            if (KEEP && more) load(next);
        }
        if (!RES || a.h) {
            stats(mean, rs);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                float n[VN];
#pragma unroll
                for (int e = 0; e < VN; ++e) n[e] = (v[i][e] - mean) * rs;
                scale(Pre{}, i, n);
                put((T*)a.h + at, i, n);
            }
        }
        if (!more) break;
        if (!KEEP) load(next);
        load_gate(next);
        row = next;
    }
}

template <class T, int TPR, int CH>
bool launch(NormArgs a, int cus, hipStream_t s) {
    constexpr int RPB = TPR == 64 ? 4 : 1, THREADS = TPR < 256 ? 256 : TPR;
    // at most four waves per SIMD, and as many rows to each workgroup
    const long long groups = ((long long)a.rows + RPB - 1) / RPB, most = cus * (1024 / THREADS);
    const long long each = (groups + most - 1) / most;
    const dim3 grid((unsigned)((groups + each - 1) / each)), block(THREADS);
    a.step = (int)(grid.x * RPB);
    const bool whole = a.cols % (16 / (int)sizeof(T)) == 0;
    if (a.y && whole) ACFUN_LAUNCH("k_norm_row", (k_norm_row<T, TPR, CH, true, true>), grid, block, 0, s, a);
    else if (a.y) ACFUN_LAUNCH("k_norm_row", (k_norm_row<T, TPR, CH, true, false>), grid, block, 0, s, a);
    else if (whole) ACFUN_LAUNCH("k_norm_row", (k_norm_row<T, TPR, CH, false, true>), grid, block, 0, s, a);
    else ACFUN_LAUNCH("k_norm_row", (k_norm_row<T, TPR, CH, false, false>), grid, block, 0, s, a);
    return check_launch("k_norm_row");
}

}  // namespace

bool norm_rows(const NormArgs& a, int type, hipStream_t s) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int VN = 16 / (int)sizeof(T);
        const int n = (a.cols + VN - 1) / VN;             // chunks of a row
        // Two chunks to a thread rather than one, so that fewer waves wait for each other: 8192
        // x 8192 bf16 97 us against 108, 4096 x 4096 fp16 12.2 against 14.7, 8 x 8192 3.9 and
        // 3.9; but one where that makes 512 threads and the rows leave CUs free: 1 x 4096 2.1
        // against 2.3.
        const int cus = num_cus();
        if (n <= 64) return launch<T, 64, 1>(a, cus, s);
        if (n <= 128) return launch<T, 64, 2>(a, cus, s);
        if (n <= 256) return launch<T, 256, 1>(a, cus, s);
        if (n <= 512) return a.rows <= cus ? launch<T, 512, 1>(a, cus, s) : launch<T, 256, 2>(a, cus, s);
        if (n <= 1024) return launch<T, 512, 2>(a, cus, s);
        if (n <= 2048) return launch<T, 1024, 2>(a, cus, s);
        if (n <= 4096) return launch<T, 1024, 4>(a, cus, s);
        if constexpr (VN == 4) return launch<T, 1024, 8>(a, cus, s);
        return false;
    });
}

}  // namespace acfun
