// k_q8.hip -- the Q8 quantizer and its inverse (layout and rounding: q8.hpp).
//
// A row's scale is known once all of it has been read, so a workgroup keeps its rows in LDS
// (columns: in registers) between the two and reads them once; past what those hold the end
// of a row is read again.  4096 x 4096 bf16 takes 10.8 us with the input in the caches, 16 to 17
// after other work, 8192 x 8192 46.  A copy's 5.55 TB/s would be 9.1 for the first; the codes' loop
// has some 100 instructions to a turn, 8 turns to a wave, 8 waves to a SIMD, which is 10.7,
// three quarters of it in turns without values (below).  Weights wait for whole columns: fp32
// [4096][8192] 53 to 55 us (3.1 TB/s).  Reading back is bound by memory: 9.9 us, and 26.6
// to 28.0 for the weights (6.0 TB/s, the codes from the caches).
#include <type_traits>

#include "mm.hpp"
#include "q8.hpp"

namespace acfun {
namespace {

typedef int i4v __attribute__((ext_vector_type(4)));

// Where the 16 codes of a row's piece p (16 k) lie.
__device__ __forceinline__ i4v* piece_at(int8_t* codes, size_t row, int kt, int p) {
    return (i4v*)(codes + ((((row >> 4) * (unsigned)kt + (p >> 2)) * 64 + 16 * (p & 3) + (row & 15)) << 4));
}

// Rows along K.  A workgroup: R rows; lane (p, r) of a step of its waves has piece
// 64 / R step + p of row r, so that a wave reads 2 KB / R of each row in 16 bits and
// writes 16 R bytes to a place.  A wave takes every 8th step and keeps NI of them.
template <class T, int R, int NI, bool WHOLE>
__global__ __launch_bounds__(kQ8RowThreads) void k_q8_quant(const T* __restrict__ x, int rows, int K,
                                                            int8_t* __restrict__ codes, float* __restrict__ scales) {
    constexpr int W = kQ8RowThreads / 64, P = 64 / R;
    typedef typename VecOf<T, 8>::type V;
    __shared__ unsigned tops[W][R];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane % R, p0 = lane / R;
    const size_t row = (size_t)blockIdx.x * R + r;
    const int kt = q8_k_tiles(K), steps = (4 * kt + P - 1) / P, end = row < (size_t)rows ? K : 0;
    const T* const xr = x + row * (unsigned)K;
    // a step's values of this thread, from memory or (at < NI) where it keeps them in LDS
    extern __shared__ __attribute__((aligned(16))) char smx[];
    struct Piece { V v[2]; };
    constexpr int VB = 8 * (int)sizeof(T);
    char* const mine = smx + threadIdx.x * 16;
    auto get = [&](int step) {
        Piece a = {};
        const int k = 16 * (P * step + p0);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (!WHOLE) a.v[h] = load_vec<T, 8>(xr + k + 8 * h, end - k - 8 * h);
            else if (k + 8 * h < end) a.v[h] = *(const V*)(xr + k + 8 * h);
        }
        return a;
    };
    union Raw { Piece a; i4v q[VB / 8]; };
    unsigned top = 0;
    auto see = [&](const Piece& a) { top = umax(top, umax(abs_max8(a.v[0]), abs_max8(a.v[1]))); };
    if constexpr (WHOLE) {
        Raw a[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (w + i * W < kt) a[i].a = get(w + i * W);
#pragma unroll
        for (int i = 0; i < NI; ++i)
            if (w + i * W < kt) {
                see(a[i].a);
#pragma unroll
                for (int j = 0; j < VB / 8; ++j) *(i4v*)(mine + (i * (VB / 8) + j) * kQ8RowThreads * 16) = a[i].q[j];
            }
    }
#pragma unroll 2
    for (int s = w + (WHOLE ? NI : 0) * W; s < steps; s += W) see(get(s));
#pragma unroll
    for (int d = R; d < 64; d *= 2) top = umax(top, __shfl_xor(top, d));
    if (p0 == 0) tops[w][r] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top = umax(top, tops[i][r]);
    const Q8Scale sc(top);
    if (w == 0 && p0 == 0) scales[row] = sc.s;
    // A turn for every 64 k of the row, though a step has 16 P of them: the turns from `steps` on,
    // 6 of a wave's 8 for R = 4 and K = 4096, find codes of zeros and store nothing.
#pragma unroll 1
    for (int i = 0; w + i * W < kt; ++i) {
        const int step = w + i * W, p = P * step + p0;
        Raw a;
        if (WHOLE && i < NI) {
#pragma unroll
            for (int j = 0; j < VB / 8; ++j) a.q[j] = *(const i4v*)(mine + (i * (VB / 8) + j) * kQ8RowThreads * 16);
        } else {
            a.a = get(step);
        }
        union { int2 h[2]; i4v v; } o;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float f[8];
            unsigned c[8];
            floats8<T>(a.a.v[h], f);
            q8_codes(sc, f, c);
            o.h[h] = bytes8(c);
        }
        if (p < 4 * kt) *piece_at(codes, row, kt, p) = o.v;
    }
}

// Four words of four neighbouring lanes, word i of lane j becoming word j of lane i.
__device__ __forceinline__ void transpose4(unsigned (&a)[4]) {
    const int l = threadIdx.x;
    auto swap = [&](unsigned& x, unsigned& y, auto CTRL, bool odd) {
        const unsigned t = lane_perm<decltype(CTRL)::value>(odd ? x : y);
        x = odd ? t : x;
        y = odd ? y : t;
    };
    swap(a[0], a[1], std::integral_constant<int, kXor1>{}, l & 1);
    swap(a[2], a[3], std::integral_constant<int, kXor1>{}, l & 1);
    swap(a[0], a[2], std::integral_constant<int, kXor2>{}, l & 2);
    swap(a[1], a[3], std::integral_constant<int, kXor2>{}, l & 2);
}

// Rows across K (weights [K][rows]).  A workgroup: 64 bytes of each k, which are TC
// rows, and all k; a wave has 64 k at once, lane 16 j + 4 c + i of it V rows (16 bytes) of k
// 16 j + 4 i .. + 3, and every 16th 64 k, NI of which it keeps.  Four lanes' codes,
// turned around, are 16 k of four rows: a store writes a whole tile, or half of two.  Neighbouring
// workgroups, which share the lines that they read, run on one XCD.
template <class T, int NI>
__global__ __launch_bounds__(kQ8ColThreads, 4) void k_q8_quant_t(const T* __restrict__ x, int rows, int K, unsigned groups,
                                                              int8_t* __restrict__ codes, float* __restrict__ scales) {
    constexpr int TC = kQ8Cols<sizeof(T)>, V = TC / 4, W = kQ8ColThreads / 64;
    typedef typename VecOf<T, V>::type VT;
    __shared__ unsigned tops[TC];
    __shared__ Q8Scale sc[TC];
    const unsigned L = xcd_tile(groups);
    if (L >= groups) return;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane >> 2 & 3, k0 = (lane >> 4) * 16 + (lane & 3) * 4, kt = q8_k_tiles(K);
    const long long row = (long long)L * TC + c * V, left = (long long)rows - row;
    const bool whole = (long long)L * TC + TC <= rows;
    const T* const xr = x + row;
    struct Piece { VT v[4]; };
    auto get = [&](int t) {
        Piece a = {};
        const int k = 64 * t + k0;
        const T* const from = xr + (size_t)k * (unsigned)rows;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (k + e < K) {
                if (whole) a.v[e] = __builtin_nontemporal_load((const VT*)(from + (size_t)e * (unsigned)rows));
                else a.v[e] = load_vec<T, V>(from + (size_t)e * (unsigned)rows, left < V ? (int)left : V);
            }
        return a;
    };
    unsigned top[V] = {};
    auto see = [&](const Piece& a) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int r = 0; r < V; ++r) top[r] = umax(top[r], bits_abs((float)a.v[e][r]));
    };
    if (threadIdx.x < TC) tops[threadIdx.x] = 0;
    __syncthreads();
    Piece a[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i)
        if (w + i * W < kt) a[i] = get(w + i * W);
#pragma unroll
    for (int i = 0; i < NI; ++i)
        if (w + i * W < kt) see(a[i]);
#pragma unroll 1
    for (int t = w + NI * W; t < kt; t += W) see(get(t));
#pragma unroll
    for (int r = 0; r < V; ++r) atomicMax(&tops[c * V + r], max_of4(top[r]));
    __syncthreads();
    if (threadIdx.x < TC) {
        const Q8Scale s(tops[threadIdx.x]);
        sc[threadIdx.x] = s;
        const long long r = (long long)L * TC + threadIdx.x;
        if (r < q8_row_tiles(rows) * 16) scales[r] = s.s;
    }
    __syncthreads();
    auto put = [&](const Piece& a, int t, auto EXACT) {         // false: some codes may be off
        bool near = true;
        unsigned o[V];
#pragma unroll
        for (int r = 0; r < V; ++r) {
            const Q8Scale s = sc[c * V + r];
            const float f[4] = {(float)a.v[0][r], (float)a.v[1][r], (float)a.v[2][r], (float)a.v[3][r]};
            unsigned q[4];
            if constexpr (decltype(EXACT)::value) q8_codes_exact(s, f, q);
            else near &= q8_codes_near(s, f, q);
            o[r] = (unsigned)low_bytes(q[0], q[1], q[2], q[3]);
        }
#pragma unroll
        for (int h = 0; h < V / 4; ++h) {
            unsigned u[4] = {o[4 * h], o[4 * h + 1], o[4 * h + 2], o[4 * h + 3]};
            transpose4(u);
            const long long r = row + 4 * h + (lane & 3);
            if (r < q8_row_tiles(rows) * 16)
                *piece_at(codes, (size_t)r, kt, 4 * t + (lane >> 4)) = i4v{(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
        }
        return near;
    };
    // few pieces, written again by one copy of the code: what runs once is fetched as it runs
    unsigned doubt = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i)
        if (w + i * W < kt && __ballot(!put(a[i], w + i * W, std::false_type{}))) doubt |= 1u << i;
#pragma unroll 1
    for (int i = 0; w + i * W < kt; ++i)
        if (i >= NI || doubt >> i & 1) put(get(w + i * W), w + i * W, std::true_type{});
}

// The other way.  A wave: 16 rows x 64 k of each of kQ8BackTiles tiles; a lane has 16
// bytes of a row's results, so that a store writes whole runs of 128 or 256 bytes, and
// reads their codes as 8 or 4 bytes.  127 times a rounded scale may pass the largest
// value, which the row had then.
template <class T>
__global__ __launch_bounds__(kQ8Threads) void k_q8_dequant(const int8_t* __restrict__ codes,
                                                           const float* __restrict__ scales, int rows, int K,
                                                           T* __restrict__ x) {
    constexpr int V = 16 / (int)sizeof(T), LPR = 64 / V, RPI = 64 / LPR, H = 16 / RPI;  // lanes to a row, rows at once
    const int kt = q8_k_tiles(K), lane = threadIdx.x & 63, q = lane % LPR, r0 = lane / LPR;
    const size_t tiles = (size_t)q8_row_tiles(rows) * (unsigned)kt;
    const size_t t0 = ((size_t)blockIdx.x * (kQ8Threads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kQ8BackTiles;
    union Codes { int w[V / 4]; int8_t b[V]; } c[kQ8BackTiles][H];
    float s[kQ8BackTiles][H];
#pragma unroll
    for (int t = 0; t < kQ8BackTiles; ++t) {
        if (t0 + t >= tiles) break;
        const size_t rt = (t0 + t) / (unsigned)kt;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int r = r0 + RPI * h;
            const int8_t* const from = codes + ((t0 + t) << 10) + (16 * (q * V >> 4) + r) * 16 + (q * V & 15);
            if constexpr (V == 8) *(int2*)c[t][h].w = *(const int2*)from;
            else c[t][h].w[0] = *(const int*)from;
            s[t][h] = scales[rt * 16 + r];
        }
    }
    const float most = sizeof(T) == 4 ? 0x1.fffffep+127f : __is_same(T, _Float16) ? 65504.f : 0x1.fep+127f;
#pragma unroll
    for (int t = 0; t < kQ8BackTiles; ++t) {
        if (t0 + t >= tiles) break;
        const size_t rt = (t0 + t) / (unsigned)kt;
        const int k = (int)(t0 + t - rt * (unsigned)kt) * 64 + q * V;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const size_t row = rt * 16 + r0 + RPI * h;
            if (row >= (size_t)rows || k >= K) continue;
            float f[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float v = (float)c[t][h].b[e] * s[t][h];
                f[e] = v > most ? most : v < -most ? -most : v;
            }
            store_vec<T, V>(x + row * (unsigned)K + k, K - k, f);
        }
    }
}

template <class T, int R, int NI, bool WHOLE>
bool rows_launch(const void* x, int rows, int K, int8_t* codes, float* scales, hipStream_t s) {
    ACFUN_LAUNCH("k_q8_quant", (k_q8_quant<T, R, NI, WHOLE>), dim3((unsigned)q8_row_groups(rows, R)), dim3(kQ8RowThreads),
                 WHOLE ? NI * kQ8RowThreads * 16 * sizeof(T) : 0, s,
                 (const T*)x, rows, K, codes, scales);
    return check_launch("k_q8_quant");
}
template <class T, int R>
bool rows_kept(const void* x, int rows, int K, int8_t* codes, float* scales, hipStream_t s) {
    if (K % 8) return rows_launch<T, R, 1, false>(x, rows, K, codes, scales, s);
    switch (q8_row_steps(K, R, sizeof(T))) {
        case 1: return rows_launch<T, R, 1, true>(x, rows, K, codes, scales, s);
        case 2: return rows_launch<T, R, 2, true>(x, rows, K, codes, scales, s);
        default: return rows_launch<T, R, sizeof(T) == 4 ? 2 : 4, true>(x, rows, K, codes, scales, s);
    }
}

}  // namespace

bool q8_quantize(const void* x, int type, int rows, int K, int trans, int8_t* codes, float* scales, hipStream_t s) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if (trans) {
            const unsigned groups = (unsigned)q8_col_groups(rows, sizeof(T));
            auto go = [&](auto N) {
                ACFUN_LAUNCH("k_q8_quant_t", (k_q8_quant_t<T, decltype(N)::value>), dim3((unsigned)xcd_groups(groups)),
                             dim3(kQ8ColThreads), 0, s, (const T*)x, rows, K, groups, codes, scales);
                return check_launch("k_q8_quant_t");
            };
            return K <= kQ8ColThreads / 64 * 64 ? go(std::integral_constant<int, 1>{})
                                                        : go(std::integral_constant<int, sizeof(T) == 4 ? 4 : 2>{});
        }
        if (q8_rows_of(rows, num_cus()) == 2) return rows_kept<T, 2>(x, rows, K, codes, scales, s);
        return rows_kept<T, 4>(x, rows, K, codes, scales, s);
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
