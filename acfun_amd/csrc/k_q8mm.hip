// k_q8mm.hip -- products of Q8 operands (q8.hpp) on the int8 MFMA: with a bias and an
// activation, or two products of the same rows, act(A B0^T + bias0) (A B1^T + bias1).
//
// The weights are the MFMA's A operand, so a lane's consecutive results are
// consecutive columns of one row of C.  Sums are exact in 32-bit integers; a result
// is (sum * row's scale) * column's scale + bias in fp32, rounded once when stored.
#include <type_traits>

#include "mm.hpp"
#include "q8.hpp"

namespace acfun {
namespace {

typedef int i4v __attribute__((ext_vector_type(4)));

struct Q8Args : Q8Product {
    int gm, gn;                     // tiles of C
    int rows;                       // of LDS for quantized rows
};

// ---------------------------------------------------------------- few rows
// 16 TM x 16 TN of C by W waves that split K between them, U 64-k tiles at a time, and
// add up through LDS.  G projections.  B comes from memory to registers, and so does A
// if X is void.  Otherwise A is float rows of X, which the workgroup quantizes into LDS.
template <class T, class X, int TM, int TN, int W, int U, int G>
__global__ __launch_bounds__(64 * W) void k_q8mm_few(Q8Args p) {
    constexpr bool ROWS = !std::is_void_v<X>;
    using E = std::conditional_t<ROWS, X, float>;
    static_assert(!ROWS || TM == 1, "rows of one tile are quantized");
    // partial sums: 16 lanes' quads, and one more, so that the threads of a row read 16
    // different banks; then the quantized rows: codes, 16 scales
    extern __shared__ __attribute__((aligned(16))) char smx[];
    i4v(*const red)[G * TM * TN][68] = (i4v(*)[G * TM * TN][68])smx;
    char* const rc = smx + q8_few_sums(TM, TN, W, G);
    const unsigned R = p.rows;                                  // room for rows, a power of two
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned total = (unsigned)p.gm * p.gn, L = xcd_tile(total);
    if (L >= total) return;
    const unsigned tn = p.gm == 1 ? L : L / p.gm, tm = L - tn * p.gm;
    const unsigned kt = q8_k_tiles(p.K), units = (kt + U - 1) / U;
    const unsigned mt = (unsigned)q8_row_tiles(p.M) - 1, nt = (unsigned)q8_row_tiles(p.N) - 1;
    unsigned* const rs = (unsigned*)(rc + kt * 64 * R);         // rows' max|x|
    const int8_t *a[TM], *b[G][TN];                             // (uniform)
    if constexpr (!ROWS)
#pragma unroll
        for (int i = 0; i < TM; ++i) a[i] = (const int8_t*)p.A + ((uint64_t)(tm * TM + i < mt ? tm * TM + i : mt) * kt << 10);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < TN; ++i) b[g][i] = p.B[g] + ((uint64_t)(tn * TN + i < nt ? tn * TN + i : nt) * kt << 10);
    const unsigned o16 = lane * 16u, j16 = lane >> 4, l16 = lane & 15;
    i4v acc[G][TM][TN];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[g][i][j] = i4v{0, 0, 0, 0};
    struct Unit {
        i4v a[U][TM], b[U][G][TN];
    };
    auto load = [&](Unit& r, unsigned u) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint64_t k = (uint64_t)(u * U + i < kt ? u * U + i : kt - 1) << 10;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int j = 0; j < TN; ++j) r.b[i][g][j] = *(const i4v*)(b[g][j] + k + o16);
            if constexpr (!ROWS)
#pragma unroll
                for (int j = 0; j < TM; ++j) r.a[i][j] = *(const i4v*)(a[j] + k + o16);
        }
    };
    // Pieces of a row and 512 k, eight values to a lane, a wave's W apart: first every
    // row's maximum, then the codes.  The codes of row r in block b (16 k) lie at place
    // r ^ b of its R, so that a piece's blocks are written to different banks.  Rows past
    // M are whatever lies there, for rows of C that are not stored.
    const unsigned rows = (unsigned)p.M - tm * 16 < 16 ? p.M - tm * 16 : 16;
    if constexpr (ROWS) {
        const E* const x = (const E*)p.A + (uint64_t)tm * 16 * (unsigned)p.K;
        const unsigned per = ((unsigned)p.K + 511) / 512, pieces = rows * per;
        if (threadIdx.x < 16) rs[threadIdx.x] = 0;
        __syncthreads();
        for (unsigned q = w; q < pieces; q += W) {
            const unsigned m = q / per, u = q - m * per;
            const int k = 512 * (int)u + 8 * lane;
            const auto v = load_vec<E, 8>(x + (uint64_t)m * (unsigned)p.K + k, p.K - k);
            unsigned top = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = umax(top, bits_abs((float)v[e]));
#pragma unroll
            for (int d = 1; d < 64; d *= 2) top = umax(top, __shfl_xor(top, d));
            if (lane == 0) atomicMax(&rs[m], top);
        }
        __syncthreads();
        for (unsigned q = w; q < pieces; q += W) {
            const unsigned m = q / per, u = q - m * per;
            const int k = 512 * (int)u + 8 * lane;
            const auto v = load_vec<E, 8>(x + (uint64_t)m * (unsigned)p.K + k, p.K - k);
            const Q8Scale sc(rs[m]);
            union { int8_t c[8]; int2 v; } c;
#pragma unroll
            for (int e = 0; e < 8; ++e) c.c[e] = (int8_t)sc.code((float)v[e]);
            const unsigned bl = (unsigned)k >> 4;
            if (bl < 4 * kt) *(int2*)(rc + (bl * R + ((m ^ bl) & (R - 1))) * 16 + (lane & 1) * 8) = c.v;
        }
        __syncthreads();
    }
    auto take_rows = [&](Unit& r, unsigned u) {
        if constexpr (ROWS)
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const unsigned t = u * U + i < kt ? u * U + i : kt - 1, bl = 4 * t + j16;
                r.a[i][0] = *(const i4v*)(rc + (bl * R + ((l16 ^ bl) & (R - 1))) * 16);
            }
    };
    for (unsigned u = w; u < units; u += W) {
        Unit c;
        load(c, u);
        take_rows(c, u);
        each<U>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            if (i > 0 && u * U + i >= kt) return;
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int y = 0; y < TM; ++y)
#pragma unroll
                    for (int x = 0; x < TN; ++x)
                        acc[g][y][x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(c.b[i][g][x], c.a[i][y], acc[g][y][x], 0, 0, 0);
        });
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int y = 0; y < TM; ++y)
#pragma unroll
            for (int x = 0; x < TN; ++x) red[w][(g * TM + y) * TN + x][lane + (lane >> 4)] = acc[g][y][x];
    __syncthreads();
    // four columns of a row to a thread
#pragma unroll
    for (int t0 = 0; t0 < TM * TN * 64; t0 += 64 * W) {
        const int t = t0 + threadIdx.x, m = t / (4 * TN), q = t % (4 * TN);
        const unsigned row = tm * (16 * TM) + m, n = tn * (16 * TN) + 4 * q;
        if (t >= TM * TN * 64 || row >= (unsigned)p.M || n >= (unsigned)p.N) continue;
        const int left = (int)(p.N - n < 4 ? p.N - n : 4);
        const float sa = p.K == 0 ? 0.f : ROWS ? Q8Scale(rs[m]).s : p.As[row];
        float o[4];
        each<G>([&](auto GC) {
            constexpr int g = decltype(GC)::value;
            const i4v* const from = &red[0][(g * TM + (m >> 4)) * TN + (q >> 2)][17 * (q & 3) + (m & 15)];
            i4v v = from[0];
#pragma unroll
            for (int i = 1; i < W; ++i) v += from[i * G * TM * TN * 68];
            const auto sb = load_vec<float, 4>(p.Bs[g] + n, p.K == 0 ? 0 : left);
            const auto bv = load_vec<float, 4>(p.bias[g] + n, p.bias[g] ? left : 0);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y = (float)v[e] * sa * sb[e] + bv[e];
                o[e] = g == 0 ? act_value<sizeof(T) == 4>(y, p.act) : o[e] * y;
            }
        });
        store_vec<T, 4>((T*)p.C + (uint64_t)row * (unsigned)p.N + n, left, o);
    }
}

template <class T, class X, int TM, int TN, int W, int U, int G>
bool launch_few(const Q8Product& p, hipStream_t s) {
    // set once per process, thread-safely, before any launch below
    static const bool attr = [] {
        (void)hipFuncSetAttribute((const void*)k_q8mm_few<T, X, TM, TN, W, U, G>,
                                  hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
        return true;
    }();
    (void)attr;
    Q8Args a;
    (Q8Product&)a = p;
    a.gm = (int)((q8_row_tiles(a.M) + TM - 1) / TM);
    a.gn = (int)((q8_row_tiles(a.N) + TN - 1) / TN);
    a.rows = few_rows(a.M);
    ACFUN_LAUNCH("k_q8mm_few", (k_q8mm_few<T, X, TM, TN, W, U, G>), dim3((unsigned)q8_groups(a.M, a.N, TM, TN)), dim3(64 * W),
                 q8_few_sums(TM, TN, W, G) + (std::is_void_v<X> ? 0 : q8_rows_lds(a.M, a.K)), s, a);
    return check_launch("k_q8mm_few");
}

}  // namespace

bool q8_gemm(const Q8Product& p, int type, hipStream_t s) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return p.gated ? launch_few<T, void, 1, 1, 8, 4, 2>(p, s) : launch_few<T, void, 1, 1, 8, 4, 1>(p, s);
    });
}

bool q8_fc(const char* who, const Q8Product& p, int type, hipStream_t s) {
    if (p.K > 0) {
        const bool fits = q8_rows_fit(p.M, p.N, p.K, p.gated);
        bool one = fits && p.M <= 16;
        if (!one) {
            // a graph would keep the addresses of temporaries that go back to the pool here
            hipStreamCaptureStatus captured = hipStreamCaptureStatusNone;
            if (!check(hipStreamIsCapturing(s, &captured), "hipStreamIsCapturing")) return false;
            one = captured != hipStreamCaptureStatusNone;
            if (one && !(fits && p.M <= kCapturedRows)) {
                set_error("%s: these sizes need temporaries, which a graph cannot keep: capture acfun_dev_quantize_q8 "
                          "and the product with buffers of the caller's", who);
                return false;
            }
        }
        if (one)
            return with_type(type, [&](auto t) {
                using T = decltype(t);
                return p.gated ? launch_few<T, T, 1, 1, 8, 4, 2>(p, s) : launch_few<T, T, 1, 1, 8, 4, 1>(p, s);
            });
    }
    Scratch codes(q8_code_bytes(p.M, p.K), s), scales(q8_scale_bytes(p.M), s);
    if (p.K > 0 && (!codes.p || !scales.p)) return false;
    Q8Product q = p;
    q.A = codes.p;
    q.As = scales.as<float>();
    return (p.K == 0 || q8_quantize(p.A, type, p.M, p.K, 0, codes.as<int8_t>(), scales.as<float>(), s)) &&
           q8_gemm(q, type, s);
}

}  // namespace acfun
