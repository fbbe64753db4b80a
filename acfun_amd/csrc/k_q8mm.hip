// k_q8mm.hip -- products of Q8 operands (q8.hpp) on the int8 MFMA: with a bias and an
// activation, or two products of the same rows, act(A B0^T + bias0) (A B1^T + bias1).
//
// The weights are the MFMA's A operand, so a lane's consecutive results are
// consecutive columns of one row of C.  Sums are exact in 32-bit integers; a result
// is (sum * row's scale) * column's scale + bias in fp32, rounded once when stored.
//
// Few rows wait for the weights' loads: 1 x 4096 x 4096 5.3 us and 16 rows 5.4, from a
// graph, three sets of operands in turn (3.2 TB/s); one row of float values with both
// projections 8192 x 4096 14.4, in one launch (4.7 TB/s).
// Many rows are bound by the int8 MFMA at the clock that its power leaves: 8192^3 437 us (2.5
// POP/s, MFMA busy 0.79 of cycles at 1.5 GHz; on registers alone it reaches 3.1 to 3.5 with
// random codes), 4096^3 62.  Both projections of a gated product share a tile of rows.
#include <type_traits>

#include "mm.hpp"
#include "q8.hpp"

namespace acfun {
namespace {

typedef int i4v __attribute__((ext_vector_type(4)));
typedef int i16v __attribute__((ext_vector_type(16)));
typedef float f4v __attribute__((ext_vector_type(4)));

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
    Q8Scale* const rs = (Q8Scale*)(rc + kt * 64 * R);           // of 16 rows
    unsigned* const tops = (unsigned*)(rs + 16);
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
    Unit r0, r1;
    // Pieces of a row and 512 k, eight values to a lane, a wave's W apart: first every
    // row's maximum, then the codes.  Up to KEEP pieces of a wave stay in registers
    // between the two, others are read again.  The codes of row r in block b (16 k) lie
    // at place r ^ b of its R, so that a piece's blocks are written to different banks.
    // Rows past M are whatever lies there, for rows of C that are not stored.
    // WHOLE: K is whole eights.
    auto quantize = [&](auto WHOLE) {
        constexpr bool whole = decltype(WHOLE)::value;
        constexpr unsigned KEEP = whole ? 4 : 1;
        const unsigned rows = (unsigned)p.M - tm * 16 < 16 ? p.M - tm * 16 : 16;
        const unsigned du = W / rows, dm = W % rows, per = ((unsigned)p.K + 511) / 512;
        const E* const x = (const E*)p.A + (uint64_t)tm * 16 * (unsigned)p.K;
        typedef typename VecOf<E, 8>::type V;
        struct Piece { unsigned u, m; };                        // 512 k, row (uniform)
        const Piece first{w / rows, w % rows};
        auto next = [&](Piece& q) {
            q.u += du, q.m += dm;
            if (q.m >= rows) q.m -= rows, ++q.u;
        };
        auto get = [&](const Piece& q) {
            const int k = 512 * (int)q.u + 8 * lane;
            const E* const from = x + (uint64_t)q.m * (unsigned)p.K + k;
            V v = {};
            if constexpr (!whole) v = load_vec<E, 8>(from, p.K - k);
            else if (k < p.K) v = *(const V*)from;
            return v;
        };
        auto top = [&](const Piece& q, const V& v, unsigned) {
            const unsigned t = wave_max(abs_max8(v));
            if (lane == 0) atomicMax(&tops[q.m], t);
        };
        uint64_t doubt = 0;                                     // the wave's pieces whose codes may be off
        auto put = [&](const Piece& q, const V& v, auto EXACT, unsigned at) {
            const unsigned bl = 32 * q.u + (lane >> 1);
            float f[8];
            unsigned c[8];
            floats8<E>(v, f);
            const Q8Scale sc = rs[q.m];
            if constexpr (decltype(EXACT)::value) q8_codes_exact(sc, f, c);
            else if (__ballot(!q8_codes_near(sc, f, c))) doubt |= 1ull << at;
            if (bl < 4 * kt) *(int2*)(rc + (bl * R + ((q.m ^ bl) & (R - 1))) * 16 + (lane & 1) * 8) = bytes8(c);
        };
        if (threadIdx.x < 16) tops[threadIdx.x] = 0;
        __syncthreads();
        V v[KEEP];
        auto kept = [&](auto f) {
            Piece q = first;
#pragma unroll
            for (unsigned i = 0; i < KEEP; ++i, next(q))
                if (q.u < per) f(q, v[i], i);
        };
        auto rest = [&](auto f) {                               // (several loads at once, for their latency)
            Piece q = first;
            unsigned n = 0;
#pragma unroll
            for (; n < KEEP; ++n) next(q);
#pragma unroll 1
            for (; q.u < per; n += KEEP) {
                V t[KEEP];
                Piece at[KEEP];
#pragma unroll
                for (unsigned i = 0; i < KEEP; ++i, next(q)) {
                    at[i] = q;
                    if (q.u < per) t[i] = get(q);
                }
#pragma unroll
                for (unsigned i = 0; i < KEEP; ++i)
                    if (at[i].u < per) f(at[i], t[i], n + i);
            }
        };
        auto near = [&](const Piece& q, const V& t, unsigned at) { put(q, t, std::false_type{}, at); };
        // before the weights' loads, behind which they would arrive
        kept([&](const Piece& q, V& t, unsigned) { t = get(q); });
        if (w < units) load(r0, w);
        if (w + W < units) load(r1, w + W);
        kept(top);
        rest(top);
        __syncthreads();
        if (threadIdx.x < 16) rs[threadIdx.x] = Q8Scale(tops[threadIdx.x]);
        __syncthreads();
        kept(near);
        rest(near);
        // few pieces, by one copy of the code: what runs once is fetched as it runs.  (LDS has
        // room for 292 pieces, so a wave has less than 64.)
#pragma unroll 1
        for (; doubt; doubt &= doubt - 1) {
            const unsigned n = w + W * (unsigned)__builtin_ctzll(doubt);
            const Piece q{n / rows, n % rows};
            put(q, get(q), std::true_type{}, 0);
        }
        __syncthreads();
    };
    auto step = [&](const Unit& c, unsigned u) {
        each<U>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            if (i > 0 && u * U + i >= kt) return;
            i4v ar[TM];
#pragma unroll
            for (int y = 0; y < TM; ++y) {
                if constexpr (ROWS) {
                    const unsigned bl = 4 * (u * U + i) + j16;
                    ar[y] = *(const i4v*)(rc + (bl * R + ((l16 ^ bl) & (R - 1))) * 16);
                } else {
                    ar[y] = c.a[i][y];
                }
            }
#pragma unroll
            for (int g = 0; g < G; ++g)
#pragma unroll
                for (int y = 0; y < TM; ++y)
#pragma unroll
                    for (int x = 0; x < TN; ++x)
                        acc[g][y][x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(c.b[i][g][x], ar[y], acc[g][y][x], 0, 0, 0);
        });
    };
    if constexpr (ROWS) {
        if (p.K % 8 == 0) quantize(std::true_type{});
        else quantize(std::false_type{});
    } else {
        if (w < units) load(r0, w);
        if (w + W < units) load(r1, w + W);
    }
    // Two units in turn: one is on its way while the other is multiplied.
    for (unsigned u = w; u < units; u += 2 * W) {
        step(r0, u);
        if (u + 2 * W < units) load(r0, u + 2 * W);
        if (u + W >= units) break;
        step(r1, u + W);
        if (u + 3 * W < units) load(r1, u + 3 * W);
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
        const float sa = p.K == 0 ? 0.f : ROWS ? rs[m].s : p.As[row];
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
                const float y = __builtin_fmaf((float)v[e] * sa, sb[e], bv[e]);
                o[e] = g == 0 ? act_value<sizeof(T) == 4>(y, p.act) : o[e] * y;
            }
        });
        store_vec<T, 4>((T*)p.C + (uint64_t)row * (unsigned)p.N + n, left, o);
    }
}

// ---------------------------------------------------------------- many rows
template <int FM, int FN>
struct Q8Tile {
    static constexpr int BM = 64 * FM, BN = 64 * FN;        // 2 x 2 waves of FM x FN blocks of 32 x 32
    static constexpr int TA = BM / 16, TB = BN / 16;        // row tiles
    static constexpr int STG = (TA + TB) * 1024, RS = 32 * FN + 4;
    static constexpr int LDS = 4 * STG;
    static_assert(4 * 32 * RS * 4 <= LDS, "a block row of each wave's sums");
};

// Tiles of BM rows and BN columns, or BN / 2 columns of each of two projections: four
// waves, operands DMA'd into LDS in chunks of 64 k, four stages.
template <class T, int FM, int FN, int G>
__global__ __launch_bounds__(256, FM * FN > 8 ? 1 : 2) void k_q8mm(Q8Args p) {
    using Tl = Q8Tile<FM, FN>;
    constexpr int CI = FM + FN;                             // DMA instructions of a wave per chunk
    constexpr int FG = FN / G, TG = Tl::TB / G;             // blocks of a wave, row tiles, of one projection
    static_assert(CI % 2 == 0 && 3 * CI < 64 && TG % 4 == 0, "whole DMA instructions per wave, vmcnt");
    extern __shared__ __attribute__((aligned(16))) char smx[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    // an XCD's run goes in groups of 4 tile rows, column-major inside: the tiles it
    // runs together are a compact patch whose operands share its L2
    const unsigned total = (unsigned)p.gm * p.gn, L = xcd_tile(total);
    if (L >= total) return;
    const unsigned grp = L / p.gn / 4, rin = L - 4 * grp * p.gn;
    const unsigned rows = p.gm - 4 * grp < 4 ? p.gm - 4 * grp : 4;
    const int tn = (int)(rin / rows), tm = (int)(4 * grp + rin % rows);
    const int kt = q8_k_tiles(p.K);
    const long long ma = q8_row_tiles(p.M) - 1 - (long long)tm * Tl::TA;
    const long long mb = q8_row_tiles(p.N) - 1 - (long long)tn * TG;
    const int8_t* const A0 = (const int8_t*)p.A + (long long)tm * Tl::TA * kt * 1024;
    const int8_t* const B0 = p.B[0] + (long long)tn * TG * kt * 1024;
    const int8_t* const B1 = G == 2 ? p.B[1] + (long long)tn * TG * kt * 1024 : nullptr;
    // offsets of this wave's row tiles, number wave + 4 t of A's TA, then of B's TB;
    // tiles past the last read the last
    unsigned oc[CI];
#pragma unroll
    for (int t = 0; t < CI; ++t) {
        const int r = t < FM ? 4 * t + wave : (4 * (t - FM) + wave) % TG;
        const long long last = t < FM ? ma : mb;
        oc[t] = (unsigned)(r < last ? r : last) * (unsigned)kt * 1024u;
    }
    // Chunk c into stage c % 4.  Past the end an empty buffer: no memory traffic, zeros
    // that are not multiplied, and the same count to wait for.
    auto issue = [&](int c, int stage, auto tile) {
        constexpr int t = decltype(tile)::value;
        const bool live = c < kt;
        lds_dma16(t < FM ? A0 : 4 * (t - FM) < TG ? B0 : B1, live, smx + stage * Tl::STG + wave * 1024 + t * 4096, lane * 16,
                  oc[t] + (live ? c : 0) * 1024u);
    };
    i16v acc[FM][FN];
    const i16v zero16 = {};
    i4v zero4 = {};
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            asm volatile("" : "+v"(zero4));                 // (or one MFMA's result would be copied)
            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(zero4, zero4, zero16, 0, 0, 0);
        }
    // lane l of a block: row l % 32 (tile l / 16 % 2), k 16 (2 step + l / 32)
    const int l16 = lane & 15, lt = (lane >> 4) & 1, lk = lane >> 5;
    const char* const ra = smx + (2 * wm * FM + lt) * 1024 + lk * 256 + l16 * 16;
    const char* const rb = smx + (Tl::TA + 2 * wn * FG + lt) * 1024 + lk * 256 + l16 * 16;
    i4v fa[2][FM], fb[2][FN];                               // the operands of 32 k, one step ahead
    auto read = [&](auto stage, auto step, auto item) {
        constexpr int s = decltype(step)::value, at = decltype(stage)::value * Tl::STG + s * 512, t = decltype(item)::value;
        if constexpr (t < FM) fa[s][t] = *(const i4v*)(ra + at + t * 2048);
        else fb[s][t - FM] = *(const i4v*)(rb + at + (t - FM) / FG * TG * 1024 + (t - FM) % FG * 2048);
    };
    // Half of chunk c (in stage q): its MFMAs, and between them the next half's reads
    // and half of a later chunk's DMA, a few to each MFMA, so that neither their queues
    // nor the MFMAs wait.
    constexpr int H1 = CI / 2;
    auto half = [&](int c, auto Q, auto S) {
        constexpr int q = decltype(Q)::value, s = decltype(S)::value;
        constexpr int items = CI + H1, per = (items + FM * FN - 1) / (FM * FN);
        using Next = std::integral_constant<int, (q + s) & 3>;                  // the next half's stage and step
        using Step = std::integral_constant<int, s ^ 1>;
        each<FM * FN>([&](auto K) {
            constexpr int k = decltype(K)::value, i = k / FN, j = k % FN;
            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[s][j], fa[s][i], acc[i][j], 0, 0, 0);
            each<per>([&](auto P) {
                constexpr int t = k * per + decltype(P)::value;
                if constexpr (t < CI) read(Next{}, Step{}, std::integral_constant<int, t>{});
                else if constexpr (t < items && s == 1) issue(c + 4, q, std::integral_constant<int, t - CI>{});
                else if constexpr (t < items) issue(c + 3, (q + 3) & 3, std::integral_constant<int, H1 + t - CI>{});
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    using Zero = std::integral_constant<int, 0>;
    using One = std::integral_constant<int, 1>;
#pragma unroll 1
    for (int c = 0; c < 3; ++c) each<CI>([&](auto i) { issue(c, c, i); });
    each<H1>([&](auto i) { issue(3, 3, i); });
    __builtin_amdgcn_s_waitcnt(vm_count(2 * CI + H1));
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    each<CI>([&](auto i) { read(Zero{}, Zero{}, i); });
    float sa[FM];                                           // of the lane's rows
#pragma unroll
    for (int i = 0; i < FM; ++i) {
        const long long m = (long long)tm * Tl::BM + (wm * FM + i) * 32 + (lane & 31);
        sa[i] = p.As[m < p.M ? m : p.M - 1];
    }
    // Chunk c + q, in stage q.  Between its halves it is in registers, everyone's, and
    // its stage is free; the next chunk has landed once the two after it are all that
    // is outstanding.
    int c = 0;
    do {
        each<4>([&](auto Q) {
            constexpr int q = decltype(Q)::value;
            if (q > 0 && c + q >= kt) return;
            half(c + q, Q, Zero{});
            __builtin_amdgcn_s_waitcnt(vm_count(2 * CI));
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            half(c + q, Q, One{});
        });
        c += 4;
    } while (c < kt);
    // Lane l, register e of a block: row l % 32, column 8 (e / 4) + 4 (l / 32) + e % 4.
    // A wave turns its sums around in LDS, 32 rows at a time, for stores of whole cache
    // lines by lanes that keep their columns' scales and biases.  16 bytes between
    // rows: 8 lanes' writes fall on different banks.
    __builtin_amdgcn_s_waitcnt(vm_count(0));                // the chunks past the end
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    constexpr int CV = 16 / (int)sizeof(T), LPR = 32 * FG / CV, RPI = 64 / LPR;   // columns to a lane, lanes to a row
    typedef typename VecOf<float, CV>::type P;
    float* const slab = (float*)smx + wave * 32 * Tl::RS;
    const long long n0 = (long long)tn * (Tl::BN / G) + wn * 32 * FG, m0 = (long long)tm * Tl::BM + wm * 32 * FM;
    const int cl = lane % LPR * CV;                         // this lane's columns, and how many of them there are
    const int left = n0 + cl < p.N ? (int)(p.N - n0 - cl < CV ? p.N - n0 - cl : CV) : 0;
    P sb[G], bv[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
        sb[g] = load_vec<float, CV>(p.Bs[g] + n0 + cl, left);
        bv[g] = load_vec<float, CV>(p.bias[g] + n0 + cl, p.bias[g] ? left : 0);
    }
    auto dump = [&](auto I) {
        constexpr int i = decltype(I)::value;
        each<FN * 4>([&](auto E) {
            constexpr int j = decltype(E)::value / 4, h = decltype(E)::value % 4;
            f4v v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)acc[i][j][4 * h + e] * sa[i];
            *(f4v*)(slab + (lane & 31) * Tl::RS + 32 * j + 8 * h + 4 * lk) = v;
        });
    };
    auto rows_out = [&](long long m, auto UNROLL, auto act) {
        const int rows = p.M - m < 32 ? (int)(p.M - m) : 32;
        T* const C = (T*)p.C + m * p.N + n0 + cl;
        if (left > 0)
#pragma unroll decltype(UNROLL)::value
            for (int r = lane / LPR; r < rows; r += RPI) {
                float o[CV];
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    const f4v* const from = (const f4v*)(slab + r * Tl::RS + 32 * FG * g + cl);
#pragma unroll
                    for (int e = 0; e < CV; ++e) {
                        const float y = __builtin_fmaf(from[e / 4][e % 4], sb[g][e], bv[g][e]);
                        o[e] = g == 0 ? act(y) : o[e] * y;
                    }
                }
                store_vec<T, CV, true>(C + (size_t)r * p.N, left, o);
            }
    };
    each<FM>([&](auto I) {
        dump(I);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        constexpr bool X = sizeof(T) == 4;
        using Four = std::integral_constant<int, 4>;
        const long long m = m0 + 32 * decltype(I)::value;
        if (p.act == 0) rows_out(m, Four{}, [](float v) { return v; });
        else if (p.act == ACT_RELU) rows_out(m, Four{}, [](float v) { return at_least(v, 0.f); });
        else if (p.act == ACT_SILU) rows_out(m, One{}, [](float v) { return act_value<X>(v, ACT_SILU); });
        else if (p.act == ACT_GELU) rows_out(m, One{}, [](float v) { return act_value<X>(v, ACT_GELU); });
        else rows_out(m, One{}, [](float v) { return act_value<X>(v, ACT_GELU_TANH); });
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    });
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
    ACFUN_LAUNCH("k_q8mm_few", (k_q8mm_few<T, X, TM, TN, W, U, G>), dim3((unsigned)xcd_groups((long long)a.gm * a.gn)), dim3(64 * W),
                 q8_few_sums(TM, TN, W, G) + (std::is_void_v<X> ? 0 : q8_rows_lds(a.M, a.K)), s, a);
    return check_launch("k_q8mm_few");
}

template <class T, int FM, int FN, int G>
bool launch_many(const Q8Product& p, hipStream_t s) {
    using Tl = Q8Tile<FM, FN>;
    static_assert(Tl::LDS <= kLds, "LDS");
    // set once per process, thread-safely, before any launch below
    static const bool attr = [] {
        (void)hipFuncSetAttribute((const void*)k_q8mm<T, FM, FN, G>, hipFuncAttributeMaxDynamicSharedMemorySize, Tl::LDS);
        return true;
    }();
    (void)attr;
    Q8Args a;
    (Q8Product&)a = p;
    a.gm = (int)(((long long)a.M + Tl::BM - 1) / Tl::BM);
    a.gn = (int)(((long long)a.N + Tl::BN / G - 1) / (Tl::BN / G));
    ACFUN_LAUNCH("k_q8mm", (k_q8mm<T, FM, FN, G>), dim3((unsigned)xcd_groups((long long)a.gm * a.gn)), dim3(256), Tl::LDS, s, a);
    return check_launch("k_q8mm");
}

}  // namespace

bool q8_gemm(const Q8Product& p, int type, hipStream_t s) {
    const Q8Kind kind = q8_choose(p.M, p.N, p.K, p.gated, num_cus());
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        auto run = [&](auto GC) {
            constexpr int G = decltype(GC)::value;
            switch (kind) {
                case Q8_FEW16: return launch_few<T, void, 1, 1, 8, 4, G>(p, s);
                case Q8_FEW32: return launch_few<T, void, 2, 2 / G, 4, 2, G>(p, s);
                case Q8_FEW64: return launch_few<T, void, 4, 4 / G, 8, 1, G>(p, s);
                case Q8_MANY128: return launch_many<T, 2, 2, G>(p, s);
                default: return launch_many<T, 4, 4, G>(p, s);
            }
        };
        return p.gated ? run(std::integral_constant<int, 2>{}) : run(std::integral_constant<int, 1>{});
    });
}

bool q8_fc(const char* who, const Q8Product& p, int type, hipStream_t s) {
    if (p.K > 0) {
        const bool fits = q8_rows_fit(p.M, p.N, p.K, p.gated);
        bool one = fits && q8_rows_one(p.M, p.K);
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
