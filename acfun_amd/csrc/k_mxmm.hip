// k_mxmm.hip -- products of MXFP4 operands (mx.hpp) on the scaled MFMA.
//
// The weights are the MFMA's A operand, so a lane's consecutive results are
// consecutive columns of one row of C.
//
// k_mxmm_few: tiles of 16, 32 or 64 on the 16 x 16 x 128 MFMA, K split between a
// workgroup's waves.  A launch's latency bounds the smallest, the latency of loads the
// others, of which a wave has one unit under way at a time.  In a graph, us: 1 x 4096 x
// 4096 with the quantization of its row 3.4 on the same operands, 4.4 with weights from
// HBM; 1 x 16384 -> 4096 7.1 and 10.7 (34 MB, 3.2 TB/s); the product 128 x 8192 x 4096 6.9
// and 9.2.
//
// k_mxmm: four waves of 2 x 2 or 4 x 4 blocks of 32 x 32, operands DMA'd into LDS in
// chunks of 128 k, four stages.  The 256 x 256 tile needs 512 bytes of LDS reads per
// MFMA, half of what 128 x 128 does.  Its loop takes 1,240 cycles a chunk, of which
// the MFMAs are 1,024; random data at that rate brings the clock down to 1.5 GHz
// (MFMAs alone, on registers, reach 6.5 PFLOP/s with them and 9.4 on zeros), and
// without its LDS reads, or without its DMA, the kernel would be 6 or 10 % faster.
// 8192^3 bf16: 242 us (4.5 PFLOP/s); 4096^3 to fp32: 40 us (3.4; one tile for each CU, so
// that its 67 MB of results are stored at once, at the end); with a wave to each 16 x
// 16 of C and operands from memory 1,800 and 190.
#include <type_traits>

#include "mm.hpp"
#include "mx.hpp"

namespace acfun {
namespace {

typedef int i4v __attribute__((ext_vector_type(4)));
typedef int i8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));

__device__ __forceinline__ i8v wide(i4v v) { return i8v{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

struct MmArgs {
    int M, N, K;
    const void* A;                  // codes, or float rows (k_mxmm_few of rows)
    const uint8_t *As, *B, *Bs;
    void* C;
    const float* bias;
    int act, gm, gn;                // tiles of C
    int rows = 0;                   // of LDS for quantized rows
};

// ---------------------------------------------------------------- few rows
// 16 TM x 16 TN of C by W waves that split K between them, U 128-k tiles at a time,
// and add up through LDS: all of a short K is under way at once.  B comes from
// memory to registers, and so does A if X is void.  Otherwise A is float rows of X,
// which the workgroup quantizes into LDS for its tile, while B's first loads are on
// their way.
template <class T, class X, int TM, int TN, int W, int U>
__global__ __launch_bounds__(64 * W) void k_mxmm_few(MmArgs p) {
    constexpr bool ROWS = !std::is_void_v<X>;
    using E = std::conditional_t<ROWS, X, float>;
    static_assert(!ROWS || TM == 1, "rows of one tile are quantized");
    // partial sums: 16 lanes' quads, and one more, so that the threads of a row read 16
    // different banks; then the quantized rows: codes, scales
    extern __shared__ __attribute__((aligned(16))) char smx[];
    f4v(*const red)[TM * TN][68] = (f4v(*)[TM * TN][68])smx;
    char* const rc = smx + kFewSums<TM, TN, W>;
    const unsigned R = p.rows;                                  // room for rows, a power of two
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned total = (unsigned)p.gm * p.gn, L = xcd_tile(total);
    if (L >= total) return;
    const unsigned tn = p.gm == 1 ? L : L / p.gm, tm = L - tn * p.gm;
    const unsigned kt = mx_k_tiles(p.K), st = mx_scale_tiles(p.K), units = (kt + U - 1) / U;
    const unsigned mt = (unsigned)mx_row_tiles(p.M) - 1, nt = (unsigned)mx_row_tiles(p.N) - 1;
    char* const rs = rc + st * 256 * R;
    const uint8_t *a[TM], *as[TM], *b[TN], *bs[TN];             // (uniform)
    if constexpr (!ROWS)
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const unsigned t = tm * TM + i < mt ? tm * TM + i : mt;
            a[i] = (const uint8_t*)p.A + ((uint64_t)t * kt << 10);
            as[i] = p.As + ((uint64_t)t * st << 8);
        }
#pragma unroll
    for (int i = 0; i < TN; ++i) {
        const unsigned t = tn * TN + i < nt ? tn * TN + i : nt;
        b[i] = p.B + ((uint64_t)t * kt << 10);
        bs[i] = p.Bs + ((uint64_t)t * st << 8);
    }
    const unsigned o16 = lane * 16u, o4 = lane * 4u, j16 = lane >> 4, l16 = lane & 15;
    const unsigned oq = (j16 * R + ((l16 ^ j16) & (R - 1))) * 16, os = (j16 * R + (l16 & (R - 1))) * 4;
    f4v acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f4v{0.f, 0.f, 0.f, 0.f};
    struct Unit {
        i4v a[U][TM], b[U][TN];
        unsigned sa[TM], sb[TN];
    };
    // A wave's units: 2^run neighbours at a time, which one load of scales serves, as long as
    // every wave has that many.
    const int run = U == 4 ? 0 : units >= 4 / U * W ? (U == 1 ? 2 : 1) : U == 1 && units >= 2 * W ? 1 : 0;
    auto unit = [&](unsigned i) { return (((i >> run) * W + w) << run) + (i & ((1 << run) - 1)); };
    auto load = [&](Unit& r, unsigned u, bool scales) {
        const uint64_t g = (uint64_t)(u * U >> 2) << 8;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const uint64_t k = (uint64_t)(u * U + i < kt ? u * U + i : kt - 1) << 10;
#pragma unroll
            for (int j = 0; j < TN; ++j) r.b[i][j] = *(const i4v*)(b[j] + k + o16);
            if constexpr (!ROWS)
#pragma unroll
                for (int j = 0; j < TM; ++j) r.a[i][j] = *(const i4v*)(a[j] + k + o16);
        }
        if (U < 4 && !scales) return;
#pragma unroll
        for (int j = 0; j < TN; ++j) r.sb[j] = *(const unsigned*)(bs[j] + g + o4);
        if constexpr (!ROWS)
#pragma unroll
            for (int j = 0; j < TM; ++j) r.sa[j] = *(const unsigned*)(as[j] + g + o4);
    };
    // Pieces of a row and 512 k, eight values to a lane; four to a wave at once, for the
    // latency of their loads, then one by one.  ENDS: 0 where K is whole pieces, 1 where
    // it ends between lanes, 2 inside a lane's eight values (a kernel fetches its code
    // as it goes, so each has its own).  Codes and scales lie as in an operand but for the
    // room, which is for R rows instead of 16, and for the place of row r's codes in
    // block j of the s-th 128 k, which is r ^ (4 s + j): a piece's blocks are written to
    // different banks.  Rows past M are whatever lies there, for rows of C that are not
    // stored.
    auto quantize = [&](auto ENDS) {
        constexpr int ends = decltype(ENDS)::value;
        const unsigned rows = (unsigned)p.M - tm * 16 < 16 ? p.M - tm * 16 : 16;
        const unsigned du = W / rows, dm = W % rows;            // from a wave's piece to its next
        unsigned u = w / rows, m = w - u * rows;
        const unsigned j = (lane >> 2) & 3, s = lane >> 4, part = lane & 3;
        const E* const x = (const E*)p.A + (uint64_t)tm * 16 * (unsigned)p.K;
        auto some = [&](auto QC) {
            constexpr int Q = decltype(QC)::value;
            typename VecOf<E, 8>::type v[Q] = {};
            unsigned to[Q], row[Q];
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                to[i] = u * 16 * R;
                row[i] = m;
                const E* const from = x + (uint64_t)m * (unsigned)p.K + 512ull * u;
                const int left = p.K - (int)(512 * u) - 8 * lane;
                if constexpr (ends == 2) v[i] = load_vec<E, 8>(from + 8u * lane, left);
                else if (ends == 0 || left > 0) v[i] = *(const typename VecOf<E, 8>::type*)(from + 8u * lane);
                u += du, m += dm;
                if (m >= rows) m -= rows, ++u;
            }
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                unsigned byte;
                const unsigned c = mx_codes_of4(v[i], byte);
                const unsigned block = (4 * s + j) * R + ((row[i] ^ (4 * s + j)) & (R - 1));
                *(unsigned*)(rc + (to[i] + block) * 16 + 4 * part) = c;
                // (all four lanes of a block have its scale byte)
                rs[to[i] + (j * R + row[i]) * 4 + s] = (char)byte;
            }
        };
        const unsigned mine = (rows * st + W - 1 - w) / W;
        unsigned n = 0;
        for (; n + 4 <= mine; n += 4) some(std::integral_constant<int, 4>{});
#pragma unroll 1
        for (; n < mine; ++n) some(std::integral_constant<int, 1>{});
    };
    auto take_rows = [&](Unit& r, unsigned u) {
        if constexpr (ROWS) {
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const unsigned t = u * U + i;
                r.a[i][0] = *(const i4v*)(rc + t * 64 * R + (oq ^ ((t & 3) * 64 & (R - 1) * 16)));
            }
            r.sa[0] = *(const unsigned*)(rs + (u * U >> 2) * 16 * R + os);
        }
    };
    Unit r;
    unsigned u = unit(0);
    if (u < units) load(r, u, true);
    if constexpr (ROWS) {
        if (p.K % 512 == 0) quantize(std::integral_constant<int, 0>{});
        else if (p.K % 8 == 0) quantize(std::integral_constant<int, 1>{});
        else quantize(std::integral_constant<int, 2>{});
        __syncthreads();
    }
    // (The copy makes the compiler wait for all of r at the end of a turn: the next unit's
    // loads overlap with this unit's MFMAs, and no more than one unit is under way.)
    for (unsigned i = 0; u < units;) {
        Unit c = r;
        const unsigned v = unit(++i);
        if (v < units) load(r, v, (i & ((1 << run) - 1)) == 0);
        take_rows(c, u);
        if constexpr (U < 4) {
            const int sh = 8 * ((u * U) & 3);
#pragma unroll
            for (int j = 0; j < TN; ++j) c.sb[j] >>= sh;
#pragma unroll
            for (int j = 0; j < TM; ++j) c.sa[j] >>= sh;
        }
        each<U>([&](auto ic) {
            constexpr int i = decltype(ic)::value;          // of the unit's U
            if (i > 0 && u * U + i >= kt) return;
#pragma unroll
            for (int y = 0; y < TM; ++y)
#pragma unroll
                for (int x = 0; x < TN; ++x)
                    acc[y][x] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                        wide(c.b[i][x]), wide(c.a[i][y]), acc[y][x], 4, 4, i, c.sb[x], i, c.sa[y]);
        });
        u = v;
    }
#pragma unroll
    for (int y = 0; y < TM; ++y)
#pragma unroll
        for (int x = 0; x < TN; ++x) red[w][y * TN + x][lane + (lane >> 4)] = acc[y][x];
    __syncthreads();
    const float lo = p.act ? 0.f : -__builtin_inff();
    // four columns of a row to a thread
#pragma unroll
    for (int t0 = 0; t0 < TM * TN * 64; t0 += 64 * W) {
        const int t = t0 + threadIdx.x, m = t / (4 * TN), q = t % (4 * TN);
        const unsigned row = tm * (16 * TM) + m, n = tn * (16 * TN) + 4 * q;
        if (t >= TM * TN * 64 || row >= (unsigned)p.M || n >= (unsigned)p.N) continue;
        const f4v* const from = &red[0][(m >> 4) * TN + (q >> 2)][17 * (q & 3) + (m & 15)];
        f4v v = from[0];
#pragma unroll
        for (int i = 1; i < W; ++i) v += from[i * TM * TN * 68];
        const int left = (int)(p.N - n < 4 ? p.N - n : 4);
        if (p.bias) {
            const auto bv = load_vec<float, 4>(p.bias + n, left);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += bv[e];
        }
        const float o[4] = {at_least(v[0], lo), at_least(v[1], lo), at_least(v[2], lo), at_least(v[3], lo)};
        store_vec<T, 4>((T*)p.C + (uint64_t)row * (unsigned)p.N + n, left, o);
    }
}

// ---------------------------------------------------------------- many rows
template <int FM, int FN>
struct MmTile {
    static constexpr int BM = 64 * FM, BN = 64 * FN;        // 2 x 2 waves of FM x FN blocks of 32 x 32
    static constexpr int TA = BM / 16, TB = BN / 16;        // row tiles
    static constexpr int STG = (TA + TB) * 1024, SCL = (TA + TB) * 256;
    static constexpr int LDS = 4 * STG + 3 * SCL;
};

template <class T, int FM, int FN>
__global__ __launch_bounds__(256, FM * FN > 8 ? 1 : 2) void k_mxmm(MmArgs p) {
    using Tl = MmTile<FM, FN>;
    constexpr int CI = FM + FN, SI = CI / 4, ITEMS = CI + SI;   // DMA instructions of a wave per 128 k
    static_assert(CI % 4 == 0 && 3 * ITEMS < 64 && (ITEMS + 1) / 2 <= CI, "whole DMA instructions per wave, vmcnt");
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
    const int kt = mx_k_tiles(p.K), st = mx_scale_tiles(p.K);
    const long long ma = mx_row_tiles(p.M) - 1 - (long long)tm * Tl::TA;
    const long long mb = mx_row_tiles(p.N) - 1 - (long long)tn * Tl::TB;
    const uint8_t* const A0 = (const uint8_t*)p.A + (long long)tm * Tl::TA * kt * 1024;
    const uint8_t* const B0 = p.B + (long long)tn * Tl::TB * kt * 1024;
    const uint8_t* const As0 = p.As + (long long)tm * Tl::TA * st * 256;
    const uint8_t* const Bs0 = p.Bs + (long long)tn * Tl::TB * st * 256;
    // offsets of this wave's row tiles, number wave + 4 t of A's TA, then of B's TB;
    // tiles past the last read the last
    unsigned oc[CI], os[CI];
#pragma unroll
    for (int t = 0; t < CI; ++t) {
        const int r = 4 * (t < FM ? t : t - FM) + wave;
        const long long last = t < FM ? ma : mb;
        const unsigned tile = (unsigned)(r < last ? r : last);
        oc[t] = tile * (unsigned)kt * 1024u;
        os[t] = tile * (unsigned)st * 256u;
    }
    // Chunk c: the codes of its 128 k into stage c % 4, and a quarter of the scales of
    // the 512 k after its own into one of three slots.  Past the end an empty buffer:
    // no memory traffic, zeros that are not multiplied, and the same count to wait for.
    auto scales = [&](int g, auto tile) {
        constexpr int t = decltype(tile)::value;
        const bool live = g < st;
        char* const to = smx + 4 * Tl::STG + g % 3 * Tl::SCL + wave * 256;
        lds_dma4(t < FM ? As0 : Bs0, live, to + t * 1024, lane * 4, os[t] + (live ? g : 0) * 256u);
    };
    auto codes = [&](int c, int stage, auto tile) {
        constexpr int t = decltype(tile)::value;
        const bool live = c < kt;
        char* const to = smx + stage * Tl::STG + wave * 1024;
        lds_dma16(t < FM ? A0 : B0, live, to + t * 4096, lane * 16, oc[t] + (live ? c : 0) * 1024u);
    };
    auto issue = [&](int c, auto stage, auto item) {
        constexpr int t = decltype(item)::value, q = decltype(stage)::value;
        if constexpr (t < CI) codes(c, q, item);
        else scales((c >> 2) + 1, std::integral_constant<int, q * SI + t - CI>{});
    };
    // zeros from an MFMA each: an eighth of the code of a move to each register
    f16v acc[FM][FN];
    const f16v zero16 = {};
    i4v zero4 = {};
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            asm volatile("" : "+v"(zero4));                 // (or one MFMA's result would be copied)
            const bf8 z = __builtin_bit_cast(bf8, zero4);
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(z, z, zero16, 0, 0, 0);
        }
    // lane l of a block: row l % 32 (tile l / 16 % 2), k-block 2 step + l / 32
    const int l16 = lane & 15, lt = (lane >> 4) & 1, lk = lane >> 5;
    const char* const ra = smx + (2 * wm * FM + lt) * 1024 + lk * 256 + l16 * 16;
    const char* const rb = smx + (Tl::TA + 2 * wn * FN + lt) * 1024 + lk * 256 + l16 * 16;
    const char* const sra = smx + 4 * Tl::STG + (2 * wm * FM + lt) * 256 + lk * 64 + l16 * 4;
    const char* const srb = smx + 4 * Tl::STG + (Tl::TA + 2 * wn * FN + lt) * 256 + lk * 64 + l16 * 4;
    i4v fa[2][FM], fb[2][FN];                               // the operands of 64 k, one step ahead
    unsigned sa[2][FM], sb[2][FN];                          // and the scales of its 512 k
    auto read = [&](auto stage, auto step, auto item) {
        constexpr int s = decltype(step)::value, at = decltype(stage)::value * Tl::STG + s * 512, t = decltype(item)::value;
        if constexpr (t < FM) fa[s][t] = *(const i4v*)(ra + at + t * 2048);
        else fb[s][t - FM] = *(const i4v*)(rb + at + (t - FM) * 2048);
    };
    auto read_scale = [&](int g, auto step, auto item) {
        constexpr int s = decltype(step)::value, t = decltype(item)::value;
        const int at = g % 3 * Tl::SCL + s * 128;
        if constexpr (t < FM) sa[s][t] = *(const unsigned*)(sra + at + t * 512);
        else sb[s][t - FM] = *(const unsigned*)(srb + at + (t - FM) * 512);
    };
    // Half of chunk c (in stage q): its MFMAs, and between them the next half's reads
    // and half of a later chunk's DMA, a few to each MFMA, so that neither their queues
    // nor the MFMAs wait.
    constexpr int H1 = (ITEMS + 1) / 2;
    auto half = [&](int c, auto Q, auto S) {
        constexpr int q = decltype(Q)::value, s = decltype(S)::value;
        constexpr int NS = (s == 1 && q == 3) || (s == 0 && q == 0) ? CI : 0;   // scales to read
        constexpr int items = NS + CI + (s == 0 ? ITEMS - H1 : H1), per = (items + FM * FN - 1) / (FM * FN);
        using Next = std::integral_constant<int, (q + s) & 3>;                  // the next half's stage and step
        using Step = std::integral_constant<int, s ^ 1>;
        each<FM * FN>([&](auto K) {
            constexpr int k = decltype(K)::value, i = k / FN, j = k % FN;
            acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wide(fb[s][j]), wide(fa[s][i]), acc[i][j], 4, 4,
                                                                       q, sb[s][j], q, sa[s][i]);
            each<per>([&](auto P) {
                constexpr int t = k * per + decltype(P)::value;
                if constexpr (t < NS)
                    read_scale((c >> 2) + s, Step{}, std::integral_constant<int, t>{});
                else if constexpr (t < NS + CI)
                    read(Next{}, Step{}, std::integral_constant<int, t - NS>{});
                else if constexpr (t < items && s == 1)
                    issue(c + 4, Q, std::integral_constant<int, t - NS - CI>{});
                else if constexpr (t < items)
                    issue(c + 3, std::integral_constant<int, (q + 3) & 3>{},
                          std::integral_constant<int, H1 + t - NS - CI>{});
            });
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    using Zero = std::integral_constant<int, 0>;
    using One = std::integral_constant<int, 1>;
    // The scales of two groups, and 3 1/2 chunks as the loop issues them: with as many
    // instructions each (in a rolled loop, so a chunk brings scales that are there
    // already), for the loop's waits count them.
    each<CI>([&](auto i) { scales(0, i); });
    each<CI>([&](auto i) { scales(1, i); });
#pragma unroll 1
    for (int c = 0; c < 3; ++c) {
        each<CI>([&](auto i) { codes(c, c, i); });
        each<SI>([&](auto i) { scales(1, i); });
    }
    each<H1>([&](auto i) { codes(3, 3, i); });
    __builtin_amdgcn_s_waitcnt(vm_count(2 * ITEMS + H1));
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    each<CI>([&](auto i) { read_scale(0, Zero{}, i); });
    each<CI>([&](auto i) { read(Zero{}, Zero{}, i); });
    // Chunk c + q, in stage q.  Between its halves it is in registers, everyone's, and
    // its stage is free; the next chunk has landed once the two after it are all that
    // is outstanding.
    float bias[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const long long n = (long long)tn * Tl::BN + (wn * FN + j) * 32 + lane;
        bias[j] = p.bias && lane < 32 && n < p.N ? p.bias[n] : 0.f;
    }
    int c = 0;
    do {
        each<4>([&](auto Q) {
            constexpr int q = decltype(Q)::value;
            if (q > 0 && c + q >= kt) return;
            half(c + q, Q, Zero{});
            __builtin_amdgcn_s_waitcnt(vm_count(2 * ITEMS));
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            half(c + q, Q, One{});
        });
        c += 4;
    } while (c < kt);
    // Lane l, register e of a block: row l % 32, column 8 (e / 4) + 4 (l / 32) + e % 4.
    // A wave turns its results around in LDS, for stores of
    // whole cache lines.  16 bytes between rows: 8 lanes' writes fall on different banks.
    __builtin_amdgcn_s_waitcnt(vm_count(0));                // the chunks past the end
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (p.bias) {
        // an fp32 MFMA of the bias and 1 (one of its two k is 0): exact
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(bias[j], lane < 32 ? 1.f : 0.f, acc[i][j], 0, 0, 0);
    }
    const float lo = p.act ? 0.f : -__builtin_inff();
    constexpr int CV = 16 / (int)sizeof(T), LPR = 32 * FN / CV, RPI = 64 / LPR;   // columns to a lane, lanes to a row
    constexpr int RS = 32 * FN + CV, SLABS = sizeof(T) == 4 ? (FM + 1) / 2 : FM;
    static_assert(4 * SLABS * 32 * RS * sizeof(T) <= Tl::LDS && FM % SLABS == 0, "LDS");
    typedef T t4 __attribute__((ext_vector_type(4)));
    typedef T tv __attribute__((ext_vector_type(CV)));
    typedef typename VecOf<T, CV>::type tvu;
    T* const slab = (T*)smx + wave * SLABS * 32 * RS;
    const long long n0 = (long long)tn * Tl::BN + wn * 32 * FN, m0 = (long long)tm * Tl::BM + wm * 32 * FM;
    const int cl = lane % LPR * CV;                         // this lane's columns, and how many of them there are
    const int left = n0 + cl < p.N ? (int)(p.N - n0 - cl < CV ? p.N - n0 - cl : CV) : 0;
    each<FM / SLABS>([&](auto G) {
        constexpr int g = decltype(G)::value * SLABS;
        each<SLABS * FN * 4>([&](auto E) {
            constexpr int i = decltype(E)::value / (4 * FN), j = decltype(E)::value / 4 % FN, h = decltype(E)::value % 4;
            t4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)at_least(acc[g + i][j][4 * h + e], lo);
            *(t4*)(slab + (32 * i + (lane & 31)) * RS + 32 * j + 8 * h + 4 * lk) = v;
        });
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const long long m = m0 + 32 * g;
        const int rows = p.M - m < 32 * SLABS ? (int)(p.M - m) : 32 * SLABS;
        T* const C = (T*)p.C + m * p.N + n0;
        if (left == CV)
#pragma unroll 8
            for (int r = lane / LPR; r < rows; r += RPI)
                __builtin_nontemporal_store(*(const tv*)(slab + r * RS + cl), (tvu*)(C + (size_t)r * p.N + cl));
        else if (left > 0)                                  // the last columns
#pragma unroll 1
            for (int r = lane / LPR; r < rows; r += RPI)
                for (int e = 0; e < left; ++e) C[(size_t)r * p.N + cl + e] = slab[r * RS + cl + e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    });
}

template <class T, class X, int TM, int TN, int W, int U>
bool launch_few(MmArgs a, hipStream_t s) {
    // set once per process, thread-safely, before any launch below
    static const bool attr = [] {
        (void)hipFuncSetAttribute((const void*)k_mxmm_few<T, X, TM, TN, W, U>,
                                  hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
        return true;
    }();
    (void)attr;
    a.gm = (int)((mx_row_tiles(a.M) + TM - 1) / TM);
    a.gn = (int)((mx_row_tiles(a.N) + TN - 1) / TN);
    a.rows = few_rows(a.M);
    const long long grid = xcd_groups((long long)a.gm * a.gn);
    ACFUN_LAUNCH("k_mxmm_few", (k_mxmm_few<T, X, TM, TN, W, U>), dim3((unsigned)grid), dim3(64 * W),
                 (kFewSums<TM, TN, W> + (std::is_void_v<X> ? 0 : few_rows_lds(a.M, a.K))), s, a);
    return check_launch("k_mxmm_few");
}

template <class T, int FM, int FN>
bool launch_many(MmArgs a, hipStream_t s) {
    using Tl = MmTile<FM, FN>;
    static_assert(Tl::LDS <= kLds, "LDS");
    // set once per process, thread-safely, before any launch below
    static const bool attr = [] {
        (void)hipFuncSetAttribute((const void*)k_mxmm<T, FM, FN>, hipFuncAttributeMaxDynamicSharedMemorySize, Tl::LDS);
        return true;
    }();
    (void)attr;
    a.gm = (int)(((long long)a.M + Tl::BM - 1) / Tl::BM);
    a.gn = (int)(((long long)a.N + Tl::BN - 1) / Tl::BN);
    const long long grid = xcd_groups((long long)a.gm * a.gn);
    ACFUN_LAUNCH("k_mxmm", (k_mxmm<T, FM, FN>), dim3((unsigned)grid), dim3(256), Tl::LDS, s, a);
    return check_launch("k_mxmm");
}

}  // namespace

bool mx_gemm(int M, int N, int K, const uint8_t* A, const uint8_t* As, const uint8_t* B, const uint8_t* Bs,
             void* C, int type, const float* bias, int act, hipStream_t s) {
    const MmArgs a{M, N, K, A, As, B, Bs, C, bias, act, 0, 0};
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        double us;
        switch (mm_choose(M, N, K, num_cus(), us)) {
            case FEW16: return launch_few<T, void, 1, 1, 8, 4>(a, s);
            case FEW32: return launch_few<T, void, 2, 2, 4, 2>(a, s);
            case FEW64: return launch_few<T, void, 4, 4, 8, 1>(a, s);
            case MANY128: return launch_many<T, 2, 2>(a, s);
            default: return launch_many<T, 4, 4>(a, s);
        }
    });
}

bool mx_fc(const void* x, int type, int M, int K, const uint8_t* B, const uint8_t* Bs, const float* bias,
           int N, void* C, int act, hipStream_t s) {
    if (K > 0) {
        const FcPlan plan = fc_plan(M, N, K, type_size(type), num_cus());
        bool one = plan.one;
        if (!one) {
            // a graph would keep the addresses of temporaries that go back to the pool here
            hipStreamCaptureStatus captured = hipStreamCaptureStatusNone;
            if (!check(hipStreamIsCapturing(s, &captured), "hipStreamIsCapturing")) return false;
            one = captured != hipStreamCaptureStatusNone;
            if (one && !plan.captured) {
                set_error("acfun_dev_fc_mxfp4: these sizes need temporaries, which a graph cannot keep: capture "
                          "acfun_dev_quantize_mxfp4 and acfun_dev_gemm_mxfp4 with buffers of the caller's");
                return false;
            }
        }
        if (one) {
            const MmArgs a{M, N, K, x, nullptr, B, Bs, C, bias, act, 0, 0};
            return with_type(type, [&](auto t) {
                using T = decltype(t);
                if (plan.tn == 1) return launch_few<T, T, 1, 1, 8, 4>(a, s);
                if (plan.tn == 2) return launch_few<T, T, 1, 2, 8, 4>(a, s);
                return launch_few<T, T, 1, 4, 8, 2>(a, s);
            });
        }
    }
    Scratch codes(mx_code_bytes(M, K), s), scales(mx_scale_bytes(M, K), s);
    if (K > 0 && (!codes.p || !scales.p)) return false;
    return (K == 0 || mx_quantize(x, type, M, K, 0, codes.as<uint8_t>(), scales.as<uint8_t>(), s)) &&
           mx_gemm(M, N, K, codes.as<uint8_t>(), scales.as<uint8_t>(), B, Bs, C, type, bias, act, s);
}

}  // namespace acfun
