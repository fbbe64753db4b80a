// k_sample.hip -- a token drawn from each row of logits.
//
//   w_i = exp((x_i - max x) / T),  tokens in order of x, the lower index first of equals;
//   kept: the first k; of these the fewest whose weights reach p of theirs; of these
//   w_i >= m.  The token is the first in order of index with sum_{j <= i} w_j > u sum w.
//
// Weights are 64-bit integers, multiples of 2^-f with f so that a row's sum fits (45 for
// 2^17 columns, 48 at most), from an exponential in 64 bits: sums do not depend on their order.
// Half a step of each weight and the exponential's 2^-39.8 of it leave a row's shares, and
// with them the borders that u and a nucleus are compared with, off by cols 2^-(f+1) + 2^-38.8 at
// most: 2^-28.9 for 2^17 columns, 2^-24.9 for 2^19 and more.  Past 2^19 columns f is taken
// from the row's own sum, in a pass of its own (1 x 2^20 fp32 with a nucleus 59 us, 50 without
// it; where the border's bin has more tokens than a list, one workgroup does the row again: 1.8 ms).
// No row is sorted.  The kept tokens are those not below one of them, the cut, in the
// order; it lies in a bin of a histogram over x whose tokens alone are put in order.  Bins are
// even in x / T, 59 to a factor of e, so that most rows spread over many.  A top-k's
// tokens, or a nucleus's, that are few are all taken out of the row, and the rest is done
// with these.
//
// A row is read three to five times from the caches, and a few rows wait for what follows one
// another: 64 x 32003 bf16 takes 7.5 us for the largest, 15.7 with a temperature, 23 with a top-k,
// 33 with a nucleus, 27 with all; 64 x 1000 fp32 3.7, 4.8, 8, 12 and 13.  A captured call has one
// workgroup to any row: 1 x 131072 fp32 with all settings 40 us, 24 in parts.  Many rows are bound by the
// instructions of a weight, the exponential in 64 bits above all: 512 x 131072 fp32 with a
// nucleus takes 207 us, half of it the one pass with weights; the first, from memory, 46.
#include <type_traits>

#include "q8.hpp"

namespace acfun {
namespace {

typedef unsigned long long u64;

// The order of the values as one of integers, equal for +0 and -0; 0 for those that are
// never drawn, NaN and -infinity.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return x > -__builtin_inff() ? (b >> 31 ? ~b : b | 0x80000000u) : 0u;
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}
// What all lanes have, in scalar registers.
__device__ __forceinline__ unsigned same(unsigned v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ u64 same(u64 v) { return (u64)same((unsigned)(v >> 32)) << 32 | same((unsigned)v); }
// A value of 4 or 8 bytes from another lane: by DPP (lanes without a source, and rows not in
// ROWS, get 0), and a lane's for all.  Sums by DPP take a third of the time that they do
// through LDS.
template <int CTRL, int ROWS = 15, class V>
__device__ __forceinline__ V dpp(V v) {
    if constexpr (sizeof(V) == 8)
        return (V)dpp<CTRL, ROWS>((unsigned)((u64)v >> 32)) << 32 | dpp<CTRL, ROWS>((unsigned)v);
    else
        return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 15, false));
}
template <class V>
__device__ __forceinline__ V from_lane(V v, int lane) {
    if constexpr (sizeof(V) == 8)
        return (V)from_lane((unsigned)((u64)v >> 32), lane) << 32 | from_lane((unsigned)v, lane);
    else
        return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ u64 lanes_of(bool b) { return __builtin_amdgcn_ballot_w64(b); }
// The lanes of a set that are before this one.
__device__ __forceinline__ unsigned before_in(u64 lanes) {
    return __builtin_amdgcn_mbcnt_hi((unsigned)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)lanes, 0));
}
// f over the first N lanes of each 16, in these lanes.
template <int N, class V, class F>
__device__ __forceinline__ V row_all(V v, F f) {
    if constexpr (N > 1) v = f(v, dpp<0xb1>(v));            // lane ^ 1
    if constexpr (N > 2) v = f(v, dpp<0x4e>(v));            // lane ^ 2
    if constexpr (N > 4) v = f(v, dpp<0x141>(v));           // 7 - lane, of each 8
    if constexpr (N > 8) v = f(v, dpp<0x140>(v));           // 15 - lane
    return v;
}
// A token's place in the order, the first the largest.
__device__ __forceinline__ u64 place_of(float x, int i) { return (u64)key_of(x) << 32 | (unsigned)~i; }

// A cut below all that can be drawn: any index with the lowest finite value.
constexpr u64 kNoCut = (u64)0x00800000 << 32;
// Whether a token is not below a cut.
struct Cut {
    float x;
    unsigned i;
    __device__ __forceinline__ explicit Cut(u64 place) : x(value_of(place >> 32)), i(~(unsigned)place) {}
    __device__ __forceinline__ bool keeps(float v, int at) const { return (v > x) | ((v == x) & ((unsigned)at <= i)); }
};

// 2^f, |f| <= 1/2, by the polynomial through it at nine Chebyshev points, off by 1.1e-12 of the
// value at most.
struct Exp2 {
    double k[8];
    __device__ __forceinline__ Exp2()
        : k{0x1.62e42fef84cf0p-1, 0x1.ebfbdff823cedp-3, 0x1.c6b08dd6fd236p-5,  0x1.3b2ab7181b77dp-7,
            0x1.5d8745a728209p-10, 0x1.4308ac85a69f8p-13, 0x1.00dc4a5344ef5p-16, 0x1.63d1363a681b4p-20} {
#pragma unroll
        for (int i = 0; i < 8; ++i) asm("" : "+s"(k[i]));       // (or each use would copy them)
    }
    __device__ __forceinline__ double operator()(double f) const {
        double p = k[7];
#pragma unroll
        for (int i = 6; i >= 0; --i) p = __builtin_fma(p, f, k[i]);
        return __builtin_fma(p, f, 1.);
    }
};

struct Weights {
    double max, least, c;                       // c: log2(e) / T
    float top, half_top, per_2x;                // the largest value; bins to two units of x
    unsigned bins;
    int frac;
    Exp2 exp2;
    // `bins` for the 50 powers of two that weigh.  No infinities, whose differences and products
    // are none: a temperature is 2^1000 at most, an infinite top is 2^128 (which it is not below,
    // and finite values are far from at the temperature 1, as they are to be at any).
    __device__ __forceinline__ Weights(float largest, float T, int f, int n) {
        const bool inf = largest == __builtin_inff();
        top = largest;
        half_top = 0.5f * top;
        max = inf ? 0x1p128 : (double)top;
        const double t = T < __builtin_inff() ? (double)T : 0x1p1000;
        c = inf ? 1. : 0x1.71547652b82fep+0 / t;
        least = inf ? -1000. : -1000. * 0x1.62e42fefa39efp-1 * t;           // -1000 / c
        per_2x = __builtin_fminf((float)n * (float)(0x1.715476p+0 / 25.) / T, 1e30f);
        bins = (unsigned)n;
        frac = f;
    }
    // In steps of 2^-f.  2^t = 2^n 2^f with n in the low bits of a number that has no others
    // below 1, added to the exponent; the result's steps again in such low bits.  2^-1000 and less
    // (-infinity, NaN) is 0 of them.
    __device__ __forceinline__ u64 operator()(float x) const {
        const double d = __builtin_fmin(__builtin_fmax((double)x - max, least), 0.);
        const double z = __builtin_fma(d, c, 0x1.8p52), f = __builtin_fma(d, c, 0x1.8p52 - z);
        const u64 p = __builtin_bit_cast(u64, exp2(f));
        const unsigned hi = (unsigned)(p >> 32) + (((unsigned)__builtin_bit_cast(u64, z) + (unsigned)frac) << 20);
        const double w = __builtin_bit_cast(double, (u64)hi << 32 | (unsigned)p) + 0x1p52;
        return __builtin_bit_cast(u64, w) & 0xfffffffffffffull;
    }
    // The weight itself, however small.
    __device__ __forceinline__ double real(float x) const {
        const double t = __builtin_fmin(__builtin_fmax(((double)x - max) * c, -4096.), 0.);
        return __builtin_amdgcn_ldexp(exp2(t - __builtin_rint(t)), (int)__builtin_rint(t));
    }
    __device__ __forceinline__ double one() const { return __builtin_amdgcn_ldexp(1., frac); }
    // from 0 for the largest value up; `bins`: no weight (so for a NaN or -infinity)
    __device__ __forceinline__ unsigned bin(float x) const {
        const float b = __builtin_fmaf(x, -0.5f, half_top) * per_2x;    // (top - x may pass fp32)
        const unsigned at = (unsigned)__builtin_fminf(b, (float)bins);
        return x == top ? 0u : at;                                      // (both infinite, b is none)
    }
    // The least key whose weight is m or more, in (0, 1]: 64 candidates at once.
    __device__ __forceinline__ unsigned least_key(double m) const {
        unsigned lo = key_of(-0x1.fffffep+127f), hi = key_of(top);
        while (lo < hi) {
            const unsigned lane = threadIdx.x & 63, k = lo + (unsigned)((u64)(hi - lo) * lane >> 6);
            const u64 past = lanes_of(real(value_of(k)) >= m);
            const int s = past ? __ffsll(past) - 1 : 64;
            if (s < 64) hi = from_lane(k, s);
            if (s > 0) lo = from_lane(k, s - 1) + 1;
        }
        return hi;
    }
};

// Up to so many tokens of a bin count those before them, each all the others.
constexpr int kSome = 256;

// A workgroup's: two bins and two entries of the list to a thread.
template <int NT>
struct Shared {
    static constexpr int kWaves = NT / 64, kBins = 2 * NT, kList = 2 * NT;
    u64 mass[kBins];
    u64 list[kList], some[kSome], some_mass[kSome], some_before[kSome];
    u64 part[kWaves];
    unsigned count[kBins];
    unsigned n, bin;
    u64 above;
};

struct Max { template <class V> __device__ V operator()(V a, V b) const { return a > b ? a : b; } };
struct Min { template <class V> __device__ V operator()(V a, V b) const { return a < b ? a : b; } };
struct Add { template <class V> __device__ V operator()(V a, V b) const { return a + b; } };

template <class V, class F>
__device__ __forceinline__ V wave_all(V v, F f) {
    v = row_all<16>(v, f);
    return f(f(from_lane(v, 0), from_lane(v, 16)), f(from_lane(v, 32), from_lane(v, 48)));
}
template <int NT, class V, class F>
__device__ __forceinline__ V block_all(V v, Shared<NT>& sm, F f) {
    typedef std::conditional_t<sizeof(V) == 8, u64, unsigned> U;
    v = wave_all(v, f);
    if ((threadIdx.x & 63) == 0) sm.part[threadIdx.x >> 6] = __builtin_bit_cast(U, v);
    __syncthreads();
    v = __builtin_bit_cast(V, (U)sm.part[threadIdx.x % (NT / 64)]);
    __syncthreads();
    return from_lane(row_all<NT / 64>(v, f), 0);
}
// The sum over the lanes up to and with this one, of the wave and of the block.
__device__ __forceinline__ u64 wave_upto(u64 v) {
    v += dpp<0x111>(v);                                     // lane - 1, 2, 4, 8 of a row of 16
    v += dpp<0x112>(v);
    v += dpp<0x114>(v);
    v += dpp<0x118>(v);
    v += dpp<0x142, 10>(v);                                 // rows 1 and 3: the row before's last lane
    return v + dpp<0x143, 12>(v);                           // rows 2 and 3: lane 31
}
template <int NT>
__device__ __forceinline__ u64 block_upto(u64 v, Shared<NT>& sm, u64& total) {
    constexpr int W = NT / 64;
    v = wave_upto(v);
    if ((threadIdx.x & 63) == 63) sm.part[threadIdx.x >> 6] = v;
    __syncthreads();
    const u64 waves = wave_upto((int)(threadIdx.x & 63) < W ? sm.part[threadIdx.x % W] : 0);
    total = from_lane(waves, W - 1);
    const int w = (int)same(threadIdx.x >> 6);
    const u64 before = from_lane(waves, w ? w - 1 : 0);
    __syncthreads();
    return w ? v + before : v;
}

// A row's values, 16 bytes of them to a lane, to f(x, index).
template <class T>
struct Row {
    static constexpr int V = 16 / (int)sizeof(T);
    typedef typename VecOf<T, V>::type VT;
    struct Some {
        VT v;
        int i;                                  // the first one's index
    };
    const T* x;
    int cols;
    // V values from index i; at the row's end its last V, those before i as -infinity
    __device__ __forceinline__ Some load(int i) const {
        if (i + V <= cols) return {*(const VT*)(x + i), i};
        if (cols < V) return {load_vec<T, V>(x + i, cols - i, -__builtin_inff()), i};
        Some s{*(const VT*)(x + cols - V), cols - V};
#pragma unroll
        for (int e = 0; e < V; ++e) s.v[e] = s.i + e < i ? (T)-__builtin_inff() : s.v[e];
        return s;
    }
    // from i0 to i1, apart by whole 64 V or at the row's end, by lanes t of `threads`: to
    // f(x, i) B neighbours at once, the first one's index i.  (One copy of f for each: what runs
    // a few times is fetched as it runs.)
    static constexpr int B = 4;
    template <int U, class F>
    __device__ __forceinline__ void fours(int i0, int i1, int t, int threads, F f) const {
        int i = i0 + t * V;
        const int step = threads * V;
        if constexpr (U > 1)
#pragma unroll 1
            for (; i + (U - 1) * step + V <= i1; i += U * step) {
                VT v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) v[u] = *(const VT*)(x + i + u * step);
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int g = 0; g < V; g += B) {
                        float y[B];
#pragma unroll
                        for (int e = 0; e < B; ++e) y[e] = (float)v[u][g + e];
                        f(y, i + u * step + g);
                    }
            }
        if (i >= i1) return;
        Some s = load(i);
#pragma unroll 1
        for (;; i += step) {
            const Some c = s;
            const bool more = i + step < i1;
            if (more) s = load(i + step);
#pragma unroll
            for (int g = 0; g < V; g += B) {
                float x[B];
#pragma unroll
                for (int e = 0; e < B; ++e) x[e] = (float)c.v[g + e];
                f(x, c.i + g);
            }
            if (!more) return;
        }
    }
    // one by one
    template <int U = 1, class F>
    __device__ __forceinline__ void each(int i0, int i1, int t, int threads, F f) const {
        fours<U>(i0, i1, t, threads, [&](const float (&x)[B], int i) {
#pragma unroll
            for (int e = 0; e < B; ++e) f(x[e], i + e);
        });
    }
};

// The first bin up to and with which the bins hold `need` (at least 1); those before it
// hold sm.above.  False if all of them hold less.
template <int NT, class V>
__device__ __forceinline__ bool find_bin(const V* bins, u64 need, Shared<NT>& sm) {
    const int t = threadIdx.x, b0 = 2 * t, b1 = b0 + 1;
    const u64 first = bins[b0], mine = first + bins[b1];
    if (t == 0) sm.bin = 2 * NT;
    u64 total;
    const u64 above = block_upto(mine, sm, total) - mine;
    if (above < need && need <= above + mine) {
        const bool zero = above + first >= need;
        sm.bin = zero ? b0 : b1;
        sm.above = zero ? above : above + first;
    }
    __syncthreads();
    return sm.bin < 2 * NT;
}

// What the histogram says of a row's first k (0: all) and p (1 or more: all): the bin that
// the next cut lies in, and whether the tokens up to it are few enough to take them all.
struct Plan {
    bool by_count, cut, take;                   // cut: there is one
    unsigned bin;
    u64 need, above;
    unsigned lo = ~0u, hi = 0;                  // the bins of the list
};

template <class T, int NT>
struct Draw {
    static constexpr int kWaves = NT / 64, kBins = 2 * NT, kList = 2 * NT, kLoads = NT == 1024 && sizeof(T) == 4 ? 2 : 1;
    static constexpr int kFew = kLoads == 2 ? 4 : 1;    // loads where nothing else needs registers
    const Row<T> row;
    const Weights w;
    Shared<NT>& sm;
    int* const token;
    float* const prob;
    const float u, m;                           // m: min_p

    // The cut, or min_p's where that is above it.
    __device__ __forceinline__ u64 with_floor(u64 cut) const {
        if (!(m > 0.f)) return cut;
        const u64 floor = (u64)w.least_key(m < 1.f ? (double)m : 1.) << 32;
        return same(floor > cut ? floor : cut);
    }
    template <class F>
    __device__ __forceinline__ void all(F f) const { row.each(0, row.cols, threadIdx.x, NT, f); }
    __device__ __forceinline__ void clear() const {
        sm.mass[threadIdx.x] = sm.mass[threadIdx.x + NT] = 0;
        sm.count[threadIdx.x] = sm.count[threadIdx.x + NT] = 0;
        if (threadIdx.x == 0) sm.n = 0;
        __syncthreads();
    }
    // The cut in bin b: the first place of its tokens, in order, up to and with which their
    // number or mass, `before` with what the earlier bins hold, is `need`.  For bins of
    // any size: by its digits, a pass for each.
    template <bool MASS>
    __device__ __forceinline__ u64 cut_by_digits(unsigned b, u64 need, u64 before) const {
        u64 prefix = 0;
        constexpr int D = NT == 1024 ? 11 : NT == 512 ? 10 : 9;
        static_assert(1 << D <= kBins, "a bin to each digit");
#pragma unroll 1
        for (int shift = 64 - D;;) {
            const int width = shift == 0 ? (64 - 1) % D + 1 : D;
            clear();
            all([&](float x, int i) {
                if (w.bin(x) != b) return;
                const u64 p = place_of(x, i);
                if (shift < 64 - D && p >> (shift + width) != prefix) return;
                const unsigned d = (1u << width) - 1 - ((unsigned)(p >> shift) & ((1u << width) - 1));   // the largest first
                if constexpr (MASS) atomicAdd(&sm.mass[d], w(x));
                else atomicAdd(&sm.count[d], 1u);
            });
            __syncthreads();
            if constexpr (MASS) find_bin(sm.mass, need - before, sm);
            else find_bin(sm.count, need - before, sm);
            prefix = prefix << width | ((1u << width) - 1 - same(sm.bin));
            before += same(sm.above);
            __syncthreads();
            if (shift == 0) return prefix;
            shift = shift > D ? shift - D : 0;
        }
    }
    // The same of a bin whose tokens are among the list's n.  While they are more than kSome, a
    // histogram over their places narrows them; then each adds up those before it, with
    // NT / kSome threads.
    __device__ __forceinline__ u64 cut_in_list(int n, unsigned b, bool mass, u64 need, u64 before) const {
        const int t = threadIdx.x;
        u64 lo = 0, hi = ~0ull;
        unsigned m;
#pragma unroll 1
        for (;;) {
            if (t == 0) sm.n = 0;
            if (t < kSome) sm.some_before[t] = 0;
            __syncthreads();
            u64 least = ~0ull, most = 0;
            each_listed(n, [&](float x, int i) {
                const u64 p = place_of(x, i);
                if (w.bin(x) != b || p < lo || p > hi) return;
                const unsigned at = atomicAdd(&sm.n, 1u);
                if (at < (unsigned)kSome) sm.some[at] = p, sm.some_mass[at] = mass ? w(x) : 1;
                least = p < least ? p : least;
                most = p > most ? p : most;
            });
            __syncthreads();
            m = sm.n;
            if (m <= (unsigned)kSome) break;
            lo = block_all(least, sm, Min{});
            hi = block_all(most, sm, Max{});
            int shift = 0;
            while ((hi - lo) >> shift >= (u64)kBins) ++shift;
            clear();
            each_listed(n, [&](float x, int i) {
                const u64 p = place_of(x, i);
                if (p >= lo && p <= hi) atomicAdd(&sm.mass[(hi - p) >> shift], mass ? w(x) : 1ull);
            });
            __syncthreads();
            find_bin(sm.mass, need - before, sm);
            before += sm.above;
            hi -= (u64)sm.bin << shift;
            const u64 last = (1ull << shift) - 1;
            lo = hi - lo > last ? hi - last : lo;
            __syncthreads();
        }
        const int e = t % kSome;
        const u64 mine = e < (int)m ? sm.some[e] : 0;
        if (mine) {
            u64 sum = 0;
#pragma unroll 2
            for (int j = t / kSome; j < (int)m; j += NT / kSome) sum += sm.some[j] > mine ? sm.some_mass[j] : 0;
            if (sum) atomicAdd(&sm.some_before[e], sum);
        }
        __syncthreads();
        if (t < (int)m) {
            before += sm.some_before[t];
            if (before < need && need <= before + sm.some_mass[t]) sm.above = mine;
        }
        __syncthreads();
        const u64 c = same(sm.above);
        __syncthreads();
        return c;
    }
    // The part p of a mass, in steps, at least one.
    __device__ __forceinline__ u64 share(float p, u64 of) const {
        const double want = __builtin_ceil((double)p * (double)of);
        return want >= 1. ? (u64)want : 1;
    }
    __device__ __forceinline__ u64 target_of(u64 total) const {
        const double at = (double)(u > 0.f ? u < 1.f ? u : 0x1.fffffep-1f : 0.f) * (double)total;
        return (u64)at < total ? (u64)at : total - 1;
    }
    __device__ __forceinline__ void put(int i, float x, u64 total) const {
        *token = i;
        if (prob) *prob = (float)(w.real(x) * w.one() / (double)total);
    }
    template <class F>
    __device__ __forceinline__ void each_listed(int n, F f) const {
#pragma unroll 1
        for (int i = threadIdx.x; i < n; i += NT) {
            const u64 p = sm.list[i];
            f(value_of(p >> 32), ~(int)p);
        }
    }

    // Draws from the list's n tokens that are not below the cut: a histogram over the index, then
    // the tokens of a bin.
    __device__ __forceinline__ void from_listed(int n, u64 cut) const {
        const int t = threadIdx.x;
        int shift = 0;
        while ((row.cols - 1) >> shift >= kBins) ++shift;
        clear();
        each_listed(n, [&](float x, int i) {
            if (place_of(x, i) >= cut) atomicAdd(&sm.mass[i >> shift], w(x));
        });
        __syncthreads();
        const u64 total = block_all(sm.mass[2 * t] + sm.mass[2 * t + 1], sm, Add{}), target = target_of(total);
        if (__builtin_expect(target == 0, 0)) { // u = 0: the first kept, however small its weight
            u64 first = ~0ull;
            each_listed(n, [&](float x, int i) {
                const u64 at = (u64)(unsigned)i << 32 | __float_as_uint(x);
                if (at < first && place_of(x, i) >= cut && w.real(x) > 0.) first = at;
            });
            first = block_all(first, sm, Min{});
            if (t == 0) put((int)(first >> 32), __uint_as_float((unsigned)first), total);
            return;
        }
        find_bin(sm.mass, target + 1, sm);
        const unsigned bin = sm.bin;
        u64 before = sm.above;
        if (t == 0) sm.n = 0;
        __syncthreads();
        each_listed(n, [&](float x, int i) {
            if ((unsigned)i >> shift != bin || place_of(x, i) < cut) return;
            const unsigned at = atomicAdd(&sm.n, 1u);
            if (at < kSome) sm.some[at] = (u64)(unsigned)i << 32 | __float_as_uint(x), sm.some_mass[at] = w(x);
        });
        __syncthreads();
        const int m = (int)sm.n;
        if (m <= kSome) {
            if (t >= m) return;
            const u64 mine = sm.some[t];
#pragma unroll 1
            for (int j = 0; j < m; ++j) before += sm.some[j] < mine ? sm.some_mass[j] : 0;
            if (before <= target && target < before + sm.some_mass[t])
                put((int)(mine >> 32), __uint_as_float((unsigned)mine), total);
            return;
        }
        const int i0 = (int)bin << shift, i1 = i0 + (1 << shift) < row.cols ? i0 + (1 << shift) : row.cols;
#pragma unroll 1
        for (int i = i0; i < i1; i += NT) {
            const float x = i + t < i1 ? (float)row.x[i + t] : -__builtin_inff();
            const u64 v = Cut(cut).keeps(x, i + t) ? w(x) : 0;
            u64 all;
            const u64 upto = before + block_upto(v, sm, all);
            if (upto > target && upto - v <= target) put(i + t, x, total);
            before += all;
        }
    }

    // The mass of the tokens a to b not below the cut, in every lane of a wave.
    __device__ __forceinline__ u64 kept_mass(int a, int b, u64 cut, int t, int threads) const {
        const Cut c(cut);
        u64 mass = 0;
        row.template fours<kLoads>(a, b, t, threads, [&](const float (&x)[4], int i) {
            u64 m[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) m[e] = w(x[e]);
#pragma unroll
            for (int e = 0; e < 4; ++e) mass += c.keeps(x[e], i + e) ? m[e] : 0;
        });
        return wave_all(mass, Add{});
    }
    // The mass of all tokens i0 to i1.
    __device__ __forceinline__ u64 mass_of(int i0, int i1) const {
        const u64 mass = kept_mass(i0, i1, kNoCut, threadIdx.x, NT);
        return block_all((threadIdx.x & 63) == 0 ? mass : 0, sm, Add{});
    }
    // A wave's run of the tokens i0 to i1: whole loads of a wave.
    static constexpr int kWaveLoad = 64 * Row<T>::V;
    static __device__ __forceinline__ int run_of(int i0, int i1) {
        return ((i1 - i0 + kWaves - 1) / kWaves + kWaveLoad - 1) / kWaveLoad * kWaveLoad;
    }
    // Draws from the tokens i0 to i1 not below the cut, those before them having the mass
    // `before` of all tokens' `total` (0: it is that of these).  `runs`: sm.part has the masses of
    // the waves' runs.  k: the row's top_k, which the cut does not hold where fewer tokens have a bin.
    __device__ __forceinline__ void from_row(int i0, int i1, u64 cut, u64 before, u64 total, bool runs, int k) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        u64 target = total ? target_of(total) : 1;
        // a run to each wave, then a part of the run that the target falls in
#pragma unroll 1
        for (; target; runs = false) {
            const int per = run_of(i0, i1);
            if (!runs) {
                const int a = i0 + wave * per < i1 ? i0 + wave * per : i1, b = a + per < i1 ? a + per : i1;
                const u64 mass = kept_mass(a, b, cut, lane, 64);
                if (lane == 0) sm.part[wave] = mass;
                __syncthreads();
            }
            const u64 upto = wave_upto(lane < kWaves ? sm.part[lane % kWaves] : 0);
            if (!total) total = from_lane(upto, kWaves - 1), target = target_of(total);
            const u64 past = lanes_of(lane < kWaves && before + upto > target);
            const int s = past ? __ffsll(past) - 1 : kWaves - 1;
            before += s ? from_lane(upto, s - 1) : 0;
            __syncthreads();
            i0 += s * per;
            i1 = i0 + per < i1 ? i0 + per : i1;
            if (per == kWaveLoad) break;
        }
        if (__builtin_expect(target == 0, 0)) { // u = 0: the first kept, however small its weight
            if (k > 0) {                        // (so also among those of the first k without a bin)
                unsigned binned = 0;
                all([&](float x, int) { binned += w.bin(x) < (unsigned)kBins; });
                binned = same(block_all(binned, sm, Add{}));
                if (binned < (unsigned)k) {
                    const u64 last = cut_by_digits<false>(kBins, (u64)k, binned);
                    cut = last > cut ? last : cut;
                }
            }
            const Cut c(cut);
            int first = row.cols;
            all([&](float x, int i) {
                if (i < first && c.keeps(x, i) && w.real(x) > 0.) first = i;
            });
            __syncthreads();
            first = block_all(first, sm, Min{});
            if (threadIdx.x == 0) put(first, (float)row.x[first], total);
            return;
        }
        if (wave) return;
        const auto v = row.load(i0 + lane * Row<T>::V < row.cols ? i0 + lane * Row<T>::V : row.cols);
        u64 m[Row<T>::V], mine = 0;
#pragma unroll
        for (int e = 0; e < Row<T>::V; ++e) {
            m[e] = v.i + e < i1 && Cut(cut).keeps((float)v.v[e], v.i + e) ? w((float)v.v[e]) : 0;
            mine += m[e];
        }
        before += wave_upto(mine) - mine;
        if (target < before || target >= before + mine) return;
        int at = 0;
        float x = 0.f;
#pragma unroll
        for (int e = 0; e < Row<T>::V; ++e) {
            if (before <= target && target < before + m[e]) at = v.i + e, x = (float)v.v[e];
            before += m[e];
        }
        put(at, x, total);
    }

    __device__ __forceinline__ Plan plan(int k, float p, bool by_count) const {
        const int t = threadIdx.x;
        Plan l{by_count, true, false, 0, (u64)k, 0};
        if (by_count) {                         // (fewer than k tokens with a bin: no limit on what weighs anything)
            l.cut = find_bin(sm.count, l.need, sm);
        } else if (p < 1.f) {
            l.need = same(share(p, block_all(sm.mass[2 * t] + sm.mass[2 * t + 1], sm, Add{})));
            find_bin(sm.mass, l.need, sm);
        } else {
            l.cut = false;
        }
        l.bin = same(sm.bin);
        l.above = same(sm.above);
        __syncthreads();
        if (!l.cut) return l;
        const unsigned few =
            (2 * t <= (int)l.bin ? sm.count[2 * t] : 0) + (2 * t + 1 <= (int)l.bin ? sm.count[2 * t + 1] : 0);
        l.take = same(block_all(few, sm, Add{})) <= (unsigned)kList;
        l.lo = l.take ? 0 : l.bin;
        l.hi = l.bin;
        return l;
    }
    // The plan of a nucleus by the bins' numbers alone, with the weight in a bin's middle: the
    // next bins on both sides are listed too while there is room (none, lo past hi: the bin alone
    // has too many), and the exact sums of the pass that lists them say whether the cut is there.
    __device__ __forceinline__ Plan guess(float p) const {
        const int t = threadIdx.x;
#pragma unroll
        for (int b = 2 * t; b < 2 * t + 2; ++b)
            sm.mass[b] = (u64)((double)sm.count[b] *
                               (double)__builtin_amdgcn_exp2f((float)w.frac - ((float)b + 0.5f) * (50.f / kBins)));
        find_bin(sm.mass, share(p, block_all(sm.mass[2 * t] + sm.mass[2 * t + 1], sm, Add{})), sm);
        Plan l{};
        l.cut = true;
        l.bin = same(sm.bin);
        l.hi = l.bin + 1 < (unsigned)kBins ? l.bin + 1 : l.bin;
        // the tokens up to there, and those of the bin and the ones beside it
        u64 upto = 0;
        for (int b = 2 * t; b < 2 * t + 2; ++b)
            if (b <= (int)l.hi) upto += sm.count[b] + (b + 1 >= (int)l.bin ? (u64)sm.count[b] << 32 : 0);
        upto = same(block_all(upto, sm, Add{}));
        l.take = (unsigned)upto <= (unsigned)kList;
        l.lo = l.take ? 0 : l.bin ? l.bin - 1 : 0;
        if (upto >> 32 > (u64)kList) {
            l.hi = l.bin;
            l.lo = same(sm.count[l.bin]) <= (unsigned)kList ? l.bin : ~0u;
        }
        __syncthreads();                        // (what follows may clear the numbers)
        return l;
    }
    // The histogram of the tokens i0 to i1: of their number, or (`mass`) of both the number and
    // the mass of those not below the cut.
    __device__ __forceinline__ void fill(int i0, int i1, bool mass, u64 cut) const {
        if (!mass)
            row.template fours<kFew>(i0, i1, threadIdx.x, NT, [&](const float (&x)[4], int) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (const unsigned b = w.bin(x[e]); b < (unsigned)kBins) atomicAdd(&sm.count[b], 1u);
            });
        else {
            const Cut c(cut);
            row.template fours<kLoads>(i0, i1, threadIdx.x, NT, [&](const float (&x)[4], int i) {
                u64 m[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) m[e] = w(x[e]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned b = w.bin(x[e]);
                    if (b >= (unsigned)kBins || !c.keeps(x[e], i + e)) continue;
                    atomicAdd(&sm.count[b], 1u);
                    atomicAdd(&sm.mass[b], m[e]);
                }
            });
        }
        __syncthreads();
    }
    // One pass over the tokens i0 to i1, a run to each wave.  To the list: those of l's bins;
    // their number is the result.  To sm.part (MASS): the masses of the runs' tokens before these
    // bins, or of all (no bins), without those below `floor`, a value's
    // first place.  To `total`: the mass of a thread's tokens.
    template <bool MASS>
    __device__ __forceinline__ unsigned sweep(int i0, int i1, const Plan& l, u64 floor, u64* total = nullptr) const {
        if (threadIdx.x == 0) sm.n = 0;
        __syncthreads();
        const int per = run_of(i0, i1), wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
        const int a = i0 + wave * per < i1 ? i0 + wave * per : i1, b = a + per < i1 ? a + per : i1;
        const float least = Cut(floor).x;
        u64 mass = 0;
        row.template fours<MASS ? kLoads : kFew>(a, b, lane, 64, [&](const float (&x)[4], int i) {
            u64 m[4] = {};
            if constexpr (MASS)
#pragma unroll
                for (int e = 0; e < 4; ++e) m[e] = w(x[e]);
            bool in[4];
            u64 has[4];
            unsigned hits = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned at = w.bin(x[e]);
                if (MASS) mass += (at < l.lo) & (x[e] >= least) ? m[e] : 0;
                if (MASS && total) *total += m[e];
                in[e] = (at >= l.lo) & (at <= l.hi);
                has[e] = lanes_of(in[e]);
                hits += __popcll(has[e]);
            }
            if (!hits) return;
            // one atomic for the wave's four
            unsigned n = 0;
            if (!before_in(lanes_of(true))) n = atomicAdd(&sm.n, hits);
            n = same(n);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned to = n + before_in(has[e]);
                if (in[e] && to < (unsigned)kList) sm.list[to] = place_of(x[e], i + e);
                n += __popcll(has[e]);
            }
        });
        if constexpr (MASS) {
            mass = wave_all(mass, Add{});
            if (lane == 0) sm.part[wave] = mass;
        }
        __syncthreads();
        const unsigned n = same(sm.n);
        __syncthreads();
        return n;
    }
    // The list's tokens not below the cut, to the masses of the runs of i0 to i1.
    __device__ __forceinline__ void add_list(int n, u64 cut, int i0, int per, u64* masses) const {
        each_listed(n, [&](float x, int i) {
            if (place_of(x, i) >= cut) atomicAdd(&masses[(i - i0) / per], w(x));
        });
        __syncthreads();
    }
    // The cut of l, from the list's n tokens of its bin (more than it holds: from the row).
    __device__ __forceinline__ u64 cut_of(const Plan& l, unsigned n) const {
        if (n > (unsigned)kList)
            return l.by_count ? cut_by_digits<false>(l.bin, l.need, l.above) : cut_by_digits<true>(l.bin, l.need, l.above);
        return cut_in_list((int)n, l.bin, !l.by_count, l.need, l.above);
    }

    // Draws from the list's n tokens, which are all those of the bins up to l's.
    __device__ __forceinline__ void from_list(int n, Plan l, float p) const {
        const bool again = l.by_count && p < 1.f;
        unsigned bin = l.bin;
        u64 need = l.need, above = l.above, cut;
#pragma unroll 1
        for (bool count = l.by_count;; count = false) {
            cut = cut_in_list(n, bin, !count, need, above);
            if (!count || !again) break;
            clear();                            // p of the tokens up to the cut
            each_listed(n, [&](float x, int i) {
                if (place_of(x, i) >= cut) atomicAdd(&sm.mass[w.bin(x)], w(x));
            });
            __syncthreads();
            need = share(p, block_all(sm.mass[2 * threadIdx.x] + sm.mass[2 * threadIdx.x + 1], sm, Add{}));
            find_bin(sm.mass, need, sm);
            bin = sm.bin;
            above = sm.above;
        }
        from_listed(n, with_floor(cut));
    }

    // A whole row, whose largest value is w.top.
    __device__ __forceinline__ void from_whole(int k, float p) const {
        const bool nucleus = p < 1.f;
        const u64 floor = with_floor(kNoCut);
        u64 cut = kNoCut;
        Plan l{};
        bool by_count = k > 0, exact = false, runs = false;
#pragma unroll 1
        for (;;) {
            if (!by_count && !nucleus) {
                cut = floor;
                break;
            }
            clear();
            fill(0, row.cols, !by_count && exact, cut);
            l = by_count || exact ? plan(k, p, by_count) : guess(p);
            if (l.lo > l.hi && l.cut) {         // no guess
                exact = true;
                continue;
            }
            if (exact) l.take = false, l.lo = l.bin;    // (a cut by number counts, the list would not know it)
            by_count = false;
            if (!l.cut) continue;               // no limit
            const bool listed_only = l.by_count && (l.take || nucleus);
            u64 total = 0;
            const unsigned n = listed_only ? sweep<false>(0, row.cols, l, floor) : sweep<true>(0, row.cols, l, floor, &total);
            const u64 mine = sm.part[threadIdx.x % kWaves];     // (what follows uses them)
            __syncthreads();
            bool past = false;                  // min_p ends before the list
            if (!l.by_count && !exact) {
                const u64 before = from_lane(row_all<kWaves>(mine, Add{}), 0);
                l.need = same(share(p, block_all(total, sm, Add{})));
                past = w.bin(value_of(floor >> 32)) < l.lo;
                exact = before >= l.need;
                if (!exact && !past) {          // the list's bin with the cut
                    clear();
                    each_listed((int)n, [&](float x, int i) { atomicAdd(&sm.mass[w.bin(x)], w(x)); });
                    __syncthreads();
                    exact = !find_bin(sm.mass, l.need - before, sm);
                    l.bin = same(sm.bin);
                    l.above = before + same(sm.above);
                    __syncthreads();
                }
                if (exact) continue;            // the guess was wrong
            }
            if (l.take) {
                from_list((int)n, l, p);
                return;
            }
            cut = past ? floor : cut_of(l, n);
            if (listed_only) {                  // a cut by number, then p of the tokens up to it
                exact = true;
                continue;
            }
            cut = cut > floor ? cut : floor;
            runs = n <= (unsigned)kList;
            if (threadIdx.x < kWaves) sm.part[threadIdx.x] = mine;
            __syncthreads();
            if (runs) add_list((int)n, cut, 0, run_of(0, row.cols), sm.part);
            break;
        }
        from_row(0, row.cols, cut, 0, 0, runs, k);
    }
};

// The largest value; -infinity for a row with nothing to draw.
template <int NT, class T>
__device__ __forceinline__ float largest_of(const Row<T>& row, int i0, int i1, Shared<NT>& sm) {
    float top = -__builtin_inff();
    row.template each<NT == 1024 ? 8 : 1>(i0, i1, threadIdx.x, NT, [&](float x, int) { top = __builtin_fmaxf(top, x); });
    return block_all(top, sm, [](float p, float q) { return __builtin_fmaxf(p, q); });
}
// What a row asks for.
struct Ask {
    float T, p, m, u;
    int k;
    __device__ __forceinline__ Ask(const SampleArgs& a, int r) {
        T = a.temp ? a.temp[r] : 1.f;
        p = a.top_p ? a.top_p[r] : 1.f;
        m = a.min_p ? a.min_p[r] : 0.f;
        u = a.u[r];
        k = a.top_k ? a.top_k[r] : 0;
        if (k < 0 || k >= a.cols) k = 0;
    }
};
// A row that needs no draw: nothing in it, or the largest asked for, of which i0 to i1 hold the first.
template <int NT, class T>
__device__ __forceinline__ void settle(const SampleArgs& a, int r, const Row<T>& row, float top, int i0, int i1, Shared<NT>& sm) {
    int first = a.cols;
    if (top > -__builtin_inff()) row.each(i0, i1, threadIdx.x, NT, [&](float x, int i) { first = x == top && i < first ? i : first; });
    first = block_all(first, sm, Min{});
    if (threadIdx.x == 0) {
        a.token[r] = first < a.cols ? first : -1;
        if (a.prob) a.prob[r] = first < a.cols ? 1.f : 0.f;
    }
}
__device__ __forceinline__ bool settled(float top, const Ask& ask) { return !(top > -__builtin_inff()) || !(ask.T > 0.f); }

// f for a row whose `cols` weights have the sum `total` in steps of 2^-frac, each off by half a step: up
// to kSampleFrac, while the sum stays below 2^62.
__device__ __forceinline__ int wide_frac(int frac, int cols, u64 total) {
    const int more = __builtin_clzll(total + (unsigned)cols) - 2;
    return frac + more < kSampleFrac ? frac + (more > 0 ? more : 0) : kSampleFrac;
}

// A workgroup to a row, which it reads three to five times (WIDE: once more).
template <class T, int NT, bool WIDE = false>
__global__ __launch_bounds__(NT) void k_sample(SampleArgs a, int frac) {
    __shared__ Shared<NT> sm;
    const int r = blockIdx.x;
    const Row<T> row{(const T*)a.x + (size_t)r * a.ld, a.cols};
    const Ask ask(a, r);
    const float top = largest_of(row, 0, a.cols, sm);
    if (settled(top, ask)) {
        settle(a, r, row, top, 0, a.cols, sm);
        return;
    }
    if constexpr (WIDE) {
        const Draw<T, NT> d{row, Weights(top, ask.T, frac, 2 * NT), sm, nullptr, nullptr, 0.f, 0.f};
        frac = wide_frac(frac, a.cols, d.mass_of(0, a.cols));
    }
    const Draw<T, NT> d{row, Weights(top, ask.T, frac, 2 * NT), sm, a.token + r, a.prob ? a.prob + r : nullptr, ask.u,
                        ask.m};
    d.from_whole(ask.k, ask.p);
}

// ---------------------------------------------------------------- few long rows
// A row's `parts` workgroups have `per` of its tokens each, in four launches: the largest,
// the histogram, the list, the draw; and, for wide rows, the sum after the largest.
struct Split {
    SampleArgs a;
    int frac, parts, per;
    char* rows;
};
constexpr int NS = 1024;                        // threads
struct SplitRow {
    u64 mass[Shared<NS>::kBins], list[Shared<NS>::kList];
    u64 kept[kSampleParts], sum[kSampleParts];
    float top[kSampleParts];
    unsigned count[Shared<NS>::kBins];
    unsigned n;
    Plan plan;
};
template <class T, bool WIDE>
struct Part {
    const int r, part, i0, i1;
    const Row<T> row;
    SplitRow& ws;
    __device__ __forceinline__ explicit Part(const Split& p)
        : r(blockIdx.y), part(blockIdx.x), i0(part * p.per), i1(i0 + p.per < p.a.cols ? i0 + p.per : p.a.cols),
          row{(const T*)p.a.x + (size_t)r * p.a.ld, p.a.cols}, ws(((SplitRow*)p.rows)[r]) {}
    __device__ __forceinline__ float top(const Split& p) const {
        const int lane = threadIdx.x & 63;
        return wave_all(lane < p.parts ? ws.top[lane] : -__builtin_inff(), [](float p, float q) { return __builtin_fmaxf(p, q); });
    }
    // the first part that holds the row's largest
    __device__ __forceinline__ int of_top(const Split& p, float top) const {
        const int lane = threadIdx.x & 63;
        return __ffsll(lanes_of(lane < p.parts && ws.top[lane] == top)) - 1;
    }
    __device__ __forceinline__ Draw<T, NS> draw(const Split& p, float top, const Ask& ask, Shared<NS>& sm) const {
        const int lane = threadIdx.x & 63;
        int frac = p.frac;
        if constexpr (WIDE) frac = wide_frac(frac, p.a.cols, wave_all(lane < p.parts ? ws.sum[lane] : 0, Add{}));
        return {row, Weights(top, ask.T, frac, 2 * NS), sm, p.a.token + r, p.a.prob ? p.a.prob + r : nullptr, ask.u,
                ask.m};
    }
};
// Those that are settled without a histogram.
__device__ __forceinline__ bool plain(float top, const Ask& ask) {
    return settled(top, ask) || (!ask.k && !(ask.p < 1.f));
}

template <class T>
__global__ __launch_bounds__(NS) void k_sample_first(Split p) {
    __shared__ Shared<NS> sm;
    const Part<T, false> q(p);
    for (int i = q.part * NS + threadIdx.x; i < 2 * NS; i += p.parts * NS) q.ws.mass[i] = 0, q.ws.count[i] = 0;
    if (q.part == 0 && threadIdx.x == 0) q.ws.n = 0;
    const float top = largest_of(q.row, q.i0, q.i1, sm);
    if (threadIdx.x == 0) q.ws.top[q.part] = top;
}

template <class T>
__global__ __launch_bounds__(NS) void k_sample_sum(Split p) {
    __shared__ Shared<NS> sm;
    const Part<T, false> q(p);
    const Ask ask(p.a, q.r);
    const float top = q.top(p);
    if (settled(top, ask)) return;
    const Draw<T, NS> d{q.row, Weights(top, ask.T, p.frac, 2 * NS), sm, nullptr, nullptr, 0.f, 0.f};
    const u64 mass = d.mass_of(q.i0, q.i1);
    if (threadIdx.x == 0) q.ws.sum[q.part] = mass;
}

template <class T, bool WIDE>
__global__ __launch_bounds__(NS) void k_sample_bins(Split p) {
    __shared__ Shared<NS> sm;
    const Part<T, WIDE> q(p);
    const Ask ask(p.a, q.r);
    const float top = q.top(p);
    if (plain(top, ask)) return;
    const auto d = q.draw(p, top, ask, sm);
    d.clear();
    d.fill(q.i0, q.i1, ask.p < 1.f, kNoCut);
#pragma unroll
    for (int i = threadIdx.x; i < 2 * NS; i += NS) {
        if (sm.count[i]) atomicAdd(&q.ws.count[i], sm.count[i]);
        if (sm.mass[i]) atomicAdd(&q.ws.mass[i], sm.mass[i]);
    }
}

// The row's histogram from memory, and its plan.
template <class T, bool WIDE>
__device__ __forceinline__ Plan plan_of(const Part<T, WIDE>& q, const Draw<T, NS>& d, const Ask& ask) {
    for (int i = threadIdx.x; i < 2 * NS; i += NS) d.sm.count[i] = q.ws.count[i], d.sm.mass[i] = q.ws.mass[i];
    __syncthreads();
    const Plan l = d.plan(ask.k, ask.p, ask.k > 0);
    return ask.k && !l.cut ? d.plan(0, ask.p, false) : l;
}
// A top-k of many tokens with a nucleus among them: one workgroup does such a row.
__device__ __forceinline__ bool hard(const Plan& l, const Ask& ask) { return l.by_count && !l.take && ask.p < 1.f; }

template <class T, bool WIDE>
__global__ __launch_bounds__(NS) void k_sample_take(Split p) {
    __shared__ Shared<NS> sm;
    const Part<T, WIDE> q(p);
    const Ask ask(p.a, q.r);
    const float top = q.top(p);
    if (settled(top, ask)) return;
    const auto d = q.draw(p, top, ask, sm);
    Plan l{};
    if (!plain(top, ask)) {
        l = plan_of(q, d, ask);
        if (q.part == 0 && threadIdx.x == 0) q.ws.plan = l;
        if (hard(l, ask)) return;
    }
    unsigned n = 0;
    u64 mass = 0;
    if (l.take) {
        n = d.template sweep<false>(q.i0, q.i1, l, 0);
    } else {
        n = d.template sweep<true>(q.i0, q.i1, l, d.with_floor(kNoCut));
        mass = block_all((threadIdx.x & 63) == 0 ? sm.part[threadIdx.x >> 6] : 0, sm, Add{});
    }
    if (threadIdx.x == 0) {
        q.ws.kept[q.part] = mass;
        sm.bin = n ? atomicAdd(&q.ws.n, n) : 0;                 // (more than the list holds: no longer of use)
    }
    __syncthreads();
    const unsigned at = sm.bin;
    for (unsigned i = threadIdx.x; i < n && i < 2 * NS && at + i < 2 * NS; i += NS) q.ws.list[at + i] = sm.list[i];
}

// A workgroup to a row.
template <class T, bool WIDE>
__global__ __launch_bounds__(NS) void k_sample_draw(Split p) {
    __shared__ Shared<NS> sm;
    __shared__ u64 kept[kSampleParts];
    const Part<T, WIDE> q(p);
    const Ask ask(p.a, q.r);
    const float top = q.top(p);
    if (settled(top, ask)) {
        const int i0 = q.of_top(p, top) * p.per;                // (-1: there is none)
        settle(p.a, q.r, q.row, top, i0, i0 + p.per < p.a.cols ? i0 + p.per : p.a.cols, sm);
        return;
    }
    const auto d = q.draw(p, top, ask, sm);
    const Plan l = plain(top, ask) ? Plan{} : q.ws.plan;
    const unsigned n = q.ws.n;
    if (l.cut && (hard(l, ask) || n > 2 * NS)) {
        d.from_whole(ask.k, ask.p);
        return;
    }
    if ((int)threadIdx.x < p.parts) kept[threadIdx.x] = q.ws.kept[threadIdx.x];
    if (l.cut)
        for (unsigned i = threadIdx.x; i < n; i += NS) sm.list[i] = q.ws.list[i];
    __syncthreads();
    if (l.take) {
        d.from_list((int)n, l, ask.p);
        return;
    }
    u64 cut = d.with_floor(kNoCut);
    if (l.cut) {
        const u64 c = d.cut_of(l, n);
        cut = c > cut ? c : cut;
        d.add_list((int)n, cut, 0, p.per, kept);
    }
    const int lane = threadIdx.x & 63;
    const u64 upto = wave_upto(lane < p.parts ? kept[lane] : 0);
    const u64 total = from_lane(upto, 63), target = d.target_of(total), past = lanes_of(upto > target);
    const int s = __ffsll(past) - 1;
    const u64 before = s ? from_lane(upto, s - 1) : 0;
    const int i0 = s * p.per;
    d.from_row(i0, i0 + p.per < p.a.cols ? i0 + p.per : p.a.cols, cut, before, total, false, ask.k);
}

template <class T, bool WIDE>
bool launch_split(const Split& p, bool cuts, hipStream_t s) {
    const dim3 grid((unsigned)p.parts, (unsigned)p.a.rows), block(NS);
    ACFUN_LAUNCH("k_sample_first", (k_sample_first<T>), grid, block, 0, s, p);
    if (WIDE) ACFUN_LAUNCH("k_sample_sum", (k_sample_sum<T>), grid, block, 0, s, p);
    if (cuts) ACFUN_LAUNCH("k_sample_bins", (k_sample_bins<T, WIDE>), grid, block, 0, s, p);
    ACFUN_LAUNCH("k_sample_take", (k_sample_take<T, WIDE>), grid, block, 0, s, p);
    ACFUN_LAUNCH("k_sample_draw", (k_sample_draw<T, WIDE>), dim3(1, (unsigned)p.a.rows), block, 0, s, p);
    return check_launch("k_sample_draw");
}

}  // namespace

bool sample_rows(const SampleArgs& a, int type, hipStream_t s) {
    const int frac = sample_frac(a.cols);
    const bool wide = a.cols > kSampleEven;
    const SamplePlan plan = sample_plan(a.rows, a.cols, num_cus());
    bool split = plan.parts > 1;
    if (split) {
        // a graph would keep the address of a temporary that goes back to the pool here
        hipStreamCaptureStatus captured = hipStreamCaptureStatusNone;
        if (!check(hipStreamIsCapturing(s, &captured), "hipStreamIsCapturing")) return false;
        split = captured == hipStreamCaptureStatusNone;
    }
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        if (split) {
            Scratch ws((size_t)a.rows * sizeof(SplitRow), s);
            const Split p{a, frac, plan.parts, plan.per, ws.as<char>()};
            const bool cuts = a.top_k || a.top_p;
            return ws.p && (wide ? launch_split<T, true>(p, cuts, s) : launch_split<T, false>(p, cuts, s));
        }
        if (plan.threads == 256)
            ACFUN_LAUNCH("k_sample", (k_sample<T, 256>), dim3(a.rows), dim3(256), 0, s, a, frac);
        else if (plan.threads == 512)
            ACFUN_LAUNCH("k_sample", (k_sample<T, 512>), dim3(a.rows), dim3(512), 0, s, a, frac);
        else if (!wide)
            ACFUN_LAUNCH("k_sample", (k_sample<T, 1024>), dim3(a.rows), dim3(1024), 0, s, a, frac);
        else
            ACFUN_LAUNCH("k_sample", (k_sample<T, 1024, true>), dim3(a.rows), dim3(1024), 0, s, a, frac);
        return check_launch("k_sample");
    });
}

}  // namespace acfun
