// k_sample.hip -- a token drawn from each row of logits.
//
//   w_i = exp((x_i - max x) / T),  tokens in order of x, the lower index first of equals;
//   kept: the first k; of these the fewest whose weights reach p of theirs; of these
//   w_i >= m.  The token is the first in order of index with sum_{j <= i} w_j > u sum w.
//
// Weights are 64-bit integers, multiples of 2^-f with f so that a row's sum fits (45 for
// 2^17 columns), from an exponential in 64 bits: sums do not depend on their order,
// and the token is the one that real numbers give but for u within about 2^-f of a border.
// No row is sorted.  The kept tokens are those not below one of them, the cut, in the
// order; it lies in a bin of a histogram over x whose tokens alone are put in order.  Bins are
// even in x / T, 59 to a factor of e, so that most rows spread over many.  A top-k's
// tokens, or a nucleus's, that are few are all taken out of the row, and the rest is done
// with these.
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
// A token's place in the order, the first the largest.
__device__ __forceinline__ u64 place_of(float x, int i) { return (u64)key_of(x) << 32 | (unsigned)~i; }

// 2^t for t <= 0: 2^f, |f| <= 1/2, by the polynomial through 2^f at nine Chebyshev points, off by
// 1.1e-12 of the value at most.
__device__ __forceinline__ double exp2_of(double t) {
    const double n = __builtin_rint(t), f = t - n;
    double p = 0x1.63d1363a681b4p-20;
    p = __builtin_fma(p, f, 0x1.00dc4a5344ef5p-16);
    p = __builtin_fma(p, f, 0x1.4308ac85a69f8p-13);
    p = __builtin_fma(p, f, 0x1.5d8745a728209p-10);
    p = __builtin_fma(p, f, 0x1.3b2ab7181b77dp-7);
    p = __builtin_fma(p, f, 0x1.c6b08dd6fd236p-5);
    p = __builtin_fma(p, f, 0x1.ebfbdff823cedp-3);
    p = __builtin_fma(p, f, 0x1.62e42fef84cf0p-1);
    p = __builtin_fma(p, f, 1.);
    return __builtin_amdgcn_ldexp(p, (int)n);
}

struct Weights {
    double max, c, one, least;                  // c: log2(e) / T; one: 2^f; least: min_p
    float top, per_2x;                          // the largest value; bins to two units of x
    int bins;
    // `bins` for the 50 powers of two that weigh; no infinity, whose product with 0 is none
    __device__ __forceinline__ Weights(float largest, float T, float m, int frac, int n) {
        max = top = largest;
        c = 0x1.71547652b82fep+0 / (double)T;
        one = (double)(1ull << frac);
        least = m > 0.f ? m < 1.f ? m : 1. : 0.;
        per_2x = __builtin_fminf((float)n * (float)(0x1.715476p+0 / 25.) / T, 1e30f);
        bins = n;
    }
    // log2 of the weight; past any float's range where there is none
    __device__ __forceinline__ double log(float x) const {
        const double t = x == top ? 0. : ((double)x - max) * c;
        return t > -1074. ? t : -4096.;
    }
    __device__ __forceinline__ double real(float x) const {
        const double t = log(x);
        return t > -4096. ? exp2_of(t) : 0.;
    }
    __device__ __forceinline__ u64 fixed(double w) const {
        return __builtin_bit_cast(u64, __builtin_fma(w, one, 0x1p52)) - 0x4330000000000000ull;
    }
    // 0 past 2^-50, which rounds to no step
    __device__ __forceinline__ u64 operator()(float x) const {
        const double t = log(x);
        return t > -50. ? fixed(exp2_of(t)) : 0;
    }
    // the same without those below min_p
    __device__ __forceinline__ u64 kept(float x) const {
        const double t = log(x);
        const double w = t > -50. ? exp2_of(t) : 0.;
        return w >= least ? fixed(w) : 0;
    }
    // from 0 for the largest value up; `bins`: no weight (so for a NaN or -infinity)
    __device__ __forceinline__ unsigned bin(float x) const {
        const float b = x == top ? 0.f : __builtin_fmaf(x, -0.5f, 0.5f * top) * per_2x;  // (top - x may pass fp32)
        return b < (float)bins ? (unsigned)b : (unsigned)bins;
    }
};

// A workgroup's: two bins and two entries of the list to a thread.
template <int NT>
struct Shared {
    static constexpr int kWaves = NT / 64, kBins = 2 * NT, kList = 2 * NT;
    u64 mass[kBins];
    u64 list[kList], some[64], some_mass[64];
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
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = f(v, (V)__shfl_xor(v, d));
    return v;
}
template <int NT, class V, class F>
__device__ __forceinline__ V block_all(V v, Shared<NT>& sm, F f) {
    typedef std::conditional_t<sizeof(V) == 8, u64, unsigned> U;
    v = wave_all(v, f);
    if ((threadIdx.x & 63) == 0) sm.part[threadIdx.x >> 6] = __builtin_bit_cast(U, v);
    __syncthreads();
    v = __builtin_bit_cast(V, (U)sm.part[threadIdx.x % (NT / 64)]);
#pragma unroll
    for (int d = 1; d < NT / 64; d *= 2) v = f(v, (V)__shfl_xor(v, d));
    __syncthreads();
    return v;
}
// The sum over the lanes up to and with this one, of the wave and of the block.
__device__ __forceinline__ u64 wave_upto(u64 v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u64 o = __shfl_up(v, d);
        if ((int)(threadIdx.x & 63) >= d) v += o;
    }
    return v;
}
template <int NT>
__device__ __forceinline__ u64 block_upto(u64 v, Shared<NT>& sm, u64& total) {
    constexpr int W = NT / 64;
    v = wave_upto(v);
    if ((threadIdx.x & 63) == 63) sm.part[threadIdx.x >> 6] = v;
    __syncthreads();
    const u64 waves = wave_upto((int)(threadIdx.x & 63) < W ? sm.part[threadIdx.x % W] : 0);
    total = __shfl(waves, W - 1);
    const int w = threadIdx.x >> 6;
    const u64 before = __shfl(waves, w ? w - 1 : 0);
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
    // from i0 to i1, apart by whole 64 V or at the row's end, by lanes t of `threads`.  (One copy
    // of f: what runs a few times is fetched as it runs.)
    template <class F>
    __device__ __forceinline__ void each(int i0, int i1, int t, int threads, F f) const {
        int i = i0 + t * V;
        const int step = threads * V;
        if (i >= i1) return;
        Some s = load(i);
#pragma unroll 1
        for (;; i += step) {
            const Some c = s;
            const bool more = i + step < i1;
            if (more) s = load(i + step);
#pragma unroll
            for (int e = 0; e < V; ++e) f((float)c.v[e], c.i + e);
            if (!more) return;
        }
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

// The list's first n entries, the largest first; the rest of it up to a power of two is 0.
template <int NT>
__device__ __forceinline__ void sort_list(u64* list, int n) {
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += NT) list[i] = 0;
    for (int run = 2; run <= size; run *= 2)
        for (int d = run / 2; d > 0; d /= 2) {
            __syncthreads();
            const int t = threadIdx.x, i = (t & ~(d - 1)) * 2 + (t & (d - 1));
            if (t < size / 2) {
                const u64 a = list[i], b = list[i + d];
                if ((a < b) == ((i & run) == 0)) list[i] = b, list[i + d] = a;
            }
        }
    __syncthreads();
}

// What the histogram says of a row's first k (0: all) and p (1 or more: all): the bin that
// the next cut lies in, and whether the tokens up to it are few enough to take them all.
struct Plan {
    bool by_count, cut, take;                   // cut: there is one
    int k;
    unsigned bin;
    u64 need, above, mass;                      // mass: of all tokens (not by_count)
};

template <class T, int NT>
struct Draw {
    static constexpr int kWaves = NT / 64, kBins = 2 * NT, kList = 2 * NT;
    const Row<T> row;
    const Weights w;
    Shared<NT>& sm;
    int* const token;
    float* const prob;
    const float u;

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
        constexpr int D = NT == 1024 ? 11 : 9;
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
            prefix = prefix << width | ((1u << width) - 1 - sm.bin);
            before += sm.above;
            __syncthreads();
            if (shift == 0) return prefix;
            shift = shift > D ? shift - D : 0;
        }
    }
    // The same of a bin whose tokens are the list's n, in order.
    __device__ __forceinline__ u64 cut_in_list(int n, bool mass, u64 need, u64 before) const {
        const int t = threadIdx.x;
        u64 p[2], m[2], total;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            p[e] = 2 * t + e < n ? sm.list[2 * t + e] : 0;
            m[e] = !p[e] ? 0 : mass ? w(value_of(p[e] >> 32)) : 1;
        }
        const u64 upto = before + block_upto(m[0] + m[1], sm, total), first = upto - m[1];
        if (first - m[0] < need && need <= upto) sm.above = first >= need ? p[0] : p[1];
        __syncthreads();
        const u64 c = sm.above;
        __syncthreads();
        return c;
    }
    // The same of a bin whose tokens are among the list's n: up to 64 of them are taken out and each
    // counts those before it; 0 if there are more.
    __device__ __forceinline__ u64 cut_of_few(int n, unsigned b, bool mass, u64 need, u64 before) const {
        const int t = threadIdx.x;
        if (t == 0) sm.n = 0;
        __syncthreads();
        each_listed(n, [&](float x, int i) {
            if (w.bin(x) != b) return;
            const unsigned at = atomicAdd(&sm.n, 1u);
            if (at < 64) sm.some[at] = place_of(x, i), sm.some_mass[at] = mass ? w(x) : 1;
        });
        __syncthreads();
        const int m = (int)sm.n;
        if (m <= 64 && t < m) {
            const u64 mine = sm.some[t];
#pragma unroll 4
            for (int j = 0; j < m; ++j) before += sm.some[j] > mine ? sm.some_mass[j] : 0;
            if (before < need && need <= before + sm.some_mass[t]) sm.above = mine;
        }
        __syncthreads();
        const u64 c = m <= 64 ? sm.above : 0;
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
        if (prob) *prob = (float)(w.real(x) * w.one / (double)total);
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
            if (place_of(x, i) >= cut) atomicAdd(&sm.mass[i >> shift], w.kept(x));
        });
        __syncthreads();
        const u64 total = block_all(sm.mass[2 * t] + sm.mass[2 * t + 1], sm, Add{}), target = target_of(total);
        if (target == 0) {                      // u = 0: the first kept, however small its weight
            u64 first = ~0ull;
            each_listed(n, [&](float x, int i) {
                if (place_of(x, i) < cut) return;
                const double v = w.real(x);
                const u64 at = (u64)(unsigned)i << 32 | __float_as_uint(x);
                if (v > 0. && v >= w.least && at < first) first = at;
            });
            first = block_all(first, sm, Min{});
            if (t == 0) put((int)(first >> 32), __uint_as_float((unsigned)first), total);
            return;
        }
        find_bin(sm.mass, target + 1, sm);
        u64 before = sm.above;
        const int i0 = (int)sm.bin << shift, i1 = i0 + (1 << shift) < row.cols ? i0 + (1 << shift) : row.cols;
#pragma unroll 1
        for (int i = i0; i < i1; i += NT) {
            const float x = i + t < i1 ? (float)row.x[i + t] : -__builtin_inff();
            const u64 v = place_of(x, i + t) >= cut ? w.kept(x) : 0;
            u64 all;
            const u64 upto = before + block_upto(v, sm, all);
            if (upto > target && upto - v <= target) put(i + t, x, total);
            before += all;
        }
    }

    // The mass of the tokens a to b not below the cut, in every lane of a wave.
    __device__ __forceinline__ u64 kept_mass(int a, int b, u64 cut, int t, int threads) const {
        u64 mass = 0;
        row.each(a, b, t, threads, [&](float x, int i) {
            if (i < b && place_of(x, i) >= cut) mass += w.kept(x);
        });
        return wave_all(mass, Add{});
    }
    // Draws from the tokens i0 to i1 not below the cut, those before them having the mass
    // `before` of all tokens' `total` (known: false if i0 to i1 are all tokens).
    __device__ __forceinline__ void from_row(int i0, int i1, u64 cut, bool known, u64 before, u64 total) const {
        constexpr int Q = 64 * Row<T>::V;       // a wave's values at once
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        u64 target = known ? target_of(total) : 1;
        // a run to each wave, then a part of the run that the target falls in
#pragma unroll 1
        while (target) {
            const int per = ((i1 - i0 + kWaves - 1) / kWaves + Q - 1) / Q * Q;
            const int a = i0 + wave * per < i1 ? i0 + wave * per : i1, b = a + per < i1 ? a + per : i1;
            const u64 mass = kept_mass(a, b, cut, lane, 64);
            if (lane == 0) sm.part[wave] = mass;
            __syncthreads();
            const u64 upto = wave_upto(lane < kWaves ? sm.part[lane % kWaves] : 0);
            if (!known) total = __shfl(upto, kWaves - 1), target = target_of(total), known = true;
            const u64 past = __ballot(lane < kWaves && before + upto > target);
            const int s = past ? __ffsll(past) - 1 : kWaves - 1;
            before += s ? __shfl(upto, s - 1) : 0;
            __syncthreads();
            i0 += s * per;
            i1 = i0 + per < i1 ? i0 + per : i1;
            if (per == Q) break;
        }
        if (target == 0) {                      // u = 0: the first kept, however small its weight
            int first = row.cols;
            all([&](float x, int i) {
                if (i >= first || place_of(x, i) < cut) return;
                const double v = w.real(x);
                if (v > 0. && v >= w.least) first = i;
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
            m[e] = v.i + e < i1 && place_of((float)v.v[e], v.i + e) >= cut ? w.kept((float)v.v[e]) : 0;
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
        Plan l{by_count, true, false, k, 0, (u64)k, 0, 0};
        if (by_count && !find_bin(sm.count, l.need, sm)) {      // fewer tokens than k that weigh anything: no limit
            l.k = 0, l.by_count = false;
            __syncthreads();
        }
        if (!l.by_count) {
            if (!(p < 1.f)) {
                l.cut = false;
                return l;
            }
            l.mass = block_all(sm.mass[2 * t] + sm.mass[2 * t + 1], sm, Add{});
            l.need = share(p, l.mass);
            find_bin(sm.mass, l.need, sm);
        }
        l.bin = sm.bin;
        l.above = sm.above;
        const unsigned few =
            (2 * t <= (int)l.bin ? sm.count[2 * t] : 0) + (2 * t + 1 <= (int)l.bin ? sm.count[2 * t + 1] : 0);
        l.take = block_all(few, sm, Add{}) <= (unsigned)kList;
        return l;
    }
    // The histogram of the tokens i0 to i1 not below the cut.
    __device__ __forceinline__ void fill(int i0, int i1, bool count, bool mass, u64 cut) const {
        row.each(i0, i1, threadIdx.x, NT, [&](float x, int i) {
            const unsigned b = w.bin(x);
            if (b >= (unsigned)kBins || i >= i1 || (cut >> 32 && place_of(x, i) < cut)) return;
            if (count) atomicAdd(&sm.count[b], 1u);
            if (mass) atomicAdd(&sm.mass[b], w(x));
        });
        __syncthreads();
    }
    // Tokens i0 to i1 of the bins up to l's (l.take) or of that alone to the list; their number.
    __device__ __forceinline__ unsigned gather(int i0, int i1, const Plan& l) const {
        if (threadIdx.x == 0) sm.n = 0;
        __syncthreads();
        const unsigned b0 = l.take ? 0 : l.bin;
        row.each(i0, i1, threadIdx.x, NT, [&](float x, int i) {
            const unsigned b = w.bin(x);
            if (b < b0 || b > l.bin || i >= i1) return;
            const unsigned at = atomicAdd(&sm.n, 1u);
            if (at < (unsigned)kList) sm.list[at] = place_of(x, i);
        });
        __syncthreads();
        const unsigned n = sm.n;
        __syncthreads();
        return n;
    }
    // The cut of l, from the list's n tokens of its bin (more than it holds: from the row).
    __device__ __forceinline__ u64 cut_of(const Plan& l, unsigned n) const {
        if (n > (unsigned)kList)
            return l.by_count ? cut_by_digits<false>(l.bin, l.need, l.above) : cut_by_digits<true>(l.bin, l.need, l.above);
        sort_list<NT>(sm.list, (int)n);
        return cut_in_list((int)n, !l.by_count, l.need, l.above);
    }

    // Draws from the list's n tokens, which are all those of the bins up to l's.
    __device__ __forceinline__ void from_list(int n, Plan l, float p) const {
        const bool again = l.by_count && p < 1.f;
        unsigned bin = l.bin;
        u64 need = l.need, above = l.above, cut;
#pragma unroll 1
        for (bool count = l.by_count;; count = false) {
            cut = cut_of_few(n, bin, !count, need, above);
            if (!cut || !count || !again) break;
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
        if (cut == 0) {                         // many in the cut's bin: all of the list in order
            sort_list<NT>(sm.list, n);
            cut = cut_in_list(n, !l.by_count, l.by_count ? (u64)l.k : l.need, 0);
            if (again) {
                u64 mass = 0;
                each_listed(n, [&](float x, int i) { mass += place_of(x, i) >= cut ? w(x) : 0; });
                cut = cut_in_list(n, true, share(p, block_all(mass, sm, Add{})), 0);
            }
        }
        from_listed(n, cut);
    }

    // A whole row, whose largest value is w.top.
    __device__ __forceinline__ void from_whole(int k, float p) const {
        u64 cut = 1ull << 32;                   // all that can be drawn
        bool by_count = k > 0;
#pragma unroll 1
        for (bool first = true; by_count || p < 1.f; first = false) {
            clear();
            fill(0, row.cols, first, p < 1.f, first ? 0 : cut);
            Plan l = plan(k, p, by_count);
            if (!l.cut) break;
            l.take &= first;
            const unsigned n = gather(0, row.cols, l);
            if (l.take) {
                from_list((int)n, l, p);
                return;
            }
            cut = cut_of(l, n);
            if (!l.by_count || !(p < 1.f)) break;
            by_count = false;                   // p of the tokens up to the cut
        }
        from_row(0, row.cols, cut, false, 0, 0);
    }
};

// A row's largest value with its lowest index, as its place; 0 for a row with nothing to draw.
template <int NT, class T>
__device__ __forceinline__ u64 first_of(const Row<T>& row, int i0, int i1, Shared<NT>& sm) {
    float top = -__builtin_inff();
    int at = 0;
    row.each(i0, i1, threadIdx.x, NT, [&](float x, int i) {
        const bool more = x > top && i < i1;
        top = more ? x : top;
        at = more ? i : at;
    });
    return block_all(top > -__builtin_inff() ? place_of(top, at) : 0, sm, Max{});
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
// A row that needs no draw: nothing in it, or the largest asked for.
__device__ __forceinline__ bool settled(const SampleArgs& a, int r, u64 first, const Ask& ask) {
    if (first && ask.T > 0.f) return false;
    if (threadIdx.x == 0) {
        a.token[r] = first ? ~(int)first : -1;
        if (a.prob) a.prob[r] = first ? 1.f : 0.f;
    }
    return true;
}

// A workgroup to a row, which it reads three to five times.
template <class T, int NT>
__global__ __launch_bounds__(NT) void k_sample(SampleArgs a, int frac) {
    __shared__ Shared<NT> sm;
    const int r = blockIdx.x;
    const Row<T> row{(const T*)a.x + (size_t)r * a.ld, a.cols};
    const Ask ask(a, r);
    const u64 first = first_of(row, 0, a.cols, sm);
    if (settled(a, r, first, ask)) return;
    const Draw<T, NT> d{row, Weights(value_of(first >> 32), ask.T, ask.m, frac, 2 * NT), sm, a.token + r,
                        a.prob ? a.prob + r : nullptr, ask.u};
    d.from_whole(ask.k, ask.p);
}

// ---------------------------------------------------------------- few long rows
// A row's `parts` workgroups have `per` of its tokens each, in four launches: the largest,
// the histogram, the list, the draw.
struct Split {
    SampleArgs a;
    int frac, parts, per;
    char* rows;
};
constexpr int NS = 1024;                        // threads
struct SplitRow {
    u64 mass[Shared<NS>::kBins], list[Shared<NS>::kList];
    u64 first[kSampleParts], kept[kSampleParts];
    unsigned count[Shared<NS>::kBins];
    unsigned n, done;
    Plan plan;
};
template <class T>
struct Part {
    const int r, part, i0, i1;
    const Row<T> row;
    SplitRow& ws;
    __device__ __forceinline__ explicit Part(const Split& p)
        : r(blockIdx.y), part(blockIdx.x), i0(part * p.per), i1(i0 + p.per < p.a.cols ? i0 + p.per : p.a.cols),
          row{(const T*)p.a.x + (size_t)r * p.a.ld, p.a.cols}, ws(((SplitRow*)p.rows)[r]) {}
    __device__ __forceinline__ u64 first(const Split& p) const {
        const int lane = threadIdx.x & 63;
        return wave_all(lane < p.parts ? ws.first[lane] : 0, Max{});
    }
    __device__ __forceinline__ Draw<T, NS> draw(const Split& p, u64 top, const Ask& ask, Shared<NS>& sm) const {
        return {row, Weights(value_of(top >> 32), ask.T, ask.m, p.frac, 2 * NS), sm, p.a.token + r,
                p.a.prob ? p.a.prob + r : nullptr, ask.u};
    }
};
// Those that are settled without a histogram.
__device__ __forceinline__ bool plain(u64 top, const Ask& ask) {
    return !top || !(ask.T > 0.f) || (!ask.k && !(ask.p < 1.f));
}

template <class T>
__global__ __launch_bounds__(NS) void k_sample_first(Split p) {
    __shared__ Shared<NS> sm;
    const Part<T> q(p);
    for (int i = q.part * NS + threadIdx.x; i < 2 * NS; i += p.parts * NS) q.ws.mass[i] = 0, q.ws.count[i] = 0;
    if (q.part == 0 && threadIdx.x == 0) q.ws.n = 0, q.ws.done = 0;
    const u64 top = first_of(q.row, q.i0, q.i1, sm);
    if (threadIdx.x == 0) q.ws.first[q.part] = top;
}

template <class T>
__global__ __launch_bounds__(NS) void k_sample_bins(Split p) {
    __shared__ Shared<NS> sm;
    const Part<T> q(p);
    const Ask ask(p.a, q.r);
    const u64 top = q.first(p);
    if (plain(top, ask)) return;
    const auto d = q.draw(p, top, ask, sm);
    d.clear();
    d.fill(q.i0, q.i1, true, ask.p < 1.f, 0);
#pragma unroll
    for (int i = threadIdx.x; i < 2 * NS; i += NS) {
        if (sm.count[i]) atomicAdd(&q.ws.count[i], sm.count[i]);
        if (sm.mass[i]) atomicAdd(&q.ws.mass[i], sm.mass[i]);
    }
}

// The row's histogram from memory, and its plan.
template <class T>
__device__ __forceinline__ Plan plan_of(const Part<T>& q, const Draw<T, NS>& d, const Ask& ask) {
    for (int i = threadIdx.x; i < 2 * NS; i += NS) d.sm.count[i] = q.ws.count[i], d.sm.mass[i] = q.ws.mass[i];
    __syncthreads();
    return d.plan(ask.k, ask.p, ask.k > 0);
}
// A top-k of many tokens with a nucleus among them: one workgroup does such a row.
__device__ __forceinline__ bool hard(const Plan& l, const Ask& ask) { return l.by_count && !l.take && ask.p < 1.f; }

template <class T>
__global__ __launch_bounds__(NS) void k_sample_take(Split p) {
    __shared__ Shared<NS> sm;
    const Part<T> q(p);
    const Ask ask(p.a, q.r);
    const u64 top = q.first(p);
    if (plain(top, ask)) return;
    const auto d = q.draw(p, top, ask, sm);
    const Plan l = plan_of(q, d, ask);
    if (q.part == 0 && threadIdx.x == 0) q.ws.plan = l;
    if (!l.cut || hard(l, ask)) return;
    const unsigned n = d.gather(q.i0, q.i1, l);
    if (n == 0) return;
    if (threadIdx.x == 0) sm.bin = atomicAdd(&q.ws.n, n);       // (more than the list holds: no longer of use)
    __syncthreads();
    const unsigned at = sm.bin;
    for (unsigned i = threadIdx.x; i < n && i < 2 * NS && at + i < 2 * NS; i += NS) q.ws.list[at + i] = sm.list[i];
}

template <class T>
__global__ __launch_bounds__(NS) void k_sample_draw(Split p) {
    __shared__ Shared<NS> sm;
    const Part<T> q(p);
    const Ask ask(p.a, q.r);
    const u64 top = q.first(p);
    if (!top || !(ask.T > 0.f)) {
        if (q.part == 0) settled(p.a, q.r, top, ask);
        return;
    }
    const auto d = q.draw(p, top, ask, sm);
    u64 cut = 1ull << 32;
    if (!plain(top, ask)) {
        const Plan l = q.ws.plan;
        const unsigned n = q.ws.n;
        if (l.cut && (hard(l, ask) || n > 2 * NS)) {
            if (q.part == 0) d.from_whole(ask.k, ask.p);
            return;
        }
        if (l.cut) {
            if (l.take && q.part) return;
            for (unsigned i = threadIdx.x; i < n; i += NS) sm.list[i] = q.ws.list[i];
            __syncthreads();
            if (l.take) {
                d.from_list((int)n, l, ask.p);
                return;
            }
            cut = d.cut_of(l, n);
        }
    }
    // every part's mass; the last workgroup to have its own draws
    const u64 mass = block_all(d.kept_mass(q.i0, q.i1, cut, threadIdx.x, NS) * ((threadIdx.x & 63) == 0), sm, Add{});
    if (threadIdx.x == 0) {
        __hip_atomic_store(&q.ws.kept[q.part], mass, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        sm.n = __hip_atomic_fetch_add(&q.ws.done, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (sm.n != (unsigned)p.parts - 1) return;
    const int lane = threadIdx.x & 63;
    const u64 upto = wave_upto(lane < p.parts ? __hip_atomic_load(&q.ws.kept[lane], __ATOMIC_RELAXED,
                                                                  __HIP_MEMORY_SCOPE_AGENT) : 0);
    const u64 total = __shfl(upto, 63), target = d.target_of(total), past = __ballot(upto > target);
    const int s = __ffsll(past) - 1;
    const u64 before = s ? __shfl(upto, s - 1) : 0;
    const int i0 = s * p.per, i1 = i0 + p.per < p.a.cols ? i0 + p.per : p.a.cols;
    d.from_row(i0, i1, cut, true, before, total);
}

template <class T>
bool launch_split(const Split& p, bool cuts, hipStream_t s) {
    const dim3 grid((unsigned)p.parts, (unsigned)p.a.rows), block(NS);
    ACFUN_LAUNCH("k_sample_first", (k_sample_first<T>), grid, block, 0, s, p);
    if (cuts) {
        ACFUN_LAUNCH("k_sample_bins", (k_sample_bins<T>), grid, block, 0, s, p);
        ACFUN_LAUNCH("k_sample_take", (k_sample_take<T>), grid, block, 0, s, p);
    }
    ACFUN_LAUNCH("k_sample_draw", (k_sample_draw<T>), grid, block, 0, s, p);
    return check_launch("k_sample_draw");
}

}  // namespace

bool sample_rows(const SampleArgs& a, int type, hipStream_t s) {
    int bits = 0;
    while ((1 << bits) < a.cols) ++bits;
    const int frac = 62 - bits < 48 ? 62 - bits : 48;
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
            return ws.p && launch_split<T>({a, frac, plan.parts, plan.per, ws.as<char>()}, a.top_k || a.top_p, s);
        }
        if (a.cols <= kSampleShort)
            ACFUN_LAUNCH("k_sample", (k_sample<T, 256>), dim3(a.rows), dim3(256), 0, s, a, frac);
        else
            ACFUN_LAUNCH("k_sample", (k_sample<T, 1024>), dim3(a.rows), dim3(1024), 0, s, a, frac);
        return check_launch("k_sample");
    });
}

}  // namespace acfun
