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
constexpr int kThreads = kSampleThreads, kWaves = kThreads / 64, kBins = 2048, kList = 2048;

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
    // from 0 for the largest value up; kBins: no weight (so for a NaN or -infinity)
    __device__ __forceinline__ unsigned bin(float x) const {
        const float b = x == top ? 0.f : __builtin_fmaf(x, -0.5f, 0.5f * top) * per_2x;  // (top - x may pass fp32)
        return b < (float)kBins ? (unsigned)b : kBins;
    }
};

struct Shared {
    u64 mass[kBins];
    u64 list[kList];
    u64 part[kWaves + 1];
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
template <class V, class F>
__device__ __forceinline__ V block_all(V v, Shared& sm, F f) {
    v = wave_all(v, f);
    if ((threadIdx.x & 63) == 0) sm.part[threadIdx.x >> 6] = __builtin_bit_cast(std::conditional_t<sizeof(V) == 8, u64, unsigned>, v);
    __syncthreads();
    auto get = [&](int i) { return __builtin_bit_cast(V, (std::conditional_t<sizeof(V) == 8, u64, unsigned>)sm.part[i]); };
    v = get(0);
    for (int i = 1; i < kWaves; ++i) v = f(v, get(i));
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
__device__ __forceinline__ u64 block_upto(u64 v, Shared& sm, u64& total) {
    v = wave_upto(v);
    if ((threadIdx.x & 63) == 63) sm.part[threadIdx.x >> 6] = v;
    __syncthreads();
    total = 0;
    for (int i = 0; i < kWaves; ++i) {
        const u64 o = sm.part[i];
        if (i < (int)(threadIdx.x >> 6)) v += o;
        total += o;
    }
    __syncthreads();
    return v;
}

// A row's values, 16 bytes of them to a lane, to f(x, index).
template <class T>
struct Row {
    static constexpr int V = 16 / (int)sizeof(T);
    typedef typename VecOf<T, V>::type VT;
    const T* x;
    int cols;
    // a lane's V values from index i
    __device__ __forceinline__ VT load(int i) const { return load_vec<T, V>(x + i, cols - i, -__builtin_inff()); }
    // from i0 to i1, both whole 64 V but for the row's end, by lanes of `threads`, U loads at once
    template <int U, class F>
    __device__ __forceinline__ void each(int i0, int i1, int t, int threads, F f) const {
        int i = i0 + t * V;
        const int step = threads * V;
        for (; i + (U - 1) * step + V <= i1; i += U * step) {
            VT v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = *(const VT*)(x + i + u * step);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < V; ++e) f((float)v[u][e], i + u * step + e);
        }
#pragma unroll 1
        for (; i < i1; i += step) {
            const VT v = load(i);
#pragma unroll
            for (int e = 0; e < V; ++e) f((float)v[e], i + e);
        }
    }
    template <int U, class F>
    __device__ __forceinline__ void all(F f) const { each<U>(0, cols, threadIdx.x, kThreads, f); }
};

// The first bin up to and with which the bins hold `need` (at least 1); those before it
// hold sm.above.  False if all of them hold less.
template <class V>
__device__ __forceinline__ bool find_bin(const V* bins, u64 need, Shared& sm) {
    const int t = threadIdx.x, b0 = 2 * t, b1 = b0 + 1;
    const u64 first = bins[b0], mine = first + bins[b1];
    if (t == 0) sm.bin = kBins;
    u64 total;
    const u64 above = block_upto(mine, sm, total) - mine;
    if (above < need && need <= above + mine) {
        const bool zero = above + first >= need;
        sm.bin = zero ? b0 : b1;
        sm.above = zero ? above : above + first;
    }
    __syncthreads();
    return sm.bin < kBins;
}

// The list's first n entries, the largest first; the rest of it up to a power of two is 0.
__device__ void sort_list(u64* list, int n) {
    int size = 64;
    while (size < n) size *= 2;
    for (int i = n + threadIdx.x; i < size; i += kThreads) list[i] = 0;
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

template <class T>
struct Draw {
    const Row<T> row;
    Weights w;
    Shared& sm;

    // Tokens of the bins b0 to b1 into the list, in order; false if they are more than it holds.
    __device__ bool gather(unsigned b0, unsigned b1) {
        if (threadIdx.x == 0) sm.n = 0;
        __syncthreads();
        row.template all<4>([&](float x, int i) {
            const unsigned b = w.bin(x);
            if (b < b0 || b > b1) return;
            const unsigned at = atomicAdd(&sm.n, 1u);
            if (at < kList) sm.list[at] = place_of(x, i);
        });
        __syncthreads();
        const unsigned n = sm.n;
        __syncthreads();
        if (n > kList) return false;
        sort_list(sm.list, (int)n);
        return true;
    }

    // The cut in bin b: the first place of its tokens, in order, up to and with which their
    // number or mass, `before` with what the earlier bins hold, is `need`; `upto` becomes the
    // mass (MASS) up to and with it.  For bins of any size: by its digits, a pass for each.
    template <bool MASS>
    __device__ u64 cut_by_digits(unsigned b, u64 need, u64 before) {
        u64 prefix = 0;
        for (int shift = 53;; shift = shift > 11 ? shift - 11 : 0) {
            const int width = shift ? 11 : 9;
            for (int i = threadIdx.x; i < kBins; i += kThreads) {
                if constexpr (MASS) sm.mass[i] = 0;
                else sm.count[i] = 0;
            }
            __syncthreads();
            row.template all<1>([&](float x, int i) {
                if (w.bin(x) != b) return;
                const u64 p = place_of(x, i);
                if (shift < 53 && p >> (shift + width) != prefix) return;
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
        }
    }
    template <bool MASS>
    __device__ u64 cut(unsigned b, u64 need, u64 before) {
        if (!gather(b, b)) return cut_by_digits<MASS>(b, need, before);
        u64 total;
        const int t = threadIdx.x, n = (int)sm.n;
        const u64 p0 = 2 * t < n ? sm.list[2 * t] : 0, p1 = 2 * t + 1 < n ? sm.list[2 * t + 1] : 0;
        u64 m0, m1;
        if constexpr (MASS) m0 = p0 ? w(value_of(p0 >> 32)) : 0, m1 = p1 ? w(value_of(p1 >> 32)) : 0;
        else m0 = p0 != 0, m1 = p1 != 0;
        const u64 upto = before + block_upto(m0 + m1, sm, total), first = upto - m1;
        if (first - m0 < need && need <= upto) sm.above = first >= need ? p0 : p1;
        __syncthreads();
        const u64 c = sm.above;
        __syncthreads();
        return c;
    }

    // Draws from the first n of the list, which is in order, with u; the total's weight.
    __device__ void from_list(int n, float u, int* token, float* prob) {
        const int t = threadIdx.x;
        u64 p[2], m[2], total;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            p[e] = 2 * t + e < n ? sm.list[2 * t + e] : 0;
            p[e] = p[e] << 32 | p[e] >> 32;     // by index: ~i is the larger half
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 2; ++e)
            if (2 * t + e < n) sm.list[2 * t + e] = p[e];
        __syncthreads();
        sort_list(sm.list, n);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            p[e] = 2 * t + e < n ? sm.list[2 * t + e] : 0;
            m[e] = p[e] ? w.kept(value_of((unsigned)p[e])) : 0;
        }
        const u64 upto = block_upto(m[0] + m[1], sm, total), before = upto - m[0] - m[1];
        const u64 target = target_of(u, total);
        if (target == 0 && u64_zero(u, n, token, prob, total)) return;
        if (before <= target && target < upto) {
            const bool one = target >= before + m[0];
            put(~(int)(p[one] >> 32), value_of((unsigned)p[one]), total, token, prob);
        }
    }
    __device__ __forceinline__ u64 target_of(float u, u64 total) const {
        const double at = (double)(u > 0.f ? u < 1.f ? u : 0x1.fffffep-1f : 0.f) * (double)total;
        return (u64)at < total ? (u64)at : total - 1;
    }
    __device__ __forceinline__ void put(int i, float x, u64 total, int* token, float* prob) const {
        *token = i;
        if (prob) *prob = (float)(w.real(x) * w.one / (double)total);
    }
    // u = 0 among the list: the first kept, however small its weight
    __device__ bool u64_zero(float, int n, int* token, float* prob, u64 total) {
        const int t = threadIdx.x;
        int first = kList;
        for (int j = 2 * t + 1; j >= 2 * t; --j)
            if (j < n) {
                const double v = w.real(value_of((unsigned)sm.list[j]));
                if (v > 0. && v >= w.least) first = j;
            }
        first = block_all(first, sm, Min{});
        if (t == 0) put(~(int)(sm.list[first] >> 32), value_of((unsigned)sm.list[first]), total, token, prob);
        return true;
    }

    // Draws from all tokens of the row not below the cut.
    __device__ void from_row(u64 cut, float u, int* token, float* prob) {
        constexpr int Q = 64 * Row<T>::V;       // a wave's values at once
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        auto kept = [&](float x, int i) { return place_of(x, i) >= cut ? w.kept(x) : 0; };
        // a run of the row to each wave, then a part of the run that it falls in
        int i0 = 0, i1 = row.cols;
        u64 before = 0, total = 0, target = 0;
        for (int level = 0;; ++level) {
            const int per = ((i1 - i0 + kWaves - 1) / kWaves + Q - 1) / Q * Q;
            const int a = i0 + wave * per < i1 ? i0 + wave * per : i1, b = a + per < i1 ? a + per : i1;
            u64 mass = 0;
            row.template each<2>(a, b, lane, 64, [&](float x, int i) { mass += i < b ? kept(x, i) : 0; });
            mass = wave_all(mass, Add{});
            if (lane == 0) sm.part[wave] = mass;
            __syncthreads();
            if (level == 0) {
                for (int i = 0; i < kWaves; ++i) total += sm.part[i];
                target = target_of(u, total);
                if (target == 0) break;
            }
            int s = 0;
            for (; s < kWaves - 1 && target >= before + sm.part[s]; ++s) before += sm.part[s];
            __syncthreads();
            i0 += s * per;
            i1 = i0 + per < i1 ? i0 + per : i1;
            if (per == Q) break;
        }
        if (target == 0) {                      // u = 0: the first kept, however small its weight
            int first = row.cols;
            row.template all<1>([&](float x, int i) {
                if (i >= first || place_of(x, i) < cut) return;
                const double v = w.real(x);
                if (v > 0. && v >= w.least) first = i;
            });
            __syncthreads();
            first = block_all(first, sm, Min{});
            if (threadIdx.x == 0) put(first, (float)row.x[first], total, token, prob);
            return;
        }
        if (wave) return;
        const auto v = row.load(i0 + lane * Row<T>::V);
        u64 mine = 0;
#pragma unroll
        for (int e = 0; e < Row<T>::V; ++e) mine += kept((float)v[e], i0 + lane * Row<T>::V + e);
        before += wave_upto(mine) - mine;
        if (target < before || target >= before + mine) return;
        for (int e = 0; e < Row<T>::V; ++e) {
            const int i = i0 + lane * Row<T>::V + e;
            const float x = (float)row.x[i];
            before += kept(x, i);
            if (before > target) {
                put(i, x, total, token, prob);
                return;
            }
        }
    }
};

template <class T>
__global__ __launch_bounds__(kThreads) void k_sample(SampleArgs a, int frac) {
    __shared__ Shared sm;
    const int t = threadIdx.x, r = blockIdx.x;
    Draw<T> d{{(const T*)a.x + (size_t)r * a.ld, a.cols}, {}, sm};
    int* const token = a.token + r;
    float* const prob = a.prob ? a.prob + r : nullptr;
    float top = -__builtin_inff();
    d.row.template all<4>([&](float x, int) { top = __builtin_fmaxf(top, x); });
    top = block_all(top, sm, [](float p, float q) { return __builtin_fmaxf(p, q); });
    if (top == -__builtin_inff()) {
        if (t == 0) {
            *token = -1;
            if (prob) *prob = 0.f;
        }
        return;
    }
    const float T0 = a.temp ? a.temp[r] : 1.f, m = a.min_p ? a.min_p[r] : 0.f, u = a.u[r];
    if (!(T0 > 0.f)) {
        int first = a.cols;
        d.row.template all<4>([&](float x, int i) { first = x == top && i < first ? i : first; });
        first = block_all(first, sm, Min{});
        if (t == 0) {
            *token = first;
            if (prob) *prob = 1.f;
        }
        return;
    }
    Weights& w = d.w;
    w.max = top;
    w.c = 0x1.71547652b82fep+0 / (double)T0;
    w.one = (double)(1ull << frac);
    w.least = m > 0.f ? m < 1.f ? m : 1. : 0.;
    w.top = top;
    // kBins for the 50 powers of two that weigh; no infinity, whose product with 0 is none
    w.per_2x = __builtin_fminf((float)(kBins / 25.) * (0x1.715476p+0f / T0), 1e30f);
    int k = a.top_k ? a.top_k[r] : 0;
    float p = a.top_p ? a.top_p[r] : 1.f;
    const bool nucleus = p < 1.f;
    u64 cut = 1ull << 32;                       // all that can be drawn
    if (k <= 0 || k >= a.cols) k = 0;
    if (k || nucleus) {
        for (int i = t; i < kBins; i += kThreads) sm.mass[i] = 0, sm.count[i] = 0;
        __syncthreads();
        d.row.template all<2>([&](float x, int) {
            const unsigned b = w.bin(x);
            if (b >= kBins) return;
            atomicAdd(&sm.count[b], 1u);
            if (nucleus) atomicAdd(&sm.mass[b], w(x));
        });
        __syncthreads();
        // (fewer tokens than k that weigh anything: no limit)
        if (k && !find_bin(sm.count, (u64)k, sm)) k = 0;
        unsigned b = sm.bin;
        u64 above = sm.above, all = 0, need = 0;
        __syncthreads();
        if (!k && !nucleus) {
            d.from_row(cut, u, token, prob);
            return;
        }
        if (nucleus) {
            u64 mine = sm.mass[2 * t] + sm.mass[2 * t + 1];
            all = block_all(mine, sm, Add{});
        }
        auto share = [&](u64 of) {
            const double want = __builtin_ceil((double)p * (double)of);
            return want >= 1. ? (u64)want : 1;
        };
        if (!k) {
            need = share(all);
            find_bin(sm.mass, need, sm);
            b = sm.bin;
            above = sm.above;
            __syncthreads();
        }
        // how many the bins up to b hold
        u64 few = 0;
        for (int i = 2 * t; i < 2 * t + 2; ++i) few += i <= (int)b ? sm.count[i] : 0;
        few = block_all(few, sm, Add{});
        if (few <= kList) {
            d.gather(0, b);
            int n = (int)sm.n;
            if (k && n > k) n = k;
            if (nucleus) {
                u64 mass[2], total;
                for (int e = 0; e < 2; ++e) mass[e] = 2 * t + e < n ? w(value_of(sm.list[2 * t + e] >> 32)) : 0;
                const u64 upto = block_upto(mass[0] + mass[1], sm, total);
                if (k) need = share(total);
                // a token is kept while those before it stay below `need`
                const u64 b1 = upto - mass[1], b0 = b1 - mass[0];
                u64 mine = (2 * t < n && b0 < need) + (2 * t + 1 < n && b1 < need);
                n = (int)block_all(mine, sm, Add{});
            }
            d.from_list(n, u, token, prob);
            return;
        }
        if (k) {
            cut = d.template cut<false>(b, (u64)k, above);
            if (nucleus) {
                // of the tokens up to the cut: their mass, and the bin that holds p of it
                for (int i = t; i < kBins; i += kThreads) sm.mass[i] = 0;
                __syncthreads();
                d.row.template all<2>([&](float x, int i) {
                    const unsigned b = w.bin(x);
                    if (b < kBins && place_of(x, i) >= cut) atomicAdd(&sm.mass[b], w(x));
                });
                __syncthreads();
                all = block_all(sm.mass[2 * t] + sm.mass[2 * t + 1], sm, Add{});
                need = share(all);
                find_bin(sm.mass, need, sm);
                b = sm.bin;
                above = sm.above;
                __syncthreads();
                cut = d.template cut<true>(b, need, above);
            }
        } else {
            cut = d.template cut<true>(b, need, above);
        }
    }
    d.from_row(cut, u, token, prob);
}

}  // namespace

bool sample_rows(const SampleArgs& a, int type, hipStream_t s) {
    int bits = 0;
    while ((1 << bits) < a.cols) ++bits;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        ACFUN_LAUNCH("k_sample", k_sample<T>, dim3(a.rows), dim3(kThreads), 0, s, a, 62 - bits < 48 ? 62 - bits : 48);
        return check_launch("k_sample");
    });
}

}  // namespace acfun
