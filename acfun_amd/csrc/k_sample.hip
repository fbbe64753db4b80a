// k_sample.hip -- a token drawn from each row of logits.
//
//   w_i = exp((x_i - max x) / T),  tokens in order of x, the lower index first of equals;
//   kept: the first k; of these the fewest whose weights reach p of theirs; of these
//   w_i >= m.  The token is the first in order of index with sum_{j <= i} w_j > u sum w.
//
// Weights are 64-bit integers, multiples of 2^-f with f so that a row's sum fits (45 for
// 2^17 columns), from an exponential in 64 bits: sums do not depend on their order,
// and the token is the one that real numbers give but for u within about 2^-f of a border.
// The kept tokens are a range of the order, given by the bits of its last value and by how
// many of the tokens with that value it has; both are found digit by digit, without sorting.
#include "q8.hpp"

namespace acfun {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 1024, kWaves = kThreads / 64, kBins = 2048;

// The order of the values as one of integers, equal for +0 and -0; 0 for those that are
// never drawn, NaN and -infinity.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return x > -__builtin_inff() ? (b >> 31 ? ~b : b | 0x80000000u) : 0u;
}
__device__ __forceinline__ float value_of(unsigned key) {
    return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

struct Weights {
    double max, inv_t, one;                     // one: 2^f
    unsigned top;                               // the largest value's key
    __device__ __forceinline__ double real(unsigned key) const {
        if (key == top || key == 0) return key ? 1. : 0.;
        const double d = (double)value_of(key) - max;
        return d < -1e300 ? 0. : exp(d * inv_t);
    }
    __device__ __forceinline__ u64 fixed(double w) const { return (u64)(w * one + 0.5); }
    __device__ __forceinline__ u64 operator()(unsigned key) const { return fixed(real(key)); }
};

struct Shared {
    u64 mass[kBins];
    unsigned count[kBins];
    u64 part[kWaves];
    unsigned ties[kWaves], found_bin;
    u64 found_above;
};

template <class V, class F>
__device__ __forceinline__ V block_all(V v, V* part, F f) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = f(v, (V)__shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = part[0];
    for (int i = 1; i < kWaves; ++i) v = f(v, part[i]);
    __syncthreads();
    return v;
}

template <class T>
struct Row {
    const T* x;
    int cols;
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        for (int i = threadIdx.x; i < cols; i += kThreads) f(key_of((float)x[i]));
    }
};

// The bin, from the last one down, in which what the bins hold passes `need` (at least 1):
// all bins above hold less.  False if all of them do.
template <class V>
__device__ __forceinline__ bool find_bin(const V* bins, u64 need, Shared& sm) {
    const int t = threadIdx.x, b1 = kBins - 1 - 2 * t, b0 = b1 - 1;
    const u64 mine = (u64)bins[b1] + bins[b0];
    u64 upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const u64 o = __shfl_up(upto, d);
        if ((t & 63) >= d) upto += o;
    }
    if ((t & 63) == 63) sm.part[t >> 6] = upto;
    if (t == 0) sm.found_bin = kBins;
    __syncthreads();
    for (int i = 0; i < t >> 6; ++i) upto += sm.part[i];
    const u64 above = upto - mine;
    if (above < need && need <= upto) {
        const bool first = above + bins[b1] >= need;
        sm.found_bin = first ? b1 : b0;
        sm.found_above = first ? above : above + bins[b1];
    }
    __syncthreads();
    return sm.found_bin < kBins;
}

// The value (as its key) at which the tokens from the largest down to and with it pass
// `need`, by their number or by their mass, and what those above it amount to.  False if
// all tokens stay below `need`.
template <bool MASS, class T>
__device__ bool find_key(const Row<T>& row, const Weights& w, u64 need, Shared& sm, unsigned& key, u64& above) {
    unsigned prefix = 0;
    above = 0;
#pragma unroll 1
    for (int shift = 21;; shift = shift == 21 ? 10 : 0) {
        const int bits = shift ? 11 : 10;
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            if constexpr (MASS) sm.mass[i] = 0;
            else sm.count[i] = 0;
        }
        __syncthreads();
        row.each([&](unsigned k) {
            if (k == 0 || (u64)k >> (shift + bits) != prefix) return;
            const unsigned d = k >> shift & ((1u << bits) - 1);
            if constexpr (MASS) atomicAdd(&sm.mass[d], w(k));
            else atomicAdd(&sm.count[d], 1u);
        });
        __syncthreads();
        bool found;
        if constexpr (MASS) found = find_bin(sm.mass, need - above, sm);
        else found = find_bin(sm.count, need - above, sm);
        if (!found) return false;
        prefix = prefix << bits | sm.found_bin;
        above += sm.found_above;
        __syncthreads();
        if (shift == 0) break;
    }
    key = prefix;
    return true;
}

template <class T>
__global__ __launch_bounds__(kThreads) void k_sample(SampleArgs a, int frac) {
    __shared__ Shared sm;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, r = blockIdx.x;
    const Row<T> row{(const T*)a.x + (size_t)r * a.ld, a.cols};
    unsigned top = 0;
    row.each([&](unsigned k) { top = k > top ? k : top; });
    top = block_all(top, sm.ties, [](unsigned p, unsigned q) { return p > q ? p : q; });
    auto put = [&](int token, float prob) {
        a.token[r] = token;
        if (a.prob) a.prob[r] = prob;
    };
    if (top == 0) {
        if (t == 0) put(-1, 0.f);
        return;
    }
    const float T0 = a.temp ? a.temp[r] : 1.f;
    const Weights w{(double)value_of(top), 1. / (double)T0, (double)(1ull << frac), top};
    unsigned key = 0, ties = 0;                 // kept: above key, and the first `ties` of those equal to it
    u64 above;
    auto kept_mass = [&] {                      // of all those above key, and the ties
        u64 s = 0;
        row.each([&](unsigned k) { s += k > key ? w(k) : 0; });
        s = block_all(s, sm.part, [](u64 p, u64 q) { return p + q; });
        return s + ties * (key ? w(key) : 0);
    };
    if (!(T0 > 0.f)) {
        key = top, ties = 1;
    } else {
        const int k = a.top_k ? a.top_k[r] : 0;
        if (k > 0 && k < a.cols && find_key<false>(row, w, (u64)k, sm, key, above)) ties = k - (unsigned)above;
        const float p = a.top_p ? a.top_p[r] : 1.f;
        if (p < 1.f) {
            const double want = __builtin_ceil((double)p * (double)kept_mass());
            const u64 need = want >= 1. ? (u64)want : 1;
            if (find_key<true>(row, w, need, sm, key, above)) {
                const u64 each = w(key);
                ties = (unsigned)((need - above + each - 1) / each);
            }
        }
    }
    const float m = a.min_p ? a.min_p[r] : 0.f;
    const double least = m > 0.f ? m < 1.f ? m : 1. : 0.;
    auto weigh = [&](unsigned k) { const double v = w.real(k); return v >= least ? w.fixed(v) : 0; };
    // A wave has a run of the row; of those equal to key the waves before it have some.
    const int per = (a.cols + kWaves - 1) / kWaves, i0 = wave * per, i1 = i0 + per < a.cols ? i0 + per : a.cols;
    const u64 one_tie = key ? weigh(key) : 0;
    u64 mass = 0;
    unsigned equal = 0;
    for (int i = i0 + lane; i < i1; i += 64) {
        const unsigned k = key_of((float)row.x[i]);
        if (k > key) mass += weigh(k);
        equal += k == key && key;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) mass += __shfl_xor(mass, d), equal += __shfl_xor(equal, d);
    if (lane == 0) sm.part[wave] = mass, sm.ties[wave] = equal;
    __syncthreads();
    u64 total = 0, before = 0;
    unsigned seen = 0, mine = 0;                // ties of the waves so far, and before this one
    for (int i = 0; i < kWaves; ++i) {
        const unsigned n = seen < ties ? (sm.ties[i] < ties - seen ? sm.ties[i] : ties - seen) : 0;
        if (i == wave) before = total, mine = seen, mass = sm.part[i] + n * one_tie;
        total += sm.part[i] + n * one_tie;
        seen += sm.ties[i];
    }
    const float u = a.u[r];
    const double at = (double)(u > 0.f ? u < 1.f ? u : 0x1.fffffep-1f : 0.f) * (double)total;
    const u64 target = (u64)at < total ? (u64)at : total - 1;
    if (target == 0) {                          // u = 0: the first kept, however small its weight
        int first = a.cols;
        for (int i = t; i < a.cols; i += kThreads) {
            const unsigned k = key_of((float)row.x[i]);
            const double v = k >= key && k ? w.real(k) : 0.;
            if (v > 0. && v >= least && i < first) first = i;
        }
        __syncthreads();
        first = block_all(first, (int*)sm.ties, [](int p, int q) { return p < q ? p : q; });
        if (t == 0) put(first, (float)(w.real(key_of((float)row.x[first])) * w.one / (double)total));
        return;
    }
    if (target < before || target >= before + mass) return;
    for (int i = i0; i < i1; i += 64) {
        const unsigned k = i + lane < i1 ? key_of((float)row.x[i + lane]) : 0;
        const bool tie = k == key && key;
        const u64 among = __ballot(tie);
        const unsigned rank = mine + __popcll(among & ((1ull << lane) - 1));
        const u64 v = k > key || (tie && rank < ties) ? weigh(k) : 0;
        u64 upto = v;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const u64 o = __shfl_up(upto, d);
            if (lane >= d) upto += o;
        }
        const u64 past = __ballot(before + upto > target);
        if (past) {
            if (lane == __ffsll(past) - 1) put(i + lane, (float)(w.real(k) * w.one / (double)total));
            return;
        }
        before += __shfl(upto, 63);
        mine += __popcll(among);
    }
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
