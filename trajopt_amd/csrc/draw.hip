// Draws from exponentiated returns: for every row of K returns the samples that pass top-k, top-p and min-p are weighed by
// w_i = exp(kappa (R_i - max R)), and given uniform numbers u pick the smallest i with  sum_{j <= i} w_j > u W.
//
// Numbers.  A return that is NaN or infinite weighs nothing, as in the planner's updates.  Weights are evaluated in fp64 and
// summed as 64-bit fixed point, q_i = round(w_i 2^S): integer sums do not depend on their order, so the histograms may use
// atomics, a row gives the same answer however it is split, and ties are exact.  The best sample weighs 1, so a mass is never
// below 2^S, and each of K roundings is off by half a unit at most: a border between two samples lies within K 2^-(S + 1) of the mass
// of where it would be without them (2^-31 for 65536 samples in LDS).  Rows in LDS take the largest S at which K weights of 1
// stay below 2^62 (at most 51, where w 2^S still fits the 52 bits of a double's fraction: 46 for the longest row); longer
// rows first sum their weights and take S from that sum, so that a row with few samples that count keeps 51 bits of them.
// Samples with kappa (max - R) > (S + 1) ln 2 round to zero; they cannot be drawn, and are left out from the start.
//
// Borders.  The samples kept by top-k and top-p are a prefix of the order (return descending, index ascending), so either
// filter is one pair (the last return that is kept, and the index up to which samples equal to it are).  It is found without
// sorting: a histogram of counts (top-k) or masses (top-p) over bins that are linear in max - R, then, while the bin with the
// border holds more than 64 samples of different returns, histograms over the bits of its keys, and last the ranks of the up to
// 64 candidates, a lane each, by comparing each with each.  (A linear bin holds about as many samples wherever it lies; bins
// of the key's leading bits would put most returns of a planner, which are of one magnitude, into one.)
//
// What bounds it.  The bytes are few (the benchmark planner's row is 16 KB); what takes the time is one pass behind the other
// over a row, with a barrier after each, and the instructions of code that runs once.  So a row stays in one workgroup's LDS as long
// as it fits, passes test values in the type of the row and evaluate fp64 exponentials only where a sample passes, and loops are
// rolled.  Per call in a row of calls (3.6 us for the smallest kernel there is): 1 x 40 fp64 with top-k 5.4 us; 1 x 4096 fp32 with
// top-p 9.3; 1024 x 512 fp32 with all three filters 8.8; 192 x 65535 bf16 with all three 17.3 or 20, one of the two for as long as a
// process runs (25 MB: 1.3 to 1.5 TB/s); 1 x 524288 fp32 with both borders 28.5; 16 x 262144 fp64 with top-p and 64 draws each 58.5.
#include "abi_common.hpp"
#include "bins.hpp"
#include "../../include/mppi_hip.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <exception>

using mppi::fail;

namespace {

// ------------------------------------------------------------------------------------------
// returns of every type as float or double, and keys that order like them
// ------------------------------------------------------------------------------------------
struct Half { uint16_t bits; };
struct Bfloat { uint16_t bits; };
__device__ __forceinline__ double value_of(double x) { return x; }
__device__ __forceinline__ float value_of(float x) { return x; }
__device__ __forceinline__ float value_of(Half x) { return (float)__builtin_bit_cast(_Float16, x.bits); }
__device__ __forceinline__ float value_of(Bfloat x) { return __uint_as_float((unsigned)x.bits << 16); }

__device__ __forceinline__ float minus_infinity(float*) { return -INFINITY; }
__device__ __forceinline__ double minus_infinity(double*) { return -INFINITY; }
__device__ __forceinline__ float lowest(float*) { return -3.402823466e38f; }
__device__ __forceinline__ double lowest(double*) { return -1.7976931348623157e308; }
__device__ __forceinline__ Half minus_infinity(Half*) { return {0xfc00}; }
__device__ __forceinline__ Bfloat minus_infinity(Bfloat*) { return {0xff80}; }

template <class T> struct Traits { using V = float; using U = uint32_t; };
template <> struct Traits<double> { using V = double; using U = uint64_t; };

// monotone in x; adding zero gives both zeros one key
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t key_of(double x) {
    const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
    return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
struct DrawArgs {
    const void* R;
    long long row_stride, col_stride;
    int rows, K, D;
    const double* u;
    mppi_draw_filter f;
    long long* index;
    float* weight;
    long long first;                  // row (long_draw: draw) of the launch's first workgroup
    int per;                          // draws of one workgroup
};

// ------------------------------------------------------------------------------------------
// sums, extremes and scans: lanes through DPP (no trip to LDS), waves through LDS
// ------------------------------------------------------------------------------------------
template <int CTRL, int ROWS, class X> __device__ __forceinline__ X dpp(X v, X other) {      // other where no lane is read from
    if constexpr (sizeof(X) == 4) {
        return __builtin_bit_cast(X, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, other), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    } else {
        const unsigned long long a = __builtin_bit_cast(unsigned long long, v), o = __builtin_bit_cast(unsigned long long, other);
        const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp((int)(unsigned)o, (int)(unsigned)a, CTRL, ROWS, 0xf, false);
        const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp((int)(o >> 32), (int)(a >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(X, (unsigned long long)hi << 32 | lo);
    }
}
template <class X> __device__ __forceinline__ X lane_value(X v, int lane) {                  // lane: the same in every lane
    if constexpr (sizeof(X) == 4) {
        return __builtin_bit_cast(X, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
    } else {
        const unsigned long long a = __builtin_bit_cast(unsigned long long, v);
        const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)a, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(a >> 32), lane);
        return __builtin_bit_cast(X, (unsigned long long)hi << 32 | lo);
    }
}
// inclusive, in the order of the lanes: within rows of 16, then the last lane of rows 0 and 2 into rows 1 and 3, then lane 31
// into rows 2 and 3
template <class X, class Op> __device__ __forceinline__ X wave_scan(X v, X none, Op op) {
    v = op(v, dpp<0x111, 0xf>(v, none));
    v = op(v, dpp<0x112, 0xf>(v, none));
    v = op(v, dpp<0x114, 0xf>(v, none));
    v = op(v, dpp<0x118, 0xf>(v, none));
    v = op(v, dpp<0x142, 0xa>(v, none));
    v = op(v, dpp<0x143, 0xc>(v, none));
    return v;
}
struct Add { template <class X> __device__ __forceinline__ X operator()(X a, X b) const { return a + b; } };
struct Max { template <class X> __device__ __forceinline__ X operator()(X a, X b) const { return a > b ? a : b; } };
struct Min { template <class X> __device__ __forceinline__ X operator()(X a, X b) const { return a < b ? a : b; } };

// Over the NT threads of a workgroup.  Two sets of slots in LDS are used in turn, so that one barrier is enough: who writes to a set
// again has passed the barrier of the other set, and with it everybody who had to read the first.
template <int NT> struct Group {
    unsigned long long* slots;                       // 2 NT / 64
    int flip = 0;
    __device__ Group(unsigned long long* s) : slots(s) {}
    template <class X> __device__ __forceinline__ X* next() {
        X* p = (X*)(slots + flip);
        flip = NT / 64 - flip;
        return p;
    }
    template <class X, class Op> __device__ __forceinline__ X reduce(X v, X none, Op op) {
        v = wave_scan(v, none, op);
        if (NT == 64) return lane_value(v, 63);
        const int lane = threadIdx.x & 63;
        X* tot = next<X>();
        if (lane == 63) tot[threadIdx.x >> 6] = v;
        __syncthreads();
        return lane_value(wave_scan(lane < NT / 64 ? tot[lane] : none, none, op), 63);      // (lanes behind the totals add nothing)
    }
    template <class X> __device__ __forceinline__ X scan(X v, X& total) {                   // exclusive sums
        const X inc = wave_scan(v, (X)0, Add());
        if (NT == 64) { total = lane_value(inc, 63); return inc - v; }
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        X* tot = next<X>();
        if (lane == 63) tot[wave] = inc;
        __syncthreads();
        const X own = lane < NT / 64 ? tot[lane] : (X)0;
        const X all = wave_scan(own, (X)0, Add());
        total = lane_value(all, 63);
        return lane_value(all - own, __builtin_amdgcn_readfirstlane(wave)) + inc - v;
    }
};

// ------------------------------------------------------------------------------------------
// parameters and targets
// ------------------------------------------------------------------------------------------
struct Param {
    double kappa, top_p, min_p;
    long long top_k;
    __device__ Param(const mppi_draw_filter& f, long long row)
        : kappa(f.kappa_of ? f.kappa_of[row] : f.kappa), top_p(f.top_p_of ? f.top_p_of[row] : f.top_p),
          min_p(f.min_p_of ? f.min_p_of[row] : f.min_p), top_k(f.top_k_of ? f.top_k_of[row] : f.top_k) {}
    // Values that the host has not seen, one per row: outside its range (or NaN) any of them leaves the row without samples.
    __device__ bool valid() const { return kappa >= 0.0 && kappa < INFINITY && top_p > 0.0 && top_p <= 1.0 && min_p >= 0.0 && min_p <= 1.0; }
};
// u in [0, 1) -> a whole number below the mass
__device__ __forceinline__ unsigned long long target_of(double u, unsigned long long mass) {
    const double want = u * (double)mass;
    const unsigned long long t = want > 0.0 ? (want < (double)mass ? (unsigned long long)want : mass) : 0ull;
    return t < mass ? t : mass - 1;
}

// top-p keeps the samples with less than share W of the mass W before them: less than this whole number; 0: none is kept
__device__ __forceinline__ unsigned long long share_of(double share, unsigned long long mass) {
    const double want = ceil(share * (double)mass);
    return want >= 1.0 ? (want < (double)mass ? (unsigned long long)want : mass) : 0ull;
}
// ------------------------------------------------------------------------------------------
// weights and masses of one row
// ------------------------------------------------------------------------------------------
// w[j] = exp(-d[j]) for 0 <= d < 700: 2^n e^r with r = -d - n ln 2, |r| <= ln 2 / 2 (ln 2 split into a part of 32 bits, whose product
// with n is exact, and the rest, as Cody and Waite do it), and the series of e^r up to r^12 / 12!, whose next term is below 2^-52.
// N of them side by side: one alone is a chain of dependent operations.
template <int N> __device__ __forceinline__ void exp_minus(const double (&d)[N], double (&w)[N]) {
    constexpr double C[13] = {1.0 / 479001600.0, 1.0 / 39916800.0, 1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0,
                              1.0 / 120.0, 1.0 / 24.0, 1.0 / 6.0, 0.5, 1.0, 1.0};
    double n[N], r[N];
#pragma unroll
    for (int j = 0; j < N; j++) n[j] = rint(d[j] * -1.4426950408889634);
#pragma unroll
    for (int j = 0; j < N; j++) r[j] = fma(n[j], -6.9314718036912382e-01, -d[j]);
#pragma unroll
    for (int j = 0; j < N; j++) { r[j] = fma(n[j], -1.9082149292705877e-10, r[j]); w[j] = C[0]; }
#pragma unroll
    for (int i = 1; i < 13; i++) {
#pragma unroll
        for (int j = 0; j < N; j++) w[j] = fma(w[j], r[j], C[i]);
        __builtin_amdgcn_sched_barrier(0);           // (the scheduler would line the chains up one behind the other)
    }
#pragma unroll
    for (int j = 0; j < N; j++) w[j] = ldexp(w[j], (int)n[j]);
}
// x in [0, 2^51] to the nearest whole number: added to 2^52, it lies in the low bits of the sum
__device__ __forceinline__ unsigned long long whole(double x) {
    return (unsigned long long)__double_as_longlong(x + 4503599627370496.0) & 0xfffffffffffffull;
}

template <class V> struct Weights {
    double kappa, scale;              // scale: 2^S
    double unit, top;                 // fp64: both ends may be apart by more than its range; then distances are taken in halves,
                                      // unit = 1/2, top = best unit, and kappa is twice what it was
    V best, from;                     // highest value of the row, lowest that takes part

    // Samples further behind than (S + 1) ln 2 / kappa have masses below half a unit.  (A margin covers the rounding of this
    // bound, and rounding to the type of the values cannot pass one of them.)
    __device__ __forceinline__ void set(double kappa_, V best_, V worst, int S) {
        kappa = kappa_;
        best = best_;
        scale = __longlong_as_double((long long)(1023 + S) << 52);
        const V bound = (V)((double)best - (S + 1.01) * 0.6931471805599453 / kappa * (1.0 + 1e-6));
        from = worst > bound ? worst : bound;        // (finite, as worst is)
        if (sizeof(V) == 8) {
            unit = (double)best - (double)from < INFINITY ? 1.0 : 0.5;       // (not a large kappa's: its `from` is near)
            top = unit * (double)best;
            kappa /= unit;
        }
    }
    // kappa (best - v) of a sample that takes part (of one that does not: that of the last that does)
    __device__ __forceinline__ double distance(V v) const {
        const double x = (double)(v > from ? v : from);
        return kappa * (sizeof(V) == 8 ? fma(-x, unit, top) : (double)best - x);
    }
    __device__ __forceinline__ double weight(V v) const {
        const double d[1] = {distance(v)};
        double w[1];
        exp_minus(d, w);
        return w[0];
    }
    __device__ __forceinline__ unsigned long long mass_of(V v) const { return whole(weight(v) * scale); }
    // masses of several samples, zero where bit j of live is not set or the weight is below `least`
    template <int N> __device__ __forceinline__ void masses(const V (&v)[N], unsigned live, double least, unsigned long long (&q)[N]) const {
        double d[N], w[N];
#pragma unroll
        for (int j = 0; j < N; j++) d[j] = distance(v[j]);
        exp_minus(d, w);
#pragma unroll
        for (int j = 0; j < N; j++) q[j] = (live >> j & 1u) && w[j] >= least ? whole(w[j] * scale) : 0ull;
#pragma unroll
        for (int j = 0; j < N; j++) asm volatile("" : "+v"(q[j]));         // (or each would be moved behind the test of its bit)
    }
};

// VEC samples from sample i on, those behind the end of the row as -inf
template <class T, int VEC> __device__ __forceinline__ void load_piece(const T* R, long long col_stride, long long i, int K, T (&v)[VEC]) {
    if (col_stride == 1 && i + VEC <= K) {
        __builtin_memcpy(v, R + i, sizeof(v));
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) v[j] = i + j < K ? R[(i + j) * col_stride] : minus_infinity((T*)nullptr);
    }
}

// ------------------------------------------------------------------------------------------
// the border of a prefix of the order
// ------------------------------------------------------------------------------------------
template <class V, int NT> struct BorderArea {
    static constexpr int BINS = NT == 64 ? 256 : 1024, LIST = 64;
    unsigned long long mass[BINS], slots[NT / 32], pick_before;
    V list_v[LIST], border;
    unsigned cnt[BINS], list_idx[LIST], n_list, pick_bin, pick_n;
    unsigned border_keep, border_all;                // of the border_all samples equal to the border, this many are kept
    unsigned border_idx;                             // the last of those that are kept; UINT_MAX: not known
};

// Among the samples of `src` in [low, high]: BY_COUNT: sample number `target` of the order.  BY_MASS: the last sample with less than
// `target` of the mass before it.  BY_SHARE: the same with `share` (< 1) of their whole mass for a target.  False: there is no such
// sample (too few of them; a share so small that nothing is kept, then src.from is raised to infinity).  `bottom`: about the lowest of
// them (the bins of the first pass reach down to it, the last one further).  `most`: as many samples as there can be.  Every thread has
// to call.
enum Aim { BY_COUNT, BY_MASS, BY_SHARE };
template <Aim AIM, int NT, class Src, class V>
__device__ bool find_border(Src& src, BorderArea<V, NT>& s, Group<NT>& group, unsigned long long target, double share, V low, V high, V bottom,
                            unsigned most) {
    using U = typename Traits<V>::U;
    using Area = BorderArea<V, NT>;
    constexpr bool MASS = AIM != BY_COUNT;
    constexpr int BINS = Area::BINS, PER = BINS / NT, LIST = Area::LIST, VEC = Src::VEC;
    // bins linear in high - v first (monotone: every step rounds monotonically); per = 0 where that range overflows
    const V per = high > bottom ? (V)BINS / (high - bottom) : (V)0;
    V lo = low, hi = high;
    int shift = -1, bin = 0;                         // -1: linear bins; else bits of key(hi) - key(v)
    U top = 0;
    unsigned long long before = 0;
    unsigned n = most;
    const auto linear = [&](V v) -> int { return bin_of((high - v) * per, BINS); };
    const auto keyed = [&](V v) -> int { return (int)((top - key_of(v)) >> shift); };
    const auto fill = [&](auto bin_of) {
        src.each(lo, hi, [&](const V (&v)[VEC], unsigned live, int) {
            unsigned long long q[VEC];
            if (MASS) src.w.masses(v, live, 0.0, q);
#pragma unroll
            for (int j = 0; j < VEC; j++)
                if (live >> j & 1u) {
                    const int b = bin_of(v[j]);
                    atomicAdd(&s.cnt[b], 1u);
                    if (MASS) atomicAdd(&s.mass[b], q[j]);
                }
        });
    };
    const auto ends = [&](auto bin_of) {             // the values of the bin, from its lowest to its highest
        V first = (V)-INFINITY, last = (V)INFINITY;
        src.each(lo, hi, [&](const V (&v)[VEC], unsigned live, int) {
#pragma unroll
            for (int j = 0; j < VEC; j++)
                if ((live >> j & 1u) && bin_of(v[j]) == bin) { first = v[j] > first ? v[j] : first; last = v[j] < last ? v[j] : last; }
        });
        lo = group.reduce(last, (V)INFINITY, Min());
        hi = group.reduce(first, (V)-INFINITY, Max());
    };
    const auto gather = [&](auto bin_of) {           // the places first, then room for all of the thread's at once
        unsigned long long hits = 0;
        const auto enlist = [&](unsigned long long bits, int first) {
            unsigned e = atomicAdd(&s.n_list, (unsigned)__popcll(bits));
#pragma unroll 1
            for (; bits; bits &= bits - 1) {
                const int at = first + __ffsll((long long)bits) - 1;
                s.list_v[e] = src.value(at / VEC, at % VEC);
                s.list_idx[e] = src.index(at / VEC, at % VEC);
                e++;
            }
        };
        src.each(lo, hi, [&](const V (&v)[VEC], unsigned live, int o) {
            unsigned hit = 0;
#pragma unroll
            for (int j = 0; j < VEC; j++) hit |= (live >> j & 1u) && bin_of(v[j]) == bin ? 1u << j : 0u;
            if (o < 64 / VEC) hits |= (unsigned long long)hit << (o * VEC);
            else if (hit) enlist(hit, o * VEC);      // (sources of more than 64 samples per thread)
        });
        if (hits) enlist(hits, 0);
    };
    if (NT == 64) __syncthreads();                   // (larger groups have just met at a barrier)
    if (threadIdx.x == 0) s.n_list = 0;
    if (most > 16) {     // (comparing more with each other costs more than the histogram: 1024 x 512 11.5 us with it, 13.9 without)
#pragma unroll 1
        while (true) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                s.cnt[threadIdx.x + i * NT] = 0;
                if (MASS) s.mass[threadIdx.x + i * NT] = 0;
            }
            __syncthreads();
            if (shift < 0) fill(linear); else fill(keyed);
            __syncthreads();
            unsigned long long own[PER], sum = 0, total;
            unsigned c[PER];
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int b = threadIdx.x * PER + i;
                c[i] = s.cnt[b];
                own[i] = MASS ? s.mass[b] : (unsigned long long)c[i];
                sum += own[i];
            }
            unsigned long long run = before + group.scan(sum, total);
            if (shift < 0) {
                if (AIM == BY_SHARE) {
                    target = share_of(share, total);
                    if (target == 0) { src.w.from = (V)INFINITY; return false; }
                }
                if (total < target) return false;
            }
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (run < target && target <= run + own[i]) {
                    s.pick_bin = threadIdx.x * PER + i;
                    s.pick_n = c[i];
                    s.pick_before = run;
                }
                run += own[i];
            }
            __syncthreads();
            bin = (int)s.pick_bin;
            n = s.pick_n;
            before = s.pick_before;
            if (n <= LIST) break;
            if (shift < 0) ends(linear); else ends(keyed);
            if (lo == hi) break;
            top = key_of(hi);
            shift = 0;
            while (((top - key_of(lo)) >> shift) >= (U)BINS) shift++;
        }
    } else {
        bin = -1;                                    // (no binning: all of them are candidates)
        __syncthreads();
    }
    if (n > LIST) {                                  // all n of one return
        if (threadIdx.x == 0) {
            s.border = lo;
            s.border_all = n;
            const unsigned long long one = MASS ? src.w.mass_of(lo) : 1ull;
            s.border_keep = (unsigned)((target - before + one - 1) / one);
            s.border_idx = UINT_MAX;
        }
        __syncthreads();
        return true;
    }
    if (bin < 0) gather([](V) { return -1; });
    else if (shift < 0) gather(linear);
    else gather(keyed);
    __syncthreads();
    if (threadIdx.x < 64) {                          // the first wave compares each with each
        static_assert(LIST == 64, "a candidate per lane");
        const int lane = threadIdx.x;
        n = __builtin_amdgcn_readfirstlane(s.n_list);
        const bool in = lane < (int)n;
        const V v = in ? s.list_v[lane] : (V)-INFINITY;
        const unsigned idx = in ? s.list_idx[lane] : UINT_MAX;
        const unsigned long long q = in ? (MASS ? src.w.mass_of(v) : 1ull) : 0ull;
        unsigned long long run = before, all = 0;    // run: what lies before this lane's candidate in the order
        unsigned rank = 0;
        const unsigned long long place = (unsigned long long)(sizeof(V) == 4 ? (U)key_of(v) : (U)0) << 32 | (unsigned)~idx;
        for (unsigned o = 0; o < n; o++) {
            bool first;
            if constexpr (sizeof(V) == 4) {          // value and index in one number
                first = lane_value(place, o) > place;
            } else {
                const V ov = lane_value(v, o);
                first = ov > v || (ov == v && lane_value(idx, o) < idx);
            }
            if (MASS) {
                const unsigned long long oq = lane_value(q, o);
                all += oq;
                run += first ? oq : 0ull;
            } else {
                rank += first ? 1u : 0u;
            }
        }
        if (!MASS) { run += rank; all = n; }
        bool some = true;
        if (bin < 0) {                               // what the histogram would have said
            if (AIM == BY_SHARE) target = share_of(share, all);
            some = target > 0 && all >= target;
            if (lane == 0) s.pick_n = some ? 1u : target == 0 ? 2u : 0u;
        }
        const unsigned long long here = __ballot(some && run < target && target <= run + q);
        if (here) {
            const int at = __builtin_amdgcn_readfirstlane(__ffsll((long long)here) - 1);
            const V border = lane_value(v, at);
            const unsigned last = lane_value(idx, at);
            const unsigned long long same = __ballot(in && v == border), kept = __ballot(in && v == border && idx <= last);
            if (lane == 0) {
                s.border = border;
                s.border_all = (unsigned)__popcll(same);
                s.border_keep = (unsigned)__popcll(kept);
                s.border_idx = last;
            }
        }
    }
    __syncthreads();
    if (bin < 0) {
        const unsigned said = s.pick_n;
        if (said == 2u) src.w.from = (V)INFINITY;
        if (said != 1u) { __syncthreads(); return false; }
    }
    return true;
}

// ------------------------------------------------------------------------------------------
// rows of up to 128 KB: one workgroup each
// ------------------------------------------------------------------------------------------
// The row lies in LDS as it came, behind its end -inf; what is not finite fails the comparison with the lowest or the highest.
// Thread t owns the C samples from t C on, in GP pieces of 16 bytes; it visits them from piece t mod GP on, so that the lanes of
// a wave read from all banks.  All loops over samples stay rolled: unrolled, or with the row in registers, a kernel of this many
// passes is larger than the instruction cache (192 x 65535 bf16: 424 us in registers, 88 with the same passes over LDS).  A pass
// tests values against the lowest one that takes part, in the type of the row (fp32 or fp64); exponentials, in fp64, are evaluated
// only for pieces with a sample that passes (88 -> 62 us).
template <class T, int NT, int BYTES> struct Shelf {
    using V = typename Traits<T>::V;
    static constexpr int VEC = 16 / sizeof(T);
    static constexpr int FEW = NT >= 512 ? 1024 : 64;          // up to this many samples that take part can move together
    static constexpr int LAST = 64;                            // up to this many are left to one wave (finish): a sample per lane
    struct alignas(16) Piece { T v[VEC]; };
    using Area = BorderArea<V, NT>;
    struct Shared {
        Piece row[BYTES / 16];
        Area b;
        __device__ unsigned* few_idx() { return (unsigned*)&row[FEW / VEC]; }       // (behind what has moved together)
        __device__ unsigned long long* ends() { return b.mass; }           // (once the borders are found; NT <= BINS)
    };
    Shared& s;
    Weights<V> w;
    int GP, start;                    // pieces of this thread, the one it begins with
    bool moved;                       // the row is what has moved together
    int C;                            // samples per thread

    V bottom;                         // about the lowest value that takes part (at first)
    Group<NT> group;
    unsigned most;                    // samples that can take part

    __device__ Shelf(Shared& s_) : s(s_), group(s_.b.slots) {}
    __device__ __forceinline__ static V at(const Piece& p, int j) { return value_of(p.v[j]); }
    // the thread's pieces in the order in which it visits them
    __device__ __forceinline__ int piece(int o) const { const int g = start + o; return (int)threadIdx.x * GP + (g < GP ? g : g - GP); }
    __device__ __forceinline__ V value(int o, int j) const { return at(s.row[piece(o)], j); }
    __device__ __forceinline__ unsigned index(int o, int j) const { return (unsigned)(piece(o) * VEC + j); }

    // f(v, live, o): the pieces with samples in [low, high]; live: bit j for sample v[j] of the o-th piece visited
    template <class F> __device__ __forceinline__ void each(V low, V high, F f) {
        const int own = (int)threadIdx.x * GP;
        int g = start;
#pragma unroll 1
        for (int o = 0; o < GP; o++) {
            const Piece p = s.row[own + g];
            V v[VEC];
            unsigned live = 0;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                v[j] = at(p, j);
                live |= v[j] >= low && v[j] <= high ? 1u << j : 0u;
            }
            if (live) f(v, live, o);
            g = g + 1 == GP ? 0 : g + 1;
        }
    }

    // Raises w.from to a value that at least k threads' own values `mine` reach (one per thread), near the highest such.
    __device__ void raise(V mine, unsigned k) {
        constexpr int BINS = Area::BINS, PER = BINS / NT;
        const V per = w.best > bottom ? (V)BINS / (w.best - bottom) : (V)0;
        const bool in = mine >= w.from;
        const int b = in ? bin_of((w.best - mine) * per, BINS) : 0;
#pragma unroll
        for (int i = 0; i < PER; i++) s.b.cnt[threadIdx.x + i * NT] = 0;
        __syncthreads();
        if (in) atomicAdd(&s.b.cnt[b], 1u);
        __syncthreads();
        unsigned own[PER], sum = 0, total;
#pragma unroll
        for (int i = 0; i < PER; i++) { own[i] = s.b.cnt[threadIdx.x * PER + i]; sum += own[i]; }
        unsigned run = group.scan(sum, total);
        if (total < k) return;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (run < k && k <= run + own[i]) s.b.pick_bin = threadIdx.x * PER + i;
            run += own[i];
        }
        __syncthreads();
        const V low = in && b <= (int)s.b.pick_bin ? mine : (V)INFINITY;
        w.from = group.reduce(low, (V)INFINITY, Min());
    }

    // If few samples take part, they move together (in their order, with their indices), and the passes that follow go over
    // them alone.  top[p]: highest value of piece p NT + t, as thread t loaded them, so that most pieces need not be looked at again.
    template <int P> __device__ void gather_few(const V (&top)[P]) {
        static_assert(P <= 8, "two words of four counts");
        unsigned long long bits = 0, mine[2] = {0, 0}, total[2] = {0, 0};  // bit p VEC + j; samples by piece, 16 bits each
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (p < GP && top[p] >= w.from) {
                const Piece x = s.row[p * NT + (int)threadIdx.x];
                unsigned in = 0;
#pragma unroll
                for (int j = 0; j < VEC; j++) in |= at(x, j) >= w.from && at(x, j) <= w.best ? 1u << j : 0u;
                bits |= (unsigned long long)in << (p * VEC);
                mine[p / 4] += (unsigned long long)__popc(in) << (p % 4 * 16);
            }
        }
        unsigned long long to[2] = {group.scan(mine[0], total[0]), group.scan(mine[1], total[1])};
        unsigned all = 0;                            // (at most 1024 threads of 8 samples: every count fits)
#pragma unroll
        for (int p = 0; p < P; p++) {
            if (all <= FEW) to[p / 4] += (unsigned long long)all << (p % 4 * 16);
            all += (unsigned)(total[p / 4] >> (p % 4 * 16) & 0xffffu);
        }
        most = all;
        if (all > FEW) return;
        // over the areas of the histogram, and from there to where the row was
        static_assert(FEW <= Area::BINS && FEW * (sizeof(T) + 4) <= BYTES, "values and indices");
        T* values = (T*)s.b.mass;
        for (int e = (int)all + (int)threadIdx.x; e < FEW; e += NT) values[e] = minus_infinity((T*)nullptr);
#pragma unroll 1
        for (; bits; bits &= bits - 1) {             // (in the order of the pieces, and in it within each)
            const int at = __ffsll((long long)bits) - 1, p = at / VEC, j = at % VEC, from = p * NT + (int)threadIdx.x;
            const int field = p % 4 * 16;
            const unsigned e = (unsigned)((p < 4 ? to[0] : to[1]) >> field & 0xffffu);
            if (p < 4) to[0] += 1ull << field; else to[1] += 1ull << field;
            values[e] = s.row[from].v[j];
            s.b.cnt[e] = (unsigned)(from * VEC + j);
        }
        __syncthreads();
        for (int e = threadIdx.x; e < FEW; e += NT) {
            s.row[e / VEC].v[e % VEC] = values[e];
            s.few_idx()[e] = s.b.cnt[e];
        }
        __syncthreads();
        moved = true;
        GP = threadIdx.x < FEW / VEC ? 1 : 0;
        start = 0;
        C = VEC;
    }

    // The rest of the way for n <= 64 samples in the order of their indices, by one wave, a sample per lane: ranks by comparing each with
    // each, masses in the order of the ranks for top-p, and in that of the indices for the draws.  The lane's sample, its weight, its
    // mass (0: it may not be drawn) and the mass before it; returns the whole mass.
    __device__ unsigned long long finish(unsigned n, const Param& par, V& v, double& weight, unsigned long long& q, unsigned long long& before) {
        const unsigned lane = threadIdx.x & 63;
        const bool by_count = par.top_k > 0 && par.top_k < (long long)n, by_share = !(par.top_p >= 1.0);
        v = lane < n ? at(s.row[lane / VEC], lane % VEC) : (V)-INFINITY;
        bool live = v >= w.from && v <= w.best;
        v = live ? v : (V)-INFINITY;
        weight = w.weight(v);
        const unsigned long long mass = whole(weight * w.scale);
        if (by_count || by_share) {
            unsigned rank = 0;
            if constexpr (sizeof(V) == 4) {          // value and index in one number (16-bit returns are often equal); the others come last
                const unsigned long long place = (unsigned long long)key_of(v) << 32 | (63u - lane);
                for (unsigned o = 0; o < n; o += 4) {
#pragma unroll
                    for (unsigned j = 0; j < 4; j++) rank += lane_value(place, o + j) > place ? 1u : 0u;
                }
            } else {                                 // how many are higher, and where there are equal ones, how many of these come first
                const V x = live ? v : (V)NAN;
                for (unsigned o = 0; o < n; o += 4) {
#pragma unroll
                    for (unsigned j = 0; j < 4; j++) rank += lane_value(x, o + j) > x ? 1u : 0u;
                }
                const unsigned all = (unsigned)__popcll(__ballot(live));
                if (lane_value(wave_scan(live ? rank : 0u, 0u, Add()), 63) != all * (all - 1) / 2) {
                    for (unsigned o = 0; o < n; o += 4) {
#pragma unroll
                        for (unsigned j = 0; j < 4; j++) rank += lane_value(x, o + j) == x && o + j < lane ? 1u : 0u;
                    }
                }
                rank = live ? rank : 63u;            // (where some lane takes no part, no rank is 63)
            }
            if (by_count) live = live && (long long)rank < par.top_k;
            if (by_share) {
                const unsigned long long m = live ? mass : 0ull;
                const int to = (int)rank * 4;
                const unsigned long long sorted = (unsigned long long)(unsigned)__builtin_amdgcn_ds_permute(to, (int)(m >> 32)) << 32 |
                                                  (unsigned)__builtin_amdgcn_ds_permute(to, (int)(unsigned)m);
                const unsigned long long inc = wave_scan(sorted, 0ull, Add()), ahead = inc - sorted;
                const unsigned long long own = (unsigned long long)(unsigned)__builtin_amdgcn_ds_bpermute(to, (int)(ahead >> 32)) << 32 |
                                               (unsigned)__builtin_amdgcn_ds_bpermute(to, (int)(unsigned)ahead);
                live = live && own < share_of(par.top_p, lane_value(inc, 63));
            }
        }
        q = live && weight >= par.min_p ? mass : 0ull;
        const unsigned long long inc = wave_scan(q, 0ull, Add());
        before = inc - q;
        return lane_value(inc, 63);
    }

    // leaves out what lies behind the border that was found
    __device__ void cut_behind() {
        w.from = s.b.border;
        const unsigned keep = s.b.border_keep;
        if (keep < s.b.border_all) {                 // of the equal ones, the first in the order of the samples stay
            unsigned mine = 0, total;
            each(w.from, w.from, [&](const V (&)[VEC], unsigned live, int) { mine += (unsigned)__popc(live); });
            unsigned rank = group.scan(mine, total);
#pragma unroll 1
            for (int g = 0; g < GP && mine > 0; g++) {
                Piece& p = s.row[(int)threadIdx.x * GP + g];
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (at(p, j) == w.from && rank++ >= keep) p.v[j] = minus_infinity((T*)nullptr);
            }
        }
        __syncthreads();                             // the border may be written again
    }
};

template <class T, int NT, int BYTES> __global__ void __launch_bounds__(NT) draw_row_kernel(DrawArgs a, int S) {
    using H = Shelf<T, NT, BYTES>;
    using V = typename H::V;
    using Piece = typename H::Piece;
    constexpr int VEC = H::VEC, NW = NT / 64;
    __shared__ typename H::Shared s;
    H h(s);
    const long long row = a.first + blockIdx.x, from_draw = row * a.D + (long long)blockIdx.y * a.per;
    const int D = min(a.per, (int)(a.D - (long long)blockIdx.y * a.per));
    const T* R = (const T*)a.R + row * a.row_stride;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    h.GP = (a.K + NT * VEC - 1) / (NT * VEC);
    h.C = h.GP * VEC;
    h.start = tid % h.GP;
    h.moved = false;
    h.most = (unsigned)a.K;
    const Param par(a.f, row);
    long long* index = a.index + from_draw;
    float* weight = a.weight ? a.weight + from_draw : nullptr;
    const double* u = a.u + from_draw;
    auto nothing = [&]() {
        for (int d = tid; d < D; d += NT) { index[d] = -1; if (weight) weight[d] = 0.0f; }
    };

    const double u_wave = wave < D ? u[wave] : 0.0, u_thread = tid < D ? u[tid] : 0.0;      // asked for before anything waits
    // the row into LDS, AHEAD pieces requested at a time
    constexpr int AHEAD = BYTES >= 65536 ? 8 : 4, DIRECT = 8;
    V best = (V)-INFINITY, some = (V)INFINITY, top[AHEAD];               // some: the lowest of every fourth sample
#pragma unroll 1
    for (int p0 = 0; p0 < h.GP; p0 += AHEAD) {                            // (once where few samples may move together)
        Piece in[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) load_piece(R, a.col_stride, (long long)((p0 + k) * NT + tid) * VEC, a.K, in[k].v);
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            if (p0 + k >= h.GP) break;
            top[k] = (V)-INFINITY;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const V v = H::at(in[k], j), fine = isfinite(v) ? v : (V)-INFINITY;
                top[k] = fine > top[k] ? fine : top[k];
                if (j % 4 == 0) some = isfinite(v) && v < some ? v : some;
            }
            best = top[k] > best ? top[k] : best;
            s.row[(p0 + k) * NT + tid] = in[k];
        }
    }
    const V mine = best;                                                  // best of what this thread loaded
    best = h.group.reduce(best, (V)-INFINITY, Max());
    some = h.group.reduce(some, (V)INFINITY, Min());
    if (NT == 64) __syncthreads();                                        // (the row is there; larger groups have just waited)
    if (!par.valid() || !(best > (V)-INFINITY)) return nothing();
    h.w.set(par.kappa, best, lowest((V*)nullptr), S);
    h.bottom = some > h.w.from && some <= best ? some : h.w.from;

    auto answer = [&](int d, int i, double w, unsigned long long mass) {
        index[d] = h.moved ? (long long)s.few_idx()[i] : i;
        if (weight) weight[d] = (float)(w * h.w.scale / (double)mass);
    };
    auto finish = [&]() __attribute__((always_inline)) {                  // few samples: the first wave does the rest
        const unsigned n = h.most;
        unsigned long long mass = 0;
        if (wave == 0) {
            V v;
            double own;
            unsigned long long q, before;
            mass = h.finish(n, par, v, own, q, before);
            if (D <= DIRECT) {
                for (int d = 0; d < D; d++) {
                    const unsigned long long target = mass ? target_of(d == 0 ? u_wave : u[d], mass) : 0ull;
                    if (target - before < q) answer(d, lane, own, mass);
                    if (mass == 0 && lane == 0) { index[d] = -1; if (weight) weight[d] = 0.0f; }
                }
                return;
            }
            s.ends()[lane] = before + q;
        }
        if (D <= DIRECT) return;
        __syncthreads();                                                  // many draws: a thread each
        const unsigned long long* ends = s.ends();
        mass = ends[63];
        if (mass == 0) return nothing();
        for (int d = tid; d < D; d += NT) {
            const unsigned long long target = target_of(d == tid ? u_thread : u[d], mass);
            int lo = 0, hi = (int)n - 1;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (ends[mid] > target) hi = mid; else lo = mid + 1;
            }
            answer(d, lo, h.w.weight(H::at(s.row[lo / VEC], lo % VEC)), mass);
        }
    };
    static_assert(AHEAD * NT * 16 >= BYTES, "the row is loaded in one go, and top[] holds all of its pieces");
    bool few = BYTES < 131072 && a.K <= H::LAST;
    // Each thread's best is one sample, so the k best threads bound the k best samples from below, and with many samples per thread
    // little else passes that bound: what passes moves together, and the passes that follow go over it alone.  Up to NT / 2: beyond,
    // more passes than can move (64 x 65535 bf16, k = 512: 56 us without the bound, 24 with it; k = 800: 55 and 56).  With two
    // pieces per thread it gains little without top-p behind it (64 x 4096 fp32, k = 200: 9.3 and 10.2, with top-p 13.2 and 12.9),
    // with four much (64 x 8192: 11.5 and 10.4, with top-p 17.9 and 13.3).
    const bool raised = NT >= 512 && par.top_k > 0 && par.top_k <= NT / 2 && h.GP > 1;
    if (raised) h.raise(mine, (unsigned)par.top_k);
    if (raised || BYTES >= 131072) {
        h.gather_few(top);
        few = h.moved && h.most <= H::LAST;
    }
    if (!few && par.top_k > 0 && par.top_k < a.K && find_border<BY_COUNT>(h, s.b, h.group, (unsigned long long)par.top_k, 0.0, h.w.from, best, h.bottom, h.most)) {
        h.cut_behind();
        h.bottom = h.w.from;
        h.most = h.most < par.top_k ? h.most : (unsigned)par.top_k;
        if (BYTES < 131072 && !h.moved && h.most <= H::LAST) {
            h.gather_few(top);
            few = true;
        }
    }
    if (few) return finish();
    if (!(par.top_p >= 1.0) && find_border<BY_SHARE>(h, s.b, h.group, 0, par.top_p, h.w.from, best, h.bottom, h.most)) h.cut_behind();

    unsigned long long sum = 0, mass;
    h.each(h.w.from, best, [&](const V (&v)[VEC], unsigned live, int) {
        unsigned long long q[VEC];
        h.w.masses(v, live, par.min_p, q);
#pragma unroll
        for (int j = 0; j < VEC; j++) sum += q[j];
    });
    const unsigned long long base = h.group.scan(sum, mass);
    if (mass == 0) return nothing();
    unsigned long long* ends = s.ends();
    ends[tid] = base + sum;
    __syncthreads();
    // mass of sample i of the row, zero if it may not be drawn
    auto mass_of_sample = [&](int i, double& w) -> unsigned long long {
        const V v = H::at(s.row[i / VEC], i % VEC);
        w = h.w.weight(v);
        return v >= h.w.from && v <= best && w >= par.min_p ? whole(w * h.w.scale) : 0ull;
    };
    const int C = h.C;
    // A wave for every draw, or a thread for every draw: a round of the waves takes about as long as two pieces of the threads' walks
    // (256 rows of 30000 fp32: 64 draws 25.3 us by waves, 25.7 by threads, 128 draws 30.1 and 26.0).
    if ((D + NW - 1) / NW * 2 - 1 <= (D + NT - 1) / NT * (C / VEC)) {
#pragma unroll 1
        for (int d = wave; d < D; d += NW) {
            const unsigned long long target = target_of(d == wave ? u_wave : u[d], mass);
            int owner = 0;                                     // number of threads that end at or below the target
#pragma unroll
            for (int k = 0; k < NW; k++) owner += __popcll(__ballot(ends[k * 64 + lane] <= target));
            const unsigned long long ahead = owner > 0 ? ends[owner - 1] : 0ull;
            double w = 0.0;
            const unsigned long long m = lane < C ? mass_of_sample(owner * C + lane, w) : 0ull;      // C <= 64
            const unsigned long long at = ahead + wave_scan(m, 0ull, Add()) - m;
            if (target - at < m) answer(d, owner * C + lane, w, mass);
        }
    } else {
        double next = u_thread;
#pragma unroll 1
        for (int d = tid; d < D; d += NT) {
            const unsigned long long target = target_of(next, mass);
            next = d + NT < D ? u[d + NT] : 0.0;
            int lo = 0, hi = NT - 1;                           // the first thread that ends above the target
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (ends[mid] > target) hi = mid; else lo = mid + 1;
            }
            unsigned long long c = lo > 0 ? ends[lo - 1] : 0ull;
#pragma unroll 1
            for (int p = lo * C / VEC; p < (lo + 1) * C / VEC; p++) {
                const Piece x = s.row[p];
                V v[VEC];
                unsigned live = 0;
                unsigned long long q[VEC], sum = 0;
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    v[j] = H::at(x, j);
                    live |= v[j] >= h.w.from && v[j] <= best ? 1u << j : 0u;
                }
                h.w.masses(v, live, par.min_p, q);
#pragma unroll
                for (int j = 0; j < VEC; j++) sum += q[j];
                if (target - c < sum) {
                    V chosen = v[0];
                    int at = 0;
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        if (target - c < q[j]) { chosen = v[j]; at = j; }
                        c += q[j];
                    }
                    answer(d, p * VEC + at, h.w.weight(chosen), mass);
                    break;
                }
                c += sum;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------
// longer rows: a workgroup for every chunk of 4096 or 8192 samples, up to five launches
// ------------------------------------------------------------------------------------------
//   chunk_best    highest, lowest and summed weight of every chunk; clears what the next ones add to
//   chunk_bins    counts and masses over bins linear in best - v, a histogram per row
//   chunk_split   the bins in which the borders can lie follow from the histogram: mass of what lies before them by chunk and by
//                 segment (the 64 VEC samples that one wave holds in one piece each), and a list of the samples in them
//   row_border    the borders among the listed samples; their masses join those of their chunks; up to 4 draws
//   long_draw     more draws, a wave for each: the chunk, then the segment, then the sample
// Rows without top-k and top-p need no list: the masses of their chunks stay as chunk_bins wrote them, and long_draw follows.
//
// Each of the first three reads the row once, and only the first finds it outside the caches (in part: an L2 holds 4 MB).  A launch
// takes 4 us by itself; by kernel, 1 x 524288 fp32 (2 MB): 3.9, 8.3, 6.7, 9.5 us; 16 x 262144 fp64 (34 MB) and 64 draws: 10.8, 13.5,
// 16.2, 15.5, 4.8 us, i.e. 3.1 TB/s for the reading alone and 2.1 to 2.5 TB/s with fp64 exponentials (some 20 operations of 4 cycles
// each for a wave) in the two that need masses.
constexpr int MOST_SEGS = 64, LT = 512, LONG_BINS = 1024, BT = 256;

// Where the borders can lie: the count border in bin k (-1: none) with so many samples and so much mass before it, the mass border in
// bins p_first ... p_last (none: p_first > p_last)
struct Where {
    int k, p_first, p_last;
    unsigned k_before;
    unsigned long long k_mass_before, mass_before;   // mass_before: before p_first
    unsigned long long mass;                         // of all bins
    bool nothing;
};
template <class V> struct LongRow {                  // what is known of a row (written by its first workgroup of chunk_bins)
    Weights<V> w;
    Where at;                                        // (of chunk_split)
    V border;                                        // kept: above the border, or equal to it with an index up to last
    unsigned last, listed;
    int state;                                       // 0: nothing to draw, 1: every sample that takes part is kept, 2: borders
};
// log2 of a chunk's samples: smaller ones where there would be up to 128 workgroups (per call, top-p alone, 4096 and 8192: 1 x 70000 39 us and 44, 1 x 524288
// 37 and 40; more of them add more to the histogram: 16 x 262144 fp64 58 and 57, 1 x 4000000 with top-k 64 and 51).
__host__ __device__ __forceinline__ int chunk_shift(size_t rows, size_t K) { return rows * K <= (size_t)1 << 20 ? 12 : 13; }
template <class V> struct LongArea {                 // the workspace, of all rows
    V *best, *worst;                                 // [rows][chunks]
    double* sum;
    unsigned long long *kept, *seg, *mass;           // mass of a chunk, [rows][chunks], and of its segments, [MOST_SEGS]; [rows][LONG_BINS]
    unsigned* cnt;
    LongRow<V>* row;
    V* list_v;                                       // [rows][K]
    unsigned* list_i;
    int chunks;
    static size_t carve(LongArea* a, char* p, size_t rows, size_t K) {
        const int shift = chunk_shift(rows, K);
        const size_t chunks = (K + (1u << shift) - 1) >> shift;
        size_t at = 0;
        auto take = [&](size_t bytes) { char* r = p + at; at += (bytes + 255) & ~(size_t)255; return r; };
        LongArea local;
        if (!a) a = &local;
        a->best = (V*)take(rows * chunks * sizeof(V));
        a->worst = (V*)take(rows * chunks * sizeof(V));
        a->sum = (double*)take(rows * chunks * 8);
        a->kept = (unsigned long long*)take(rows * chunks * 8);
        a->seg = (unsigned long long*)take(rows * chunks * MOST_SEGS * 8);
        a->mass = (unsigned long long*)take(rows * LONG_BINS * 8);
        a->cnt = (unsigned*)take(rows * LONG_BINS * 4);
        a->row = (LongRow<V>*)take(rows * sizeof(LongRow<V>));
        a->list_v = (V*)take(rows * K * sizeof(V));
        a->list_i = (unsigned*)take(rows * K * 4);
        a->chunks = (int)chunks;
        return at;
    }
};

// the chunk of this workgroup, HELD samples per thread, in pieces of VEC neighbours
template <class T> constexpr int segment = 64 * (16 / (int)sizeof(T));       // samples that one wave holds in a piece per lane
template <class T, int CHUNK> struct Chunk {
    using V = typename Traits<T>::V;
    static constexpr int HELD = CHUNK / LT, VEC = 16 / sizeof(T), PIECES = HELD / VEC, SEGS = CHUNK / segment<T>;
    static_assert(SEGS <= MOST_SEGS, "");
    V x[PIECES][VEC];
    int first;                                       // index of x[0][0]
    __device__ __forceinline__ int index(int p, int j) const { return first + p * LT * VEC + j; }
    __device__ __forceinline__ void load(const DrawArgs& a, long long row, int chunk) {
        const T* R = (const T*)a.R + row * a.row_stride;
        T raw[PIECES][VEC];
        first = chunk * CHUNK + (int)threadIdx.x * VEC;
#pragma unroll
        for (int p = 0; p < PIECES; p++) load_piece(R, a.col_stride, index(p, 0), a.K, raw[p]);
#pragma unroll
        for (int p = 0; p < PIECES; p++)
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                x[p][j] = value_of(raw[p][j]);
                x[p][j] = isfinite(x[p][j]) ? x[p][j] : (V)-INFINITY;
            }
    }
    // mass of every segment and of the chunk from those of the thread's pieces
    __device__ __forceinline__ static void store(const unsigned long long (&sum)[PIECES], Group<LT>& group, unsigned long long* seg, unsigned long long* kept) {
        unsigned long long all = 0;
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
            const unsigned long long inc = wave_scan(sum[p], 0ull, Add());
            if ((threadIdx.x & 63) == 63) seg[p * (LT / 64) + (threadIdx.x >> 6)] = inc;
            all += sum[p];
        }
        all = group.reduce(all, 0ull, Add());
        if (threadIdx.x == 0) *kept = all;
    }
    __device__ __forceinline__ unsigned live(int p, V low) const {
        unsigned bits = 0;
#pragma unroll
        for (int j = 0; j < VEC; j++) bits |= x[p][j] >= low ? 1u << j : 0u;
        return bits;
    }
};

__device__ __forceinline__ bool wants_border(const Param& par, int K) { return (par.top_k > 0 && par.top_k < K) || !(par.top_p >= 1.0); }

template <class T, int CHUNK> __global__ void __launch_bounds__(LT, 4) chunk_best_kernel(DrawArgs a, LongArea<typename Traits<T>::V> l) {
    using V = typename Traits<T>::V;
    __shared__ unsigned long long s_slots[LT / 32];
    Group<LT> group(s_slots);
    const long long row = blockIdx.x / l.chunks;
    const int chunk = (int)(blockIdx.x - row * l.chunks);
    Chunk<T, CHUNK> c;
    c.load(a, row, chunk);
    const Param par(a.f, row);
    for (int i = chunk * LT + (int)threadIdx.x; i < LONG_BINS; i += l.chunks * LT) {
        l.mass[row * LONG_BINS + i] = 0;
        l.cnt[row * LONG_BINS + i] = 0;
    }
    if (chunk == 0 && threadIdx.x == 0) l.row[row].listed = 0;
    V best = (V)-INFINITY, worst = (V)INFINITY;
#pragma unroll
    for (int p = 0; p < c.PIECES; p++)
#pragma unroll
        for (int j = 0; j < c.VEC; j++) {
            const V v = c.x[p][j];
            best = v > best ? v : best;
            worst = v > (V)-INFINITY && v < worst ? v : worst;
        }
    best = group.reduce(best, (V)-INFINITY, Max());
    worst = group.reduce(worst, (V)INFINITY, Min());
    double sum = 0.0;
    if (par.valid() && best > (V)-INFINITY) {
        Weights<V> w;
        w.set(par.kappa, best, worst, 51);
        float some = 0.0f;                           // (it says how large the sums become; fp32 is enough for that)
#pragma unroll
        for (int p = 0; p < c.PIECES; p++)
#pragma unroll
            for (int j = 0; j < c.VEC; j++) some += c.x[p][j] >= w.from ? __expf(-(float)w.distance(c.x[p][j])) : 0.0f;
        sum = some;
    }
    sum = group.reduce(sum, 0.0, Add());
    if (threadIdx.x == 0) {
        l.best[blockIdx.x] = best;
        l.worst[blockIdx.x] = worst;
        l.sum[blockIdx.x] = sum;
    }
}

// bins of a long row
template <class V> struct LongBins {
    V best, per;
    __device__ LongBins(const Weights<V>& w) : best(w.best), per(w.best > w.from ? (V)LONG_BINS / (w.best - w.from) : (V)0) {}
    __device__ __forceinline__ int of(V v) const { return bin_of((best - v) * per, LONG_BINS); }
};

template <class T, int CHUNK> __global__ void __launch_bounds__(LT, 4) chunk_bins_kernel(DrawArgs a, LongArea<typename Traits<T>::V> l) {
    using V = typename Traits<T>::V;
    __shared__ unsigned long long s_slots[LT / 32], s_mass[LONG_BINS];
    Group<LT> group(s_slots);
    __shared__ unsigned s_cnt[LONG_BINS];
    const long long row = blockIdx.x / l.chunks;
    const int chunk = (int)(blockIdx.x - row * l.chunks);
    Chunk<T, CHUNK> c;
    c.load(a, row, chunk);
    const Param par(a.f, row);
    // the row's best, worst and mass from those of its chunks
    V best = (V)-INFINITY, worst = (V)INFINITY;
    for (int i = threadIdx.x; i < l.chunks; i += LT) {
        const V b = l.best[row * l.chunks + i], w = l.worst[row * l.chunks + i];
        best = b > best ? b : best;
        worst = w < worst ? w : worst;
    }
    best = group.reduce(best, (V)-INFINITY, Max());
    worst = group.reduce(worst, (V)INFINITY, Min());
    const bool some = par.valid() && best > (V)-INFINITY;
    Weights<V> w;
    int state = 0;
    if (some) {
        w.set(par.kappa, best, worst, 51);
        double sum = 0.0;
        for (int i = threadIdx.x; i < l.chunks; i += LT) {
            const V b = l.best[row * l.chunks + i];
            if (b >= w.from) sum += l.sum[row * l.chunks + i] * w.weight(b);
        }
        sum = group.reduce(sum, 0.0, Add());
        int e;
        (void)frexp(sum * 1.001, &e);                 // the sum is below 2^e (the weights of chunk_best are good to 10^-5)
        const int S = 62 - e < 51 ? 62 - e : 51;
        w.set(par.kappa, best, worst, S);
        state = wants_border(par, a.K) ? 2 : 1;
    }
    if (chunk == 0 && threadIdx.x == 0) {
        LongRow<V>& r = l.row[row];
        r.w = w;
        r.border = w.from;
        r.last = UINT_MAX;
        r.state = state;
    }
    if (state == 2) {
        for (int i = threadIdx.x; i < LONG_BINS; i += LT) { s_cnt[i] = 0; s_mass[i] = 0; }
        __syncthreads();
    }
    const LongBins<V> bins(w);
    unsigned long long kept[c.PIECES];
#pragma unroll
    for (int p = 0; p < c.PIECES; p++) kept[p] = 0;
    if (state != 0) {
#pragma unroll
        for (int p = 0; p < c.PIECES; p++) {
            const unsigned live = c.live(p, w.from);
            if (live) {
                unsigned long long q[c.VEC];
                w.masses(c.x[p], live, state == 1 ? par.min_p : 0.0, q);
#pragma unroll
                for (int j = 0; j < c.VEC; j++) {
                    kept[p] += q[j];
                    if (state == 2 && (live >> j & 1u)) {
                        const int b = bins.of(c.x[p][j]);
                        atomicAdd(&s_cnt[b], 1u);
                        atomicAdd(&s_mass[b], q[j]);
                    }
                }
            }
        }
    }
    if (state != 2) {
        c.store(kept, group, l.seg + (size_t)blockIdx.x * MOST_SEGS, l.kept + blockIdx.x);
        return;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < LONG_BINS; i += LT)
        if (s_cnt[i]) {
            atomicAdd(&l.cnt[row * LONG_BINS + i], s_cnt[i]);
            atomicAdd(&l.mass[row * LONG_BINS + i], s_mass[i]);
        }
}

struct WhereArea {
    unsigned long long k_mass_before, k_mass, p_before;
    unsigned k_before;
    int k, first, last;
};
template <int NT> __device__ Where where(const Param& par, int K, const unsigned* cnt, const unsigned long long* mass, WhereArea& s, Group<NT>& group) {
    constexpr int PER = LONG_BINS / NT;
    unsigned c[PER], csum = 0, ctotal;
    unsigned long long m[PER], msum = 0, mtotal;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        c[i] = cnt[threadIdx.x * PER + i];
        m[i] = mass[threadIdx.x * PER + i];
        csum += c[i];
        msum += m[i];
    }
    const unsigned crun0 = group.scan(csum, ctotal);
    const unsigned long long mrun0 = group.scan(msum, mtotal);
    Where r;
    r.k = -1;
    r.p_first = 1; r.p_last = 0;
    r.k_before = 0;
    r.k_mass_before = r.mass_before = 0;
    r.mass = mtotal;
    r.nothing = false;
    unsigned long long least = mtotal, most = mtotal;          // bounds of the mass that top-k keeps
    if (par.top_k > 0 && par.top_k < K && (unsigned long long)par.top_k <= ctotal) {
        const unsigned k = (unsigned)par.top_k;
        unsigned crun = crun0;
        unsigned long long mrun = mrun0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (crun < k && k <= crun + c[i]) { s.k = threadIdx.x * PER + i; s.k_before = crun; s.k_mass_before = mrun; s.k_mass = m[i]; }
            crun += c[i];
            mrun += m[i];
        }
        __syncthreads();
        r.k = s.k;
        r.k_before = s.k_before;
        r.k_mass_before = least = s.k_mass_before;
        most = least + s.k_mass;
    }
    if (!(par.top_p >= 1.0)) {
        const unsigned long long to = share_of(par.top_p, most);
        unsigned long long from = share_of(par.top_p, least);
        if (to == 0) { r.nothing = true; return r; }
        from = from > 0 ? from : 1;
        unsigned long long mrun = mrun0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (mrun < from && from <= mrun + m[i]) { s.first = threadIdx.x * PER + i; s.p_before = mrun; }
            if (mrun < to && to <= mrun + m[i]) s.last = threadIdx.x * PER + i;
            mrun += m[i];
        }
        __syncthreads();
        r.p_first = s.first;
        r.p_last = s.last;
        r.mass_before = s.p_before;
    }
    return r;
}

template <class T, int CHUNK> __global__ void __launch_bounds__(LT, 4) chunk_split_kernel(DrawArgs a, LongArea<typename Traits<T>::V> l) {
    using V = typename Traits<T>::V;
    __shared__ WhereArea s;
    __shared__ unsigned long long s_slots[LT / 32];
    __shared__ unsigned s_listed, s_at;
    Group<LT> group(s_slots);
    const long long row = blockIdx.x / l.chunks;
    const int chunk = (int)(blockIdx.x - row * l.chunks);
    if (l.row[row].state != 2) return;
    Chunk<T, CHUNK> c;
    c.load(a, row, chunk);
    const Param par(a.f, row);
    const Weights<V> w = l.row[row].w;
    const LongBins<V> bins(w);
    if (threadIdx.x == 0) s_listed = 0;
    const Where at = where<LT>(par, a.K, l.cnt + row * LONG_BINS, l.mass + row * LONG_BINS, s, group);
    if (chunk == 0 && threadIdx.x == 0) l.row[row].at = at;
    // before `first` everything is kept; with neither border (top-k of more samples than there are) that is all of it
    const int first = at.nothing ? 0 : at.p_first <= at.p_last ? at.p_first : at.k >= 0 ? at.k : LONG_BINS;
    unsigned long long kept[c.PIECES];
    unsigned mine = 0;
    unsigned hits[c.PIECES];
#pragma unroll
    for (int p = 0; p < c.PIECES; p++) {
        hits[p] = 0;
        kept[p] = 0;
        const unsigned live = at.nothing ? 0u : c.live(p, w.from);
        if (live) {
            unsigned sure = 0;
#pragma unroll
            for (int j = 0; j < c.VEC; j++) {
                const int b = bins.of(c.x[p][j]);
                const unsigned bit = live & 1u << j;
                sure |= b < first ? bit : 0u;
                hits[p] |= (b >= at.p_first && b <= at.p_last) || b == at.k ? bit : 0u;
            }
            mine += (unsigned)__popc(hits[p]);
            if (sure) {
                unsigned long long q[c.VEC];
                w.masses(c.x[p], sure, par.min_p, q);
#pragma unroll
                for (int j = 0; j < c.VEC; j++) kept[p] += q[j];
            }
        }
    }
    __syncthreads();                                  // (s_listed)
    unsigned to = mine ? atomicAdd(&s_listed, mine) : 0u;
    c.store(kept, group, l.seg + (size_t)blockIdx.x * MOST_SEGS, l.kept + blockIdx.x);
    if (threadIdx.x == 0) {
        s_at = s_listed ? atomicAdd(&l.row[row].listed, s_listed) : 0u;
    }
    __syncthreads();
    to += s_at;
    if (mine) {
#pragma unroll
        for (int p = 0; p < c.PIECES; p++)
#pragma unroll
            for (int j = 0; j < c.VEC; j++)
                if (hits[p] >> j & 1u) {
                    l.list_v[row * a.K + to] = c.x[p][j];
                    l.list_i[row * a.K + to] = (unsigned)c.index(p, j);
                    to++;
                }
    }
}

// The listed samples of a row as a source of find_border.  BY_INDEX: only those equal to `only`, ordered by their index alone (an index
// below 2^24 is exact as a float).
template <class V, bool BY_INDEX> struct Listed {
    static constexpr int VEC = 4;
    const V* v;
    const unsigned* i;
    unsigned n;
    V only;
    Weights<V> w;
    __device__ __forceinline__ static unsigned place(int o, int j) { return threadIdx.x + (o * VEC + j) * BT; }
    __device__ __forceinline__ V value(int o, int j) const { return BY_INDEX ? -(V)i[place(o, j)] : v[place(o, j)]; }
    __device__ __forceinline__ unsigned index(int o, int j) const { return i[place(o, j)]; }
    template <class F> __device__ __forceinline__ void each(V low, V high, F f) {
#pragma unroll 1
        for (int o = 0; place(o, 0) < n; o++) {
            const unsigned e = place(o, 0);
            V x[VEC];
            unsigned live = 0;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const unsigned at = e + j * BT < n ? e + j * BT : e;
                x[j] = v[at];
                const bool in = e + j * BT < n && (!BY_INDEX || x[j] == only);
                if (BY_INDEX) x[j] = -(V)i[at];
                live |= in && x[j] >= low && x[j] <= high ? 1u << j : 0u;
            }
            if (live) f(x, live, o);
        }
    }
};

// what is kept of a row: above the border, or equal to it with an index up to last
template <class V> struct Kept {
    V border;
    unsigned last;
    bool some;
};
template <class T, class V = typename Traits<T>::V>
__device__ Kept<V> keep_listed(const DrawArgs& a, const LongArea<V>& l, long long row, const LongRow<V>& r, const Param& par, BorderArea<V, BT>& s,
                               Group<BT>& group) {
    const Kept<V> nothing{(V)0, 0, false};
    const Where at = r.at;
    if (at.nothing) return nothing;
    const Weights<V> w = r.w;
    if (at.k < 0 && at.p_first > at.p_last) return {w.from, UINT_MAX, true};             // all of them are kept
    const LongBins<V> bins(w);
    const int shift = chunk_shift(a.rows, a.K);
    const auto add = [&](unsigned idx, unsigned long long q) {
        const long long chunk = row * l.chunks + (idx >> shift);
        atomicAdd(&l.kept[chunk], q);
        atomicAdd(&l.seg[chunk * MOST_SEGS + (idx & ((1u << shift) - 1u)) / segment<T>], q);
    };
    const bool share = at.p_first <= at.p_last;
    if (r.listed <= BT) {
        // A thread for each: ranks by comparing each with each, masses in the order of the ranks (1 x 524288 fp32: 8.6 us, by the
        // histograms below 11.6).  The bins of the mass border come first in that order, behind them, if it is another, the
        // bin of the count border.
        const unsigned n = r.listed, t = threadIdx.x;
        V* line_v = (V*)(s.mass + BT);
        static_assert(3 * BT <= BorderArea<V, BT>::BINS, "masses, values and ranks");
        const bool in = t < n;
        const V v = in ? l.list_v[row * a.K + t] : (V)-INFINITY;
        const unsigned idx = in ? l.list_i[row * a.K + t] : UINT_MAX;
        line_v[t] = v;
        s.cnt[t] = idx;
        const int bin = in ? bins.of(v) : LONG_BINS;
        const double weight = w.weight(v);
        const unsigned long long q = in ? whole(weight * w.scale) : 0ull;
        const unsigned before_k = group.reduce(bin < at.k ? 1u : 0u, 0u, Add());             // (and line_v, cnt are there)
        unsigned rank = 0;
#pragma unroll 2
        for (unsigned o = 0; o < n; o += 4) {
#pragma unroll
            for (unsigned j = 0; j < 4; j++) rank += line_v[o + j] > v || (line_v[o + j] == v && s.cnt[o + j] < idx) ? 1u : 0u;
        }
        bool keep = in && (at.k < 0 || bin < at.k || (bin == at.k && (long long)(rank - before_k) < par.top_k - (long long)at.k_before));
        if (share) {
            const unsigned long long some = group.reduce(keep && bin == at.k ? q : 0ull, 0ull, Add());
            const unsigned long long target = share_of(par.top_p, at.k >= 0 ? at.k_mass_before + some : at.mass);
            if (target == 0) return nothing;
            if (in) s.mass[rank] = q;
            __syncthreads();
            unsigned long long total;
            const unsigned long long ahead = group.scan(in ? s.mass[t] : 0ull, total);
            s.mass[2 * BT + t] = at.mass_before + ahead;
            __syncthreads();
            keep = keep && bin <= at.p_last && s.mass[2 * BT + rank] < target;
        }
        const unsigned last = group.reduce(keep ? rank : 0u, 0u, Max());                     // (some sample is kept)
        if (keep && rank == last) { s.border = v; s.border_idx = idx; }
        if (keep && weight >= par.min_p && q) {
            add(idx, q);
        }
        __syncthreads();
        return {s.border, s.border_idx, true};
    }
    Listed<V, false> list{l.list_v + row * a.K, l.list_i + row * a.K, r.listed, (V)0, w};
    // values of the listed samples in bins first ... last
    auto range = [&](int first, int last, V low, V& lo, V& hi) {
        V least = (V)INFINITY, most = (V)-INFINITY;
        list.each(low, w.best, [&](const V (&x)[4], unsigned live, int) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int b = bins.of(x[j]);
                if ((live >> j & 1u) && b >= first && b <= last) { least = x[j] < least ? x[j] : least; most = x[j] > most ? x[j] : most; }
            }
        });
        lo = group.reduce(least, (V)INFINITY, Min());
        hi = group.reduce(most, (V)-INFINITY, Max());
    };
    V border = w.from, lo, hi;
    unsigned keep = 0, all = 0, last = UINT_MAX;
    auto found = [&]() { border = s.border; keep = s.border_keep; all = s.border_all; last = s.border_idx; __syncthreads(); };
    unsigned long long mass = 0;                      // of what top-k keeps, where top-p asks
    if (at.k >= 0) {
        range(at.k, at.k, w.from, lo, hi);
        (void)find_border<BY_COUNT>(list, s, group, (unsigned long long)par.top_k - at.k_before, 0.0, lo, hi, lo, list.n);
        found();
        if (share) {
            unsigned long long sum = 0;
            list.each(border, hi, [&](const V (&x)[4], unsigned live, int) {
                unsigned above = 0;
                unsigned long long q[4];
#pragma unroll
                for (int j = 0; j < 4; j++) above |= x[j] > border ? live & 1u << j : 0u;
                w.masses(x, above, 0.0, q);
#pragma unroll
                for (int j = 0; j < 4; j++) sum += q[j];
            });
            mass = at.k_mass_before + group.reduce(sum, 0ull, Add()) + keep * w.mass_of(border);
        }
    } else {
        mass = at.mass;
    }
    if (share) {
        const unsigned long long target = share_of(par.top_p, mass);
        if (target == 0) return nothing;
        range(at.p_first, at.p_last, border, lo, hi);
        if (find_border<BY_MASS>(list, s, group, target - at.mass_before, 0.0, lo, hi, lo, list.n)) found();
    }
    if (keep >= all) {
        last = UINT_MAX;
    } else if (last == UINT_MAX) {
        // more equal ones than a list of candidates holds: the keep-th of them by index
        Listed<V, true> equal{list.v, list.i, list.n, border, w};
        (void)find_border<BY_COUNT>(equal, s, group, keep, 0.0, -(V)a.K, (V)0, -(V)a.K, list.n);
        last = s.border_idx;
    }
    // what the list keeps joins the chunks
    list.each(border, w.best, [&](const V (&x)[4], unsigned live, int o) {
        unsigned in = 0;
        unsigned idx[4];
        unsigned long long q[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            idx[j] = live >> j & 1u ? list.index(o, j) : 0u;
            in |= x[j] > border || idx[j] <= last ? live & 1u << j : 0u;
        }
        w.masses(x, in, par.min_p, q);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (q[j]) add(idx[j], q[j]);
    });
    return {border, last, true};
}

// Draw number `at` of all by one wave: the chunk, its segment, the sample.  FRESH: masses that this workgroup has just added to.
template <class T, bool FRESH, class V = typename Traits<T>::V>
__device__ void draw_one(const DrawArgs& a, const LongArea<V>& l, long long row, long long at, const Param& par, const Weights<V>& w, const Kept<V>& r) {
    constexpr int SEG = segment<T>, VEC = SEG / 64;
    const int lane = threadIdx.x & 63, shift = chunk_shift(a.rows, a.K);
    const auto mass_at = [](const unsigned long long* p) { return FRESH ? __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *p; };
    const unsigned long long* kept = l.kept + row * l.chunks;
    unsigned long long mass = 0, target = 0, run = 0;
    int chunk = 0;
    if (r.some) {
        const int PER = (l.chunks + 63) / 64;                   // neighbouring chunks of a lane
        unsigned long long sum = 0;
        for (int i = 0; i < PER; i++) {
            const int c = lane * PER + i;
            sum += c < l.chunks ? mass_at(kept + c) : 0ull;
        }
        const unsigned long long inc = wave_scan(sum, 0ull, Add());
        mass = lane_value(inc, 63);
        if (mass != 0) {
            target = target_of(a.u[at], mass);
            run = inc - sum;
            const int owner = __builtin_amdgcn_readfirstlane(__ffsll((long long)__ballot(target - run < sum)) - 1);
            run = lane_value(run, owner);
            chunk = owner * PER;
            for (int i = 0; i < PER - 1; i++) {                  // (the same in every lane)
                const unsigned long long m = mass_at(kept + chunk);
                if (target - run < m) break;
                run += m;
                chunk++;
            }
        }
    }
    if (mass == 0) {
        if (lane == 0) { a.index[at] = -1; if (a.weight) a.weight[at] = 0.0f; }
        return;
    }
    const unsigned long long m = lane < (1 << shift) / SEG ? mass_at(l.seg + (row * l.chunks + chunk) * MOST_SEGS + lane) : 0ull;
    const unsigned long long inc = wave_scan(m, 0ull, Add());
    const int seg = __builtin_amdgcn_readfirstlane(__ffsll((long long)__ballot(target - (run + inc - m) < m)) - 1);
    run += lane_value(inc - m, seg);

    const int first = (chunk << shift) + seg * SEG + lane * VEC;
    T raw[VEC];
    load_piece((const T*)a.R + row * a.row_stride, a.col_stride, (long long)first, a.K, raw);
    V v[VEC];
    unsigned live = 0;
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        v[j] = value_of(raw[j]);
        live |= v[j] < (V)INFINITY && (v[j] > r.border || (v[j] == r.border && (unsigned)(first + j) <= r.last)) ? 1u << j : 0u;
    }
    unsigned long long q[VEC], sum = 0;
    w.masses(v, live, par.min_p, q);
#pragma unroll
    for (int j = 0; j < VEC; j++) sum += q[j];
    run += wave_scan(sum, 0ull, Add()) - sum;
    if (target - run < sum) {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            if (target - run < q[j]) {
                a.index[at] = first + j;
                if (a.weight) a.weight[at] = (float)(w.weight(v[j]) * w.scale / (double)mass);
            }
            run += q[j];
        }
    }
}

// DRAW: the rows' draws as well, a wave each by those that found the borders: less than another launch for one round of them (16 x
// 262144 fp64, per call: 4 draws 51.2 us, 52.0 with a launch of their own; 8 draws 53.1 and 51.6, 64 draws 81 and 53).
constexpr int FEW_DRAWS = BT / 64;
template <class T, bool DRAW> __global__ void __launch_bounds__(BT) row_border_kernel(DrawArgs a, LongArea<typename Traits<T>::V> l) {
    using V = typename Traits<T>::V;
    __shared__ BorderArea<V, BT> s;
    Group<BT> group(s.slots);
    const long long row = blockIdx.x;
    LongRow<V>& r = l.row[row];
    const Param par(a.f, row);
    const int state = r.state;
    if (!DRAW && state != 2) return;
    Kept<V> k{r.border, UINT_MAX, state != 0};
    if (state == 2) {
        k = keep_listed<T>(a, l, row, r, par, s, group);
        if (!DRAW && threadIdx.x == 0) {
            r.border = k.border;
            r.last = k.last;
            r.state = k.some ? 2 : 0;
        }
    }
    if (DRAW) {
        __threadfence();                             // (the masses added by any of the threads, for all of them)
        __syncthreads();
        const int d = threadIdx.x >> 6;
        if (d < a.D) draw_one<T, true>(a, l, row, row * a.D + d, par, r.w, k);
    }
}
template <class T> __global__ void __launch_bounds__(64) long_draw_kernel(DrawArgs a, LongArea<typename Traits<T>::V> l) {
    const long long at = a.first + blockIdx.x, row = (unsigned)at / (unsigned)a.D;       // (below 2^31)
    const LongRow<typename Traits<T>::V>& r = l.row[row];
    draw_one<T, false>(a, l, row, at, Param(a.f, row), r.w, {r.border, r.last, r.state != 0});
}

int ceil_log2(int n) {
    int e = 0;
    while ((1ll << e) < n) e++;
    return e;
}

constexpr size_t SHELF = 131072;                     // bytes of the longest row that one workgroup holds in LDS

// Long rows of which there are few are cut into chunks also where one workgroup could hold them: its passes take the longer the longer the
// row is, those over chunks the longer the more samples there are in all (per call, LDS and chunks, top-p alone: 1 x 20000 fp32 26 us and
// 23, 32 rows 28 and 27, 64 rows 27 and 32; 1 x 32768 34 and 25, 64 rows 35 and 34, 128 rows 35 and 47; 1 x 65536 bf16 69 and 28, 128
// rows 68 and 68, 192 rows 68 and 89; no filter: 28 and 13, 30 and 31, 31 and 40; 1 x 16384 fp64 24 and 24).
bool few_long_rows(size_t rows, size_t K) { return K > 16384 && rows * 512 <= K; }

// A grid has at most 2^32 - 1 threads along its first axis: more workgroups than that go into several launches.  `f(count)` makes
// one of workgroups a.first ... a.first + count - 1.
template <class F> int in_grids(DrawArgs& a, long long groups, int threads, F f) {
    const long long most = 0xffffffffll / threads;
    for (a.first = 0; a.first < groups; a.first += most) {
        f((unsigned)std::min(most, groups - a.first));
        HIP_OK(hipGetLastError());
    }
    return 0;
}
template <class T, int NT, int BYTES> int launch_rows(DrawArgs a, hipStream_t s) {
    // K units of half 2^-S at most in error, and sums below 2^62
    const int S = std::min(51, 62 - ceil_log2(a.K));
    // Many draws are shared by as many workgroups as leave no CU idle, each of which finds the kept samples for itself; fewer than NT / 4
    // draws of one pay for no further one.  (1 row of 4096 fp32 and 300000 draws: 11.5 us for 256 workgroups, 13.8 for 512, 1403 for one;
    // 16 rows of 30000 and 16384 draws each: 32, 50 and 228 us.)
    const long long want = std::max(1ll, 256ll / a.rows);
    const long long per = std::max({(long long)NT / 4, (a.D + want - 1) / want, ((long long)a.D + 65534) / 65535});
    const unsigned parts = (unsigned)((a.D + per - 1) / per);
    a.per = (int)std::min(per, (long long)a.D);
    return in_grids(a, a.rows, NT, [&](unsigned n) { hipLaunchKernelGGL((draw_row_kernel<T, NT, BYTES>), dim3(n, parts), dim3(NT), 0, s, a, S); });
}
template <class T, int CHUNK> int launch_chunks(const DrawArgs& a, const LongArea<typename Traits<T>::V>& l, unsigned n, bool borders, hipStream_t s) {
    hipLaunchKernelGGL((chunk_best_kernel<T, CHUNK>), dim3(n), dim3(LT), 0, s, a, l);
    HIP_OK(hipGetLastError());
    hipLaunchKernelGGL((chunk_bins_kernel<T, CHUNK>), dim3(n), dim3(LT), 0, s, a, l);
    HIP_OK(hipGetLastError());
    if (borders) {
        hipLaunchKernelGGL((chunk_split_kernel<T, CHUNK>), dim3(n), dim3(LT), 0, s, a, l);
        HIP_OK(hipGetLastError());
    }
    return 0;
}
template <class T> int launch(DrawArgs a, void* workspace, size_t workspace_bytes, hipStream_t s) {
    using V = typename Traits<T>::V;
    // (Not where top-k leaves little to do behind the first pass: 1 x 65536 bf16 with k = 64 22 us and 25, 64 rows 25 and 41.  Nor for very
    // many draws, which evaluate their segment's weights each: 1 x 32768 fp32, 16384 draws 23 and 24, 65536 24 and 51; 32 rows, 256 draws
    // each 25 and 19, 1024 each 24 and 34.)
    const bool few = few_long_rows(a.rows, a.K) && (a.f.top_k_of || a.f.top_k == 0 || a.f.top_k > 512) && (long long)a.rows * a.D <= 16384;
    if ((size_t)a.K * sizeof(T) <= SHELF && !few) {
        // One wave needs no barriers, but has every pass to itself: 1024 x 512 fp32 with all filters 9.8 us by 64 threads, 18.7 by 512;
        // 1 x 512 and 64 draws 9.3 and 10.3, 200 draws 11.4 and 10.4.  More than 512 threads pay where a row would otherwise be more
        // than 64 KB, or 64 samples per thread: 1024 x 4096 fp32 21 us by 512 threads, 64 by 1024; 1 x 8192 11.7 and 15.9; 1024 x
        // 16384 40 and 64; 1 x 16384 15.8 and 14.9.  (Two sizes of 512: with LDS for 64 KB fewer workgroups share a CU, 1024 x 8192
        // fp32 26 us with 32 KB, 33 with 64.)
        if (a.K <= 512 && a.D <= 64) return launch_rows<T, 64, 512 * sizeof(T)>(a, s);
        if (a.K * sizeof(T) <= 32768) return launch_rows<T, 512, 32768>(a, s);
        if constexpr (sizeof(T) >= 4)
            if (a.K * sizeof(T) <= 65536) return launch_rows<T, 512, 65536>(a, s);
        return launch_rows<T, 1024, SHELF>(a, s);
    }
    LongArea<V> l;
    if (!workspace || workspace_bytes < LongArea<V>::carve(&l, (char*)workspace, a.rows, a.K))
        return fail(-1, "workspace too small (mppi_draw_workspace)");
    const long long n = (long long)a.rows * l.chunks;
    if (n > 0xffffffffll / LT || (long long)a.rows * a.D > INT_MAX)
        return fail(-6, "more than 2^23 - 1 chunks of 8192 samples, or than 2^31 - 1 draws, in one call of long rows");
    const bool borders = a.f.top_k_of || a.f.top_p_of || (a.f.top_k > 0 && a.f.top_k < a.K) || a.f.top_p < 1.0;
    const int rc = chunk_shift(a.rows, a.K) == 12 ? launch_chunks<T, 4096>(a, l, (unsigned)n, borders, s) : launch_chunks<T, 8192>(a, l, (unsigned)n, borders, s);
    if (rc) return rc;
    if (borders) {
        if (a.D <= FEW_DRAWS)
            hipLaunchKernelGGL((row_border_kernel<T, true>), dim3(a.rows), dim3(BT), 0, s, a, l);
        else
            hipLaunchKernelGGL((row_border_kernel<T, false>), dim3(a.rows), dim3(BT), 0, s, a, l);
        HIP_OK(hipGetLastError());
        if (a.D <= FEW_DRAWS) return 0;
    }
    return in_grids(a, (long long)a.rows * a.D, 64, [&](unsigned n) { hipLaunchKernelGGL((long_draw_kernel<T>), dim3(n), dim3(64), 0, s, a, l); });
}

size_t workspace_of(int dtype, size_t rows, size_t K) {
    const size_t size = dtype == MPPI_F64 ? 8 : dtype == MPPI_F32 ? 4 : 2;
    if (K * size <= SHELF && !few_long_rows(rows, K)) return 0;
    return dtype == MPPI_F64 ? LongArea<double>::carve(nullptr, nullptr, rows, K) : LongArea<float>::carve(nullptr, nullptr, rows, K);
}

int check_filter(const mppi_draw_filter* f) {
    if (!f->kappa_of && !(f->kappa >= 0.0 && std::isfinite(f->kappa))) return fail(-1, "kappa must be finite and not negative");
    if (!f->top_k_of && f->top_k < 0) return fail(-1, "top_k must not be negative (0: every sample)");
    if (!f->top_p_of && !(f->top_p > 0.0 && f->top_p <= 1.0)) return fail(-1, "top_p must lie in (0, 1]");
    if (!f->min_p_of && !(f->min_p >= 0.0 && f->min_p <= 1.0)) return fail(-1, "min_p must lie in [0, 1]");
    return 0;
}

}  // namespace

extern "C" {

int mppi_draw_workspace(int32_t dtype, int32_t rows, int32_t K, size_t* bytes) try {
    if (!bytes) return fail(-1, "null argument");
    if (rows < 0 || K < 1) return fail(-1, "rows must not be negative, K must be positive");
    if (dtype < MPPI_F32 || dtype > MPPI_BF16) return fail(-1, "dtype must be MPPI_F32, MPPI_F64, MPPI_F16 or MPPI_BF16");
    if (K > MPPI_DRAW_MAX_K) return fail(-6, "K = " + std::to_string(K) + " exceeds " + std::to_string(MPPI_DRAW_MAX_K) + " samples");
    *bytes = workspace_of(dtype, (size_t)rows, (size_t)K);
    return 0;
} catch (const std::exception& e) {
    return fail(-8, std::string("host exception: ") + e.what());
}

int mppi_draw_from_returns(int32_t device, const void* d_R, int32_t dtype, int32_t rows, int32_t K, int64_t row_stride,
                           int64_t col_stride, const double* d_u, int32_t D, const mppi_draw_filter* filter, int64_t* d_index,
                           float* d_weight, void* d_workspace, size_t workspace_bytes, void* stream) try {
    if (!filter) return fail(-1, "null argument");
    if (rows < 0 || K < 1 || D < 0) return fail(-1, "rows and D must not be negative, K must be positive");
    if (K > MPPI_DRAW_MAX_K)
        return fail(-6, "mppi_draw_from_returns: K = " + std::to_string(K) + " exceeds " + std::to_string(MPPI_DRAW_MAX_K) + " samples");
    if (row_stride < 0 || col_stride < 0) return fail(-1, "strides must not be negative");
    if (dtype < MPPI_F32 || dtype > MPPI_BF16) return fail(-1, "dtype must be MPPI_F32, MPPI_F64, MPPI_F16 or MPPI_BF16");
    const int rc = check_filter(filter);
    if (rc) return rc;
    if (rows == 0 || D == 0) return 0;
    if (!d_R || !d_u || !d_index) return fail(-1, "null argument");
    if (workspace_bytes < workspace_of(dtype, (size_t)rows, (size_t)K) || ((uintptr_t)d_workspace & 255))
        return fail(-1, "workspace too small (mppi_draw_workspace) or not aligned to 256 bytes");
    mppi::DeviceGuard guard;
    HIP_OK(guard.enter(device));
    DrawArgs a{};
    a.R = d_R; a.row_stride = row_stride; a.col_stride = col_stride;
    a.rows = rows; a.K = K; a.D = D;
    a.u = d_u; a.f = *filter;
    a.index = (long long*)d_index; a.weight = d_weight;
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
    case MPPI_F32: return launch<float>(a, d_workspace, workspace_bytes, s);
    case MPPI_F64: return launch<double>(a, d_workspace, workspace_bytes, s);
    case MPPI_F16: return launch<Half>(a, d_workspace, workspace_bytes, s);
    default: return launch<Bfloat>(a, d_workspace, workspace_bytes, s);
    }
} catch (const std::exception& e) {
    return fail(-8, std::string("host exception: ") + e.what());
}

}  // extern "C"
