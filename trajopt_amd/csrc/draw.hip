// Draws from exponentiated returns: for every row of K returns the samples that pass top-k, top-p and min-p are weighed by
// w_i = exp(kappa (R_i - max R)), and given uniform numbers u pick the smallest i with  sum_{j <= i} w_j > u W.
//
// Numbers.  A return that is NaN or infinite weighs nothing, as in the planner's updates.  Weights are evaluated in fp64 and
// summed as 64-bit fixed point, q_i = round(w_i 2^S): integer sums do not depend on their order, so the histograms may use
// atomics, a row gives the same answer however it is split, and ties are exact.  S is chosen from the row's own mass (its
// fp64 sum, rounded up to a power of two), so the sum stays below 2^63 and K roundings of half a unit are at most
// K 2^-62 of the mass.  Samples with kappa (max - R) > (S + 1) ln 2 round to zero; they cannot be drawn, so they are left
// out from the start.
//
// Borders.  The samples kept by top-k and top-p are a prefix of the order (return descending, index ascending), so either
// filter is one pair (key of the last kept return, how many of the samples equal to it are kept).  It is found without
// sorting: a histogram of counts (top-k) or masses (top-p) over bins that are linear in kappa (max - R), then, while the bin
// with the border holds more than LIST samples of different returns, histograms over the bits of its keys, and last the
// ranks of the LIST candidates by comparing each with each.
#include "abi_common.hpp"
#include "../../include/mppi_hip.h"

#include <climits>
#include <cmath>
#include <cstdint>
#include <exception>
#include <new>

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
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
__device__ __forceinline__ double of_key(uint64_t k) {
    return __longlong_as_double((long long)((k & 0x8000000000000000ull) ? k ^ 0x8000000000000000ull : ~k));
}

struct DrawArgs {
    const void* R;
    long long row_stride, col_stride;
    int rows, K, D;
    const double* u;
    mppi_draw_filter f;
    long long* index;
    float* weight;
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

// over the NT threads of a workgroup; s_tot: NT / 64 values nobody else uses before the next barrier
template <int NT, class X, class Op> __device__ __forceinline__ X group_reduce(X v, X none, X* s_tot, Op op) {
    v = wave_scan(v, none, op);
    if (NT == 64) return lane_value(v, 63);
    const int lane = threadIdx.x & 63;
    if (lane == 63) s_tot[threadIdx.x >> 6] = v;
    __syncthreads();
    v = wave_scan(lane < NT / 64 ? s_tot[lane] : none, none, op);       // (the lanes behind the totals add nothing)
    __syncthreads();
    return lane_value(v, 63);
}
template <int NT, class X> __device__ __forceinline__ X group_scan(X v, X* s_tot, X& total) {        // exclusive sums
    const int wave = threadIdx.x >> 6;
    const X inc = wave_scan(v, (X)0, Add());
    if (NT == 64) { total = lane_value(inc, 63); return inc - v; }
    const int lane = threadIdx.x & 63;
    if (lane == 63) s_tot[wave] = inc;
    __syncthreads();
    const X own = lane < NT / 64 ? s_tot[lane] : (X)0;
    const X tot = wave_scan(own, (X)0, Add());
    __syncthreads();
    total = lane_value(tot, 63);
    return lane_value(tot - own, __builtin_amdgcn_readfirstlane(wave)) + inc - v;
}

// ------------------------------------------------------------------------------------------
// one row per workgroup, read from memory in every pass
// ------------------------------------------------------------------------------------------
template <class T, int NT> struct Row {
    using V = typename Traits<T>::V;
    using U = typename Traits<T>::U;
    static constexpr int VEC = 16 / sizeof(T);          // samples a thread takes at a time: 16 bytes
    static constexpr int BINS = NT, LIST = 256;
    struct Shared {
        unsigned cnt[BINS];
        unsigned long long mass[BINS];
        unsigned long long tot[NT / 64 + 1];
        U list_key[LIST];
        unsigned list_idx[LIST];
        unsigned long long list_q[LIST], list_before[LIST];
        unsigned list_rank[LIST], list_ties[LIST];
        unsigned n_list;
        unsigned long long pick_before;
        unsigned pick_bin, pick_n;
        U border_key;
        unsigned border_keep, border_all;
    };
    const T* R;
    long long cs;
    int K, S;
    double kappa, best, cut;          // cut: kappa (best - R) beyond which a sample is left out
    Shared& s;

    __device__ Row(Shared& s_) : s(s_) {}

    __device__ double distance(V x) const { return kappa > 0.0 ? kappa * (best - (double)x) : 0.0; }
    __device__ unsigned long long mass_of(V x) const { return (unsigned long long)__double2ull_rn(ldexp(exp(-distance(x)), S)); }

    // f(x, i): every sample in reach; those left out come as -inf
    template <class F> __device__ void each(F f) const {
        for (long long i0 = (long long)threadIdx.x * VEC; i0 < K; i0 += (long long)NT * VEC) {
#pragma unroll
            for (int j = 0; j < VEC; j++)
                if (i0 + j < K) f(load(i0 + j), (int)(i0 + j));
        }
    }
    __device__ V load(long long i) const {
        const V x = value_of(R[i * cs]);
        if (!isfinite(x)) return (V)-INFINITY;
        return distance(x) > cut ? (V)-INFINITY : x;
    }

    // Border of a prefix of the order: `target` counts samples (MASS false: the border is the target-th sample) or mass (the
    // last sample with less than the target before it).  Only samples with keys >= from take part.  A target beyond what
    // there is leaves no border (false).
    template <bool MASS> __device__ bool border(unsigned long long target, U from) {
        // range of kappa (best - R) over the samples in reach
        double far = 0.0;
        each([&](V x, int) {
            if (x > (V)-INFINITY && key_of(x) >= from) far = fmax(far, distance(x));
        });
        far = group_reduce<NT>(far, 0.0, (double*)s.tot, Max());
        const double per = far > 0.0 ? BINS / far : 0.0;
        U lo = from, hi = ~(U)0;
        int shift = -1;                                  // -1: bins linear in the distance; else bits of hi - key
        unsigned long long before = 0;
        unsigned n = 0;
        auto bin_of = [&](V x, U key) -> int {
            if (shift >= 0) return (int)((hi - key) >> shift);
            const int b = (int)(distance(x) * per);
            return b < BINS ? b : BINS - 1;
        };
        while (true) {
            s.cnt[threadIdx.x] = 0;
            s.mass[threadIdx.x] = 0;
            __syncthreads();
            each([&](V x, int) {
                const U key = key_of(x);
                if (x > (V)-INFINITY && key >= lo && key <= hi) {
                    const int b = bin_of(x, key);
                    atomicAdd(&s.cnt[b], 1u);
                    if (MASS) atomicAdd(&s.mass[b], mass_of(x));
                }
            });
            __syncthreads();
            const unsigned long long v = MASS ? s.mass[threadIdx.x] : (unsigned long long)s.cnt[threadIdx.x];
            unsigned long long total;
            const unsigned long long at = before + group_scan<NT>(v, s.tot, total);
            if (before + total < target) return false;   // (first pass only: later ones hold the border)
            if (at < target && target <= at + v) {
                s.pick_bin = threadIdx.x;
                s.pick_n = s.cnt[threadIdx.x];
                s.pick_before = at;
            }
            __syncthreads();
            const int b = (int)s.pick_bin;
            n = s.pick_n;
            before = s.pick_before;
            // keys of that bin
            if (shift < 0) {
                U klo = ~(U)0, khi = 0;
                each([&](V x, int) {
                    const U key = key_of(x);
                    if (x > (V)-INFINITY && key >= lo && bin_of(x, key) == b) { klo = key < klo ? key : klo; khi = key > khi ? key : khi; }
                });
                klo = group_reduce<NT>(klo, ~(U)0, (U*)s.tot, Min());
                khi = group_reduce<NT>(khi, (U)0, (U*)s.tot, Max());
                lo = klo;
                hi = khi;
            } else {
                const U top = hi - ((U)b << shift), width = ((U)1 << shift) - 1;
                lo = top - lo > width ? top - width : lo;
                hi = top;
            }
            if (n <= LIST || lo == hi) break;
            shift = 0;
            while (((hi - lo) >> shift) >= (U)BINS) shift++;
        }
        if (lo == hi) {                                  // all n of one return
            if (threadIdx.x == 0) {
                s.border_key = lo;
                s.border_all = n;
                if (MASS) {
                    const unsigned long long q = mass_of(of_key(lo));
                    s.border_keep = (unsigned)((target - before + q - 1) / q);
                } else {
                    s.border_keep = (unsigned)(target - before);
                }
            }
            __syncthreads();
            return true;
        }
        if (threadIdx.x == 0) s.n_list = 0;
        if (threadIdx.x < LIST) { s.list_rank[threadIdx.x] = 0; s.list_before[threadIdx.x] = 0; s.list_ties[threadIdx.x] = 0; }
        __syncthreads();
        each([&](V x, int i) {
            const U key = key_of(x);
            if (x > (V)-INFINITY && key >= lo && key <= hi) {
                const unsigned at = atomicAdd(&s.n_list, 1u);
                s.list_key[at] = key;
                s.list_idx[at] = (unsigned)i;
                s.list_q[at] = MASS ? mass_of(x) : 0;
            }
        });
        __syncthreads();
        // rank of every candidate: the threads share the comparisons
        const unsigned parts = NT / n;                   // n <= LIST <= NT
        const unsigned e = threadIdx.x / parts, part = threadIdx.x % parts;
        if (e < n) {
            const U key = s.list_key[e];
            const unsigned idx = s.list_idx[e];
            unsigned rank = 0, ties = 0;
            unsigned long long ahead = 0;
            for (unsigned o = part; o < n; o += parts) {
                const U ok = s.list_key[o];
                const bool first = ok > key || (ok == key && s.list_idx[o] < idx);
                rank += first ? 1u : 0u;
                ties += ok == key ? (first ? 0x10001u : 0x1u) : 0u;        // low half: all equal ones, high half: those ahead
                if (MASS) ahead += first ? s.list_q[o] : 0ull;
            }
            atomicAdd(&s.list_rank[e], rank);
            atomicAdd(&s.list_ties[e], ties);
            if (MASS) atomicAdd(&s.list_before[e], ahead);
        }
        __syncthreads();
        if (threadIdx.x < n) {
            const unsigned long long at = before + (MASS ? s.list_before[threadIdx.x] : (unsigned long long)s.list_rank[threadIdx.x]);
            const unsigned long long own = MASS ? s.list_q[threadIdx.x] : 1ull;
            if (at < target && target <= at + own) {
                s.border_key = s.list_key[threadIdx.x];
                s.border_all = s.list_ties[threadIdx.x] & 0xffffu;
                s.border_keep = (s.list_ties[threadIdx.x] >> 16) + 1;
            }
        }
        __syncthreads();
        return true;
    }
};

template <class T, int NT> __global__ void __launch_bounds__(NT) draw_rows_kernel(DrawArgs a) {
    using W = Row<T, NT>;
    using V = typename W::V;
    using U = typename W::U;
    __shared__ typename W::Shared s;
    W r(s);
    const long long row = blockIdx.x;
    r.R = (const T*)a.R + row * a.row_stride;
    r.cs = a.col_stride;
    r.K = a.K;
    r.kappa = a.f.kappa_of ? a.f.kappa_of[row] : a.f.kappa;
    const double top_p = a.f.top_p_of ? a.f.top_p_of[row] : a.f.top_p;
    const double min_p = a.f.min_p_of ? a.f.min_p_of[row] : a.f.min_p;
    const long long top_k = a.f.top_k_of ? a.f.top_k_of[row] : a.f.top_k;
    long long* index = a.index + row * a.D;
    float* weight = a.weight ? a.weight + row * a.D : nullptr;
    const double* u = a.u + row * a.D;

    auto nothing = [&]() {
        for (int d = threadIdx.x; d < a.D; d += NT) { index[d] = -1; if (weight) weight[d] = 0.0f; }
    };
    if (!(r.kappa >= 0.0 && r.kappa < INFINITY)) return nothing();

    // best return, then the scale from the mass
    r.best = 0.0;
    r.cut = INFINITY;
    V best = (V)-INFINITY;
    r.each([&](V x, int) { best = x > best ? x : best; });
    best = group_reduce<NT>(best, (V)-INFINITY, (V*)s.tot, Max());
    if (!(best > (V)-INFINITY)) return nothing();
    r.best = (double)best;
    double mass = 0.0;
    r.each([&](V x, int) { if (x > (V)-INFINITY) mass += exp(-r.distance(x)); });
    mass = group_reduce<NT>(mass, 0.0, (double*)s.tot, Add());
    int e;
    (void)frexp(mass, &e);                                // mass < 2^e
    r.S = 62 - e;
    r.cut = (r.S + 1) * 0.6931471805599453;

    U from = 0;                                           // border: keys above it, and the first `keep` samples that equal it
    unsigned keep = UINT_MAX, ties = 0;
    if (top_k > 0 && top_k < a.K && r.template border<false>((unsigned long long)top_k, 0)) {
        from = s.border_key; keep = s.border_keep; ties = s.border_all;
    }
    __syncthreads();
    auto kept_mass = [&](double least) {                  // of the samples with w >= least inside the border
        unsigned long long sum = 0;
        r.each([&](V x, int) {
            if (x > (V)-INFINITY) {
                const U key = key_of(x);
                if (key > from || (key == from && keep >= ties)) {
                    const double w = exp(-r.distance(x));
                    if (w >= least) sum += __double2ull_rn(ldexp(w, r.S));
                }
            }
        });
        sum = group_reduce<NT>(sum, 0ull, s.tot, Add());
        if (keep < ties && exp(-r.distance(of_key(from))) >= least) sum += keep * r.mass_of(of_key(from));
        return sum;
    };
    if (!(top_p >= 1.0)) {
        const unsigned long long all = kept_mass(0.0);
        const double part = ceil(top_p * (double)all);    // a whole number: "mass before < top_p W" is "mass before < part"
        if (!(part >= 1.0)) return nothing();
        const unsigned long long target = part < (double)all ? (unsigned long long)part : all;
        if (r.template border<true>(target, from)) {
            // inside the samples that top-k kept: its own border never lies behind theirs
            if (s.border_key != from || s.border_keep < keep) { from = s.border_key; keep = s.border_keep; ties = s.border_all; }
        }
        __syncthreads();
    }
    const unsigned long long all = kept_mass(min_p);
    if (all == 0) return nothing();

    // running mass in the order of the samples, a tile of NT VEC samples at a time
    unsigned long long running = 0;
    unsigned equal = 0;
    for (long long t0 = 0; t0 < a.K; t0 += (long long)NT * W::VEC) {
        V x[W::VEC];
        unsigned mine = 0;
#pragma unroll
        for (int j = 0; j < W::VEC; j++) {
            const long long i = t0 + (long long)threadIdx.x * W::VEC + j;
            x[j] = i < a.K ? r.load(i) : (V)-INFINITY;
            mine += x[j] > (V)-INFINITY && key_of(x[j]) == from ? 1u : 0u;
        }
        unsigned tile_equal;
        unsigned rank = equal + group_scan<NT>(mine, (unsigned*)s.tot, tile_equal);
        unsigned long long q[W::VEC], sum = 0;
#pragma unroll
        for (int j = 0; j < W::VEC; j++) {
            q[j] = 0;
            if (x[j] > (V)-INFINITY) {
                const U key = key_of(x[j]);
                const bool in = key > from || (key == from && rank < keep);
                rank += key == from ? 1u : 0u;
                if (in) {
                    const double w = exp(-r.distance(x[j]));
                    q[j] = w >= min_p ? __double2ull_rn(ldexp(w, r.S)) : 0ull;
                }
            }
            sum += q[j];
        }
        unsigned long long tile;
        const unsigned long long at = running + group_scan<NT>(sum, s.tot, tile);
        for (int d = 0; d < a.D; d++) {
            const double want = u[d] * (double)all;
            unsigned long long target = want > 0.0 ? (want < (double)all ? (unsigned long long)want : all) : 0ull;
            target = target < all ? target : all - 1;
            if (target >= at && target < at + sum) {
                unsigned long long c = at;
#pragma unroll
                for (int j = 0; j < W::VEC; j++) {
                    if (target >= c && target < c + q[j]) {
                        index[d] = t0 + (long long)threadIdx.x * W::VEC + j;
                        if (weight) weight[d] = (float)(ldexp(exp(-r.distance(x[j])), r.S) / (double)all);
                    }
                    c += q[j];
                }
            }
        }
        running += tile;
        equal += tile_equal;
    }
}

// ------------------------------------------------------------------------------------------
// one row per workgroup, held in registers
// ------------------------------------------------------------------------------------------
struct Param {
    double kappa, top_p, min_p;
    long long top_k;
    __device__ Param(const mppi_draw_filter& f, long long row)
        : kappa(f.kappa_of ? f.kappa_of[row] : f.kappa), top_p(f.top_p_of ? f.top_p_of[row] : f.top_p),
          min_p(f.min_p_of ? f.min_p_of[row] : f.min_p), top_k(f.top_k_of ? f.top_k_of[row] : f.top_k) {}
    __device__ bool valid() const { return kappa >= 0.0 && kappa < INFINITY; }
};
// u in [0, 1) -> a whole number below the mass
__device__ __forceinline__ unsigned long long target_of(double u, unsigned long long mass) {
    const double want = u * (double)mass;
    const unsigned long long t = want > 0.0 ? (want < (double)mass ? (unsigned long long)want : mass) : 0ull;
    return t < mass ? t : mass - 1;
}

// The row lies in LDS as it came (what takes no part as -inf of its type).  Thread t owns the C samples from t C on, in GP
// pieces of 16 bytes; it visits them from piece t mod GP on, so that the lanes of a wave read from all banks.  All loops over
// samples stay rolled: unrolled, a kernel of this many passes is larger than the instruction cache.  A pass tests values
// against the lowest one that takes part, in the type of the row (fp32 or fp64); exponentials, in fp64, are evaluated only for
// samples that pass.
template <class T, int NT, int BYTES> struct Shelf {
    using V = typename Traits<T>::V;
    using U = typename Traits<T>::U;
    static constexpr int VEC = 16 / sizeof(T);
    static constexpr int BINS = NT == 64 ? 256 : 1024, PER = BINS / NT, LIST = NT == 64 ? 64 : 128;
    static constexpr int FEW = BYTES >= 131072 ? 1024 : 0;     // up to this many samples that take part move together
    struct alignas(16) Piece { T v[VEC]; };
    struct Shared {
        Piece row[(BYTES / (int)sizeof(T) + FEW) / VEC];
        unsigned few_idx[FEW ? FEW : 1];
        union {
            unsigned long long mass[BINS];
            unsigned long long ends[NT];             // (once the borders are found)
        };
        unsigned long long tot[32], list_q[LIST], list_before[LIST], pick_before;
        V list_v[LIST], border;
        unsigned cnt[BINS], list_idx[LIST], list_rank[LIST], list_ties[LIST], n_list, pick_bin, pick_n, border_keep, border_all;
    };
    Shared& s;
    int GP, start, base;              // pieces of this thread, the one it begins with, the row's first piece
    int C;                            // samples per thread
    double kappa, scale;
    V best, from;                     // from: the lowest value that takes part

    __device__ Shelf(Shared& s_) : s(s_) {}
    __device__ __forceinline__ static V at(const Piece& p, int j) { return value_of(p.v[j]); }
    // kappa (best - v); both ends of fp64 may be apart by more than its range, and 0 times that is 0
    __device__ __forceinline__ double distance(V v) const {
        const double d = (double)best - (double)v;
        return kappa * (sizeof(V) == 8 ? fmin(d, 1.7976931348623157e308) : d);
    }
    __device__ __forceinline__ double weight(V v) const { return exp(-distance(v)); }
    __device__ __forceinline__ unsigned long long mass_of(V v) const { return __double2ull_rn(weight(v) * scale); }

    // f(v, live, i): the pieces with samples that take part; live: bit j for sample v[j], whose index is i + j
    template <class F> __device__ __forceinline__ void each(V low, V high, F f) {
        const int own = (int)threadIdx.x * GP;
        int g = start;
#pragma unroll 1
        for (int n = 0; n < GP; n++) {
            const Piece p = s.row[base + own + g];
            V v[VEC];
            unsigned live = 0;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                v[j] = at(p, j);
                live |= v[j] >= low && v[j] <= high ? 1u << j : 0u;
            }
            if (live) f(v, live, (own + g) * VEC);
            g = g + 1 == GP ? 0 : g + 1;
        }
    }
    // masses of a piece side by side: their exponentials are long chains of dependent operations
    __device__ __forceinline__ void masses(const V (&v)[VEC], unsigned live, double least, unsigned long long (&q)[VEC]) const {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const double w = weight(v[j]);
            q[j] = (live >> j & 1u) && w >= least ? __double2ull_rn(w * scale) : 0ull;
        }
#pragma unroll
        for (int j = 0; j < VEC; j++) asm volatile("" : "+v"(q[j]));       // (or each would be moved behind the test of its bit)
    }

    // Border of a prefix of the order among the samples that take part (none below `low`).  MASS false: the border is sample
    // number `count` of the order; there is none (false) if there are fewer.  MASS true: it is the last sample with less
    // than `part` of the mass before it (part < 1).
    template <bool MASS> __device__ bool border(unsigned long long count, double part, V low) {
        // bins linear in best - v first (monotone: every step rounds monotonically); per = 0 where that range overflows
        const V per = best > low ? (V)BINS / (best - low) : (V)0;
        V lo = from, hi = best;
        int shift = -1, bin = 0;                     // -1: linear bins; else bits of key(hi) - key(v)
        U top = key_of(hi);
        unsigned long long before = 0, target = count;
        unsigned n = 0;
        auto bin_of = [&](V v) -> int {
            if (shift >= 0) return (int)((top - key_of(v)) >> shift);
            const int b = (int)((best - v) * per);
            return b < BINS ? b : BINS - 1;
        };
#pragma unroll 1
        while (true) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                s.cnt[threadIdx.x + i * NT] = 0;
                if (MASS) s.mass[threadIdx.x + i * NT] = 0;
            }
            if (threadIdx.x == 0) s.n_list = 0;
            if (threadIdx.x < LIST) { s.list_rank[threadIdx.x] = 0; s.list_before[threadIdx.x] = 0; s.list_ties[threadIdx.x] = 0; }
            __syncthreads();
            each(lo, hi, [&](const V (&v)[VEC], unsigned live, int) {
                unsigned long long q[VEC];
                if (MASS) masses(v, live, 0.0, q);
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (live >> j & 1u) {
                        const int b = bin_of(v[j]);
                        atomicAdd(&s.cnt[b], 1u);
                        if (MASS) atomicAdd(&s.mass[b], q[j]);
                    }
            });
            __syncthreads();
            unsigned long long own[PER], sum = 0, total;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int b = threadIdx.x * PER + i;
                own[i] = MASS ? s.mass[b] : (unsigned long long)s.cnt[b];
                sum += own[i];
            }
            unsigned long long run = before + group_scan<NT>(sum, s.tot, total);
            if (shift < 0) {
                if (MASS) {
                    // a whole number: "mass before < part W" is "mass before < ceil(part W)"
                    const double want = ceil(part * (double)total);
                    if (!(want >= 1.0)) { from = (V)INFINITY; return false; }     // nothing is kept
                    target = want < (double)total ? (unsigned long long)want : total;
                }
                if (total < target) return false;
            }
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (run < target && target <= run + own[i]) {
                    s.pick_bin = threadIdx.x * PER + i;
                    s.pick_n = s.cnt[threadIdx.x * PER + i];
                    s.pick_before = run;
                }
                run += own[i];
            }
            __syncthreads();
            bin = (int)s.pick_bin;
            n = s.pick_n;
            before = s.pick_before;
            if (n <= LIST) break;
            // the values of that bin, from its lowest to its highest
            V least = (V)INFINITY, most = (V)-INFINITY;
            each(lo, hi, [&](const V (&v)[VEC], unsigned live, int) {
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if ((live >> j & 1u) && bin_of(v[j]) == bin) { least = v[j] < least ? v[j] : least; most = v[j] > most ? v[j] : most; }
            });
            lo = group_reduce<NT>(least, (V)INFINITY, (V*)s.tot, Min());
            hi = group_reduce<NT>(most, (V)-INFINITY, (V*)s.tot, Max());
            if (lo == hi) break;
            top = key_of(hi);
            shift = 0;
            while (((top - key_of(lo)) >> shift) >= (U)BINS) shift++;
        }
        if (n > LIST) {                              // all n of one return
            if (threadIdx.x == 0) {
                s.border = lo;
                s.border_all = n;
                const unsigned long long one = MASS ? mass_of(lo) : 1ull;
                s.border_keep = (unsigned)((target - before + one - 1) / one);
            }
        } else {
            each(lo, hi, [&](const V (&v)[VEC], unsigned live, int i) {
                unsigned hit = 0;
#pragma unroll
                for (int j = 0; j < VEC; j++) hit |= (live >> j & 1u) && bin_of(v[j]) == bin ? 1u << j : 0u;
                if (hit) {
#pragma unroll 1
                    for (int j = 0; j < VEC; j++)
                        if (hit >> j & 1u) {
                            const unsigned e = atomicAdd(&s.n_list, 1u);
                            s.list_v[e] = at(s.row[base + i / VEC], j);
                            s.list_idx[e] = (unsigned)(i + j);
                        }
                }
            });
            __syncthreads();
            if (MASS) {
                if (threadIdx.x < n) s.list_q[threadIdx.x] = mass_of(s.list_v[threadIdx.x]);
                __syncthreads();
            }
            // rank of every candidate: the threads share the comparisons
            const unsigned parts = NT / n;           // 1 <= n <= LIST <= NT
            const unsigned e = threadIdx.x / parts, first = threadIdx.x - e * parts;
            if (e < n) {
                const V v = s.list_v[e];
                const unsigned idx = s.list_idx[e];
                unsigned rank = 0, ties = 0;
                unsigned long long ahead = 0;
                for (unsigned o = first; o < n; o += parts) {
                    const V ov = s.list_v[o];
                    const bool lead = ov > v || (ov == v && s.list_idx[o] < idx);
                    rank += lead ? 1u : 0u;
                    ties += ov == v ? (lead ? 0x10001u : 0x1u) : 0u;       // low half: all equal ones, high half: those ahead
                    if (MASS) ahead += lead ? s.list_q[o] : 0ull;
                }
                atomicAdd(&s.list_rank[e], rank);
                atomicAdd(&s.list_ties[e], ties);
                if (MASS) atomicAdd(&s.list_before[e], ahead);
            }
            __syncthreads();
            if (threadIdx.x < n) {
                const unsigned long long run = before + (MASS ? s.list_before[threadIdx.x] : (unsigned long long)s.list_rank[threadIdx.x]);
                const unsigned long long own = MASS ? s.list_q[threadIdx.x] : 1ull;
                if (run < target && target <= run + own) {
                    s.border = s.list_v[threadIdx.x];
                    s.border_all = s.list_ties[threadIdx.x] & 0xffffu;
                    s.border_keep = (s.list_ties[threadIdx.x] >> 16) + 1;
                }
            }
        }
        __syncthreads();
        return true;
    }

    // raises `from` to a value that at least k threads' own values `mine` reach (one per thread), near the highest such
    __device__ void raise(V mine, unsigned k) {
        const V per = best > from ? (V)BINS / (best - from) : (V)0;
        const bool in = mine >= from;
        int b = in ? (int)((best - mine) * per) : 0;
        b = b < BINS ? b : BINS - 1;
#pragma unroll
        for (int i = 0; i < PER; i++) s.cnt[threadIdx.x + i * NT] = 0;
        __syncthreads();
        if (in) atomicAdd(&s.cnt[b], 1u);
        __syncthreads();
        unsigned own[PER], sum = 0, total;
#pragma unroll
        for (int i = 0; i < PER; i++) { own[i] = s.cnt[threadIdx.x * PER + i]; sum += own[i]; }
        unsigned run = group_scan<NT>(sum, (unsigned*)s.tot, total);
        if (total < k) return;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (run < k && k <= run + own[i]) s.pick_bin = threadIdx.x * PER + i;
            run += own[i];
        }
        __syncthreads();
        const V low = in && b <= (int)s.pick_bin ? mine : (V)INFINITY;
        from = group_reduce<NT>(low, (V)INFINITY, (V*)s.tot, Min());
    }

    // If few samples take part, they move together (in their order, with their indices), and the passes that follow go over
    // them alone.
    __device__ void gather_few() {
        unsigned mine = 0, pieces = 0, total;
        const int own = (int)threadIdx.x * GP;
        each(from, best, [&](const V (&)[VEC], unsigned live, int i) {
            mine += (unsigned)__popc(live);
            pieces |= 1u << (i / VEC - own);
        });
        unsigned to = group_scan<NT>(mine, (unsigned*)s.tot, total);
        if (total > FEW) return;
        constexpr int first = BYTES / 16;
        if (threadIdx.x < FEW / VEC) {
#pragma unroll
            for (int j = 0; j < VEC; j++) s.row[first + threadIdx.x].v[j] = minus_infinity((T*)nullptr);
        }
        __syncthreads();
#pragma unroll 1
        for (; pieces; pieces &= pieces - 1) {
            const int p = own + __ffs(pieces) - 1;
#pragma unroll 1
            for (int j = 0; j < VEC; j++)
                if (at(s.row[p], j) >= from) {
                    s.row[first + to / VEC].v[to % VEC] = s.row[p].v[j];
                    s.few_idx[to] = (unsigned)(p * VEC + j);
                    to++;
                }
        }
        __syncthreads();
        base = first;
        GP = threadIdx.x < FEW / VEC ? 1 : 0;
        start = 0;
        C = VEC;
    }

    // leaves out what lies behind the border that was found
    __device__ void cut_behind() {
        from = s.border;
        const unsigned keep = s.border_keep;
        if (keep < s.border_all) {                   // of the equal ones, the first in the order of the samples stay
            unsigned mine = 0, total;
            each(from, from, [&](const V (&)[VEC], unsigned live, int) { mine += (unsigned)__popc(live); });
            unsigned rank = group_scan<NT>(mine, (unsigned*)s.tot, total);
#pragma unroll 1
            for (int g = 0; g < GP && mine > 0; g++) {
                Piece& p = s.row[base + (int)threadIdx.x * GP + g];
#pragma unroll
                for (int j = 0; j < VEC; j++)
                    if (at(p, j) == from && rank++ >= keep) p.v[j] = minus_infinity((T*)nullptr);
            }
        }
        __syncthreads();                             // s.border may be written again
    }
};

template <class T, int NT, int BYTES> __global__ void __launch_bounds__(NT) draw_row_kernel(DrawArgs a, int S) {
    using H = Shelf<T, NT, BYTES>;
    using V = typename H::V;
    using Piece = typename H::Piece;
    constexpr int VEC = H::VEC;
    __shared__ typename H::Shared s;
    H h(s);
    const long long row = blockIdx.x;
    const T* R = (const T*)a.R + row * a.row_stride;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    h.GP = (a.K + NT * VEC - 1) / (NT * VEC);
    h.C = h.GP * VEC;
    h.start = tid % h.GP;
    h.base = 0;
    const Param par(a.f, row);
    long long* index = a.index + row * a.D;
    float* weight = a.weight ? a.weight + row * a.D : nullptr;
    const double* u = a.u + row * a.D;
    auto nothing = [&]() {
        for (int d = tid; d < a.D; d += NT) { index[d] = -1; if (weight) weight[d] = 0.0f; }
    };

    const double u_wave = wave < a.D ? u[wave] : 0.0, u_thread = tid < a.D ? u[tid] : 0.0;      // asked for before anything waits
    // the row into LDS, AHEAD pieces requested at a time
    constexpr int AHEAD = BYTES >= 131072 ? 8 : 4;
    V best = (V)-INFINITY, worst = (V)INFINITY;
#pragma unroll 1
    for (int p0 = 0; p0 < h.GP; p0 += AHEAD) {
        Piece in[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            const int i = ((p0 + k) * NT + tid) * VEC;
            if (a.col_stride == 1 && i + VEC <= a.K) {
                __builtin_memcpy(&in[k], R + i, 16);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j++) in[k].v[j] = i + j < a.K ? R[(long long)(i + j) * a.col_stride] : minus_infinity((T*)nullptr);
            }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            if (p0 + k >= h.GP) break;
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const V v = H::at(in[k], j);
                if (!isfinite(v)) {
                    in[k].v[j] = minus_infinity((T*)nullptr);
                } else {
                    best = v > best ? v : best;
                    worst = v < worst ? v : worst;
                }
            }
            s.row[(p0 + k) * NT + tid] = in[k];
        }
    }
    const V mine = best;                                                  // best of what this thread loaded
    best = group_reduce<NT>(best, (V)-INFINITY, (V*)s.tot, Max());
    worst = group_reduce<NT>(worst, (V)INFINITY, (V*)s.tot, Min());
    __syncthreads();
    if (!par.valid() || !(best > (V)-INFINITY)) return nothing();
    h.kappa = par.kappa;
    h.best = best;
    h.scale = __longlong_as_double((long long)(1023 + S) << 52);          // 2^S
    // samples this far behind have masses below half a unit, with a margin for the rounding of the bound itself
    h.from = fmax(worst, (V)((double)best - (S + 1.01) * 0.6931471805599453 / h.kappa * (1.0 + 1e-6)));
    // Each thread's best is one sample, so the k best threads bound the k best samples from below: with many samples per
    // thread next to nothing else passes that bound.
    if (BYTES >= 131072 && par.top_k > 0 && par.top_k <= NT / 4 && h.GP > 1) h.raise(mine, (unsigned)par.top_k);
    if (H::FEW && h.GP > 1) h.gather_few();
    if (par.top_k > 0 && par.top_k < a.K && h.template border<false>((unsigned long long)par.top_k, 0.0, h.from)) h.cut_behind();
    if (!(par.top_p >= 1.0) && h.template border<true>(0, par.top_p, h.from)) h.cut_behind();

    unsigned long long sum = 0, mass;
    h.each(h.from, h.best, [&](const V (&v)[VEC], unsigned live, int) {
        unsigned long long q[VEC];
        h.masses(v, live, par.min_p, q);
#pragma unroll
        for (int j = 0; j < VEC; j++) sum += q[j];
    });
    const unsigned long long base = group_scan<NT>(sum, s.tot, mass);
    if (mass == 0) return nothing();
    s.ends[tid] = base + sum;
    __syncthreads();
    // mass of sample i of the row, zero if it may not be drawn
    auto mass_of_sample = [&](int i, double& w) -> unsigned long long {
        const V v = H::at(s.row[h.base + i / VEC], i % VEC);
        w = h.weight(v);
        return v >= h.from && w >= par.min_p ? __double2ull_rn(w * h.scale) : 0ull;
    };
    auto answer = [&](int d, int i, double w) {
        index[d] = h.base ? (long long)s.few_idx[i] : i;
        if (weight) weight[d] = (float)(w * h.scale / (double)mass);
    };
    const int C = h.C;
    // A wave for every draw (about 500 cycles each) or a thread for every draw (about 150 cycles for every sample it walks over)
    if ((long long)(a.D + NT / 64 - 1) / (NT / 64) * 500 <= (long long)((a.D + NT - 1) / NT) * C * 150) {
#pragma unroll 1
        for (int d = wave; d < a.D; d += NT / 64) {
            const unsigned long long target = target_of(d == wave ? u_wave : u[d], mass);
            int owner = 0;                                     // number of threads that end at or below the target
#pragma unroll
            for (int k = 0; k < NT / 64; k++) owner += __popcll(__ballot(s.ends[k * 64 + lane] <= target));
            const unsigned long long ahead = owner > 0 ? s.ends[owner - 1] : 0ull;
            unsigned long long m[(BYTES / (int)sizeof(T) / NT + 63) / 64], run = ahead;
            double w;
#pragma unroll
            for (int k = 0; k < (int)(sizeof(m) / sizeof(m[0])); k++) {
                const int j = k * 64 + lane;
                m[k] = j < C ? mass_of_sample(owner * C + j, w) : 0ull;
                const unsigned long long inc = wave_scan(m[k], 0ull, Add());
                if (target - (run + inc - m[k]) < m[k]) answer(d, owner * C + j, w);
                run += lane_value(inc, 63);
            }
        }
    } else {
#pragma unroll 1
        for (int d = tid; d < a.D; d += NT) {
            const unsigned long long target = target_of(d == tid ? u_thread : u[d], mass);
            int lo = 0, hi = NT - 1;                           // the first thread that ends above the target
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (s.ends[mid] > target) hi = mid; else lo = mid + 1;
            }
            unsigned long long c = lo > 0 ? s.ends[lo - 1] : 0ull;
#pragma unroll 1
            for (int i = lo * C; i < (lo + 1) * C; i++) {
                double w;
                const unsigned long long m = mass_of_sample(i, w);
                if (target - c < m) { answer(d, i, w); break; }
                c += m;
            }
        }
    }
}

int ceil_log2(int n) {
    int e = 0;
    while ((1ll << e) < n) e++;
    return e;
}

template <class T> hipError_t launch(const DrawArgs& a, hipStream_t s) {
    const int S = 62 - ceil_log2(a.K);
    const size_t bytes = (size_t)a.K * sizeof(T);
    if (a.K <= 512)
        hipLaunchKernelGGL((draw_row_kernel<T, 64, 512 * sizeof(T)>), dim3(a.rows), dim3(64), 0, s, a, S);
    else if (a.K <= 4096)
        hipLaunchKernelGGL((draw_row_kernel<T, 256, 4096 * sizeof(T)>), dim3(a.rows), dim3(256), 0, s, a, S);
    else if (bytes <= 131072)
        hipLaunchKernelGGL((draw_row_kernel<T, 1024, 131072>), dim3(a.rows), dim3(1024), 0, s, a, S);
    else
        hipLaunchKernelGGL((draw_rows_kernel<T, 1024>), dim3(a.rows), dim3(1024), 0, s, a);
    return hipGetLastError();
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

int mppi_draw_from_returns(int32_t device, const void* d_R, int32_t dtype, int32_t rows, int32_t K, int64_t row_stride,
                           int64_t col_stride, const double* d_u, int32_t D, const mppi_draw_filter* filter, int64_t* d_index,
                           float* d_weight, void* stream) try {
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
    mppi::DeviceGuard guard;
    HIP_OK(guard.enter(device));
    DrawArgs a;
    a.R = d_R; a.row_stride = row_stride; a.col_stride = col_stride;
    a.rows = rows; a.K = K; a.D = D;
    a.u = d_u; a.f = *filter;
    a.index = (long long*)d_index; a.weight = d_weight;
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
    case MPPI_F32: HIP_OK(launch<float>(a, s)); break;
    case MPPI_F64: HIP_OK(launch<double>(a, s)); break;
    case MPPI_F16: HIP_OK(launch<Half>(a, s)); break;
    default: HIP_OK(launch<Bfloat>(a, s)); break;
    }
    return 0;
} catch (const std::exception& e) {
    return fail(-8, std::string("host exception: ") + e.what());
}

}  // extern "C"
