// Global norm of the gradients of many tensors, and clipping to a largest norm.
//
//     l2: sqrt(sum g^2)      max: max |g|        over all entries of all tensors
//     out = g s,  s = max_norm / norm if norm > max_norm, else 1; a norm that is not finite changes nothing
//
// Numbers.  Squares and their sums are fp64, so no fp32 gradient overflows or vanishes in them, and every sum has a fixed order: a
// thread adds what it reads, the lanes of a workgroup are added by a tree, and so are the partial sums of the workgroups, of
// which the sizes of the tensors alone say what each covers.  Entries are scaled in fp64 (the scale of large gradients may lie below
// fp32's range) and rounded to fp32; 16-bit ones from there to their type, of whose step the first rounding is at most 2^-14
// (fp16) or 2^-17 (bf16).
//
// Two passes over the data: no entry can be scaled before all have been read.  Large sets are bound by memory: 1.07 GB of fp32 read
// in 155 us (6.9 TB/s), 268 MB of bf16 read in 48 us and read again and written in 85 to 92 (6 TB/s; what a copy moves here: 4.8).  Small
// ones are bound by launches and by the host: the six tensors of a critic take one launch, 6.3 us per call; 384 small tensors four,
// of which two carry tables of addresses, 28 to 35 us per call, of which the GPU works 12.
#include "abi_common.hpp"
#include "../../include/mppi_hip.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <vector>

using mppi::fail;

namespace {

constexpr int BT = 256;                  // threads of a workgroup
// Bytes of one tensor that a workgroup takes at a time: two rounds of its loads, or one where there would be too few workgroups (per
// call, clipping bf16 out of place, 16, 32 and 64 KB: 8 MB 10.8, 11.1 and 14.0 us, 48 MB 30.0, 27.5 and 26.3, 256 MB 129.7, 128.1 and
// 128.6; tensors end inside a chunk, so that smaller ones are filled better).
constexpr int CHUNK = 32768, SMALL_CHUNK = 16384;
constexpr int GROUPS = 1024;             // most workgroups of a launch (four per CU), and so most partial sums (512 MB: 258 us, 2048: 261, 512: 8 % more)
constexpr int AHEAD = 4;                 // loads of 16 bytes that a thread has under way (268 MB of bf16: 2: 135.7 us, 4: 133.4, 8: 134.3)
constexpr size_t STREAMED = 24 << 20;    // bytes from which on what is clipped goes past the caches (gradient_clip_kernel),
constexpr size_t READ_ONCE = 128 << 20;  // and what only a norm is taken of (gradient_partials_kernel)
constexpr int TABLE = 168;               // tensors whose table travels in a kernel's arguments (4 KB at most)

struct Entry {
    const void* g;
    void* out;
    unsigned first;                      // chunks of the tensors before it
    unsigned last_type;                  // 4 times the entries of its last chunk, plus its type
    __host__ __device__ __forceinline__ int type() const { return (int)(last_type & 3u); }
    __device__ __forceinline__ int per(int chunk) const { return type() == MPPI_F32 ? chunk / 4 : chunk / 2; }       // entries
};
static_assert(MPPI_F32 < 4 && MPPI_F16 < 4 && MPPI_BF16 < 4, "two bits");
struct Table {
    Entry e[TABLE];
    int tensors, chunk;                  // chunk: bytes
    unsigned chunks;
};
static_assert(sizeof(Table) + 40 <= 4096, "and the kernels' other arguments");
struct FarTable {                        // of more tensors: in the workspace, put there by table_kernel
    const Entry* e;
    int tensors, chunk;                  // chunk: bytes
    unsigned chunks;
};

template <class T> struct Io;
template <> struct Io<float> {
    static constexpr int VEC = 4;
    using B = uint32_t;
    static __device__ __forceinline__ float get(B b) { return __uint_as_float(b); }
    static __device__ __forceinline__ B scaled(B b, double s) { return __float_as_uint((float)((double)get(b) * s)); }
};
template <> struct Io<_Float16> {
    static constexpr int VEC = 8;
    using B = uint16_t;
    static __device__ __forceinline__ float get(B b) { return (float)__builtin_bit_cast(_Float16, b); }
    static __device__ __forceinline__ B scaled(B b, double s) { return __builtin_bit_cast(B, (_Float16)(float)((double)get(b) * s)); }
};
template <> struct Io<__bf16> {
    static constexpr int VEC = 8;
    using B = uint16_t;
    static __device__ __forceinline__ float get(B b) { return __uint_as_float((uint32_t)b << 16); }
    static __device__ __forceinline__ B scaled(B b, double s) { return __builtin_bit_cast(B, (__bf16)(float)((double)get(b) * s)); }
};
typedef uint32_t Words __attribute__((ext_vector_type(4)));
typedef Words LooseWords __attribute__((aligned(2), may_alias));
template <class T> struct Pack {         // 16 bytes of entries, wherever they lie
    using B = typename Io<T>::B;
    static constexpr int PER = 4 / (int)sizeof(B);              // entries per word
    Words w;
    template <bool STREAM = false> __device__ __forceinline__ void load(const B* p) {
        w = STREAM ? __builtin_nontemporal_load((const LooseWords*)p) : *(const LooseWords*)p;
    }
    template <bool STREAM> __device__ __forceinline__ void store(B* p) const {
        if (STREAM) __builtin_nontemporal_store(w, (LooseWords*)p);
        else *(LooseWords*)p = w;
    }
    __device__ __forceinline__ B get(int j) const { return (B)(w[j / PER] >> (j % PER * 16)); }
    __device__ __forceinline__ void scale(double s) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (PER == 1) {
                w[i] = Io<T>::scaled(get(i), s);
            } else {
                const uint32_t lo = Io<T>::scaled(get(2 * i), s), hi = Io<T>::scaled(get(2 * i + 1), s);
                w[i] = hi << 16 | lo;
            }
        }
    }
};

// tensor that holds chunk c, and the chunk's entries [lo, hi) in it
template <class Tab> __device__ __forceinline__ const Entry& locate(const Tab& t, unsigned c, long long& lo, long long& hi) {
    // the lanes look at 64 tensors at a time: a wait or two, where halving the table would wait eight times and more
    const int lane = threadIdx.x & 63;
    int a = 0, b = t.tensors;
    while (b - a > 1) {
        const int step = (b - a + 63) >> 6, i = a + lane * step;
        a += (__popcll(__ballot(i < b && t.e[i < b ? i : a].first <= c)) - 1) * step;
        b = a + step < b ? a + step : b;
    }
    const Entry& e = t.e[a];
    const unsigned end = a + 1 < t.tensors ? t.e[a + 1].first : t.chunks;
    const int per = e.per(t.chunk);
    lo = (long long)(c - e.first) * per;
    hi = lo + (c + 1 < end ? per : (int)(e.last_type >> 2));
    return e;
}

// one entry into a running sum of squares, or largest magnitude (as its bits: NaN is above infinity)
template <bool MAX> __device__ __forceinline__ void take(double& acc, uint32_t& top, float x) {
    if (MAX) {
        const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
        top = b > top ? b : top;
    } else {
        acc = fma((double)x, (double)x, acc);
    }
}
template <bool MAX, int NT> __device__ double group_total(double acc, uint32_t top, double* s) {
    double v = MAX ? (double)top : acc;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const double o = __shfl_xor(v, d, 64);
        v = MAX ? fmax(v, o) : v + o;
    }
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
    for (int w = 1; w < NT / 64; w++) v = MAX ? fmax(v, s[w]) : v + s[w];
    __syncthreads();
    return v;
}
template <bool MAX> __device__ __forceinline__ double norm_of_total(double v) { return MAX ? (double)__uint_as_float((uint32_t)v) : sqrt(v); }

// entries [lo, hi) of a tensor by NT threads (tid: which one), AHEAD packs of a thread under way at a time
template <class T, bool MAX, int NT, bool STREAM> __device__ __forceinline__ void read_span(const void* p, int tid, long long lo, long long hi, double (&acc)[4], uint32_t& top) {
    using B = typename Io<T>::B;
    constexpr int VEC = Io<T>::VEC, STEP = NT * VEC;
    const B* g = (const B*)p;
    long long i = lo + tid * VEC;
    for (; i + (AHEAD - 1) * STEP + VEC <= hi; i += AHEAD * STEP) {
        Pack<T> x[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) x[k].template load<STREAM>(g + i + k * STEP);
#pragma unroll
        for (int k = 0; k < AHEAD; k++)
#pragma unroll
            for (int j = 0; j < VEC; j++) take<MAX>(acc[j % 4], top, Io<T>::get(x[k].get(j)));
    }
    for (; i + VEC <= hi; i += STEP) {
        Pack<T> x;
        x.template load<STREAM>(g + i);
#pragma unroll
        for (int j = 0; j < VEC; j++) take<MAX>(acc[j % 4], top, Io<T>::get(x.get(j)));
    }
    for (; i < hi; i++) take<MAX>(acc[0], top, Io<T>::get(g[i]));      // the last, shorter pack
}
// times the scale, or bit for bit
template <class T, bool SCALED, int NT, bool STREAM> __device__ __forceinline__ void write_span(const void* from, void* to, int tid, long long lo, long long hi, double scale) {
    using B = typename Io<T>::B;
    constexpr int VEC = Io<T>::VEC, STEP = NT * VEC;
    const B* g = (const B*)from;
    B* out = (B*)to;
    long long i = lo + tid * VEC;
    for (; i + (AHEAD - 1) * STEP + VEC <= hi; i += AHEAD * STEP) {
        Pack<T> x[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; k++) x[k].template load<STREAM>(g + i + k * STEP);
#pragma unroll
        for (int k = 0; k < AHEAD; k++) {
            if (SCALED) x[k].scale(scale);
            x[k].template store<STREAM>(out + i + k * STEP);
        }
    }
    for (; i + VEC <= hi; i += STEP) {
        Pack<T> x;
        x.template load<STREAM>(g + i);
        if (SCALED) x.scale(scale);
        x.template store<STREAM>(out + i);
    }
    for (; i < hi; i++) out[i] = SCALED ? Io<T>::scaled(g[i], scale) : g[i];
}
template <bool MAX, int NT, bool STREAM> __device__ __forceinline__ void read_chunk(const Entry& e, int tid, long long lo, long long hi, double (&acc)[4], uint32_t& top) {
    if (e.type() == MPPI_F32) read_span<float, MAX, NT, STREAM>(e.g, tid, lo, hi, acc, top);
    else if (e.type() == MPPI_F16) read_span<_Float16, MAX, NT, STREAM>(e.g, tid, lo, hi, acc, top);
    else read_span<__bf16, MAX, NT, STREAM>(e.g, tid, lo, hi, acc, top);
}
template <int NT, bool STREAM> __device__ __forceinline__ void write_chunk(const Entry& e, int tid, long long lo, long long hi, bool clip, double scale) {
    if (!clip && e.out == e.g) return;
    if (e.type() == MPPI_F32) {
        if (clip) write_span<float, true, NT, STREAM>(e.g, e.out, tid, lo, hi, scale);
        else write_span<float, false, NT, STREAM>(e.g, e.out, tid, lo, hi, scale);
    } else if (!clip) {
        write_span<__bf16, false, NT, STREAM>(e.g, e.out, tid, lo, hi, scale);      // (bits are bits)
    } else if (e.type() == MPPI_F16) {
        write_span<_Float16, true, NT, STREAM>(e.g, e.out, tid, lo, hi, scale);
    } else {
        write_span<__bf16, true, NT, STREAM>(e.g, e.out, tid, lo, hi, scale);
    }
}

__global__ void __launch_bounds__(BT) table_kernel(Table t, Entry* __restrict__ far) {
    for (int i = threadIdx.x; i < t.tensors; i += BT) far[i] = t.e[i];
}

// STREAM: nothing is read again, and what is read need not push anything out of the caches (per call, the norm of bf16 with and without:
// 128 MB 25.4 and 26.2 us, 256 MB 44 and 48, 512 MB 82 and 92; 1.07 GB of fp32 158 and 183, i.e. 6.8 TB/s).
// FAR: t holds the last tensors only, those before it, with `before` chunks, lie in far; it is put behind them for the second pass
template <bool MAX, bool FAR, bool STREAM> __global__ void __launch_bounds__(BT) gradient_partials_kernel(Table t, Entry* far, int tensors, unsigned before, double* __restrict__ partials) {
    __shared__ double s[BT / 64];
    double acc[4] = {0.0, 0.0, 0.0, 0.0};      // four chains of dependent additions
    uint32_t top = 0;
    for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        long long lo, hi;
        const Entry& e = FAR && c < before ? locate(FarTable{far, tensors, t.chunk, before}, c, lo, hi) : locate(t, c, lo, hi);
        read_chunk<MAX, BT, STREAM>(e, threadIdx.x, lo, hi, acc, top);
    }
    if (FAR && blockIdx.x == 0)
        for (int i = threadIdx.x; i < t.tensors; i += BT) far[tensors + i] = t.e[i];
    const double v = group_total<MAX, BT>((acc[0] + acc[1]) + (acc[2] + acc[3]), top, s);
    if (threadIdx.x == 0) partials[blockIdx.x] = v;
}

template <bool MAX> __device__ double norm_of(const double* __restrict__ partials, int n, double* s) {
    double acc = 0.0, v[GROUPS / BT];                // (all asked for at once)
#pragma unroll
    for (int k = 0; k < GROUPS / BT; k++) v[k] = (int)threadIdx.x + k * BT < n ? partials[threadIdx.x + k * BT] : 0.0;
#pragma unroll
    for (int k = 0; k < GROUPS / BT; k++) acc = MAX ? fmax(acc, v[k]) : acc + v[k];
    return norm_of_total<MAX>(group_total<MAX, BT>(acc, (uint32_t)acc, s));
}

template <bool MAX> __global__ void __launch_bounds__(BT) gradient_norm_kernel(const double* __restrict__ partials, int n, float* __restrict__ norm_out) {
    __shared__ double s[BT / 64];
    const double norm = norm_of<MAX>(partials, n, s);
    if (threadIdx.x == 0) *norm_out = (float)norm;
}

// Every workgroup takes the chunks it took for the norm, the last one first: that one may still lie in its caches.  STREAM: above 24 MB
// loads and stores go past them, or the next call's reads wait for this one's writes to leave (per call out of place, with and
// without: 16 MB 11.8 and 11.7 us, 32 MB 15.3 and 18.4, 256 MB 125 and 158; in place 64 MB 33.5 and 34.3, 256 MB 128 and 155).
template <class Tab, bool MAX, bool STREAM> __global__ void __launch_bounds__(BT) gradient_clip_kernel(Tab t, const double* __restrict__ partials, int n_partials,
                                                                                       double max_norm, float* __restrict__ norm_out) {
    __shared__ double s[BT / 64];
    unsigned c = blockIdx.x + (t.chunks - 1 - blockIdx.x) / gridDim.x * gridDim.x;
    long long lo, hi;
    const Entry* e = &locate(t, c, lo, hi);          // (while the partial sums are on their way)
    const double norm = norm_of<MAX>(partials, n_partials, s);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const bool clip = norm > max_norm && norm < INFINITY;
    const double scale = clip ? max_norm / norm : 1.0;
    while (true) {
        write_chunk<BT, STREAM>(*e, threadIdx.x, lo, hi, clip, scale);
        if (c < gridDim.x) break;
        c -= gridDim.x;
        e = &locate(t, c, lo, hi);
    }
}

// Few entries: one workgroup does all of it, a wave for every PIECE, and its second reading comes from the cache of its XCD.  A
// round of 16 pieces takes about a microsecond, and three rounds as long as two launches (per call, this and two launches: 32 full
// pieces 7.9 and 9.5 us, 45 full ones 10.6 and 9.6, 47 of 400 bytes 7.1 and 10.2); MOST_BYTES stops the full ones earlier.
constexpr int ST = 1024, PIECE = 4096 /* bytes */, MOST_PIECES = 48;
constexpr size_t MOST_BYTES = 128 << 10;
template <bool MAX> __global__ void __launch_bounds__(ST) gradient_small_kernel(Table t, bool write, double max_norm, float* __restrict__ norm_out) {
    __shared__ double s[ST / 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Lane l knows tensor l and where its pieces lie among all of them: the tensor of a piece is then a ballot away, where a search
    // through the arguments would wait for a scalar load at every step.
    const Entry& own = t.e[lane < t.tensors ? lane : 0];
    const unsigned long long g = (unsigned long long)own.g, out = (unsigned long long)own.out;
    const int type = own.type(), per = type == MPPI_F32 ? PIECE / 4 : PIECE / 2;
    const int n = (int)((lane + 1 < t.tensors ? t.e[lane + 1].first : t.chunks) - own.first - 1) * own.per(t.chunk) + (int)(own.last_type >> 2);
    const int count = lane < t.tensors ? (n + per - 1) / per : 0;
    int end = count;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(end, d, 64);
        if (lane >= d) end += o;
    }
    const auto far = [](unsigned long long v, int l) {
        const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, l), hi = (unsigned)__builtin_amdgcn_readlane((int)(v >> 32), l);
        return (unsigned long long)hi << 32 | lo;
    };
    const int all = __builtin_amdgcn_readlane(end, 63);
    const auto pieces = [&](auto f) {                // f(tensor, entries of a piece): this wave's pieces
        for (int p = wave; p < all; p += ST / 64) {
            const int k = __popcll(__ballot(end <= p));
            Entry e;
            e.g = (const void*)far(g, k);
            e.out = (void*)far(out, k);
            e.first = 0;
            e.last_type = (unsigned)__builtin_amdgcn_readlane(type, k);
            const int size = e.type() == MPPI_F32 ? PIECE / 4 : PIECE / 2;
            const int lo = (p - __builtin_amdgcn_readlane(end - count, k)) * size, all_of = __builtin_amdgcn_readlane(n, k);
            f(e, (long long)lo, (long long)(lo + size < all_of ? lo + size : all_of));
        }
    };
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    uint32_t top = 0;
    pieces([&](const Entry& e, long long lo, long long hi) { read_chunk<MAX, 64, false>(e, lane, lo, hi, acc, top); });
    const double norm = norm_of_total<MAX>(group_total<MAX, ST>((acc[0] + acc[1]) + (acc[2] + acc[3]), top, s));
    if (threadIdx.x == 0) *norm_out = (float)norm;
    if (!write) return;
    const bool clip = norm > max_norm && norm < INFINITY;
    const double scale = clip ? max_norm / norm : 1.0;
    pieces([&](const Entry& e, long long lo, long long hi) { write_chunk<64, false>(e, lane, lo, hi, clip, scale); });
}

int element_size(int dtype) { return dtype == MPPI_F32 ? 4 : 2; }

// What is written may be read only as the same tensor (in place) and written only once.
int check_overlap(int32_t n, const void* const* g, void* const* out, const int64_t* sizes, const int32_t* dtypes) {
    struct Span { uintptr_t lo, hi; int who; };
    const auto by_address = [](const Span& a, const Span& b) { return a.lo < b.lo; };
    std::vector<Span> written, read;
    written.reserve(n);
    for (int i = 0; i < n; i++) {
        if (sizes[i] == 0) continue;
        const uintptr_t bytes = (uintptr_t)sizes[i] * element_size(dtypes[i]);
        written.push_back({(uintptr_t)out[i], (uintptr_t)out[i] + bytes, i});
        if (g[i] != out[i]) read.push_back({(uintptr_t)g[i], (uintptr_t)g[i] + bytes, i});
    }
    for (std::vector<Span>* v : {&written, &read})               // (allocations and views of a buffer mostly ascend)
        if (!std::is_sorted(v->begin(), v->end(), by_address)) std::sort(v->begin(), v->end(), by_address);
    const auto refuse = [](int i) { return fail(-1, "clipped gradients overlap each other or their inputs (tensor " + std::to_string(i) + ")"); };
    for (size_t i = 1; i < written.size(); i++)
        if (written[i].lo < written[i - 1].hi) return refuse(written[i].who);
    size_t w = 0;                                                // the first written span that ends behind the read one's start
    for (const Span& r : read) {
        // spans that are read may overlap each other, but their starts ascend
        while (w < written.size() && written[w].hi <= r.lo) w++;
        if (w < written.size() && written[w].lo < r.hi) return refuse(r.who);
    }
    return 0;
}

// second pass: the norm, and what it does to the entries
template <class Tab, bool MAX> int second(const Tab& t, int groups, size_t bytes, const double* partials, const double* max_norm, float* norm, hipStream_t s) {
    if (!max_norm)
        hipLaunchKernelGGL((gradient_norm_kernel<MAX>), dim3(1), dim3(BT), 0, s, partials, groups, norm);
    else if (bytes > STREAMED)
        hipLaunchKernelGGL((gradient_clip_kernel<Tab, MAX, true>), dim3(groups), dim3(BT), 0, s, t, partials, groups, *max_norm, norm);
    else
        hipLaunchKernelGGL((gradient_clip_kernel<Tab, MAX, false>), dim3(groups), dim3(BT), 0, s, t, partials, groups, *max_norm, norm);
    HIP_OK(hipGetLastError());
    return 0;
}
template <bool MAX> int run(const std::vector<Entry>& e, int chunk, unsigned chunks, size_t pieces, size_t bytes, char* workspace, const double* max_norm, float* norm, hipStream_t s) {
    const int groups = (int)std::min<unsigned>(chunks, (unsigned)GROUPS);
    double* partials = (double*)workspace;
    Entry* far = (Entry*)(workspace + GROUPS * sizeof(double));
    Table t;
    t.chunk = chunk;
    t.chunks = chunks;
    size_t at = 0;
    for (;; at += TABLE) {                                   // all tables but the last go ahead
        t.tensors = (int)std::min((size_t)TABLE, e.size() - at);
        std::copy(e.begin() + at, e.begin() + at + t.tensors, t.e);
        if (at + t.tensors == e.size()) break;
        hipLaunchKernelGGL(table_kernel, dim3(1), dim3(BT), 0, s, t, far + at);
        HIP_OK(hipGetLastError());
    }
    const bool once = !max_norm && bytes > READ_ONCE;
    if (at > 0) {
        if (once)
            hipLaunchKernelGGL((gradient_partials_kernel<MAX, true, true>), dim3(groups), dim3(BT), 0, s, t, far, (int)at, e[at].first, partials);
        else
            hipLaunchKernelGGL((gradient_partials_kernel<MAX, true, false>), dim3(groups), dim3(BT), 0, s, t, far, (int)at, e[at].first, partials);
        HIP_OK(hipGetLastError());
        return second<FarTable, MAX>(FarTable{far, (int)e.size(), chunk, chunks}, groups, bytes, partials, max_norm, norm, s);
    }
    if (pieces <= MOST_PIECES && bytes <= MOST_BYTES && t.tensors <= 64) {
        hipLaunchKernelGGL((gradient_small_kernel<MAX>), dim3(1), dim3(ST), 0, s, t, max_norm != nullptr, max_norm ? *max_norm : 0.0, norm);
        HIP_OK(hipGetLastError());
        return 0;
    }
    if (once)
        hipLaunchKernelGGL((gradient_partials_kernel<MAX, false, true>), dim3(groups), dim3(BT), 0, s, t, (Entry*)nullptr, 0, 0u, partials);
    else
        hipLaunchKernelGGL((gradient_partials_kernel<MAX, false, false>), dim3(groups), dim3(BT), 0, s, t, (Entry*)nullptr, 0, 0u, partials);
    HIP_OK(hipGetLastError());
    return second<Table, MAX>(t, groups, bytes, partials, max_norm, norm, s);
}

int gradients(int32_t device, int32_t n, const void* const* g, void* const* out, const int64_t* sizes, const int32_t* dtypes,
              int32_t norm_type, const double* max_norm, float* d_norm, void* d_workspace, size_t workspace_bytes, void* stream) {
    if (n < 0) return fail(-1, "the number of tensors must not be negative");
    if (norm_type != MPPI_NORM_L2 && norm_type != MPPI_NORM_MAX) return fail(-1, "norm_type must be MPPI_NORM_L2 or MPPI_NORM_MAX");
    if (max_norm && !(*max_norm >= 0.0)) return fail(-1, "max_norm must not be negative or NaN");
    if (!d_norm || (n > 0 && (!g || !sizes || !dtypes))) return fail(-1, "null argument");
    for (int i = 0; i < n; i++) {
        if (sizes[i] < 0) return fail(-1, "tensor " + std::to_string(i) + ": negative size");
        if (dtypes[i] != MPPI_F32 && dtypes[i] != MPPI_F16 && dtypes[i] != MPPI_BF16)
            return fail(-1, "tensor " + std::to_string(i) + ": dtype must be MPPI_F32, MPPI_F16 or MPPI_BF16");
        if (sizes[i] > 0 && (!g[i] || (max_norm && !out[i]))) return fail(-1, "tensor " + std::to_string(i) + ": null address");
        if (sizes[i] > ((int64_t)1 << 40)) return fail(-6, "tensor " + std::to_string(i) + ": more than 2^40 entries");
        const uintptr_t odd = (uintptr_t)element_size(dtypes[i]) - 1;
        if (((uintptr_t)g[i] & odd) || (max_norm && ((uintptr_t)out[i] & odd)))
            return fail(-1, "tensor " + std::to_string(i) + ": address is not a multiple of its element's size");
    }
    if (max_norm) {
        const int rc = check_overlap(n, g, out, sizes, dtypes);
        if (rc) return rc;
    }
    size_t bytes = 0, pieces = 0;
    for (int i = 0; i < n; i++) {
        const size_t size = (size_t)sizes[i] * element_size(dtypes[i]);
        bytes += size;
        pieces += (size + PIECE - 1) / PIECE;
    }
    const int chunk = bytes <= (size_t)GROUPS * SMALL_CHUNK ? SMALL_CHUNK : CHUNK;
    std::vector<Entry> entries;
    entries.reserve(n);
    long long chunks = 0;
    for (int i = 0; i < n; i++) {
        if (sizes[i] == 0) continue;
        const int64_t per = chunk / element_size(dtypes[i]), parts = (sizes[i] + per - 1) / per;
        entries.push_back({g[i], max_norm ? out[i] : nullptr, (unsigned)chunks, (unsigned)(sizes[i] - (parts - 1) * per) << 2 | (unsigned)dtypes[i]});
        chunks += parts;
        if (chunks > 0x7fffffffll) return fail(-6, "more entries than one call can take");
    }
    size_t need = 0;
    (void)mppi_gradient_workspace(n, &need);
    if (!d_workspace || workspace_bytes < need) return fail(-1, "workspace too small (mppi_gradient_workspace)");
    if ((uintptr_t)d_workspace & 7) return fail(-1, "workspace must be a multiple of 8 bytes");
    mppi::DeviceGuard guard;
    HIP_OK(guard.enter(device));
    char* ws = (char*)d_workspace;
    return norm_type == MPPI_NORM_MAX ? run<true>(entries, chunk, (unsigned)chunks, pieces, bytes, ws, max_norm, d_norm, (hipStream_t)stream)
                                      : run<false>(entries, chunk, (unsigned)chunks, pieces, bytes, ws, max_norm, d_norm, (hipStream_t)stream);
}

}  // namespace

extern "C" {

int mppi_gradient_workspace(int32_t n, size_t* bytes) {
    if (n < 0 || !bytes) return fail(-1, "bad argument");
    *bytes = GROUPS * sizeof(double) + (n > TABLE ? (size_t)n * sizeof(Entry) : 0);
    return 0;
}

int mppi_gradient_norm(int32_t device, int32_t n, const void* const* d_grads, const int64_t* sizes, const int32_t* dtypes,
                       int32_t norm_type, float* d_norm, void* d_workspace, size_t workspace_bytes, void* stream) try {
    return gradients(device, n, d_grads, nullptr, sizes, dtypes, norm_type, nullptr, d_norm, d_workspace, workspace_bytes, stream);
} catch (const std::exception& e) {
    return fail(-8, std::string("host exception: ") + e.what());
}

int mppi_clip_gradients(int32_t device, int32_t n, const void* const* d_grads, void* const* d_out, const int64_t* sizes,
                        const int32_t* dtypes, int32_t norm_type, double max_norm, float* d_norm, void* d_workspace,
                        size_t workspace_bytes, void* stream) try {
    if (n > 0 && !d_out) return fail(-1, "null argument");
    return gradients(device, n, d_grads, d_out, sizes, dtypes, norm_type, &max_norm, d_norm, d_workspace, workspace_bytes, stream);
} catch (const std::exception& e) {
    return fail(-8, std::string("host exception: ") + e.what());
}

}  // extern "C"
