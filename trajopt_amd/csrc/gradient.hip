// Global norm of the gradients of many tensors, and clipping to a largest norm.
//
//     l2: sqrt(sum g^2)      max: max |g|        over all entries of all tensors
//     out = g s,  s = max_norm / norm if norm > max_norm, else 1; a norm that is not finite changes nothing
//
// Numbers.  Squares and their sums are fp64, so no fp32 gradient overflows or vanishes in them, and every sum has a fixed
// order: a thread adds what it reads, the lanes of a workgroup are added by a tree, the workgroups in the order of their
// partial sums, of which the launch shape alone says what each covers.  fp32 gradients are scaled in fp64 and rounded once;
// 16-bit ones are exact in fp32, scaled there and rounded once more (the first rounding is 2^-16 of the second's step).
//
// Two passes over the data: no entry can be scaled before all have been read.
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
constexpr int CHUNK = 16384;             // entries of one tensor that a workgroup takes at a time
constexpr int MAX_GROUPS = 1024;         // workgroups (= partial sums) of all norm launches together
constexpr int TABLE = 128;               // tensors per launch: the table travels in the kernel's arguments (4 KB at most)

struct Table {
    const void* g[TABLE];
    void* out[TABLE];
    long long n[TABLE];
    unsigned first[TABLE];               // chunks of the tensors before it in this launch
    int tensors;
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
    static __device__ __forceinline__ B scaled(B b, double s) { return __builtin_bit_cast(B, (_Float16)(get(b) * (float)s)); }
};
template <> struct Io<__bf16> {
    static constexpr int VEC = 8;
    using B = uint16_t;
    static __device__ __forceinline__ float get(B b) { return __uint_as_float((uint32_t)b << 16); }
    static __device__ __forceinline__ B scaled(B b, double s) { return __builtin_bit_cast(B, (__bf16)(get(b) * (float)s)); }
};
template <class T> struct Pack {         // 16 bytes of entries, wherever they lie
    typename Io<T>::B v[Io<T>::VEC];
    __device__ __forceinline__ void load(const typename Io<T>::B* p) { __builtin_memcpy(this, p, 16); }
    __device__ __forceinline__ void store(typename Io<T>::B* p) const { __builtin_memcpy(p, this, 16); }
};

// tensor that holds chunk c, and the chunk's entries [lo, hi) in it
__device__ __forceinline__ int locate(const Table& t, unsigned c, long long& lo, long long& hi) {
    int a = 0, b = t.tensors - 1;
    while (a < b) {
        const int m = (a + b + 1) >> 1;
        if (t.first[m] <= c) a = m; else b = m - 1;
    }
    lo = (long long)(c - t.first[a]) * CHUNK;
    hi = lo + CHUNK < t.n[a] ? lo + CHUNK : t.n[a];
    return a;
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
template <bool MAX> __device__ double group_total(double acc, uint32_t top, double* s) {
    double v = MAX ? (double)top : acc;
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const double o = __shfl_xor(v, d, 64);
        v = MAX ? fmax(v, o) : v + o;
    }
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s[0];
    for (int w = 1; w < BT / 64; w++) v = MAX ? fmax(v, s[w]) : v + s[w];
    __syncthreads();
    return v;
}

template <class T, bool MAX> __global__ void __launch_bounds__(BT) gradient_partials_kernel(Table t, double* __restrict__ partials) {
    using B = typename Io<T>::B;
    constexpr int VEC = Io<T>::VEC;
    __shared__ double s[BT / 64];
    double acc = 0.0;
    uint32_t top = 0;
    for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        long long lo, hi;
        const B* g = (const B*)t.g[locate(t, c, lo, hi)];
        long long i = lo + threadIdx.x * VEC;
        for (; i + VEC <= hi; i += BT * VEC) {
            Pack<T> p;
            p.load(g + i);
#pragma unroll
            for (int j = 0; j < VEC; j++) take<MAX>(acc, top, Io<T>::get(p.v[j]));
        }
        for (; i < hi; i++) take<MAX>(acc, top, Io<T>::get(g[i]));      // the last, shorter pack
    }
    const double v = group_total<MAX>(acc, top, s);
    if (threadIdx.x == 0) partials[blockIdx.x] = v;
}

template <bool MAX> __device__ double norm_of(const double* __restrict__ partials, int n, double* s) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += BT) acc = MAX ? fmax(acc, partials[i]) : acc + partials[i];
    acc = group_total<MAX>(acc, (uint32_t)acc, s);
    return MAX ? (double)__uint_as_float((uint32_t)acc) : sqrt(acc);
}

template <bool MAX> __global__ void __launch_bounds__(BT) gradient_norm_kernel(const double* __restrict__ partials, int n, float* __restrict__ norm_out) {
    __shared__ double s[BT / 64];
    const double norm = norm_of<MAX>(partials, n, s);
    if (threadIdx.x == 0) *norm_out = (float)norm;
}

template <class T, bool MAX> __global__ void __launch_bounds__(BT) gradient_clip_kernel(Table t, const double* __restrict__ partials, int n_partials,
                                                                                     double max_norm, float* __restrict__ norm_out) {
    using B = typename Io<T>::B;
    constexpr int VEC = Io<T>::VEC;
    __shared__ double s[BT / 64];
    const double norm = norm_of<MAX>(partials, n_partials, s);
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    const bool clip = norm > max_norm && norm < INFINITY;
    const double scale = clip ? max_norm / norm : 1.0;
    for (unsigned c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        long long lo, hi;
        const int k = locate(t, c, lo, hi);
        const B* g = (const B*)t.g[k];
        B* out = (B*)t.out[k];
        if (!clip && out == g) continue;
        long long i = lo + threadIdx.x * VEC;
        for (; i + VEC <= hi; i += BT * VEC) {
            Pack<T> p;
            p.load(g + i);
            if (clip) {
#pragma unroll
                for (int j = 0; j < VEC; j++) p.v[j] = Io<T>::scaled(p.v[j], scale);
            }
            p.store(out + i);
        }
        for (; i < hi; i++) out[i] = clip ? Io<T>::scaled(g[i], scale) : g[i];
    }
}

// tensors of one element type, in launches of at most TABLE
struct Batch {
    Table t;
    int dtype;
    int groups, first_partial;
};

template <bool MAX> hipError_t launch_partials(const Batch& b, double* partials, hipStream_t s) {
    double* at = partials + b.first_partial;
    switch (b.dtype) {
    case MPPI_F32: hipLaunchKernelGGL((gradient_partials_kernel<float, MAX>), dim3(b.groups), dim3(BT), 0, s, b.t, at); break;
    case MPPI_F16: hipLaunchKernelGGL((gradient_partials_kernel<_Float16, MAX>), dim3(b.groups), dim3(BT), 0, s, b.t, at); break;
    default: hipLaunchKernelGGL((gradient_partials_kernel<__bf16, MAX>), dim3(b.groups), dim3(BT), 0, s, b.t, at); break;
    }
    return hipGetLastError();
}
template <bool MAX> hipError_t launch_clip(const Batch& b, const double* partials, int n, double max_norm, float* norm, hipStream_t s) {
    const int groups = (int)std::min<unsigned>(b.t.chunks, 2048u);
    switch (b.dtype) {
    case MPPI_F32: hipLaunchKernelGGL((gradient_clip_kernel<float, MAX>), dim3(groups), dim3(BT), 0, s, b.t, partials, n, max_norm, norm); break;
    case MPPI_F16: hipLaunchKernelGGL((gradient_clip_kernel<_Float16, MAX>), dim3(groups), dim3(BT), 0, s, b.t, partials, n, max_norm, norm); break;
    default: hipLaunchKernelGGL((gradient_clip_kernel<__bf16, MAX>), dim3(groups), dim3(BT), 0, s, b.t, partials, n, max_norm, norm); break;
    }
    return hipGetLastError();
}

int element_size(int dtype) { return dtype == MPPI_F32 ? 4 : 2; }

// What is written may be read only as the same tensor (in place) and written only once.
int check_overlap(int32_t n, const void* const* g, void* const* out, const int64_t* sizes, const int32_t* dtypes) {
    struct Span { uintptr_t lo, hi; int who; bool written; };
    std::vector<Span> spans;
    spans.reserve(2 * (size_t)n);
    for (int i = 0; i < n; i++) {
        if (sizes[i] == 0) continue;
        const uintptr_t bytes = (uintptr_t)sizes[i] * element_size(dtypes[i]);
        spans.push_back({(uintptr_t)out[i], (uintptr_t)out[i] + bytes, i, true});
        if (g[i] != out[i]) spans.push_back({(uintptr_t)g[i], (uintptr_t)g[i] + bytes, i, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.lo < b.lo; });
    uintptr_t any_end = 0, written_end = 0;
    for (const Span& x : spans) {
        if (x.lo < written_end || (x.written && x.lo < any_end)) return fail(-1, "clipped gradients overlap each other or their inputs (tensor " + std::to_string(x.who) + ")");
        any_end = std::max(any_end, x.hi);
        if (x.written) written_end = std::max(written_end, x.hi);
    }
    return 0;
}

template <bool MAX> int run(std::vector<Batch>& batches, int n_partials, double* partials, const double* max_norm, float* norm, hipStream_t s) {
    for (const Batch& b : batches) HIP_OK(launch_partials<MAX>(b, partials, s));
    if (!max_norm || batches.empty()) {
        hipLaunchKernelGGL((gradient_norm_kernel<MAX>), dim3(1), dim3(BT), 0, s, (const double*)partials, n_partials, norm);
        HIP_OK(hipGetLastError());
        return 0;
    }
    for (size_t i = 0; i < batches.size(); i++) HIP_OK(launch_clip<MAX>(batches[i], partials, n_partials, *max_norm, i == 0 ? norm : nullptr, s));
    return 0;
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
    std::vector<Batch> batches;
    for (const int dtype : {MPPI_F32, MPPI_F16, MPPI_BF16}) {
        Batch* b = nullptr;
        for (int i = 0; i < n; i++) {
            if (dtypes[i] != dtype || sizes[i] == 0) continue;
            const long long chunks = (sizes[i] + CHUNK - 1) / CHUNK;
            if (!b || b->t.tensors == TABLE || (long long)b->t.chunks + chunks > 0x7fffffffll) {
                batches.emplace_back();
                b = &batches.back();
                b->dtype = dtype;
                b->t.tensors = 0;
                b->t.chunks = 0;
            }
            const int k = b->t.tensors++;
            b->t.g[k] = g[i]; b->t.out[k] = max_norm ? out[i] : nullptr; b->t.n[k] = sizes[i]; b->t.first[k] = b->t.chunks;
            b->t.chunks += (unsigned)chunks;
        }
    }
    // every launch gets its share of the partial sums
    int n_partials = 0;
    const int most = batches.empty() ? 0 : std::max(1, MAX_GROUPS / (int)batches.size());
    for (Batch& b : batches) {
        b.groups = (int)std::min<unsigned>(b.t.chunks, (unsigned)most);
        b.first_partial = n_partials;
        n_partials += b.groups;
    }
    size_t need = 0;
    (void)mppi_gradient_workspace(n, &need);
    if ((size_t)n_partials * 8 > need) return fail(-8, "workspace formula");
    if (n_partials > 0 && (!d_workspace || workspace_bytes < (size_t)n_partials * 8)) return fail(-1, "workspace too small (mppi_gradient_workspace)");
    if ((uintptr_t)d_workspace & 7) return fail(-1, "workspace must be a multiple of 8 bytes");
    mppi::DeviceGuard guard;
    HIP_OK(guard.enter(device));
    double* partials = (double*)d_workspace;
    return norm_type == MPPI_NORM_MAX ? run<true>(batches, n_partials, partials, max_norm, d_norm, (hipStream_t)stream)
                                      : run<false>(batches, n_partials, partials, max_norm, d_norm, (hipStream_t)stream);
}

}  // namespace

extern "C" {

int mppi_gradient_workspace(int32_t n, size_t* bytes) {
    if (n < 0 || !bytes) return fail(-1, "bad argument");
    // launches of at least one partial sum each: up to n / TABLE full ones and one more per element type
    *bytes = (size_t)(MAX_GROUPS + n / TABLE + 3) * 8;
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
