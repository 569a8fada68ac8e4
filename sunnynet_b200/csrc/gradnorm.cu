// The norm of a model's gradients and their clipping, over many tensors of any
// of the float types at once (no counterpart among the reference's kernels: its
// training loop leaves it to torch).
//
//   norm = sqrt(sum of g^2),  factor = min(1, max_norm / (norm + 1e-6)),  g = g * factor
//
// Squares of the values of one 16-byte load are added in fp32, everything above
// that in fp64, in an order that the sizes, types and addresses modulo 16 decide; a
// load whose sum leaves fp32's normal numbers is squared in fp64 as well, so that values
// from 2^-149 to the largest count (loads of zeros go that way too, which costs nothing
// beside HBM: 32000 x 768 values with nine rows of ten empty, or all, take as long as
// without).
//
// Bound by HBM: the norm reads every value once, clipping once more, and writes
// it. The tensors are cut into runs of 16 KB of memory, which one wave of CTAs
// takes in turn (a stretch of neighbouring runs to each CTA was a fifth slower:
// DRAM pages), with the next run's loads, and the search for its tensor, on their
// way before the last one's values are used. What the first pass read last is still
// in L2 when the second begins, so that goes from the last run to the first. 12 layers of 768 in fp32
// (280 MB): squares 45 us (6.2 TB/s), with the scaling 138, three passes at 6.1 TB/s.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

#include "caller.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace sn {
namespace {

constexpr int kThreads = 256;
constexpr int kWave = 148 * 4;          // CTAs at most, each with one part of the sum
constexpr int kPacks = 4;               // 16-byte loads of a thread for a run
constexpr int kRun = kPacks * kThreads;  // packs of a run
constexpr int kFew = 32, kMany = 1280;  // tensors of a launch: 30 of the 32 KB of parameters

struct Run {
    void* p;
    long long n;
    int first;  // its first run among the launch's
    int dtype;
};

template <int N>
struct Runs {
    int count, runs;
    Run t[N];
};

template <int N>
__device__ __forceinline__ int find(const Runs<N>& a, int c) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.t[mid].first <= c)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return __float2bfloat16_rn(x);
    else
        return __float2half_rn(x);
}

template <typename T>
union Pack {
    uint4 w;
    T v[16 / sizeof(T)];
};

template <typename T>
__device__ __forceinline__ double squares(const uint4& w) {
    constexpr int V = 16 / sizeof(T);
    Pack<T> q;
    q.w = w;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float x = to_f(q.v[i]);
        s = fmaf(x, x, s);
    }
    if (s >= 0x1p-80f && s <= 0x1p120f) return (double)s;
    double d = 0.0;  // zeros, mostly
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const double x = (double)to_f(q.v[i]);
        d = fma(x, x, d);
    }
    return d;
}

// A tensor as 16-byte packs of memory: its first and last may be its own in part.
struct Packs {
    char* base;
    int before;       // bytes of the first pack that lie before the tensor
    long long bytes;  // from the first pack's begin to the tensor's end
    long long p;      // this thread's first pack of the run
    int dtype;
    __device__ __forceinline__ bool has(int k) const { return (p + k * kThreads) * 16 < bytes; }
    __device__ __forceinline__ bool whole(int k) const {
        const long long at = (p + k * kThreads) * 16;
        return at >= before && at + 16 <= bytes;
    }
    __device__ __forceinline__ uint4* at(int k) const {
        return reinterpret_cast<uint4*>(base + (p + k * kThreads) * 16);
    }
    // f(16-bit word of the tensor, its place in the pack) for a pack in part
    template <typename F>
    __device__ __forceinline__ void words(int k, F&& f) const {
        const long long at = (p + k * kThreads) * 16;
        for (int i = 0; i < 8; ++i)
            if (at + 2 * i >= before && at + 2 * i < bytes) f(reinterpret_cast<uint16_t*>(base + at + 2 * i), i);
    }
};

template <int N>
__device__ __forceinline__ Packs packs_of(const Runs<N>& a, int c) {
    const Run& t = a.t[find(a, c)];
    Packs x;
    x.before = (int)(reinterpret_cast<uintptr_t>(t.p) & 15);
    x.base = static_cast<char*>(t.p) - x.before;
    x.bytes = x.before + t.n * (t.dtype == SN_F32 ? 4 : 2);
    x.p = (long long)(c - t.first) * kRun + threadIdx.x;
    x.dtype = t.dtype;
    return x;
}

__device__ __forceinline__ void load(uint4* w, const Packs& x) {
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
        w[k] = make_uint4(0, 0, 0, 0);
        if (x.whole(k)) {
            w[k] = *x.at(k);
        } else if (x.has(k)) {
            uint32_t part[4] = {};
            x.words(k, [&](const uint16_t* from, int i) { part[i / 2] |= (uint32_t)*from << i % 2 * 16; });
            w[k] = make_uint4(part[0], part[1], part[2], part[3]);
        }
    }
}

__device__ __forceinline__ void store(const uint4* w, const Packs& x) {
#pragma unroll
    for (int k = 0; k < kPacks; ++k) {
        if (x.whole(k)) {
            __stcs(x.at(k), w[k]);  // (nothing here reads it again)
        } else if (x.has(k)) {
            const uint32_t part[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
            x.words(k, [&](uint16_t* to, int i) { *to = (uint16_t)(part[i / 2] >> i % 2 * 16); });
        }
    }
}

template <typename T>
__device__ __forceinline__ uint4 scaled(const uint4& w, float f) {
    Pack<T> q;
    q.w = w;
#pragma unroll
    for (int j = 0; j < (int)(16 / sizeof(T)); ++j) q.v[j] = from_f<T>(to_f(q.v[j]) * f);
    return q.w;
}

// f(a type's zero) for the type of a tensor.
template <typename F>
__device__ __forceinline__ void by_type(int dtype, F&& f) {
    if (dtype == SN_F32)
        f(0.0f);
    else if (dtype == SN_BF16)
        f(__nv_bfloat16());
    else
        f(__half());
}

// f(packs, their values) for this CTA's runs, from the first or (BACK) the last on.
template <bool BACK, int N, typename F>
__device__ __forceinline__ void each_run(const Runs<N>& a, F&& f) {
    const auto run = [&](int i) { return BACK ? a.runs - 1 - i : i; };
    int i = blockIdx.x;
    if (i >= a.runs) return;
    Packs x = packs_of(a, run(i));
    uint4 w[kPacks];
    load(w, x);
    for (;;) {
        const int next = i + gridDim.x;
        Packs y = x;
        uint4 v[kPacks];
        if (next < a.runs) {
            y = packs_of(a, run(next));
            load(v, y);
        }
        f(x, w);
        if (next >= a.runs) break;
        x = y;
#pragma unroll
        for (int k = 0; k < kPacks; ++k) w[k] = v[k];
        i = next;
    }
}

// Sum over the CTA, in thread 0 of it.
__device__ __forceinline__ double cta_sum(double x) {
    __shared__ double s[kThreads / 32];
#pragma unroll
    for (int d = 16; d; d /= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int i = 1; i < kThreads / 32; ++i) x += s[i];
    return x;
}

template <int N>
__global__ void __launch_bounds__(kThreads, 4) square_kernel(const __grid_constant__ Runs<N> a, double* parts) {
    pdl_trigger();
    double sum = 0.0;
    each_run<false>(a, [&](const Packs& x, const uint4* w) {
        by_type(x.dtype, [&](auto t) {
#pragma unroll
            for (int k = 0; k < kPacks; ++k) sum += squares<decltype(t)>(w[k]);
        });
    });
    sum = cta_sum(sum);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

// The norm and the factor from the parts: in every thread of the CTA.
__device__ __forceinline__ float2 finish(const double* parts, int n, double max_norm) {
    __shared__ float2 out;
    double x = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) x += parts[i];
    x = cta_sum(x);
    if (threadIdx.x == 0) {
        const double norm = sqrt(x);
        // (a NaN makes the factor one; an infinite norm below an infinite bound does not)
        out = make_float2((float)norm, norm + 1e-6 <= max_norm ? 1.0f : (float)(max_norm / (norm + 1e-6)));
    }
    __syncthreads();
    return out;
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double* parts, int n, double max_norm, float* norm,
                                                        float* factor) {
    pdl_wait();
    const float2 r = finish(parts, n, max_norm);
    if (threadIdx.x == 0) {
        if (norm) *norm = r.x;
        if (factor) *factor = r.y;
    }
}

// Each CTA sums the parts for itself: a launch between would cost more.
template <int N>
__global__ void __launch_bounds__(kThreads, 4)
scale_kernel(const __grid_constant__ Runs<N> a, const double* parts, int n_parts, double max_norm, float* norm,
             float* factor) {
    pdl_wait();
    const float2 r = finish(parts, n_parts, max_norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (norm) *norm = r.x;
        if (factor) *factor = r.y;
    }
    if (r.y == 1.0f) return;
    each_run<true>(a, [&](const Packs& x, uint4* w) {
        by_type(x.dtype, [&](auto t) {
#pragma unroll
            for (int k = 0; k < kPacks; ++k) w[k] = scaled<decltype(t)>(w[k], r.y);
        });
        store(w, x);
    });
}

// Launched so that it may start when the kernel before has, and waits for it.
template <typename... P, typename... A>
int launch_behind(void (*kernel)(P...), unsigned ctas, cudaStream_t st, A... args) {
    return cuda_check(launch_pdl(kernel, dim3(ctas), dim3(kThreads), 0, st, args...), "grad_norm launch");
}

struct Call {
    int count;
    void* const* grads;
    const int64_t* sizes;
    const int32_t* dtypes;
};

int check_list(const char* what, const Call& c, double max_norm, long long* total) {
    if (c.count < 0 || (c.count && (!c.grads || !c.sizes || !c.dtypes)))
        return fail(SN_E_INVAL, "%s: null list", what);
    if (!(max_norm >= 0.0)) return fail(SN_E_INVAL, "%s: max_norm is not a number of at least 0", what);
    *total = 0;
    for (int i = 0; i < c.count; ++i) {
        if (c.sizes[i] < 0) return fail(SN_E_INVAL, "%s: negative size", what);
        if (!dtype_size(c.dtypes[i])) return fail(SN_E_INVAL, "%s: dtype %d", what, c.dtypes[i]);
        if (c.sizes[i] && !c.grads[i]) return fail(SN_E_INVAL, "%s: null pointer", what);
        if (c.sizes[i] > (1ll << 46) - *total) return fail(SN_E_INVAL, "%s: too many values", what);
        *total += c.sizes[i];
    }
    return SN_OK;
}

// f(runs, CTAs, parts before them) for each launch of up to kMany tensors and
// kWave CTAs; how many parts there are. Where an address and type are not at hand
// yet, the most that they may take.
template <typename F>
int each_launch(const Call& c, long long* parts, F&& f) {
    *parts = 0;
    for (int i = 0; i < c.count;) {
        Runs<kMany> a;
        a.count = 0;
        long long n = 0;
        for (; i < c.count && a.count < kMany; ++i)
            if (c.sizes[i]) {
                const int type = c.dtypes ? c.dtypes[i] : SN_F32;
                const long long before = c.grads ? (long long)((uintptr_t)c.grads[i] & 15) : 15;
                const long long bytes = before + c.sizes[i] * (type == SN_F32 ? 4 : 2);
                const long long more = (bytes + 16 * kRun - 1) / (16 * kRun);
                if (n + more > 0x7fffffffll - kWave) {
                    if (a.count) break;
                    return fail(SN_E_INVAL, "grad_norm: a tensor of %lld values", (long long)c.sizes[i]);
                }
                a.t[a.count++] = {c.grads ? c.grads[i] : nullptr, c.sizes[i], (int)n, type};
                n += more;
            }
        if (!a.count) break;
        a.runs = (int)n;
        const unsigned ctas = (unsigned)std::min(n, (long long)kWave);
        if (a.count <= kFew) {
            Runs<kFew> b;
            b.count = a.count, b.runs = a.runs;
            for (int k = 0; k < a.count; ++k) b.t[k] = a.t[k];
            SN_TRY(f(b, ctas, *parts));
        } else {
            SN_TRY(f(a, ctas, *parts));
        }
        *parts += ctas;
    }
    return SN_OK;
}

int norm_or_clip(const char* what, const Call& c, double max_norm, bool clip, float* norm, float* factor, void* ws,
                 int64_t ws_bytes, void* cuda_stream) {
    CallerDevice dev;
    long long total;
    SN_TRY(check_list(what, c, max_norm, &total));
    long long n = 0;
    SN_TRY(each_launch(c, &n, [](const auto&, unsigned, long long) { return SN_OK; }));
    if (n && (!ws || ws_bytes < n * 8)) return fail(SN_E_INVAL, "%s: a workspace of %lld bytes is wanted", what, n * 8);
    for (int i = 0; i < c.count; ++i)
        if (c.sizes[i]) SN_TRY(dev.add(what, {c.grads[i], dtype_size(c.dtypes[i])}));
    for (const ArgPtr& p : {ArgPtr{norm, 4}, {factor, 4}, {ws, 8}}) SN_TRY(dev.add(what, p));
    SN_TRY(dev.select(what));
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    double* parts = static_cast<double*>(ws);
    SN_TRY(each_launch(c, &n, [&](const auto& a, unsigned ctas, long long before) {
        constexpr int N = sizeof(a.t) / sizeof(a.t[0]);
        square_kernel<N><<<ctas, kThreads, 0, st>>>(a, parts + before);
        return cuda_check(cudaGetLastError(), "grad_norm launch");
    }));
    const int count = (int)n;
    if (!clip || !n) return launch_behind(norm_kernel, 1u, st, (const double*)parts, count, max_norm, norm, factor);
    return each_launch(c, &n, [&](const auto& a, unsigned ctas, long long before) {
        constexpr int N = sizeof(a.t) / sizeof(a.t[0]);
        // (only the first of several may start early: its launch is the one behind the squares)
        if (!before)
            return launch_behind(scale_kernel<N>, ctas, st, a, (const double*)parts, count, max_norm, norm, factor);
        scale_kernel<N><<<ctas, kThreads, 0, st>>>(a, parts, count, max_norm, nullptr, nullptr);
        return cuda_check(cudaGetLastError(), "clip_grads launch");
    });
}

}  // namespace
}  // namespace sn

using namespace sn;

extern "C" {

int64_t sn_abi_grad_norm_ws(int32_t count, const int64_t* sizes) {
    if (count < 0 || (count && !sizes)) return -1;
    long long total = 0;
    for (int i = 0; i < count; ++i) {
        if (sizes[i] < 0 || sizes[i] > (1ll << 46) - total) return -1;
        total += sizes[i];
    }
    long long n = 0;
    const int rc = each_launch({count, nullptr, sizes, nullptr}, &n, [](const auto&, unsigned, long long) { return SN_OK; });
    return rc == SN_OK ? 8 * n : -1;
}

sn_status sn_abi_grad_norm(int32_t count, const void* const* grads, const int64_t* sizes, const int32_t* dtypes,
                           double max_norm, float* norm, float* factor, void* ws, int64_t ws_bytes,
                           void* cuda_stream) {
    return norm_or_clip("grad_norm", {count, const_cast<void* const*>(grads), sizes, dtypes}, max_norm, false, norm,
                        factor, ws, ws_bytes, cuda_stream);
}

sn_status sn_abi_clip_grads(int32_t count, void* const* grads, const int64_t* sizes, const int32_t* dtypes,
                            double max_norm, float* norm, float* factor, void* ws, int64_t ws_bytes,
                            void* cuda_stream) {
    return norm_or_clip("clip_grads", {count, grads, sizes, dtypes}, max_norm, true, norm, factor, ws, ws_bytes,
                        cuda_stream);
}

}  // extern "C"
