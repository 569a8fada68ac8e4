// The norm of a model's gradients and their clipping, over many tensors of any
// of the float types at once (no counterpart among the reference's kernels: its
// training loop leaves it to torch).
//
//   norm = sqrt(sum of g^2),  factor = min(1, max_norm / (norm + 1e-6)),  g = g * factor
//
// Squares of the values of one 16-byte load are added in fp32, everything above
// that in fp64, in an order that only the sizes decide; a load whose sum leaves
// fp32's normal numbers is squared in fp64 as well, so that values from 2^-149
// to the largest count.
//
// Bound by HBM: the norm reads every value once, clipping once more, and writes
// it. One wave of CTAs takes the tensors' runs of a few thousand values in turn;
// what the first pass read last is still in L2 when the second begins, so that
// goes from the last run to the first.
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
constexpr int kWave = 148 * 8;     // CTAs at most, each with one part of the sum
constexpr int kRun = 16384, kShort = 4096;  // values of a run; of a small model's, for more CTAs
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
    int per;  // values of a run
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

// Values of a run before its first multiple of 16 bytes.
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
    const int k = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) % 16 / sizeof(T));
    return k < n ? k : n;
}

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

constexpr int kAhead = 4;  // loads of a thread on their way

template <typename T>
__device__ __forceinline__ double square_run(const T* p, int n) {
    constexpr int V = 16 / sizeof(T);
    const int head = head_of(p, n), packs = (n - head) / V, tail = head + packs * V;
    double sum = 0.0;
    for (int i = threadIdx.x; i < head + (n - tail); i += kThreads) {
        const double x = (double)to_f(p[i < head ? i : tail + (i - head)]);
        sum = fma(x, x, sum);
    }
    const uint4* at = reinterpret_cast<const uint4*>(p + head);
    for (int i = threadIdx.x; i < packs; i += kAhead * kThreads) {
        uint4 w[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            w[k] = i + k * kThreads < packs ? at[i + k * kThreads] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) sum += squares<T>(w[k]);
    }
    return sum;
}

template <typename T>
__device__ __forceinline__ void scale_run(T* p, int n, float f) {
    constexpr int V = 16 / sizeof(T);
    const int head = head_of(p, n), packs = (n - head) / V, tail = head + packs * V;
    for (int i = threadIdx.x; i < head + (n - tail); i += kThreads) {
        T* at = p + (i < head ? i : tail + (i - head));
        *at = from_f<T>(to_f(*at) * f);
    }
    uint4* at = reinterpret_cast<uint4*>(p + head);
    const auto scaled = [&](const uint4& w) {
        Pack<T> q;
        q.w = w;
#pragma unroll
        for (int j = 0; j < V; ++j) q.v[j] = from_f<T>(to_f(q.v[j]) * f);
        return q.w;
    };
    for (int i = threadIdx.x; i < packs; i += kAhead * kThreads) {
        uint4 w[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (i + k * kThreads < packs) w[k] = at[i + k * kThreads];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            if (i + k * kThreads < packs) at[i + k * kThreads] = scaled(w[k]);
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

// f(values, how many) of run c.
template <int N, typename F>
__device__ __forceinline__ void with_run(const Runs<N>& a, int c, F&& f) {
    const Run& t = a.t[find(a, c)];
    const long long lo = (long long)(c - t.first) * a.per, left = t.n - lo;
    const int n = left < a.per ? (int)left : a.per;
    if (t.dtype == SN_F32)
        f(static_cast<float*>(t.p) + lo, n);
    else if (t.dtype == SN_BF16)
        f(static_cast<__nv_bfloat16*>(t.p) + lo, n);
    else
        f(static_cast<__half*>(t.p) + lo, n);
}

template <int N>
__global__ void __launch_bounds__(kThreads) square_kernel(const __grid_constant__ Runs<N> a, double* parts) {
    pdl_trigger();
    double x = 0.0;
    for (int c = blockIdx.x; c < a.runs; c += gridDim.x)
        with_run(a, c, [&](const auto* p, int n) { x += square_run(p, n); });
    x = cta_sum(x);
    if (threadIdx.x == 0) parts[blockIdx.x] = x;
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
__global__ void __launch_bounds__(kThreads)
scale_kernel(const __grid_constant__ Runs<N> a, const double* parts, int n_parts, double max_norm, float* norm,
             float* factor) {
    pdl_wait();
    const float2 r = finish(parts, n_parts, max_norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (norm) *norm = r.x;
        if (factor) *factor = r.y;
    }
    if (r.y == 1.0f) return;
    for (int c = a.runs - 1 - blockIdx.x; c >= 0; c -= gridDim.x)
        with_run(a, c, [&](auto* p, int n) { scale_run(p, n, r.y); });
}

// Launched so that it may start when the kernel before has, and waits for it.
template <typename... P, typename... A>
int launch_behind(void (*kernel)(P...), unsigned ctas, cudaStream_t st, A... args) {
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(ctas);
    c.blockDim = dim3(kThreads);
    c.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &at;
    c.numAttrs = 1;
    return cuda_check(cudaLaunchKernelEx(&c, kernel, args...), "grad_norm launch");
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

// How a list is cut up: launches of up to kMany tensors, each of up to kWave CTAs.
int run_values(long long total) { return total >= 2ll * kWave * kRun ? kRun : kShort; }

// f(runs, CTAs, parts before them) for each launch; how many parts there are.
template <typename F>
int each_launch(const Call& c, int per, long long* parts, F&& f) {
    *parts = 0;
    for (int i = 0; i < c.count;) {
        Runs<kMany> a;
        a.count = 0;
        a.per = per;
        long long n = 0;
        for (; i < c.count && a.count < kMany; ++i)
            if (c.sizes[i]) {
                const long long more = (c.sizes[i] + per - 1) / per;
                if (n + more > 0x7fffffffll - kWave) {
                    if (a.count) break;
                    return fail(SN_E_INVAL, "grad_norm: a tensor of %lld values", (long long)c.sizes[i]);
                }
                a.t[a.count++] = {c.grads ? c.grads[i] : nullptr, c.sizes[i], (int)n, c.dtypes ? c.dtypes[i] : 0};
                n += more;
            }
        if (!a.count) break;
        a.runs = (int)n;
        const unsigned ctas = (unsigned)std::min(n, (long long)kWave);
        if (a.count <= kFew) {
            Runs<kFew> b;
            b.count = a.count, b.runs = a.runs, b.per = per;
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
    long long total;
    SN_TRY(check_list(what, c, max_norm, &total));
    const int per = run_values(total);
    long long n = 0;
    SN_TRY(each_launch(c, per, &n, [](const auto&, unsigned, long long) { return SN_OK; }));
    if (n && (!ws || ws_bytes < n * 8)) return fail(SN_E_INVAL, "%s: a workspace of %lld bytes is wanted", what, n * 8);
    CallerDevice dev;
    for (int i = 0; i < c.count; ++i)
        if (c.sizes[i]) SN_TRY(dev.add(what, {c.grads[i], dtype_size(c.dtypes[i])}));
    for (const ArgPtr& p : {ArgPtr{norm, 4}, {factor, 4}, {ws, 8}}) SN_TRY(dev.add(what, p));
    SN_TRY(dev.select(what));
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    double* parts = static_cast<double*>(ws);
    SN_TRY(each_launch(c, per, &n, [&](const auto& a, unsigned ctas, long long before) {
        constexpr int N = sizeof(a.t) / sizeof(a.t[0]);
        square_kernel<N><<<ctas, kThreads, 0, st>>>(a, parts + before);
        return cuda_check(cudaGetLastError(), "grad_norm launch");
    }));
    const int count = (int)n;
    if (!clip || !n) return launch_behind(norm_kernel, 1u, st, (const double*)parts, count, max_norm, norm, factor);
    return each_launch(c, per, &n, [&](const auto& a, unsigned ctas, long long before) {
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
    const int rc = each_launch({count, nullptr, sizes, nullptr}, run_values(total), &n,
                               [](const auto&, unsigned, long long) { return SN_OK; });
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
