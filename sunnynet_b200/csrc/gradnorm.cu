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
// it. One wave of CTAs takes the values, each one run of one tensor; what the
// first pass read last is still in L2 when the second begins, so that goes
// through each run from its end.
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
constexpr int kWave = 148 * 8;     // runs that the values are cut into (and one more for each tensor)
constexpr int kLeast = 4096;       // values of a run, or a multiple
constexpr int kFew = 32, kMany = 1280;  // tensors of a launch: 30 of the 32 KB of parameters

struct Run {
    void* p;
    long long n;
    int first;  // its first run among the launch's
    int dtype;
};

template <int N>
struct Runs {
    int count;
    long long per;  // values of a run
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
__device__ __forceinline__ long long head_of(const T* p, long long n) {
    const long long k = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) % 16 / sizeof(T);
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
__device__ __forceinline__ double square_run(const T* p, long long n) {
    constexpr int V = 16 / sizeof(T);
    const long long head = head_of(p, n), packs = (n - head) / V, tail = head + packs * V;
    double sum = 0.0;
    for (long long i = threadIdx.x; i < head + (n - tail); i += kThreads) {
        const double x = (double)to_f(p[i < head ? i : tail + (i - head)]);
        sum = fma(x, x, sum);
    }
    const uint4* at = reinterpret_cast<const uint4*>(p + head);
    long long i = threadIdx.x;
    for (; i + (kAhead - 1) * kThreads < packs; i += kAhead * kThreads) {
        uint4 w[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) w[k] = at[i + k * kThreads];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) sum += squares<T>(w[k]);
    }
    for (; i < packs; i += kThreads) sum += squares<T>(at[i]);
    return sum;
}

template <typename T>
__device__ __forceinline__ void scale_run(T* p, long long n, float f) {
    constexpr int V = 16 / sizeof(T);
    const long long head = head_of(p, n), packs = (n - head) / V, tail = head + packs * V;
    for (long long i = threadIdx.x; i < head + (n - tail); i += kThreads) {
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
    long long i = packs - 1 - threadIdx.x;
    for (; i - (kAhead - 1) * kThreads >= 0; i -= kAhead * kThreads) {
        uint4 w[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) w[k] = at[i - k * kThreads];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) at[i - k * kThreads] = scaled(w[k]);
    }
    for (; i >= 0; i -= kThreads) at[i] = scaled(at[i]);
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
__global__ void __launch_bounds__(kThreads) square_kernel(const __grid_constant__ Runs<N> a, double* parts) {
    pdl_trigger();
    const Run& t = a.t[find(a, blockIdx.x)];
    const long long lo = (blockIdx.x - t.first) * a.per, n = min(a.per, t.n - lo);
    double x;
    if (t.dtype == SN_F32)
        x = square_run(static_cast<const float*>(t.p) + lo, n);
    else if (t.dtype == SN_BF16)
        x = square_run(static_cast<const __nv_bfloat16*>(t.p) + lo, n);
    else
        x = square_run(static_cast<const __half*>(t.p) + lo, n);
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
    const Run& t = a.t[find(a, blockIdx.x)];
    const long long lo = (blockIdx.x - t.first) * a.per, n = min(a.per, t.n - lo);
    if (t.dtype == SN_F32)
        scale_run(static_cast<float*>(t.p) + lo, n, r.y);
    else if (t.dtype == SN_BF16)
        scale_run(static_cast<__nv_bfloat16*>(t.p) + lo, n, r.y);
    else
        scale_run(static_cast<__half*>(t.p) + lo, n, r.y);
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

long long run_values(long long total) {
    const long long per = (total + kWave - 1) / kWave;
    return std::max(1ll, (per + kLeast - 1) / kLeast) * kLeast;
}

long long runs_of(const Call& c, long long per) {
    long long n = 0;
    for (int i = 0; i < c.count; ++i) n += (c.sizes[i] + per - 1) / per;
    return n;
}

// Launches of up to kMany tensors: f(runs, ctas, runs before them).
template <typename F>
int each_launch(const Call& c, long long per, F&& f) {
    long long before = 0;
    for (int i = 0; i < c.count;) {
        Runs<kMany> a;
        a.count = 0;
        a.per = per;
        long long n = 0;
        for (; i < c.count && a.count < kMany; ++i)
            if (c.sizes[i]) {
                a.t[a.count++] = {c.grads[i], c.sizes[i], (int)n, c.dtypes[i]};
                n += (c.sizes[i] + per - 1) / per;
            }
        if (!a.count) break;
        if (a.count <= kFew) {
            Runs<kFew> b;
            b.count = a.count;
            b.per = per;
            for (int k = 0; k < a.count; ++k) b.t[k] = a.t[k];
            SN_TRY(f(b, (unsigned)n, before));
        } else {
            SN_TRY(f(a, (unsigned)n, before));
        }
        before += n;
    }
    return SN_OK;
}

int norm_or_clip(const char* what, const Call& c, double max_norm, bool clip, float* norm, float* factor, void* ws,
                 int64_t ws_bytes, void* cuda_stream) {
    long long total;
    SN_TRY(check_list(what, c, max_norm, &total));
    const long long per = run_values(total), n = runs_of(c, per);
    if (n > 0x7fffffffll) return fail(SN_E_INVAL, "%s: too many tensors", what);
    if (n && (!ws || ws_bytes < n * 8)) return fail(SN_E_INVAL, "%s: a workspace of %lld bytes is wanted", what, n * 8);
    CallerDevice dev;
    for (int i = 0; i < c.count; ++i)
        if (c.sizes[i]) SN_TRY(dev.add(what, {c.grads[i], dtype_size(c.dtypes[i])}));
    for (const ArgPtr& p : {ArgPtr{norm, 4}, {factor, 4}, {ws, 8}}) SN_TRY(dev.add(what, p));
    SN_TRY(dev.select(what));
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    double* parts = static_cast<double*>(ws);
    SN_TRY(each_launch(c, per, [&](const auto& a, unsigned ctas, long long before) {
        constexpr int N = sizeof(a.t) / sizeof(a.t[0]);
        square_kernel<N><<<ctas, kThreads, 0, st>>>(a, parts + before);
        return cuda_check(cudaGetLastError(), "grad_norm launch");
    }));
    if (!clip || !n) return launch_behind(norm_kernel, 1u, st, (const double*)parts, (int)n, max_norm, norm, factor);
    return each_launch(c, per, [&](const auto& a, unsigned ctas, long long before) {
        constexpr int N = sizeof(a.t) / sizeof(a.t[0]);
        (void)before;
        // (only the first of several may start early: its launch is the one behind the squares)
        if (!before)
            return launch_behind(scale_kernel<N>, ctas, st, a, (const double*)parts, (int)n, max_norm, norm, factor);
        scale_kernel<N><<<ctas, kThreads, 0, st>>>(a, parts, (int)n, max_norm, nullptr, nullptr);
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
    return 8 * runs_of({count, nullptr, sizes, nullptr}, run_values(total));
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
