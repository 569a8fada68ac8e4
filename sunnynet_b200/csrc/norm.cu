// Layer norm and its gradients (no counterpart among the reference's kernels:
// its CenteredScaleNorm, model.py / ops.py:38-47, is this with
// eps = s_min^2 + 1e-5, computed by torch in training).
//
//   y  = (x - mean) * rstd * w + b       mean, rstd = 1/sqrt(var + eps) of a row
//   dx = rstd * (du - mean(du) - xhat * mean(du * xhat)),   du = dy * w
//   dw = sum over rows of dy * xhat,   db = sum over rows of dy
//
// Both passes are bound by HBM: forward reads x and writes y, backward reads
// x and dy and writes dx. A row lives in the registers of a group of threads
// (4 to 32 lanes of a warp, or a whole CTA) between its one read and its
// write, so the variance is the two-pass one (sum of squared differences
// from the mean) at no extra traffic. All sums are fp32.
//
// The weight gradients need a sum down the rows: each thread of the backward
// kernel keeps the sums of its own columns in registers over all the rows its
// group walks, a CTA adds its groups up in shared memory in a fixed order and
// writes one row of partial sums, and a second small kernel adds the CTAs'
// rows in order. No atomics: the same input gives the same bits.
//
// Rows wider than the register forms hold (kMaxWarpCols etc. below) take the
// *_wide kernels, one CTA per row, which read a row again from cache for each
// pass over it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "caller.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace sn {
namespace {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// PACK neighbouring elements moved by one load or store (16 bytes, or one
// element where the rows' addresses allow no more).
template <typename T, int PACK>
struct alignas(sizeof(T) * PACK) Pack {
    T v[PACK];
};

template <typename T, int PACK>
__device__ __forceinline__ void load_pack(const T* p, float (&f)[PACK]) {
    const Pack<T, PACK> r = *reinterpret_cast<const Pack<T, PACK>*>(p);
#pragma unroll
    for (int j = 0; j < PACK; ++j) f[j] = to_f(r.v[j]);
}

template <typename T, int PACK>
__device__ __forceinline__ void store_pack(T* p, const float (&f)[PACK]) {
    Pack<T, PACK> r;
#pragma unroll
    for (int j = 0; j < PACK; ++j) r.v[j] = from_f<T>(f[j]);
    *reinterpret_cast<Pack<T, PACK>*>(p) = r;
}

// Weight or bias columns [c, c + PACK): fp32, or the rows' own type.
template <typename T, int PACK>
__device__ __forceinline__ void load_param(const void* w, int wide, int c, float other,
                                           float (&f)[PACK]) {
    if (!w) {
#pragma unroll
        for (int j = 0; j < PACK; ++j) f[j] = other;
    } else if (wide) {
        constexpr int Q = PACK < 4 ? PACK : 4;
#pragma unroll
        for (int k = 0; k < PACK; k += Q) {
            float q[Q];
            load_pack<float, Q>(static_cast<const float*>(w) + c + k, q);
#pragma unroll
            for (int j = 0; j < Q; ++j) f[k + j] = q[j];
        }
    } else {
        load_pack<T, PACK>(static_cast<const T*>(w) + c, f);
    }
}

// Sum over the threads that share a row; every one of them gets it. G lanes
// of a warp, or (G == 0) the CTA, through `red` (32 floats, a buffer of its
// own for each call between two of the same buffer's barriers).
template <int G>
__device__ __forceinline__ float row_sum(float v, float* red) {
    constexpr int S = G ? G : 32;
#pragma unroll
    for (int o = S / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (G == 0) {
        const int w = threadIdx.x >> 5, nw = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0) red[w] = v;
        __syncthreads();
        v = 0.0f;
        for (int k = 0; k < nw; ++k) v += red[k];
    }
    return v;
}

struct FwdArgs {
    const void* x;
    const void* w;
    const void* b;
    void* y;
    float* mean;
    float* rstd;
    long long rows, ldx;
    int D, wide;  // wide: w and b are fp32
    float eps;
};

template <typename T, int PACK, int G, int NP>
__global__ void __launch_bounds__(G ? 128 : 512) norm_fwd_kernel(const FwdArgs a) {
    __shared__ float red[2][32];
    const int lane = G ? (int)(threadIdx.x % (G ? G : 1)) : (int)threadIdx.x;
    const int stride = G ? G : (int)blockDim.x;
    const long long row0 =
        G ? blockIdx.x * (long long)(blockDim.x / (G ? G : 1)) + threadIdx.x / (G ? G : 1)
          : blockIdx.x;
    const bool live = row0 < a.rows;  // the other lanes still take part in the shuffles
    const long long row = live ? row0 : 0;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float v[NP][PACK];
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int c = (i * stride + lane) * PACK;
        if (c < a.D) {
            load_pack<T, PACK>(x + c, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < PACK; ++j) v[i][j] = 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < PACK; ++j) sum += v[i][j];
    const float mean = __fdiv_rn(row_sum<G>(sum, red[0]), (float)a.D);
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const bool in = (i * stride + lane) * PACK < a.D;
#pragma unroll
        for (int j = 0; j < PACK; ++j) {
            v[i][j] -= mean;
            sq = in ? fmaf(v[i][j], v[i][j], sq) : sq;
        }
    }
    const float rstd =
        __frsqrt_rn(__fdiv_rn(row_sum<G>(sq, red[1]), (float)a.D) + a.eps);
    if (!live) return;
    if (lane == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.D;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int c = (i * stride + lane) * PACK;
        if (c >= a.D) continue;
        float w[PACK], b[PACK];
        load_param<T, PACK>(a.w, a.wide, c, 1.0f, w);
        load_param<T, PACK>(a.b, a.wide, c, 0.0f, b);
#pragma unroll
        for (int j = 0; j < PACK; ++j) v[i][j] = fmaf(v[i][j] * rstd, w[j], b[j]);
        store_pack<T, PACK>(y + c, v[i]);
    }
}

// Any width: three passes over the row, the last two from cache.
template <typename T>
__global__ void __launch_bounds__(512) norm_fwd_wide_kernel(const FwdArgs a) {
    __shared__ float red[2][32];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    float sum = 0.0f, sq = 0.0f;
    for (int c = threadIdx.x; c < a.D; c += blockDim.x) sum += to_f(x[c]);
    const float mean = __fdiv_rn(row_sum<0>(sum, red[0]), (float)a.D);
    for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
        const float d = to_f(x[c]) - mean;
        sq = fmaf(d, d, sq);
    }
    const float rstd = __frsqrt_rn(__fdiv_rn(row_sum<0>(sq, red[1]), (float)a.D) + a.eps);
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.D;
    for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
        float w[1], b[1];
        load_param<T, 1>(a.w, a.wide, c, 1.0f, w);
        load_param<T, 1>(a.b, a.wide, c, 0.0f, b);
        y[c] = from_f<T>(fmaf((to_f(x[c]) - mean) * rstd, w[0], b[0]));
    }
}

struct BwdArgs {
    const void* dy;
    const void* x;
    const void* w;
    const float* mean;
    const float* rstd;
    void* dx;       // may be null
    float* part;    // [2][gridDim.x][D] partial sums of dw and db; null: not wanted
    long long rows, ldx, lddy;
    int D, wide;
};

constexpr int kBwdThreads = 256;    // CTA of the warp-group forms
constexpr int kMaxWarpCols = 1024;  // columns a warp-group form can hold

template <typename T, int PACK, int G, int NP>
__global__ void __launch_bounds__(G ? kBwdThreads : 512) norm_bwd_kernel(const BwdArgs a) {
    __shared__ float red[4][32];
    __shared__ float colsum[G ? 2 * G * NP * PACK : 1];
    const int lane = G ? (int)(threadIdx.x % (G ? G : 1)) : (int)threadIdx.x;
    const int stride = G ? G : (int)blockDim.x;
    const int per = G ? (int)(blockDim.x / (G ? G : 1)) : 1;  // rows a CTA has in hand
    const int mine = G ? (int)(threadIdx.x / (G ? G : 1)) : 0;
    const float inv = __fdiv_rn(1.0f, (float)a.D);
    float aw[NP][PACK], ab[NP][PACK];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < PACK; ++j) aw[i][j] = ab[i][j] = 0.0f;

    int buf = 0;
    for (long long base = (long long)blockIdx.x * per; base < a.rows;
         base += (long long)gridDim.x * per) {
        const bool live = base + mine < a.rows;
        const long long row = live ? base + mine : 0;
        const T* x = static_cast<const T*>(a.x) + row * a.ldx;
        const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
        float xv[NP][PACK], gv[NP][PACK];
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = (i * stride + lane) * PACK;
            if (live && c < a.D) {
                load_pack<T, PACK>(x + c, xv[i]);
                load_pack<T, PACK>(dy + c, gv[i]);
            } else {
#pragma unroll
                for (int j = 0; j < PACK; ++j) xv[i][j] = gv[i][j] = 0.0f;
            }
        }
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s1 = 0.0f, s2 = 0.0f;  // sums of du and du * xhat
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = (i * stride + lane) * PACK;
            if (!(live && c < a.D)) continue;
            float w[PACK];
            load_param<T, PACK>(a.w, a.wide, c, 1.0f, w);
#pragma unroll
            for (int j = 0; j < PACK; ++j) {
                xv[i][j] = (xv[i][j] - mean) * rstd;
                aw[i][j] = fmaf(gv[i][j], xv[i][j], aw[i][j]);
                ab[i][j] += gv[i][j];
                gv[i][j] *= w[j];
                s1 += gv[i][j];
                s2 = fmaf(gv[i][j], xv[i][j], s2);
            }
        }
        if (!a.dx) continue;  // the whole grid alike
        s1 = row_sum<G>(s1, red[buf]) * inv;
        s2 = row_sum<G>(s2, red[buf + 1]) * inv;
        buf ^= 2;  // a buffer is written again only behind the next row's barriers
        if (live) {
            T* dx = static_cast<T*>(a.dx) + row * a.D;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int c = (i * stride + lane) * PACK;
                if (c >= a.D) continue;
                float o[PACK];
#pragma unroll
                for (int j = 0; j < PACK; ++j)
                    o[j] = rstd * (gv[i][j] - s1 - xv[i][j] * s2);
                store_pack<T, PACK>(dx + c, o);
            }
        }
    }
    if (!a.part) return;
    float* pw = a.part + (size_t)blockIdx.x * a.D;
    float* pb = pw + (size_t)gridDim.x * a.D;
    if (G == 0) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = (i * stride + lane) * PACK;
            if (c >= a.D) continue;
#pragma unroll
            for (int j = 0; j < PACK; ++j) {
                pw[c + j] = aw[i][j];
                pb[c + j] = ab[i][j];
            }
        }
        return;
    }
    // groups of one warp by shuffles, then the warps one after the other
    constexpr int cols = (G ? G : 1) * NP * PACK;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < PACK; ++j)
#pragma unroll
            for (int o = 16; o >= (G ? G : 32); o >>= 1) {
                aw[i][j] += __shfl_xor_sync(0xffffffffu, aw[i][j], o);
                ab[i][j] += __shfl_xor_sync(0xffffffffu, ab[i][j], o);
            }
    for (int k = 0; k < (int)(blockDim.x >> 5); ++k) {
        if ((int)(threadIdx.x >> 5) == k && (int)(threadIdx.x & 31) < (G ? G : 32)) {
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int j = 0; j < PACK; ++j) {
                    const int c = (i * stride + lane) * PACK + j;
                    colsum[c] = (k ? colsum[c] : 0.0f) + aw[i][j];
                    colsum[cols + c] = (k ? colsum[cols + c] : 0.0f) + ab[i][j];
                }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
        pw[c] = colsum[c];
        pb[c] = colsum[cols + c];
    }
}

// dx of rows of any width: two passes over the row, the second from cache.
template <typename T>
__global__ void __launch_bounds__(512) norm_dx_wide_kernel(const BwdArgs a) {
    __shared__ float red[2][32];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const float mean = a.mean[row], rstd = a.rstd[row], inv = __fdiv_rn(1.0f, (float)a.D);
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
        float w[1];
        load_param<T, 1>(a.w, a.wide, c, 1.0f, w);
        const float g = to_f(dy[c]) * w[0];
        s1 += g;
        s2 = fmaf(g, (to_f(x[c]) - mean) * rstd, s2);
    }
    s1 = row_sum<0>(s1, red[0]) * inv;
    s2 = row_sum<0>(s2, red[1]) * inv;
    T* dx = static_cast<T*>(a.dx) + row * a.D;
    for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
        float w[1];
        load_param<T, 1>(a.w, a.wide, c, 1.0f, w);
        dx[c] = from_f<T>(rstd * (to_f(dy[c]) * w[0] - s1 - (to_f(x[c]) - mean) * rstd * s2));
    }
}

// Partial dw, db of any width: 32 columns per CTA column, the rows of slice
// blockIdx.y over its 8 warps.
template <typename T>
__global__ void __launch_bounds__(256) norm_cols_wide_kernel(const BwdArgs a) {
    __shared__ float sw[8][32], sb[8][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    const long long lo = a.rows * blockIdx.y / gridDim.y, hi = a.rows * (blockIdx.y + 1) / gridDim.y;
    float aw = 0.0f, ab = 0.0f;
    if (c < a.D)
        for (long long r = lo + w; r < hi; r += 8) {
            const float g = to_f(static_cast<const T*>(a.dy)[r * a.lddy + c]);
            const float xh = (to_f(static_cast<const T*>(a.x)[r * a.ldx + c]) - a.mean[r]) * a.rstd[r];
            aw = fmaf(g, xh, aw);
            ab += g;
        }
    sw[w][lane] = aw;
    sb[w][lane] = ab;
    __syncthreads();
    if (w < 2 && c < a.D) {
        float s = 0.0f;
        for (int k = 0; k < 8; ++k) s += w ? sb[k][lane] : sw[k][lane];
        a.part[((size_t)w * gridDim.y + blockIdx.y) * a.D + c] = s;
    }
}

// out[c] = sum of P partial rows, in order within each of 16 slices, then the
// slices; blockIdx.y: 0 dw, 1 db.
template <typename W>
__global__ void __launch_bounds__(512)
    norm_cols_kernel(const float* __restrict__ part, int P, int D, W* dw, W* db) {
    __shared__ float s[16][32];
    W* out = blockIdx.y ? db : dw;
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    const float* p = part + (size_t)blockIdx.y * P * D + c;
    pdl_wait();
    float v = 0.0f;
    if (out && c < D)
        for (int r = k; r < P; r += 16) v += p[(size_t)r * D];
    s[k][lane] = v;
    __syncthreads();
    if (k == 0 && out && c < D) {
        v = s[0][lane];
        for (int i = 1; i < 16; ++i) v += s[i][lane];
        out[c] = from_f<W>(v);
    }
}

// How a row is laid over threads: G lanes of a warp (0: a CTA of `threads`),
// NP packs of PACK elements each.
struct Form {
    int G, NP, threads;
};

int round32(int v) { return (v + 31) / 32 * 32; }

// most: elements of a row a thread may hold. G == -1: no register form.
Form pick(int D, int pack, int most, int cta_threads) {
    const int packs = (D + pack - 1) / pack, np = most / pack;
    if (pack > 1)
        for (int g = 4; g < 32; g *= 2)
            if (packs <= g) return {g, 1, 0};
    const int need = (packs + 31) / 32;
    for (int n : {1, 2, 3, 4, 6, 8, 16, 32})
        if (n <= np && need <= n && n * 32 * pack <= kMaxWarpCols) return {32, n, 0};
    for (int n : {1, 2, 4, 8, 16, 32})
        if (n <= np && round32((packs + n - 1) / n) <= cta_threads)
            return {0, n, round32((packs + n - 1) / n)};
    return {-1, 0, 0};
}

constexpr int kFwdMost = 32, kBwdMost = 16, kBwdWarpMost = 24;

template <typename T, int PACK, int G, int NP>
int fwd_launch(const FwdArgs& a, int threads, cudaStream_t st) {
    const int per = G ? 128 / (G ? G : 1) : 1;
    const long long blocks = (a.rows + per - 1) / per;
    norm_fwd_kernel<T, PACK, G, NP><<<(unsigned)blocks, G ? 128 : threads, 0, st>>>(a);
    return cuda_check(cudaGetLastError(), "layer_norm launch");
}

template <typename T, int PACK>
int fwd_dispatch(const FwdArgs& a, cudaStream_t st) {
    const Form f = pick(a.D, PACK, kFwdMost, 512);
#define SN_FWD(g, n) \
    if (f.G == g && f.NP == n) return fwd_launch<T, PACK, g, n>(a, f.threads, st)
    if constexpr (PACK > 1) {
        SN_FWD(4, 1);
        SN_FWD(8, 1);
        SN_FWD(16, 1);
    }
    SN_FWD(32, 1);
    SN_FWD(32, 2);
    SN_FWD(32, 3);
    SN_FWD(32, 4);
    if constexpr (PACK <= 4) {
        SN_FWD(32, 6);
        SN_FWD(32, 8);
        SN_FWD(0, 8);
    }
    if constexpr (PACK == 1) {
        SN_FWD(32, 16);
        SN_FWD(32, 32);
        SN_FWD(0, 16);
        SN_FWD(0, 32);
    }
    SN_FWD(0, 1);
    SN_FWD(0, 2);
    SN_FWD(0, 4);
#undef SN_FWD
    norm_fwd_wide_kernel<T><<<(unsigned)a.rows, 512, 0, st>>>(a);
    return cuda_check(cudaGetLastError(), "layer_norm launch");
}

template <typename T>
int fwd_typed(const FwdArgs& a, bool vec, cudaStream_t st) {
    return vec ? fwd_dispatch<T, 16 / sizeof(T)>(a, st) : fwd_dispatch<T, 1>(a, st);
}

Form bwd_form(int D, int pack) {
    const Form f = pick(D, pack, kBwdWarpMost, 512);
    return f.G ? f : pick(D, pack, kBwdMost, 512);
}

// CTAs of the backward kernel: rows of the partial sums.
int bwd_parts(long long rows, int D, int pack, int sms) {
    const Form f = bwd_form(D, pack);
    long long want, cap;
    if (f.G < 0) {  // slices of norm_cols_wide_kernel
        const int cols = (D + 31) / 32;
        want = (rows + 63) / 64;
        cap = (8ll * sms + cols - 1) / cols;
    } else if (f.G) {
        const int per = kBwdThreads / f.G;
        want = (rows + per - 1) / per;
        cap = 2ll * sms;
    } else {
        want = rows;
        cap = (long long)sms * (f.threads <= 128 ? 4 : f.threads <= 256 ? 2 : 1);
    }
    const long long p = want < cap ? want : cap;
    return (int)(p < 1 ? 1 : p);
}

template <typename T, int PACK, int G, int NP>
int bwd_launch(const BwdArgs& a, int threads, int parts, cudaStream_t st) {
    norm_bwd_kernel<T, PACK, G, NP><<<parts, G ? kBwdThreads : threads, 0, st>>>(a);
    return cuda_check(cudaGetLastError(), "layer_norm_bwd launch");
}

template <typename T, int PACK>
int bwd_dispatch(const BwdArgs& a, int parts, cudaStream_t st) {
    const Form f = bwd_form(a.D, PACK);
#define SN_BWD(g, n) \
    if (f.G == g && f.NP == n) return bwd_launch<T, PACK, g, n>(a, f.threads, parts, st)
    if constexpr (PACK > 1) {
        SN_BWD(4, 1);
        SN_BWD(8, 1);
        SN_BWD(16, 1);
    }
    SN_BWD(32, 1);
    SN_BWD(32, 2);
    SN_BWD(32, 3);
    if constexpr (PACK <= 4) {
        SN_BWD(32, 4);
        SN_BWD(32, 6);
        SN_BWD(0, 4);
    }
    if constexpr (PACK == 1) {
        SN_BWD(32, 8);
        SN_BWD(32, 16);
        SN_BWD(0, 8);
        SN_BWD(0, 16);
    }
    SN_BWD(0, 1);
    SN_BWD(0, 2);
#undef SN_BWD
    if (a.dx) norm_dx_wide_kernel<T><<<(unsigned)a.rows, 512, 0, st>>>(a);
    SN_TRY(cuda_check(cudaGetLastError(), "layer_norm_bwd launch"));
    if (a.part) norm_cols_wide_kernel<T><<<dim3((a.D + 31) / 32, parts), 256, 0, st>>>(a);
    return cuda_check(cudaGetLastError(), "layer_norm_bwd launch");
}

template <typename T>
int bwd_typed(const BwdArgs& a, bool vec, int sms, void* dw, void* db, cudaStream_t st) {
    const int pack = vec ? 16 / (int)sizeof(T) : 1;
    const int parts = a.rows ? bwd_parts(a.rows, a.D, pack, sms) : 0;
    if (a.rows && (a.dx || a.part)) {
        if (vec)
            SN_TRY((bwd_dispatch<T, 16 / sizeof(T)>(a, parts, st)));
        else
            SN_TRY((bwd_dispatch<T, 1>(a, parts, st)));
    }
    if (!dw && !db) return SN_OK;
    const dim3 grid((a.D + 31) / 32, 2);
    return cuda_check(
        a.wide ? launch_pdl(norm_cols_kernel<float>, grid, dim3(512), 0, st, (const float*)a.part,
                            parts, a.D, (float*)dw, (float*)db)
               : launch_pdl(norm_cols_kernel<T>, grid, dim3(512), 0, st, (const float*)a.part,
                            parts, a.D, (T*)dw, (T*)db),
        "layer_norm_bwd launch");
}

// 16-byte loads and stores need 16-byte rows throughout.
bool rows16(const void* p, long long ld, unsigned size) {
    return ((uintptr_t)p & 15) == 0 && (ld * size) % 16 == 0;
}

bool shape_ok(long long rows, int D, long long ld) {
    return rows >= 0 && rows < (1ll << 31) && D > 0 && ld >= D;
}

}  // namespace
}  // namespace sn

using namespace sn;

extern "C" {

sn_status sn_abi_layer_norm(const void* x, int64_t ldx, const void* w, const void* b, void* y,
                            float* mean, float* rstd, int32_t dtype, int32_t wdtype,
                            int64_t rows, int32_t D, float eps, void* cuda_stream) {
    const unsigned size = dtype_size(dtype), ws = dtype_size(wdtype);
    if (!size || !ws || (wdtype != SN_F32 && wdtype != dtype))
        return fail(SN_E_INVAL, "layer_norm: dtype %d with weights of %d", dtype, wdtype);
    if (!shape_ok(rows, D, ldx)) return fail(SN_E_INVAL, "layer_norm: bad dimension");
    if (!(eps >= 0.0f)) return fail(SN_E_INVAL, "layer_norm: eps must not be negative");
    if (rows == 0) return SN_OK;
    if (!x || !y) return fail(SN_E_INVAL, "layer_norm: null pointer");
    CallerDevice dev;
    SN_TRY(dev.enter("layer_norm", {{x, size}, {w, ws}, {b, ws}, {y, size}, {mean, 4}, {rstd, 4}}));
    const FwdArgs a{x, w, b, y, mean, rstd, rows, ldx, D, wdtype == SN_F32, eps};
    const bool vec = rows16(x, ldx, size) && rows16(y, D, size) && (!w || rows16(w, 0, ws)) &&
                     (!b || rows16(b, 0, ws)) && D % (16 / size) == 0;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    switch (dtype) {
        case SN_F32: return fwd_typed<float>(a, vec, st);
        case SN_BF16: return fwd_typed<__nv_bfloat16>(a, vec, st);
        default: return fwd_typed<__half>(a, vec, st);
    }
}

int64_t sn_abi_layer_norm_bwd_ws(int64_t rows, int32_t D, int32_t dtype) {
    const unsigned size = dtype_size(dtype);
    if (!size || !shape_ok(rows, D, D)) return 0;
    CallerDevice dev;
    const int sms = dev.select("layer_norm_bwd_ws") == SN_OK ? dev.num_sms() : 148;
    const int a = bwd_parts(rows, D, 1, sms), b = bwd_parts(rows, D, 16 / (int)size, sms);
    return 8ll * (a > b ? a : b) * D;
}

sn_status sn_abi_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx,
                                const void* w, const float* mean, const float* rstd, void* dx,
                                void* dw, void* db, void* ws, int64_t ws_bytes, int32_t dtype,
                                int32_t wdtype, int64_t rows, int32_t D, void* cuda_stream) {
    const unsigned size = dtype_size(dtype), wsz = dtype_size(wdtype);
    if (!size || !wsz || (wdtype != SN_F32 && wdtype != dtype))
        return fail(SN_E_INVAL, "layer_norm_bwd: dtype %d with weights of %d", dtype, wdtype);
    if (!shape_ok(rows, D, ldx) || lddy < D)
        return fail(SN_E_INVAL, "layer_norm_bwd: bad dimension");
    if (rows && (!dy || !x || !mean || !rstd))
        return fail(SN_E_INVAL, "layer_norm_bwd: null pointer");
    if (!dx && !dw && !db) return SN_OK;
    CallerDevice dev;
    SN_TRY(dev.enter("layer_norm_bwd", {{dy, size}, {x, size}, {w, wsz}, {mean, 4}, {rstd, 4},
                                        {dx, size}, {dw, wsz}, {db, wsz}, {ws, 4}}));
    const bool sums = dw || db;
    if (sums && rows && (!ws || ws_bytes < sn_abi_layer_norm_bwd_ws(rows, D, dtype)))
        return fail(SN_E_INVAL, "layer_norm_bwd: the workspace needs %lld bytes",
                    (long long)sn_abi_layer_norm_bwd_ws(rows, D, dtype));
    const BwdArgs a{dy, x, w, mean, rstd, dx, sums ? static_cast<float*>(ws) : nullptr, rows,
                    ldx, lddy, D, wdtype == SN_F32};
    const bool vec = rows16(dy, lddy, size) && rows16(x, ldx, size) && (!w || rows16(w, 0, wsz)) &&
                     (!dx || rows16(dx, D, size)) && D % (16 / size) == 0;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    switch (dtype) {
        case SN_F32: return bwd_typed<float>(a, vec, dev.num_sms(), dw, db, st);
        case SN_BF16: return bwd_typed<__nv_bfloat16>(a, vec, dev.num_sms(), dw, db, st);
        default: return bwd_typed<__half>(a, vec, dev.num_sms(), dw, db, st);
    }
}

}  // extern "C"
