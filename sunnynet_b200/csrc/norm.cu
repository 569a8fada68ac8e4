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
// from the mean) at no extra traffic. All sums are fp32. 32768 x 768 in fp32:
// forward 37 us, backward with the weights' gradients 57 (0.83 and 0.80 of the
// copy rate); in bf16 25 and 39 (0.62, 0.59), where a row's instructions and the
// rows that the registers leave room for count as much as its bytes.
//
// The weight gradients need a sum down the rows: each thread of the backward
// kernel keeps the sums of its own columns in registers over all the rows its
// group walks, a CTA adds its groups up in shared memory in a fixed order and
// writes one row of partial sums, and a second small kernel adds the CTAs'
// rows in order. No atomics: the same input gives the same bits.
//
// Rows of an odd width start anywhere in a 16-byte unit. They are still moved in
// 16-byte packs: the packs are those of memory, a row's first and last being
// partly its neighbours' (EDGE: those two element by element). A group of
// threads that walks rows takes those at one distance from a boundary only, so
// a thread keeps the same columns throughout.
//
// Rows wider than the register forms hold (see pick) take the *_wide kernels,
// one CTA per row, which read a row again from cache for each pass over it (1000
// x 33000 in fp32: forward 78 us, 0.52 of the copy rate, backward 171, 0.35).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

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

// Columns [c, c + PACK) of a row at p as they are in memory, 0 where a row of D
// has none (EDGE; c may be negative).
template <typename T, int PACK, bool EDGE>
__device__ __forceinline__ Pack<T, PACK> load_cols(const T* p, int c, int D) {
    Pack<T, PACK> r;
    if (c >= (EDGE ? 0 : c) && c + PACK <= D) {
        r = *reinterpret_cast<const Pack<T, PACK>*>(p + c);
    } else {
#pragma unroll
        for (int j = 0; j < PACK; ++j)
            r.v[j] = EDGE && c + j >= 0 && c + j < D ? p[c + j] : from_f<T>(0.0f);
    }
    return r;
}

template <typename T, int PACK, bool EDGE>
__device__ __forceinline__ void store_cols(T* p, int c, int D, const float (&f)[PACK]) {
    if (!EDGE || (c >= 0 && c + PACK <= D)) {
        store_pack<T, PACK>(p + c, f);
    } else {
#pragma unroll
        for (int j = 0; j < PACK; ++j)
            if (c + j >= 0 && c + j < D) p[c + j] = from_f<T>(f[j]);
    }
}

// Weight or bias columns [c, c + PACK): fp32, or the rows' own type.
template <typename T, int PACK, bool EDGE>
__device__ __forceinline__ void load_param(const void* w, int wide, int c, int D, float other,
                                           float (&f)[PACK]) {
    if (!w) {
#pragma unroll
        for (int j = 0; j < PACK; ++j) f[j] = other;
    } else if (EDGE) {  // at no boundary of their own
#pragma unroll
        for (int j = 0; j < PACK; ++j) {
            const int k = min(max(c + j, 0), D - 1);
            f[j] = wide ? static_cast<const float*>(w)[k] : to_f(static_cast<const T*>(w)[k]);
        }
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

// Whether some of columns [c, c + PACK) are none of a row of D, so that each has
// to be asked for. The first and the last pack of a row that a CTA shares (8190
// columns in bf16 take 48 us so, 52 where every column is asked for); of a row
// in a warp, where most warps hold such a pack, always (20000 x 333 in bf16 20
// us, and 22 with a branch).
template <int PACK, int G>
__device__ __forceinline__ bool sticks_out(int c, int D) {
    return G || c < 0 || c + PACK > D;
}

// Elements from the 16-byte boundary at or before p to p.
template <typename T, bool EDGE>
__device__ __forceinline__ int past_boundary(const T* p) {
    return EDGE ? (int)((uintptr_t)p & 15) / (int)sizeof(T) : 0;
}

// Sums over the threads that share a row; every one of them gets them. G lanes
// of a warp, or (G == 0) the CTA, through `red` (a buffer that is not written
// again before another barrier of these).
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

template <int G>
__device__ __forceinline__ float2 row_sums(float2 v, float2* red) {
    constexpr int S = G ? G : 32;
#pragma unroll
    for (int o = S / 2; o; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if (G == 0) {
        const int w = threadIdx.x >> 5, nw = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0) red[w] = v;
        __syncthreads();
        v = make_float2(0.0f, 0.0f);
        for (int k = 0; k < nw; ++k) v.x += red[k].x, v.y += red[k].y;
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

// A group of threads per row. (Groups that walk rows, each loading its next row
// before it works on the one in hand, were slower: 43 us instead of 37 for
// 32768 x 768 in fp32. Their registers cost more warps than the rows in flight
// gain.)
template <typename T, int PACK, int G, int NP, bool EDGE>
__global__ void __launch_bounds__(G ? 128 : 512) norm_fwd_kernel(const FwdArgs a) {
    constexpr int W = G ? G : 1;
    __shared__ float red[2][32];
    const int lane = G ? (int)(threadIdx.x % W) : (int)threadIdx.x;
    const int stride = G ? G : (int)blockDim.x;
    const long long row0 =
        G ? blockIdx.x * (long long)(blockDim.x / W) + threadIdx.x / W : (long long)blockIdx.x;
    const bool live = row0 < a.rows;  // the other lanes still take part in the shuffles
    const long long row = live ? row0 : 0;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const int skip = past_boundary<T, EDGE>(x);
    float v[NP][PACK];
    float sum = 0.0f;
    {
        Pack<T, PACK> p[NP];
#pragma unroll
        for (int i = 0; i < NP; ++i)
            p[i] = load_cols<T, PACK, EDGE>(x, (i * stride + lane) * PACK - skip, a.D);
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int j = 0; j < PACK; ++j) {
                v[i][j] = to_f(p[i].v[j]);
                sum += v[i][j];
            }
    }
    const float mean = __fdiv_rn(row_sum<G>(sum, red[0]), (float)a.D);
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int c = (i * stride + lane) * PACK - skip;
#pragma unroll
        for (int j = 0; j < PACK; ++j) v[i][j] -= mean;
        if (sticks_out<PACK, G>(c, a.D)) {
#pragma unroll
            for (int j = 0; j < PACK; ++j)
                if (EDGE ? c + j < 0 || c + j >= a.D : c >= a.D) v[i][j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < PACK; ++j) sq = fmaf(v[i][j], v[i][j], sq);
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
        const int c = (i * stride + lane) * PACK - skip;
        if (c >= a.D) continue;
        float w[PACK], b[PACK];
        load_param<T, PACK, EDGE>(a.w, a.wide, c, a.D, 1.0f, w);
        load_param<T, PACK, EDGE>(a.b, a.wide, c, a.D, 0.0f, b);
#pragma unroll
        for (int j = 0; j < PACK; ++j) v[i][j] = fmaf(v[i][j] * rstd, w[j], b[j]);
        store_cols<T, PACK, EDGE>(y, c, a.D, v[i]);
    }
}

// Any width: three passes over the row, the last two from cache.
template <typename T, int PACK, bool EDGE>
__global__ void __launch_bounds__(512) norm_fwd_wide_kernel(const FwdArgs a) {
    __shared__ float red[2][32];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const int skip = past_boundary<T, EDGE>(x), c0 = (int)threadIdx.x * PACK - skip;
    const int by = (int)blockDim.x * PACK;
    float sum = 0.0f, sq = 0.0f;
#pragma unroll 4
    for (int c = c0; c < a.D; c += by) {
        const Pack<T, PACK> p = load_cols<T, PACK, EDGE>(x, c, a.D);
#pragma unroll
        for (int j = 0; j < PACK; ++j) sum += to_f(p.v[j]);
    }
    const float mean = __fdiv_rn(row_sum<0>(sum, red[0]), (float)a.D);
#pragma unroll 4
    for (int c = c0; c < a.D; c += by) {
        const Pack<T, PACK> p = load_cols<T, PACK, EDGE>(x, c, a.D);
#pragma unroll
        for (int j = 0; j < PACK; ++j) {
            const float d = to_f(p.v[j]) - mean;
            sq = !EDGE || (c + j >= 0 && c + j < a.D) ? fmaf(d, d, sq) : sq;
        }
    }
    const float rstd = __frsqrt_rn(__fdiv_rn(row_sum<0>(sq, red[1]), (float)a.D) + a.eps);
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[row] = mean;
        if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.D;
#pragma unroll 2
    for (int c = c0; c < a.D; c += by) {
        const Pack<T, PACK> p = load_cols<T, PACK, EDGE>(x, c, a.D);
        float w[PACK], b[PACK], o[PACK];
        load_param<T, PACK, EDGE>(a.w, a.wide, c, a.D, 1.0f, w);
        load_param<T, PACK, EDGE>(a.b, a.wide, c, a.D, 0.0f, b);
#pragma unroll
        for (int j = 0; j < PACK; ++j) o[j] = fmaf((to_f(p.v[j]) - mean) * rstd, w[j], b[j]);
        store_cols<T, PACK, EDGE>(y, c, a.D, o);
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

// Threads of a CTA of the warp-group forms: each CTA leaves a row of partial
// sums, so few large ones where registers allow.
constexpr int bwd_threads(int elems) { return elems <= 8 ? 256 : 128; }

// Rows of a group on their way or in hand: 3, or 2 where a thread's part of a
// row is large (a CTA's slots then leave room for others on the SM).
constexpr int bwd_ahead(int bytes) { return bytes >= 64 ? 2 : 3; }

// Bytes of a thread's slots: those rows of x and dy, and its weights in fp32.
constexpr int bwd_slot_bytes(int elem, int elems) {
    return elems * (2 * bwd_ahead(elem * elems) * elem + 4);
}

// A thread's PACK fp32 values of its i-th pack, in runs of 16 bytes so that a
// warp's accesses meet no bank twice.
template <int PACK, typename Q>
__device__ __forceinline__ void put_wide(Q* to, int i, const float* v) {
    constexpr int R = sizeof(Q) / sizeof(float);
#pragma unroll
    for (int h = 0; h < PACK / R; ++h) {
        Q q;
#pragma unroll
        for (int j = 0; j < R; ++j) q.v[j] = v[h * R + j];
        to[(i * (PACK / R) + h) * (int)blockDim.x] = q;
    }
}

template <int PACK, typename Q>
__device__ __forceinline__ void get_wide(const Q* from, int i, float* v) {
    constexpr int R = sizeof(Q) / sizeof(float);
#pragma unroll
    for (int h = 0; h < PACK / R; ++h) {
        const Q q = from[(i * (PACK / R) + h) * (int)blockDim.x];
#pragma unroll
        for (int j = 0; j < R; ++j) v[h * R + j] = q.v[j];
    }
}

// The rows a group has yet to work on wait in shared memory, brought in by
// cp.async: registers for them would cost the warps that hide what is left
// (each thread reads back only what it copied itself, so no barrier is due).
template <typename T, int PACK, int G, int NP, bool EDGE>
__global__ void __launch_bounds__(G ? bwd_threads(PACK * NP) : 512) norm_bwd_kernel(const BwdArgs a) {
    constexpr int W = G ? G : 1, kAhead = bwd_ahead(sizeof(T) * PACK * NP);
    typedef Pack<T, PACK> P;
    extern __shared__ __align__(128) unsigned char slots[];
    __shared__ float2 red[2][32];
    __shared__ float colsum[G ? 2 * W * NP * PACK : 1];
    const int lane = G ? (int)(threadIdx.x % W) : (int)threadIdx.x;
    const int stride = G ? G : (int)blockDim.x;
    // a CTA has `per` rows in hand; the step from one to the next of a group is
    // a multiple of 8, after which rows begin at the same place in a 16-byte unit
    const int per = G ? (int)(blockDim.x / W) : 1;
    const int mine = G ? (int)(threadIdx.x / W) : 0;
    const float inv = __fdiv_rn(1.0f, (float)a.D);
    const long long step = (long long)gridDim.x * per;
    long long base = (long long)blockIdx.x * per;
    const int skip = past_boundary<T, EDGE>(static_cast<const T*>(a.x) +
                                            min(base + mine, a.rows - 1) * a.ldx);
    const auto col = [&](int i) { return (i * stride + lane) * PACK - skip; };
    P* const rows = reinterpret_cast<P*>(slots) + threadIdx.x;  // [kAhead][2][NP][threads]
    const auto slot = [&](int stage, int which, int i) -> P* {
        return rows + ((stage * 2 + which) * NP + i) * (int)blockDim.x;
    };
    Pack<float, PACK <= 4 ? PACK : 4>* const weights =
        reinterpret_cast<Pack<float, PACK <= 4 ? PACK : 4>*>(reinterpret_cast<P*>(slots) +
                                                            kAhead * 2 * NP * blockDim.x) +
        threadIdx.x;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        Pack<float, PACK> w;
#pragma unroll
        for (int j = 0; j < PACK; ++j) w.v[j] = 0.0f;
        if (col(i) < a.D) load_param<T, PACK, EDGE>(a.w, a.wide, col(i), a.D, 1.0f, w.v);
        put_wide<PACK>(weights, i, w.v);
    }
    float aw[NP][PACK], ab[NP][PACK];
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
        for (int j = 0; j < PACK; ++j) aw[i][j] = ab[i][j] = 0.0f;

    const auto fetch = [&](long long row, int stage) {
        if (row < a.rows) {
            const T* from[2] = {static_cast<const T*>(a.x) + row * a.ldx,
                                static_cast<const T*>(a.dy) + row * a.lddy};
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int c = col(i);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if constexpr (sizeof(P) != 16) {
                        *slot(stage, k, i) = load_cols<T, PACK, EDGE>(from[k], c, a.D);
                    } else if (!EDGE || (c >= 0 && c + PACK <= a.D)) {
                        if (c < a.D) cp_async16(slot(stage, k, i), from[k] + c, 16);
                    } else if (c < a.D) {
                        // partly a neighbouring row's, which is there to be read
                        // but in front of the first row and behind the last
                        const long long ld = k ? a.lddy : a.ldx, at = row * ld + c;
                        if (at >= 0 && at + PACK <= (a.rows - 1) * ld + a.D)
                            cp_async16(slot(stage, k, i), from[k] + c, 16);
                        else
                            *slot(stage, k, i) = load_cols<T, PACK, EDGE>(from[k], c, a.D);
                    }
                }
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < kAhead - 1; ++k) fetch(base + mine + k * step, k);
    int stage = 0;
    // a row's statistics are asked for while the row before it is worked on, in 16
    // bits (32768 x 768: 42 us without, 38 with; in fp32, where the rows take
    // longer to come, their registers cost as much: 57 and 59)
    constexpr bool kAsk = sizeof(T) == 2;
    float mean = 0.0f, rstd = 0.0f, next_mean = 0.0f, next_rstd = 0.0f;
    if (kAsk && base + mine < a.rows) next_mean = a.mean[base + mine], next_rstd = a.rstd[base + mine];
    for (int buf = 0; base < a.rows; base += step, buf ^= 1) {
        const long long row = base + mine;
        const bool live = row < a.rows;
        if (kAsk) {
            mean = next_mean, rstd = next_rstd;
            if (row + step < a.rows) next_mean = a.mean[row + step], next_rstd = a.rstd[row + step];
        } else {
            mean = live ? a.mean[row] : 0.0f, rstd = live ? a.rstd[row] : 0.0f;
        }
        fetch(row + (kAhead - 1) * step, stage == 0 ? kAhead - 1 : stage - 1);
        cp_async_wait_group<kAhead - 1>();
        float xv[NP][PACK], gv[NP][PACK];
        float2 sum = make_float2(0.0f, 0.0f);  // of du and du * xhat
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = col(i);
            if (!(live && c < a.D)) {
#pragma unroll
                for (int j = 0; j < PACK; ++j) xv[i][j] = gv[i][j] = 0.0f;
                continue;
            }
            const P x = *slot(stage, 0, i), g = *slot(stage, 1, i);
            Pack<float, PACK> w;
            get_wide<PACK>(weights, i, w.v);
#pragma unroll
            for (int j = 0; j < PACK; ++j) {
                xv[i][j] = (to_f(x.v[j]) - mean) * rstd;
                gv[i][j] = to_f(g.v[j]);
                if (EDGE && (c + j < 0 || c + j >= a.D)) xv[i][j] = gv[i][j] = 0.0f;
                aw[i][j] = fmaf(gv[i][j], xv[i][j], aw[i][j]);
                ab[i][j] += gv[i][j];
                gv[i][j] *= w.v[j];
                sum.x += gv[i][j];
                sum.y = fmaf(gv[i][j], xv[i][j], sum.y);
            }
        }
        stage = stage == kAhead - 1 ? 0 : stage + 1;
        if (!a.dx) continue;  // the whole grid alike
        sum = row_sums<G>(sum, red[buf]);
        const float s1 = sum.x * inv, s2 = sum.y * inv;
        if (live) {
            T* dx = static_cast<T*>(a.dx) + row * a.D;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int c = col(i);
                if (c >= a.D) continue;
                float o[PACK];
#pragma unroll
                for (int j = 0; j < PACK; ++j)
                    o[j] = rstd * (gv[i][j] - s1 - xv[i][j] * s2);
                store_cols<T, PACK, EDGE>(dx, c, a.D, o);
            }
        }
    }
    if (!a.part) return;
    float* pw = a.part + (size_t)blockIdx.x * a.D;
    float* pb = pw + (size_t)gridDim.x * a.D;
    if (G == 0) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int j = 0; j < PACK; ++j) {
                const int c = (i * stride + lane) * PACK + j - skip;
                if (c >= 0 && c < a.D) {
                    pw[c] = aw[i][j];
                    pb[c] = ab[i][j];
                }
            }
        return;
    }
    // groups of one warp by shuffles (where they share columns), then the warps
    // one after the other
    constexpr int cols = W * NP * PACK;
    if (!EDGE) {
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int j = 0; j < PACK; ++j)
#pragma unroll
                for (int o = 16; o >= (G ? G : 32); o >>= 1) {
                    aw[i][j] += __shfl_xor_sync(0xffffffffu, aw[i][j], o);
                    ab[i][j] += __shfl_xor_sync(0xffffffffu, ab[i][j], o);
                }
    } else {
        for (int c = threadIdx.x; c < 2 * cols; c += blockDim.x) colsum[c] = 0.0f;
        __syncthreads();
    }
    for (int k = 0; k < (EDGE ? per : (int)(blockDim.x >> 5)); ++k) {
        if (EDGE ? mine == k : (int)(threadIdx.x >> 5) == k && (int)(threadIdx.x & 31) < W) {
#pragma unroll
            for (int i = 0; i < NP; ++i)
#pragma unroll
                for (int j = 0; j < PACK; ++j) {
                    const int c = (i * stride + lane) * PACK + j - skip;
                    if (EDGE && (c < 0 || c >= a.D)) continue;
                    colsum[c] = (EDGE || k ? colsum[c] : 0.0f) + aw[i][j];
                    colsum[cols + c] = (EDGE || k ? colsum[cols + c] : 0.0f) + ab[i][j];
                }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < a.D; c += blockDim.x) {
        pw[c] = colsum[c];
        pb[c] = colsum[cols + c];
    }
}

// Forward over many 16-bit rows of an odd width: a lane's columns lie at no
// boundary of the weights, and loading these one by one for each row took most
// of norm_fwd_kernel's time (3000 x 8190 in bf16: 86 us, and 48 here). Here
// groups walk rows that lie alike, as in the backward kernel, a thread's weights
// and biases in its slots beside the rows on their way. The CTAs that an SM
// holds, and the loads on their way with them, are the bound now.
template <typename T, int PACK, int G, int NP>
__global__ void __launch_bounds__(G ? 128 : 512) norm_fwd_walk_kernel(const FwdArgs a) {
    constexpr int W = G ? G : 1, kAhead = bwd_ahead(sizeof(T) * PACK * NP);
    typedef Pack<T, PACK> P;
    typedef Pack<float, PACK <= 4 ? PACK : 4> F;
    extern __shared__ __align__(128) unsigned char slots[];
    __shared__ float red[4][32];
    const int lane = G ? (int)(threadIdx.x % W) : (int)threadIdx.x;
    const int stride = G ? G : (int)blockDim.x;
    const int per = G ? (int)(blockDim.x / W) : 1;
    const int mine = G ? (int)(threadIdx.x / W) : 0;
    const long long step = (long long)gridDim.x * per;  // a multiple of 8
    long long base = (long long)blockIdx.x * per;
    const int skip = past_boundary<T, true>(static_cast<const T*>(a.x) +
                                            min(base + mine, a.rows - 1) * a.ldx);
    const auto col = [&](int i) { return (i * stride + lane) * PACK - skip; };
    P* const rows = reinterpret_cast<P*>(slots) + threadIdx.x;  // [kAhead][NP][threads]
    const auto slot = [&](int stage, int i) -> P* {
        return rows + (stage * NP + i) * (int)blockDim.x;
    };
    F* const weights = reinterpret_cast<F*>(reinterpret_cast<P*>(slots) +
                                            kAhead * NP * blockDim.x) + threadIdx.x;
    F* const biases = weights + NP * (PACK <= 4 ? 1 : PACK / 4) * blockDim.x;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        Pack<float, PACK> w, b;
        load_param<T, PACK, true>(a.w, a.wide, col(i), a.D, 1.0f, w.v);
        load_param<T, PACK, true>(a.b, a.wide, col(i), a.D, 0.0f, b.v);
        put_wide<PACK>(weights, i, w.v);
        put_wide<PACK>(biases, i, b.v);
    }
    const auto fetch = [&](long long row, int stage) {
        if (row < a.rows) {
            const T* x = static_cast<const T*>(a.x) + row * a.ldx;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int c = col(i);
                const long long at = row * a.ldx + c;
                // (partly a neighbouring row's, as in the backward kernel)
                if (c < a.D && at >= 0 && at + PACK <= (a.rows - 1) * a.ldx + a.D)
                    cp_async16(slot(stage, i), x + c, 16);
                else
                    *slot(stage, i) = load_cols<T, PACK, true>(x, c, a.D);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int k = 0; k < kAhead - 1; ++k) fetch(base + mine + k * step, k);
    int stage = 0;
    for (int buf = 0; base < a.rows; base += step, buf ^= 2) {
        const long long row = base + mine;
        const bool live = row < a.rows;
        fetch(row + (kAhead - 1) * step, stage == 0 ? kAhead - 1 : stage - 1);
        cp_async_wait_group<kAhead - 1>();
        float v[NP][PACK];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = col(i);
            P x;
            if (live) x = *slot(stage, i);
            const bool all = live && !sticks_out<PACK, G>(c, a.D);
#pragma unroll
            for (int j = 0; j < PACK; ++j) {
                v[i][j] = all || (live && c + j >= 0 && c + j < a.D) ? to_f(x.v[j]) : 0.0f;
                sum += v[i][j];
            }
        }
        stage = stage == kAhead - 1 ? 0 : stage + 1;
        const float mean = __fdiv_rn(row_sum<G>(sum, red[buf]), (float)a.D);
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = col(i);
            const bool all = !sticks_out<PACK, G>(c, a.D);
#pragma unroll
            for (int j = 0; j < PACK; ++j) {
                v[i][j] -= mean;
                sq = all || (c + j >= 0 && c + j < a.D) ? fmaf(v[i][j], v[i][j], sq) : sq;
            }
        }
        const float rstd =
            __frsqrt_rn(__fdiv_rn(row_sum<G>(sq, red[buf + 1]), (float)a.D) + a.eps);
        if (!live) continue;
        if (lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        T* y = static_cast<T*>(a.y) + row * a.D;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int c = col(i);
            if (c >= a.D) continue;
            Pack<float, PACK> w, b;
            get_wide<PACK>(weights, i, w.v);
            get_wide<PACK>(biases, i, b.v);
#pragma unroll
            for (int j = 0; j < PACK; ++j) v[i][j] = fmaf(v[i][j] * rstd, w.v[j], b.v[j]);
            store_cols<T, PACK, true>(y, c, a.D, v[i]);
        }
    }
}

// dx of rows of any width: two passes over the row, the second from cache.
template <typename T, int PACK, bool EDGE>
__global__ void __launch_bounds__(512) norm_dx_wide_kernel(const BwdArgs a) {
    __shared__ float2 red[32];
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const int skip = past_boundary<T, EDGE>(x), c0 = (int)threadIdx.x * PACK - skip;
    const int by = (int)blockDim.x * PACK;
    const float mean = a.mean[row], rstd = a.rstd[row], inv = __fdiv_rn(1.0f, (float)a.D);
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll 2
    for (int c = c0; c < a.D; c += by) {
        const Pack<T, PACK> p = load_cols<T, PACK, EDGE>(x, c, a.D);
        const Pack<T, PACK> g = load_cols<T, PACK, EDGE>(dy, c, a.D);
        float w[PACK];
        load_param<T, PACK, EDGE>(a.w, a.wide, c, a.D, 1.0f, w);
#pragma unroll
        for (int j = 0; j < PACK; ++j) {
            const float du = to_f(g.v[j]) * w[j];
            sum.x += du;
            sum.y = fmaf(du, (to_f(p.v[j]) - mean) * rstd, sum.y);
        }
    }
    sum = row_sums<0>(sum, red);
    const float s1 = sum.x * inv, s2 = sum.y * inv;
    T* dx = static_cast<T*>(a.dx) + row * a.D;
#pragma unroll 2
    for (int c = c0; c < a.D; c += by) {
        const Pack<T, PACK> p = load_cols<T, PACK, EDGE>(x, c, a.D);
        const Pack<T, PACK> g = load_cols<T, PACK, EDGE>(dy, c, a.D);
        float w[PACK], o[PACK];
        load_param<T, PACK, EDGE>(a.w, a.wide, c, a.D, 1.0f, w);
#pragma unroll
        for (int j = 0; j < PACK; ++j)
            o[j] = rstd * (to_f(g.v[j]) * w[j] - s1 - (to_f(p.v[j]) - mean) * rstd * s2);
        store_cols<T, PACK, EDGE>(dx, c, a.D, o);
    }
}

// Partial dw, db of any width: a lane's columns lie 32 apart, kColsWide to a
// CTA, the rows of slice blockIdx.y over its 8 warps.
constexpr int kColsWide = 128;

template <typename T>
__global__ void __launch_bounds__(256) norm_cols_wide_kernel(const BwdArgs a) {
    constexpr int N = kColsWide / 32;
    __shared__ float sums[2][8][kColsWide];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int c0 = blockIdx.x * kColsWide + lane;
    const long long lo = a.rows * blockIdx.y / gridDim.y, hi = a.rows * (blockIdx.y + 1) / gridDim.y;
    float aw[N] = {}, ab[N] = {};
#pragma unroll 4
    for (long long r = lo + w; r < hi; r += 8) {
        const T* dy = static_cast<const T*>(a.dy) + r * a.lddy;
        const T* x = static_cast<const T*>(a.x) + r * a.ldx;
        const float mean = a.mean[r], rstd = a.rstd[r];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int c = c0 + 32 * j;
            const float g = c < a.D ? to_f(dy[c]) : 0.0f;
            const float xh = c < a.D ? (to_f(x[c]) - mean) * rstd : 0.0f;
            aw[j] = fmaf(g, xh, aw[j]);
            ab[j] += g;
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        sums[0][w][lane + 32 * j] = aw[j];
        sums[1][w][lane + 32 * j] = ab[j];
    }
    __syncthreads();
    const int k = threadIdx.x / kColsWide, j = threadIdx.x % kColsWide;
    const int c = blockIdx.x * kColsWide + j;
    if (c < a.D) {
        float s = 0.0f;
        for (int i = 0; i < 8; ++i) s += sums[k][i][j];
        a.part[((size_t)k * gridDim.y + blockIdx.y) * a.D + c] = s;
    }
}

// out[c] = sum of P partial rows, in order within each of 32 slices, then the
// slices; blockIdx.y: 0 dw, 1 db. A few dozen CTAs: it takes as long as its
// chains of loads, so these are many and short.
template <typename W>
__global__ void __launch_bounds__(1024)
    norm_cols_kernel(const float* __restrict__ part, int P, int D, W* dw, W* db) {
    __shared__ float s[32][33];
    W* out = blockIdx.y ? db : dw;
    const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    const float* p = part + (size_t)blockIdx.y * P * D + c;
    pdl_wait();
    float v = 0.0f;
    if (out && c < D) {
#pragma unroll 16
        for (int r = k; r < P; r += 32) v += p[(size_t)r * D];
    }
    s[k][lane] = v;
    __syncthreads();
    v = s[lane][k];  // column k of these, its slices over the lanes
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0 && out && blockIdx.x * 32 + k < D) out[blockIdx.x * 32 + k] = from_f<W>(v);
}

// How a row is laid over threads: G lanes of a warp (0: a CTA of `threads`),
// NP packs of PACK elements each. G == -1: no register form holds it.
struct Form {
    int G, NP, threads;
};

int round32(int v) { return (v + 31) / 32 * 32; }

// A warp holds `warp_most` elements a lane at most, a thread of a CTA
// `cta_most`, a CTA has 128 to 512 threads. A row in one warp needs no barrier
// between its loads and its stores, so warps come first, with as many elements
// as leave registers for some 16 warps on an SM; the CTA forms take the most
// packs that still give 128 threads, for more rows in flight.
Form pick(int packs, int pack, int warp_most, int cta_most) {
    if (pack > 1)
        for (int g = 4; g < 32; g *= 2)
            if (packs <= g) return {g, 1, 0};
    for (int n : {1, 2, 3, 4, 6, 8, 12, 16, 32})
        if (n * pack <= warp_most && packs <= n * 32) return {32, n, 0};
    for (int n : {32, 16, 8, 4, 2, 1})
        if (n * pack <= cta_most && (packs + n - 1) / n > 96 && round32((packs + n - 1) / n) <= 512)
            return {0, n, round32((packs + n - 1) / n)};
    return {-1, 0, 0};
}

// Packs of a row, one more where it may begin within one.
int packs_of(int D, int pack, bool edge) { return (D + (edge ? pack - 1 : 0) + pack - 1) / pack; }

// CTAs of a kernel that an SM holds, asked once for each size of CTA.
template <typename K>
int resident(K kern, int threads, size_t dyn, std::atomic<int>* known) {
    int held = known[threads / 32].load(std::memory_order_relaxed);
    if (!held) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kern, threads, dyn) != cudaSuccess)
            cudaGetLastError();
        held = held < 1 ? 1 : held;
        known[threads / 32].store(held, std::memory_order_relaxed);
    }
    return held;
}

template <typename K>
int allow_smem(K kern, size_t dyn, const char* what) {
    if (dyn <= 40 * 1024) return SN_OK;
    return cuda_check(
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)dyn), what);
}

template <typename T, int PACK, int G, int NP, bool EDGE>
int fwd_launch(const FwdArgs& a, int threads, int sms, cudaStream_t st) {
    if constexpr (EDGE && sizeof(T) == 2) {
        // With eight rows for each group of an SM. 16-bit, before and now: 4000
        // x 5003 62 and 30 us, 40000 x 601 68 and 45, 8192 x 2047 50 and 35; 600
        // rows of 4001, four for each, 9.7 and 10.4. In fp32, where twice the
        // packs carry the same loads of weights, 3000 x 8190 goes from 52 to 58
        // us and the others stay within 2 us.
        static std::atomic<int> known[17];
        const auto kern = norm_fwd_walk_kernel<T, PACK, G, NP>;
        const int n = G ? 128 : threads, per = G ? n / (G ? G : 1) : 1;
        const size_t dyn =
            (size_t)n * NP * PACK * (bwd_ahead(sizeof(T) * PACK * NP) * sizeof(T) + 8);
        if ((a.w || a.b) && dyn <= 200 * 1024 && a.rows >= 8ll * sms * per) {
            SN_TRY(allow_smem(kern, dyn, "layer_norm"));
            const long long cap = (long long)sms * resident(kern, n, dyn, known) / 8 * 8;
            const long long want = (a.rows / 3 + per - 1) / per;
            const long long ctas = want < cap ? (want + 7) / 8 * 8 : cap;
            kern<<<(unsigned)ctas, n, dyn, st>>>(a);
            return cuda_check(cudaGetLastError(), "layer_norm launch");
        }
    }
    const int per = G ? 128 / (G ? G : 1) : 1;
    const long long blocks = (a.rows + per - 1) / per;
    norm_fwd_kernel<T, PACK, G, NP, EDGE><<<(unsigned)blocks, G ? 128 : threads, 0, st>>>(a);
    return cuda_check(cudaGetLastError(), "layer_norm launch");
}

template <typename T, int PACK, bool EDGE>
int fwd_dispatch(const FwdArgs& a, int sms, cudaStream_t st) {
    // 48 elements a lane: 1536 fp32 columns in one warp; single elements are
    // the rare case of rows that share no boundary with their outputs
    const Form f = pick(packs_of(a.D, PACK, EDGE), PACK, PACK == 1 ? 32 : 48, 32);
#define SN_FWD(g, n) \
    if (f.G == g && f.NP == n) return fwd_launch<T, PACK, g, n, EDGE>(a, f.threads, sms, st)
    if constexpr (PACK > 1) {
        SN_FWD(4, 1);
        SN_FWD(8, 1);
        SN_FWD(16, 1);
    }
    SN_FWD(32, 1);
    SN_FWD(32, 2);
    SN_FWD(32, 3);
    SN_FWD(32, 4);
    SN_FWD(32, 6);
    if constexpr (PACK <= 4) {
        SN_FWD(32, 8);
        SN_FWD(32, 12);
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
    norm_fwd_wide_kernel<T, PACK, EDGE><<<(unsigned)a.rows, 512, 0, st>>>(a);
    return cuda_check(cudaGetLastError(), "layer_norm launch");
}

// How rows may be moved: in packs that begin where the rows do, in packs of
// memory, or one element at a time.
enum Move { kWhole, kEdge, kSingle };

template <typename T>
int fwd_typed(const FwdArgs& a, Move move, int sms, cudaStream_t st) {
    constexpr int P = 16 / sizeof(T);
    return move == kWhole  ? fwd_dispatch<T, P, false>(a, sms, st)
           : move == kEdge ? fwd_dispatch<T, P, true>(a, sms, st)
                           : fwd_dispatch<T, 1, false>(a, sms, st);
}

// Launches the backward kernel; a == nullptr: the CTAs of it that an SM holds.
template <typename T, int PACK, int G, int NP, bool EDGE>
int bwd_launch(const BwdArgs* a, int threads, int parts, cudaStream_t st) {
    static std::atomic<int> known[17];  // by warps of a CTA
    const auto kern = norm_bwd_kernel<T, PACK, G, NP, EDGE>;
    const int n = G ? bwd_threads(PACK * NP) : threads;
    const size_t dyn = (size_t)n * bwd_slot_bytes(sizeof(T), PACK * NP);
    SN_TRY(allow_smem(kern, dyn, "layer_norm_bwd"));
    if (!a) return resident(kern, n, dyn, known);
    kern<<<parts, n, dyn, st>>>(*a);
    return cuda_check(cudaGetLastError(), "layer_norm_bwd launch");
}

template <typename T, int PACK, bool EDGE>
int bwd_dispatch(const BwdArgs* a, const Form& f, int parts, cudaStream_t st) {
#define SN_BWD(g, n) \
    if (f.G == g && f.NP == n) return bwd_launch<T, PACK, g, n, EDGE>(a, f.threads, parts, st)
    if constexpr (PACK > 1) {
        SN_BWD(4, 1);
        SN_BWD(8, 1);
        SN_BWD(16, 1);
    }
    SN_BWD(32, 1);
    SN_BWD(32, 2);
    SN_BWD(32, 3);
    SN_BWD(32, 4);
    if constexpr (PACK <= 4) {
        SN_BWD(32, 6);
        SN_BWD(32, 8);
        SN_BWD(0, 4);
    }
    if constexpr (PACK == 1) {
        SN_BWD(32, 12);
        SN_BWD(32, 16);
        SN_BWD(0, 8);
        SN_BWD(0, 16);
    }
    SN_BWD(0, 1);
    SN_BWD(0, 2);
#undef SN_BWD
    if (!a) return 1;
    if (a->dx) norm_dx_wide_kernel<T, PACK, EDGE><<<(unsigned)a->rows, 512, 0, st>>>(*a);
    SN_TRY(cuda_check(cudaGetLastError(), "layer_norm_bwd launch"));
    if (a->part)
        norm_cols_wide_kernel<T>
            <<<dim3((a->D + kColsWide - 1) / kColsWide, parts), 256, 0, st>>>(*a);
    return cuda_check(cudaGetLastError(), "layer_norm_bwd launch");
}

template <typename T>
int bwd_moved(const BwdArgs* a, const Form& f, Move move, int parts, cudaStream_t st) {
    constexpr int P = 16 / sizeof(T);
    return move == kWhole  ? bwd_dispatch<T, P, false>(a, f, parts, st)
           : move == kEdge ? bwd_dispatch<T, P, true>(a, f, parts, st)
                           : bwd_dispatch<T, 1, false>(a, f, parts, st);
}

int bwd_any(const BwdArgs* a, const Form& f, Move move, int dtype, int parts, cudaStream_t st) {
    switch (dtype) {
        case SN_F32: return bwd_moved<float>(a, f, move, parts, st);
        case SN_BF16: return bwd_moved<__nv_bfloat16>(a, f, move, parts, st);
        default: return bwd_moved<__half>(a, f, move, parts, st);
    }
}

Form bwd_form(int D, Move move, int dtype) {
    const int pack = move == kSingle ? 1 : 16 / (int)dtype_size(dtype);
    return pick(packs_of(D, pack, move == kEdge), pack, pack == 1 ? 16 : 32, 16);
}

// CTAs of the backward kernel, which are the rows of the partial sums: as many
// as the SMs hold; a multiple of 8 where the rows are moved in packs of memory.
int bwd_parts(long long rows, int D, Move move, int dtype, int sms) {
    const Form f = bwd_form(D, move, dtype);
    long long want, cap;
    if (f.G < 0) {  // slices of norm_cols_wide_kernel
        const int cols = (D + kColsWide - 1) / kColsWide;
        want = (rows + 63) / 64;
        cap = (8ll * sms + cols - 1) / cols;
    } else {
        // a CTA's partial sums are worth two of its rows: four rows to a group,
        // as far as that leaves every SM a CTA
        const int pack = move == kSingle ? 1 : 16 / (int)dtype_size(dtype);
        const int per = f.G ? bwd_threads(f.NP * pack) / f.G : 1;
        want = (rows + per - 1) / per;
        want = want / 4 > sms ? want / 4 : want < sms ? want : sms;
        const int held = bwd_any(nullptr, f, move, dtype, 0, nullptr);
        cap = (long long)sms * (held < 1 ? 1 : held);
    }
    long long p = want < cap ? want : cap;
    if (move == kEdge && f.G >= 0) p = (p + 7) / 8 * 8;
    return (int)(p < 1 ? 1 : p);
}

template <typename W>
int cols_launch(const float* part, int parts, int D, void* dw, void* db, cudaStream_t st) {
    return cuda_check(launch_pdl(norm_cols_kernel<W>, dim3((D + 31) / 32, 2), dim3(1024), 0, st,
                                 part, parts, D, static_cast<W*>(dw), static_cast<W*>(db)),
                      "layer_norm_bwd launch");
}

// Two arrays of rows whose rows lie alike in 16-byte units.
bool alike(const void* p, long long ldp, const void* q, long long ldq, unsigned size) {
    return ((uintptr_t)p - (uintptr_t)q) % 16 == 0 && (ldp - ldq) * (long long)size % 16 == 0;
}

bool whole16(const void* p, long long ld, unsigned size) {
    return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0;
}

// The widest row: the wide kernels count columns in 32 bits, up to four steps of
// 512 packs beyond the row's end.
constexpr int kMaxWidth = 0x7fffffff - 0x4000 + 1;

bool shape_ok(long long rows, int D, long long ld) {
    return rows >= 0 && rows < (1ll << 31) && D > 0 && D <= kMaxWidth && ld >= D;
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
    const bool like = alike(x, ldx, y, D, size);
    const Move move = like && whole16(x, ldx, size) && D % (16 / size) == 0 &&
                              (!w || whole16(w, 0, ws)) && (!b || whole16(b, 0, ws))
                          ? kWhole
                      : like ? kEdge
                             : kSingle;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    switch (dtype) {
        case SN_F32: return fwd_typed<float>(a, move, dev.num_sms(), st);
        case SN_BF16: return fwd_typed<__nv_bfloat16>(a, move, dev.num_sms(), st);
        default: return fwd_typed<__half>(a, move, dev.num_sms(), st);
    }
}

int64_t sn_abi_layer_norm_bwd_ws(int64_t rows, int32_t D, int32_t dtype) {
    const unsigned size = dtype_size(dtype);
    if (!size || !shape_ok(rows, D, D)) return 0;
    CallerDevice dev;
    const int sms = dev.select("layer_norm_bwd_ws") == SN_OK ? dev.num_sms() : 148;
    int parts = 0;  // the most that any addresses lead to
    for (Move move : {kWhole, kEdge, kSingle}) {
        const int p = bwd_parts(rows, D, move, dtype, sms);
        parts = p > parts ? p : parts;
    }
    return 8ll * parts * D;
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
    const bool like = alike(x, ldx, dy, lddy, size) && (!dx || alike(x, ldx, dx, D, size));
    const Move move = like && whole16(x, ldx, size) && D % (16 / size) == 0 &&
                              (!w || whole16(w, 0, wsz))
                          ? kWhole
                      : like ? kEdge
                             : kSingle;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const int parts = rows ? bwd_parts(rows, D, move, dtype, dev.num_sms()) : 0;
    if (rows && (dx || sums))
        SN_TRY(bwd_any(&a, bwd_form(D, move, dtype), move, dtype, parts, st));
    if (!sums) return SN_OK;
    switch (wdtype) {
        case SN_F32: return cols_launch<float>(a.part, parts, D, dw, db, st);
        case SN_BF16: return cols_launch<__nv_bfloat16>(a.part, parts, D, dw, db, st);
        default: return cols_launch<__half>(a.part, parts, D, dw, db, st);
    }
}

}  // extern "C"
