// Pieces of the linear-attention kernels: tiles of tokens in shared memory as
// one to three bf16 planes, their matrix fragments, and the decays of a chunk.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "caller.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace sn {
namespace la {

typedef __nv_bfloat16 bf16;

// Planes a type's values take: bf16 is one itself, float16 the sum of two, float32
// of three; nothing is lost (but that fp32 values from 3.396e38 on, the last 512th of
// the range, round to infinity in their first part).
template <typename T>
constexpr int planes_of = std::is_same<T, bf16>::value ? 1 : std::is_same<T, float>::value ? 3 : 2;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x) {
    if constexpr (std::is_same<T, float>::value)
        return x;
    else if constexpr (std::is_same<T, bf16>::value)
        return __float2bfloat16_rn(x);
    else
        return __float2half_rn(x);
}

// Two floats as bf16, the first in the low half.
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ float low(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void mma(float* c, const uint32_t* a, const uint32_t* b) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

__device__ __forceinline__ void stsm4(uint32_t at, const uint32_t* r) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3])
                 : "memory");
}

// P planes of a pair of values, the first in the low halves.
template <int P>
__device__ __forceinline__ void split2(float u, float v, uint32_t (*to)[4], int r) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
        to[p][r] = pack2(u, v);
        if (p + 1 < P) u -= low(to[p][r]), v -= high(to[p][r]);
    }
}

// The product of A (PA planes) and B (PB planes) into two neighbouring column
// tiles of eight. Planes i and j are 2^-8(i + j) of the whole: those products are
// left out that fp32 (three planes on either side), or a 16-bit result, does not
// hold.
template <int PA, int PB, int LIM = (PA > PB ? PA : PB)>
__device__ __forceinline__ void mma2(float (*c)[4], const uint32_t (*a)[4], const uint32_t (*b)[4]) {
#pragma unroll
    for (int i = PA - 1; i >= 0; --i)  // the small ones first
#pragma unroll
        for (int j = PB - 1; j >= 0; --j)
            if (i + j < LIM) {
                mma(c[0], a[i], b[j]);
                mma(c[1], a[i], b[j] + 2);
            }
}

// The same with the products of the first parts in `c` and the others in `rest`,
// which the caller adds to it: a matrix instruction cuts its sums off, and six of
// them into one sum lean by as many times 2^-24.
template <int PA, int PB, int LIM>
__device__ __forceinline__ void mma2(float (*c)[4], float (*rest)[4], const uint32_t (*a)[4],
                                     const uint32_t (*b)[4]) {
#pragma unroll
    for (int i = PA - 1; i >= 0; --i)
#pragma unroll
        for (int j = PB - 1; j >= 0; --j)
            if (i + j < LIM) {
                mma(i + j ? rest[0] : c[0], a[i], b[j]);
                mma(i + j ? rest[1] : c[1], a[i], b[j] + 2);
            }
}

// A tile in shared memory: rows of LD bf16 (8 more than their D values, so that
// the eight rows that ldmatrix reads at once lie in different banks), its
// planes `step` values apart. The four ways a 16 x 16 block of it is read, at
// (row, col):
struct Tile {
    uint32_t at;    // shared-memory address
    uint32_t ld;    // bytes from one row to the next
    uint32_t step;  // bytes from one plane to the next
    // A(m, k) = tile[row + m][col + k]
    __device__ __forceinline__ void a(uint32_t* r, int row, int col, int plane) const {
        const int l = lane_id();
        ldsm4(r, at + plane * step + (row + (l & 15)) * ld + (col + (l >> 4) * 8) * 2);
    }
    // A(m, k) = tile[row + k][col + m]
    __device__ __forceinline__ void a_t(uint32_t* r, int row, int col, int plane) const {
        const int l = lane_id();
        ldsm4t(r, at + plane * step + (row + (l & 7) + (l >> 4) * 8) * ld + (col + (l >> 3 & 1) * 8) * 2);
    }
    // B(k, n) = tile[row + n][col + k], n of two column tiles
    __device__ __forceinline__ void b(uint32_t* r, int row, int col, int plane) const {
        const int l = lane_id();
        ldsm4(r, at + plane * step + (row + (l & 7) + (l >> 4) * 8) * ld + (col + (l >> 3 & 1) * 8) * 2);
    }
    // B(k, n) = tile[row + k][col + n]
    __device__ __forceinline__ void b_t(uint32_t* r, int row, int col, int plane) const {
        const int l = lane_id();
        ldsm4t(r, at + plane * step + (row + (l & 15)) * ld + (col + (l >> 4) * 8) * 2);
    }
};

// A tile of tokens on its way to shared memory: [t0, t0 + C) of one head, `d`
// values each (D with zeros behind them), `stride` values from one token to the
// next; tokens from `end` on are zeros, whatever lies there. `whole`: base and
// stride are multiples of 16 bytes (of 8 for float16) and d fills whole packs.
// fetch() asks for the values and put() brings them, between which the caller may
// work; bf16 goes by cp.async in fetch(), for which the caller waits instead.
template <typename T, int C, int D, int THREADS>
struct Fetch {
    static constexpr bool DIRECT = std::is_same<T, bf16>::value;
    static constexpr int W = DIRECT ? 8 : 4;  // values of a pack
    static constexpr int N = C * D / W / THREADS, LD = D + 8, PLANE = C * LD;
    static_assert(C * D / W % THREADS == 0, "whole rounds of packs");
    typedef typename std::conditional<sizeof(T) == 4, float4, uint2>::type Raw;
    Raw raw[DIRECT ? 1 : N];

    // Packs of a row are the work of neighbouring threads; a thread's rows lie ROWS apart.
    static constexpr int PER_ROW = D / W, ROWS = THREADS / PER_ROW;
    static_assert(THREADS % PER_ROW == 0, "whole rows for the threads");

    __device__ __forceinline__ void fetch(bf16* dst, const T* src, long long stride, int t0, int end, int d,
                                          bool whole) {
        if (whole) {
            const int row = threadIdx.x / PER_ROW, col = threadIdx.x % PER_ROW * W;
            const int rows = col < d ? end - t0 - row : 0;  // of the thread's that hold values
            const T* from = src + (long long)(t0 + row) * stride + col;
            bf16* to = dst + row * LD + col;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const bool in = n * ROWS < rows;
                if constexpr (DIRECT)
                    cp_async16(to + n * ROWS * LD, in ? from : src, in ? 16 : 0);
                else
                    raw[n] = in ? *reinterpret_cast<const Raw*>(from) : Raw();
                from += ROWS * stride;
            }
        } else if constexpr (DIRECT) {
            for (int i = threadIdx.x; i < C * D; i += THREADS) {
                const int row = i / D, col = i % D;
                dst[row * LD + col] = t0 + row < end && col < d ? src[(long long)(t0 + row) * stride + col]
                                                                : __float2bfloat16_rn(0.0f);
            }
        }
    }

    __device__ __forceinline__ void put(bf16* dst, const T* src, long long stride, int t0, int end, int d,
                                        bool whole) {
        if constexpr (!DIRECT) {
            if (whole) {
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int i = n * THREADS + threadIdx.x, row = i / (D / W), col = i % (D / W) * W;
                    bf16* to = dst + row * LD + col;
                    float x[4];
                    if constexpr (sizeof(T) == 4) {
                        x[0] = raw[n].x, x[1] = raw[n].y, x[2] = raw[n].z, x[3] = raw[n].w;
                    } else {
                        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw[n].x));
                        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&raw[n].y));
                        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
                    }
#pragma unroll
                    for (int p = 0; p < planes_of<T>; ++p) {
                        const uint2 part = {pack2(x[0], x[1]), pack2(x[2], x[3])};
                        *reinterpret_cast<uint2*>(to + p * PLANE) = part;
                        x[0] -= low(part.x), x[1] -= high(part.x), x[2] -= low(part.y), x[3] -= high(part.y);
                    }
                }
            } else {
                for (int i = threadIdx.x; i < C * D; i += THREADS) {
                    const int row = i / D, col = i % D;
                    const bool in = t0 + row < end && col < d;
                    float x = in ? to_f(src[(long long)(t0 + row) * stride + col]) : 0.0f;
#pragma unroll
                    for (int p = 0; p < planes_of<T>; ++p) {
                        const bf16 part = __float2bfloat16_rn(x);
                        dst[p * PLANE + row * LD + col] = part;
                        x -= __bfloat162float(part);
                    }
                }
            }
        }
    }
};

// The sums c of a chunk's log decays in powers of two, up to and with each
// token. near + far is c to 2^-28: near a multiple of 1/16, so that near_t -
// near_s is exact and the decay between two tokens as good as their
// difference, however far both are from the chunk's start.
template <int C>
struct alignas(16) Decays {
    float near[C], far[C];
    float from_start[C];  // 2^c_t
    float to_end[C];      // 2^(c_C - c_t)
    float whole;          // 2^c_C
    float unused[3];
    // 2^(c_t - c_s)
    __device__ __forceinline__ float between(int t, int s) const;
};

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int C>
__device__ __forceinline__ float Decays<C>::between(int t, int s) const {
    return exp2_of(near[t] - near[s] + (far[t] - far[s]));
}

// By one whole warp, from a lane's C / 32 log decays (zeros behind the end), in
// the tokens' order. The sums are whole numbers of 2^-40: no rounding, and half
// the latency of fp64. A log decay beyond 256 (in powers of two) either way leaves
// nothing, or no finite number, in 32 bits: it is taken as 256, infinities too. A
// NaN makes every sum from its token on one.
template <int C>
__device__ __forceinline__ void decays(Decays<C>* to, const float* g) {
    constexpr int N = C / 32;
    constexpr float kLog2e = 1.44269504088896340736f, kRest = 1.92596299e-8f;  // their sum is log2(e) to 2^-50
    const int l = lane_id();
    long long c[N], sum = 0;
    int bad = N;  // the lane's first NaN
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (bad == N && g[i] != g[i]) bad = i;
        const float x = fminf(fmaxf(g[i], -178.0f), 178.0f);
        const float hi = x * kLog2e, lo = fmaf(x, kLog2e, -hi) + x * kRest;
        c[i] = sum += __float2ll_rn(hi * 0x1p40f) + __float2ll_rn(lo * 0x1p40f);
    }
    const unsigned wrong = __ballot_sync(0xffffffffu, bad < N);
    const int first = wrong ? __ffs(wrong) - 1 : 32;  // the lane of the first NaN
    long long before = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const long long y = __shfl_up_sync(0xffffffffu, before, d);
        if (l >= d) before += y;
    }
    const long long all = __shfl_sync(0xffffffffu, before, 31);
    before -= sum;
    const float nan = __int_as_float(0x7fffffff);
    const auto value = [](long long x) {  // (the high part is exact)
        const int whole = (int)(x >> 36);
        return make_float2((float)whole * 0.0625f, (float)(x - ((long long)whole << 36)) * 0x1p-40f);
    };
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool poor = l > first || (l == first && i >= bad);
        const float2 x = value(before + c[i]), y = value(all - before - c[i]);
        to->near[l * N + i] = poor ? nan : x.x;
        to->far[l * N + i] = x.y;
        to->from_start[l * N + i] = poor ? nan : exp2_of(x.x + x.y);
        to->to_end[l * N + i] = wrong ? nan : exp2_of(y.x + y.y);
    }
    if (l == 0) {
        const float2 x = value(all);
        to->whole = wrong ? nan : exp2_of(x.x + x.y);
    }
}

struct Strides {
    long long b, t, h;
};

// A call's sizes and arrays.
struct Job {
    const void *q, *k, *v;
    Strides qs, ks, vs, gs;
    const float* g;
    const int* lengths;
    int B, T, H, share, dk, dv;
    float scale;
    int whole;  // bit 0: q, 1: k, 2: v, 3: dout come in whole packs
    int chunks;  // of a sequence
    bool apart;  // each chunk's sum by a CTA of its own
};

// The gradients that a call wants, and those it is given.
struct Wanted {
    const void* dout;
    Strides ds;
    const float* dstate_out;
    void *dq, *dk, *dv;
    float *dg, *dstate;
    bool gates_alike;
};

// The launches of a call (linattn_kernels.cuh); with `need`, the bytes of workspace
// alone.
template <typename T>
int forward(const Job& j, const float* first, void* out, float* state_out, char* ws, long long ws_bytes,
            long long* need, cudaStream_t st);
template <typename T>
int backward(const Job& j, const float* first, const Wanted& w, char* ws, long long ws_bytes, long long* need,
             cudaStream_t st);

}  // namespace la
}  // namespace sn
