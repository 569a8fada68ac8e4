// Pieces of the linear-attention kernels: tiles of tokens in shared memory as
// one or two bf16 planes, their matrix fragments, and the decays of a chunk.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "ptx.cuh"

namespace sn {
namespace la {

typedef __nv_bfloat16 bf16;

// Planes a type's values take: bf16 is one itself; float16 (exactly) and
// float32 (to 2^-17 of the value) are the sum of two.
template <typename T>
constexpr int planes_of = std::is_same<T, bf16>::value ? 1 : 2;

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
// What two values have beyond their bf16 halves.
__device__ __forceinline__ uint32_t rest2(float a, float b, uint32_t hi) {
    return pack2(a - low(hi), b - high(hi));
}

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
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

// The product of A (PA planes) and B (PB planes) into two neighbouring column
// tiles of eight: all pairs of planes but the two low ones.
template <int PA, int PB>
__device__ __forceinline__ void mma2(float (*c)[4], const uint32_t (*a)[4], const uint32_t (*b)[4]) {
#pragma unroll
    for (int i = 0; i < PA; ++i)
#pragma unroll
        for (int j = 0; j < PB; ++j)
            if (i + j < 2) {
                mma(c[0], a[i], b[j]);
                mma(c[1], a[i], b[j] + 2);
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

// Tokens [t0, t0 + C) of one head, `d` values each (D with zeros behind them),
// `stride` values from one token to the next; tokens from `end` on are zeros,
// whatever lies there. `whole`: base and stride are multiples of 16 bytes (of 8
// for float16) and d fills whole packs. bf16 goes by cp.async: the caller waits.
template <typename T, int C, int D, int THREADS>
__device__ __forceinline__ void load_tokens(bf16* dst, const T* src, long long stride, int t0, int end,
                                            int d, bool whole) {
    constexpr int LD = D + 8, PLANE = C * LD;
    if (whole) {
        constexpr int W = std::is_same<T, bf16>::value ? 8 : 4;  // values of a pack
        constexpr int PACKS = C * D / W;
#pragma unroll
        for (int n = 0; n < PACKS / THREADS; ++n) {
            const int i = n * THREADS + threadIdx.x, row = i / (D / W), col = i % (D / W) * W;
            const bool in = t0 + row < end && col < d;
            const T* from = src + (in ? (long long)(t0 + row) * stride + col : 0);
            bf16* to = dst + row * LD + col;
            if constexpr (std::is_same<T, bf16>::value) {
                cp_async16(to, from, in ? 16 : 0);
            } else {
                float x[4] = {};
                if (in) {
                    if constexpr (std::is_same<T, float>::value) {
                        const float4 f = *reinterpret_cast<const float4*>(from);
                        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
                    } else {
                        const uint2 f = *reinterpret_cast<const uint2*>(from);
                        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&f.x));
                        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&f.y));
                        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
                    }
                }
                const uint2 hi = {pack2(x[0], x[1]), pack2(x[2], x[3])};
                const uint2 lo = {rest2(x[0], x[1], hi.x), rest2(x[2], x[3], hi.y)};
                *reinterpret_cast<uint2*>(to) = hi;
                *reinterpret_cast<uint2*>(to + PLANE) = lo;
            }
        }
    } else {
        for (int i = threadIdx.x; i < C * D; i += THREADS) {
            const int row = i / D, col = i % D;
            const bool in = t0 + row < end && col < d;
            const float x = in ? to_f(src[(long long)(t0 + row) * stride + col]) : 0.0f;
            const bf16 hi = __float2bfloat16_rn(x);
            dst[row * LD + col] = hi;
            if constexpr (planes_of<T> == 2)
                dst[PLANE + row * LD + col] = __float2bfloat16_rn(x - __bfloat162float(hi));
        }
    }
}

// The sums c of a chunk's log decays in powers of two, up to and with each
// token. near + far is c to 2^-29: near a multiple of 1/16, so that near_t -
// near_s is exact and the decay between two tokens as good as their
// difference, however far both are from the chunk's start.
template <int C>
struct alignas(16) Decays {
    float near[C], far[C];
    float from_start[C];  // 2^c_t
    float to_end[C];      // 2^(c_C - c_t)
    float whole;          // 2^c_C
};

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// By one whole warp. A log decay below -256 (in powers of two) leaves nothing
// in 32 bits, however long the chunk: it is taken as -256, minus infinity too.
template <int C>
__device__ __forceinline__ void decays(Decays<C>* to, const float* g, long long stride, int t0, int end) {
    constexpr int N = C / 32;
    const int l = lane_id();
    double c[N], sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int t = t0 + l * N + i;
        double x = t < end ? (double)g[(long long)t * stride] * 1.4426950408889634074 : 0.0;
        if (x < -256.0) x = -256.0;  // (a NaN stays)
        c[i] = sum += x;
    }
    double before = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const double y = __shfl_up_sync(0xffffffffu, before, d);
        if (l >= d) before += y;
    }
    const double all = __shfl_sync(0xffffffffu, before, 31);
    before -= sum;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const double x = before + c[i];
        const float near = rintf((float)x * 16.0f) * 0.0625f;
        to->near[l * N + i] = near;
        to->far[l * N + i] = (float)(x - (double)near);
        to->from_start[l * N + i] = exp2_of((float)x);
        to->to_end[l * N + i] = exp2_of((float)(all - x));
    }
    if (l == 0) to->whole = exp2_of((float)all);
}

}  // namespace la
}  // namespace sn
