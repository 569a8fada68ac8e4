// The kernels of linear attention, for one type of values (included by a source
// file for each, which are compiled side by side).
#pragma once
#include <algorithm>
#include <cmath>

#include "linattn.cuh"

namespace sn {
namespace la {
namespace {

// Tokens of a sequence.
__device__ __forceinline__ int tokens_of(const Job& j, int b) {
    return j.lengths ? max(0, min(j.T, j.lengths[b])) : j.T;
}

template <typename T>
__device__ __forceinline__ const T* head_of(const void* x, const Strides& s, int b, int h) {
    return static_cast<const T*>(x) + b * s.b + h * s.h;
}

template <int NT>
__device__ __forceinline__ void clear(float (*x)[4]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = 0.0f;
}

// S += sum over the tokens of scale w_t x_t y_t^T: 16 rows (values `row` on of x),
// NT column tiles (values `cb` on of y). x w in fp32, in three planes: what comes of
// it is an fp32 result. (The planes of a bf16 x formed by packed bf16 instructions,
// four in place of three, are a third of the work, but the fourth product of each made
// the whole 8% slower.) The chunk has `tokens`; a block of 16 with none is left out.
template <int NP, int NT, int C>
__device__ __forceinline__ void add_outer(float (*S)[4], const Tile& x, const Tile& y, const float* w,
                                          float scale, int row, int cb, int tokens) {
    const int q = lane_id() & 3;
    const auto block = [&](int kt) {
        uint32_t xr[NP][4], a[3][4];
#pragma unroll
        for (int p = 0; p < NP; ++p) x.a_t(xr[p], kt * 16, row, p);
        float2 f[2];
        f[0] = *reinterpret_cast<const float2*>(w + kt * 16 + 2 * q);
        f[1] = *reinterpret_cast<const float2*>(w + kt * 16 + 2 * q + 8);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float u = low(xr[NP - 1][r]), v = high(xr[NP - 1][r]);
#pragma unroll
            for (int p = NP - 2; p >= 0; --p) u += low(xr[p][r]), v += high(xr[p][r]);
            split2<3>(u * (f[r / 2].x * scale), v * (f[r / 2].y * scale), a, r);
        }
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
            uint32_t b[NP][4];
#pragma unroll
            for (int p = 0; p < NP; ++p) y.b_t(b[p], kt * 16, cb + n * 16, p);
            mma2<3, NP>(S + 2 * n, a, b);
        }
    };
    if (tokens > C - 16) {
#pragma unroll
        for (int kt = 0; kt < C / 16; ++kt) block(kt);
    } else {
#pragma unroll 1
        for (int kt = 0; kt * 16 < tokens; ++kt) block(kt);
    }
}

// A second sum for the products of later parts, where fp32 results count on them:
// add() puts it into the first.
template <int NP, int NT>
struct Rest {
    static constexpr bool ON = NP == 3;
    float x[ON ? NT : 1][4];
    __device__ __forceinline__ Rest() {
        if constexpr (ON) clear<NT>(x);
    }
    template <int PA, int PB, int LIM>
    __device__ __forceinline__ void mma(float (*c)[4], int n, const uint32_t (*a)[4], const uint32_t (*b)[4]) {
        if constexpr (ON)
            mma2<PA, PB, LIM>(c + n, x + n, a, b);
        else
            mma2<PA, PB, LIM>(c + n, a, b);
    }
    __device__ __forceinline__ void add(float (*c)[4]) const {
        if constexpr (ON) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) c[n][i] += x[n][i];
        }
    }
};

// out (16 rows from `ra` of A, columns from `cb` of B) += A B over D: A's rows
// are tokens, B(k, n) = tile[n][k], or tile[k][n] where TRANS.
template <int PA, int PB, int D, int NT, bool TRANS>
__device__ __forceinline__ void product(float (*out)[4], const Tile& A, int ra, const Tile& B, int cb) {
    Rest<PA, NT> rest;
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
        uint32_t a[PA][4];
#pragma unroll
        for (int p = 0; p < PA; ++p) A.a(a[p], ra, kt * 16, p);
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
            uint32_t b[PB][4];
#pragma unroll
            for (int p = 0; p < PB; ++p) {
                if constexpr (TRANS)
                    B.b_t(b[p], kt * 16, cb + n * 16, p);
                else
                    B.b(b[p], cb + n * 16, kt * 16, p);
            }
            rest.template mma<PA, PB, (PA > PB ? PA : PB)>(out, 2 * n, a, b);
        }
    }
    rest.add(out);
}

// Scores of 16 tokens of A with a strip of NB blocks of 16 tokens of B from
// block `jb` on, of which [j0, j1) are wanted.
template <int NP, int D, int NB, int LIM = NP>
__device__ __forceinline__ void scores(float (*p)[4], const Tile& A, int ra, const Tile& B, int jb, int j0,
                                       int j1) {
    clear<2 * NB>(p);
    Rest<NP, 2 * NB> rest;
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
        uint32_t a[NP][4];
#pragma unroll
        for (int i = 0; i < NP; ++i) A.a(a[i], ra, kt * 16, i);
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (jb + j >= j0 && jb + j < j1) {
                uint32_t b[NP][4];
#pragma unroll
                for (int i = 0; i < NP; ++i) B.b(b[i], (jb + j) * 16, kt * 16, i);
                rest.template mma<NP, NP, LIM>(p, 2 * j, a, b);
            }
    }
    rest.add(p);
}

// out += P Y, P such scores as they lie in registers (PP planes of them), Y the
// tokens' tile.
template <int PP, int NP, int NB, int NT>
__device__ __forceinline__ void weighted(float (*out)[4], const float (*p)[4], const Tile& Y, int cb, int jb,
                                         int j0, int j1) {
    Rest<PP, NT> rest;
#pragma unroll
    for (int j = 0; j < NB; ++j)
        if (jb + j >= j0 && jb + j < j1) {
            uint32_t a[PP][4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
                split2<PP>(p[2 * j + r / 2][r % 2 * 2], p[2 * j + r / 2][r % 2 * 2 + 1], a, r);
#pragma unroll
            for (int n = 0; n < NT / 2; ++n) {
                uint32_t b[NP][4];
#pragma unroll
                for (int i = 0; i < NP; ++i) Y.b_t(b[i], (jb + j) * 16, cb + n * 16, i);
                rest.template mma<PP, NP, (PP > NP ? PP : NP)>(out, 2 * n, a, b);
            }
        }
    rest.add(out);
}

// The same for one block, whose tokens do not all see each other: a value of Y
// that is not finite stays away from the rows before its own, which in a matrix
// product would meet it with a weight of zero.
template <int NP, int NT>
__device__ __forceinline__ void weighted_apart(float (*out)[4], const float (*p)[4], const bf16* Y, int ld,
                                               int step, int cb) {
    const int l = lane_id();
#pragma unroll
    for (int s = 0; s < 16; ++s) {
        const int from = (l & ~3) | ((s & 7) >> 1);
        const float p0 = __shfl_sync(0xffffffffu, p[s / 8][s & 1], from);
        const float p1 = __shfl_sync(0xffffffffu, p[s / 8][2 + (s & 1)], from);
        const bf16* y = Y + s * ld + cb + (l & 3) * 2;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(y + n * 8);
            float a = low(w), b = high(w);
#pragma unroll
            for (int p = 1; p < NP; ++p) {
                const uint32_t w2 = *reinterpret_cast<const uint32_t*>(y + p * step + n * 8);
                a += low(w2), b += high(w2);
            }
            if (s <= (l >> 2)) out[n][0] += p0 * a, out[n][1] += p0 * b;
            if (s <= (l >> 2) + 8) out[n][2] += p1 * a, out[n][3] += p1 * b;
        }
    }
}

template <int NT>
__device__ __forceinline__ void scale_rows(float (*x)[4], float r0, float r1) {
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n][0] *= r0, x[n][1] *= r0, x[n][2] *= r1, x[n][3] *= r1;
}
// A strip of scores from block jb on, by its columns' factors: column(s) is the
// address of those of s and s + 1.
template <int NB, typename F>
__device__ __forceinline__ void scale_columns(float (*p)[4], F&& column, int jb) {
#pragma unroll
    for (int n = 0; n < 2 * NB; ++n) {
        const float2 f = *reinterpret_cast<const float2*>(column(jb * 16 + n * 8 + (lane_id() & 3) * 2));
        p[n][0] *= f.x, p[n][1] *= f.y, p[n][2] *= f.x, p[n][3] *= f.y;
    }
}
// The scores of block rb's tokens (rows) with themselves, decayed; later columns are zeros.
template <int C>
__device__ __forceinline__ void near_decays(float (*p)[4], const Decays<C>& d, int rb, float scale) {
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = (l >> 2) + (i >> 1) * 8, s = n * 8 + (l & 3) * 2 + (i & 1);
            p[n][i] = s <= t ? p[n][i] * (d.between(rb * 16 + t, rb * 16 + s) * scale) : 0.0f;
        }
}

// 16 rows of a state in fp32 (dk, dv), in NT column tiles, from and to registers.
template <int NT>
__device__ __forceinline__ void load_state(float (*S)[4], const float* from, int row, int dk, int dv) {
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row + (l >> 2) + (i >> 1) * 8, c = n * 8 + (l & 3) * 2 + (i & 1);
            S[n][i] = from && r < dk && c < dv ? from[r * dv + c] : 0.0f;
        }
}
template <int NT>
__device__ __forceinline__ void store_state(const float (*S)[4], float* to, int row, int dk, int dv) {
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row + (l >> 2) + (i >> 1) * 8, c = n * 8 + (l & 3) * 2 + (i & 1);
            if (r < dk && c < dv) to[r * dv + c] = S[n][i];
        }
}

// The same as PN bf16 planes with rows of D values and `plane` values each, by way of 16 rows of shared memory of the
// warp's own, in packs of 16 bytes.
template <int PN, int D, int NT>
__device__ __forceinline__ void state_planes(const float (*S)[4], bf16* to, int plane, int row, bf16* by) {
    constexpr int LD = NT * 8 + 8, ROWS = 32 / NT;  // NT lanes to a row
    const int l = lane_id();
    const uint32_t at = smem_u32(by + (l & 15) * LD + (l >> 4) * 8);
#pragma unroll
    for (int p = 0; p < PN; ++p) {
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
            uint32_t r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float u = S[n + i / 2][i % 2 * 2], v = S[n + i / 2][i % 2 * 2 + 1];
                r[i] = pack2(u, v);
                for (int q = 0; q < p; ++q) {
                    u -= low(r[i]), v -= high(r[i]);
                    r[i] = pack2(u, v);
                }
            }
            stsm4(at + n * 16, r);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 16; i += ROWS)
            *reinterpret_cast<uint4*>(to + p * plane + (row + l / NT + i) * D + l % NT * 8) =
                *reinterpret_cast<const uint4*>(by + (l / NT + i) * LD + l % NT * 8);
        __syncwarp();
    }
}

// 16 rows of tokens from t0 on, their columns from `cb`: rows from `end` on are zeros.
template <typename T, int NT>
__device__ __forceinline__ void store_rows(const float (*x)[4], T* to, long long stride, int t0, int cb,
                                           int end, int T_, int d) {
    const int l = lane_id();
    const bool pairs = d % 2 == 0 && stride % 2 == 0 && reinterpret_cast<uintptr_t>(to) % (2 * sizeof(T)) == 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = t0 + (l >> 2) + i * 8;
        if (t >= T_) continue;
        T* row = to + (long long)t * stride;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int c = cb + n * 8 + (l & 3) * 2;
            const float u = t < end ? x[n][2 * i] : 0.0f, v = t < end ? x[n][2 * i + 1] : 0.0f;
            if (pairs && c < d) {
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<float2*>(row + c) = make_float2(u, v);
                } else {
                    T two[2] = {from_f<T>(u), from_f<T>(v)};
                    uint32_t w;
                    __builtin_memcpy(&w, two, 4);
                    *reinterpret_cast<uint32_t*>(row + c) = w;
                }
            } else {
                if (c < d) row[c] = from_f<T>(u);
                if (c + 1 < d) row[c + 1] = from_f<T>(v);
            }
        }
    }
}

// The same for 16-bit values by way of 16 rows of shared memory (LD values apart,
// the warp's own), where the rows come in whole packs of 16 bytes.
template <typename T, int NT, int LD>
__device__ __forceinline__ void store_rows_by(bf16* by, const float (*x)[4], T* to, long long stride, int t0,
                                              int cb, int end, int T_, int d) {
    if constexpr (sizeof(T) == 2) {
        if (d % 8 == 0 && stride % 8 == 0 && reinterpret_cast<uintptr_t>(to) % 16 == 0) {
            const int l = lane_id();
            const uint32_t at = smem_u32(by + (l & 15) * LD + (l >> 4) * 8);
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t r[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = x[n + i / 2][i % 2 * 2], v = x[n + i / 2][i % 2 * 2 + 1];
                    if constexpr (std::is_same<T, bf16>::value) {
                        r[i] = pack2(u, v);
                    } else {
                        const __half2 h = __floats2half2_rn(u, v);
                        r[i] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                }
                stsm4(at + n * 16, r);
            }
            __syncwarp();
            constexpr int ROWS = 32 / NT;  // a lane for each pack of a row, rows at once
            const int row = l / NT, col = cb + l % NT * 8;
            T* p = to + (long long)(t0 + row) * stride + col;
            if (col < d) {
#pragma unroll
                for (int i = 0; i < 16; i += ROWS) {
                    const int t = t0 + row + i;
                    uint4 w = *reinterpret_cast<const uint4*>(by + (row + i) * LD + l % NT * 8);
                    if (t >= end) w = make_uint4(0, 0, 0, 0);
                    if (t < T_) *reinterpret_cast<uint4*>(p) = w;
                    p += ROWS * stride;
                }
            }
            __syncwarp();
            return;
        }
    }
    store_rows<T, NT>(x, to, stride, t0, cb, end, T_, d);
}

// Rows [t0, t1) of zeros.
template <typename T>
__device__ __forceinline__ void zero_rows(T* to, long long stride, int t0, int t1, int d) {
    for (long long i = threadIdx.x; i < (long long)max(0, t1 - t0) * d; i += blockDim.x)
        to[(t0 + i / d) * stride + i % d] = from_f<T>(0.0f);
}

// The CTA of a kernel: NW warps share a chunk's C / 16 blocks of tokens, and where
// there are more warps than blocks, a block's columns. In bf16 with heads of up to 64
// there is a warp to a block: with two, both computed its scores (outputs of 16 x 2048 x
// 12 heads 69 us instead of 50, gradients 296 instead of 223; chunks of 128 tokens with
// eight warps 62 and 254); the other forms have too much to do for four warps.
template <typename T_, int KD_, int VD_, int C_>
struct Shape {
    typedef T_ T;
    static constexpr int NP = planes_of<T_>, C = C_, NW = NP == 1 && KD_ == 64 && VD_ == 64 ? 4 : 8, THREADS = NW * 32;
    static constexpr int KD = KD_, VD = VD_, LK = KD + 8, LV = VD + 8;  // rows of keys, of values and of states
    static constexpr int KT = NP * C * LK, VT = NP * C * LV, STATE = KD * LV;
    static constexpr int RB = C / 16, CG = NW / RB, NK = KD / CG / 8, NV = VD / CG / 8;
    static_assert(NW % RB == 0 && NK % 2 == 0 && NV % 2 == 0, "whole blocks for the warps");
    // a states' pass: a warp for every 16 rows (with half of the columns to a warp, the rows' planes were
    // formed twice: a fifth slower)
    static constexpr int SW = KD / 16, ST = SW * 32, SNT = VD / 8;
};

__device__ __forceinline__ Tile tile(const bf16* p, int ld, int step) {
    return {smem_u32(p), (uint32_t)ld * 2, (uint32_t)step * 2};
}

// ------------------------------------------------------------------ states
// What a pass over a sequence adds up: x y^T over its tokens, forwards (keys and
// values) or backwards (queries and the gradient of the outputs).
struct Pass {
    const void *x, *y;
    Strides xs, ys;
    const float* start;    // the first state, or null
    float *sums, *factor;  // what each chunk adds to a state of zeros (KD x VD), and its decay
    bf16* kept;            // the state before (backwards: behind) each chunk, planes of KD x VD
    float* end;            // the last state, or null
    bool back;
};

// The states alone: with KEEP a CTA goes through the chunks of a head; without,
// each chunk has a CTA, which leaves its sum and factor. The decays of the next
// chunk are the work of one more warp, and its tiles are on their way meanwhile. PN:
// planes of the kept states. A warp has 16 rows of the state in registers, all its columns.
// 16 x 2048 x 12 of 64 in bf16: 62 us, and both passes of a gradient 116 (3.8 TB/s; matrix
// instructions 37% of the time): a chunk's sum waits for its weighted values, which take
// as long to form in three parts as to multiply, and the next chunk waits for it. A state's
// rows on two CTAs, which would fill the SMs more evenly, gained nothing and took 164.
// Where keys are wider than 64 the ninth warp, of the decays, leaves a thread 168 registers
// (96 where two CTAs share an SM), and the walk spills: up to 256 bytes stored in bf16, 332
// in fp16, 520 in fp32 (224 there for values wider than 64). 16 x 2048 x 12 of 128 take
// 0.40 ms in bf16, 1.07 in fp16, 1.67 in fp32, with gradients 1.8, 3.9 and 5.2.
template <class S_, bool KEEP, int PN>
__global__ void __launch_bounds__(S_::ST + 32, KEEP && S_::SNT > 8 ? 1 : 2)
state_kernel(const Job j, const Pass p0, const Pass p1, Decays<S_::C>* dec_out) {
    pdl_trigger();
    typedef typename S_::T T;
    constexpr int NP = S_::NP, KD = S_::KD, VD = S_::VD, C = S_::C, NT = S_::SNT;
    // (three planes leave room for one stage, which is filled when every warp is done with it)
    constexpr int STAGES = NP == 3 || !KEEP ? 1 : NP == 2 ? 2 : 3;
    constexpr int AHEAD = NP == 1 && KEEP ? 2 : 1;  // stages on their way
    constexpr int STAGE = S_::KT + S_::VT;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* const tiles = reinterpret_cast<bf16*>(smem);
    __shared__ Decays<C> dec_[2];
    __shared__ __align__(16) bf16 by_[KEEP ? S_::SW : 1][KEEP ? 16 * (NT * 8 + 8) : 8];
    const Pass& p = blockIdx.y ? p1 : p0;
    const long long bh = KEEP ? blockIdx.x : blockIdx.x / j.chunks;
    const int b = (int)(bh / j.H), h = (int)(bh % j.H), end = tokens_of(j, b);
    const int c0 = KEEP ? 0 : blockIdx.x % j.chunks;
    const int live = KEEP ? (end + C - 1) / C : c0 + (c0 * C < end), n = live - c0;
    const auto chunk = [&](int i) { return p.back ? live - 1 - i : c0 + i; };
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;

    if (warp == S_::SW) {  // the decays
        constexpr int M = C / 32;
        const float* g = j.g + b * j.gs.b + h * j.gs.h;
        constexpr int FAR = 4;  // chunks whose log decays are on their way
        float x[FAR][M];
        const auto ask = [&](float* to, int i) {
#pragma unroll
            for (int k = 0; k < M; ++k) {
                const int t = chunk(i) * C + l * M + k;
                to[k] = i < n && t < end ? g[(long long)t * j.gs.t] : 0.0f;
            }
        };
#pragma unroll
        for (int i = 0; i < FAR; ++i) ask(x[i], i);
        if (n) decays<C>(&dec_[0], x[0]);
        for (int i = 0; i < n; ++i) {
            __syncthreads();  // (what is written behind it was read a chunk ago)
            if (!blockIdx.y) {
                const float4* from = reinterpret_cast<const float4*>(&dec_[i & 1]);
                float4* to = reinterpret_cast<float4*>(dec_out + bh * j.chunks + chunk(i));
                for (int k = l; k < (int)sizeof(Decays<C>) / 16; k += 32) to[k] = from[k];
            }
#pragma unroll
            for (int a = 0; a + 1 < FAR; ++a)
#pragma unroll
                for (int k = 0; k < M; ++k) x[a][k] = x[a + 1][k];
            ask(x[FAR - 1], i + FAR);
            if (i + 1 < n) decays<C>(&dec_[(i + 1) & 1], x[0]);
#pragma unroll
            for (int k = 1; k < (STAGES == 1 ? 2 : 1); ++k) __syncthreads();
        }
        return;
    }

    const int row = warp * 16;
    const T* x = head_of<T>(p.x, p.xs, b, h / j.share);
    const T* y = head_of<T>(p.y, p.ys, b, h);
    const bool wx = j.whole >> (p.back ? 0 : 1) & 1, wy = j.whole >> (p.back ? 3 : 2) & 1;
    Fetch<T, C, KD, S_::ST> lx;
    Fetch<T, C, VD, S_::ST> ly;
    const auto fetch = [&](int i, int stage) {
        if (i < n) {
            bf16* to = tiles + stage * STAGE;
            lx.fetch(to, x, p.xs.t, chunk(i) * C, end, j.dk, wx);
            ly.fetch(to + S_::KT, y, p.ys.t, chunk(i) * C, end, j.dv, wy);
        }
        cp_async_commit();
    };
    const auto put = [&](int i, int stage) {
        if (i < n) {
            bf16* to = tiles + stage * STAGE;
            lx.put(to, x, p.xs.t, chunk(i) * C, end, j.dk, wx);
            ly.put(to + S_::KT, y, p.ys.t, chunk(i) * C, end, j.dv, wy);
        }
    };
    for (int i = 0; i < AHEAD; ++i) fetch(i, i);
    put(0, 0);
    float S[NT][4];
    if constexpr (KEEP)
        load_state<NT>(S, p.start ? p.start + bh * j.dk * j.dv : nullptr, row, j.dk, j.dv);
    else
        clear<NT>(S);
    int stage = 0;
    for (int i = 0; i < n; ++i) {
        const Decays<C>& dec = dec_[i & 1];
        cp_async_wait_group<AHEAD - 1>();
        __syncthreads();
        fetch(i + AHEAD, (stage + AHEAD) % STAGES);
        if constexpr (KEEP)
            state_planes<PN, VD, NT>(S, p.kept + (bh * j.chunks + chunk(i)) * PN * KD * VD, KD * VD, row, by_[warp]);
        const bf16* from = tiles + stage * STAGE;
        float sum[NT][4];
        clear<NT>(sum);
        add_outer<NP, NT, C>(sum, tile(from, S_::LK, C * S_::LK), tile(from + S_::KT, S_::LV, C * S_::LV),
                             p.back ? dec.from_start : dec.to_end, p.back ? j.scale : 1.0f, row, 0, end - chunk(i) * C);
        // The chunk's sum is added here, not in the matrix instruction, which cuts its sums off: over a
        // sequence that leaned by 2^-24 of the state a step.
        const float f = dec.whole;
#pragma unroll
        for (int m = 0; m < NT; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[m][e] = fmaf(S[m][e], f, sum[m][e]);
        if constexpr (STAGES == 1) __syncthreads();
        stage = (stage + 1) % STAGES;
        put(i + 1, stage);
    }
    if constexpr (!KEEP) {
        if (!n) return;
        float* const to = p.sums + (bh * j.chunks + c0) * KD * VD;
#pragma unroll
        for (int m = 0; m < NT; ++m)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                *reinterpret_cast<float2*>(to + (row + (l >> 2) + i * 8) * VD + m * 8 + (l & 3) * 2) =
                    make_float2(S[m][2 * i], S[m][2 * i + 1]);
        if (threadIdx.x == 0) p.factor[bh * j.chunks + c0] = dec_[0].whole;
    } else if (p.end) {
        store_state<NT>(S, p.end + bh * j.dk * j.dv, row, j.dk, j.dv);
    }
}

// The kept states and the last one from the chunks' sums: a thread for four
// neighbouring values of a state. Bound by HBM and the chunks' order: 8192 x 12 of 128 in bf16
// 28 us, 150 MB at 5.4 TB/s.
template <int KD, int VD, int C, int PN>
__global__ void __launch_bounds__(256) scan_kernel(const Job j, const Pass p0, const Pass p1) {
    pdl_trigger();
    const Pass& p = blockIdx.y ? p1 : p0;
    const long long i = blockIdx.x * 256ll + threadIdx.x, bh = i / (KD * VD / 4);
    if (bh >= (long long)j.B * j.H) return;
    const int e = (int)(i % (KD * VD / 4)) * 4, r = e / VD, c = e % VD;
    const int live = (tokens_of(j, (int)(bh / j.H)) + C - 1) / C;
    constexpr int SIZE = KD * VD;
    float S[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
        S[k] = p.start && r < j.dk && c + k < j.dv ? p.start[(bh * j.dk + r) * j.dv + c + k] : 0.0f;
    const float* const sums = p.sums + bh * j.chunks * SIZE + e;
    const float* const factor = p.factor + bh * j.chunks;
    bf16* const kept = p.kept + bh * j.chunks * PN * SIZE + e;
    constexpr int U = 8;  // asked for together
    for (int k0 = 0; k0 < live; k0 += U) {
        float4 add[U];
        float by[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = min(k0 + u, live - 1), k = p.back ? live - 1 - at : at;
            add[u] = *reinterpret_cast<const float4*>(sums + (long long)k * SIZE);
            by[u] = factor[k];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k0 + u < live) {
                const int k = p.back ? live - 1 - k0 - u : k0 + u;
                float part[4] = {S[0], S[1], S[2], S[3]};
#pragma unroll
                for (int q = 0; q < PN; ++q) {
                    const uint2 w = {pack2(part[0], part[1]), pack2(part[2], part[3])};
                    *reinterpret_cast<uint2*>(kept + ((long long)k * PN + q) * SIZE) = w;
                    part[0] -= low(w.x), part[1] -= high(w.x), part[2] -= low(w.y), part[3] -= high(w.y);
                }
                S[0] = by[u] * S[0] + add[u].x, S[1] = by[u] * S[1] + add[u].y;
                S[2] = by[u] * S[2] + add[u].z, S[3] = by[u] * S[3] + add[u].w;
            }
    }
    if (p.end) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (r < j.dk && c + k < j.dv) p.end[(bh * j.dk + r) * j.dv + c + k] = S[k];
    }
}

// ----------------------------------------------------------------- outputs
// A CTA for each chunk: the states before them are there, so all run at once.
// Heads go side by side: they lie so in memory. 16 x 2048 x 12 of 64 in bf16: 53 us, 240 MB
// at 4.6 TB/s (0.7 of a copy's rate); the rest are waits between products that follow
// from one another. Blocks of 16 without tokens are left out (64 sequences of up to 257
// tokens in fp32: 192 -> 182 us).
struct Chunk {
    int b, h, c;
    long long bh;
    __device__ __forceinline__ explicit Chunk(const Job& j) {
        const long long n = blockIdx.x / j.H;
        h = blockIdx.x % j.H;
        c = (int)(n % j.chunks);
        b = (int)(n / j.chunks);
        bh = (long long)b * j.H + h;
    }
};

// A tile of kept states (PN planes of KD x VD), and a chunk's decays, by cp.async.
template <class S_, int PN>
__device__ __forceinline__ void load_kept(bf16* dst, const bf16* from) {
    constexpr int PACKS = S_::KD * S_::VD / 8, ROW = S_::VD / 8;
#pragma unroll
    for (int n = 0; n < PN * PACKS / S_::THREADS; ++n) {
        const int i = n * S_::THREADS + threadIdx.x;
        cp_async16(dst + i / PACKS * S_::STATE + i % PACKS / ROW * S_::LV + i % ROW * 8, from + i * 8, 16);
    }
}
template <int C>
__device__ __forceinline__ void load_decays(Decays<C>* to, const Decays<C>* from) {
    if (threadIdx.x < sizeof(Decays<C>) / 16)
        cp_async16(reinterpret_cast<float4*>(to) + threadIdx.x, reinterpret_cast<const float4*>(from) + threadIdx.x,
                   16);
}

template <class S_, int MIN>
__global__ void __launch_bounds__(S_::THREADS, MIN)
out_kernel(const Job j, const bf16* kept, const Decays<S_::C>* decs, void* out_) {
    typedef typename S_::T T;
    constexpr int NP = S_::NP, KD = S_::KD, C = S_::C, LK = S_::LK, LV = S_::LV, NT = S_::NV, NB = 2;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* const sq = reinterpret_cast<bf16*>(smem);
    bf16 *const sk = sq + S_::KT, *const sv = sk + S_::KT, *const ss = sv + S_::VT;
    __shared__ Decays<C> dec;
    const Chunk at(j);
    const int end = tokens_of(j, at.b), c0 = at.c * C;
    const long long ot = (long long)j.H * j.dv;
    T* out = static_cast<T*>(out_) + (long long)at.b * j.T * ot + (long long)at.h * j.dv;
    if (c0 >= end) {
        zero_rows(out, ot, c0, min(c0 + C, j.T), j.dv);
        pdl_wait();  // (where no sequence has a token, all CTAs leave here: not before the states are there)
        return;
    }
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;
    const int rb = warp % S_::RB, cb = warp / S_::RB * NT * 8;
    const bool on = rb * 16 < end - c0;  // the warp's block holds tokens
    const T* q = head_of<T>(j.q, j.qs, at.b, at.h / j.share);
    const T* k = head_of<T>(j.k, j.ks, at.b, at.h / j.share);
    const T* v = head_of<T>(j.v, j.vs, at.b, at.h);
    Fetch<T, C, KD, S_::THREADS> lq, lk;
    Fetch<T, C, S_::VD, S_::THREADS> lv;
    lq.fetch(sq, q, j.qs.t, c0, end, j.dk, j.whole & 1);
    pdl_wait();  // (the call's inputs were there before its first launch)
    load_kept<S_, NP>(ss, kept + (at.bh * j.chunks + at.c) * NP * KD * S_::VD);
    load_decays<C>(&dec, decs + at.bh * j.chunks + at.c);
    cp_async_commit();
    lk.fetch(sk, k, j.ks.t, c0, end, j.dk, j.whole >> 1 & 1);
    lv.fetch(sv, v, j.vs.t, c0, end, j.dv, j.whole >> 2 & 1);
    cp_async_commit();
    lq.put(sq, q, j.qs.t, c0, end, j.dk, j.whole & 1);
    lk.put(sk, k, j.ks.t, c0, end, j.dk, j.whole >> 1 & 1);
    lv.put(sv, v, j.vs.t, c0, end, j.dv, j.whole >> 2 & 1);
    cp_async_wait_group<1>();
    __syncthreads();
    const Tile tq = tile(sq, LK, C * LK), tk = tile(sk, LK, C * LK), tv = tile(sv, LV, C * LV),
               ts = tile(ss, LV, S_::STATE);

    // Between the blocks of 16 tokens a decay is 2^(c_t - c_r) 2^(c_r - c_s), r the
    // last token before the row's block: a factor of the row, which the state's
    // part shares, and one of the column, which the warp writes down once (behind the
    // rows of its block's queries, four to a row). Both are at most 1. Within a block
    // each pair has its own.
    static_assert(C <= 64, "room behind the rows");
    const auto column = [&](int s) { return reinterpret_cast<float*>(sq + (rb * 16 + s / 4) * LK + KD) + s % 4; };
    for (int s = l; s < rb * 16; s += 32) *column(s) = dec.between(rb * 16 - 1, s);
    __syncwarp();
    float O[NT][4];
    const int t = rb * 16 + (l >> 2);
    const float r0 = (rb ? dec.between(t, rb * 16 - 1) : dec.from_start[t]) * j.scale;
    const float r1 = (rb ? dec.between(t + 8, rb * 16 - 1) : dec.from_start[t + 8]) * j.scale;
    const auto before = [&] {
        product<NP, NP, KD, NT, true>(O, tq, rb * 16, ts, cb);
        if (rb) {
            const float begin = dec.from_start[rb * 16 - 1];
            scale_rows<NT>(O, begin, begin);
        }
    };
    const auto chunk = [&](bool apart) {
        for (int jb = 0; jb < rb; jb += NB) {
            float P[2 * NB][4];
            scores<NP, KD, NB>(P, tq, rb * 16, tk, jb, 0, rb);
            scale_columns<NB>(P, column, jb);
            weighted<NP, NP, NB, NT>(O, P, tv, cb, jb, 0, rb);
        }
        scale_rows<NT>(O, r0, r1);
        float P[2][4];
        scores<NP, KD, 1>(P, tq, rb * 16, tk, rb, rb, rb + 1);
        near_decays<C>(P, dec, rb, j.scale);
        if (apart)
            weighted_apart<NP, NT>(O, P, sv + rb * 16 * LV, LV, C * LV, cb);
        else
            weighted<NP, NP, 1, NT>(O, P, tv, cb, rb, rb, rb + 1);
    };
    clear<NT>(O);
    if (on) before();
    cp_async_wait_all();
    __syncthreads();
    if (on) {
        chunk(false);
        // a value of v that is not finite reaches every row of its block (times zero, in those before it)
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) sum = fmaf(O[n][0], 0.0f, fmaf(O[n][1], 0.0f, sum));
        if (__any_sync(0xffffffffu, sum != 0.0f)) {
            clear<NT>(O);
            before();
            chunk(true);
        }
    }
    if constexpr (S_::VD <= KD) {  // by way of these rows' queries, which are done with
        if constexpr (S_::CG > 1) named_bar_sync(rb + 1, S_::CG * 32);
        store_rows_by<T, NT, LK>(sq + rb * 16 * LK + cb, O, out, ot, c0 + rb * 16, cb, end, j.T, j.dv);
    } else {
        store_rows<T, NT>(O, out, ot, c0 + rb * 16, cb, end, j.T, j.dv);
    }
}

// ---------------------------------------------------------------- gradients
// A CTA for each chunk again. First by rows s (dk, dv, with the gradient behind the chunk),
// then by rows t (dq, with the state before it), so that every product finds its left
// side in the warp's registers; the scores of do and v are computed for both. 16 x 2048 x
// 12 of 64 in bf16: 223 us, 643 MB at 2.9 TB/s, matrix instructions 30% of the time: 168
// registers and 66 KB leave three CTAs of four warps on an SM, which wait for their states,
// for ldmatrix and for one another. 3 x 1001 x 6 of 40 and 72 in fp32: 77 us, two waves of
// one CTA an SM.
struct Grads {
    const void* dout;
    Strides ds;
    const bf16 *before, *behind;  // the states before the chunks, their gradients behind them
    void *dq, *dk, *dv;
    float *dq32, *dk32;  // in place of dq, dk: each head's own, where heads share q and k
    float* dg;           // (B, T, H), or null
};

// A row of 16-bit pairs (or more planes of them) times a block of products: each
// lane's part of the sums over the columns, for its rows g and g + 8.
template <int NP, int NT>
__device__ __forceinline__ void row_dots(const float (*x)[4], const bf16* tile, int ld, int step, int r,
                                         int cb, float* sum) {
    const int l = lane_id();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float s = 0.0f;
        const bf16* at = tile + (r + (l >> 2) + i * 8) * ld + cb + (l & 3) * 2;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(at + n * 8);
            float u = low(w), v = high(w);
#pragma unroll
            for (int p = 1; p < NP; ++p) {
                const uint32_t w2 = *reinterpret_cast<const uint32_t*>(at + p * step + n * 8);
                u += low(w2), v += high(w2);
            }
            s = fmaf(x[n][2 * i], u, s);
            s = fmaf(x[n][2 * i + 1], v, s);
        }
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        sum[i] = s;
    }
}

// Sums over the eight lanes that hold the same columns, of N values of each: the
// lanes share them out, and each ends with one (or, of fewer than eight, with one
// that others have too). Returns which.
template <int N>
__device__ __forceinline__ int column_sums(float* v) {
    const int l = lane_id();
    int which = 0;
#pragma unroll
    for (int d = 16, n = N; d >= 4; d /= 2) {
        if (n > 1) {
            n /= 2;
            const bool upper = l & d;
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const float keep = upper ? v[n + i] : v[i], give = upper ? v[i] : v[n + i];
                v[i] = keep + __shfl_xor_sync(0xffffffffu, give, d);
            }
            if (upper) which += n;
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], d);
        }
    }
    return which;
}

// A 16 x 16 block of products becomes, row by row, its sums from each column on.
__device__ __forceinline__ void pairs_from(float (*x)[4]) {
    const int q = lane_id() & 3;
#pragma unroll
    for (int h = 0; h < 4; h += 2) {  // rows g and g + 8
        float after = 0.0f;           // of the later columns
#pragma unroll
        for (int n = 1; n >= 0; --n) {
            float s = x[n][h] + x[n][h + 1];
#pragma unroll
            for (int d = 1; d < 4; d *= 2) {
                const float y = __shfl_down_sync(0xffffffffu, s, d, 4);
                if (q + d < 4) s += y;
            }
            const float y = __shfl_down_sync(0xffffffffu, s, 1, 4), whole = __shfl_sync(0xffffffffu, s, 0, 4);
            x[n][h + 1] += (q < 3 ? y : 0.0f) + after;
            x[n][h] += x[n][h + 1];
            after += whole;
        }
    }
}

// Sums over the lanes before (behind) this one among W neighbours.
template <int W>
__device__ __forceinline__ float sum_before(float x) {
    const int l = lane_id() % W;
#pragma unroll
    for (int d = 1; d < W; d *= 2) {
        const float y = __shfl_up_sync(0xffffffffu, x, d, W);
        if (l >= d) x += y;
    }
    x = __shfl_up_sync(0xffffffffu, x, 1, W);  // (the sum less its own x would lose small others)
    return l ? x : 0.0f;
}
template <int W>
__device__ __forceinline__ float sum_behind(float x) {
    const int l = lane_id() % W;
#pragma unroll
    for (int d = 1; d < W; d *= 2) {
        const float y = __shfl_down_sync(0xffffffffu, x, d, W);
        if (l + d < W) x += y;
    }
    x = __shfl_down_sync(0xffffffffu, x, 1, W);
    return l + 1 < W ? x : 0.0f;
}

template <class S_, int MIN>
__global__ void __launch_bounds__(S_::THREADS, MIN)
grad_kernel(const Job j, const Grads G, const Decays<S_::C>* decs) {
    pdl_trigger();
    typedef typename S_::T T;
    constexpr int NP = S_::NP, KD = S_::KD, VD = S_::VD, C = S_::C, LK = S_::LK, LV = S_::LV, NK = S_::NK, NV = S_::NV;
    constexpr int RB = S_::RB, CG = S_::CG;
    constexpr int NB = 2;  // blocks of a strip: two accumulators and two strips of scores are held
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* const sq = reinterpret_cast<bf16*>(smem);
    bf16 *const sk = sq + S_::KT, *const sv = sk + S_::KT, *const so = sv + S_::VT;
    bf16* const ss = so + S_::VT;  // the gradient behind the chunk, then the state before it
    __shared__ Decays<C> dec;
    // parts of dg: by row block (of each block's own pairs: by token), and by column group where the columns are split
    __shared__ float col_part[RB][C], row_part[C], dq_part[CG][C], dk_part[CG][C], dot_part[S_::NW];
    const Chunk at(j);
    const int end = tokens_of(j, at.b), c0 = at.c * C, c1 = min(c0 + C, j.T);
    const long long kt = (long long)j.H * j.dk, vt = (long long)j.H * j.dv;
    const long long k0 = (long long)at.b * j.T * kt + (long long)at.h * j.dk;
    T* dv = static_cast<T*>(G.dv) + (long long)at.b * j.T * vt + (long long)at.h * j.dv;
    float* dg = G.dg ? G.dg + (long long)at.b * j.T * j.H + at.h : nullptr;
    if (c0 >= end) {
        zero_rows(dv, vt, c0, c1, j.dv);
        if (G.dq32) {
            zero_rows(G.dq32 + k0, kt, c0, c1, j.dk);
            zero_rows(G.dk32 + k0, kt, c0, c1, j.dk);
        } else {
            zero_rows(static_cast<T*>(G.dq) + k0, kt, c0, c1, j.dk);
            zero_rows(static_cast<T*>(G.dk) + k0, kt, c0, c1, j.dk);
        }
        if (dg) zero_rows(dg, j.H, c0, c1, 1);
        pdl_wait();  // (as in out_kernel)
        return;
    }
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;
    const int rb = warp % RB, cg = warp / RB, ck = cg * NK * 8, cv = cg * NV * 8;
    const int live = min(RB, (end - c0 + 15) / 16);  // blocks that hold tokens
    const bool on = rb < live;
    // (in two and three parts the loops run to the chunk's end: with the other bound 6% slower, and 1% faster in one)
    const int blocks = NP == 1 ? live : RB;
    const Tile tq = tile(sq, LK, C * LK), tk = tile(sk, LK, C * LK), tv = tile(sv, LV, C * LV),
               to = tile(so, LV, C * LV), ts = tile(ss, LV, S_::STATE);
    const long long kept = (at.bh * j.chunks + at.c) * 3 * KD * VD;
    {
        const T* q = head_of<T>(j.q, j.qs, at.b, at.h / j.share);
        const T* k = head_of<T>(j.k, j.ks, at.b, at.h / j.share);
        const T* v = head_of<T>(j.v, j.vs, at.b, at.h);
        const T* dout = head_of<T>(G.dout, G.ds, at.b, at.h);
        Fetch<T, C, KD, S_::THREADS> lq, lk;
        Fetch<T, C, VD, S_::THREADS> lv, lo;
        lk.fetch(sk, k, j.ks.t, c0, end, j.dk, j.whole >> 1 & 1);
        pdl_wait();
        load_kept<S_, 3>(ss, G.behind + kept);
        load_decays<C>(&dec, decs + at.bh * j.chunks + at.c);
        lv.fetch(sv, v, j.vs.t, c0, end, j.dv, j.whole >> 2 & 1);
        cp_async_commit();
        lk.put(sk, k, j.ks.t, c0, end, j.dk, j.whole >> 1 & 1);
        lv.put(sv, v, j.vs.t, c0, end, j.dv, j.whole >> 2 & 1);
        lq.fetch(sq, q, j.qs.t, c0, end, j.dk, j.whole & 1);
        lo.fetch(so, dout, G.ds.t, c0, end, j.dv, j.whole >> 3 & 1);
        cp_async_commit();
        lq.put(sq, q, j.qs.t, c0, end, j.dk, j.whole & 1);
        lo.put(so, dout, G.ds.t, c0, end, j.dv, j.whole >> 3 & 1);
    }
    cp_async_wait_group<1>();
    __syncthreads();
    // (by way of the states' place, a part of it for each warp)
    constexpr int BK = NK * 8 + 8, BV = NV * 8 + 8, BY = BK > BV ? BK : BV;
    static_assert(S_::NW * 16 * BY <= 3 * S_::STATE, "room for every warp's rows");
    bf16* const by = ss + warp * 16 * BY;
    const auto store_head = [&](const float(*x)[4], void* to16, float* to32) {
        if (to32)
            store_rows<float, NK>(x, to32 + k0, kt, c0 + rb * 16, ck, end, j.T, j.dk);
        else
            store_rows_by<T, NK, BK>(by, x, static_cast<T*>(to16) + k0, kt, c0 + rb * 16, ck, end, j.T, j.dk);
    };
    // factors of columns, as in out_kernel
    const auto column = [&](int s) { return reinterpret_cast<float*>(sq + (rb * 16 + s / 4) * LK + KD) + s % 4; };
    constexpr int FINE = NP == 2 ? 3 : NP;  // (the scores' products in full: dg is an fp32 result)
    float part[2];
    const int t = rb * 16 + (l >> 2);  // the lane's tokens: this and 8 behind
    {
        // rows s, columns u >= s. Between blocks a decay is 2^(c_u - c_r) 2^(c_r - c_s), r
        // the last token of the row's block
        const int r = rb * 16 + 15;
        const float b0 = dec.between(r, t), b1 = dec.between(r, t + 8), behind = dec.to_end[r];
        float V[NV][4], K[NK][4], across[2] = {0.0f, 0.0f};
        clear<NV>(V);
        clear<NK>(K);
        if (on) {
            product<NP, NP, KD, NV, true>(V, tk, rb * 16, ts, cv);
            scale_rows<NV>(V, behind, behind);
            product<NP, 3, VD, NK, false>(K, tv, rb * 16, ts, ck);
            scale_rows<NK>(K, behind, behind);
            row_dots<NP, NK>(K, sk, LK, C * LK, rb * 16, ck, part);
            if ((l & 3) == 0) dk_part[cg][t] = part[0] * b0, dk_part[cg][t + 8] = part[1] * b1;
        }
        cp_async_wait_all();  // queries and the gradient of the outputs
        for (int u = r + 1 + l; u < C; u += 32) *column(u) = dec.between(u, r) * j.scale;
        __syncthreads();
        if (on) {
            for (int jb = (rb + 1) / NB * NB; jb < blocks; jb += NB) {
                float P[2 * NB][4], Q[2 * NB][4], down[4 * NB];
                scores<NP, KD, NB, FINE>(P, tk, rb * 16, tq, jb, rb + 1, RB);
                scores<NP, VD, NB, FINE>(Q, tv, rb * 16, to, jb, rb + 1, RB);
#pragma unroll
                for (int n = 0; n < 2 * NB; ++n) {
                    const int u = jb * 16 + n * 8 + (l & 3) * 2;
                    const float2 f = *reinterpret_cast<const float2*>(column(u));
                    const bool in = jb + n / 2 > rb;  // (the factors of other blocks are not there)
                    const float x0 = P[n][0] * Q[n][0], x1 = P[n][1] * Q[n][1], x2 = P[n][2] * Q[n][2],
                                x3 = P[n][3] * Q[n][3];
                    down[2 * n] = in ? (x0 * b0 + x2 * b1) * f.x : 0.0f;
                    down[2 * n + 1] = in ? (x1 * b0 + x3 * b1) * f.y : 0.0f;
                    across[0] += in ? x0 * f.x + x1 * f.y : 0.0f;
                    across[1] += in ? x2 * f.x + x3 * f.y : 0.0f;
                    P[n][0] *= f.x, P[n][1] *= f.y, P[n][2] *= f.x, P[n][3] *= f.y;
                    Q[n][0] *= f.x, Q[n][1] *= f.y, Q[n][2] *= f.x, Q[n][3] *= f.y;
                }
                const int which = column_sums<4 * NB>(down);
                if (cg == 0) col_part[rb][jb * 16 + which / 2 * 8 + (l & 3) * 2 + which % 2] = down[0];
                weighted<NP, NP, NB, NV>(V, P, to, cv, jb, rb + 1, RB);
                weighted<NP, NP, NB, NK>(K, Q, tq, ck, jb, rb + 1, RB);
            }
            scale_rows<NV>(V, b0, b1);
            scale_rows<NK>(K, b0, b1);
            across[0] *= b0, across[1] *= b1;
            float P[2][4], Q[2][4], A[2][4], down[4] = {};
            scores<NP, KD, 1, FINE>(P, tk, rb * 16, tq, rb, rb, rb + 1);
            scores<NP, VD, 1, FINE>(Q, tv, rb * 16, to, rb, rb, rb + 1);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int s = t + (i >> 1) * 8, u = rb * 16 + n * 8 + (l & 3) * 2 + (i & 1);
                    const float w = dec.between(u, s) * j.scale, p = P[n][i] * w;
                    A[n][i] = u > s ? p * Q[n][i] : 0.0f;
                    P[n][i] = u >= s ? p : 0.0f;
                    Q[n][i] = u >= s ? Q[n][i] * w : 0.0f;
                }
            // the block's own pairs: of the rows before each column, the sums from it on
            pairs_from(A);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if ((l >> 2) + (i >> 1) * 8 < n * 8 + (l & 3) * 2 + (i & 1)) down[2 * n + (i & 1)] += A[n][i];
            const int which = column_sums<4>(down);
            if (cg == 0) col_part[rb][rb * 16 + which / 2 * 8 + (l & 3) * 2 + which % 2] = down[0];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                across[i] += __shfl_xor_sync(0xffffffffu, across[i], 1);
                across[i] += __shfl_xor_sync(0xffffffffu, across[i], 2);
            }
            if (cg == 0 && (l & 3) == 0) row_part[t] = across[0], row_part[t + 8] = across[1];
            weighted<NP, NP, 1, NV>(V, P, to, cv, rb, rb, rb + 1);
            weighted<NP, NP, 1, NK>(K, Q, tq, ck, rb, rb, rb + 1);
        }
        // <R, S>, and then their place is free
        float dot = 0.0f;
        if (dg) {
            const uint4* from = reinterpret_cast<const uint4*>(G.before + kept);
            constexpr int PACKS = KD * VD / 8, ROW = VD / 8;
#pragma unroll 2
            for (int i = threadIdx.x; i < PACKS; i += S_::THREADS) {
                uint4 x[3], r[3];
#pragma unroll
                for (int p = 0; p < 3; ++p) {
                    x[p] = from[p * PACKS + i];
                    r[p] = *reinterpret_cast<const uint4*>(ss + p * S_::STATE + i / ROW * LV + i % ROW * 8);
                }
                const auto add = [&](uint32_t a0, uint32_t a1, uint32_t a2, uint32_t b0, uint32_t b1, uint32_t b2) {
                    dot = fmaf(low(a0) + (low(a1) + low(a2)), low(b0) + (low(b1) + low(b2)), dot);
                    dot = fmaf(high(a0) + (high(a1) + high(a2)), high(b0) + (high(b1) + high(b2)), dot);
                };
                add(x[0].x, x[1].x, x[2].x, r[0].x, r[1].x, r[2].x);
                add(x[0].y, x[1].y, x[2].y, r[0].y, r[1].y, r[2].y);
                add(x[0].z, x[1].z, x[2].z, r[0].z, r[1].z, r[2].z);
                add(x[0].w, x[1].w, x[2].w, r[0].w, r[1].w, r[2].w);
            }
        }
#pragma unroll
        for (int d = 16; d; d /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (l == 0) dot_part[warp] = dot;
        __syncthreads();
        store_rows_by<T, NV, BV>(by, V, dv, vt, c0 + rb * 16, cv, end, j.T, j.dv);
        store_head(K, G.dk, G.dk32);
    }
    __syncthreads();
    load_kept<S_, 3>(ss, G.before + kept);
    cp_async_wait_all();
    for (int s = l; s < rb * 16; s += 32) *column(s) = dec.between(rb * 16 - 1, s);
    __syncthreads();
    {
        // rows u, columns s <= u, as the outputs
        float X[NK][4], P[2][4];
        clear<NK>(X);
        if (on) {
            product<NP, 3, VD, NK, false>(X, to, rb * 16, ts, ck);
            const float begin = rb ? dec.from_start[rb * 16 - 1] : 1.0f;
            scale_rows<NK>(X, begin, begin);
            const float r0 = (rb ? dec.between(t, rb * 16 - 1) : dec.from_start[t]) * j.scale;
            const float r1 = (rb ? dec.between(t + 8, rb * 16 - 1) : dec.from_start[t + 8]) * j.scale;
            row_dots<NP, NK>(X, sq, LK, C * LK, rb * 16, ck, part);
            if ((l & 3) == 0) dq_part[cg][t] = part[0] * r0, dq_part[cg][t + 8] = part[1] * r1;
            for (int jb = 0; jb < rb; jb += NB) {
                float Q[2 * NB][4];
                scores<NP, VD, NB>(Q, to, rb * 16, tv, jb, 0, rb);
                scale_columns<NB>(Q, column, jb);
                weighted<NP, NP, NB, NK>(X, Q, tk, ck, jb, 0, rb);
            }
            scale_rows<NK>(X, r0, r1);
            scores<NP, VD, 1>(P, to, rb * 16, tv, rb, rb, rb + 1);
            near_decays<C>(P, dec, rb, j.scale);
            weighted<NP, NP, 1, NK>(X, P, tk, ck, rb, rb, rb + 1);
        }
        __syncthreads();
        store_head(X, G.dq, G.dq32);
    }
    if (warp == 0 && dg) {
        // A sum for each token t of what passes its gate, and nothing taken away again, so that a
        // small one is as good as its terms: sums over the chunk from t on of what the outputs have of
        // the state before it, up to t of what the tokens leave in the one behind; of the pairs those
        // within t's block, those of its tokens before t with later blocks, of earlier blocks with its
        // tokens from t on, and of earlier with later blocks.
        constexpr int M = C / 32, LANES = 16 / M;  // tokens of a lane, lanes of a block
        const int K = l / LANES;
        float behind[M], ahead[M], rows[M], cols[M], own[M], all = 0.0f, b = 0.0f, a = 0.0f, r = 0.0f, c = 0.0f;
        float far[RB + 1] = {};
#pragma unroll
        for (int i = 0; i < S_::NW; ++i) all += dot_part[i];
        all *= dec.whole;
#pragma unroll
        for (int i = M - 1; i >= 0; --i) {
            const int u = l * M + i;
            own[i] = 0.0f;
            if (K < live) {
#pragma unroll
                for (int g = 0; g < CG; ++g) b += dq_part[g][u];
                float x = 0.0f;
#pragma unroll
                for (int g = 0; g < RB; ++g)
                    if (g < K) {
                        x += col_part[g][u];
                        if (g + 1 < K) far[g + 1] += x;  // of blocks up to g with this one
                    }
                c += x;
                own[i] = col_part[K][u];
            }
            behind[i] = b, cols[i] = c;
        }
#pragma unroll
        for (int i = 0; i < M; ++i) {
            ahead[i] = a, rows[i] = r;
            if (K < live) {
#pragma unroll
                for (int g = 0; g < CG; ++g) a += dk_part[g][l * M + i];
                r += row_part[l * M + i];
            }
        }
        const float outside = sum_behind<32>(b) + sum_before<32>(a);
        float pairs = sum_before<LANES>(r) + sum_behind<LANES>(c);
#pragma unroll
        for (int g = 1; g + 1 < RB; ++g) {
            float x = far[g];
#pragma unroll
            for (int d = 16; d; d /= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
            if (g == K) pairs += x;
        }
#pragma unroll
        for (int i = 0; i < M; ++i) {
            const int u = c0 + l * M + i;
            if (u < j.T)
                dg[(long long)u * j.H] =
                    u < end ? all + (behind[i] + ahead[i] + outside) + (own[i] + rows[i] + cols[i] + pairs) : 0.0f;
        }
    }
}

// Sums over the heads that share one of q and k.
template <typename T>
__global__ void __launch_bounds__(256) fold_kernel(const float* x, const float* y, T* to_x, T* to_y,
                                                   int share, int d, long long n) {
    pdl_trigger();
    pdl_wait();
    const float* from = blockIdx.y ? y : x;
    T* to = blockIdx.y ? to_y : to_x;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
        const float* at = from + i / d * share * d + i % d;
        float s = 0.0f;
        for (int r = 0; r < share; ++r) s += at[(long long)r * d];
        to[i] = from_f<T>(s);
    }
}

// dg (n, H) summed down its rows, in fp64 and always in one order: a CTA for
// each part of the rows, the parts by a second launch of one.
__global__ void __launch_bounds__(256) gate_kernel(const float* dg, const double* parts, double* to_parts,
                                                   float* out, long long n, int H, int count) {
    pdl_trigger();
    pdl_wait();
    __shared__ double s[8];
    for (int h = blockIdx.y; h < H; h += gridDim.y) {
        double x = 0.0;
        if (dg) {
            for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll)
                x += (double)dg[i * H + h];
        } else {
            for (int i = threadIdx.x; i < count; i += 256) x += parts[(long long)h * count + i];
        }
#pragma unroll
        for (int d = 16; d; d /= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int i = 1; i < 8; ++i) x += s[i];
            if (dg)
                to_parts[(long long)h * gridDim.x + blockIdx.x] = x;
            else
                out[h] = (float)x;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ launches
template <class S_>
struct Sizes {
    static constexpr int sum = (S_::KT + S_::VT) * 2, state = (4 - S_::NP) * sum;
    static constexpr int out = (2 * S_::KT + S_::VT + S_::NP * S_::STATE) * 2;
    static constexpr int grad = (2 * S_::KT + 2 * S_::VT + 3 * S_::STATE) * 2;
};

template <typename K>
int allow(K* kernel, int bytes, const char* what) {
    return cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
}

// A launch that may start while the one before ends, whose results it waits for
// itself. (A call's first launch is an ordinary one: all that came before is done.)
template <typename... P, typename... A>
int behind(void (*kernel)(P...), dim3 ctas, int threads, int bytes, cudaStream_t st, A... args) {
    return cuda_check(launch_pdl(kernel, ctas, dim3(threads), bytes, st, args...), "linear_attention launch");
}

// Whether each chunk's sum gets a CTA: where the heads alone leave SMs idle. (The
// sums cost a write and a read of a state in fp32 for each chunk; one prompt of 8192
// tokens and 12 heads of 128 otherwise waits for 128 chunks, one after the other. 2048 tokens
// of 64, walked or apart: bf16 48 heads 66 and 43 us, 74 72 and 55, 148 90 and 100, 296 143
// and 193; fp32 74 heads 244 and 154, 148 340 and 293, 192 422 and 373, 296 557 and 565. Of
// 128 in bf16: 74 heads 193 and 168, 148 248 and 311. Gradients in bf16, of twice as many
// walks: 48 heads 185 and 156, 74 220 and 221, 148 340 and 410.)
void cut(Job* j, int C, int passes) {
    j->chunks = (j->T + C - 1) / C;
    j->apart = j->chunks > 1 && (long long)j->B * j->H * passes < 148;
}

constexpr int kGateParts = 64;

// The workspace, in bytes from its start (each a multiple of 256).
struct Space {
    long long sums, factor, back, back_factor, decays, kept, kept_back, dq32, dk32, dg, gates, bytes;
};
long long up(long long n) { return (n + 255) / 256 * 256; }

template <class S_>
Space space_of(const Job& j, bool back, bool gates_alike) {
    Space s = {};
    const long long bh = (long long)j.B * j.H, plane = bh * j.chunks * S_::KD * S_::VD * 2;
    long long at = 0;
    const auto take = [&](long long bytes) {
        const long long a = at;
        at += up(bytes);
        return a;
    };
    for (int i = 0; i < 1 + back; ++i)
        if (j.apart) {
            (i ? s.back : s.sums) = take(plane * 2);
            (i ? s.back_factor : s.factor) = take(bh * j.chunks * 4);
        }
    s.decays = take(bh * j.chunks * sizeof(Decays<S_::C>));
    s.kept = take(plane * (back ? 3 : S_::NP));
    if (back) {
        s.kept_back = take(plane * 3);
        if (j.share > 1) {
            s.dq32 = take(bh * j.T * j.dk * 4);
            s.dk32 = take(bh * j.T * j.dk * 4);
        }
        if (gates_alike) {
            s.dg = take(bh * j.T * 4);
            s.gates = take((long long)kGateParts * j.H * 8);
        }
    }
    s.bytes = at;
    return s;
}

// The states that the chunks need.
template <class S_, int PN>
int states(const Job& j, const Pass& p0, const Pass& p1, bool both, Decays<S_::C>* dec, cudaStream_t st) {
    const long long bh = (long long)j.B * j.H;
    constexpr int threads = S_::ST + 32, bytes = Sizes<S_>::state, SIZE = S_::KD * S_::VD;
    static_assert(bytes <= 180 * 1024, "shared memory of a CTA");
    if (j.apart) {
        auto* sum = state_kernel<S_, false, PN>;
        SN_TRY(allow(sum, Sizes<S_>::sum, "linear_attention"));
        sum<<<dim3((unsigned)(bh * j.chunks), 1 + both), threads, Sizes<S_>::sum, st>>>(j, p0, p1, dec);
        // (not launched early: where CTAs of the sums leave first, it would crowd, 10 us instead of 5)
        scan_kernel<S_::KD, S_::VD, S_::C, PN>
            <<<dim3((unsigned)((bh * SIZE / 4 + 255) / 256), 1 + both), 256, 0, st>>>(j, p0, p1);
    } else {
        auto* keep = state_kernel<S_, true, PN>;
        SN_TRY(allow(keep, bytes, "linear_attention"));
        keep<<<dim3((unsigned)bh, 1 + both), threads, bytes, st>>>(j, p0, p1, dec);
    }
    return cuda_check(cudaGetLastError(), "linear_attention launch");
}

int check_space(const Job& j, const Space& s, const char* what, const char* ws, long long ws_bytes) {
    if (s.bytes > ws_bytes || (s.bytes && !ws))
        return fail(SN_E_INVAL, "%s: a workspace of %lld bytes is wanted", what, s.bytes);
    if ((long long)j.B * j.H * j.chunks > 0x7fffffffll)
        return fail(SN_E_INVAL, "%s: too many chunks", what);
    return SN_OK;
}

template <class S_>
int forward_as(Job j, const float* first, void* out, float* state_out, char* ws, long long ws_bytes, long long* need,
            cudaStream_t st) {
    cut(&j, S_::C, 1);
    const Space s = space_of<S_>(j, false, false);
    if (need) {
        *need = s.bytes;
        return SN_OK;
    }
    SN_TRY(check_space(j, s, "linear_attention", ws, ws_bytes));
    Pass p = {j.k, j.v, j.ks, j.vs};
    p.start = first;
    p.sums = reinterpret_cast<float*>(ws + s.sums), p.factor = reinterpret_cast<float*>(ws + s.factor);
    p.kept = reinterpret_cast<bf16*>(ws + s.kept);
    p.end = state_out;
    auto* dec = reinterpret_cast<Decays<S_::C>*>(ws + s.decays);
    SN_TRY((states<S_, S_::NP>(j, p, p, false, dec, st)));
    if (!j.chunks) return SN_OK;
    constexpr int bytes = Sizes<S_>::out;
    static_assert(bytes <= 220 * 1024, "shared memory of a CTA");
    auto* kernel = out_kernel<S_, bytes <= 40 * 1024 ? 5 : bytes <= 72 * 1024 ? 3 : bytes <= 96 * 1024 ? 2 : 1>;
    SN_TRY(allow(kernel, bytes, "linear_attention"));
    return behind(kernel, dim3((unsigned)((long long)j.B * j.H * j.chunks)), S_::THREADS, bytes, st, j, p.kept, dec, out);
}

template <class S_>
int backward_as(Job j, const float* first, const Wanted& g, char* ws, long long ws_bytes, long long* need,
             cudaStream_t st) {
    typedef typename S_::T T;
    cut(&j, S_::C, 2);
    const Space s = space_of<S_>(j, true, g.gates_alike);
    if (need) {
        *need = s.bytes;
        return SN_OK;
    }
    SN_TRY(check_space(j, s, "linear_attention_bwd", ws, ws_bytes));
    const auto floats = [&](long long at) { return reinterpret_cast<float*>(ws + at); };
    Pass p = {j.k, j.v, j.ks, j.vs}, r = {j.q, g.dout, j.qs, g.ds};
    p.start = first, r.start = g.dstate_out;
    p.sums = floats(s.sums), p.factor = floats(s.factor);
    p.kept = reinterpret_cast<bf16*>(ws + s.kept);
    r.sums = floats(s.back), r.factor = floats(s.back_factor);
    r.kept = reinterpret_cast<bf16*>(ws + s.kept_back);
    r.end = g.dstate;
    r.back = true;
    auto* dec = reinterpret_cast<Decays<S_::C>*>(ws + s.decays);
    SN_TRY((states<S_, 3>(j, p, r, true, dec, st)));
    Grads G = {};
    G.dout = g.dout, G.ds = g.ds;
    G.before = p.kept, G.behind = r.kept;
    G.dq = g.dq, G.dk = g.dk, G.dv = g.dv;
    if (j.share > 1) G.dq32 = floats(s.dq32), G.dk32 = floats(s.dk32);
    G.dg = !g.dg ? nullptr : g.gates_alike ? floats(s.dg) : g.dg;
    constexpr int bytes = Sizes<S_>::grad;
    static_assert(bytes <= 220 * 1024, "shared memory of a CTA");
    auto* kernel = grad_kernel<S_, bytes <= 66 * 1024 ? 3 : bytes <= 102 * 1024 ? 2 : 1>;
    SN_TRY(allow(kernel, bytes, "linear_attention_bwd"));
    if (j.chunks)
        SN_TRY(behind(kernel, dim3((unsigned)((long long)j.B * j.H * j.chunks)), S_::THREADS, bytes, st, j, G, dec));
    const long long rows = (long long)j.B * j.T;
    if (j.share > 1 && rows) {
        const long long n = rows * (j.H / j.share) * j.dk;
        SN_TRY(behind(fold_kernel<T>, dim3((unsigned)std::min((n + 255) / 256, 8ll * 148), 2), 256, 0, st, G.dq32, G.dk32,
                      static_cast<T*>(g.dq), static_cast<T*>(g.dk), j.share, j.dk, n));
    }
    if (g.dg && g.gates_alike) {
        double* parts = reinterpret_cast<double*>(ws + s.gates);
        const unsigned ys = (unsigned)std::min(j.H, 65535);
        SN_TRY(behind(gate_kernel, dim3(kGateParts, ys), 256, 0, st, G.dg, nullptr, parts, nullptr, rows, j.H, 0));
        SN_TRY(behind(gate_kernel, dim3(1, ys), 256, 0, st, nullptr, parts, nullptr, g.dg, 0, j.H, kGateParts));
    }
    return SN_OK;
}

// The widths that the keys and the values are laid out in, and the tokens of a
// chunk: 64, but where the tiles and a state of two or three parts would not fit.
template <typename T, typename F>
int by_width(const Job& j, F&& f) {
    if (j.dk <= 64) return j.dv <= 64 ? f(Shape<T, 64, 64, 64>()) : f(Shape<T, 64, 128, 64>());
    return j.dv <= 64 ? f(Shape<T, 128, 64, 64>()) : f(Shape<T, 128, 128, planes_of<T> == 1 ? 64 : 32>());
}

}  // namespace

template <typename T>
int forward(const Job& j, const float* first, void* out, float* state_out, char* ws, long long ws_bytes,
            long long* need, cudaStream_t st) {
    return by_width<T>(j, [&](auto s) {
        return forward_as<decltype(s)>(j, first, out, state_out, ws, ws_bytes, need, st);
    });
}

template <typename T>
int backward(const Job& j, const float* first, const Wanted& w, char* ws, long long ws_bytes, long long* need,
             cudaStream_t st) {
    return by_width<T>(j, [&](auto s) { return backward_as<decltype(s)>(j, first, w, ws, ws_bytes, need, st); });
}

}  // namespace la
}  // namespace sn
