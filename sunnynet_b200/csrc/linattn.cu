// Linear attention with a decay for each head (no counterpart among the
// reference's kernels; its baselines leave it to torch):
//
//   S_t = 2^(g_t) S_(t-1) + k_t v_t^T      (dk x dv, fp32)      o_t = scale S_t^T q_t
//
// in chunks of C tokens. With c_t the sum of a chunk's log decays g up to t and
// S the state before the chunk,
//
//   o_t  = scale (2^(c_t) S^T q_t + sum over s <= t of 2^(c_t - c_s) (q_t . k_s) v_s)
//   S'   = 2^(c_C) S + sum over s of 2^(c_C - c_s) k_s v_s^T
//
// and for the gradients, with R that of the state behind the chunk,
//
//   dq_t = scale (2^(c_t) S do_t + sum over s <= t of 2^(c_t - c_s) (do_t . v_s) k_s)
//   dk_s = 2^(c_C - c_s) R v_s   + scale sum over t >= s of 2^(c_t - c_s) (do_t . v_s) q_t
//   dv_s = 2^(c_C - c_s) R^T k_s + scale sum over t >= s of 2^(c_t - c_s) (q_t . k_s) do_t
//   R'   = 2^(c_C) R + scale sum over t of 2^(c_t) q_t do_t^T
//   dg_t = 2^(c_C) <R, S> + sum over u >= t of q_u . (its dq from S) + sum over s < t of
//          k_s . (its dk from R) + sum over u >= t > s of scale 2^(c_u - c_s) (q_u . k_s) (do_u . v_s)
//
// (dg sums only what passes token t's gate: the shorter form by differences
// q.dq - k.dk from the sequence's end loses all digits over long sequences.)
//
// All products are m16n8k16 matrix instructions on bf16 with fp32 sums. bf16
// values are taken as they are; float16 and float32 ones, and what is computed
// on the way to an fp32 result (the states, dg), as the sum of two bf16 (2^-17
// of a value), three products for one. What goes to a 16-bit output alone is
// rounded to one. The state stays in registers from chunk to chunk, a warp
// holding 16 rows of it. tcgen05 was not taken: with heads of 64 its products
// here have 64 columns, and an instruction of 128 x 64 x 16 takes as long as one
// of 128 x 128 x 16 (90 cycles); the 24 that a chunk of 128 tokens needs would
// fill three quarters of the time that HBM leaves it, while the decays need the
// scores in registers and the state rounded anew for each chunk.
#include <algorithm>
#include <cmath>

#include "caller.cuh"
#include "linattn.cuh"
#include "runtime.cuh"

namespace sn {
namespace la {
namespace {

struct Strides {
    long long b, t, h;
};

struct Job {
    const void *q, *k, *v;
    Strides qs, ks, vs, gs;
    const float* g;
    const int* lengths;
    int B, T, H, share, dk, dv;
    float scale;
    int whole;  // bit 0: q, 1: k, 2: v, 3: dout come in whole packs
    int nseg, per_seg;  // parts of a sequence that run side by side, and their chunks
};

// What one CTA works on.
struct Place {
    int b, h, seg, end, c0, c1, live;  // chunks [c0, c1), those from `live` on lie behind the sequence's end
    long long bh;
    template <int C>
    __device__ __forceinline__ static Place of(const Job& j) {
        Place p;
        p.seg = blockIdx.x % j.nseg;
        p.bh = blockIdx.x / j.nseg;
        p.b = (int)(p.bh / j.H);
        p.h = (int)(p.bh % j.H);
        p.end = j.T;
        if (j.lengths) p.end = max(0, min(j.T, j.lengths[p.b]));
        const int n = (j.T + C - 1) / C;
        p.c0 = min(n, p.seg * j.per_seg);
        p.c1 = min(n, p.c0 + j.per_seg);
        p.live = max(p.c0, min(p.c1, (p.end + C - 1) / C));
        return p;
    }
};

template <typename T>
__device__ __forceinline__ const T* head_of(const void* x, const Strides& s, int b, int h) {
    return static_cast<const T*>(x) + b * s.b + h * s.h;
}

// S += sum over the chunk's tokens of w_t x_t y_t^T: 16 rows (values `row` on
// of x), all columns.
template <int NP, int D, int C>
__device__ __forceinline__ void add_outer(float (*S)[4], const Tile& x, const Tile& y, const float* w,
                                          float scale, int row) {
    const int q = lane_id() & 3;
#pragma unroll
    for (int kt = 0; kt < C / 16; ++kt) {
        uint32_t xr[NP][4], a[2][4];
#pragma unroll
        for (int p = 0; p < NP; ++p) x.a_t(xr[p], kt * 16, row, p);
        float2 f[2];
        f[0] = *reinterpret_cast<const float2*>(w + kt * 16 + 2 * q);
        f[1] = *reinterpret_cast<const float2*>(w + kt * 16 + 2 * q + 8);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float u = low(xr[0][r]), v = high(xr[0][r]);
            if constexpr (NP == 2) u += low(xr[1][r]), v += high(xr[1][r]);
            u *= f[r / 2].x * scale, v *= f[r / 2].y * scale;
            a[0][r] = pack2(u, v);
            a[1][r] = rest2(u, v, a[0][r]);
        }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
            uint32_t b[NP][4];
#pragma unroll
            for (int p = 0; p < NP; ++p) y.b_t(b[p], kt * 16, n * 16, p);
            mma2<2, NP>(S + 2 * n, a, b);
        }
    }
}

// out (16 rows from `ra` of A, columns from `cb` of B) += A B over D: A's rows
// are tokens, B(k, n) = tile[n][k], or tile[k][n] where TRANS.
template <int PA, int PB, int D, int NT, bool TRANS>
__device__ __forceinline__ void product(float (*out)[4], const Tile& A, int ra, const Tile& B, int cb) {
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
            mma2<PA, PB>(out + 2 * n, a, b);
        }
    }
}

// Scores of 16 tokens of A with the blocks [j0, j1) of 16 tokens of B.
template <int NP, int D, int C>
__device__ __forceinline__ void scores(float (*p)[4], const Tile& A, int ra, const Tile& B, int j0, int j1) {
#pragma unroll
    for (int n = 0; n < C / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[n][i] = 0.0f;
#pragma unroll
    for (int kt = 0; kt < D / 16; ++kt) {
        uint32_t a[NP][4];
#pragma unroll
        for (int i = 0; i < NP; ++i) A.a(a[i], ra, kt * 16, i);
#pragma unroll
        for (int j = 0; j < C / 16; ++j)
            if (j >= j0 && j < j1) {
                uint32_t b[NP][4];
#pragma unroll
                for (int i = 0; i < NP; ++i) B.b(b[i], j * 16, kt * 16, i);
                mma2<NP, NP>(p + 2 * j, a, b);
            }
    }
}

// out += P Y, P the scores of blocks [j0, j1) as they lie in registers (PP
// planes of them), Y the tokens' tile.
template <int PP, int NP, int C, int NT>
__device__ __forceinline__ void weighted(float (*out)[4], const float (*p)[4], const Tile& Y, int cb, int j0,
                                         int j1) {
#pragma unroll
    for (int j = 0; j < C / 16; ++j)
        if (j >= j0 && j < j1) {
            uint32_t a[PP][4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float u = p[2 * j + r / 2][r % 2 * 2], v = p[2 * j + r / 2][r % 2 * 2 + 1];
                a[0][r] = pack2(u, v);
                if constexpr (PP == 2) a[1][r] = rest2(u, v, a[0][r]);
            }
#pragma unroll
            for (int n = 0; n < NT / 2; ++n) {
                uint32_t b[NP][4];
#pragma unroll
                for (int i = 0; i < NP; ++i) Y.b_t(b[i], j * 16, cb + n * 16, i);
                mma2<PP, NP>(out + 2 * n, a, b);
            }
        }
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
            if constexpr (NP == 2) {
                const uint32_t w2 = *reinterpret_cast<const uint32_t*>(y + step + n * 8);
                a += low(w2), b += high(w2);
            }
            if (s <= (l >> 2)) out[n][0] += p0 * a, out[n][1] += p0 * b;
            if (s <= (l >> 2) + 8) out[n][2] += p1 * a, out[n][3] += p1 * b;
        }
    }
}

// A state in fp32 (dk, dv) to and from the registers that hold 16 rows of it.
template <int D>
__device__ __forceinline__ void load_state(float (*S)[4], const float* from, int row, int dk, int dv) {
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row + (l >> 2) + (i >> 1) * 8, c = n * 8 + (l & 3) * 2 + (i & 1);
            S[n][i] = from && r < dk && c < dv ? from[r * dv + c] : 0.0f;
        }
}
template <int D>
__device__ __forceinline__ void store_state(const float (*S)[4], float* to, float f, int row, int dk, int dv) {
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row + (l >> 2) + (i >> 1) * 8, c = n * 8 + (l & 3) * 2 + (i & 1);
            if (r < dk && c < dv) to[r * dv + c] = S[n][i] * f;
        }
}

// The same as PN bf16 planes of a tile with rows of LD values.
template <int PN, int D>
__device__ __forceinline__ void state_planes(const float (*S)[4], bf16* to, int row, int ld, int step) {
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            bf16* at = to + (row + (l >> 2) + i * 8) * ld + n * 8 + (l & 3) * 2;
            const uint32_t hi = pack2(S[n][2 * i], S[n][2 * i + 1]);
            *reinterpret_cast<uint32_t*>(at) = hi;
            if constexpr (PN == 2)
                *reinterpret_cast<uint32_t*>(at + step) = rest2(S[n][2 * i], S[n][2 * i + 1], hi);
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

// Rows [t0, t1) of zeros.
template <typename T>
__device__ __forceinline__ void zero_rows(T* to, long long stride, int t0, int t1, int d) {
    for (long long i = threadIdx.x; i < (long long)max(0, t1 - t0) * d; i += blockDim.x)
        to[(t0 + i / d) * stride + i % d] = from_f<T>(0.0f);
}

// The layout of a kernel's shared memory, in bf16 values, and its CTA: as many
// warps as the state has rows of 16; they share the chunk's C / 16 blocks of
// tokens, and the columns of a block where there are more warps than blocks.
template <typename T_, int D_, int C_>
struct Shape {
    typedef T_ T;
    static constexpr int NP = planes_of<T_>, D = D_, C = C_, NW = D / 16, THREADS = NW * 32;
    static constexpr int LD = D + 8, TILE = NP * C * LD, STATE = D * LD;
    static constexpr int RB = C / 16, CG = NW / RB, NT = D / CG / 8;
    static_assert(NW % RB == 0, "whole blocks for the warps");
};

__device__ __forceinline__ Tile tile(const bf16* p, int ld, int step) {
    return {smem_u32(p), (uint32_t)ld * 2, (uint32_t)step * 2};
}

// ------------------------------------------------------------------ states
// The states alone. Without KEEP: what each part of the sequence adds to a
// state of zeros, and its decay (the last part's is not needed). BACK: of
// gradients, x and y being q and dout. With KEEP: the state before every chunk,
// as two planes of D x D, from the parts' starts.
template <class S_, bool KEEP, bool BACK>
__global__ void __launch_bounds__(S_::THREADS)
state_kernel(const Job j, const void* xs, Strides xst, const void* ys, Strides yst, const float* start,
             float* sums, float* factor, bf16* kept) {
    typedef typename S_::T T;
    constexpr int NP = S_::NP, D = S_::D, C = S_::C, LD = S_::LD;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* const sx = reinterpret_cast<bf16*>(smem);
    __shared__ Decays<C> dec;
    const Place at = Place::of<C>(j);
    if (!KEEP && at.seg == (BACK ? 0 : j.nseg - 1)) return;
    const int warp = threadIdx.x >> 5, row = warp * 16;
    const T* x = head_of<T>(xs, xst, at.b, at.h / j.share);
    const T* y = head_of<T>(ys, yst, at.b, at.h);
    const float* g = j.g + at.b * j.gs.b + at.h * j.gs.h;
    const Tile tx = tile(sx, LD, C * LD), ty = tile(sx + S_::TILE, LD, C * LD);
    const int N = (j.T + C - 1) / C;
    const bool wx = j.whole >> (BACK ? 0 : 1) & 1, wy = j.whole >> (BACK ? 3 : 2) & 1;
    float S[D / 8][4];
    load_state<D>(S, KEEP && start ? start + (at.bh * j.nseg + at.seg) * j.dk * j.dv : nullptr, row, j.dk,
                  j.dv);
    float f = 1.0f;
    for (int i = at.c0; i < at.live; ++i) {
        const int c = BACK ? at.live - 1 - (i - at.c0) : i;
        load_tokens<T, C, D, S_::THREADS>(sx, x, xst.t, c * C, at.end, j.dk, wx);
        load_tokens<T, C, D, S_::THREADS>(sx + S_::TILE, y, yst.t, c * C, at.end, j.dv, wy);
        if (warp == 0) decays<C>(&dec, g, j.gs.t, c * C, at.end);
        if constexpr (KEEP)
            state_planes<2, D>(S, kept + (at.bh * N + c) * 2 * D * D, row, D, D * D);
        cp_async_wait_all();
        __syncthreads();
        const float w = dec.whole;
        f *= w;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[n][e] *= w;
        add_outer<NP, D, C>(S, tx, ty, BACK ? dec.from_start : dec.to_end, BACK ? j.scale : 1.0f, row);
        __syncthreads();
    }
    if constexpr (!KEEP) {
        store_state<D>(S, sums + (at.bh * j.nseg + at.seg) * j.dk * j.dv, 1.0f, row, j.dk, j.dv);
        if (threadIdx.x == 0) factor[at.bh * j.nseg + at.seg] = f;
    }
}

// From what each part adds, in place, the state that each starts with (BACK:
// the state's gradient at its end), `first` being the sequence's.
template <bool BACK>
__global__ void __launch_bounds__(256) join_kernel(float* sums, const float* factor, const float* first,
                                                   int nseg, long long size, long long total) {
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    if (i >= total) return;
    const long long bh = i / size;
    float* at = sums + bh * nseg * size + i % size;
    const float* f = factor + bh * nseg;
    float S = first ? first[i] : 0.0f;
#pragma unroll 8
    for (int k = 0; k < nseg; ++k) {
        const int s = BACK ? nseg - 1 - k : k;
        const bool last = k == nseg - 1;
        const float add = last ? 0.0f : at[s * size];
        at[s * size] = S;
        S = (last ? 0.0f : f[s]) * S + add;
    }
}

// ----------------------------------------------------------------- outputs
template <class S_>
__global__ void __launch_bounds__(S_::THREADS)
out_kernel(const Job j, const float* start, void* out_, float* state_out) {
    typedef typename S_::T T;
    constexpr int NP = S_::NP, D = S_::D, C = S_::C, LD = S_::LD, NT = S_::NT;
    constexpr int BUFS = NP == 1 ? 2 : 1;  // bf16 tiles are copied while the chunk before is worked on
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* const sq = reinterpret_cast<bf16*>(smem);
    bf16* const ss = sq + BUFS * 3 * S_::TILE;
    __shared__ Decays<C> dec_[BUFS];
    const Place at = Place::of<C>(j);
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, row = warp * 16;
    const int rb = warp % S_::RB, cb = warp / S_::RB * NT * 8;
    const T* q = head_of<T>(j.q, j.qs, at.b, at.h / j.share);
    const T* k = head_of<T>(j.k, j.ks, at.b, at.h / j.share);
    const T* v = head_of<T>(j.v, j.vs, at.b, at.h);
    const float* g = j.g + at.b * j.gs.b + at.h * j.gs.h;
    const long long ot = (long long)j.H * j.dv;
    T* out = static_cast<T*>(out_) + (long long)at.b * j.T * ot + (long long)at.h * j.dv;

    const auto load = [&](int c, int buf) {
        bf16* to = sq + buf * 3 * S_::TILE;
        load_tokens<T, C, D, S_::THREADS>(to, q, j.qs.t, c * C, at.end, j.dk, j.whole & 1);
        load_tokens<T, C, D, S_::THREADS>(to + S_::TILE, k, j.ks.t, c * C, at.end, j.dk, j.whole >> 1 & 1);
        load_tokens<T, C, D, S_::THREADS>(to + 2 * S_::TILE, v, j.vs.t, c * C, at.end, j.dv,
                                          j.whole >> 2 & 1);
        if (warp == 0) decays<C>(&dec_[buf], g, j.gs.t, c * C, at.end);
    };

    float S[D / 8][4];
    load_state<D>(S, start ? start + (at.bh * j.nseg + at.seg) * j.dk * j.dv : nullptr, row, j.dk, j.dv);
    if (at.c0 < at.live) load(at.c0, 0);
    state_planes<NP, D>(S, ss, row, LD, S_::STATE);
    for (int c = at.c0; c < at.live; ++c) {
        const int buf = BUFS == 2 ? (c - at.c0) & 1 : 0;
        cp_async_wait_all();
        __syncthreads();
        if (BUFS == 2 && c + 1 < at.live) load(c + 1, buf ^ 1);
        const bf16* from = sq + buf * 3 * S_::TILE;
        const Tile tq = tile(from, LD, C * LD), tk = tile(from + S_::TILE, LD, C * LD),
                   tv = tile(from + 2 * S_::TILE, LD, C * LD), ts = tile(ss, LD, S_::STATE);
        const Decays<C>& dec = dec_[buf];

        float P[C / 8][4], O[NT][4];
        scores<NP, D, C>(P, tq, rb * 16, tk, 0, rb + 1);
        const int t = rb * 16 + (l >> 2);
        {
            const float n0 = dec.near[t], n1 = dec.near[t + 8], f0 = dec.far[t], f1 = dec.far[t + 8];
#pragma unroll
            for (int n = 0; n < C / 8; ++n)
                if (n < 2 * (rb + 1)) {
                    const int s = n * 8 + (l & 3) * 2;
                    const float2 nn = *reinterpret_cast<const float2*>(dec.near + s);
                    const float2 ff = *reinterpret_cast<const float2*>(dec.far + s);
                    const float e0 = exp2_of(n0 - nn.x + (f0 - ff.x)), e1 = exp2_of(n0 - nn.y + (f0 - ff.y));
                    const float e2 = exp2_of(n1 - nn.x + (f1 - ff.x)), e3 = exp2_of(n1 - nn.y + (f1 - ff.y));
                    P[n][0] = s <= t ? P[n][0] * (e0 * j.scale) : 0.0f;
                    P[n][1] = s + 1 <= t ? P[n][1] * (e1 * j.scale) : 0.0f;
                    P[n][2] = s <= t + 8 ? P[n][2] * (e2 * j.scale) : 0.0f;
                    P[n][3] = s + 1 <= t + 8 ? P[n][3] * (e3 * j.scale) : 0.0f;
                }
        }
        const float r0 = dec.from_start[t] * j.scale, r1 = dec.from_start[t + 8] * j.scale;
        const auto before = [&] {  // what the state gives
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) O[n][i] = 0.0f;
            product<NP, NP, D, NT, true>(O, tq, rb * 16, ts, cb);
#pragma unroll
            for (int n = 0; n < NT; ++n) O[n][0] *= r0, O[n][1] *= r0, O[n][2] *= r1, O[n][3] *= r1;
        };
        before();
        weighted<NP, NP, C, NT>(O, P, tv, cb, 0, rb + 1);
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum = fmaf(O[n][i], 0.0f, sum);
        if (__any_sync(0xffffffffu, sum != 0.0f)) {  // a NaN or an infinity
            before();
            weighted<NP, NP, C, NT>(O, P, tv, cb, 0, rb);
#pragma unroll
            for (int i = 0; i < C / 16; ++i)
                if (i == rb)
                    weighted_apart<NP, NT>(O, P + 2 * i, from + 2 * S_::TILE + i * 16 * LD, LD, C * LD, cb);
        }
        store_rows<T, NT>(O, out, ot, c * C + rb * 16, cb, at.end, j.T, j.dv);

        const float w = dec.whole;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) S[n][i] *= w;
        add_outer<NP, D, C>(S, tk, tv, dec.to_end, 1.0f, row);
        __syncthreads();
        if (c + 1 < at.live) {
            state_planes<NP, D>(S, ss, row, LD, S_::STATE);
            if (BUFS == 1) load(c + 1, 0);
        }
    }
    zero_rows(out, ot, max(at.live, at.c0) * C, min(at.c1 * C, j.T), j.dv);
    if (at.seg == j.nseg - 1) store_state<D>(S, state_out + at.bh * j.dk * j.dv, 1.0f, row, j.dk, j.dv);
}

// ---------------------------------------------------------------- gradients
struct Grads {
    const void* dout;
    Strides ds;
    const bf16* kept;   // the states before the chunks
    const float* end;   // the state's gradient at each part's end, or null
    void *dq, *dk, *dv;
    float *dq32, *dk32;  // in place of dq, dk: each head's own, where heads share q and k
    float* dg;           // (B, T, H), or null
    float* dstate;       // or null
};

// A row of 16-bit pairs (or two planes of them) times a block of products: each
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
            if constexpr (NP == 2) {
                const uint32_t w2 = *reinterpret_cast<const uint32_t*>(at + step + n * 8);
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

template <class S_>
__global__ void __launch_bounds__(S_::THREADS)
grad_kernel(const Job j, const Grads G) {
    typedef typename S_::T T;
    constexpr int NP = S_::NP, D = S_::D, C = S_::C, LD = S_::LD, NT = S_::NT, RB = S_::RB, CG = S_::CG;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* const sq = reinterpret_cast<bf16*>(smem);
    bf16 *const sk = sq + S_::TILE, *const sv = sk + S_::TILE, *const so = sv + S_::TILE;
    bf16 *const ss = so + S_::TILE, *const sr = ss + 2 * S_::STATE;
    __shared__ Decays<C> dec;
    // parts of dg: by row block, and by column group where the columns are split
    __shared__ float col_part[RB][C], row_part[C], dq_part[CG][C], dk_part[CG][C], dot_part[S_::NW];
    const Place at = Place::of<C>(j);
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, row = warp * 16;
    const int rb = warp % RB, cg = warp / RB, cb = cg * NT * 8;
    const T* q = head_of<T>(j.q, j.qs, at.b, at.h / j.share);
    const T* k = head_of<T>(j.k, j.ks, at.b, at.h / j.share);
    const T* v = head_of<T>(j.v, j.vs, at.b, at.h);
    const T* dout = head_of<T>(G.dout, G.ds, at.b, at.h);
    const float* g = j.g + at.b * j.gs.b + at.h * j.gs.h;
    const long long kt = (long long)j.H * j.dk, vt = (long long)j.H * j.dv;
    const long long k0 = (long long)at.b * j.T * kt + (long long)at.h * j.dk;
    T* dv = static_cast<T*>(G.dv) + (long long)at.b * j.T * vt + (long long)at.h * j.dv;
    const int N = (j.T + C - 1) / C;
    const Tile tq = tile(sq, LD, C * LD), tk = tile(sk, LD, C * LD), tv = tile(sv, LD, C * LD),
               to = tile(so, LD, C * LD), ts = tile(ss, LD, S_::STATE), tr = tile(sr, LD, S_::STATE);

    const auto load = [&](int c) {
        load_tokens<T, C, D, S_::THREADS>(sq, q, j.qs.t, c * C, at.end, j.dk, j.whole & 1);
        load_tokens<T, C, D, S_::THREADS>(sk, k, j.ks.t, c * C, at.end, j.dk, j.whole >> 1 & 1);
        load_tokens<T, C, D, S_::THREADS>(sv, v, j.vs.t, c * C, at.end, j.dv, j.whole >> 2 & 1);
        load_tokens<T, C, D, S_::THREADS>(so, dout, G.ds.t, c * C, at.end, j.dv, j.whole >> 3 & 1);
        const bf16* from = G.kept + (at.bh * N + c) * 2 * D * D;
#pragma unroll
        for (int n = 0; n < 2 * D * D / 8 / S_::THREADS; ++n) {
            const int i = n * S_::THREADS + threadIdx.x;
            cp_async16(ss + i / (D * D / 8) * S_::STATE + i % (D * D / 8) / (D / 8) * LD + i % (D / 8) * 8,
                       from + i * 8, 16);
        }
        if (warp == 0) decays<C>(&dec, g, j.gs.t, c * C, at.end);
    };
    const auto store_head = [&](const float(*x)[4], void* to16, float* to32, int t0) {
        if (to32)
            store_rows<float, NT>(x, to32 + k0, kt, t0, cb, at.end, j.T, j.dk);
        else
            store_rows<T, NT>(x, static_cast<T*>(to16) + k0, kt, t0, cb, at.end, j.T, j.dk);
    };

    float R[D / 8][4];
    load_state<D>(R, G.end ? G.end + (at.bh * j.nseg + at.seg) * j.dk * j.dv : nullptr, row, j.dk, j.dv);
    if (at.c0 < at.live) load(at.live - 1);
    state_planes<2, D>(R, sr, row, LD, S_::STATE);
    for (int c = at.live - 1; c >= at.c0; --c) {
        cp_async_wait_all();
        __syncthreads();
        float X[NT][4], part[2];
        const int t = rb * 16 + (l >> 2);  // the lane's tokens: this and 8 behind
        const float n0 = dec.near[t], n1 = dec.near[t + 8], f0 = dec.far[t], f1 = dec.far[t + 8];
        const float b0 = dec.to_end[t], b1 = dec.to_end[t + 8];
        const int t0 = c * C + rb * 16;
        {
            // rows s, columns u >= s
            float P[C / 8][4], Q[C / 8][4];
            scores<NP, D, C>(P, tk, rb * 16, tq, rb, RB);
            scores<NP, D, C>(Q, tv, rb * 16, to, rb, RB);
            float across[2] = {0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < C / 8; ++n) {
                float down[2] = {0.0f, 0.0f};
                if (n >= 2 * rb) {
                    const int u = n * 8 + (l & 3) * 2;
                    const float2 nn = *reinterpret_cast<const float2*>(dec.near + u);
                    const float2 ff = *reinterpret_cast<const float2*>(dec.far + u);
                    const float e[4] = {exp2_of(nn.x - n0 + (ff.x - f0)), exp2_of(nn.y - n0 + (ff.y - f0)),
                                        exp2_of(nn.x - n1 + (ff.x - f1)), exp2_of(nn.y - n1 + (ff.y - f1))};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int s = t + (i >> 1) * 8, uu = u + (i & 1);
                        const float p = P[n][i], w = j.scale * e[i];
                        P[n][i] = uu >= s ? p * w : 0.0f;
                        const float a = uu > s ? p * w * Q[n][i] : 0.0f;
                        Q[n][i] = uu >= s ? Q[n][i] * w : 0.0f;
                        across[i >> 1] += a;
                        down[i & 1] += a;
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    down[i] += __shfl_xor_sync(0xffffffffu, down[i], 4);
                    down[i] += __shfl_xor_sync(0xffffffffu, down[i], 8);
                    down[i] += __shfl_xor_sync(0xffffffffu, down[i], 16);
                }
                if (cg == 0 && l < 4) {
                    col_part[rb][n * 8 + l * 2] = down[0];
                    col_part[rb][n * 8 + l * 2 + 1] = down[1];
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                across[i] += __shfl_xor_sync(0xffffffffu, across[i], 1);
                across[i] += __shfl_xor_sync(0xffffffffu, across[i], 2);
            }
            if (cg == 0 && (l & 3) == 0) row_part[t] = across[0], row_part[t + 8] = across[1];

#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) X[n][i] = 0.0f;
            product<NP, NP, D, NT, true>(X, tk, rb * 16, tr, cb);
#pragma unroll
            for (int n = 0; n < NT; ++n) X[n][0] *= b0, X[n][1] *= b0, X[n][2] *= b1, X[n][3] *= b1;
            weighted<NP, NP, C, NT>(X, P, to, cb, rb, RB);
            store_rows<T, NT>(X, dv, vt, t0, cb, at.end, j.T, j.dv);

#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) X[n][i] = 0.0f;
            product<NP, 2, D, NT, false>(X, tv, rb * 16, tr, cb);
#pragma unroll
            for (int n = 0; n < NT; ++n) X[n][0] *= b0, X[n][1] *= b0, X[n][2] *= b1, X[n][3] *= b1;
            row_dots<NP, NT>(X, sk, LD, C * LD, rb * 16, cb, part);
            if ((l & 3) == 0) dk_part[cg][t] = part[0], dk_part[cg][t + 8] = part[1];
            weighted<NP, NP, C, NT>(X, Q, tq, cb, rb, RB);
            store_head(X, G.dk, G.dk32, t0);
        }
        {
            // rows u, columns s <= u
            float Q[C / 8][4];
            scores<NP, D, C>(Q, to, rb * 16, tv, 0, rb + 1);
#pragma unroll
            for (int n = 0; n < C / 8; ++n)
                if (n < 2 * (rb + 1)) {
                    const int s = n * 8 + (l & 3) * 2;
                    const float2 nn = *reinterpret_cast<const float2*>(dec.near + s);
                    const float2 ff = *reinterpret_cast<const float2*>(dec.far + s);
                    const float e[4] = {exp2_of(n0 - nn.x + (f0 - ff.x)), exp2_of(n0 - nn.y + (f0 - ff.y)),
                                        exp2_of(n1 - nn.x + (f1 - ff.x)), exp2_of(n1 - nn.y + (f1 - ff.y))};
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        Q[n][i] = s + (i & 1) <= t + (i >> 1) * 8 ? Q[n][i] * e[i] * j.scale : 0.0f;
                }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) X[n][i] = 0.0f;
            product<NP, 2, D, NT, false>(X, to, rb * 16, ts, cb);
            const float r0 = dec.from_start[t] * j.scale, r1 = dec.from_start[t + 8] * j.scale;
#pragma unroll
            for (int n = 0; n < NT; ++n) X[n][0] *= r0, X[n][1] *= r0, X[n][2] *= r1, X[n][3] *= r1;
            row_dots<NP, NT>(X, sq, LD, C * LD, rb * 16, cb, part);
            if ((l & 3) == 0) dq_part[cg][t] = part[0], dq_part[cg][t + 8] = part[1];
            weighted<NP, NP, C, NT>(X, Q, tk, cb, 0, rb + 1);
            store_head(X, G.dq, G.dq32, t0);
        }
        const float w = dec.whole;
        float dot = 0.0f;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const bf16* s = ss + (row + (l >> 2) + i * 8) * LD + n * 8 + (l & 3) * 2;
                const uint32_t hi = *reinterpret_cast<const uint32_t*>(s);
                const uint32_t lo = *reinterpret_cast<const uint32_t*>(s + S_::STATE);
                dot = fmaf(R[n][2 * i], low(hi) + low(lo), dot);
                dot = fmaf(R[n][2 * i + 1], high(hi) + high(lo), dot);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) R[n][i] *= w;
        }
#pragma unroll
        for (int d = 16; d; d /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (l == 0) dot_part[warp] = dot * w;
        add_outer<NP, D, C>(R, tq, to, dec.from_start, j.scale, row);
        __syncthreads();
        if (warp == 0 && G.dg) {
            // behind: sum over u >= t of (rho_u + r_u) - sum over s >= t of kappa_s; ahead: sum over s < t of l_s
            constexpr int M = C / 32;
            float behind[M], ahead[M], all = 0.0f, b = 0.0f, a = 0.0f;
#pragma unroll
            for (int i = 0; i < S_::NW; ++i) all += dot_part[i];
#pragma unroll
            for (int i = M - 1; i >= 0; --i) {
                const int u = l * M + i;
                float x = -row_part[u];
#pragma unroll
                for (int r = 0; r < RB; ++r)
                    if (r <= u / 16) x += col_part[r][u];
#pragma unroll
                for (int r = 0; r < CG; ++r) x += dq_part[r][u];
                behind[i] = b += x;
            }
#pragma unroll
            for (int i = 0; i < M; ++i) {
                ahead[i] = a;
#pragma unroll
                for (int r = 0; r < CG; ++r) a += dk_part[r][l * M + i];
            }
            float bs = b, as = a;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const float y = __shfl_down_sync(0xffffffffu, bs, d), z = __shfl_up_sync(0xffffffffu, as, d);
                if (l + d < 32) bs += y;
                if (l >= d) as += z;
            }
            bs -= b, as -= a;
#pragma unroll
            for (int i = 0; i < M; ++i) {
                const int u = c * C + l * M + i;
                if (u < j.T)
                    G.dg[((long long)at.b * j.T + u) * j.H + at.h] =
                        u < at.end ? all + behind[i] + bs + ahead[i] + as : 0.0f;
            }
        }
        if (c > at.c0) {
            state_planes<2, D>(R, sr, row, LD, S_::STATE);
            __syncwarp();
            load(c - 1);
        }
    }
    const int z0 = max(at.live, at.c0) * C, z1 = min(at.c1 * C, j.T);
    zero_rows(dv, vt, z0, z1, j.dv);
    if (G.dq32) {
        zero_rows(G.dq32 + k0, kt, z0, z1, j.dk);
        zero_rows(G.dk32 + k0, kt, z0, z1, j.dk);
    } else {
        zero_rows(static_cast<T*>(G.dq) + k0, kt, z0, z1, j.dk);
        zero_rows(static_cast<T*>(G.dk) + k0, kt, z0, z1, j.dk);
    }
    if (G.dg)
        zero_rows(G.dg + (long long)at.b * j.T * j.H + at.h, j.H, z0, z1, 1);
    if (G.dstate && at.seg == 0)
        store_state<D>(R, G.dstate + at.bh * j.dk * j.dv, 1.0f, row, j.dk, j.dv);
}

// Sums over the heads that share one of q and k.
template <typename T>
__global__ void __launch_bounds__(256) fold_kernel(const float* x, const float* y, T* to_x, T* to_y,
                                                   int share, int d, long long n) {
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

// -------------------------------------------------------------- single token
// A CTA for each sequence and head: its state goes through once. Lanes stand
// side by side along a row of the state, so that every access is one run.
template <typename T, int VEC>
__global__ void __launch_bounds__(128)
step_kernel(const T* q_, const T* k_, const T* v_, Strides qs, Strides ks, Strides vs, const float* g,
            long long gb, long long gh, float* state, long long sb, T* out, int H, int share, int dk, int dv,
            float scale) {
    __shared__ float sq[128], sk[128];
    __shared__ float part[128 * VEC];
    const int b = blockIdx.x / H, h = blockIdx.x % H, tid = threadIdx.x;
    const T* q = q_ + b * qs.b + h / share * qs.h;
    const T* k = k_ + b * ks.b + h / share * ks.h;
    const T* v = v_ + b * vs.b + h * vs.h;
    float* S = state + b * sb + (long long)h * dk * dv;
    const int packs = dv / VEC;
    int lanes = 1;  // of a row
    while (lanes < packs) lanes *= 2;
    const int rows = 128 / lanes, r0 = tid / lanes, c = tid % lanes;
    const bool in = c < packs;
    if (tid < dk) {
        sq[tid] = to_f(q[tid]) * scale;
        sk[tid] = to_f(k[tid]);
    }
    const double gate = (double)g[b * gb + h * gh] * 1.4426950408889634074;
    const float f = exp2_of(gate < -256.0 ? -256.0f : (float)gate);
    float x[VEC], o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        x[i] = in ? to_f(v[c * VEC + i]) : 0.0f;
        o[i] = 0.0f;
    }
    __syncthreads();
    if (in) {
        constexpr int U = 8;
        for (int r = r0; r < dk; r += rows * U) {
            float s[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * rows < dk) {
                    const float* at = S + (r + u * rows) * dv + c * VEC;
                    if constexpr (VEC == 4) {
                        const float4 y = *reinterpret_cast<const float4*>(at);
                        s[u][0] = y.x, s[u][1] = y.y, s[u][2] = y.z, s[u][3] = y.w;
                    } else {
                        s[u][0] = *at;
                    }
                }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * rows < dk) {
                    const float kk = sk[r + u * rows], qq = sq[r + u * rows];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        s[u][i] = fmaf(kk, x[i], f * s[u][i]);
                        o[i] = fmaf(qq, s[u][i], o[i]);
                    }
                    float* at = S + (r + u * rows) * dv + c * VEC;
                    if constexpr (VEC == 4)
                        *reinterpret_cast<float4*>(at) = make_float4(s[u][0], s[u][1], s[u][2], s[u][3]);
                    else
                        *at = s[u][0];
                }
        }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) part[(r0 * lanes + c) * VEC + i] = o[i];
    __syncthreads();
    for (int i = tid; i < dv; i += 128) {
        float y = 0.0f;
        for (int r = 0; r < rows; ++r) y += part[(r * lanes + i / VEC) * VEC + i % VEC];
        out[((long long)b * H + h) * dv + i] = from_f<T>(y);
    }
}

// ------------------------------------------------------------------ launches
constexpr int kMaxHead = 128;

template <class S_>
struct Sizes {
    static constexpr int out = (S_::NP == 1 ? 6 : 3) * S_::TILE * 2 + S_::NP * S_::STATE * 2;
    static constexpr int state = 2 * S_::TILE * 2;
    static constexpr int grad = 4 * S_::TILE * 2 + 4 * S_::STATE * 2;
};

template <typename K>
int allow(K* kernel, int bytes, const char* what) {
    return cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
}

// Parts of a sequence side by side: enough CTAs for `per_sm` on every SM, none
// shorter than four chunks (the states of its start cost a pass over the keys
// and values, half of what the outputs read).
void split(Job* j, int C, int sms, int per_sm) {
    const int n = (j->T + C - 1) / C;
    const long long heads = (long long)j->B * j->H;
    long long parts = heads ? ((long long)sms * per_sm) / heads : 1;
    parts = std::max(1ll, std::min(parts, (long long)n / 4));
    j->per_seg = std::max(1, (int)((n + parts - 1) / parts));
    j->nseg = std::max(1, (n + j->per_seg - 1) / j->per_seg);
}

constexpr int kGateParts = 64;

// The workspace, in bytes from its start (each a multiple of 256).
struct Space {
    long long sums, factor, back, back_factor, kept, dq32, dk32, dg, gates, bytes;
};
long long up(long long n) { return (n + 255) / 256 * 256; }

template <class S_>
Space space_of(const Job& j, bool back, bool gates_alike) {
    Space s = {};
    const long long bh = (long long)j.B * j.H, n = (j.T + S_::C - 1) / S_::C;
    long long at = 0;
    const auto take = [&](long long bytes) {
        const long long a = at;
        at += up(bytes);
        return a;
    };
    if (j.nseg > 1) {
        s.sums = take(bh * j.nseg * j.dk * j.dv * 4);
        s.factor = take(bh * j.nseg * 4);
    }
    if (back) {
        if (j.nseg > 1) {
            s.back = take(bh * j.nseg * j.dk * j.dv * 4);
            s.back_factor = take(bh * j.nseg * 4);
        }
        s.kept = take(bh * n * 2 * S_::D * S_::D * 2);
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

template <class S_, bool BACK>
int starts(const Job& j, const void* x, const Strides& xs, const void* y, const Strides& ys, const float* first,
           float* sums, float* factor, cudaStream_t st) {
    const long long bh = (long long)j.B * j.H, size = (long long)j.dk * j.dv;
    auto* kernel = state_kernel<S_, false, BACK>;
    SN_TRY(allow(kernel, Sizes<S_>::state, "linear_attention"));
    kernel<<<(unsigned)(bh * j.nseg), S_::THREADS, Sizes<S_>::state, st>>>(j, x, xs, y, ys, nullptr, sums,
                                                                           factor, nullptr);
    join_kernel<BACK><<<(unsigned)((bh * size + 255) / 256), 256, 0, st>>>(sums, factor, first, j.nseg, size,
                                                                           bh * size);
    return cuda_check(cudaGetLastError(), "linear_attention launch");
}

template <class S_>
int forward(Job j, int sms, const float* first, void* out, float* state_out, char* ws, long long ws_bytes,
            long long* need, cudaStream_t st) {
    split(&j, S_::C, sms, S_::D == 64 ? 3 : 1);
    const Space s = space_of<S_>(j, false, false);
    if (need) {
        *need = s.bytes;
        return SN_OK;
    }
    if (s.bytes > ws_bytes || (s.bytes && !ws))
        return fail(SN_E_INVAL, "linear_attention: a workspace of %lld bytes is wanted", s.bytes);
    if ((long long)j.B * j.H * j.nseg > 0x7fffffffll) return fail(SN_E_INVAL, "linear_attention: too many heads");
    if (j.nseg > 1) {
        float* sums = reinterpret_cast<float*>(ws + s.sums);
        SN_TRY((starts<S_, false>(j, j.k, j.ks, j.v, j.vs, first, sums,
                                  reinterpret_cast<float*>(ws + s.factor), st)));
        first = sums;
    }
    static_assert(Sizes<S_>::out <= 220 * 1024, "shared memory of a CTA");
    SN_TRY(allow(out_kernel<S_>, Sizes<S_>::out, "linear_attention"));
    out_kernel<S_><<<(unsigned)((long long)j.B * j.H * j.nseg), S_::THREADS, Sizes<S_>::out, st>>>(j, first, out,
                                                                                                  state_out);
    return cuda_check(cudaGetLastError(), "linear_attention launch");
}

struct Wanted {
    const void* dout;
    Strides ds;
    const float* dstate_out;
    void *dq, *dk, *dv;
    float *dg, *dstate;
    bool gates_alike;
};

template <class S_>
int backward(Job j, int sms, const float* first, const Wanted& g, char* ws, long long ws_bytes, long long* need,
             cudaStream_t st) {
    typedef typename S_::T T;
    split(&j, S_::C, sms, S_::D == 64 ? 2 : 1);
    const Space s = space_of<S_>(j, true, g.gates_alike);
    if (need) {
        *need = s.bytes;
        return SN_OK;
    }
    if (s.bytes > ws_bytes || (s.bytes && !ws))
        return fail(SN_E_INVAL, "linear_attention_bwd: a workspace of %lld bytes is wanted", s.bytes);
    if ((long long)j.B * j.H * j.nseg > 0x7fffffffll)
        return fail(SN_E_INVAL, "linear_attention_bwd: too many heads");
    const auto floats = [&](long long at) { return reinterpret_cast<float*>(ws + at); };
    Grads G = {};
    G.dout = g.dout, G.ds = g.ds;
    G.end = g.dstate_out;
    if (j.nseg > 1) {
        SN_TRY((starts<S_, false>(j, j.k, j.ks, j.v, j.vs, first, floats(s.sums), floats(s.factor), st)));
        SN_TRY((starts<S_, true>(j, j.q, j.qs, g.dout, g.ds, g.dstate_out, floats(s.back),
                                 floats(s.back_factor), st)));
        first = floats(s.sums);
        G.end = floats(s.back);
    }
    bf16* kept = reinterpret_cast<bf16*>(ws + s.kept);
    const unsigned ctas = (unsigned)((long long)j.B * j.H * j.nseg);
    auto* keep = state_kernel<S_, true, false>;
    SN_TRY(allow(keep, Sizes<S_>::state, "linear_attention_bwd"));
    keep<<<ctas, S_::THREADS, Sizes<S_>::state, st>>>(j, j.k, j.ks, j.v, j.vs, first, nullptr, nullptr, kept);
    G.kept = kept;
    G.dq = g.dq, G.dk = g.dk, G.dv = g.dv;
    if (j.share > 1) G.dq32 = floats(s.dq32), G.dk32 = floats(s.dk32);
    G.dg = !g.dg ? nullptr : g.gates_alike ? floats(s.dg) : g.dg;
    G.dstate = g.dstate;
    static_assert(Sizes<S_>::grad <= 220 * 1024, "shared memory of a CTA");
    SN_TRY(allow(grad_kernel<S_>, Sizes<S_>::grad, "linear_attention_bwd"));
    grad_kernel<S_><<<ctas, S_::THREADS, Sizes<S_>::grad, st>>>(j, G);
    const long long rows = (long long)j.B * j.T;
    if (j.share > 1 && rows) {
        const long long n = rows * (j.H / j.share) * j.dk;
        fold_kernel<T><<<dim3((unsigned)std::min((n + 255) / 256, 8ll * sms), 2), 256, 0, st>>>(
            G.dq32, G.dk32, static_cast<T*>(g.dq), static_cast<T*>(g.dk), j.share, j.dk, n);
    }
    if (g.dg && g.gates_alike) {
        double* parts = reinterpret_cast<double*>(ws + s.gates);
        const unsigned ys = (unsigned)std::min(j.H, 65535);
        gate_kernel<<<dim3(kGateParts, ys), 256, 0, st>>>(G.dg, nullptr, parts, nullptr, rows, j.H, 0);
        gate_kernel<<<dim3(1, ys), 256, 0, st>>>(nullptr, parts, nullptr, g.dg, 0, j.H, kGateParts);
    }
    return cuda_check(cudaGetLastError(), "linear_attention_bwd launch");
}

// The chunk: 64 tokens; 32 in the gradients of heads above 64 in two planes,
// whose tiles and states fill the shared memory.
template <typename T, bool BACK, typename F>
int by_width(const Job& j, F&& f) {
    if (std::max(j.dk, j.dv) <= 64) return f(Shape<T, 64, 64>());
    return f(Shape<T, 128, BACK && planes_of<T> == 2 ? 32 : 64>());
}
template <bool BACK, typename F>
int by_type(int dtype, const Job& j, F&& f) {
    return dtype == SN_F32    ? by_width<float, BACK>(j, f)
           : dtype == SN_BF16 ? by_width<bf16, BACK>(j, f)
                              : by_width<__half, BACK>(j, f);
}

// Whether loads of whole packs (16 bytes; 8 for float16) are aligned.
bool packs(const void* p, const Strides& s, int d, int dtype, bool one_seq, bool one_head) {
    const int w = dtype == SN_BF16 ? 8 : 4;
    const unsigned bytes = w * dtype_size(dtype);
    return (uintptr_t)p % bytes == 0 && d % w == 0 && s.t % w == 0 && (one_seq || s.b % w == 0) &&
           (one_head || s.h % w == 0);
}

Strides strides(const int64_t* s) { return {s[0], s[1], s[2]}; }

int read_job(const SnAbiLinearAttention* a, const char* what, Job* j) {
    if (!a) return fail(SN_E_INVAL, "%s: null arguments", what);
    if (!dtype_size(a->dtype)) return fail(SN_E_INVAL, "%s: dtype %d", what, a->dtype);
    if (a->B < 0 || a->T < 0 || a->H < 1 || a->Hk < 1 || a->H % a->Hk)
        return fail(SN_E_INVAL, "%s: sizes B %d T %d, heads %d over %d", what, a->B, a->T, a->H, a->Hk);
    if (a->dk < 1 || a->dv < 1 || a->dk > kMaxHead || a->dv > kMaxHead)
        return fail(SN_E_INVAL, "%s: heads have 1 to %d values, not %d and %d", what, kMaxHead, a->dk, a->dv);
    if (a->T > 0x7fffffff - 128 || (long long)a->B * a->H > 0x7fffffffll)
        return fail(SN_E_INVAL, "%s: sizes beyond 31 bits", what);
    if (!std::isfinite(a->scale)) return fail(SN_E_INVAL, "%s: the scale is not finite", what);
    j->q = a->q, j->k = a->k, j->v = a->v, j->g = a->log_decay;
    j->qs = strides(a->q_stride), j->ks = strides(a->k_stride), j->vs = strides(a->v_stride);
    j->gs = strides(a->log_decay_stride);
    j->lengths = a->lengths;
    j->B = a->B, j->T = a->T, j->H = a->H, j->share = a->H / a->Hk, j->dk = a->dk, j->dv = a->dv;
    j->scale = a->scale;
    j->nseg = 1, j->per_seg = 1;
    j->whole = (int)packs(j->q, j->qs, j->dk, a->dtype, a->B < 2, a->Hk < 2) |
               (int)packs(j->k, j->ks, j->dk, a->dtype, a->B < 2, a->Hk < 2) << 1 |
               (int)packs(j->v, j->vs, j->dv, a->dtype, a->B < 2, a->H < 2) << 2;
    return SN_OK;
}

constexpr int kSms = 148;  // of a B200: the split of a sequence does not ask the device

}  // namespace
}  // namespace la
}  // namespace sn

using namespace sn;

extern "C" {

int64_t sn_abi_linear_attention_ws(const SnAbiLinearAttention* a, int32_t backward, int32_t head_gates) {
    la::Job j;
    if (la::read_job(a, "linear_attention_ws", &j) != SN_OK) return -1;
    if (!a->B) return 0;
    long long need = 0;
    if (backward) {
        la::Wanted w = {};
        w.gates_alike = head_gates != 0;
        la::by_type<true>(a->dtype, j, [&](auto s) {
            return la::backward<decltype(s)>(j, la::kSms, nullptr, w, nullptr, 0, &need, nullptr);
        });
    } else {
        la::by_type<false>(a->dtype, j, [&](auto s) {
            return la::forward<decltype(s)>(j, la::kSms, nullptr, nullptr, nullptr, nullptr, 0, &need, nullptr);
        });
    }
    return need;
}

sn_status sn_abi_linear_attention(const SnAbiLinearAttention* a, void* out, float* state_out, void* ws,
                                  int64_t ws_bytes, void* cuda_stream) {
    la::Job j;
    SN_TRY(la::read_job(a, "linear_attention", &j));
    if (!a->B) return SN_OK;
    if (!state_out || (a->T && (!a->log_decay || !a->q || !a->k || !a->v || !out)))
        return fail(SN_E_INVAL, "linear_attention: null pointer");
    const unsigned e = dtype_size(a->dtype);
    CallerDevice dev;
    SN_TRY(dev.enter("linear_attention", {{a->q, e}, {a->k, e}, {a->v, e}, {a->log_decay, 4}, {a->state, 4},
                                          {a->lengths, 4}, {out, e}, {state_out, 4}, {ws, 16}}));
    return la::by_type<false>(a->dtype, j, [&](auto s) {
        return la::forward<decltype(s)>(j, la::kSms, a->state, out, state_out, static_cast<char*>(ws), ws_bytes,
                                        nullptr, static_cast<cudaStream_t>(cuda_stream));
    });
}

sn_status sn_abi_linear_attention_bwd(const SnAbiLinearAttention* a, const void* dout,
                                      const int64_t* dout_stride, const float* dstate_out, void* dq, void* dk,
                                      void* dv, float* dlog_decay, int32_t head_gates, float* dstate, void* ws,
                                      int64_t ws_bytes, void* cuda_stream) {
    la::Job j;
    SN_TRY(la::read_job(a, "linear_attention_bwd", &j));
    if (!a->B) {
        if (dlog_decay && head_gates) return fail(SN_E_INVAL, "linear_attention_bwd: no sequences");
        return SN_OK;
    }
    if (!dout_stride ||
        (a->T && (!a->log_decay || !a->q || !a->k || !a->v || !dout || !dq || !dk || !dv)))
        return fail(SN_E_INVAL, "linear_attention_bwd: null pointer");
    const unsigned e = dtype_size(a->dtype);
    CallerDevice dev;
    SN_TRY(dev.enter("linear_attention_bwd",
                     {{a->q, e}, {a->k, e}, {a->v, e}, {a->log_decay, 4}, {a->state, 4}, {a->lengths, 4},
                      {dout, e}, {dstate_out, 4}, {dq, e}, {dk, e}, {dv, e}, {dlog_decay, 4}, {dstate, 4},
                      {ws, 16}}));
    la::Wanted w = {dout, la::strides(dout_stride), dstate_out, dq, dk, dv, dlog_decay, dstate,
                    head_gates != 0};
    j.whole |= (int)la::packs(dout, w.ds, j.dv, a->dtype, a->B < 2, a->H < 2) << 3;
    return la::by_type<true>(a->dtype, j, [&](auto s) {
        return la::backward<decltype(s)>(j, la::kSms, a->state, w, static_cast<char*>(ws), ws_bytes, nullptr,
                                         static_cast<cudaStream_t>(cuda_stream));
    });
}

sn_status sn_abi_linear_attention_step(const SnAbiLinearAttention* a, float* state, int64_t state_stride,
                                       void* out, void* cuda_stream) {
    la::Job j;
    SN_TRY(la::read_job(a, "linear_attention_step", &j));
    if (a->T != 1) return fail(SN_E_INVAL, "linear_attention_step: one token, not %d", a->T);
    if (!a->B) return SN_OK;
    const long long size = (long long)j.H * j.dk * j.dv;
    if (!a->q || !a->k || !a->v || !a->log_decay || !state || !out)
        return fail(SN_E_INVAL, "linear_attention_step: null pointer");
    if (a->B > 1 && state_stride < size)
        return fail(SN_E_INVAL, "linear_attention_step: states overlap");
    const unsigned e = dtype_size(a->dtype);
    CallerDevice dev;
    SN_TRY(dev.enter("linear_attention_step",
                     {{a->q, e}, {a->k, e}, {a->v, e}, {a->log_decay, 4}, {state, 4}, {out, e}}));
    const bool four = (uintptr_t)state % 16 == 0 && j.dv % 4 == 0 && (a->B < 2 || state_stride % 4 == 0);
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const auto go = [&](auto t, auto vec) {
        typedef decltype(t) T;
        la::step_kernel<T, decltype(vec)::value><<<(unsigned)((long long)j.B * j.H), 128, 0, st>>>(
            static_cast<const T*>(j.q), static_cast<const T*>(j.k), static_cast<const T*>(j.v), j.qs, j.ks, j.vs,
            j.g, j.gs.b, j.gs.h, state, state_stride, static_cast<T*>(out), j.H, j.share, j.dk, j.dv, j.scale);
        return cuda_check(cudaGetLastError(), "linear_attention_step launch");
    };
    const auto typed = [&](auto t) {
        return four ? go(t, std::integral_constant<int, 4>()) : go(t, std::integral_constant<int, 1>());
    };
    return a->dtype == SN_F32 ? typed(0.0f) : a->dtype == SN_BF16 ? typed(la::bf16()) : typed(__half());
}

}  // extern "C"
