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
    int chunks;         // of a sequence
    int nseg, per_seg;  // parts of a sequence whose states run side by side, and their chunks
};

// Tokens of a sequence, and its chunks that hold some.
__device__ __forceinline__ int tokens_of(const Job& j, int b) {
    return j.lengths ? max(0, min(j.T, j.lengths[b])) : j.T;
}

template <typename T>
__device__ __forceinline__ const T* head_of(const void* x, const Strides& s, int b, int h) {
    return static_cast<const T*>(x) + b * s.b + h * s.h;
}

// S += sum over the tokens of w_t x_t y_t^T: 16 rows (values `row` on of x), NT
// column tiles (values `cb` on of y). x w is taken apart as it is formed: the
// product of the high parts rounded, what that leaves (which bf16 holds exactly),
// and the products with the low parts: 2^-16 of a value, in three or four
// instructions for two.
template <int NP, int NT, int C>
__device__ __forceinline__ void add_outer(float (*S)[4], const Tile& x, const Tile& y, const uint2* w, int row,
                                          int cb) {
    const int q = lane_id() & 3;
#pragma unroll
    for (int kt = 0; kt < C / 16; ++kt) {
        uint32_t xr[NP][4], a[2][4];
#pragma unroll
        for (int p = 0; p < NP; ++p) x.a_t(xr[p], kt * 16, row, p);
        const uint2 f[2] = {w[kt * 8 + q], w[kt * 8 + 4 + q]};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            a[0][r] = fma2(xr[0][r], f[r / 2].x, 0x80008000u);
            a[1][r] = fma2(xr[0][r], f[r / 2].x, neg2(a[0][r]));
            a[1][r] = fma2(xr[0][r], f[r / 2].y, a[1][r]);
            if constexpr (NP == 2) a[1][r] = fma2(xr[1][r], f[r / 2].x, a[1][r]);
        }
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
            uint32_t b[NP][4];
#pragma unroll
            for (int p = 0; p < NP; ++p) y.b_t(b[p], kt * 16, cb + n * 16, p);
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

// Scores of 16 tokens of A with a strip of NB blocks of 16 tokens of B from
// block `jb` on, of which [j0, j1) are wanted.
template <int NP, int D, int NB>
__device__ __forceinline__ void scores(float (*p)[4], const Tile& A, int ra, const Tile& B, int jb, int j0,
                                       int j1) {
#pragma unroll
    for (int n = 0; n < 2 * NB; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[n][i] = 0.0f;
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
                mma2<NP, NP>(p + 2 * j, a, b);
            }
    }
}

// out += P Y, P such scores as they lie in registers (PP planes of them), Y the
// tokens' tile.
template <int PP, int NP, int NB, int NT>
__device__ __forceinline__ void weighted(float (*out)[4], const float (*p)[4], const Tile& Y, int cb, int jb,
                                         int j0, int j1) {
#pragma unroll
    for (int j = 0; j < NB; ++j)
        if (jb + j >= j0 && jb + j < j1) {
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
                for (int i = 0; i < NP; ++i) Y.b_t(b[i], (jb + j) * 16, cb + n * 16, i);
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

template <int NT>
__device__ __forceinline__ void clear(float (*x)[4]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) x[n][i] = 0.0f;
}
template <int NT>
__device__ __forceinline__ void scale_rows(float (*x)[4], float r0, float r1) {
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n][0] *= r0, x[n][1] *= r0, x[n][2] *= r1, x[n][3] *= r1;
}
// A strip of scores from block jb on, by its columns' factors.
template <int NB>
__device__ __forceinline__ void scale_columns(float (*p)[4], const float* column, int jb) {
#pragma unroll
    for (int n = 0; n < 2 * NB; ++n) {
        const float2 f = *reinterpret_cast<const float2*>(column + jb * 16 + n * 8 + (lane_id() & 3) * 2);
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

// 16 rows and NT column tiles of a state in fp32 (dk, dv), from and to registers.
template <int NT>
__device__ __forceinline__ void load_state(float (*S)[4], const float* from, int row, int cb, int dk, int dv) {
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row + (l >> 2) + (i >> 1) * 8, c = cb + n * 8 + (l & 3) * 2 + (i & 1);
            S[n][i] = from && r < dk && c < dv ? from[r * dv + c] : 0.0f;
        }
}
template <int NT>
__device__ __forceinline__ void store_state(const float (*S)[4], float* to, int row, int cb, int dk, int dv) {
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = row + (l >> 2) + (i >> 1) * 8, c = cb + n * 8 + (l & 3) * 2 + (i & 1);
            if (r < dk && c < dv) to[r * dv + c] = S[n][i];
        }
}

// The same as PN bf16 planes of D x D.
template <int PN, int D, int NT>
__device__ __forceinline__ void state_planes(const float (*S)[4], bf16* to, int row, int cb) {
    const int l = lane_id();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            bf16* at = to + (row + (l >> 2) + i * 8) * D + cb + n * 8 + (l & 3) * 2;
            const uint32_t hi = pack2(S[n][2 * i], S[n][2 * i + 1]);
            *reinterpret_cast<uint32_t*>(at) = hi;
            if constexpr (PN == 2)
                *reinterpret_cast<uint32_t*>(at + D * D) = rest2(S[n][2 * i], S[n][2 * i + 1], hi);
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
// there are more warps than blocks, a block's columns.
template <typename T_, int D_, int C_, int NW_>
struct Shape {
    typedef T_ T;
    static constexpr int NP = planes_of<T_>, D = D_, C = C_, NW = NW_, THREADS = NW * 32;
    static constexpr int LD = D + 8, TILE = NP * C * LD, STATE = D * LD;
    static constexpr int SUB = C < 64 ? C : 64, STAGE = NP * SUB * LD;  // tokens of a stage of the states' pass
    static constexpr int RB = C / 16, CG = NW / RB, NT = D / CG / 8;
    // a states' pass: warps of 16 rows and half of the columns
    static constexpr int SR = D / 16, SW = 2 * SR, ST = SW * 32, SNT = D / 16;
    static_assert(NW % RB == 0 && NT % 2 == 0, "whole blocks for the warps");
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
    const float* start;  // each part's first state, or null
    float *sums, *factor;  // what each part adds to a state of zeros, and its decay
    bf16* kept;            // the state before (backwards: behind) each chunk, planes of D x D
    float* end;            // the last state, or null
    bool back;
};

// The states alone; without KEEP, sums and factor of every part but the last.
// The decays of the next chunk are the work of one more warp, and its tiles are on
// their way meanwhile. PN: planes of the kept states.
template <class S_, bool KEEP, int PN>
__global__ void __launch_bounds__(S_::ST + 32)
state_kernel(const Job j, const Pass p0, const Pass p1, Decays<S_::C>* dec_out) {
    typedef typename S_::T T;
    constexpr int NP = S_::NP, D = S_::D, C = S_::C, LD = S_::LD, NT = S_::SNT, SUB = S_::SUB, PER = C / SUB;
    constexpr int STAGES = NP == 1 ? 3 : 2;
    typedef Fetch<T, SUB, D, S_::ST> Load;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* const tiles = reinterpret_cast<bf16*>(smem);
    __shared__ Decays<C> dec_[2];
    __shared__ Weights<C> weights_[2];
    const Pass& p = blockIdx.y ? p1 : p0;
    const int seg = blockIdx.x % j.nseg;
    const long long bh = blockIdx.x / j.nseg;
    const int b = (int)(bh / j.H), h = (int)(bh % j.H);
    if (!KEEP && seg == (p.back ? 0 : j.nseg - 1)) return;
    const int end = tokens_of(j, b), c0 = min(j.chunks, seg * j.per_seg);
    const int live = max(c0, min(min(j.chunks, c0 + j.per_seg), (end + C - 1) / C)), n = live - c0;
    const auto chunk = [&](int i) { return p.back ? live - 1 - i : c0 + i; };
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;

    if (warp == S_::SW) {  // the decays
        constexpr int M = C / 32;
        const float* g = j.g + b * j.gs.b + h * j.gs.h;
        float x[M], y[M];
        const auto ask = [&](float* to, int i) {
#pragma unroll
            for (int k = 0; k < M; ++k) {
                const int t = chunk(i) * C + l * M + k;
                to[k] = i < n && t < end ? g[(long long)t * j.gs.t] : 0.0f;
            }
        };
        ask(x, 0);
        ask(y, 1);
        if (n) decays<C>(&dec_[0], &weights_[0], x, p.back, j.scale);
        for (int i = 0; i < n; ++i) {
            __syncthreads();  // (what is written behind it was read a chunk ago)
            if (KEEP && dec_out && !blockIdx.y) {
                const float4* from = reinterpret_cast<const float4*>(&dec_[i & 1]);
                float4* to = reinterpret_cast<float4*>(dec_out + bh * j.chunks + chunk(i));
                for (int k = l; k < (int)sizeof(Decays<C>) / 16; k += 32) to[k] = from[k];
            }
#pragma unroll
            for (int k = 0; k < M; ++k) x[k] = y[k];
            ask(y, i + 2);
            if (i + 1 < n) decays<C>(&dec_[(i + 1) & 1], &weights_[(i + 1) & 1], x, p.back, j.scale);
#pragma unroll
            for (int k = 1; k < PER; ++k) __syncthreads();
        }
        return;
    }

    const int row = warp % S_::SR * 16, cb = warp / S_::SR * NT * 8;
    const T* x = head_of<T>(p.x, p.xs, b, h / j.share);
    const T* y = head_of<T>(p.y, p.ys, b, h);
    const bool wx = j.whole >> (p.back ? 0 : 1) & 1, wy = j.whole >> (p.back ? 3 : 2) & 1;
    Load lx, ly;
    // stage u of the pass: tokens [first(u), first(u) + SUB)
    const int stages = n * PER;
    const auto first = [&](int u) { return chunk(u / PER) * C + u % PER * SUB; };
    const auto fetch = [&](int u, int stage) {
        if (u < stages) {
            bf16* to = tiles + stage * 2 * S_::STAGE;
            lx.fetch(to, x, p.xs.t, first(u), end, j.dk, wx);
            ly.fetch(to + S_::STAGE, y, p.ys.t, first(u), end, j.dv, wy);
        }
        cp_async_commit();
    };
    const auto put = [&](int u, int stage) {
        if (u < stages) {
            bf16* to = tiles + stage * 2 * S_::STAGE;
            lx.put(to, x, p.xs.t, first(u), end, j.dk, wx);
            ly.put(to + S_::STAGE, y, p.ys.t, first(u), end, j.dv, wy);
        }
    };
    for (int u = 0; u < STAGES - 1; ++u) fetch(u, u);
    put(0, 0);
    float S[NT][4];
    load_state<NT>(S, KEEP && p.start ? p.start + (bh * j.nseg + seg) * j.dk * j.dv : nullptr, row, cb, j.dk,
                   j.dv);
    float f = 1.0f;
    int stage = 0;
    for (int i = 0; i < n; ++i) {
        const Decays<C>& dec = dec_[i & 1];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const int u = i * PER + k;
            cp_async_wait_group<STAGES - 2>();
            __syncthreads();
            fetch(u + STAGES - 1, (stage + STAGES - 1) % STAGES);
            if (k == 0) {
                if constexpr (KEEP)
                    state_planes<PN, D, NT>(S, p.kept + (bh * j.chunks + chunk(i)) * PN * D * D, row, cb);
                const float w = dec.whole;
                f *= w;
#pragma unroll
                for (int m = 0; m < NT; ++m)
#pragma unroll
                    for (int e = 0; e < 4; ++e) S[m][e] *= w;
            }
            const bf16* from = tiles + stage * 2 * S_::STAGE;
            add_outer<NP, NT, SUB>(S, tile(from, LD, SUB * LD), tile(from + S_::STAGE, LD, SUB * LD),
                                   weights_[i & 1].pair + k * SUB / 2, row, cb);
            stage = (stage + 1) % STAGES;
            put(u + 1, stage);
        }
    }
    if constexpr (!KEEP) {
        store_state<NT>(S, p.sums + (bh * j.nseg + seg) * j.dk * j.dv, row, cb, j.dk, j.dv);
        if (threadIdx.x == 0) p.factor[bh * j.nseg + seg] = f;
    } else if (p.end && seg == (p.back ? 0 : j.nseg - 1)) {
        store_state<NT>(S, p.end + bh * j.dk * j.dv, row, cb, j.dk, j.dv);
    }
}

// From what each part adds, in place, the state that each starts with, `first`
// being the sequence's.
__global__ void __launch_bounds__(256) join_kernel(float* sums, const float* factor, const float* first,
                                                   bool back, int nseg, long long size, long long total) {
    const long long i = blockIdx.x * 256ll + threadIdx.x;
    if (i >= total) return;
    const long long bh = i / size;
    float* at = sums + bh * nseg * size + i % size;
    const float* f = factor + bh * nseg;
    float S = first ? first[i] : 0.0f;
    constexpr int U = 16;  // asked for together
    for (int k0 = 0; k0 < nseg; k0 += U) {
        float add[U], by[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = back ? nseg - 1 - k0 - u : k0 + u;
            const bool in = k0 + u < nseg - 1;  // (nothing is added up for the last)
            add[u] = in ? at[s * size] : 0.0f;
            by[u] = in ? f[s] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = back ? nseg - 1 - k0 - u : k0 + u;
            if (k0 + u < nseg) at[s * size] = S;
            S = by[u] * S + add[u];
        }
    }
}

// ----------------------------------------------------------------- outputs
// A CTA for each chunk: the states before them are there, so all run at once.
// Heads go side by side: they lie so in memory.
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

// A tile of kept states (PN planes of D x D), and a chunk's decays, by cp.async.
template <class S_, int PN>
__device__ __forceinline__ void load_kept(bf16* dst, const bf16* from) {
    constexpr int D = S_::D;
#pragma unroll
    for (int n = 0; n < PN * D * D / 8 / S_::THREADS; ++n) {
        const int i = n * S_::THREADS + threadIdx.x;
        cp_async16(dst + i / (D * D / 8) * S_::STATE + i % (D * D / 8) / (D / 8) * S_::LD + i % (D / 8) * 8,
                   from + i * 8, 16);
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
    constexpr int NP = S_::NP, D = S_::D, C = S_::C, LD = S_::LD, NT = S_::NT, NB = 2;
    typedef Fetch<T, C, D, S_::THREADS> Load;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* const sq = reinterpret_cast<bf16*>(smem);
    bf16 *const sk = sq + S_::TILE, *const sv = sk + S_::TILE, *const ss = sv + S_::TILE;
    __shared__ Decays<C> dec;
    const Chunk at(j);
    const int end = tokens_of(j, at.b), c0 = at.c * C;
    const long long ot = (long long)j.H * j.dv;
    T* out = static_cast<T*>(out_) + (long long)at.b * j.T * ot + (long long)at.h * j.dv;
    if (c0 >= end) return zero_rows(out, ot, c0, min(c0 + C, j.T), j.dv);
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;
    const int rb = warp % S_::RB, cb = warp / S_::RB * NT * 8;
    const T* q = head_of<T>(j.q, j.qs, at.b, at.h / j.share);
    const T* k = head_of<T>(j.k, j.ks, at.b, at.h / j.share);
    const T* v = head_of<T>(j.v, j.vs, at.b, at.h);
    Load lq, lk, lv;
    lq.fetch(sq, q, j.qs.t, c0, end, j.dk, j.whole & 1);
    load_kept<S_, NP>(ss, kept + (at.bh * j.chunks + at.c) * NP * D * D);
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
    const Tile tq = tile(sq, LD, C * LD), tk = tile(sk, LD, C * LD), tv = tile(sv, LD, C * LD),
               ts = tile(ss, LD, S_::STATE);

    // Between the blocks of 16 tokens a decay is 2^(c_t - c_r) 2^(c_r - c_s), r the
    // last token before the row's block: a factor of the row, which the state's
    // part shares, and one of the column, which the warp writes down once. Both are
    // at most 1. Within a block each pair has its own.
    __shared__ float column_[S_::NW][C];
    float* const column = column_[warp];
    for (int s = l; s < rb * 16; s += 32) column[s] = dec.between(rb * 16 - 1, s);
    __syncwarp();
    float O[NT][4];
    const int t = rb * 16 + (l >> 2);
    const float r0 = (rb ? dec.between(t, rb * 16 - 1) : dec.from_start[t]) * j.scale;
    const float r1 = (rb ? dec.between(t + 8, rb * 16 - 1) : dec.from_start[t + 8]) * j.scale;
    const auto before = [&] {
        clear<NT>(O);
        product<NP, NP, D, NT, true>(O, tq, rb * 16, ts, cb);
        if (rb) {
            const float begin = dec.from_start[rb * 16 - 1];
            scale_rows<NT>(O, begin, begin);
        }
    };
    const auto chunk = [&](bool apart) {
        for (int jb = 0; jb < rb; jb += NB) {
            float P[2 * NB][4];
            scores<NP, D, NB>(P, tq, rb * 16, tk, jb, 0, rb);
            scale_columns<NB>(P, column, jb);
            weighted<NP, NP, NB, NT>(O, P, tv, cb, jb, 0, rb);
        }
        scale_rows<NT>(O, r0, r1);
        float P[2][4];
        scores<NP, D, 1>(P, tq, rb * 16, tk, rb, rb, rb + 1);
        near_decays<C>(P, dec, rb, j.scale);
        if (apart)
            weighted_apart<NP, NT>(O, P, sv + rb * 16 * LD, LD, C * LD, cb);
        else
            weighted<NP, NP, 1, NT>(O, P, tv, cb, rb, rb, rb + 1);
    };
    before();
    cp_async_wait_all();
    __syncthreads();
    chunk(false);
    // a value of v that is not finite reaches every row of its block (times zero, in those before it)
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) sum = fmaf(O[n][0], 0.0f, fmaf(O[n][1], 0.0f, sum));
    if (__any_sync(0xffffffffu, sum != 0.0f)) {
        before();
        chunk(true);
    }
    if constexpr (S_::CG > 1) named_bar_sync(rb + 1, S_::CG * 32);  // the queries of these rows are done with
    store_rows_by<T, NT, LD>(sq + rb * 16 * LD + cb, O, out, ot, c0 + rb * 16, cb, end, j.T, j.dv);
}

// ---------------------------------------------------------------- gradients
struct Grads {
    const void* dout;
    Strides ds;
    const bf16 *before, *behind;  // the states before the chunks, their gradients behind them
    void *dq, *dk, *dv;
    float *dq32, *dk32;  // in place of dq, dk: each head's own, where heads share q and k
    float* dg;           // (B, T, H), or null
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

template <class S_, int MIN>
__global__ void __launch_bounds__(S_::THREADS, MIN)
grad_kernel(const Job j, const Grads G, const Decays<S_::C>* decs) {
    typedef typename S_::T T;
    constexpr int NP = S_::NP, D = S_::D, C = S_::C, LD = S_::LD, NT = S_::NT, RB = S_::RB, CG = S_::CG;
    constexpr int NB = 2;  // blocks of a strip: two accumulators and two strips of scores are held
    typedef Fetch<T, C, D, S_::THREADS> Load;
    extern __shared__ __align__(16) unsigned char smem[];
    bf16* const sq = reinterpret_cast<bf16*>(smem);
    bf16 *const sk = sq + S_::TILE, *const sv = sk + S_::TILE, *const so = sv + S_::TILE;
    bf16* const ss = so + S_::TILE;  // the gradient behind the chunk, then the state before it
    __shared__ Decays<C> dec;
    __shared__ float column_[S_::NW][C];
    // parts of dg: by row block, and by column group where the columns are split
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
        return;
    }
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31;
    const int rb = warp % RB, cg = warp / RB, cb = cg * NT * 8;
    const Tile tq = tile(sq, LD, C * LD), tk = tile(sk, LD, C * LD), tv = tile(sv, LD, C * LD),
               to = tile(so, LD, C * LD), ts = tile(ss, LD, S_::STATE);
    const long long kept = (at.bh * j.chunks + at.c) * 2 * D * D;
    {
        const T* q = head_of<T>(j.q, j.qs, at.b, at.h / j.share);
        const T* k = head_of<T>(j.k, j.ks, at.b, at.h / j.share);
        const T* v = head_of<T>(j.v, j.vs, at.b, at.h);
        const T* dout = head_of<T>(G.dout, G.ds, at.b, at.h);
        Load lq, lk, lv, lo;
        lq.fetch(sq, q, j.qs.t, c0, end, j.dk, j.whole & 1);
        lk.fetch(sk, k, j.ks.t, c0, end, j.dk, j.whole >> 1 & 1);
        load_kept<S_, 2>(ss, G.behind + kept);
        load_decays<C>(&dec, decs + at.bh * j.chunks + at.c);
        lq.put(sq, q, j.qs.t, c0, end, j.dk, j.whole & 1);
        lk.put(sk, k, j.ks.t, c0, end, j.dk, j.whole >> 1 & 1);
        lv.fetch(sv, v, j.vs.t, c0, end, j.dv, j.whole >> 2 & 1);
        lo.fetch(so, dout, G.ds.t, c0, end, j.dv, j.whole >> 3 & 1);
        lv.put(sv, v, j.vs.t, c0, end, j.dv, j.whole >> 2 & 1);
        lo.put(so, dout, G.ds.t, c0, end, j.dv, j.whole >> 3 & 1);
    }
    cp_async_wait_all();
    __syncthreads();
    // (by way of the states' place, a part of it for each warp)
    constexpr int BY = NT * 8 + 8;
    static_assert(S_::NW * 16 * BY <= 2 * S_::STATE, "room for every warp's rows");
    bf16* const by = ss + warp * 16 * BY;
    const auto store_head = [&](const float(*x)[4], void* to16, float* to32) {
        if (to32)
            store_rows<float, NT>(x, to32 + k0, kt, c0 + rb * 16, cb, end, j.T, j.dk);
        else
            store_rows_by<T, NT, BY>(by, x, static_cast<T*>(to16) + k0, kt, c0 + rb * 16, cb, end, j.T, j.dk);
    };
    float* const column = column_[warp];
    float part[2];
    const int t = rb * 16 + (l >> 2);  // the lane's tokens: this and 8 behind
    {
        // rows s, columns u >= s. Between blocks a decay is 2^(c_u - c_r) 2^(c_r - c_s), r
        // the last token of the row's block
        const int r = rb * 16 + 15;
        for (int u = r + 1 + l; u < C; u += 32) column[u] = dec.between(u, r) * j.scale;
        __syncwarp();
        const float b0 = dec.between(r, t), b1 = dec.between(r, t + 8), behind = dec.to_end[r];
        float V[NT][4], K[NT][4], across[2] = {0.0f, 0.0f};
        clear<NT>(V);
        product<NP, NP, D, NT, true>(V, tk, rb * 16, ts, cb);
        scale_rows<NT>(V, behind, behind);
        clear<NT>(K);
        product<NP, 2, D, NT, false>(K, tv, rb * 16, ts, cb);
        scale_rows<NT>(K, behind, behind);
        row_dots<NP, NT>(K, sk, LD, C * LD, rb * 16, cb, part);
        if ((l & 3) == 0) dk_part[cg][t] = part[0] * b0, dk_part[cg][t + 8] = part[1] * b1;
        for (int jb = (rb + 1) / NB * NB; jb < RB; jb += NB) {
            float P[2 * NB][4], Q[2 * NB][4], down[4 * NB];
            scores<NP, D, NB>(P, tk, rb * 16, tq, jb, rb + 1, RB);
            scores<NP, D, NB>(Q, tv, rb * 16, to, jb, rb + 1, RB);
#pragma unroll
            for (int n = 0; n < 2 * NB; ++n) {
                const int u = jb * 16 + n * 8 + (l & 3) * 2;
                const float2 f = *reinterpret_cast<const float2*>(column + u);
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
            weighted<NP, NP, NB, NT>(V, P, to, cb, jb, rb + 1, RB);
            weighted<NP, NP, NB, NT>(K, Q, tq, cb, jb, rb + 1, RB);
        }
        scale_rows<NT>(V, b0, b1);
        scale_rows<NT>(K, b0, b1);
        across[0] *= b0, across[1] *= b1;
        float P[2][4], Q[2][4], down[4] = {};
        scores<NP, D, 1>(P, tk, rb * 16, tq, rb, rb, rb + 1);
        scores<NP, D, 1>(Q, tv, rb * 16, to, rb, rb, rb + 1);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int s = t + (i >> 1) * 8, u = rb * 16 + n * 8 + (l & 3) * 2 + (i & 1);
                const float w = dec.between(u, s) * j.scale, p = P[n][i] * w;
                const float a = u > s ? p * Q[n][i] : 0.0f;
                P[n][i] = u >= s ? p : 0.0f;
                Q[n][i] = u >= s ? Q[n][i] * w : 0.0f;
                across[i >> 1] += a;
                down[2 * n + (i & 1)] += a;
            }
        const int which = column_sums<4>(down);
        if (cg == 0) col_part[rb][rb * 16 + which / 2 * 8 + (l & 3) * 2 + which % 2] = down[0];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            across[i] += __shfl_xor_sync(0xffffffffu, across[i], 1);
            across[i] += __shfl_xor_sync(0xffffffffu, across[i], 2);
        }
        if (cg == 0 && (l & 3) == 0) row_part[t] = across[0], row_part[t + 8] = across[1];
        weighted<NP, NP, 1, NT>(V, P, to, cb, rb, rb, rb + 1);
        weighted<NP, NP, 1, NT>(K, Q, tq, cb, rb, rb, rb + 1);
        // <R, S>, and then their place is free
        float dot = 0.0f;
        if (dg) {
            const uint4* from = reinterpret_cast<const uint4*>(G.before + kept);
            constexpr int PACKS = D * D / 8;
#pragma unroll 4
            for (int i = threadIdx.x; i < PACKS; i += S_::THREADS) {
                const uint4 hi = from[i], lo = from[PACKS + i];
                const uint4 r = *reinterpret_cast<const uint4*>(ss + i / (D / 8) * LD + i % (D / 8) * 8);
                const uint4 r2 = *reinterpret_cast<const uint4*>(ss + S_::STATE + i / (D / 8) * LD + i % (D / 8) * 8);
                const uint32_t a[4] = {r.x, r.y, r.z, r.w}, b[4] = {r2.x, r2.y, r2.z, r2.w};
                const uint32_t x[4] = {hi.x, hi.y, hi.z, hi.w}, y[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    dot = fmaf(low(a[e]) + low(b[e]), low(x[e]) + low(y[e]), dot);
                    dot = fmaf(high(a[e]) + high(b[e]), high(x[e]) + high(y[e]), dot);
                }
            }
        }
#pragma unroll
        for (int d = 16; d; d /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (l == 0) dot_part[warp] = dot;
        __syncthreads();
        store_rows_by<T, NT, BY>(by, V, dv, vt, c0 + rb * 16, cb, end, j.T, j.dv);
        store_head(K, G.dk, G.dk32);
    }
    __syncthreads();
    load_kept<S_, 2>(ss, G.before + kept);
    cp_async_wait_all();
    for (int s = l; s < rb * 16; s += 32) column[s] = dec.between(rb * 16 - 1, s);
    __syncthreads();
    {
        // rows u, columns s <= u, as the outputs
        float X[NT][4], P[2][4];
        clear<NT>(X);
        product<NP, 2, D, NT, false>(X, to, rb * 16, ts, cb);
        const float begin = rb ? dec.from_start[rb * 16 - 1] : 1.0f;
        scale_rows<NT>(X, begin, begin);
        const float r0 = (rb ? dec.between(t, rb * 16 - 1) : dec.from_start[t]) * j.scale;
        const float r1 = (rb ? dec.between(t + 8, rb * 16 - 1) : dec.from_start[t + 8]) * j.scale;
        row_dots<NP, NT>(X, sq, LD, C * LD, rb * 16, cb, part);
        if ((l & 3) == 0) dq_part[cg][t] = part[0] * r0, dq_part[cg][t + 8] = part[1] * r1;
        for (int jb = 0; jb < rb; jb += NB) {
            float Q[2 * NB][4];
            scores<NP, D, NB>(Q, to, rb * 16, tv, jb, 0, rb);
            scale_columns<NB>(Q, column, jb);
            weighted<NP, NP, NB, NT>(X, Q, tk, cb, jb, 0, rb);
        }
        scale_rows<NT>(X, r0, r1);
        scores<NP, D, 1>(P, to, rb * 16, tv, rb, rb, rb + 1);
        near_decays<C>(P, dec, rb, j.scale);
        weighted<NP, NP, 1, NT>(X, P, tk, cb, rb, rb, rb + 1);
        __syncthreads();
        store_head(X, G.dq, G.dq32);
    }
    if (warp == 0 && dg) {
        // behind: sum over u >= t of (rho_u + r_u) - sum over s >= t of kappa_s; ahead: sum over s < t of l_s
        constexpr int M = C / 32;
        float behind[M], ahead[M], all = 0.0f, b = 0.0f, a = 0.0f;
#pragma unroll
        for (int i = 0; i < S_::NW; ++i) all += dot_part[i];
        all *= dec.whole;
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
            const int u = c0 + l * M + i;
            if (u < j.T) dg[(long long)u * j.H] = u < end ? all + behind[i] + bs + ahead[i] + as : 0.0f;
        }
    }
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
    static constexpr int state = (S_::NP == 1 ? 6 : 4) * S_::STAGE * 2;
    static constexpr int out = 3 * S_::TILE * 2 + S_::NP * S_::STATE * 2;
    static constexpr int grad = 4 * S_::TILE * 2 + 2 * S_::STATE * 2;
};

template <typename K>
int allow(K* kernel, int bytes, const char* what) {
    return cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
}

constexpr int kSms = 148;  // of a B200: the split of a sequence does not ask the device

// Parts of a sequence whose states run side by side: enough CTAs for `per_sm` on
// every SM, none shorter than four chunks.
void split(Job* j, int C, int per_sm) {
    j->chunks = (j->T + C - 1) / C;
    const long long heads = (long long)j->B * j->H;
    long long parts = heads ? kSms * per_sm / heads : 1;
    parts = std::max(1ll, std::min(parts, (long long)j->chunks / 4));
    j->per_seg = std::max(1, (int)((j->chunks + parts - 1) / parts));
    j->nseg = std::max(1, (j->chunks + j->per_seg - 1) / j->per_seg);
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
    const long long bh = (long long)j.B * j.H, plane = bh * j.chunks * S_::D * S_::D * 2;
    long long at = 0;
    const auto take = [&](long long bytes) {
        const long long a = at;
        at += up(bytes);
        return a;
    };
    for (int i = 0; i < 1 + back; ++i)
        if (j.nseg > 1) {
            (i ? s.back : s.sums) = take(bh * j.nseg * j.dk * j.dv * 4);
            (i ? s.back_factor : s.factor) = take(bh * j.nseg * 4);
        }
    s.decays = take(bh * j.chunks * sizeof(Decays<S_::C>));
    s.kept = take(plane * (back ? 2 : S_::NP));
    if (back) {
        s.kept_back = take(plane * 2);
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

// The states that the chunks need: in parts, joined, where there are several.
template <class S_, int PN>
int states(const Job& j, Pass p0, Pass p1, bool both, const float* first0, const float* first1,
           Decays<S_::C>* dec, cudaStream_t st) {
    const long long bh = (long long)j.B * j.H, size = (long long)j.dk * j.dv;
    const dim3 grid((unsigned)(bh * j.nseg), both ? 2 : 1);
    constexpr int threads = S_::ST + 32, bytes = Sizes<S_>::state;
    static_assert(bytes <= 220 * 1024, "shared memory of a CTA");
    p0.start = first0, p1.start = first1;
    if (j.nseg > 1) {
        auto* sum = state_kernel<S_, false, PN>;
        SN_TRY(allow(sum, bytes, "linear_attention"));
        sum<<<grid, threads, bytes, st>>>(j, p0, p1, nullptr);
        const unsigned ctas = (unsigned)((bh * size + 255) / 256);
        join_kernel<<<ctas, 256, 0, st>>>(p0.sums, p0.factor, first0, p0.back, j.nseg, size, bh * size);
        if (both)
            join_kernel<<<ctas, 256, 0, st>>>(p1.sums, p1.factor, first1, p1.back, j.nseg, size, bh * size);
        p0.start = p0.sums, p1.start = p1.sums;
    }
    auto* keep = state_kernel<S_, true, PN>;
    SN_TRY(allow(keep, bytes, "linear_attention"));
    keep<<<grid, threads, bytes, st>>>(j, p0, p1, dec);
    return cuda_check(cudaGetLastError(), "linear_attention launch");
}

int check_space(const Job& j, const Space& s, const char* what, const char* ws, long long ws_bytes) {
    if (s.bytes > ws_bytes || (s.bytes && !ws))
        return fail(SN_E_INVAL, "%s: a workspace of %lld bytes is wanted", what, s.bytes);
    if ((long long)j.B * j.H * std::max(j.nseg, j.chunks) > 0x7fffffffll)
        return fail(SN_E_INVAL, "%s: too many chunks", what);
    return SN_OK;
}

template <class S_>
int forward(Job j, const float* first, void* out, float* state_out, char* ws, long long ws_bytes, long long* need,
            cudaStream_t st) {
    split(&j, S_::C, 2);
    const Space s = space_of<S_>(j, false, false);
    if (need) {
        *need = s.bytes;
        return SN_OK;
    }
    SN_TRY(check_space(j, s, "linear_attention", ws, ws_bytes));
    Pass p = {j.k, j.v, j.ks, j.vs};
    p.sums = reinterpret_cast<float*>(ws + s.sums), p.factor = reinterpret_cast<float*>(ws + s.factor);
    p.kept = reinterpret_cast<bf16*>(ws + s.kept);
    p.end = state_out;
    auto* dec = reinterpret_cast<Decays<S_::C>*>(ws + s.decays);
    SN_TRY((states<S_, S_::NP>(j, p, p, false, first, nullptr, dec, st)));
    if (!j.chunks) return SN_OK;
    constexpr int bytes = Sizes<S_>::out;
    static_assert(bytes <= 220 * 1024, "shared memory of a CTA");
    auto* kernel = out_kernel<S_, bytes <= 66 * 1024 ? 3 : bytes <= 96 * 1024 ? 2 : 1>;
    SN_TRY(allow(kernel, bytes, "linear_attention"));
    kernel<<<(unsigned)((long long)j.B * j.H * j.chunks), S_::THREADS, bytes, st>>>(j, p.kept, dec, out);
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
    split(&j, S_::C, 1);
    const Space s = space_of<S_>(j, true, g.gates_alike);
    if (need) {
        *need = s.bytes;
        return SN_OK;
    }
    SN_TRY(check_space(j, s, "linear_attention_bwd", ws, ws_bytes));
    const auto floats = [&](long long at) { return reinterpret_cast<float*>(ws + at); };
    Pass p = {j.k, j.v, j.ks, j.vs}, r = {j.q, g.dout, j.qs, g.ds};
    p.sums = floats(s.sums), p.factor = floats(s.factor);
    p.kept = reinterpret_cast<bf16*>(ws + s.kept);
    r.sums = floats(s.back), r.factor = floats(s.back_factor);
    r.kept = reinterpret_cast<bf16*>(ws + s.kept_back);
    r.end = g.dstate;
    r.back = true;
    auto* dec = reinterpret_cast<Decays<S_::C>*>(ws + s.decays);
    SN_TRY((states<S_, 2>(j, p, r, true, first, g.dstate_out, dec, st)));
    Grads G = {};
    G.dout = g.dout, G.ds = g.ds;
    G.before = p.kept, G.behind = r.kept;
    G.dq = g.dq, G.dk = g.dk, G.dv = g.dv;
    if (j.share > 1) G.dq32 = floats(s.dq32), G.dk32 = floats(s.dk32);
    G.dg = !g.dg ? nullptr : g.gates_alike ? floats(s.dg) : g.dg;
    constexpr int bytes = Sizes<S_>::grad;
    static_assert(bytes <= 220 * 1024, "shared memory of a CTA");
    auto* kernel = grad_kernel<S_, bytes <= 96 * 1024 ? 2 : 1>;
    SN_TRY(allow(kernel, bytes, "linear_attention_bwd"));
    if (j.chunks)
        kernel<<<(unsigned)((long long)j.B * j.H * j.chunks), S_::THREADS, bytes, st>>>(j, G, dec);
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

// Tokens of a chunk: the longer, the fewer states are kept and read again (in
// bf16 with heads of up to 64, the states of a chunk of 128 take half of what its
// keys do), and the more shared memory the tiles take.
template <typename T, typename F>
int by_width(const Job& j, F&& f) {
    constexpr bool one = planes_of<T> == 1;
    if (std::max(j.dk, j.dv) <= 64) return f(Shape<T, 64, one ? 128 : 64, 8>());
    return f(Shape<T, 128, 64, 8>());
}
template <typename F>
int by_type(int dtype, const Job& j, F&& f) {
    return dtype == SN_F32    ? by_width<float>(j, f)
           : dtype == SN_BF16 ? by_width<bf16>(j, f)
                              : by_width<__half>(j, f);
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
    j->chunks = 0, j->nseg = 1, j->per_seg = 1;
    j->whole = (int)packs(j->q, j->qs, j->dk, a->dtype, a->B < 2, a->Hk < 2) |
               (int)packs(j->k, j->ks, j->dk, a->dtype, a->B < 2, a->Hk < 2) << 1 |
               (int)packs(j->v, j->vs, j->dv, a->dtype, a->B < 2, a->H < 2) << 2;
    return SN_OK;
}

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
        la::by_type(a->dtype, j, [&](auto s) {
            return la::backward<decltype(s)>(j, la::kSms, nullptr, w, nullptr, 0, &need, nullptr);
        });
    } else {
        la::by_type(a->dtype, j, [&](auto s) {
            return la::forward<decltype(s)>(j, nullptr, nullptr, nullptr, nullptr, 0, &need, nullptr);
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
    return la::by_type(a->dtype, j, [&](auto s) {
        return la::forward<decltype(s)>(j, a->state, out, state_out, static_cast<char*>(ws), ws_bytes,
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
    return la::by_type(a->dtype, j, [&](auto s) {
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
