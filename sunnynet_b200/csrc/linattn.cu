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
// (dg sums only what passes token t's gate, so that it is as good as its own terms: the
// shorter form by differences q.dq - k.dk from the sequence's end loses all digits over
// long sequences, and differences of the pairs' sums within a chunk those of fast decays.)
//
// All products are m16n8k16 matrix instructions on bf16 with fp32 sums. bf16
// values are taken as they are, float16 ones as the sum of two bf16 and float32
// ones of three, which loses nothing; the products of their parts are left out
// that a result does not hold. What is computed on the way to an fp32 result (the
// states, dg) is taken apart in three as well, and so keeps fp32's accuracy; what
// goes to 16-bit outputs alone is rounded to one part (bf16) or two (float16). tcgen05 was
// not taken: with heads of 64 its products here have 64 columns, and an instruction
// of 128 x 64 x 16 takes as long as one of 128 x 128 x 16 (90 cycles); the 24 that
// a chunk of 128 tokens needs would fill three quarters of the time that HBM leaves
// it, while the decays need the scores in registers and the states anew for each chunk.
// Heads of 128 would fill the instruction; there the traffic of the states is what bounds
// the calls (see state_kernel), and tcgen05 was not tried.
#include <algorithm>
#include <cmath>

#include "linattn.cuh"

namespace sn {
namespace la {

// The kernels of each type are compiled in a file of their own.
#define SN_LA_EXTERN(T)                                                                                      \
    extern template int forward<T>(const Job&, const float*, void*, float*, char*, long long, long long*,    \
                                   cudaStream_t);                                                            \
    extern template int backward<T>(const Job&, const float*, const Wanted&, char*, long long, long long*,   \
                                    cudaStream_t);
SN_LA_EXTERN(float)
SN_LA_EXTERN(bf16)
SN_LA_EXTERN(__half)

namespace {

// -------------------------------------------------------------- single token
// A CTA for each sequence and head: its state goes through once. Lanes stand
// side by side along a row of the state, so that every access is one run. Bound by HBM: 256
// sequences x 12 heads of 64 take 17.5 us, one call after the other, 102 MB at 5.8 TB/s.
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
    constexpr int U = 8;  // rows on their way at once; the first are, while the factor is formed
    float s[U][VEC];
    const auto fetch = [&](int r) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (in && r + u * rows < dk) {
                const float* at = S + (r + u * rows) * dv + c * VEC;
                if constexpr (VEC == 4) {
                    const float4 y = *reinterpret_cast<const float4*>(at);
                    s[u][0] = y.x, s[u][1] = y.y, s[u][2] = y.z, s[u][3] = y.w;
                } else {
                    s[u][0] = *at;
                }
            }
    };
    const float gate = g[b * gb + h * gh];
    fetch(r0);
    // exp(g) in two parts: a slow decay's factor is the same at every token, and what it is off adds up over
    // 1 / (1 - f) of them (4096 tokens of decays about 2^-11: 3e-4 by ex2.approx, 8e-6 so: the states' roundings)
    float f, rest = 0.0f;
    if (fabsf(gate) < 0.5f) {
        const float e = expm1f(gate);
        f = 1.0f + e;
        rest = e - (f - 1.0f);  // (exactly what the sum lost)
    } else {
        f = expf(gate);
    }
    float x[VEC], o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        x[i] = in ? to_f(v[c * VEC + i]) : 0.0f;
        o[i] = 0.0f;
    }
    __syncthreads();
    if (in) {
        for (int r = r0; r < dk; r += rows * U) {
            if (r > r0) fetch(r);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (r + u * rows < dk) {
                    const float kk = sk[r + u * rows], qq = sq[r + u * rows];
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        s[u][i] = fmaf(f, s[u][i], fmaf(rest, s[u][i], kk * x[i]));
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

constexpr int kMaxHead = 128;

template <typename F>
int by_type(int dtype, F&& f) {
    return dtype == SN_F32 ? f(0.0f) : dtype == SN_BF16 ? f(bf16()) : f(__half());
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
    j->chunks = 0, j->apart = false;
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
        la::by_type(a->dtype, [&](auto t) {
            return la::backward<decltype(t)>(j, nullptr, w, nullptr, 0, &need, nullptr);
        });
    } else {
        la::by_type(a->dtype, [&](auto t) {
            return la::forward<decltype(t)>(j, nullptr, nullptr, nullptr, nullptr, 0, &need, nullptr);
        });
    }
    return need;
}

sn_status sn_abi_linear_attention(const SnAbiLinearAttention* a, void* out, float* state_out, void* ws,
                                  int64_t ws_bytes, void* cuda_stream) {
    CallerDevice dev;
    la::Job j;
    SN_TRY(la::read_job(a, "linear_attention", &j));
    if (!a->B) return SN_OK;
    if (!state_out || (a->T && (!a->log_decay || !a->q || !a->k || !a->v || !out)))
        return fail(SN_E_INVAL, "linear_attention: null pointer");
    const unsigned e = dtype_size(a->dtype);
    SN_TRY(dev.enter("linear_attention", {{a->q, e}, {a->k, e}, {a->v, e}, {a->log_decay, 4}, {a->state, 4},
                                          {a->lengths, 4}, {out, e}, {state_out, 4}, {ws, 16}}));
    return la::by_type(a->dtype, [&](auto t) {
        return la::forward<decltype(t)>(j, a->state, out, state_out, static_cast<char*>(ws), ws_bytes,
                                        nullptr, static_cast<cudaStream_t>(cuda_stream));
    });
}

sn_status sn_abi_linear_attention_bwd(const SnAbiLinearAttention* a, const void* dout,
                                      const int64_t* dout_stride, const float* dstate_out, void* dq, void* dk,
                                      void* dv, float* dlog_decay, int32_t head_gates, float* dstate, void* ws,
                                      int64_t ws_bytes, void* cuda_stream) {
    CallerDevice dev;
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
    SN_TRY(dev.enter("linear_attention_bwd",
                     {{a->q, e}, {a->k, e}, {a->v, e}, {a->log_decay, 4}, {a->state, 4}, {a->lengths, 4},
                      {dout, e}, {dstate_out, 4}, {dq, e}, {dk, e}, {dv, e}, {dlog_decay, 4}, {dstate, 4},
                      {ws, 16}}));
    la::Wanted w = {dout, la::strides(dout_stride), dstate_out, dq, dk, dv, dlog_decay, dstate,
                    head_gates != 0};
    j.whole |= (int)la::packs(dout, w.ds, j.dv, a->dtype, a->B < 2, a->H < 2) << 3;
    return la::by_type(a->dtype, [&](auto t) {
        return la::backward<decltype(t)>(j, a->state, w, static_cast<char*>(ws), ws_bytes, nullptr,
                                         static_cast<cudaStream_t>(cuda_stream));
    });
}

sn_status sn_abi_linear_attention_step(const SnAbiLinearAttention* a, float* state, int64_t state_stride,
                                       void* out, void* cuda_stream) {
    CallerDevice dev;
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
    return la::by_type(a->dtype, typed);
}

}  // extern "C"
