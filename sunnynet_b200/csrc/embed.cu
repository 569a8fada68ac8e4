// The rows of an embedding for given tokens, scaled, and the gradient of the
// embedding (no counterpart among the reference's kernels: its decode copies one
// row a step, its training loop leaves both to torch).
//
//   out[i] = scale * W[token_i]        dW[v] = scale * sum of dout[i] over token_i = v
//
// Forward: a copy, bound by HBM. A token outside the vocabulary gives a row of
// NaN, and no gradient: the device has no other way to tell.
//
// Gradient: the tokens are sorted by a stable radix sort of eight bits a pass, so
// that each row's tokens lie side by side in their order and are added in it, a row
// of many in pieces, which end where its chunks of sorted tokens do: an order that the
// call's tokens and sizes decide, the same bits every time, no atomics on values. Up to kNear tokens are sorted by one
// cluster of eight CTAs in one launch (5003 tokens, two passes: 11 us; four launches
// of many CTAs took 12, and 10 more of the host's time; 32768 tokens 28 us against
// 18), more of them by two launches a pass: the counts of every tile, then ranks and
// places. Bound by HBM (dout read, dW written once) from some ten thousand tokens on,
// and by latency below. While they sort, further CTAs of the same launches fill dW with zeros,
// which costs nothing then: most rows of a vocabulary occur in no batch, and those
// that do are overwritten. 32768 tokens of 32000 x 768 in bf16, rows 14 us, the sort
// 18, the sums 17 and the joins of rows of many tokens 7.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "caller.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace sn {
namespace {

template <typename T>
__device__ __forceinline__ float to_f(T x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return __bfloat162float(x);
    else
        return __half2float(x);
}
template <typename T>
__device__ __forceinline__ T from_f(float x) {
    if constexpr (sizeof(T) == 4)
        return x;
    else if constexpr (std::is_same<T, __nv_bfloat16>::value)
        return __float2bfloat16_rn(x);
    else
        return __float2half_rn(x);
}

// N values of T, read and written at once.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// The row of token i, or -1.
__device__ __forceinline__ long long row_of(const void* tokens, bool wide, long long i, long long V) {
    const long long t = wide ? static_cast<const long long*>(tokens)[i] : static_cast<const int*>(tokens)[i];
    return t >= 0 && t < V ? t : -1;
}

// x * f for a pack, rounded once to fp32 and once to T.
template <typename T, int N>
__device__ __forceinline__ Pack<T, N> scaled(const Pack<T, N>& x, float f) {
    Pack<T, N> y;
#pragma unroll
    for (int k = 0; k < N; ++k) y.v[k] = from_f<T>(to_f(x.v[k]) * f);
    return y;
}

// ----------------------------------------------------------------- forward
constexpr int kThreads = 256;

// LANES neighbouring threads copy a row, U packs of each on their way at once.
template <typename T, int N, int LANES>
__global__ void __launch_bounds__(kThreads)
rows_kernel(const void* tokens, bool wide, const T* W, long long ld, long long V, T* out, long long n, int D,
            float scale) {
    constexpr int U = LANES == 32 ? 4 : 2;
    const long long i = (blockIdx.x * (long long)kThreads + threadIdx.x) / LANES;
    if (i >= n) return;
    const long long row = row_of(tokens, wide, i, V);
    const float f = row >= 0 ? scale : __int_as_float(0x7fffffff);
    const T* from = W + (row >= 0 ? row * ld : 0);
    T* to = out + i * D;
    for (int c = threadIdx.x % LANES * N; c < D; c += U * LANES * N) {
        Pack<T, N> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = c + u * LANES * N;
            if (at < D && V) x[u] = *reinterpret_cast<const Pack<T, N>*>(from + at);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = c + u * LANES * N;
            if (at < D) *reinterpret_cast<Pack<T, N>*>(to + at) = scaled(x[u], f);
        }
    }
}

// -------------------------------------------------------------------- sort
constexpr int kTiles = 148;  // at most: a tile of the tokens for each SM
constexpr int kBins = 256;
constexpr int kSort = 1024;  // threads of a CTA: tokens of a tile that are placed at once

struct Sorting {
    const void* tokens;  // of the first pass
    bool wide;
    long long V;
    const uint2* from;  // of the others: token and place
    uint2* to;
    int* counts;  // tiles x kBins
    int n, tiles, per, shift;
    int* joins;  // how many rows a later kernel joins: set to none by the first launch
    float4* zeros;  // what further CTAs fill
    long long zero_packs;
    int zero_rest;  // bytes behind those
};

__device__ __forceinline__ uint2 entry(const Sorting& s, int i) {
    if (s.from) return __ldcg(s.from + i);  // (written in this launch, or the one before)
    const long long r = row_of(s.tokens, s.wide, i, s.V);
    return make_uint2((unsigned)(r < 0 ? s.V : r), (unsigned)i);  // strangers behind all others
}

__device__ __forceinline__ void fill_zeros(const Sorting& s) {
    const long long ctas = gridDim.x - s.tiles;
    for (long long i = (blockIdx.x - s.tiles) * (long long)blockDim.x + threadIdx.x; i < s.zero_packs;
         i += ctas * blockDim.x)
        s.zeros[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (blockIdx.x == (unsigned)s.tiles && threadIdx.x < (unsigned)s.zero_rest)
        reinterpret_cast<char*>(s.zeros + s.zero_packs)[threadIdx.x] = 0;
}

__global__ void __launch_bounds__(kSort) count_kernel(const Sorting s) {
    pdl_trigger();
    if (blockIdx.x == 0 && threadIdx.x == 0 && !s.from) *s.joins = 0;
    if (blockIdx.x >= (unsigned)s.tiles) return fill_zeros(s);  // (dW is this call's own since its first launch)
    __shared__ int count[kBins];
    for (int i = threadIdx.x; i < kBins; i += blockDim.x) count[i] = 0;
    __syncthreads();
    pdl_wait();
    const int lo = blockIdx.x * s.per, hi = min(s.n, lo + s.per);
    for (int i = lo + threadIdx.x; i < hi; i += blockDim.x) atomicAdd(&count[entry(s, i).x >> s.shift & (kBins - 1)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += blockDim.x) s.counts[blockIdx.x * kBins + i] = count[i];
}

// What placing a tile's tokens keeps in shared memory.
struct Placing {
    int at[kBins];                      // where the next token of each bin goes
    int seen[kSort / 32][kBins];        // of a warp, in this round
    int part[kSort / kBins][kBins][2];  // of the counts: of all tiles, of those before this one
    int warp_sum[kBins / 32];
};

// at: behind the tokens of lower bins, and of earlier tiles; count(t, bin) is tile t's.
template <typename F>
__device__ __forceinline__ void first_places(Placing& m, int tile, int tiles, F&& count) {
    constexpr int PARTS = kSort / kBins;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, bin = tid % kBins;
    int all = 0, before = 0;
#pragma unroll 16
    for (int t = tid / kBins; t < tiles; t += PARTS) {
        const int c = count(t, bin);
        all += c;
        before += t < tile ? c : 0;
    }
    m.part[tid / kBins][bin][0] = all;
    m.part[tid / kBins][bin][1] = before;
    __syncthreads();
    int sum = 0;
    if (tid < kBins) {
        all = before = 0;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) all += m.part[p][tid][0], before += m.part[p][tid][1];
        sum = all;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, sum, d);
            if (lane >= d) sum += y;
        }
        if (lane == 31) m.warp_sum[warp] = sum;
    }
    __syncthreads();
    if (tid < kBins) {
        for (int w = 0; w < warp; ++w) sum += m.warp_sum[w];
        m.at[tid] = sum - all + before;
    }
    __syncthreads();
}

// Places tokens [lo, hi): a thread for each, kSort at a time, in their order.
__device__ __forceinline__ void place_tokens(Placing& m, const Sorting& s, int lo, int hi) {
    constexpr int WARPS = kSort / 32;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (int base = lo; base < hi; base += kSort) {
        for (int j = tid; j < WARPS * kBins; j += kSort) (&m.seen[0][0])[j] = 0;
        __syncthreads();
        const int i = base + tid;
        const bool in = i < hi;
        const uint2 e = in ? entry(s, i) : make_uint2(0, 0);
        const unsigned d = e.x >> s.shift & (kBins - 1);
        const unsigned peers = __match_any_sync(0xffffffffu, in ? d : kBins);
        const int rank = __popc(peers & ((1u << lane) - 1));
        if (in && rank == 0) m.seen[warp][d] = __popc(peers);
        __syncthreads();
        if (tid < kBins) {  // counts of the warps become their first places
            int next = m.at[tid];
#pragma unroll 8
            for (int w = 0; w < WARPS; ++w) {
                const int c = m.seen[w][tid];
                m.seen[w][tid] = next;
                next += c;
            }
            m.at[tid] = next;
        }
        __syncthreads();
        if (in) s.to[m.seen[warp][d] + rank] = e;
        __syncthreads();
    }
}

__global__ void __launch_bounds__(kSort) place_kernel(const Sorting s) {
    pdl_trigger();
    if (blockIdx.x >= (unsigned)s.tiles) return fill_zeros(s);
    __shared__ Placing m;
    pdl_wait();
    first_places(m, blockIdx.x, s.tiles, [&](int t, int bin) { return s.counts[t * kBins + bin]; });
    const int lo = blockIdx.x * s.per;
    place_tokens(m, s, lo, min(s.n, lo + s.per));
}

// All passes in one launch: the first cluster sorts, each of its CTAs a tile, the
// others fill zeros.
constexpr int kCluster = 8, kNear = kCluster * kSort;

__global__ void __launch_bounds__(kSort) __cluster_dims__(kCluster, 1, 1)
sort_kernel(Sorting s, uint2* list0, uint2* list1, int passes) {
    pdl_trigger();
    if (blockIdx.x >= kCluster) return fill_zeros(s);
    __shared__ Placing m;
    __shared__ int count[kBins];
    const int tile = blockIdx.x, lo = min(s.n, tile * s.per), hi = min(s.n, lo + s.per);
    if (tile == 0 && threadIdx.x == 0) *s.joins = 0;
    for (int p = 0; p < passes; ++p) {
        s.shift = 8 * p;
        s.from = p == 0 ? nullptr : p & 1 ? list0 : list1;
        s.to = p & 1 ? list1 : list0;
        for (int i = threadIdx.x; i < kBins; i += kSort) count[i] = 0;
        __syncthreads();
        for (int i = lo + threadIdx.x; i < hi; i += kSort)
            atomicAdd(&count[entry(s, i).x >> s.shift & (kBins - 1)], 1);
        cluster_sync();
        first_places(m, tile, kCluster, [&](int t, int bin) {
            int c;
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(c) : "r"(dsmem_addr(&count[bin], t)) : "memory");
            return c;
        });
        cluster_sync();  // (the counts are read: they may be overwritten)
        place_tokens(m, s, lo, hi);
        __threadfence();
        cluster_sync();  // every token is in its place
    }
}

// --------------------------------------------------------------------- sums
// The sorted tokens in chunks of `per`. A row whose tokens are at most `per`
// belongs to the chunk in which they begin, and is written by it; those of a
// longer one are summed up to each chunk's border and joined by a second
// kernel: a piece that began in its chunk lies in slot 2 c + 1, one that goes
// on in it from the last in slot 2 c.
constexpr int kMaxChunk = 512;
constexpr int kColumns = 128;  // threads of a CTA, each with a pack of columns

struct Summing {
    const uint2* sorted;
    int n, per;
    long long V, ld;
    int D;
    float* pieces;  // slots x D
    int *joins, *list;  // the chunks in which a row of several pieces begins, in any order
    float scale;
};

template <typename T, int N>
__global__ void __launch_bounds__(kColumns) sum_kernel(const Summing s, const T* dout, T* dW) {
    pdl_trigger();
    pdl_wait();
    extern __shared__ uint2 window[];  // sorted tokens [a - per, b + per + 1)
    __shared__ int first_, last_;
    const int per = s.per, a = blockIdx.x * per, b = min(s.n, a + per), w0 = max(0, a - per);
    const int w1 = (int)min((long long)s.n, (long long)b + per + 1);
    for (int i = w0 + threadIdx.x; i < w1; i += kColumns) window[i - w0] = s.sorted[i];
    if (threadIdx.x == 0) first_ = a, last_ = b;
    __syncthreads();
    const auto key = [&](int i) { return window[i - w0].x; };
    // where the tokens of the row of token i (in the chunk) begin, or a - per
    const auto begin_of = [&](int i) {
        const unsigned r = key(i);
        int lo = w0, hi = i;  // the first of r in [w0, i]
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (key(mid) >= r)
                hi = mid;
            else
                lo = mid + 1;
        }
        return lo;
    };
    const auto long_row = [&](int begin, unsigned r) { return (long long)begin + per < w1 && key(begin + per) == r; };
    const unsigned ra = key(a), rb = key(b - 1);
    const bool on = a > 0 && key(a - 1) == ra;  // the first row began before
    const int sa = begin_of(a), sb = begin_of(b - 1);
    // (where it began at or before w0 > 0, token a itself is `per` behind w0: long)
    const bool long_a = long_row(sa, ra), long_b = long_row(sb, rb);
    if (on && !long_a)
        for (int i = a + threadIdx.x; i < w1; i += kColumns)
            if (key(i) != ra && key(i - 1) == ra) first_ = i;
    if (on && !long_a && threadIdx.x == 0 && key(w1 - 1) == ra) first_ = w1;  // none behind it
    if (b < s.n && key(b) == rb && !long_b)
        for (int i = b + threadIdx.x; i < w1; i += kColumns)
            if (key(i - 1) == rb && (i + 1 == w1 || key(i + 1) != rb) && key(i) == rb) last_ = i + 1;
    __syncthreads();
    const bool cut = b < s.n && key(b) == rb && long_b;  // the last row goes on behind
    if (cut && rb < s.V && !(on && ra == rb) && blockIdx.y == 0 && threadIdx.x == 0)
        s.list[atomicAdd(s.joins, 1)] = blockIdx.x;
    const int first = first_;
    int last = last_;
    if (key(last - 1) >= s.V) {  // strangers are no one's
        int lo = first < last ? first : last, hi = last;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (key(mid) >= s.V)
                hi = mid;
            else
                lo = mid + 1;
        }
        last = lo;
    }
    const int col = (blockIdx.y * kColumns + threadIdx.x) * N;
    // (a short row's tokens behind b are this chunk's only if they begin in it)
    if (first >= b || first >= last || col >= s.D) return;
    constexpr int U = 8;
    const T* const from = dout + col;
    float sum[N] = {};
    for (int i0 = first; i0 < last; i0 += U) {
        Pack<T, N> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            x[u] = *reinterpret_cast<const Pack<T, N>*>(from + (long long)window[min(i0 + u, last - 1) - w0].y * s.ld);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u;
            if (i < last) {
#pragma unroll
                for (int k = 0; k < N; ++k) sum[k] += to_f(x[u].v[k]);
                const unsigned r = key(i);
                if (i + 1 == last || key(i + 1) != r) {  // the row's last token in this chunk
                    const bool head = on && long_a && r == ra, tail = cut && r == rb;
                    if (head || tail) {
                        float* to = s.pieces + (2ll * blockIdx.x + (head ? 0 : 1)) * s.D + col;
#pragma unroll
                        for (int k = 0; k < N; ++k) to[k] = sum[k];
                    } else {
                        Pack<T, N> y;
#pragma unroll
                        for (int k = 0; k < N; ++k) y.v[k] = from_f<T>(sum[k] * s.scale);
                        *reinterpret_cast<Pack<T, N>*>(dW + (long long)r * s.D + col) = y;
                    }
#pragma unroll
                    for (int k = 0; k < N; ++k) sum[k] = 0.0f;
                }
            }
        }
    }
}

// The pieces of the rows that have several, a slab of 128 columns of a row at a
// time: each warp takes every kJoin-th piece, and the warps' sums are added in
// their order.
constexpr int kJoin = 8;  // warps

template <typename T>
__global__ void __launch_bounds__(kJoin * 32) join_kernel(const Summing s, T* dW) {
    pdl_wait();
    __shared__ float part[kJoin][128];
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, slabs = (s.D + 127) / 128, todo = *s.joins * slabs;
    for (int item = blockIdx.x; item < todo; item += gridDim.x) {
        const int first = s.list[item / slabs], col = item % slabs * 128 + l;
        const unsigned r = s.sorted[(first + 1) * s.per].x;  // (it goes on in the next chunk)
        // the last chunk whose first token is the row's: 32 places of what is left at once
        int last = first + 1, hi = (s.n - 1) / s.per;
        while (last < hi) {
            const int step = (hi - last + 32) / 32, m = last + l * step;
            const int yes = __popc(__ballot_sync(0xffffffffu, m <= hi && s.sorted[min(m, hi) * s.per].x == r));
            last += (yes - 1) * step;
            hi = min(hi, last + step - 1);
        }
        float sum[4] = {};
#pragma unroll 8
        for (int c = first + warp; c <= last; c += kJoin) {
            const float* from = s.pieces + (2ll * c + (c == first)) * s.D;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (col + k * 32 < s.D) sum[k] += from[col + k * 32];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) part[warp][k * 32 + l] = sum[k];
        __syncthreads();
        const int c = item % slabs * 128 + threadIdx.x;
        if (threadIdx.x < 128 && c < s.D) {
            float x = part[0][threadIdx.x];
#pragma unroll
            for (int w = 1; w < kJoin; ++w) x += part[w][threadIdx.x];
            dW[(long long)r * s.D + c] = from_f<T>(x * s.scale);
        }
        __syncthreads();
    }
}

template <typename... P, typename... A>
int launch_behind(void (*kernel)(P...), dim3 ctas, int threads, int smem, cudaStream_t st, A... args) {
    return cuda_check(launch_pdl(kernel, ctas, dim3(threads), smem, st, args...), "embedding launch");
}

// Bytes of the widest access that fits addresses, strides and width.
int width_of(const void* a, const void* b, long long ld, int D, unsigned e) {
    int w = 16;
    while (w > (int)e && ((uintptr_t)a % w || (uintptr_t)b % w || ld * e % w || (long long)D * e % w)) w /= 2;
    return w;
}

template <typename F>
int by_type(int dtype, F&& f) {
    return dtype == SN_F32 ? f(0.0f) : dtype == SN_BF16 ? f(__nv_bfloat16()) : f(__half());
}
// f(type, values of an access)
template <typename F>
int by_access(int dtype, int width, F&& f) {
    return by_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        constexpr int E = sizeof(T);
        if (width == 16) return f(t, std::integral_constant<int, 16 / E>());
        if (width == 8) return f(t, std::integral_constant<int, 8 / E>());
        if constexpr (E == 2)
            if (width == 4) return f(t, std::integral_constant<int, 2>());
        return f(t, std::integral_constant<int, 1>());
    });
}

// (tokens: their indexes plus a tile's stay in 31 bits; columns: a grid's second axis)
constexpr long long kMostTokens = 0x7ffff000;
constexpr int kMostColumns = 1 << 22;

int check_call(const char* what, int64_t n, int64_t V, int32_t D, int64_t ld, int32_t dtype, float scale) {
    if (!dtype_size(dtype)) return fail(SN_E_INVAL, "%s: dtype %d", what, dtype);
    if (n < 0 || V < 0 || D < 0 || n > kMostTokens || V >= 0x7fffffffll || D > kMostColumns)
        return fail(SN_E_INVAL, "%s: %lld tokens, %lld rows of %d", what, (long long)n, (long long)V, D);
    if (ld < 0 || ld >= 1ll << 44) return fail(SN_E_INVAL, "%s: rows %lld values apart", what, (long long)ld);
    if (!std::isfinite(scale)) return fail(SN_E_INVAL, "%s: the scale is not finite", what);
    return SN_OK;
}

// How the tokens are cut up, and the workspace in bytes.
struct Plan {
    int tiles, per, passes, chunk;
    long long chunks, list, counts, joins, pieces, bytes;
};
Plan plan_of(long long n, long long V, int D) {
    Plan p;
    const auto up = [](long long b) { return (b + 255) / 256 * 256; };
    p.tiles = n <= kNear ? kCluster : (int)std::min((long long)kTiles, (n + kSort - 1) / kSort);
    p.per = (int)((n + p.tiles - 1) / p.tiles);
    p.passes = 1;
    while (V >> 8 * p.passes) ++p.passes;  // (V itself marks strangers)
    // about 14 chunks to an SM, of 16 tokens at least
    p.chunk = 16;
    while (p.chunk < kMaxChunk && (n + p.chunk - 1) / p.chunk > 148 * 14) p.chunk *= 2;
    p.chunks = (n + p.chunk - 1) / p.chunk;
    p.list = up(n * 8);
    p.counts = up((long long)p.tiles * kBins * 4);
    p.joins = up((p.chunks + 1) * 4);
    p.pieces = up(p.chunks * 2 * D * 4);
    p.bytes = 2 * p.list + p.counts + p.joins + p.pieces;
    return p;
}

}  // namespace
}  // namespace sn

using namespace sn;

extern "C" {

sn_status sn_abi_embedding(const void* tokens, int32_t token_bits, int64_t n, const void* W, int64_t ld, int64_t V,
                           int32_t D, int32_t dtype, float scale, void* out, void* cuda_stream) {
    CallerDevice dev;
    SN_TRY(check_call("embedding", n, V, D, ld, dtype, scale));
    if (token_bits != 32 && token_bits != 64) return fail(SN_E_INVAL, "embedding: tokens have 32 or 64 bits");
    if (!n || !D) return SN_OK;
    if (!tokens || !out || (V && !W)) return fail(SN_E_INVAL, "embedding: null pointer");
    const unsigned e = dtype_size(dtype);
    SN_TRY(dev.enter("embedding", {{tokens, (unsigned)token_bits / 8}, {W, e}, {out, e}}));
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    return by_access(dtype, width_of(W, out, ld, D, e), [&](auto t, auto vec) {
        typedef decltype(t) T;
        constexpr int N = decltype(vec)::value;
        const auto go = [&](auto lanes) {
            constexpr int L = decltype(lanes)::value;
            rows_kernel<T, N, L><<<(unsigned)((n * L + kThreads - 1) / kThreads), kThreads, 0, st>>>(
                tokens, token_bits == 64, static_cast<const T*>(W), ld, V, static_cast<T*>(out), n, D, scale);
        };
        // a warp to a row, or as many lanes as it has packs
        if (D / N > 16)
            go(std::integral_constant<int, 32>());
        else if (D / N > 4)
            go(std::integral_constant<int, 8>());
        else
            go(std::integral_constant<int, 2>());
        return cuda_check(cudaGetLastError(), "embedding launch");
    });
}

int64_t sn_abi_embedding_bwd_ws(int64_t n, int64_t V, int32_t D) {
    if (check_call("embedding_bwd_ws", n, V, D, 0, SN_F32, 1.0f) != SN_OK) return -1;
    return n && V && D ? plan_of(n, V, D).bytes : 0;
}

sn_status sn_abi_embedding_bwd(const void* tokens, int32_t token_bits, int64_t n, const void* dout, int64_t ld,
                               int64_t V, int32_t D, int32_t dtype, float scale, void* dW, void* ws,
                               int64_t ws_bytes, void* cuda_stream) {
    CallerDevice dev;
    SN_TRY(check_call("embedding_bwd", n, V, D, ld, dtype, scale));
    if (token_bits != 32 && token_bits != 64) return fail(SN_E_INVAL, "embedding_bwd: tokens have 32 or 64 bits");
    if (!V || !D) return SN_OK;
    if (!dW || (n && (!tokens || !dout))) return fail(SN_E_INVAL, "embedding_bwd: null pointer");
    const unsigned e = dtype_size(dtype);
    SN_TRY(dev.enter("embedding_bwd",
                     {{tokens, n ? (unsigned)token_bits / 8 : 1}, {dout, n ? e : 1}, {dW, e}, {ws, 16}}));
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    const long long bytes = V * (long long)D * e;
    if (!n) return cuda_check(cudaMemsetAsync(dW, 0, bytes, st), "embedding_bwd");
    const Plan p = plan_of(n, V, D);
    if (!ws || ws_bytes < p.bytes)
        return fail(SN_E_INVAL, "embedding_bwd: a workspace of %lld bytes is wanted", p.bytes);
    char* at = static_cast<char*>(ws);
    uint2* lists[2] = {reinterpret_cast<uint2*>(at), reinterpret_cast<uint2*>(at + p.list)};
    Sorting s = {};
    s.tokens = tokens, s.wide = token_bits == 64, s.V = V;
    s.counts = reinterpret_cast<int*>(at + 2 * p.list);
    s.joins = reinterpret_cast<int*>(at + 2 * p.list + p.counts);
    s.n = (int)n, s.tiles = p.tiles, s.per = p.per;
    // the zeros, a part to each launch; where they do not begin at a pack, by one of their own
    const int launches = n <= kNear ? 1 : 2 * p.passes;
    const bool packed = (uintptr_t)dW % 16 == 0;
    const long long packs = packed ? bytes / 16 : 0, share = (packs + launches - 1) / launches;
    if (!packed) SN_TRY(cuda_check(cudaMemsetAsync(dW, 0, bytes, st), "embedding_bwd"));
    long long done = 0;
    const auto zeros = [&] {
        s.zeros = reinterpret_cast<float4*>(dW) + done;
        s.zero_packs = std::min(share, packs - done);
        done += s.zero_packs;
        s.zero_rest = packed && done == packs ? (int)(bytes % 16) : 0;
        return (unsigned)std::min((s.zero_packs + 4095) / 4096 + (s.zero_rest > 0), 148ll * 4);
    };
    if (n <= kNear) {
        const unsigned more = (zeros() + kCluster - 1) / kCluster * kCluster;
        sort_kernel<<<kCluster + more, kSort, 0, st>>>(s, lists[0], lists[1], p.passes);
        SN_TRY(cuda_check(cudaGetLastError(), "embedding launch"));
    } else {
        for (int i = 0; i < p.passes; ++i) {
            s.shift = 8 * i;
            s.from = i ? lists[(i - 1) & 1] : nullptr;
            s.to = lists[i & 1];
            unsigned more = zeros();
            if (i == 0) {
                count_kernel<<<p.tiles + more, kSort, 0, st>>>(s);
                SN_TRY(cuda_check(cudaGetLastError(), "embedding launch"));
            } else {
                SN_TRY(launch_behind(count_kernel, dim3(p.tiles + more), kSort, 0, st, s));
            }
            more = zeros();
            SN_TRY(launch_behind(place_kernel, dim3(p.tiles + more), kSort, 0, st, s));
        }
    }
    Summing m = {};
    m.sorted = lists[(p.passes - 1) & 1];
    m.n = (int)n, m.per = p.chunk, m.V = V, m.ld = ld, m.D = D;
    m.joins = s.joins, m.list = s.joins + 1;
    m.pieces = reinterpret_cast<float*>(at + 2 * p.list + p.counts + p.joins);
    m.scale = scale;
    SN_TRY(by_access(dtype, width_of(dout, dW, ld, D, e), [&](auto t, auto vec) {
        typedef decltype(t) T;
        constexpr int N = decltype(vec)::value;
        const unsigned slabs = (unsigned)((D / N + kColumns - 1) / kColumns);
        return launch_behind(sum_kernel<T, N>, dim3((unsigned)p.chunks, slabs), kColumns, (3 * p.chunk + 1) * 8, st, m,
                             static_cast<const T*>(dout), static_cast<T*>(dW));
    }));
    return by_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        const long long most = (p.chunks + 1) / 2 * ((D + 127) / 128);  // (a row of several pieces has two chunks)
        return launch_behind(join_kernel<T>, dim3((unsigned)std::min(most, 148ll * 8)), kJoin * 32, 0, st, m,
                             static_cast<T*>(dW));
    });
}

}  // extern "C"
