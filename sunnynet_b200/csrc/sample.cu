// The next token of each row of logits, drawn with temperature, top-k, top-p
// and min-p from given uniform numbers: the rule of the reference's
// sample_logits (serve.py:30-57, numpy on the host, row by row) plus min-p.
//
//   T <= 0: the lowest id of the largest logit. Otherwise
//   w_i = exp((x_i - max) / T)                        weight of id i
//   top-k: ids with x_i >= the k-th largest logit     (equal ones all stay)
//   top-p: of those in descending order, equal ones by id, each id whose
//          predecessors weigh less than p of them all
//   min-p: ids with w_i >= min_p                      (max has weight 1)
//   token: the first id, by id, whose weight and those before it exceed u
//          times the kept weight.
//
// Which id a draw meets is decided by differences between sums, so weights
// are whole numbers: w_i * 2^44 (2^44 = the largest logit's; fewer bits above
// 2^18 ids, so that a row's sum stays below 2^62), from an exponential in 64
// bits that is right to 2^-46. Their sums are exact in any order: the result
// depends on no scheduling, and differs from the rule in real numbers only
// where u meets a border to about 2^-40.
//
// A row is read from HBM once, by a cluster of 1 to 8 CTAs that each keep a
// slice of it in shared memory as order-preserving 32-bit keys. Neither top-k
// nor top-p sorts: both look for one border key, the largest with "count (or
// weight) of the larger keys < target <= that plus its own". A histogram over
// 512 bins between the row's largest logit and the point where weights vanish
// gives the border's bin; the bin's few keys are gathered and compared with
// one another. A bin of more than kList keys is cut into 512 bins again, by
// key, until it is small or holds a single key (at most five rounds). The
// CTAs of a cluster read one another's histograms and lists through
// distributed shared memory and come to the same border by themselves.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>

#include "caller.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace sn {
namespace {

typedef unsigned long long u64;
typedef unsigned int u32;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kBins = 512;     // two to a thread
constexpr int kList = 256;     // keys resolved by comparing them all: one to a thread
constexpr int kMaxCluster = 8;
constexpr u32 kNothing = 0x007fffffu;  // key of -infinity (and of NaN)
constexpr u32 kInfinite = 0xff800000u; // key of +infinity

struct Setting {  // one value, or one for each row
    const double* rows;
    double one;
    __device__ double at(int r) const { return rows ? rows[r] : one; }
};

struct SampleArgs {
    const void* logits;
    const void* u;
    const int* top_k;
    int32_t* out;
    Setting temperature, top_p, min_p;
    long long ld;
    int one_k, u_wide, V, slice, bits;
};

// Bits of x ordered like the numbers, -0 taken for 0 and NaN for -infinity.
__device__ __forceinline__ u32 key_of(float x) {
    if (!(x == x)) return kNothing;
    const u32 b = __float_as_uint(x + 0.0f);
    return b ^ ((u32)((int)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ float value_of(u32 k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ u32 peer_u32(const u32* local, u32 rank) {
    u32 v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(dsmem_addr(local, rank)) : "memory");
    return v;
}

__device__ __forceinline__ void peer_store(u64* local, u32 rank, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dsmem_addr(local, rank)), "l"(v)
                 : "memory");
}

struct Shared {
    double pow16[16];        // 2^(j/16)
    u64 told[9][kMaxCluster];  // a value of each CTA, one line per exchange
    u64 red[kWarps];
    u64 warp_sum[kWarps];
    u32 lo[kBins], hi[kBins];  // a bin's count or weight, as two words
    u32 list[2][kList], listed[2];  // keys of the border's bin, of top-k and of top-p
    u32 least, most;         // their range
    u32 all[kList];          // every CTA's list
    u64 weight[kList];
    u64 found[4];
};

// One row's numbers, the same in every thread of the cluster.
struct Row {
    double max, scale;  // w = 2^((x - max) * scale)
    int shift;          // 52 - bits
    float max_f, bin;   // linear bins: (max - x) * bin
};

// 2^((x - max) * scale) * 2^bits, cut to a whole number. The fraction f of the
// exponent in 16ths is left to the exponential series of f ln2 / 16 < 0.0434:
// its eighth term is below 2^-51.
__device__ __forceinline__ u64 weigh(const Row& r, const Shared& s, u32 key) {
    const double d = ((double)value_of(key) - r.max) * r.scale;
    if (!(d >= -64.0)) return 0;  // too far below, -infinity among them
    const double n = floor(d * 16.0);
    const double f = fma(n, -0.0625, d) * 0.69314718055994530942;
    double e = 1.0 / 5040;
    e = fma(e, f, 1.0 / 720);
    e = fma(e, f, 1.0 / 120);
    e = fma(e, f, 1.0 / 24);
    e = fma(e, f, 1.0 / 6);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
    e = fma(e, f, 1.0);
    const int i = (int)n;  // -1024 .. 0
    const u64 v = (u64)__double_as_longlong(e * s.pow16[i & 15]);  // near [1, 2)
    const u64 m = (v & 0xfffffffffffffull) | 0x10000000000000ull;
    const int sh = r.shift + 1023 - (int)(v >> 52) - (i >> 4);
    return sh < 64 ? m >> sh : 0;
}

__device__ __forceinline__ int linear_bin(const Row& r, float x) {
    return (int)fminf((r.max_f - x) * r.bin, (float)(kBins - 1));
}

// A barrier over the CTAs of a row.
__device__ __forceinline__ void row_sync(u32 ctas) {
    if (ctas == 1)
        __syncthreads();
    else
        cluster_sync();
}

__device__ __forceinline__ u64 warp_max(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const u64 w = __shfl_xor_sync(0xffffffffu, v, o);
        v = w > v ? w : v;
    }
    return v;
}

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ u64 warp_upto(u64 v) {  // inclusive prefix sum
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 w = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += w;
    }
    return v;
}

// Inclusive prefix sum over the CTA's threads.
__device__ __forceinline__ u64 block_upto(Shared& s, u64 v) {
    v = warp_upto(v);
    const int w = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 31) s.red[w] = v;
    __syncthreads();
    for (int k = 0; k < w; ++k) v += s.red[k];
    __syncthreads();  // red is free again
    return v;
}

template <typename T>
__device__ __forceinline__ float number(T v);
template <>
__device__ __forceinline__ float number<float>(float v) { return v; }
template <>
__device__ __forceinline__ float number<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float number<__half>(__half v) { return __half2float(v); }

// A CTA's slice [first, first + n) of a row: its keys from shared memory, or
// (rows too long for it) from the logits again.
template <typename T, bool HELD>
struct Slice {
    const T* x;
    const u32* held;
    int n, first;
    __device__ __forceinline__ u32 operator[](int i) const {
        return HELD ? held[i] : key_of(number<T>(x[i]));
    }
};

// What the border of top-k or top-p is.
struct Border {
    u32 key;
    u64 ahead;  // count or weight of the larger keys
    u64 ties;   // ids that have this key
    u64 target;
};

// The weight that top-p's ids have to reach: p of the whole, at least 1 (the
// largest logit's id always stays).
__device__ __forceinline__ u64 share(double p, u64 whole) {
    const double want = ceil(p * (double)whole);
    return want < 1.0 ? 1 : want < (double)whole ? (u64)want : whole;
}

// The border key: count (or, BY_WEIGHT, weight) of larger keys < target <=
// that and its own. Candidates are keys >= floor; `few`: they are known to
// be kList at most. BY_WEIGHT the target is p of all candidates' weight.
template <bool BY_WEIGHT, typename S>
__device__ Border border(Shared& s, const Row& r, const S& x, u32 floor_key, u32 top, u64 target,
                         double p, bool few, u32 rank, u32 ctas) {
    const int tid = threadIdx.x;
    u32* list = s.list[BY_WEIGHT];
    u64(*told)[kMaxCluster] = s.told + (BY_WEIGHT ? 4 : 1);  // three lines
    u32 from = floor_key, to = top;
    u64 base = 0;
    int shift = -1;  // -1: linear bins
    int bin = -1;
    for (;;) {
        if (!few) {
            for (int b = tid; b < kBins; b += kThreads) s.lo[b] = s.hi[b] = 0;
            __syncthreads();
            for (int i = tid; i < x.n; i += kThreads) {
                const u32 k = x[i];
                if (k < from || k > to) continue;
                const int b = shift < 0 ? linear_bin(r, value_of(k)) : (int)((to - k) >> shift);
                if (BY_WEIGHT) {
                    const u64 w = weigh(r, s, k);
                    const u32 a = (u32)w, old = atomicAdd(&s.lo[b], a);
                    const u32 c = (u32)(w >> 32) + (old + a < old ? 1u : 0u);
                    if (c) atomicAdd(&s.hi[b], c);
                } else {
                    atomicAdd(&s.lo[b], 1u);
                }
            }
            row_sync(ctas);
            u64 v[2] = {0, 0};
            for (u32 c = 0; c < ctas; ++c)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int b = 2 * tid + j;
                    v[j] += (u64)peer_u32(&s.lo[b], c);
                    if (BY_WEIGHT) v[j] += (u64)peer_u32(&s.hi[b], c) << 32;
                }
            const u64 upto = block_upto(s, v[0] + v[1]);
            if (BY_WEIGHT && target == 0) {
                if (tid == kThreads - 1) s.found[0] = upto;
                __syncthreads();
                target = share(p, s.found[0]);
                __syncthreads();
            }
            const u64 before = upto - v[0] - v[1];
            if (base + before < target && target <= base + upto) {
                const bool second = base + before + v[0] < target;
                s.found[0] = second ? before + v[0] : before;
                s.found[1] = 2 * tid + second;
            }
            __syncthreads();
            base += s.found[0];
            bin = (int)s.found[1];
        }
        // the keys of the bin: their number and range, and themselves while there is room
        if (tid == 0) s.listed[BY_WEIGHT] = 0, s.least = 0xffffffffu, s.most = 0;
        __syncthreads();
        u32 least = 0xffffffffu, most = 0;
        for (int i = tid; i < x.n; i += kThreads) {
            const u32 k = x[i];
            if (k < from || k > to) continue;
            if (!few &&
                (shift < 0 ? linear_bin(r, value_of(k)) : (int)((to - k) >> shift)) != bin)
                continue;
            least = min(least, k);
            most = max(most, k);
            const u32 at = atomicAdd(&s.listed[BY_WEIGHT], 1u);
            if (at < kList) list[at] = k;
        }
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        if ((tid & 31) == 0) {
            atomicMin(&s.least, least);
            atomicMax(&s.most, most);
        }
        __syncthreads();
        if (tid < (int)ctas) {
            peer_store(&told[0][rank], tid, s.listed[BY_WEIGHT]);
            peer_store(&told[1][rank], tid, s.least);
            peer_store(&told[2][rank], tid, s.most);
        }
        row_sync(ctas);
        u64 count = 0;
        for (u32 c = 0; c < ctas; ++c) {
            count += told[0][c];
            least = min(least, (u32)told[1][c]);
            most = max(most, (u32)told[2][c]);
        }
        from = __reduce_min_sync(0xffffffffu, least);
        to = __reduce_max_sync(0xffffffffu, most);
        if (from == to) {  // one key, however often
            if (BY_WEIGHT && target == 0) target = share(p, count * weigh(r, s, from));
            return {from, base, count, target};
        }
        if (count <= kList) {
            u32 at = 0;
            for (u32 c = 0; c < ctas; ++c) {
                const u32 n = (u32)told[0][c];
                for (u32 j = tid; j < n; j += kThreads) s.all[at + j] = peer_u32(&list[j], c);
                at += n;
            }
            __syncthreads();
            const bool in = tid < (int)count;
            const u32 mine = in ? s.all[tid] : 0;
            if (BY_WEIGHT) {
                const u64 w = in ? weigh(r, s, mine) : 0;
                s.weight[tid] = w;
                if (target == 0) {  // p of the listed candidates
                    const u64 upto = block_upto(s, w);
                    if (tid == kThreads - 1) s.found[0] = upto;
                    __syncthreads();
                    target = share(p, s.found[0]);
                }
                __syncthreads();
            }
            if (in) {
                u64 more = 0, own = 0, ties = 0;
                for (int j = 0; j < (int)count; ++j) {
                    const u32 k = s.all[j];
                    const u64 w = BY_WEIGHT ? s.weight[j] : 1;
                    more += k > mine ? w : 0;
                    own += k == mine ? w : 0;
                    ties += k == mine;
                }
                if (base + more < target && target <= base + more + own) {  // all its ties say the same
                    s.found[1] = mine;
                    s.found[2] = base + more;
                    s.found[3] = ties;
                }
            }
            __syncthreads();
            return {(u32)s.found[1], s.found[2], s.found[3], target};
        }
        const u32 span = to - from;
        shift = max(0, 32 - __clz(span) - 9);  // span >> shift < 512
        few = false;
    }
}

// First id, by id, at which the running sum of measure(i, key) over the row
// exceeds the target that aim(total) gives; -1 in CTAs that do not hold it.
template <typename S, typename M, typename A>
__device__ int first_beyond(Shared& s, const S& x, u64* told, u32 rank, u32 ctas, M measure,
                            A aim) {
    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
    const int part = (x.n + kThreads - 1) / kThreads * 32;  // a warp's run of ids
    const int lo = min(w * part, x.n), hi = min(lo + part, x.n);
    u64 sum = 0;
    for (int i = lo + lane; i < hi; i += 32) sum += measure(i, x[i]);
    sum = warp_add(sum);
    if (lane == 0) s.warp_sum[w] = sum;
    __syncthreads();
    u64 mine = 0;
    for (int k = 0; k < kWarps; ++k) mine += s.warp_sum[k];
    if (tid < (int)ctas) peer_store(told + rank, tid, mine);
    row_sync(ctas);
    u64 total = 0, before = 0;
    for (u32 c = 0; c < ctas; ++c) {
        if (c == rank) before = total;
        total += told[c];
    }
    const u64 target = aim(total);
    if (target < before || target >= before + mine) return -1;
    int k = 0;
    while (target >= before + s.warp_sum[k]) before += s.warp_sum[k++];
    // the run of warp k, a few ids to each thread
    const int a = min(k * part, x.n), b = min(a + part, x.n);
    const int n = (b - a + kThreads - 1) / kThreads;
    const int from = min(a + tid * n, b), to = min(from + n, b);
    sum = 0;
    for (int i = from; i < to; ++i) sum += measure(i, x[i]);
    u64 upto = before + block_upto(s, sum);
    if (tid == 0) s.found[0] = ~0ull;
    __syncthreads();
    if (target < upto && target >= upto - sum) {
        u64 at = upto - sum;
        int i = from;
        for (; i < to - 1; ++i) {
            at += measure(i, x[i]);
            if (at > target) break;
        }
        s.found[0] = (u64)i;
    }
    __syncthreads();
    return (int)s.found[0];
}

template <typename T, bool HELD>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) u32 held[];
    __shared__ Shared s;
    const int tid = threadIdx.x;
    const u32 ctas = cluster_size(), rank = cluster_rank();
    const int row = blockIdx.x / ctas;
    Slice<T, HELD> x;
    x.first = min((long long)rank * a.slice, (long long)a.V);
    x.n = min(a.slice, a.V - x.first);
    x.x = static_cast<const T*>(a.logits) + row * a.ld + x.first;
    x.held = held;
    if (tid < 16) s.pow16[tid] = exp2(tid / 16.0);

    // keys, the largest with its lowest id, the smallest above -infinity
    u64 best = 0;
    u32 least = 0xffffffffu;
    const auto take = [&](int i, float v) {
        const u32 k = key_of(v);
        if (HELD) held[i] = k;
        const u64 c = (u64)k << 32 | (0xffffffffu - (u32)(x.first + i));
        best = c > best ? c : best;
        if (k > kNothing) least = min(least, k);
    };
    {
        constexpr int P = 16 / sizeof(T), U = 4;
        struct alignas(16) Pack {
            T v[P];
        };
        const int head = min(x.n, (int)((16 - ((uintptr_t)x.x & 15)) % 16 / sizeof(T)));
        const int packs = (x.n - head) / P;
        const Pack* px = reinterpret_cast<const Pack*>(x.x + head);
        for (int q = tid; q < packs; q += U * kThreads) {
            Pack v[U];
#pragma unroll
            for (int j = 0; j < U; ++j)
                if (q + j * kThreads < packs) v[j] = px[q + j * kThreads];
#pragma unroll
            for (int j = 0; j < U; ++j)
                if (q + j * kThreads < packs)
#pragma unroll
                    for (int e = 0; e < P; ++e)
                        take(head + (q + j * kThreads) * P + e, number<T>(v[j].v[e]));
        }
        for (int i = tid; i < head; i += kThreads) take(i, number<T>(x.x[i]));
        for (int i = head + packs * P + tid; i < x.n; i += kThreads) take(i, number<T>(x.x[i]));
    }
    best = warp_max(best);
    least = __reduce_min_sync(0xffffffffu, least);
    if ((tid & 31) == 0) {
        s.red[tid >> 5] = best;
        s.warp_sum[tid >> 5] = least;
    }
    __syncthreads();
    for (int k = 0; k < kWarps; ++k) {
        best = s.red[k] > best ? s.red[k] : best;
        least = min(least, (u32)s.warp_sum[k]);
    }
    if (tid < (int)ctas) {
        peer_store(&s.told[0][rank], tid, best);
        peer_store(&s.told[7][rank], tid, least);
    }
    row_sync(ctas);
    for (u32 c = 0; c < ctas; ++c) {
        best = s.told[0][c] > best ? s.told[0][c] : best;
        least = min(least, (u32)s.told[7][c]);
    }

    const u32 top = (u32)(best >> 32);
    const double T_ = a.temperature.at(row);
    if (top <= kNothing || top >= kInfinite || !(T_ > 0.0)) {
        // nothing to draw, or nothing but the largest (its lowest id)
        if (rank == 0 && tid == 0)
            a.out[row] = top <= kNothing ? -1 : (int)(0xffffffffu - (u32)best);
        return;
    }
    Row r;
    r.max_f = value_of(top);
    r.max = r.max_f;
    r.scale = fmin(1.4426950408889634074 / T_, 1e300);
    r.shift = 52 - a.bits;
    // beyond 46 / log2(e) temperatures below the largest every weight is 0
    const float range = fminf((float)fmin(32.0 * T_, 3e38), r.max_f - value_of(least));
    r.bin = fminf(kBins / range, 3e38f);

    const int k = a.top_k ? a.top_k[row] : a.one_k;
    const double p = a.top_p.at(row);
    u32 key = 0;              // kept: larger keys, and of the equal ones ids up to `last`
    int last = 0x7fffffff;
    bool few = false;
    if (k > 0 && k < a.V) {
        const Border b = border<false>(s, r, x, 0, top, (u64)k, 0.0, false, rank, ctas);
        key = b.key;
        few = b.ahead + b.ties <= kList;
    }
    if (p > 0.0 && p < 1.0) {
        const Border b = border<true>(s, r, x, key, top, 0, p, few, rank, ctas);
        key = b.key;
        const u64 w = weigh(r, s, key);
        const u64 stay = w ? (b.target - b.ahead + w - 1) / w : b.ties;
        if (stay < b.ties) {
            const int i = first_beyond(
                s, x, s.told[7], rank, ctas, [&](int, u32 q) { return (u64)(q == key); },
                [&](u64) { return stay - 1; });
            if (i >= 0 && tid < (int)ctas) peer_store(&s.told[0][0], tid, (u64)(x.first + i));
            row_sync(ctas);
            last = (int)s.told[0][0];
        }
    }
    const double least_w = fmin(a.min_p.at(row), 1.0) * exp2((double)a.bits);
    const u64 w_floor = least_w > 0.0 ? (u64)ceil(least_w) : 0;
    const double u = a.u_wide ? static_cast<const double*>(a.u)[row]
                              : (double)static_cast<const float*>(a.u)[row];
    const int i = first_beyond(
        s, x, s.told[8], rank, ctas,
        [&](int j, u32 q) -> u64 {
            if (q < key || (q == key && x.first + j > last)) return 0;
            const u64 w = weigh(r, s, q);
            return w < w_floor ? 0 : w;
        },
        [&](u64 total) {
            const double t = u * (double)total;
            return !(t > 0.0) ? 0ull : t >= (double)total ? total - 1 : min((u64)t, total - 1);
        });
    if (i >= 0 && tid == 0) a.out[row] = x.first + i;
    row_sync(ctas);  // no CTA ends while another may still store into it
}

template <typename T>
int launch(const SampleArgs& a, int B, int ctas, cudaStream_t st) {
    const size_t held = (size_t)(a.slice + 3) / 4 * 16;
    const bool fits = held <= 200 * 1024;
    const auto kern = fits ? sample_kernel<T, true> : sample_kernel<T, false>;
    if (fits && held + sizeof(Shared) > 48 * 1024)
        SN_TRY(cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               200 * 1024),
                          "sample"));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)B * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = fits ? held : 0;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_check(cudaLaunchKernelEx(&cfg, kern, a), "sample launch");
}

}  // namespace
}  // namespace sn

using namespace sn;

extern "C" sn_status sn_abi_sample(const void* logits, int64_t ld, int32_t dtype, const void* u,
                                   int32_t u_f64, const double* temperature, double temperature0,
                                   const int32_t* top_k, int32_t top_k0, const double* top_p,
                                   double top_p0, const double* min_p, double min_p0, int32_t B,
                                   int32_t V, int32_t* tokens, void* cuda_stream) {
    const unsigned size = dtype_size(dtype);
    if (!size) return fail(SN_E_INVAL, "sample: dtype %d", dtype);
    if (B < 0 || V <= 0 || ld < V) return fail(SN_E_INVAL, "sample: bad dimension");
    if ((!temperature && !(temperature0 < INFINITY)) || (!min_p && !(min_p0 <= 1.0)) ||
        (!top_p && !(top_p0 == top_p0)))
        return fail(SN_E_INVAL, "sample: a temperature that is not finite, min_p above 1 or NaN");
    if (B == 0) return SN_OK;
    if (!logits || !u || !tokens) return fail(SN_E_INVAL, "sample: null pointer");
    if (B > 0x7fffffff / kMaxCluster) return fail(SN_E_INVAL, "sample: %d rows", B);
    CallerDevice dev;
    SN_TRY(dev.enter("sample", {{logits, size}, {u, u_f64 ? 8u : 4u}, {temperature, 8},
                                {top_k, 4}, {top_p, 8}, {min_p, 8}, {tokens, 4}}));
    // slices of 8192 keys (32 KB) leave room for six CTAs on an SM, so that one
    // row's reads run under another's arithmetic; a few rows are cut further,
    // until the SMs have two CTAs each
    int ctas = 1;
    while (ctas < kMaxCluster &&
           ((long long)ctas * 8192 < V ||
            ((long long)B * ctas < 2ll * dev.num_sms() && (long long)ctas * 2048 < V)))
        ctas *= 2;
    SampleArgs a{logits, u, top_k, tokens, {temperature, temperature0}, {top_p, top_p0},
                 {min_p, min_p0}, ld, top_k0, u_f64, V, 0, 44};
    a.slice = (int)(((long long)V + ctas - 1) / ctas + 7) / 8 * 8;
    while (std::ldexp((double)V, a.bits) >= std::ldexp(1.0, 62)) --a.bits;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    switch (dtype) {
        case SN_F32: return launch<float>(a, B, ctas, st);
        case SN_BF16: return launch<__nv_bfloat16>(a, B, ctas, st);
        default: return launch<__half>(a, B, ctas, st);
    }
}
