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
// where u, or top-p's target, meets a border to about 2^-40 (two equal largest
// logits, the others 31 temperatures below and p of exactly 0.5: the second is
// in by what those weigh, which is nothing here). An id below 2^-45 of the
// largest is never drawn.
//
// What bounds a batch of rows is not HBM but the instructions spent on a logit:
// an exact weight takes about 40, 14 of them in 64 bits. So what can be kept is
// narrowed first. A histogram over 1024 bins, linear from the largest logit down,
// counts the logits; for top-k the bins down to the k-th, for top-p those whose
// count times the bin's least weight reaches p of the row's weight (estimated
// from above in fp32) hold every id that can stay. The ids of those bins are
// listed by id, and only they get exact weights. Top-p's target p * (weight of
// all) needs the rest's weight too: it comes from the fp32 estimate with its
// worst-case error; where the two ends of that error do not lead to the same
// ids (a percent of the rows) the row's weight is summed exactly.
//
// Neither top-k nor top-p sorts: both look for one border key, the largest
// with "count (or weight) of the larger keys < target <= that plus its own".
// The first histogram leaves a range of keys for it; the range is cut into 512
// bins by key, whose counts or weights give the border's bin, until a bin's
// keys are kList or fewer, or one (at most five rounds); these are gathered and
// compared with one another. A top-k row with at most kList listed ids, the
// usual case, is finished by one CTA that compares all of them.
//
// A row belongs to a cluster of 1 to 8 CTAs. With few rows each CTA keeps a
// slice of the row in shared memory, and the CTAs read one another's
// histograms and lists through distributed shared memory. With rows enough
// for every SM a row belongs to one CTA, which keeps no more than the list and
// reads the row from L2 again: the cost of a CTA's fixed steps (scans,
// searches) is then spread over the whole row.
//
// One row of 32000 fp32 logits with top-k 40 and top-p 0.95 takes 13.5 us, a chain
// of waits; 1024 of them 60 us with top-k 40 (greedy, which is the pass over the
// logits alone, 25), and 122 us with top-p 0.9, which keeps some thousands of
// each. A border beyond the bins (fewer ids allowed than top-k, or a k-th logit
// 32 temperatures below the first) leaves every id in its range: 256 x 16384 take
// 61 us with ten allowed ids and top-k 40, and 18 where the border lies in the
// bins.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstddef>

#include "caller.cuh"
#include "ptx.cuh"
#include "runtime.cuh"

namespace sn {
namespace {

typedef unsigned long long u64;
typedef unsigned int u32;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kCut = 1024;     // bins of the first histogram, four to a thread
constexpr int kBins = 512;     // of the others, two to a thread
constexpr int kList = 256;     // keys resolved by comparing them all: one to a thread
constexpr int kCand = 8192;    // logits a CTA that keeps no slice can list, at least: 32 KB,
                               // four CTAs on an SM
constexpr int kProbe = 4 * kThreads;  // first logits of a row, from which the bins take their place
constexpr int kPow = 128;      // table of 2^(j/128)
constexpr int kMaxCluster = 8;
constexpr u32 kNothing = 0x007fffffu;  // key of -infinity

// 2^(j/128) by the exponential series, computed by the compiler.
struct PowTable {
    double v[kPow];
    constexpr PowTable() : v{} {
        for (int j = 0; j < kPow; ++j) {
            double x = j * 0.69314718055994530942 / kPow, e = 1.0;
            for (int k = 24; k > 0; --k) e = 1.0 + e * x / k;
            v[j] = e;
        }
    }
};
__device__ constexpr PowTable g_pow{};

__device__ __forceinline__ double two_to(int n) { return __hiloint2double((1023 + n) << 20, 0); }

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
    int one_k, u_wide, V, slice, bits, cand;
};

// Bits of x ordered like the numbers, -0 taken for 0.
__device__ __forceinline__ u32 key_of(float x) {
    const u32 b = __float_as_uint(x + 0.0f);
    return b ^ ((u32)((int)b >> 31) | 0x80000000u);
}

__device__ __forceinline__ float value_of(u32 k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

struct Shared {
    double pow[kPow];           // 2^(j/128)
    u64 told[14][kMaxCluster];  // a value of each CTA, one line per exchange
    u64 red[kWarps];
    u64 warp_sum[kWarps];
    u64 third[kWarps];
    alignas(16) u32 count[kCut];  // of cut()
    alignas(16) u32 lo[kBins], hi[kBins];  // a bin's count or weight, as two words, of border()
    u32 list[2][kList], listed[2];  // keys of the border's bin, of top-k and of top-p
    u32 least, most;           // their range
    u32 all[kList];            // every CTA's list
    u64 weight[kList];
    u64 found[4];
    u32 edge[2];
};
static_assert(offsetof(Shared, told) % 8 == 0 && offsetof(Shared, count) % 16 == 0 &&
                  offsetof(Shared, lo) % 16 == 0 && offsetof(Shared, hi) % 16 == 0,
              "vector loads of other CTAs' counters");

// The CTAs of a row: a cluster, or (ONE) a CTA by itself.
template <bool ONE>
struct Team {
    u32 rank, ctas;
    __device__ Team() : rank(ONE ? 0 : cluster_rank()), ctas(ONE ? 1 : cluster_size()) {}
    __device__ __forceinline__ void sync() const {
        if (ONE || ctas == 1)
            __syncthreads();
        else
            cluster_sync();
    }
    // Another CTA's shared memory may be touched once that CTA runs: each says so
    // when it starts, and waits for the others in front of its first tell(). The
    // pass over the row lies between the two, so the wait is over by then.
    __device__ __forceinline__ void started() const {
        if (!ONE && ctas > 1) cluster_arrive_relaxed();
    }
    __device__ __forceinline__ void all_started() const {
        if (!ONE && ctas > 1) cluster_wait();
    }
    // Reads of another CTA's shared memory take several hundred cycles: the
    // callers issue all of theirs before they use the first.
    __device__ __forceinline__ u32 read(const u32* local, u32 from) const {
        if (ONE) return *local;
        u32 v;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(dsmem_addr(local, from)));
        return v;
    }
    // N counters from each CTA, added up
    template <int N>
    __device__ __forceinline__ void add_up(const u32* local, u64 (&sum)[N]) const {
        static_assert(N == 2 || N == 4, "a vector load each");
        u32 v[ONE ? 1 : kMaxCluster][N];
#pragma unroll
        for (int c = 0; c < (ONE ? 1 : kMaxCluster); ++c) {
            if (ONE) {
                for (int j = 0; j < N; ++j) v[c][j] = local[j];
            } else if (c < (int)ctas) {
                const u32 at = dsmem_addr(local, c);
                if constexpr (N == 4)
                    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(v[c][0]), "=r"(v[c][1]), "=r"(v[c][2]), "=r"(v[c][3])
                                 : "r"(at));
                else
                    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];"
                                 : "=r"(v[c][0]), "=r"(v[c][1])
                                 : "r"(at));
            } else {
                for (int j = 0; j < N; ++j) v[c][j] = 0;
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            sum[j] = 0;
#pragma unroll
            for (int c = 0; c < (ONE ? 1 : kMaxCluster); ++c) sum[j] += v[c][j];
        }
    }
    // Thread i's place among the CTAs' lists, laid one behind the other: of
    // which CTA (ctas: behind them all) and where in its list; count[c] long.
    __device__ __forceinline__ u32 place(const u64* count, u32 i, u32* at) const {
        u32 c = 0;
        *at = i;
#pragma unroll
        for (int k = 0; k < (ONE ? 1 : kMaxCluster); ++k)
            if (k < (int)ctas && c == (u32)k && *at >= (u32)count[k]) *at -= (u32)count[k], ++c;
        return c;
    }
    // v into the place of *local in CTA `to`
    __device__ __forceinline__ void store(u64* local, u32 to, u64 v) const {
        if (ONE)
            *local = v;
        else
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(dsmem_addr(local, to)), "l"(v)
                         : "memory");
    }
    // v of this CTA into every CTA's line, by the first threads
    __device__ __forceinline__ void tell(u64* line, u64 v) const {
        if (threadIdx.x < ctas) store(line + rank, threadIdx.x, v);
    }
};

// One row's numbers, the same in every thread of the cluster.
struct Row {
    double max, scale;  // w = 2^((x - max) * scale)
    double unit;        // 2^(52 - bits): a double near it ends at 2^-bits
    float max_f, scale_f;
    float ref, bin;     // linear bins: (ref - x) * bin
    float cutoff;       // logits below weigh nothing
};

// 2^((x - max) * scale) * 2^bits to the nearest whole number. The exponent's
// nearest 128th goes to the table, the rest |f| <= 2^-8 to the exponential
// series of f ln2, whose fifth term is below 2^-49.
__device__ __forceinline__ u64 weigh(const Row& r, const Shared& s, float x) {
    constexpr double whole128 = 1.5 * 0x1p45;  // doubles near it are 128ths
    constexpr double ln2 = 0.69314718055994530942;
    const double below = (double)fmaxf(x, r.cutoff) - r.max;
    const double near = fma(below, r.scale, whole128);
    const double f = fma(below, r.scale, whole128 - near);
    double e = ln2 * ln2 * ln2 * ln2 / 24;
    e = fma(e, f, ln2 * ln2 * ln2 / 6);
    e = fma(e, f, ln2 * ln2 / 2);
    e = fma(e, f, ln2);
    e = fma(e, f, 1.0);
    const int i = __double2loint(near);  // 128ths, 0 down to -8320
    e *= s.pow[i & (kPow - 1)];
    e = __hiloint2double(__double2hiint(e) + ((i >> 7) << 20), __double2loint(e));
    e += r.unit;
    const u64 w = (u64)(__double_as_longlong(e) - __double_as_longlong(r.unit));
    return x < r.cutoff ? 0 : w;
}

// Bin of x, its distance below ref to the nearest, the first and the last bin
// taking what is beyond them: adding 2^23 leaves the rounded number in the low
// bits.
__device__ __forceinline__ int linear_bin(const Row& r, float x) {
    const float v = __saturatef((r.ref - x) * (r.bin * (1.0f / (kCut - 1))));
    return __float_as_int(fmaf(v, (float)(kCut - 1), 8388608.0f)) - 0x4b000000;
}

// 2^x to 2^-22 of itself.
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

// Three of those at once.
__device__ __forceinline__ void block_upto3(Shared& s, u64 (&v)[3], u64 (&all)[3]) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const u64 x = __shfl_up_sync(0xffffffffu, v[j], o);
            if (lane >= o) v[j] += x;
        }
    if (lane == 31) s.red[w] = v[0], s.warp_sum[w] = v[1], s.third[w] = v[2];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 3; ++j) all[j] = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
        if (k == w)
#pragma unroll
            for (int j = 0; j < 3; ++j) v[j] += all[j];
        all[0] += s.red[k], all[1] += s.warp_sum[k], all[2] += s.third[k];
    }
    __syncthreads();
}

// Sum over the CTA's threads, the same in all.
__device__ __forceinline__ u64 block_add(Shared& s, u64 v) {
    v = warp_add(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) v += s.warp_sum[k];
    return v;
}

template <typename T>
__device__ __forceinline__ float number(T v);
template <>
__device__ __forceinline__ float number<float>(float v) { return fmaxf(v, -INFINITY); }
template <>
__device__ __forceinline__ float number<__nv_bfloat16>(__nv_bfloat16 v) {
    return fmaxf(__bfloat162float(v), -INFINITY);
}
template <>
__device__ __forceinline__ float number<__half>(__half v) {
    return fmaxf(__half2float(v), -INFINITY);
}

template <typename T, int P>
struct alignas(sizeof(T) * P) Pack {
    T v[P];
};

// A CTA's slice of a row in the caller's memory, from the 16-byte boundary at or
// before its first logit: the `skip` places in front of that, those behind the
// last and NaN read as -infinity.
template <typename T>
struct Far {
    static constexpr int P = 16 / sizeof(T), U = 16 / P;  // logits of a pack, packs in flight
    const T* x;
    int n, skip;  // n: places, skipped ones among them
    __device__ __forceinline__ float value(int i) const {
        return i < skip ? -INFINITY : number<T>(x[i]);
    }
    __device__ __forceinline__ int id(int i) const { return i - skip; }
    __device__ __forceinline__ int packs() const { return (n + P - 1) / P; }
    __device__ __forceinline__ void load(int i, float (&v)[P]) const {
        if (i * P >= skip && (i + 1) * P <= n) {
            const Pack<T, P> p = reinterpret_cast<const Pack<T, P>*>(x)[i];
#pragma unroll
            for (int j = 0; j < P; ++j) v[j] = number<T>(p.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < P; ++j) v[j] = i * P + j < n ? value(i * P + j) : -INFINITY;
        }
    }
};

template <typename T>
__device__ __forceinline__ T nothing();
template <>
__device__ __forceinline__ float nothing<float>() { return -INFINITY; }
template <>
__device__ __forceinline__ __nv_bfloat16 nothing<__nv_bfloat16>() {
    return __ushort_as_bfloat16(0xff80);
}
template <>
__device__ __forceinline__ __half nothing<__half>() { return __ushort_as_half(0xfc00); }

// A walk over a slice in the caller's memory in tiles of kTile packs to a
// thread, the next kRing - 1 of them on their way to shared memory (cp.async)
// meanwhile. Loads into registers had 4 packs in flight and none while they
// were worked on: 20 us instead of 14 for the first 592 rows of 32000 fp32
// logits. A warp reads back what its own lanes copied.
constexpr int kRing = 4, kTile = 2;

template <typename T>
struct Walk {
    static constexpr int P = 16 / sizeof(T);
    const Far<T>& x;
    Pack<T, P>* ring;  // [kRing][warps][kTile][32]
    int packs, tiles, ahead = 0;
    __device__ Walk(const Far<T>& far, void* shared)
        : x(far), ring(static_cast<Pack<T, P>*>(shared)), packs(far.packs()),
          tiles((far.packs() + kTile * kThreads - 1) / (kTile * kThreads)) {
        for (int k = 0; k < kRing - 1; ++k) fetch();
    }
    // First pack of the calling warp's part of tile t: kTile * 32 packs.
    __device__ __forceinline__ int first(int t) const {
        return (t * kThreads + (int)(threadIdx.x & ~31)) * kTile;
    }
    __device__ __forceinline__ Pack<T, P>* part(int t) const {
        return ring + ((t % kRing) * kThreads + (threadIdx.x & ~31)) * kTile;
    }
    __device__ __forceinline__ bool inner(int t) const { return t > 0 && t + 1 < tiles; }
    __device__ __forceinline__ void fetch() {
        const int lane = threadIdx.x & 31;
        Pack<T, P>* to = part(ahead);
        const int q0 = first(ahead);
        if (inner(ahead)) {
#pragma unroll
            for (int n = 0; n < kTile; ++n)
                cp_async16(to + n * 32 + lane, x.x + (long long)(q0 + n * 32 + lane) * P, 16);
        } else if (ahead < tiles) {
#pragma unroll
            for (int n = 0; n < kTile; ++n) {
                const int q = q0 + n * 32 + lane;
                if (q * P >= x.skip && (q + 1) * P <= x.n) {
                    cp_async16(to + n * 32 + lane, x.x + (long long)q * P, 16);
                } else {  // in part or wholly beside the slice
                    Pack<T, P> p;
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        const int i = q * P + j;
                        p.v[j] = i >= x.skip && i < x.n ? x.x[i] : nothing<T>();
                    }
                    to[n * 32 + lane] = p;
                }
            }
        }
        cp_async_commit();
        ++ahead;
    }
    // The warp's part of tile t, once it is there. (What is fetched next goes
    // where the tile before this one lay.)
    __device__ __forceinline__ const Pack<T, P>* tile(int t) {
        __syncwarp();
        fetch();
        cp_async_wait_group<kRing - 1>();
        __syncwarp();
        return part(t);
    }
};

// f(place, logit, position in its pack) for each, padding included, ascending
// within a thread.
template <typename T, typename F>
__device__ __forceinline__ void walk_all(const Far<T>& x, void* ring, F f) {
    Walk<T> walk(x, ring);
    const int lane = threadIdx.x & 31;
    for (int t = 0; t < walk.tiles; ++t) {
        const auto* part = walk.tile(t);
        const int q0 = walk.first(t) + lane;
#pragma unroll
        for (int n = 0; n < kTile; ++n) {
            const auto p = part[n * 32 + lane];
#pragma unroll
            for (int e = 0; e < Walk<T>::P; ++e)
                f((q0 + n * 32) * Walk<T>::P + e, number<T>(p.v[e]), e);
        }
    }
}

// The same in shared memory, in fp32 and whole packs.
struct Near {
    static constexpr int P = 4, U = 1;
    const float* x;
    int n, skip;
    __device__ __forceinline__ float value(int i) const { return x[i]; }
    __device__ __forceinline__ int id(int i) const { return i - skip; }
    __device__ __forceinline__ int packs() const { return (n + 3) / 4; }
    __device__ __forceinline__ void load(int i, float (&v)[4]) const {
        const float4 f = reinterpret_cast<const float4*>(x)[i];
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    }
};

// Of a slice in shared memory: the places of what can stay, in order.
struct NearListed {
    static constexpr int P = 1, U = 4;
    Near of;
    const unsigned short* at;
    int n;
    __device__ __forceinline__ float value(int i) const { return of.x[at[i]]; }
    __device__ __forceinline__ int id(int i) const { return of.id(at[i]); }
    __device__ __forceinline__ int packs() const { return n; }
    __device__ __forceinline__ void load(int i, float (&v)[1]) const { v[0] = value(i); }
};

// Of a whole row that is not kept: the logits of what can stay, in order of
// id. Their ids are found again for the one that is drawn.
struct FarListed {
    static constexpr int P = 1, U = 4;
    const float* x;
    int n;
    __device__ __forceinline__ float value(int i) const { return x[i]; }
    __device__ __forceinline__ int id(int i) const { return i; }
    __device__ __forceinline__ int packs() const { return n; }
    __device__ __forceinline__ void load(int i, float (&v)[1]) const { v[0] = x[i]; }
};

// f(place, logit, position in its pack) for each of a slice, padding included,
// in no order, but ascending within a thread.
template <typename S, typename F>
__device__ __forceinline__ void each(const S& x, F f) {
    const int packs = x.packs();
    for (int q = threadIdx.x; q < packs; q += S::U * kThreads) {
        float v[S::U][S::P];
#pragma unroll
        for (int j = 0; j < S::U; ++j)
            if (q + j * kThreads < packs) x.load(q + j * kThreads, v[j]);
#pragma unroll
        for (int j = 0; j < S::U; ++j) {
            if (q + j * kThreads >= packs) break;
#pragma unroll
            for (int e = 0; e < S::P; ++e) f((q + j * kThreads) * S::P + e, v[j][e], e);
        }
    }
}

// f(logit, weight) for each of a slice; the weights of a pack, or of the packs
// of one, are formed side by side (each is a chain of a dozen operations).
template <typename S, typename F>
__device__ __forceinline__ void each_weighed(const Row& r, const Shared& s, const S& x, F f) {
    constexpr int P = S::P, G = P == 1 ? S::U : 1;  // packs weighed side by side
    const int packs = x.packs();
    for (int q = threadIdx.x; q < packs; q += S::U * kThreads) {
        float v[S::U][P];
#pragma unroll
        for (int j = 0; j < S::U; ++j) {
            if (q + j * kThreads < packs) {
                x.load(q + j * kThreads, v[j]);
            } else {
#pragma unroll
                for (int e = 0; e < P; ++e) v[j][e] = -INFINITY;
            }
        }
#pragma unroll
        for (int j0 = 0; j0 < S::U; j0 += G) {
            u64 w[G][P];
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int e = 0; e < P; ++e) w[j][e] = weigh(r, s, v[j0 + j][e]);
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int e = 0; e < P; ++e) f(v[j0 + j][e], w[j][e]);
        }
    }
}

// The weight that top-p's ids have to reach: p of the whole, at least 1 (the
// largest logit's id always stays).
__device__ __forceinline__ u64 share(double p, u64 whole) {
    const double want = ceil(p * (double)whole);
    return want < 1.0 ? 1 : want < (double)whole ? (u64)want : whole;
}

// Where a border key can be: [from, to]; keys above `to` lie ahead of it, and
// number `ahead` (top-k); `keys`: how many it is among.
struct Range {
    u32 from, to;
    u64 ahead;
    u32 keys;
};

// What the border of top-k or top-p is.
struct Border {
    u32 key;
    u64 ahead;  // count or weight of the larger keys
    u64 ties;   // ids that have this key
    u64 total, target;  // weight of what it is among, and top-p's target
};

// The weight of a row's ids that are not in hand, in units of the weights: at
// least and at most. `below`: they are in hand, as keys below the range.
struct Rest {
    u64 least, most;
    bool below;
};

// The border key: count (or, BY_WEIGHT, weight) of larger keys < target <=
// that and its own. The target of a weight is p of the weight of all keys >=
// in.from and of the rest.
template <bool BY_WEIGHT, bool ONE, typename S>
__device__ Border border(Shared& s, const Row& r, const S& x, const Range& in, u64 target,
                         double p, Rest rest, Team<ONE> t) {
    const int tid = threadIdx.x;
    u32* list = s.list[BY_WEIGHT];
    // three lines; no call follows one of its kind without a barrier between
    u64(*told)[kMaxCluster] = s.told + (BY_WEIGHT ? 4 : 1);
    u32 from = in.from, to = in.to;
    u64 base = BY_WEIGHT ? 0 : in.ahead;
    int shift = max(0, 32 - __clz(to - from) - 9);  // (to - from) >> shift < 512
    int bin = -1;
    bool few = in.keys <= kList;  // enough to gather at once
    u64 total = 0;
    for (bool first = true;; first = false) {  // (or a first round of `few` that were not)
        if (!few) {
            for (int b = tid; b < kBins; b += kThreads) s.lo[b] = s.hi[b] = 0;
            __syncthreads();
            u64 above = 0, below = 0;
            if (BY_WEIGHT) {
                each_weighed(r, s, x, [&](float f, u64 w) {
                    const u32 k = key_of(f);
                    above += first && k > to ? w : 0;
                    below += first && k < from ? w : 0;
                    if (k < from || k > to || w == 0) return;
                    const u32 b = (to - k) >> shift, a = (u32)w, old = atomicAdd(&s.lo[b], a);
                    const u32 c = (u32)(w >> 32) + (old + a < old ? 1u : 0u);
                    if (c) atomicAdd(&s.hi[b], c);
                });
            } else {
                each(x, [&](int, float f, int) {
                    const u32 k = key_of(f);
                    if (k >= from && k <= to) atomicAdd(&s.lo[(to - k) >> shift], 1u);
                });
            }
            if (BY_WEIGHT && first) {
                t.tell(s.told[10], block_add(s, above));
                if (rest.below) t.tell(s.told[11], block_add(s, below));
            }
            t.sync();
            if (BY_WEIGHT && first)
                for (u32 c = 0; c < t.ctas; ++c) {
                    base += s.told[10][c];
                    if (rest.below) total += s.told[11][c];
                }
            u64 v[2];
            t.add_up(&s.lo[2 * tid], v);
            if (BY_WEIGHT) {
                u64 high[2];
                t.add_up(&s.hi[2 * tid], high);
                v[0] += high[0] << 32, v[1] += high[1] << 32;
            }
            const u64 upto = block_upto(s, v[0] + v[1]);
            if (BY_WEIGHT && target == 0) {
                if (tid == kThreads - 1) s.found[0] = upto;
                __syncthreads();
                total += base + s.found[0];
                target = share(p, total + rest.least);
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
        const auto gather = [&](u32 k) {
            least = min(least, k);
            most = max(most, k);
            const u32 at = atomicAdd(&s.listed[BY_WEIGHT], 1u);
            if (at < kList) list[at] = k;
        };
        if (BY_WEIGHT && few) {  // the first round, without a histogram before
            u64 above = 0, below = 0;
            each_weighed(r, s, x, [&](float f, u64 w) {
                const u32 k = key_of(f);
                above += k > to ? w : 0;
                below += k < from ? w : 0;
                if (k >= from && k <= to) gather(k);
            });
            t.tell(s.told[10], block_add(s, above));
            if (rest.below) t.tell(s.told[11], block_add(s, below));
        } else {
            each(x, [&](int, float f, int) {
                const u32 k = key_of(f);
                if (k >= from && k <= to && (few || (int)((to - k) >> shift) == bin)) gather(k);
            });
        }
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        if ((tid & 31) == 0 && least <= most) {
            atomicMin(&s.least, least);
            atomicMax(&s.most, most);
        }
        __syncthreads();
        t.tell(told[0], s.listed[BY_WEIGHT]);
        t.tell(told[1], s.least);
        t.tell(told[2], s.most);
        t.sync();
        u64 count = 0;
        least = 0xffffffffu, most = 0;
        for (u32 c = 0; c < t.ctas; ++c) {
            if (BY_WEIGHT && few) {
                base += s.told[10][c];
                if (rest.below) total += s.told[11][c];
            }
            count += told[0][c];
            least = min(least, (u32)told[1][c]);
            most = max(most, (u32)told[2][c]);
        }
        from = least;
        to = most;
        if (from == to) {  // one key, however often
            if (BY_WEIGHT && target == 0) {
                total += base + count * weigh(r, s, value_of(from));
                target = share(p, total + rest.least);
            }
            return {from, base, count, total, target};
        }
        if (count <= kList) {
            u32 at;
            const u32 c = t.place(told[0], tid, &at);
            const bool mine_in = c < t.ctas;
            const u32 mine = mine_in ? t.read(&list[at], c) : 0;
            const u64 w = BY_WEIGHT && mine_in ? weigh(r, s, value_of(mine)) : 0;
            s.all[tid] = mine;  // no key behind the last
            if (BY_WEIGHT) s.weight[tid] = w;
            if (BY_WEIGHT && target == 0) {
                total += base + block_add(s, w);
                target = share(p, total + rest.least);
            }
            __syncthreads();
            if (mine_in) {
                u64 more = 0;
                u32 ties = 0;
#pragma unroll 8
                for (int j = 0; j < (int)(count + 7) / 8 * 8; ++j) {
                    const u32 k = s.all[j];
                    more += k > mine ? (BY_WEIGHT ? s.weight[j] : 1) : 0;
                    ties += k == mine;
                }
                const u64 own = ties * (BY_WEIGHT ? s.weight[tid] : 1);
                if (base + more < target && target <= base + more + own) {  // all its ties say the same
                    s.found[1] = mine;
                    s.found[2] = base + more;
                    s.found[3] = ties;
                }
            }
            __syncthreads();
            return {(u32)s.found[1], s.found[2], s.found[3], total, target};
        }
        shift = max(0, 32 - __clz(to - from) - 9);
        few = false;
    }
}

// Index (in x) of the first id at which the running sum of measure(i, logit) over
// the row exceeds the target that aim(total) gives; -1 in CTAs that do not
// hold it.
template <bool ONE, typename S, typename M, typename A>
__device__ int first_beyond(Shared& s, const S& x, u64* told, Team<ONE> t, M measure, A aim) {
    const int tid = threadIdx.x, w = tid >> 5, lane = tid & 31;
    const int packs = x.packs(), part = (packs + kThreads - 1) / kThreads * 32;
    const int lo = min(w * part, packs), hi = min(lo + part, packs);  // a warp's run
    u64 sum = 0;
    for (int i = lo + lane; i < hi; i += 32 * S::U) {
        float v[S::U][S::P];
#pragma unroll
        for (int j = 0; j < S::U; ++j)
            if (i + 32 * j < hi) x.load(i + 32 * j, v[j]);
#pragma unroll
        for (int j = 0; j < S::U; ++j) {
            if (i + 32 * j >= hi) break;
#pragma unroll
            for (int e = 0; e < S::P; ++e) sum += measure((i + 32 * j) * S::P + e, v[j][e]);
        }
    }
    const u64 mine = block_add(s, sum);
    t.tell(told, mine);
    t.sync();
    u64 total = 0, before = 0;
    for (u32 c = 0; c < t.ctas; ++c) {
        if (c == t.rank) before = total;
        total += told[c];
    }
    const u64 target = aim(total);
    if (target < before || target >= before + mine) return -1;
    int k = 0;
    while (target >= before + s.warp_sum[k]) before += s.warp_sum[k++];
    // the run of warp k, a few ids to each thread
    const int a = min(k * part * S::P, x.n), b = min((k + 1) * part * S::P, x.n);
    const int n = (b - a + kThreads - 1) / kThreads;
    const int from = min(a + tid * n, b), to = min(from + n, b);
    sum = 0;
    for (int i = from; i < to; ++i) sum += measure(i, x.value(i));
    const u64 upto = before + block_upto(s, sum);
    if (target < upto && target >= upto - sum) {
        u64 at = upto - sum;
        int i = from;
        for (; i < to - 1; ++i) {
            at += measure(i, x.value(i));
            if (at > target) break;
        }
        s.found[0] = (u64)i;
    }
    __syncthreads();
    return (int)s.found[0];
}

// Key of the smallest number whose linear bin is `bin` or nearer, by the lanes
// of a warp: it lies in (out, in], at first within 256 keys of the bin's edge in
// real numbers where those ends say so, cut to a 32nd by each step. One above
// the row's largest where that lies in a farther bin.
__device__ u32 near_edge(const Row& r, int bin) {
    const u32 lane = threadIdx.x & 31, top = key_of(r.max_f);
    if (linear_bin(r, r.max_f) > bin) return top + 1;
    const u32 guess = key_of(fminf(fmaxf(r.ref - (bin + 0.5f) / r.bin, -3e38f), r.max_f));
    u32 out = guess - 256, in = min(guess + 256, top);
    if (!(out > kNothing && out < in && linear_bin(r, value_of(out)) > bin)) out = kNothing;
    if (linear_bin(r, value_of(in)) > bin) in = top;
    while (in - out > 1) {
        const u32 step = (in - out + 31) / 32;
        const u32 at = min((u64)out + (u64)step * (lane + 1), (u64)in);
        const u32 near = __ballot_sync(0xffffffffu, linear_bin(r, value_of(at)) <= bin);
        const int f = __ffs(near) - 1;  // the last lane's is `in` itself
        const u32 low = out;
        out = f ? (u32)min((u64)low + (u64)step * f, (u64)in) : low;
        in = (u32)min((u64)low + (u64)step * (f + 1), (u64)in);
    }
    return in;
}

// Narrows where the border is, from the counts of the linear bins and, for
// top-p, the estimate `sum` of the weight of all relative to ref's. Returns how
// many ids lie in the range or above; 0: the bins lie in the wrong place.
template <bool ONE>
__device__ u32 cut(Shared& s, const Row& r, int V, int k, double p, int bits, Team<ONE> t,
                   double sum, Range* range) {
    constexpr int N = kCut / kThreads;
    const int tid = threadIdx.x;
    u64 whole[2] = {0, 0};
    if (k <= 0) {
        // 2^-12 is more than its terms' 2^-22, the roundings of exponents up to
        // 200 (3 * 2^-24 * 200 * ln 2 < 2^-15) and those of sums of 2^10 terms
        sum *= fast_exp2((float)(((double)r.ref - r.max) * r.scale));
        if (!(sum >= 0.5 && sum < 2.0 * V)) return 0;  // ref is too far off
        const double units = sum * two_to(bits);
        whole[0] = (u64)(units * (1 - 0x1p-12));
        whole[1] = (u64)(units * (1 + 0x1p-12));
    }
    u64 sums[N];
    u32 n[N], own = 0;
    t.add_up(&s.count[N * tid], sums);
#pragma unroll
    for (int j = 0; j < N; ++j) own += n[j] = (u32)sums[j];
    // found: the border's bin or a farther one, ids up to it, ids ahead of the
    // range; and how many nearest bins are surely ahead of the border
    if (k > 0) {
        u32 counted = (u32)block_upto(s, own) - own;  // before this thread's bins
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (counted < (u32)k && (u32)k <= counted + n[j]) {
                s.found[0] = s.found[3] = N * tid + j;
                s.found[1] = counted + n[j];
                s.found[2] = counted;
            }
            counted += n[j];
        }
    } else {  // the weight of a bin's ids is between those of its edges
        const float step = (float)(r.scale / r.bin), unit_f = (float)two_to(bits);
        const float d0 = (float)(((double)r.ref - r.max) * r.scale);  // bin 0's middle
        const float slack = 0x1p-16f + 0x1p-21f * fabsf(d0);
        u64 lo[N], hi[N], upto[3] = {0, 0, own}, all[3];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int b = N * tid + j;
            const float far = fminf(d0 - (b + 0.5f) * step * (1 + 0x1p-18f), 0.0f);
            const float near = b == 0 ? 0.0f : fminf(d0 - (b - 0.5f) * step * (1 - 0x1p-18f), 0.0f);
            // (the last bin has no far edge: -infinity lies in it)
            lo[j] = b == kCut - 1 ? 0 : (u64)(n[j] * (unit_f * (1 - slack) * fast_exp2(far)));
            hi[j] = (u64)(n[j] * (unit_f * (1 + slack) * fast_exp2(near))) + n[j];
            upto[0] += lo[j];
            upto[1] += hi[j];
        }
        const u64 lo_own = upto[0], hi_own = upto[1];
        block_upto3(s, upto, all);
        u64 lo_upto = upto[0] - lo_own, hi_upto = upto[1] - hi_own;
        u32 counted = (u32)upto[2] - own;
        // A bin lies at the border or behind it if the bins up to it reach p of
        // the whole, or those behind it weigh no more than the rest; it lies
        // ahead if those up to it do not, or those behind it weigh more. The
        // bounds are a bin's width apart in what they sum up: for p near 1 the
        // sums from behind are the sharper.
        const u64 sure = share(p, whole[1]), may = share(p, whole[0]);
        const u64 room = (u64)fmax(0.0, (1.0 - p) * (double)whole[0] - 2.0);
        const u64 room_most = (u64)((1.0 - p) * (double)whole[1]) + 2;
        u64 not_enough = 0, ahead = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            lo_upto += lo[j];
            hi_upto += hi[j];
            not_enough += !(lo_upto >= sure || all[1] - hi_upto <= room);
            ahead += hi_upto < may || all[0] - lo_upto > room_most;  // (both descend along the bins)
        }
        const u64 both = block_add(s, not_enough << 32 | ahead);
        const u32 bin = (u32)(both >> 32), near = min((u32)both, bin);
        if (tid == 0) s.found[0] = bin, s.found[3] = near, s.found[2] = 0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) {
            counted += n[j];
            if (bin == (u32)(N * tid + j)) s.found[1] = counted;
            if (near == (u32)(N * tid + j + 1)) s.found[2] = counted;
        }
    }
    __syncthreads();
    // no bin, the last, which has no far edge, or the one before it: every id can stay
    const int bin = (int)s.found[0], ahead = (int)s.found[3];
    const bool open = bin >= kCut - 2;
    if (tid < 32) {
        const u32 e = open ? kNothing : near_edge(r, bin);
        if (tid == 0) s.edge[0] = e;
    } else if (tid < 64) {
        const u32 e = ahead > 0 ? near_edge(r, min(ahead, kCut - 1) - 1) - 1 : key_of(r.max_f);
        if (tid == 32) s.edge[1] = e;
    }
    __syncthreads();
    range->from = s.edge[0];
    range->to = s.edge[1];
    const u32 all = open ? (u32)V : (u32)s.found[1];  // (bins behind the border's are in, too)
    range->ahead = s.found[2];
    range->keys = all - (u32)s.found[2];
    __syncthreads();
    return all;
}

// put(position, place) for each marked place of a slice, [skip, n) (skip < 32), in
// order; returns their number. Places beside the slice, in the first and the last
// word, may be marked (they read as -infinity, which is no less than a `least` of
// -infinity), and are unmarked here: masks where the marks are made took 2 us more
// of 122 (1024 x 32000 with top-p) and 5 of 17 (64 x 65521 with min-p).
template <typename F>
__device__ int give_marked(Shared& s, int skip, int n, u32* marks, F put) {
    const int tid = threadIdx.x, words = (n + 31) / 32;
    __syncthreads();
    if (tid == 0 && words > 0) {
        marks[0] &= ~0u << skip;
        marks[words - 1] &= ~0u >> (words * 32 - n);
    }
    __syncthreads();
    // a few neighbouring words to each thread
    const int each = (words + kThreads - 1) / kThreads;
    const int lo = min(tid * each, words), hi = min(lo + each, words);
    u32 mine = 0;
    for (int w = lo; w < hi; ++w) mine += __popc(marks[w]);
    const u32 upto = (u32)block_upto(s, mine);
    if (tid == kThreads - 1) s.found[0] = upto;
    u32 at = upto - mine;
    for (int w = lo; w < hi; ++w)
        for (u32 m = marks[w]; m; m &= m - 1) put(at++, w * 32 + __ffs(m) - 1);
    __syncthreads();
    return (int)s.found[0];
}

// Marks the places of a slice's logits >= least, a bit each in words of 32, then
// gives put(position, place) for each in order; returns their number. REST: the
// weight of the others is estimated and added to *rest.
template <bool REST, typename S, typename F>
__device__ int list(Shared& s, const Row& r, const S& x, float least, u32* marks, double* rest,
                    F put) {
    constexpr int U = 8;
    const int tid = threadIdx.x, words = (x.n + 31) / 32;
    for (int w0 = (tid >> 5) * U; w0 < words; w0 += kWarps * U) {
        float v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int i = (w0 + j) * 32 + (tid & 31);
            v[j] = i < x.n ? x.value(i) : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const u32 m = __ballot_sync(0xffffffffu, v[j] >= least);
            if ((tid & 31) == j && w0 + j < words) marks[w0 + j] = m;
        }
        if (REST) {
#pragma unroll
            for (int j = 0; j < U; ++j)
                v[j] = v[j] >= least ? 0.0f : fast_exp2((v[j] - r.max_f) * r.scale_f);
            *rest += (double)(((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])));
        }
    }
    return give_marked(s, x.skip, x.n, marks, put);
}

// The same over a row that is not kept.
template <bool REST, typename T, typename F>
__device__ int list(Shared& s, const Row& r, const Far<T>& x, void* ring, float least, u32* marks,
                    double* rest, F put) {
    constexpr int N = kTile * 16 / sizeof(T);  // words of a warp's part of a tile
    const int lane = threadIdx.x & 31, words = (x.n + 31) / 32;
    Walk<T> walk(x, ring);
    for (int t = 0; t < walk.tiles; ++t) {
        const T* part = reinterpret_cast<const T*>(walk.tile(t));
        const int w0 = walk.first(t) * Walk<T>::P / 32;
        float v[N];
        u32 mine = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            v[j] = number<T>(part[j * 32 + lane]);
            const u32 m = __ballot_sync(0xffffffffu, v[j] >= least);
            mine = lane == j ? m : mine;
        }
        if (lane < N && w0 + lane < words) marks[w0 + lane] = mine;
        if (REST) {
            float sum[2] = {0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < N; ++j)
                sum[j & 1] += v[j] >= least ? 0.0f : fast_exp2((v[j] - r.max_f) * r.scale_f);
            *rest += (double)(sum[0] + sum[1]);
        }
    }
    return give_marked(s, x.skip, x.n, marks, put);
}

// Place of the m-th marked, from 0, in the thread that finds it; -1 in others.
__device__ __forceinline__ int marked_place(Shared& s, int n, const u32* marks, u32 m) {
    const int words = (n + 31) / 32, each = (words + kThreads - 1) / kThreads;
    const int lo = min((int)threadIdx.x * each, words), hi = min(lo + each, words);
    u32 mine = 0;
    for (int w = lo; w < hi; ++w) mine += __popc(marks[w]);
    u32 at = (u32)block_upto(s, mine) - mine;
    if (m < at || m >= at + mine) return -1;
    for (int w = lo; w < hi; ++w)
        for (u32 b = marks[w]; b; b &= b - 1)
            if (at++ == m) return w * 32 + __ffs(b) - 1;
    return -1;
}

struct Rule {
    int k;              // 0: none
    double p, u;        // p of 1: none
    u64 w_floor;        // least weight
    __device__ __forceinline__ u64 aim(u64 total) const {  // u of the kept weight
        const double t = u * (double)total;
        return !(t > 0.0) ? 0ull : t >= (double)total ? total - 1 : min((u64)t, total - 1);
    }
};

// The draw among the listed ids of a top-k row, if they are kList at most in all
// CTAs together (what was listed counts here, not what the bins foretold), by the
// CTA of rank 0: a thread for each id, which counts and weighs those ahead of
// it. The lists are in order of id. *drawn: the id (first + x.id), -1 in other
// CTAs. False, in every CTA alike, where they are more.
template <bool ONE, typename L>
__device__ bool draw_few(Shared& s, const Row& r, const L& x, int first, const Rule& g,
                         Team<ONE> t, int* drawn) {
    const int tid = threadIdx.x;
    u64* told = s.told[13];  // (a line of top-p without top-k)
    // each CTA leaves its keys and ids where rank 0 reads them
    for (int i = tid; i < min(x.n, kList); i += kThreads) {
        s.list[0][i] = key_of(x.value(i));
        s.list[1][i] = (u32)(first + x.id(i));
    }
    t.tell(told, (u64)x.n);
    t.sync();
    u64 count = 0;
    for (u32 c = 0; c < t.ctas; ++c) count += told[c];
    if (count > kList) return false;
    if (t.rank == 0) {
        u32 at;
        const u32 c = t.place(told, tid, &at);
        const bool in = c < t.ctas;
        const u32 mine = in ? t.read(&s.list[0][at], c) : 0;
        const u32 id = in ? t.read(&s.list[1][at], c) : 0;
        const u64 w = in ? weigh(r, s, value_of(mine)) : 0;
        s.all[tid] = mine;  // no key behind the last
        s.weight[tid] = w;
        __syncthreads();
        int more = 0;   // larger ones
        u64 ahead = 0;  // weight of the ids before this in descending order
        if (in) {
#pragma unroll 8
            for (int j = 0; j < (int)(count + 7) / 8 * 8; ++j) {
                const u32 k = s.all[j];
                more += k > mine;
                ahead += k > mine || (k == mine && j < tid) ? s.weight[j] : 0;
            }
        }
        bool stays = in && more < g.k;
        const u64 target = g.p < 1.0 ? share(g.p, block_add(s, stays ? w : 0)) : ~0ull;
        stays = stays && ahead < target && w >= g.w_floor;
        const u64 upto = block_upto(s, stays ? w : 0);
        if (tid == kThreads - 1) s.found[1] = upto;
        __syncthreads();
        const u64 goal = g.aim(s.found[1]);
        if (stays && goal < upto && goal >= upto - w) s.found[0] = id;
    }
    t.sync();  // no CTA ends while rank 0 may still read from it
    *drawn = t.rank == 0 ? (int)s.found[0] : -1;
    return true;
}

// The draw among the ids of x (all of the slice's, or its listed ones) by the
// whole cluster. rest: of the ids that x leaves out, whose weight exact(key)
// gives as that of smaller keys. Returns the index in x, -1 in other CTAs.
template <bool ONE, typename S, typename E>
__device__ int draw(Shared& s, const Row& r, const S& x, int first, const Rule& g, Range range,
                    Rest rest, Team<ONE> t, E exact) {
    u32 key = 0;            // kept: larger keys, and of the equal ones ids up to `last`
    int last = 0x7fffffff;
    if (g.k > 0) {
        const Border b = border<false>(s, r, x, range, (u64)g.k, 0.0, rest, t);
        key = b.key;
        range = {key, key_of(r.max_f), 0, (u32)min(b.ahead + b.ties, (u64)0xffffffffu)};
        rest = {0, 0, false};
    }
    if (g.p < 1.0) {
        Border b;
        u64 stay;
        for (;;) {
            b = border<true>(s, r, x, range, 0, g.p, rest, t);
            const u64 w = weigh(r, s, value_of(b.key));
            stay = w ? (b.target - b.ahead + w - 1) / w : b.ties;
            if (rest.least == rest.most) break;
            // the other end of the estimate: the same key, and as many of its ties?
            const u64 most = share(g.p, b.total + rest.most);
            if (most <= b.ahead + b.ties * w && (most - b.ahead + w - 1) / w == stay) break;
            t.sync();
            rest.least = rest.most = exact(range.from);
        }
        key = b.key;
        if (stay < b.ties) {
            const int i = first_beyond(
                s, x, s.told[7], t, [&](int, float v) { return (u64)(key_of(v) == key); },
                [&](u64) { return stay - 1; });
            if (i >= 0 && threadIdx.x < t.ctas)
                t.store(&s.told[0][0], threadIdx.x, (u64)(first + x.id(i)));
            t.sync();
            last = (int)s.told[0][0];
        }
    }
    return first_beyond(
        s, x, s.told[8], t,
        [&](int j, float v) -> u64 {
            const u32 q = key_of(v);
            const u64 w = weigh(r, s, v);  // for all: in a warp some lane needs it
            return q < key || (q == key && first + x.id(j) > last) || w < g.w_floor ? 0 : w;
        },
        [&](u64 total) { return g.aim(total); });
}

// HELD: the slice is kept in shared memory, in front of a list of its places (as
// many as it has). Otherwise the list is of a.cand logits.
template <typename T, bool HELD, bool ONE>
__global__ void __launch_bounds__(kThreads, 4) sample_kernel(const SampleArgs a) {
    extern __shared__ __align__(16) float dyn[];
    __shared__ Shared s;
    const int tid = threadIdx.x;
    const Team<ONE> t;
    t.started();
    const int row = blockIdx.x / t.ctas;
    const int first = min((long long)t.rank * a.slice, (long long)a.V);
    Far<T> far;
    {
        const T* x = static_cast<const T*>(a.logits) + row * a.ld + first;
        far.skip = (int)((uintptr_t)x & 15) / (int)sizeof(T);
        far.x = x - far.skip;
        far.n = min(a.slice, a.V - first) + far.skip;
    }
    const double T_ = a.temperature.at(row);
    const bool greedy = !(T_ > 0.0);
    Rule g;
    g.k = a.top_k ? a.top_k[row] : a.one_k;
    if (g.k < 0 || g.k >= a.V) g.k = 0;
    g.p = a.top_p.at(row);
    if (!(g.p > 0.0 && g.p < 1.0)) g.p = 1.0;
    const double q = fmin(a.min_p.at(row), 1.0);
    const double least_w = q * two_to(a.bits);
    g.w_floor = least_w > 0.0 ? (u64)ceil(least_w) : 0;
    g.u = a.u_wide ? static_cast<const double*>(a.u)[row]
                   : (double)static_cast<const float*>(a.u)[row];
    Row r;
    r.scale = fmin(1.4426950408889634074 / T_, 1e300);
    r.scale_f = (float)fmin(r.scale, 3e38);
    r.unit = two_to(52 - a.bits);
    const double reach = 64.0 / r.scale;
    // (a scale that fp32 does not hold well: no estimates)
    const bool bins = !greedy && (g.k > 0 || g.p < 1.0) && r.scale > 1e-30 && r.scale < 1e30 &&
                      a.V < 1 << 20;
    if (tid < kPow) s.pow[tid] = g_pow.v[tid];
    if (bins) {
        // The bins have to be in place before the row is read, its largest logit
        // not known: they reach from 24 temperatures above the largest of the
        // first kProbe logits to 32 below (beyond, every weight is 0), and at
        // high temperatures over 112 at most. Where that is the wrong place the
        // first or the last bin holds what matters, and the row goes on as if
        // it had not been counted.
        float v = -INFINITY;
        const T* x = static_cast<const T*>(a.logits) + row * a.ld;
#pragma unroll
        for (int j = 0; j < kProbe / kThreads; ++j)
            if (j * kThreads + tid < a.V) v = fmaxf(v, number<T>(x[j * kThreads + tid]));
        const u32 k = __reduce_max_sync(0xffffffffu, key_of(v));
        if ((tid & 31) == 0) s.warp_sum[tid >> 5] = k;
        for (int b = tid; b < kCut; b += kThreads) s.count[b] = 0;
        __syncthreads();
        u32 first_most = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) first_most = max(first_most, (u32)s.warp_sum[w]);
        const float t8 = (float)fmin(8.0 * T_, 16.0);
        r.ref = (first_most == kNothing ? 0.0f : fminf(value_of(first_most), 3e38f)) + 3.0f * t8;
        r.bin = fminf((kCut - 4) / (7.0f * t8), 3e38f);
    }

    // one pass over the slice: the largest; its id (greedy); the counts; the
    // sum of the weights' estimates (top-p alone)
    float best = -INFINITY, e[4] = {0, 0, 0, 0};
    int best_at = 0;
    const auto pass = [&](auto f) {
        if constexpr (HELD) {
            constexpr int P = Far<T>::P, U = Far<T>::U;
            const int packs = far.packs();
            for (int q = tid; q < packs; q += U * kThreads) {
                float v[U][P];
#pragma unroll
                for (int j = 0; j < U; ++j)
                    if (q + j * kThreads < packs) far.load(q + j * kThreads, v[j]);
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    if (q + j * kThreads >= packs) break;
#pragma unroll
                    for (int i = 0; i < P; i += 4)
                        reinterpret_cast<float4*>(dyn)[((q + j * kThreads) * P + i) / 4] =
                            make_float4(v[j][i], v[j][i + 1], v[j][i + 2], v[j][i + 3]);
#pragma unroll
                    for (int i = 0; i < P; ++i) f(v[j][i], i);
                }
            }
        } else if constexpr (ONE) {
            walk_all(far, dyn, [&](int, float v, int i) { f(v, i); });
        } else {
            each(far, [&](int, float v, int i) { f(v, i); });
        }
    };
    if (greedy) {
        const auto keep = [&](int i, float v, int) {
            best_at = v > best ? i : best_at;
            best = fmaxf(best, v);
        };
        if constexpr (!HELD && ONE)
            walk_all(far, dyn, keep);
        else
            each(far, keep);
    } else if (!bins) {
        pass([&](float v, int) { best = fmaxf(best, v); });
    } else if (g.k > 0) {
        pass([&](float v, int) {
            best = fmaxf(best, v);
            atomicAdd(&s.count[linear_bin(r, v)], 1u);
        });
    } else {
        pass([&](float v, int i) {
            best = fmaxf(best, v);
            atomicAdd(&s.count[linear_bin(r, v)], 1u);
            e[i & 3] += fast_exp2((v - r.ref) * r.scale_f);
        });
    }
    double sum = 0.0;
    if (bins && g.k <= 0) {
        sum = ((double)e[0] + e[1]) + ((double)e[2] + e[3]);
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        __syncthreads();
        if ((tid & 31) == 0) s.warp_sum[tid >> 5] = (u64)__double_as_longlong(sum);
    }
    u64 most = __reduce_max_sync(0xffffffffu, key_of(best));
    const u32 id = (u32)most == key_of(best) ? (u32)(first + far.id(best_at)) : 0xffffffffu;
    most = most << 32 | ~__reduce_min_sync(0xffffffffu, greedy ? id : 0);
    if ((tid & 31) == 0) s.red[tid >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kWarps; ++k) most = s.red[k] > most ? s.red[k] : most;
    t.all_started();
    if (bins && g.k <= 0) {  // in the order of the warps, then of the CTAs
        sum = 0.0;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) sum += __longlong_as_double((long long)s.warp_sum[k]);
        t.tell(s.told[9], (u64)__double_as_longlong(sum));
    }
    t.tell(s.told[0], most);
    t.sync();
    sum = 0.0;
#pragma unroll
    for (int c = 0; c < (ONE ? 1 : kMaxCluster); ++c)
        if (c < (int)t.ctas) {
            most = s.told[0][c] > most ? s.told[0][c] : most;
            if (bins && g.k <= 0) sum += __longlong_as_double((long long)s.told[9][c]);
        }

    const u32 top = (u32)(most >> 32);
    if (top == kNothing || greedy) {
        if (t.rank == 0 && tid == 0)
            a.out[row] = top == kNothing ? -1 : (int)~(u32)most;
        return;
    }
    r.max_f = value_of(top);
    const auto x = [&] {
        if constexpr (HELD)
            return Near{dyn, far.n, far.skip};
        else
            return far;
    }();
    if (r.max_f == INFINITY) {  // nothing but the largest: its lowest id
        const int i = first_beyond(
            s, x, s.told[8], t, [&](int, float v) { return (u64)(v == INFINITY); },
            [](u64) { return 0ull; });
        if (i >= 0 && tid == 0) a.out[row] = first + x.id(i);
        t.sync();  // no CTA ends while another may still read from it
        return;
    }
    r.max = r.max_f;
    r.cutoff = fmaxf(__double2float_ru(r.max - reach), -3.402823466e38f);
    Range range{kNothing, top, 0, (u32)a.V};
    const auto exact = [&](u32 from) {
        u64 sum = 0;
        each_weighed(r, s, x, [&](float v, u64 w) { sum += key_of(v) < from ? w : 0; });
        t.tell(s.told[12], block_add(s, sum));
        t.sync();
        sum = 0;
        for (u32 c = 0; c < t.ctas; ++c) sum += s.told[12][c];
        return sum;
    };
    u32 listed = 0;   // ids that can stay, where they are to be listed
    float least = 0;  // their least logit
    if (bins) {
        Range found;
        const u32 n = cut(s, r, a.V, g.k, g.p, a.bits, t, sum, &found);
        if (n) range = found;
        // every CTA of the cluster decides alike
        if (n && (HELD ? n <= (u32)a.V / 2 : ONE && n <= (u32)a.cand)) listed = n;
        least = value_of(range.from);
    } else if (g.w_floor > 0 && g.k == 0 && g.p == 1.0 && (HELD || ONE)) {
        // where x < max + T ln(min_p) by more than the roundings here, w is below min_p
        const double edge = T_ * log(q);
        least = __double2float_rd(r.max + edge - 1e-9 * fabs(edge));
        listed = (u32)a.V;
    }
    if constexpr (HELD || ONE) {
        if (listed) {
            double others = 0.0;  // estimate of the weight that is not listed (top-p alone)
            const auto finish = [&](const auto& l) {
                int few;
                if (g.k > 0 && listed <= kList && draw_few(s, r, l, first, g, t, &few)) return few;
                Rest rest{0, 0, false};
                if (g.k <= 0 && g.p < 1.0) {
                    // Each 2^d is off by 2^-22 of itself, by the roundings of the
                    // difference and the product and by the scale's in fp32,
                    // (2 * 2^-24 + that) |d| ln 2, and by 10 of sums in fp32. The
                    // mean of |d|, by weight, is the entropy of the weights less
                    // log2 of their sum, at most log2(V / sum).
                    double v = others;
#pragma unroll
                    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
                    __syncthreads();
                    if ((tid & 31) == 0) s.warp_sum[tid >> 5] = (u64)__double_as_longlong(v);
                    __syncthreads();
                    v = 0.0;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) v += __longlong_as_double((long long)s.warp_sum[w]);
                    t.tell(s.told[13], (u64)__double_as_longlong(v));
                    t.sync();
                    v = 0.0;
                    for (u32 c = 0; c < t.ctas; ++c) v += __longlong_as_double((long long)s.told[13][c]);
                    if (v > 0x1p-100) {
                        const double mean = ilogb(a.V / v) + 1;
                        const double scale = fabs(r.scale_f / r.scale - 1.0);
                        const double off = 0x1p-22 + 10 * 0x1p-24 +
                                           (2 * 0x1p-24 + scale) * 0.694 * mean;
                        const double units = v * two_to(a.bits), err = 1.01 * off * units + a.V;
                        rest.least = units > err ? (u64)(units - err) : 0;
                        rest.most = (u64)(units + err);  // (exact weights are rounded, too)
                    } else {
                        rest.most = a.V;
                    }
                }
                const int i = draw(s, r, l, first, g, range, rest, t, exact);
                t.sync();
                return i < 0 ? -1 : first + l.id(i);
            };
            const auto listing = [&](u32* marks, auto put) {
                if constexpr (HELD)
                    return g.k <= 0 && g.p < 1.0 ? list<true>(s, r, x, least, marks, &others, put)
                                                 : list<false>(s, r, x, least, marks, &others, put);
                else
                    return g.k <= 0 && g.p < 1.0
                               ? list<true>(s, r, x, dyn, least, marks, &others, put)
                               : list<false>(s, r, x, dyn, least, marks, &others, put);
            };
            if constexpr (HELD) {
                unsigned short* at = reinterpret_cast<unsigned short*>(dyn + a.slice + 8);
                u32* marks = reinterpret_cast<u32*>(at + a.slice + 8);
                const int n = listing(marks, [&](u32 pos, int i) {
                    at[pos] = (unsigned short)i;
                });
                const int id = finish(NearListed{x, at, n});
                if (id >= 0 && tid == 0) a.out[row] = id;
                return;
            } else {
                u32* marks = reinterpret_cast<u32*>(dyn + a.cand);
                u32* at = reinterpret_cast<u32*>(dyn);  // places first, then the logits there
                const int n = listing(marks, [&](u32 pos, int i) {
                    if (pos < (u32)a.cand) at[pos] = (u32)i;
                });
                if (n <= a.cand) {  // always where the bins counted them
#pragma unroll 8
                    for (int i = tid; i < n; i += kThreads) dyn[i] = x.value((int)at[i]);
                    __syncthreads();
                    const int m = finish(FarListed{dyn, n});
                    const int i = marked_place(s, x.n, marks, (u32)m);
                    if (i >= 0) a.out[row] = x.id(i);
                    return;
                }
            }
        }
    }
    const int i = draw(s, r, x, first, g, range, Rest{0, 0, g.k <= 0}, t, exact);
    if (i >= 0 && tid == 0) a.out[row] = first + x.id(i);
    t.sync();
}

template <typename T, bool HELD, bool ONE>
int start(const SampleArgs& a, int B, int ctas, size_t dyn, cudaStream_t st) {
    const auto kern = sample_kernel<T, HELD, ONE>;
    if (dyn + sizeof(Shared) > 48 * 1024)
        SN_TRY(cuda_check(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               200 * 1024),
                          "sample"));
    if (ONE) {
        kern<<<B, kThreads, dyn, st>>>(a);
        return cuda_check(cudaGetLastError(), "sample launch");
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)B * ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = dyn;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cuda_check(cudaLaunchKernelEx(&cfg, kern, a), "sample launch");
}

template <typename T>
int launch(SampleArgs& a, int B, int sms, cudaStream_t st) {
    // A row for every SM: a row to a CTA (256 x 32000 top-k takes 24 us so, 48 in
    // clusters of 4; 160 x 32000 23 and 33). Fewer: slices of 8192 logits, cut
    // further down to 2048 while the SMs have less than two CTAs each (one row
    // of 32000 takes 13 us in eight CTAs).
    const bool one = B >= sms;
    int ctas = 1;
    while (!one && ctas < kMaxCluster &&
           ((long long)ctas * 8192 < a.V ||
            ((long long)B * ctas < 2ll * sms && (long long)ctas * 2048 < a.V)))
        ctas *= 2;
    a.slice = (int)(((long long)a.V + ctas - 1) / ctas + 7) / 8 * 8;
    // the slice in fp32 behind up to 7 skipped places, a list of places in 16
    // bits, and a bit for each
    const size_t marks = (size_t)(a.slice + 8 + 31) / 32 * 4, held = (size_t)(a.slice + 8) * 6 + marks;
    if (ctas == 1 && a.slice > 8192) {
        // the more rows an SM has at once the shorter their lists
        a.cand = B >= 4 * sms ? kCand : B >= 2 * sms ? 3 * kCand / 2 : 11 * kCand / 4;
        if (4 * (size_t)a.cand + marks > 200 * 1024) a.cand = kCand;
        const size_t dyn = 4 * (size_t)a.cand + marks;
        if (dyn <= 200 * 1024) return start<T, false, true>(a, B, 1, dyn, st);
    }
    if (held > 200 * 1024) return start<T, false, false>(a, B, ctas, 0, st);
    return ctas == 1 ? start<T, true, true>(a, B, 1, held, st)
                     : start<T, true, false>(a, B, ctas, held, st);
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
    SampleArgs a{logits, u, top_k, tokens, {temperature, temperature0}, {top_p, top_p0},
                 {min_p, min_p0}, ld, top_k0, u_f64, V, 0, 44, 0};
    while (std::ldexp((double)V, a.bits) >= std::ldexp(1.0, 62)) --a.bits;
    const cudaStream_t st = static_cast<cudaStream_t>(cuda_stream);
    switch (dtype) {
        case SN_F32: return launch<float>(a, B, dev.num_sms(), st);
        case SN_BF16: return launch<__nv_bfloat16>(a, B, dev.num_sms(), st);
        default: return launch<__half>(a, B, dev.num_sms(), st);
    }
}
