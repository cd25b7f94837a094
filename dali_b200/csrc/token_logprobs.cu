// Log probabilities of given tokens, the entropy of the distribution they are drawn from and its most probable tokens, from
// rows of logits z, and the gradient: dalib200_token_logprobs, dalib200_token_logprobs_backward.
//
//   lse = log sum_j exp z_j,  log p_j = z_j - lse,  logprob = log p_t,  H = - sum_j p_j log p_j
//   dz_j = g ([j = t] - p_j) - w p_j (log p_j + H)         for the gradients g of logprob and w of H
//
// One pass over the row with the running maximum m and, relative to it, s = sum exp(z - m) and u = sum (z - m) exp(z - m):
// lse = m + log s and H = log s - u / s, a sum of two terms that are not negative.  When m grows to m', both sums are scaled
// by c = exp(m - m') after u has been moved: u' = c (u + (m - m') s).
//
// An entry of -infinity is one that cannot be drawn (p = 0, 0 log 0 = 0); a row of nothing else has lse = -infinity,
// logprob = -infinity and H = 0.  The alternatives are ordered by value and, among equal values, by index; NaN ranks last.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "op_device.cuh"
#include "op_host.h"

namespace dalib {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = DALIB200_MAX_TOP;

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float log_of(float x) { return logf(x); }
__device__ __forceinline__ double log_of(double x) { return log(x); }
__device__ __forceinline__ float nan_of(float) { return __int_as_float(0x7fffffff); }
__device__ __forceinline__ double nan_of(double) { return __longlong_as_double(0x7fffffffffffffffll); }
__device__ __forceinline__ float infinity_of(float) { return __int_as_float(0x7f800000); }
__device__ __forceinline__ double infinity_of(double) { return __longlong_as_double(0x7ff0000000000000ll); }
// the larger of two numbers, NaN if one is NaN
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ double max_nan(double a, double b) { return a != a ? a : b != b ? b : a > b ? a : b; }
template <typename A> struct Lowest;
template <> struct Lowest<float> { static __device__ __forceinline__ float value() { return -FLT_MAX; } };
template <> struct Lowest<double> { static __device__ __forceinline__ double value() { return -DBL_MAX; } };
// exp(d) is 0 in either type below this; differences are not let fall lower, so that 0 * d stays 0 for d = -infinity
template <typename A> __device__ __forceinline__ A floor_of_difference() { return sizeof(A) == 8 ? (A)-1000 : (A)-200; }

// m >= every entry seen and >= the lowest finite number; s, u relative to m.  NaN or +infinity in the row make s and u NaN.
template <typename A>
struct Running {
    A m, s, u;
    __device__ __forceinline__ void clear() { m = Lowest<A>::value(); s = 0; u = 0; }
    __device__ __forceinline__ void raise(A to) {      // to >= m
        const A d = max_nan(m - to, floor_of_difference<A>());
        const A c = exp_of(d);
        u = c * (u + d * s);
        s = c * s;
        m = to;
    }
    __device__ __forceinline__ void add(A z) {         // z <= m, or NaN
        const A d = max_nan(z - m, floor_of_difference<A>());
        const A e = exp_of(d);
        s += e;
        u += d * e;
    }
    __device__ __forceinline__ void take(A z) {
        if (z > m) raise(z);
        add(z);
    }
    __device__ __forceinline__ void merge(Running o) {
        if (o.m > m) raise(o.m);
        else if (m > o.m) o.raise(m);
        s += o.s;
        u += o.u;
    }
};

// Values ordered as unsigned integers: larger value, larger key; -0 equals +0; NaN is 0.
__device__ __forceinline__ uint32_t ordered(float z) {
    if (z != z) return 0;
    const uint32_t b = __float_as_uint(z + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long ordered(double z) {
    if (z != z) return 0;
    const unsigned long long b = (unsigned long long)__double_as_longlong(z + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
// (value, index): larger value first, then smaller index
template <typename A>
struct Ranked {
    decltype(ordered(A())) value;
    uint32_t index;
    __device__ __forceinline__ bool before(const Ranked& o) const { return value > o.value || (value == o.value && index < o.index); }
};

// What a thread of the row's CTA has to say when the statistics are known.
template <typename A>
__device__ __forceinline__ void finish_row(const Running<A>& all, long long row, A* logprob, A* entropy, A* lse_out, A* lse) {
    A l, h;
    if (all.s == 0) {              // nothing but -infinity
        l = -infinity_of(A());
        h = 0;
    } else {
        const A ls = log_of(all.s);
        l = all.m + ls;
        h = ls - all.u / all.s;
    }
    *lse = l;
    if (entropy) entropy[row] = h;
    if (lse_out) lse_out[row] = l;
    (void)logprob;
}

// log p of an entry
template <typename A>
__device__ __forceinline__ A log_p(A z, A lse) { return lse == -infinity_of(A()) ? lse : z - lse; }

// ---------------------------------------------------------------------------------------------- f64 rows
// A CTA per row, one entry a thread and step; the alternatives one after another, each by another walk over the row.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_rows_kernel(const T* __restrict__ logits, long long ld, long long rows, int vocab,
                                                                 const int* __restrict__ tokens, typename AccOf<T>::type* logprob,
                                                                 typename AccOf<T>::type* entropy, typename AccOf<T>::type* lse_out,
                                                                 int top, typename AccOf<T>::type* top_logprobs, int* top_tokens) {
    typedef typename AccOf<T>::type A;
    __shared__ Running<A> sm[kThreads / 32];
    __shared__ Ranked<A> best[kThreads / 32];
    dependent_prologue();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* z = logits + row * ld;
        Running<A> r;
        r.clear();
        for (int j = threadIdx.x; j < vocab; j += kThreads) r.take(widen(z[j]));
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) {
            Running<A> o;
            o.m = __shfl_xor_sync(0xffffffffu, r.m, m);
            o.s = __shfl_xor_sync(0xffffffffu, r.s, m);
            o.u = __shfl_xor_sync(0xffffffffu, r.u, m);
            r.merge(o);
        }
        __syncthreads();
        if (lane == 0) sm[warp] = r;
        __syncthreads();
        Running<A> all = sm[0];
        for (int w = 1; w < kThreads / 32; ++w) all.merge(sm[w]);
        A lse;
        if (threadIdx.x == 0) {
            finish_row(all, row, logprob, entropy, lse_out, &lse);
            if (logprob) {
                const int t = tokens[row];
                logprob[row] = t < 0 ? (A)0 : t >= vocab ? nan_of(A()) : log_p((A)widen(z[t]), lse);
            }
        }
        Ranked<A> last;
        for (int k = 0; k < top; ++k) {
            Ranked<A> b = {0, 0xffffffffu};
            for (int j = threadIdx.x; j < vocab; j += kThreads) {
                const Ranked<A> c = {ordered(widen(z[j])), (uint32_t)j};
                if ((k == 0 || last.before(c)) && c.before(b)) b = c;
            }
#pragma unroll
            for (int m = 16; m > 0; m >>= 1) {
                Ranked<A> o;
                o.value = __shfl_xor_sync(0xffffffffu, b.value, m);
                o.index = __shfl_xor_sync(0xffffffffu, b.index, m);
                if (o.before(b)) b = o;
            }
            __syncthreads();
            if (lane == 0) best[warp] = b;
            __syncthreads();
            last = best[0];
            for (int w = 1; w < kThreads / 32; ++w)
                if (best[w].before(last)) last = best[w];
            if (threadIdx.x == 0) {
                top_tokens[row * top + k] = (int)last.index;
                top_logprobs[row * top + k] = log_p((A)widen(z[last.index]), lse);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- f32 and bf16 rows
// A cluster of S CTAs shares a row, each a contiguous slice of its 16-byte packets; a thread takes every kThreads-th packet of
// its CTA's slice, kBatch of them at a time, and keeps (m, s, u) in units of log 2: t = (z - m) log2 e, s = sum 2^t,
// u = sum t 2^t.  (z - m is formed before it is scaled: a row of the type's lowest value is uniform, not -infinity.)
//
// The alternatives cost no work in that pass.  The entries of one thread are a GROUP; a thread remembers in which batch its
// maximum was raised last.  At least `top` entries are >= the top-th largest group maximum tau (by value, then index: a total order),
// and every entry >= tau lies in one of those `top` groups: only they are read again (from L2, 1 / 256 of a CTA's slice each), and
// what is >= tau in them, hardly more than `top` entries, is sorted.  Lists of 32 keys, one a lane, are sorted and merged
// bitonically.
constexpr int kBatch = 4;
constexpr int kWarps = kThreads / 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kFloor = -290.0f;              // 2^t is 0 in fp32 below; t does not fall lower, so that 0 * t stays 0 for t = -infinity

__device__ __forceinline__ float exp2_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// the largest value of some packets (NaN counts only if there is nothing else)
__device__ __forceinline__ uint32_t max_of_pairs(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <int B>
__device__ __forceinline__ float largest(const uint4 (&q)[B], float*) {
    float m = __uint_as_float(q[0].x);
#pragma unroll
    for (int i = 0; i < B; ++i)
        m = fmaxf(fmaxf(m, __uint_as_float(q[i].x)), fmaxf(fmaxf(__uint_as_float(q[i].y), __uint_as_float(q[i].z)), __uint_as_float(q[i].w)));
    return m;
}
template <int B>
__device__ __forceinline__ float largest(const uint4 (&q)[B], bf16_s*) {
    uint32_t m = q[0].x;
#pragma unroll
    for (int i = 0; i < B; ++i) m = max_of_pairs(max_of_pairs(m, q[i].x), max_of_pairs(max_of_pairs(q[i].y, q[i].z), q[i].w));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ uint4 packet_of_minus_infinity();
template <> __device__ __forceinline__ uint4 packet_of_minus_infinity<float>() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
template <> __device__ __forceinline__ uint4 packet_of_minus_infinity<bf16_s>() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }

// (m, s, u) in units of log 2
struct Running2 {
    float m, s, u;
    __device__ __forceinline__ void raise(float to) {
        const float t = max_nan((m - to) * kLog2e, kFloor);
        const float c = exp2_of(t);
        u = c * (u + t * s);
        s = c * s;
        m = to;
    }
    __device__ __forceinline__ void merge(Running2 o) {
        if (o.m > m) raise(o.m);
        else if (m > o.m) o.raise(m);
        s += o.s;
        u += o.u;
    }
};

// Keys: (ordered value, ~index), so that a larger key is a larger value or the same value at a lower index; no two entries share
// one; 0 is no entry.
typedef unsigned long long Key;
__device__ __forceinline__ Key key_of(float z, int index) { return ((Key)ordered(z) << 32) | (uint32_t)~index; }
__device__ __forceinline__ int index_of(Key k) { return (int)~(uint32_t)k; }
__device__ __forceinline__ Key exchange(Key k, int mask) { return __shfl_xor_sync(0xffffffffu, k, mask); }
__device__ __forceinline__ Key keep(Key mine, Key other, bool larger) { return (mine > other) == larger ? mine : other; }
// one key a lane; descending from lane 0
__device__ __forceinline__ Key merge_down(Key k, int lane) {
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) k = keep(k, exchange(k, j), (lane & j) == 0);
    return k;
}
__device__ __forceinline__ Key sort_down(Key k, int lane) {
#pragma unroll
    for (int w = 2; w <= 32; w <<= 1)
#pragma unroll
        for (int j = w >> 1; j > 0; j >>= 1) k = keep(k, exchange(k, j), ((lane & j) == 0) == ((lane & w) == 0 || w == 32));
    return k;
}
// the 32 largest of two descending lists; b is read backwards from memory
__device__ __forceinline__ Key join(Key a, const Key* b, int lane) {
    const Key o = b[31 - lane];
    return merge_down(a > o ? a : o, lane);
}
// The 32 largest keys of `n` (a power of two <= 2 * kWarps) descending lists in shared memory, left in list 0.
__device__ __forceinline__ void join_lists(Key (*lists)[32], int n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncthreads();
    for (int half = n >> 1; half > 0; half >>= 1) {
        if (warp < half) lists[warp][lane] = join(lists[warp][lane], lists[warp + half], lane);
        __syncthreads();
    }
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// the same shared-memory word in CTA 0 of the cluster
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)));
    return r;
}
__device__ __forceinline__ void store_remote(uint32_t at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }
__device__ __forceinline__ void store_remote(uint32_t at, Key v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }

constexpr int kMaxCluster = 16;

// A row as the kernel walks it: `head` entries up to the 16-byte grid, whole packets, `tail` entries.
template <typename T>
struct RowSplit {
    static constexpr int N = Packet<T>::N;
    const T* z;
    int head, tail, packets;
    __device__ __forceinline__ RowSplit(const T* row, int vocab) : z(row) {
        const int off = (int)(((uintptr_t)row & 15) / sizeof(T));
        head = off ? min(N - off, vocab) : 0;
        packets = (vocab - head) / N;
        tail = vocab - head - packets * N;
    }
    __device__ __forceinline__ int first_of(int packet) const { return head + packet * N; }
    __device__ __forceinline__ uint4 packet(int p) const { return *reinterpret_cast<const uint4*>(z + first_of(p)); }
    // the i-th of the head + tail entries
    __device__ __forceinline__ int edge(int i) const { return i < head ? i : i + packets * N; }
};

template <typename T>
__device__ __forceinline__ float entry(uint4 q, int e);
template <> __device__ __forceinline__ float entry<float>(uint4 q, int e) { return __uint_as_float(e == 0 ? q.x : e == 1 ? q.y : e == 2 ? q.z : q.w); }
template <> __device__ __forceinline__ float entry<bf16_s>(uint4 q, int e) {
    const uint32_t w = (e >> 1) == 0 ? q.x : (e >> 1) == 1 ? q.y : (e >> 1) == 2 ? q.z : q.w;
    return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
}

// The `top` largest entries of the CTA's packets [begin, end) (and, in the first CTA, of the row's edges) as a descending list in lists[0].
// best_batch: the thread's batch whose maximum raised its own last, -1: none did (nothing but -infinity and NaN).
template <typename T>
__device__ __forceinline__ void top_of_slice(const RowSplit<T>& row, int begin, int end, bool edges, int top, int best_batch, Key (*lists)[32],
                                             Key (*pending)[64]) {
    constexpr int N = Packet<T>::N;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n_edges = edges ? row.head + row.tail : 0;
    // the thread's largest key: its place is looked up in the batch that holds it
    Key mine = 0;
    {
        const int from = best_batch >= 0 ? best_batch : begin + tid;
        const int until = best_batch >= 0 ? min(end, best_batch + kBatch * kThreads) : end;
        for (int p = from; p < until; p += kThreads) {
            const uint4 q = row.packet(p);
#pragma unroll
            for (int e = 0; e < N; ++e) mine = max(mine, key_of(entry<T>(q, e), row.first_of(p) + e));
        }
        if (tid < n_edges) mine = max(mine, key_of(widen(row.z[row.edge(tid)]), row.edge(tid)));
    }
    lists[warp][lane] = sort_down(mine, lane);
    join_lists(lists, kWarps);
    const Key tau = max(lists[0][top - 1], (Key)1);
    const Key chosen = lane < top ? lists[0][lane] : 0;
    __syncthreads();
    // a warp reads every kWarps-th of the chosen groups
    Key best = 0;
    int waiting = 0;
    auto offer = [&](Key k) {
        const bool take = k >= tau;
        const uint32_t who = __ballot_sync(0xffffffffu, take);
        if (who == 0) return;
        if (take) pending[warp][waiting + __popc(who & ((1u << lane) - 1))] = k;
        waiting += __popc(who);
        __syncwarp();
        if (waiting >= 32) {
            const Key k32 = sort_down(pending[warp][lane], lane);
            const Key rest = pending[warp][32 + lane];
            __syncwarp();
            pending[warp][lane] = rest;
            const Key other = __shfl_sync(0xffffffffu, k32, 31 - lane);
            best = merge_down(best > other ? best : other, lane);
            waiting -= 32;
            __syncwarp();
        }
    };
    for (int g = warp; g < top; g += kWarps) {
        const Key k = __shfl_sync(0xffffffffu, chosen, g);
        if (k == 0) break;
        const int index = index_of(k);
        const bool at_edge = index < row.head || index >= row.head + row.packets * N;
        const int who = at_edge ? (index < row.head ? index : index - row.packets * N) : ((index - row.head) / N - begin) % kThreads;
        for (int p0 = begin + who; p0 < end; p0 += 32 * kThreads) {
            const int p = p0 + lane * kThreads;
            const bool there = p < end;
            uint4 q = packet_of_minus_infinity<T>();
            if (there) q = row.packet(p);
#pragma unroll
            for (int e = 0; e < N; ++e) offer(there ? key_of(entry<T>(q, e), row.first_of(p) + e) : 0);
        }
        if (who < n_edges) offer(lane == 0 ? key_of(widen(row.z[row.edge(who)]), row.edge(who)) : 0);
    }
    {
        const Key k32 = sort_down(lane < waiting ? pending[warp][lane] : 0, lane);
        const Key other = __shfl_sync(0xffffffffu, k32, 31 - lane);
        best = merge_down(best > other ? best : other, lane);
    }
    lists[warp][lane] = best;
    join_lists(lists, kWarps);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_kernel(const T* __restrict__ logits, long long ld, long long rows, int vocab,
                                                            const int* __restrict__ tokens, float* __restrict__ logprob,
                                                            float* __restrict__ entropy, float* __restrict__ lse_out, int top,
                                                            float* __restrict__ top_logprobs, int* __restrict__ top_tokens, int cluster) {
    constexpr int N = Packet<T>::N;
    __shared__ Running2 sm[kWarps];
    __shared__ Running2 from_cta[kMaxCluster];
    __shared__ Key lists[kMaxCluster][32];
    __shared__ Key pending[kWarps][64];
    __shared__ Key from_cta_keys[kMaxCluster][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    if (cluster > 1) cluster_arrive();          // every CTA of the cluster runs before its shared memory is written from another
    dependent_prologue();
    bool started = cluster == 1;
    for (long long r = blockIdx.x / cluster; r < rows; r += gridDim.x / cluster) {
        const RowSplit<T> row(logits + r * ld, vocab);
        const int share = (row.packets + cluster - 1) / cluster;
        const int begin = min(row.packets, rank * share), end = min(row.packets, begin + share);
        Running2 me = {Lowest<float>::value(), 0, 0};
        float seen = -infinity_of(0.0f);
        int best_batch = -1;
        {
            Two s2 = two(0, 0), u2 = two(0, 0);
            auto raise = [&](float to) {
                float a, b, c, d;
                parts(s2, a, b);
                parts(u2, c, d);
                me.s = a + b;
                me.u = c + d;
                me.raise(to);
                s2 = two(me.s, 0);
                u2 = two(me.u, 0);
            };
            for (int b = begin + tid; b < end; b += kBatch * kThreads) {
                uint4 q[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) q[i] = b + i * kThreads < end ? row.packet(b + i * kThreads) : packet_of_minus_infinity<T>();
                const float high = largest(q, (T*)nullptr);
                if (high > seen) {
                    seen = high;
                    best_batch = b;
                    if (high > me.m) raise(high);
                }
                const Two minus = two(-me.m, -me.m), scale = two(kLog2e, kLog2e);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    Two z[N / 2];
                    pairs_of(q[i], z, (T*)nullptr);
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) {
                        float t0, t1;
                        parts((z[e] + minus) * scale, t0, t1);
                        t0 = max_nan(t0, kFloor);
                        t1 = max_nan(t1, kFloor);
                        const Two p = two(exp2_of(t0), exp2_of(t1));
                        s2 = s2 + p;
                        u2 = multiply_add(two(t0, t1), p, u2);
                    }
                }
            }
            if (rank == 0 && tid < row.head + row.tail) {
                const float z = widen(row.z[row.edge(tid)]);
                if (z > me.m) raise(z);
                const float t = max_nan((z - me.m) * kLog2e, kFloor), p = exp2_of(t);
                s2 = s2 + two(p, 0);
                u2 = u2 + two(t * p, 0);
            }
            raise(me.m);
        }
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) {
            Running2 o;
            o.m = __shfl_xor_sync(0xffffffffu, me.m, m);
            o.s = __shfl_xor_sync(0xffffffffu, me.s, m);
            o.u = __shfl_xor_sync(0xffffffffu, me.u, m);
            me.merge(o);
        }
        __syncthreads();          // the row before has been written
        if (lane == 0) sm[warp] = me;
        if (top > 0) top_of_slice(row, begin, end, rank == 0, top, best_batch, lists, pending);
        else __syncthreads();
        if (cluster > 1) {
            if (!started) { cluster_wait(); started = true; }
            if (warp == 0) {
                if (lane == 0) {
                    Running2 all = sm[0];
#pragma unroll
                    for (int w = 1; w < kWarps; ++w) all.merge(sm[w]);
                    store_remote(in_first_cta(&from_cta[rank].m), all.m);
                    store_remote(in_first_cta(&from_cta[rank].s), all.s);
                    store_remote(in_first_cta(&from_cta[rank].u), all.u);
                }
                if (top > 0) store_remote(in_first_cta(&from_cta_keys[rank][lane]), lists[0][lane]);
            }
            cluster_arrive();
            cluster_wait();
            if (rank == 0 && top > 0) {
                for (int w = warp; w < cluster; w += kWarps) lists[w][lane] = from_cta_keys[w][lane];
                join_lists(lists, cluster);
            }
        }
        if (rank == 0 && warp == 0) {
            Running2 all = cluster > 1 ? from_cta[0] : sm[0];
            for (int w = 1; w < (cluster > 1 ? cluster : kWarps); ++w) all.merge(cluster > 1 ? from_cta[w] : sm[w]);
            float l, h;
            if (all.s == 0) {          // nothing but -infinity
                l = -infinity_of(0.0f);
                h = 0;
            } else {
                const float ls = logf(all.s);
                l = all.m + ls;
                h = ls - kLn2 * (all.u / all.s);
            }
            if (lane == 0) {
                if (entropy) entropy[r] = h;
                if (lse_out) lse_out[r] = l;
                if (logprob) {
                    const int t = tokens[r];
                    logprob[r] = t < 0 ? 0.0f : t >= vocab ? nan_of(0.0f) : log_p(widen(row.z[t]), l);
                }
            }
            if (lane < top) {
                const int index = index_of(lists[0][lane]);
                top_tokens[r * top + lane] = index;
                top_logprobs[r * top + lane] = log_p(widen(row.z[index]), l);
            }
        }
        if (cluster > 1) {           // the first CTA has read what the others sent for this row
            cluster_arrive();
            cluster_wait();
        }
    }
    if (!started) cluster_wait();
}

// ---------------------------------------------------------------------------------------------- gradient
// f64 rows, and rows of logits and gradients that do not lie alike on the 16-byte grid: a CTA per row, element by element.
template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_backward_rows_kernel(const T* logits, long long ld, long long rows, int vocab,
                                                                          const int* __restrict__ tokens,
                                                                          const typename AccOf<T>::type* __restrict__ lse,
                                                                          const typename AccOf<T>::type* __restrict__ entropy,
                                                                          const typename AccOf<T>::type* __restrict__ dlogprob,
                                                                          const typename AccOf<T>::type* __restrict__ dentropy, T* dlogits,
                                                                          long long ldd) {
    typedef typename AccOf<T>::type A;
    dependent_prologue();
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* z = logits + row * ld;
        T* out = dlogits + row * ldd;
        int t = dlogprob ? tokens[row] : -1;
        A g = t < 0 ? (A)0 : dlogprob[row];
        const A w = dentropy ? dentropy[row] : (A)0, h = dentropy ? entropy[row] : (A)0, l = lse[row];
        if (t >= vocab) g = nan_of(A());
        const bool nothing = (g == 0 && w == 0) || l == -infinity_of(A());
        for (int j = threadIdx.x; j < vocab; j += kThreads) {
            A d = 0;
            if (!nothing) {
                const A lp = max_nan((A)widen(z[j]) - l, floor_of_difference<A>());
                const A p = exp_of(lp);
                d = -p * (g + w * (lp + h));
                if (j == t) d += g;
            }
            out[j] = Narrow<T>::of(d);
        }
    }
}

// Everything else streams: a CTA takes kBatch packets a thread of one row, all loaded before the first is worked on, and p is
// exp2 of t = (z - lse) log2 e.  With dentropy:  dz = -p (g + w (log p + H)) = -p (a + b t),  a = g + w H, b = w / log2 e.
template <typename T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads) logprobs_backward_kernel(const T* logits, long long ld, long long pieces, int per_row, int vocab,
                                                                     const int* __restrict__ tokens, const float* __restrict__ lse,
                                                                     const float* __restrict__ entropy, const float* __restrict__ dlogprob,
                                                                     const float* __restrict__ dentropy, T* dlogits, long long ldd) {
    constexpr int N = Packet<T>::N;
    dependent_prologue();
    for (long long piece = blockIdx.x; piece < pieces; piece += gridDim.x) {
        const long long r = piece / per_row;
        const int part = (int)(piece - r * per_row);
        const RowSplit<T> row(logits + r * ld, vocab);
        T* out = dlogits + r * ldd;
        const int t = dlogprob ? tokens[r] : -1;
        const float g = t < 0 ? 0.0f : t >= vocab ? nan_of(0.0f) : dlogprob[r], l = lse[r];
        const float w = ENTROPY ? dentropy[r] : 0.0f, h = ENTROPY ? entropy[r] : 0.0f;
        const bool nothing = (g == 0 && w == 0) || l == -infinity_of(0.0f);
        const float a = -(g + w * h), b = -w * kLn2;
        const int begin = part * kBatch * kThreads + threadIdx.x;
        if (nothing) {          // 0 whatever the logits hold: they are not read
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (begin + i * kThreads < row.packets) *reinterpret_cast<uint4*>(out + row.first_of(begin + i * kThreads)) = make_uint4(0, 0, 0, 0);
            if (part == 0 && (int)threadIdx.x < row.head + row.tail) out[row.edge(threadIdx.x)] = Narrow<T>::of(0.0f);
            continue;
        }
        uint4 q[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (begin + i * kThreads < row.packets) q[i] = row.packet(begin + i * kThreads);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int p = begin + i * kThreads;
            if (p >= row.packets) break;
            Two z[N / 2];
            pairs_of(q[i], z, (const T*)nullptr);
#pragma unroll
            for (int e = 0; e < N / 2; ++e) {
                float t0, t1;
                parts((z[e] + both(-l)) * both(kLog2e), t0, t1);
                if (ENTROPY) {
                    t0 = max_nan(t0, kFloor);
                    t1 = max_nan(t1, kFloor);
                }
                const Two prob = two(exp2_of(t0), exp2_of(t1));
                z[e] = prob * (ENTROPY ? multiply_add(two(t0, t1), both(b), both(a)) : both(a));
            }
            const int j = t - row.first_of(p);
            if (j >= 0 && j < N) {
#pragma unroll
                for (int e = 0; e < N / 2; ++e) z[e] = z[e] + two(j == 2 * e ? g : 0.0f, j == 2 * e + 1 ? g : 0.0f);
            }
            *reinterpret_cast<uint4*>(out + row.first_of(p)) = packet_of(z, (const T*)nullptr);
        }
        if (part == 0 && (int)threadIdx.x < row.head + row.tail) {
            const int j = row.edge(threadIdx.x);
            const float t0 = max_nan((widen(row.z[j]) - l) * kLog2e, kFloor);
            out[j] = Narrow<T>::of(exp2_of(t0) * (t0 * b + a) + (j == t ? g : 0.0f));
        }
    }
}

long long capped(long long want, long long most) { return std::max<long long>(1, std::min(want, most)); }

template <typename T>
cudaError_t forward(cudaStream_t s, const Rows& z, const int* tokens, void* logprob, void* entropy, void* lse, int top, void* top_logprobs,
                    int* top_tokens) {
    // as many CTAs a row as fill the machine, none with less than one batch of packets for its threads
    const long long packets = z.cols / Packet<T>::N;
    int cluster = 1;
    while (cluster < kMaxCluster && z.rows * cluster < kSms * 8 && packets >= 2ll * cluster * kBatch * kThreads) cluster *= 2;
    if (cluster > 8) {
        static std::atomic<unsigned long long> allowed(0);      // by device
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e == cudaSuccess && !(allowed.load() >> (device & 63) & 1)) {
            e = cudaFuncSetAttribute(logprobs_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e == cudaSuccess) allowed.fetch_or(1ull << (device & 63));
        }
        if (e != cudaSuccess) return e;
    }
    const long long clusters = std::min<long long>(z.rows, (1ll << 30) / cluster);
    return launch(logprobs_kernel<T>, dim3((unsigned)(clusters * cluster)), kThreads, 0, s, cluster, (const T*)z.data, (long long)z.stride,
                  (long long)z.rows, (int)z.cols, tokens, (float*)logprob, (float*)entropy, (float*)lse, top, (float*)top_logprobs, top_tokens,
                  cluster);
}

template <>
cudaError_t forward<double>(cudaStream_t s, const Rows& z, const int* tokens, void* logprob, void* entropy, void* lse, int top,
                            void* top_logprobs, int* top_tokens) {
    return launch(logprobs_rows_kernel<double>, dim3((unsigned)capped(z.rows, kSms * 64)), kThreads, 0, s, 1, (const double*)z.data,
                  (long long)z.stride, (long long)z.rows, (int)z.cols, tokens, (double*)logprob, (double*)entropy, (double*)lse, top,
                  (double*)top_logprobs, top_tokens);
}

template <typename T>
cudaError_t backward(cudaStream_t s, const Rows& z, const int* tokens, const void* lse, const void* entropy, const void* dlogprob,
                     const void* dentropy, const Rows& dz) {
    typedef typename AccOf<T>::type A;
    const bool alike = ((uintptr_t)z.data - (uintptr_t)dz.data) % 16 == 0 && (z.rows < 2 || (z.stride - dz.stride) * z.size % 16 == 0);
    if constexpr (sizeof(T) < 8) {
        if (alike) {
            const long long packets = z.cols / Packet<T>::N, per_row = std::max<long long>(1, (packets + kBatch * kThreads - 1) / (kBatch * kThreads));
            const long long pieces = z.rows * per_row;
            return launch(dentropy ? logprobs_backward_kernel<T, true> : logprobs_backward_kernel<T, false>, dim3((unsigned)capped(pieces, 1 << 30)),
                          kThreads, 0, s, 1, (const T*)z.data, (long long)z.stride, pieces, (int)per_row, (int)z.cols, tokens, (const float*)lse,
                          (const float*)entropy, (const float*)dlogprob, (const float*)dentropy, (T*)dz.data, (long long)dz.stride);
        }
    }
    return launch(logprobs_backward_rows_kernel<T>, dim3((unsigned)capped(z.rows, kSms * 64)), kThreads, 0, s, 1, (const T*)z.data,
                  (long long)z.stride, (long long)z.rows, (int)z.cols, tokens, (const A*)lse, (const A*)entropy, (const A*)dlogprob,
                  (const A*)dentropy, (T*)dz.data, (long long)dz.stride);
}

std::string wrong_vector(const char* name, const void* p, int size) {
    if (p && (uintptr_t)p % size) return std::string(name) + " is not aligned to its elements";
    return "";
}

}  // namespace
}  // namespace dalib

using namespace dalib;

extern "C" int dalib200_token_logprobs(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits,
                                       int64_t row_stride, const int32_t* tokens, void* logprob, void* entropy, void* lse, int top,
                                       void* top_logprobs, int32_t* top_tokens) {
    return guarded("dalib200_token_logprobs", [&]() -> int {
        const std::string what = "dalib200_token_logprobs: ";
        if (!floating(dtype)) return refuse(what + "dtype must be f32, f64 or bf16");
        if (rows < 0 || vocab < 1) return refuse(what + "rows must be >= 0 and vocab >= 1");
        if (vocab > INT32_MAX) return refuse(what + "tokens are int32: the vocabulary has to end below 2^31");
        if (top < 0 || top > kMaxTop || top > vocab) return refuse(what + "top must lie between 0 and " + std::to_string(kMaxTop) + " and not exceed vocab");
        if (top > 0 && rows > 0 && (!top_logprobs || !top_tokens)) return refuse(what + "top alternatives need top_logprobs and top_tokens");
        if (rows == 0) return OnDevice(device).status;
        if (!logprob && !entropy && !lse && top == 0) return refuse(what + "no result is asked for");
        if (logprob && !tokens) return refuse(what + "logprob needs tokens");
        const Rows z = {"logits", logits, rows, vocab, row_stride, size_of(dtype)};
        std::string w = wrong(z);
        const int acc = dtype == DALIB200_F64 ? 8 : 4;
        const struct { const char* name; void* p; size_t bytes; int size; } outs[] = {
            {"logprob", logprob, (size_t)rows * acc, acc}, {"entropy", entropy, (size_t)rows * acc, acc}, {"lse", lse, (size_t)rows * acc, acc},
            {"top_logprobs", top ? top_logprobs : nullptr, (size_t)rows * top * acc, acc}, {"top_tokens", top ? top_tokens : nullptr, (size_t)rows * top * 4, 4}};
        for (const auto& o : outs) {
            if (w.empty()) w = wrong_vector(o.name, o.p, o.size);
            if (w.empty() && meets(o.p, o.bytes, logits, (size_t)(z.end() - z.begin()))) w = std::string(o.name) + " overlaps logits";
            if (w.empty() && logprob && meets(o.p, o.bytes, tokens, (size_t)rows * 4)) w = std::string(o.name) + " overlaps tokens";
            for (const auto& other : outs)
                if (w.empty() && &other < &o && meets(o.p, o.bytes, other.p, other.bytes)) w = std::string(o.name) + " overlaps " + other.name;
        }
        if (w.empty() && logprob) w = wrong_vector("tokens", tokens, 4);
        if (!w.empty()) return refuse(what + w);
        OnDevice on(device);
        if (on.status != DALIB200_OK) return on.status;
        cudaStream_t s = (cudaStream_t)stream;
        cudaError_t e;
        if (dtype == DALIB200_F32) e = forward<float>(s, z, tokens, logprob, entropy, lse, top, top_logprobs, top_tokens);
        else if (dtype == DALIB200_F64) e = forward<double>(s, z, tokens, logprob, entropy, lse, top, top_logprobs, top_tokens);
        else e = forward<bf16_s>(s, z, tokens, logprob, entropy, lse, top, top_logprobs, top_tokens);
        return launched("dalib200_token_logprobs", e);
    });
}

extern "C" int dalib200_token_logprobs_backward(int device, void* stream, int dtype, int64_t rows, int64_t vocab, const void* logits,
                                                int64_t row_stride, const int32_t* tokens, const void* lse, const void* entropy,
                                                const void* dlogprob, const void* dentropy, void* dlogits, int64_t dlogits_row_stride) {
    return guarded("dalib200_token_logprobs_backward", [&]() -> int {
        const std::string what = "dalib200_token_logprobs_backward: ";
        if (!floating(dtype)) return refuse(what + "dtype must be f32, f64 or bf16");
        if (rows < 0 || vocab < 1) return refuse(what + "rows must be >= 0 and vocab >= 1");
        if (vocab > INT32_MAX) return refuse(what + "tokens are int32: the vocabulary has to end below 2^31");
        if (rows == 0) return OnDevice(device).status;
        if (!lse) return refuse(what + "lse is a null pointer");
        if (!dlogprob && !dentropy) return refuse(what + "neither dlogprob nor dentropy is given");
        if (dlogprob && !tokens) return refuse(what + "dlogprob needs tokens");
        if (dentropy && !entropy) return refuse(what + "dentropy needs entropy");
        const int acc = dtype == DALIB200_F64 ? 8 : 4;
        const Rows z = {"logits", logits, rows, vocab, row_stride, size_of(dtype)};
        const Rows dz = {"dlogits", dlogits, rows, vocab, dlogits_row_stride, size_of(dtype)};
        std::string w = wrong(z);
        if (w.empty()) w = wrong(dz);
        if (w.empty() && clash(z, dz)) w = "dlogits overlaps logits without being logits";
        const struct { const char* name; const void* p; int size; } ins[] = {{"tokens", dlogprob ? tokens : nullptr, 4}, {"lse", lse, acc},
            {"entropy", dentropy ? entropy : nullptr, acc}, {"dlogprob", dlogprob, acc}, {"dentropy", dentropy, acc}};
        for (const auto& i : ins) {
            if (w.empty()) w = wrong_vector(i.name, i.p, i.size);
            if (w.empty() && meets(i.p, (size_t)rows * i.size, dlogits, (size_t)(dz.end() - dz.begin()))) w = std::string("dlogits overlaps ") + i.name;
        }
        if (!w.empty()) return refuse(what + w);
        OnDevice on(device);
        if (on.status != DALIB200_OK) return on.status;
        cudaStream_t s = (cudaStream_t)stream;
        cudaError_t e;
        if (dtype == DALIB200_F32) e = backward<float>(s, z, tokens, lse, entropy, dlogprob, dentropy, dz);
        else if (dtype == DALIB200_F64) e = backward<double>(s, z, tokens, lse, entropy, dlogprob, dentropy, dz);
        else e = backward<bf16_s>(s, z, tokens, lse, entropy, dlogprob, dentropy, dz);
        return launched("dalib200_token_logprobs_backward", e);
    });
}
