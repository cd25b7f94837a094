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
// Index of an entry where a loop steps past the row's end: vocab + kThreads may exceed 2^31 - 1, 2^32 - 1 it does not.
typedef uint32_t Place;

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

// A row's normaliser, the largest entry and the logarithm of the sum apart: log p = (z - m) - log s does not depend on what all
// entries have in common, while m + log s rounded to fp32 (the lse that is written) is off by 2^-24 of it.  (64 x 50000 f32 logits around
// 1e4: largest error 9.1e-7; z - lse 4.8e-4.)
template <typename A>
struct Normaliser {
    A m, log_s, lse;
    __device__ __forceinline__ A log_p(A z) const { return lse == -infinity_of(A()) ? lse : (z - m) - log_s; }
};
// from the row's sums; u in the units of a difference z - m times `unit`
template <typename A, typename R>
__device__ __forceinline__ Normaliser<A> finish_row(const R& all, A unit, A* entropy) {
    if (all.s == 0) {              // nothing but -infinity
        *entropy = 0;
        return {all.m, 0, -infinity_of(A())};
    }
    const A log_s = log_of(all.s);
    *entropy = log_s - unit * (all.u / all.s);
    return {all.m, log_s, all.m + log_s};
}

// ---------------------------------------------------------------------------------------------- f64 rows
// A CTA per row, one entry a thread and step; the alternatives one after another, each by another walk over the row.
// 8 CTAs an SM, 32 registers a thread: with one more, 1000 x 50001 with 5 alternatives no longer runs in one wave (844 -> 1060 us).
template <typename T>
__global__ void __launch_bounds__(kThreads, 8) logprobs_rows_kernel(const T* __restrict__ logits, long long ld, long long rows, int vocab,
                                                                 const int* __restrict__ tokens, typename AccOf<T>::type* logprob,
                                                                 typename AccOf<T>::type* entropy, typename AccOf<T>::type* lse_out,
                                                                 int top, typename AccOf<T>::type* top_logprobs, int* top_tokens) {
    typedef typename AccOf<T>::type A;
    __shared__ Running<A> sm[kThreads / 32];
    __shared__ Ranked<A> best[kThreads / 32];
    __shared__ Normaliser<A> norm;          // of the first thread; in registers it would cost every thread some
    dependent_prologue();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* z = logits + row * ld;
        Running<A> r;
        r.clear();
        for (Place j = threadIdx.x; j < (Place)vocab; j += kThreads) r.take(widen(z[j]));
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
        if (threadIdx.x == 0) {
            A h;
            norm = finish_row(all, (A)1, &h);
            if (entropy) entropy[row] = h;
            if (lse_out) lse_out[row] = norm.lse;
            if (logprob) {
                const int t = tokens[row];
                logprob[row] = t < 0 ? (A)0 : t >= vocab ? nan_of(A()) : norm.log_p(widen(z[t]));
            }
        }
        Ranked<A> last;
        for (int k = 0; k < top; ++k) {
            Ranked<A> b = {0, 0xffffffffu};
            for (Place j = threadIdx.x; j < (Place)vocab; j += kThreads) {
                const Ranked<A> c = {ordered(widen(z[j])), j};
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
                top_logprobs[row * top + k] = norm.log_p(widen(z[last.index]));
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- f32 and bf16 rows
// A team of one warp (short rows), of the CTA's eight, or of a cluster of CTAs shares a row, each CTA a contiguous slice of its
// 16-byte packets; a thread takes every TEAM-th packet of its slice, kBatch of them at a time, and keeps (m, s, u) in units of log 2:
// t = (z - m) log2 e, s = sum 2^t, u = sum t 2^t.  (z - m is formed before it is scaled: a row of the type's lowest value is uniform,
// not -infinity.)
//
// The alternatives cost no work in that pass.  A thread remembers its largest entry; the largest of a few neighbouring threads is
// their GROUP's.  At least `top` entries are >= the top-th largest group maximum tau, and every entry >= tau is one of a thread whose own
// maximum is >= tau: only those threads' entries, hardly more than `top` threads', are read again (from L2), and what is >= tau
// among them, hardly more than `top` entries, goes to a pool and is put in order by counting for each how many are larger.
// Where many entries equal tau the pool overflows: then tau is told apart by index too (a larger value, or the same
// at a lower index; no two entries are the same), for which every thread looks its maximum's place up.  Should even so the
// pool be too small (all of a few threads' entries larger than every other's), entries are sorted 32 at a time and merged.
//
// What bounds it, beside the 6570 GB/s of a copy: memory for f32 rows (4096 x 32768 85 us, 96%); for bf16 rows, with twice the entries a
// byte, the exponential of each (that unit is busy 65% of the time, 70% of the issue slots are taken) and, in a long run, the clock that
// is left under the power limit (8192 x 65536 177 us alone, 92%; 211 us one call after the other, at 1.7 GHz).  20 alternatives
// of each of those rows add 80 us, and 5 of 1000 x 50001 f32 13 us: the row's threads wait for one another several times while no row
// is read.
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
    // the team's: raised to the largest m first, so that sums are left to add; over LANES neighbouring lanes
    template <int LANES>
    __device__ __forceinline__ void over_lanes() {
        float high = m;
#pragma unroll
        for (int k = LANES / 2; k > 0; k >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, k));
        raise(high);
#pragma unroll
        for (int k = LANES / 2; k > 0; k >>= 1) {
            s += __shfl_xor_sync(0xffffffffu, s, k);
            u += __shfl_xor_sync(0xffffffffu, u, k);
        }
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
// the threads of a team meet
template <int WR>
__device__ __forceinline__ void team_barrier() {
    if (WR == 1) __syncwarp();
    else __syncthreads();
}
// The 32 largest keys of `n` (a power of two <= 2 * WR) descending lists in shared memory, left in list 0.
template <int WR>
__device__ __forceinline__ void join_lists(Key (*lists)[32], int n) {
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % WR;
    team_barrier<WR>();
    for (int half = n >> 1; half > 0; half >>= 1) {
        if (warp < half) lists[warp][lane] = join(lists[warp][lane], lists[warp + half], lane);
        team_barrier<WR>();
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

// the e-th entry of a packet
template <typename T>
__device__ __forceinline__ float entry(uint4 q, int e) {
    const int w = sizeof(T) == 4 ? e : e >> 1;
    const uint32_t word = w & 2 ? (w & 1 ? q.w : q.z) : (w & 1 ? q.y : q.x);
    return __uint_as_float(sizeof(T) == 4 ? word : e & 1 ? word & 0xffff0000u : word << 16);
}
// one bit for each entry of a packet that is >= z
template <typename T>
__device__ __forceinline__ uint32_t reaching(uint4 q, float z) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            if (__uint_as_float(w[i]) >= z) bits |= 1u << i;
        } else {
            if (__uint_as_float(w[i] << 16) >= z) bits |= 1u << 2 * i;
            if (__uint_as_float(w[i] & 0xffff0000u) >= z) bits |= 2u << 2 * i;
        }
    }
    return bits;
}

// `count` distinct keys in shared memory (a zero behind an odd count) -> the 32 largest in descending order in sorted[] (which held
// zeros).  SPLIT neighbouring threads count for one key.
template <int TEAM, int SPLIT>
__device__ __forceinline__ void order_by(const Key* keys, int count, Key* sorted) {
    const int t = threadIdx.x % TEAM, part = t % SPLIT;
    for (int i0 = 0; i0 < count; i0 += TEAM / SPLIT) {
        const int i = i0 + t / SPLIT;
        const Key mine = i < count ? keys[i] : 0;
        int larger = 0;
#pragma unroll 4
        for (int j = 2 * part; j < count; j += 2 * SPLIT) {
            const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(keys + j);
            larger += (o.x > mine) + (o.y > mine);
        }
#pragma unroll
        for (int m = 1; m < SPLIT; m <<= 1) larger += __shfl_xor_sync(0xffffffffu, larger, m);
        if (part == 0 && mine != 0 && larger < 32) sorted[larger] = mine;
    }
}
template <int TEAM>
__device__ __forceinline__ void order(const Key* keys, int count, Key* sorted) {
    if (TEAM > 32 && count <= TEAM / 8) order_by<TEAM, 8>(keys, count, sorted);
    else if (TEAM > 32 && count <= TEAM / 4) order_by<TEAM, 4>(keys, count, sorted);
    else order_by<TEAM, TEAM == 32 ? 1 : 2>(keys, count, sorted);
}

template <int WR>
struct alignas(16) Picking {
    // of 64 groups the 32nd largest leaves 64 log 2 = 44 entries above it, of 32 the last one about 32 (1 + 1/2 + ... + 1/32) = 130
    static constexpr int GROUPS = WR == 1 ? 32 : 64, MEMBERS = 32 * WR / GROUPS, POOL = WR == 1 ? 256 : 128;
    Key groups[WR == 1 ? 2 : GROUPS], sorted[WR == 1 ? 2 : 32], pool[POOL + 2];
    int in_pool;
};

// The `top` largest entries of the team's packets [begin, end) (and, in the first CTA, of the row's edges) as a descending list in
// lists[0], zeros behind them if there are fewer.  seen: the thread's largest entry among its packets; best_batch: the batch of its
// packets that holds it, -1 if there is nothing but -infinity and NaN.
template <typename T, int WR>
__device__ __forceinline__ void top_of_slice(const RowSplit<T>& row, int begin, int end, bool edges, int top, float seen, int best_batch,
                                             Key (*lists)[32], Picking<WR>& pick, Key* pending) {
    constexpr int N = Packet<T>::N, TEAM = 32 * WR, MEMBERS = Picking<WR>::MEMBERS;
    const int t = threadIdx.x % TEAM, lane = t & 31, warp = t >> 5;
    const int n_edges = edges ? row.head + row.tail : 0;
    const bool has_edge = t < n_edges;
    const float edge = has_edge ? widen(row.z[row.edge(t)]) : 0.0f;
    auto packet_at = [&](int p) { return p < end ? row.packet(p) : packet_of_minus_infinity<T>(); };
    auto entry_key = [&](uint4 q, int p, int e) { return key_of(entry<T>(q, e), row.first_of(p) + e); };
    enum { BY_VALUE, BY_PLACE, SORTED };
#pragma unroll 1
    for (int attempt = BY_VALUE;; ++attempt) {
        // the thread's largest key (BY_VALUE: told apart by thread, and below any real key of its value)
        Key mine = 0;
        if (attempt == BY_VALUE) {
            if (begin + t < end) mine = (Key)ordered(seen) << 32;
            if (has_edge) mine = max(mine, (Key)ordered(edge) << 32);
            if (mine) mine |= (uint32_t)(kThreads - t);
        } else {
            const int from = best_batch >= 0 ? best_batch : begin + t, until = best_batch >= 0 ? min(end, best_batch + kBatch * TEAM) : end;
#pragma unroll 1
            for (int p = from; p < until; p += TEAM) {
                const uint4 q = row.packet(p);
#pragma unroll 1
                for (int e = 0; e < N; ++e) mine = max(mine, entry_key(q, p, e));
            }
            if (has_edge) mine = max(mine, key_of(edge, row.edge(t)));
        }
        Key group = mine;
#pragma unroll
        for (int m = 1; m < MEMBERS; m <<= 1) group = max(group, exchange(group, m));
        if (t == 0) pick.in_pool = 0;
        Key tau;
        if constexpr (WR == 1) {
            tau = __shfl_sync(0xffffffffu, sort_down(group, lane), top - 1);
            __syncwarp();
        } else {
            if (t % MEMBERS == 0) pick.groups[t / MEMBERS] = group;
            if (t < 32) {
                pick.sorted[t] = 0;
                lists[0][t] = 0;
            }
            team_barrier<WR>();
            order<TEAM>(pick.groups, Picking<WR>::GROUPS, pick.sorted);
            team_barrier<WR>();
            tau = pick.sorted[top - 1];
        }
        if (attempt == BY_VALUE) tau = tau >> 32 << 32;
        tau = max(tau, (Key)1);
        // (where tau is a NaN's or nobody's, every entry needs a closer look than its value)
        const bool all_pass = (tau >> 32) == 0;
        const uint32_t tau_bits = (uint32_t)(tau >> 32);
        const float tau_value = __uint_as_float(tau_bits & 0x80000000u ? tau_bits & 0x7fffffffu : ~tau_bits);

        Key best = 0;          // SORTED: the warp's list
        int waiting = 0;
        auto flush = [&](Key k) {
            const Key k32 = sort_down(k, lane), other = __shfl_sync(0xffffffffu, k32, 31 - lane);
            best = merge_down(best > other ? best : other, lane);
        };
        // one key a lane (0: none): those >= tau to the pool, or to the warp's list
        auto offer = [&](Key k) {
            const bool passes = k >= tau;
            const uint32_t who = __ballot_sync(0xffffffffu, passes);
            if (who == 0) return;
            const int before = __popc(who & ((1u << lane) - 1));
            if (attempt != SORTED) {
                int at = 0;
                if (lane == 0) at = atomicAdd(&pick.in_pool, __popc(who));
                at = __shfl_sync(0xffffffffu, at, 0) + before;
                if (passes && at < Picking<WR>::POOL) pick.pool[at] = k;
                return;
            }
            if (passes) pending[waiting + before] = k;
            waiting += __popc(who);
            __syncwarp();
            if (waiting >= 32) {
                const Key first = pending[lane], rest = pending[32 + lane];
                __syncwarp();
                pending[lane] = rest;
                flush(first);
                waiting -= 32;
                __syncwarp();
            }
        };
        // each lane its own packets, or all lanes one holder's after the other's, kBatch of them under way at a time
        const uint32_t holders = __ballot_sync(0xffffffffu, mine >= tau);
        const int per = (end - begin + TEAM - 1) / TEAM;          // packets of a thread
        const bool own = per <= __popc(holders) * ((per + 31) / 32);
        const int stride = own ? TEAM : 32 * TEAM;
        uint32_t left = own ? (per > 0 ? 1u : 0u) : holders;      // what is still to be read: threads (own: all at once)
        int first = own ? begin + warp * 32 : begin + warp * 32 + __ffs(left) - 1;          // lane 0's packet
        if (first >= end) left = 0;
#pragma unroll 1
        while (left) {
            uint4 q[kBatch];
            int at[kBatch];
            uint32_t bits = 0;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                at[i] = left ? first + (own ? lane : lane * TEAM) : end;
                q[i] = packet_at(at[i]);
                first += stride;
                if (left && first >= end) {
                    left &= left - 1;
                    first = begin + warp * 32 + __ffs(left) - 1;
                }
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (at[i] < end) bits |= (all_pass ? (1u << N) - 1 : reaching<T>(q[i], tau_value)) << N * i;
#pragma unroll 1
            while (__any_sync(0xffffffffu, bits)) {
                const int bit = __ffs(bits) - 1, i = bit / N, e = bit % N;
                const uint4 w = i & 2 ? (i & 1 ? q[3] : q[2]) : (i & 1 ? q[1] : q[0]);
                const int p = i & 2 ? (i & 1 ? at[3] : at[2]) : (i & 1 ? at[1] : at[0]);
                offer(bits ? entry_key(w, p, e) : 0);
                bits &= bits - 1;
            }
        }
        if (n_edges > 0 && warp == 0) offer(has_edge ? key_of(edge, row.edge(t)) : 0);
        if (attempt == SORTED) {
            flush(lane < waiting ? pending[lane] : 0);
            lists[warp][lane] = best;
            join_lists<WR>(lists, WR);
            return;
        }
        team_barrier<WR>();
        const int count = pick.in_pool;
        if (count <= Picking<WR>::POOL && (count >= top || attempt == BY_PLACE)) {
            if constexpr (WR == 1) {          // (a warp sorts and merges faster than it counts)
                for (int i = 0; i < count; i += 32) flush(i + lane < count ? pick.pool[i + lane] : 0);
                lists[0][lane] = best;
                __syncwarp();
                return;
            }
            if (t == 0 && (count & 1)) pick.pool[count] = 0;
            team_barrier<WR>();
            order<TEAM>(pick.pool, count, lists[0]);
            team_barrier<WR>();
            return;
        }
        team_barrier<WR>();          // everybody has read in_pool
    }
}

template <typename T, int WR, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) logprobs_kernel(const T* __restrict__ logits, long long ld, long long rows, int vocab,
                                                            const int* __restrict__ tokens, float* __restrict__ logprob,
                                                            float* __restrict__ entropy, float* __restrict__ lse_out, int top_asked,
                                                            float* __restrict__ top_logprobs, int* __restrict__ top_tokens, int cluster) {
    const int top = TOP ? top_asked : 0;
    constexpr int N = Packet<T>::N, TEAM = 32 * WR, TEAMS = kThreads / TEAM;
    __shared__ Running2 sm[kWarps];
    __shared__ Running2 from_cta[WR == 1 ? 1 : kMaxCluster];
    __shared__ Key all_lists[WR == 1 ? kWarps : kMaxCluster][32];
    __shared__ Key pending[TOP ? kWarps : 1][64];
    __shared__ Key from_cta_keys[WR == 1 ? 1 : kMaxCluster][32];
    __shared__ Picking<WR> picking[TOP ? TEAMS : 1];
    const int team = threadIdx.x / TEAM, t = threadIdx.x % TEAM, lane = t & 31, warp = t >> 5;
    Key(*lists)[32] = all_lists + team * WR;
    const int rank = cluster > 1 ? (int)cluster_rank() : 0;
    if (cluster > 1) cluster_arrive();          // every CTA of the cluster runs before its shared memory is written from another
    dependent_prologue();
    bool started = cluster == 1;
    const long long step = (long long)(gridDim.x / cluster) * TEAMS;
    for (long long r = (long long)(blockIdx.x / cluster) * TEAMS + team; r < rows; r += step) {
        const RowSplit<T> row(logits + r * ld, vocab);
        const int share = (row.packets + cluster - 1) / cluster;
        const int begin = min(row.packets, rank * share), end = min(row.packets, begin + share);
        Running2 me = {Lowest<float>::value(), 0, 0};
        float seen = -infinity_of(0.0f);
        int best_batch = -1;
        {
            Two s2 = two(0, 0), u2 = two(0, 0);
            auto raise = [&](float to) {
                me.s = total(s2);
                me.u = total(u2);
                me.raise(to);
                s2 = two(me.s, 0);
                u2 = two(me.u, 0);
            };
            uint4 ahead[kBatch];          // the next batch is on its way while one is worked on
#pragma unroll
            for (int i = 0; i < kBatch; ++i) ahead[i] = begin + t + i * TEAM < end ? row.packet(begin + t + i * TEAM) : packet_of_minus_infinity<T>();
            for (int b = begin + t; b < end; b += kBatch * TEAM) {
                uint4 q[kBatch];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    q[i] = ahead[i];
                    const int p = b + (kBatch + i) * TEAM;
                    ahead[i] = p < end ? row.packet(p) : packet_of_minus_infinity<T>();
                }
                const float high = largest(q, (T*)nullptr);
                if (high > seen) {
                    seen = high;
                    best_batch = b;
                    if (high > me.m) raise(high);
                }
                const Two minus = both(-me.m), scale = both(kLog2e);
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
            if (rank == 0 && t < row.head + row.tail) {
                const float z = widen(row.z[row.edge(t)]);
                if (z > me.m) raise(z);
                const float d = max_nan((z - me.m) * kLog2e, kFloor), p = exp2_of(d);
                s2 = s2 + two(p, 0);
                u2 = u2 + two(d * p, 0);
            }
            me.s = total(s2);
            me.u = total(u2);
        }
        me.over_lanes<32>();
        if (WR > 1) {
            __syncthreads();          // the row before has been written
            if (lane == 0) sm[warp] = me;
        }
        if constexpr (TOP) top_of_slice<T, WR>(row, begin, end, rank == 0, top, seen, best_batch, lists, picking[team], pending[threadIdx.x >> 5]);
        else if (WR > 1) __syncthreads();
        if (WR > 1 && cluster > 1) {
            if (!started) { cluster_wait(); started = true; }
            if (warp == 0) {
                me = sm[lane % kWarps];
                me.over_lanes<kWarps>();
                if (lane == 0) {
                    store_remote(in_first_cta(&from_cta[rank].m), me.m);
                    store_remote(in_first_cta(&from_cta[rank].s), me.s);
                    store_remote(in_first_cta(&from_cta[rank].u), me.u);
                }
                if (top > 0) store_remote(in_first_cta(&from_cta_keys[rank][lane]), lists[0][lane]);
            }
            cluster_arrive();
            cluster_wait();
            if (rank == 0 && top > 0) {
                for (int w = warp; w < cluster; w += kWarps) lists[w][lane] = from_cta_keys[w][lane];
                join_lists<WR>(lists, cluster);
            }
        }
        if (rank == 0 && warp == 0) {
            if (WR > 1 && cluster > 1) {
                me = from_cta[lane % cluster];          // (every CTA's sums 32 / cluster times)
                me.over_lanes<32>();
                me.s *= cluster * (1.0f / 32);
                me.u *= cluster * (1.0f / 32);
            } else if (WR > 1) {
                me = sm[lane % kWarps];
                me.over_lanes<kWarps>();
            }
            float h;
            const Normaliser<float> norm = finish_row(me, kLn2, &h);
            if (lane == 0) {
                if (entropy) entropy[r] = h;
                if (lse_out) lse_out[r] = norm.lse;
                if (logprob) {
                    const int given = tokens[r];
                    logprob[r] = given < 0 ? 0.0f : given >= vocab ? nan_of(0.0f) : norm.log_p(widen(row.z[given]));
                }
            }
            if (lane < top) {
                const int index = index_of(lists[0][lane]);
                top_tokens[r * top + lane] = index;
                top_logprobs[r * top + lane] = norm.log_p(widen(row.z[index]));
            }
        }
        if (WR > 1 && cluster > 1) {           // the first CTA has read what the others sent for this row
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
        for (Place j = threadIdx.x; j < (Place)vocab; j += kThreads) {
            A d = 0;
            if (!nothing) {
                const A lp = max_nan((A)widen(z[j]) - l, floor_of_difference<A>());
                const A p = exp_of(lp);
                d = -p * (g + w * (lp + h));
                if ((int)j == t) d += g;
            }
            out[j] = Narrow<T>::of(d);
        }
    }
}

// Everything else streams: a CTA (a warp, where rows are short) takes kBatch packets a thread of one row, all loaded before the first
// is worked on, and p is exp2 of t = (z - lse) log2 e.  With dentropy:  dz = -p (g + w (log p + H)) = -p (a + b t),  a = g + w H,
// b = w / log2 e.  Bound by memory: 8192 x 65536 bf16 322 us, the rate of a copy (with dentropy 336); 373 when a row's numbers
// were read with its packets and the stores went through the caches.
template <typename T, int WR, bool ENTROPY>
__global__ void __launch_bounds__(kThreads) logprobs_backward_kernel(const T* logits, long long ld, long long pieces, int per_row, int vocab,
                                                                     const int* __restrict__ tokens, const float* __restrict__ lse,
                                                                     const float* __restrict__ entropy, const float* __restrict__ dlogprob,
                                                                     const float* __restrict__ dentropy, T* dlogits, long long ldd) {
    constexpr int N = Packet<T>::N, TEAM = 32 * WR, TEAMS = kThreads / TEAM;
    const int me = threadIdx.x % TEAM;
    const long long mine = (long long)blockIdx.x * TEAMS + threadIdx.x / TEAM, step = (long long)gridDim.x * TEAMS;
    dependent_prologue();
    // what a row's entries need, read a piece ahead: the packets can be asked for at once
    struct Row { int t; float g, l, w, h; };
    auto row_of = [&](long long piece) {
        const long long r = piece / per_row;
        Row v;
        v.t = dlogprob ? tokens[r] : -1;
        v.g = dlogprob ? dlogprob[r] : 0.0f;
        v.l = lse[r];
        v.w = ENTROPY ? dentropy[r] : 0.0f;
        v.h = ENTROPY ? entropy[r] : 0.0f;
        return v;
    };
    Row next = {};
    if (mine < pieces) next = row_of(mine);
    for (long long piece = mine; piece < pieces; piece += step) {
        const long long r = piece / per_row;
        const int part = (int)(piece - r * per_row);
        const RowSplit<T> row(logits + r * ld, vocab);
        T* out = dlogits + r * ldd;
        const int t = next.t;
        const float g = t < 0 ? 0.0f : t >= vocab ? nan_of(0.0f) : next.g, l = next.l, w = next.w, h = next.h;
        if (piece + step < pieces) next = row_of(piece + step);
        const bool nothing = (g == 0 && w == 0) || l == -infinity_of(0.0f);
        const float a = -(g + w * h), b = -w * kLn2;
        const int begin = part * kBatch * TEAM + me;
        if (nothing) {          // 0 whatever the logits hold: they are not read
#pragma unroll
            for (int i = 0; i < kBatch; ++i)
                if (begin + i * TEAM < row.packets) *reinterpret_cast<uint4*>(out + row.first_of(begin + i * TEAM)) = make_uint4(0, 0, 0, 0);
            if (part == 0 && me < row.head + row.tail) out[row.edge(me)] = Narrow<T>::of(0.0f);
            continue;
        }
        uint4 q[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (begin + i * TEAM < row.packets) q[i] = row.packet(begin + i * TEAM);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int p = begin + i * TEAM;
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
            __stcs(reinterpret_cast<uint4*>(out + row.first_of(p)), packet_of(z, (const T*)nullptr));
        }
        if (part == 0 && me < row.head + row.tail) {
            const int j = row.edge(me);
            const float t0 = max_nan((widen(row.z[j]) - l) * kLog2e, kFloor);
            out[j] = Narrow<T>::of(exp2_of(t0) * (t0 * b + a) + (j == t ? g : 0.0f));
        }
    }
}

long long capped(long long want, long long most) { return std::max<long long>(1, std::min(want, most)); }

template <typename T>
cudaError_t forward(cudaStream_t s, const Rows& z, const int* tokens, void* logprob, void* entropy, void* lse, int top, void* top_logprobs,
                    int* top_tokens) {
    // A warp per row where that is a few batches for it, or where there are rows for every warp of the machine (16384 x 8192 bf16: 49 us, a
    // CTA per row 89); else a CTA per row, and several for so few rows that two CTAs a SM are not reached with one (64 x 131072 bf16:
    // 9 us with eight, 20 with one; 1000 x 50001 f32: 35 us with one, 48 with two), none with less than one batch for its
    // threads.
    const long long packets = z.cols / Packet<T>::N;
    const bool warp_each = packets <= 32 * kBatch * 2 || (packets <= 32 * kBatch * 8 && z.rows >= kSms * 8);
    int cluster = 1;
    while (!warp_each && cluster < kMaxCluster && z.rows * cluster <= kSms * 2 && packets >= 2ll * cluster * kBatch * kThreads) cluster *= 2;
    auto kernel = warp_each ? (top ? logprobs_kernel<T, 1, true> : logprobs_kernel<T, 1, false>)
                            : (top ? logprobs_kernel<T, kWarps, true> : logprobs_kernel<T, kWarps, false>);
    if (cluster > 8) {
        static std::atomic<unsigned long long> allowed[2];      // by device
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e == cudaSuccess && !(allowed[top > 0].load() >> (device & 63) & 1)) {
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e == cudaSuccess) allowed[top > 0].fetch_or(1ull << (device & 63));
        }
        if (e != cudaSuccess) return e;
    }
    const int teams = warp_each ? kWarps : 1;
    const long long clusters = std::min<long long>((z.rows + teams - 1) / teams, (1ll << 30) / cluster);
    return launch(kernel, dim3((unsigned)(clusters * cluster)), kThreads, 0, s, cluster, (const T*)z.data, (long long)z.stride,
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
            const long long packets = z.cols / Packet<T>::N;
            const bool warp_each = packets <= 32 * kBatch * 4;          // (16384 x 1000 f32: 41 us with a CTA per row)
            const long long piece = kBatch * (warp_each ? 32 : kThreads), per_row = std::max<long long>(1, (packets + piece - 1) / piece);
            const long long pieces = z.rows * per_row;
            auto kernel = warp_each ? (dentropy ? logprobs_backward_kernel<T, 1, true> : logprobs_backward_kernel<T, 1, false>)
                                    : (dentropy ? logprobs_backward_kernel<T, kWarps, true> : logprobs_backward_kernel<T, kWarps, false>);
            return launch(kernel, dim3((unsigned)capped(warp_each ? (pieces + kWarps - 1) / kWarps : pieces, kSms * 8)),
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
