// Layer normalisation along rows and its gradient: dalib200_layer_norm, dalib200_layer_norm_backward.
//
//   mean = sum x / n,  var = sum (x - mean)^2 / n,  r = 1 / sqrt(var + eps),  h = (x - mean) r
//   y = h gamma + beta
//   a = dy gamma
//   dx = r (a - mean(a) - h mean(a h)),  dgamma = sum over the rows of dy h,  dbeta = sum over the rows of dy
//
// The backward pass takes x and no saved statistics: it has to read x anyway, and mean and r of a row that is at hand cost
// no memory traffic.  Statistics and sums are held in fp32 (fp64 for fp64 rows).
#include <algorithm>
#include <atomic>

#include "op_device.cuh"
#include "op_host.h"

namespace dalib {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------------------------- rows of any length
// f64 rows, and rows that do not fit a CTA's registers.  A CTA walks a row W elements at a time, once for the mean, once for the squared
// deviations, and once to write it; behind the first walk the row comes from L2.  W is a packet's where the matrices lie alike on the
// 16-byte grid (the elements in front of it and behind it one by one), else 1.  1 x 17744 f32: 14.3 us with 256 threads and
// W = 1, 8.6 with 1024 and packets; 3000 x 32768 f32 gradient 819 and 576.  Not everywhere: 4000 x 20000 f32 takes 264 us
// (37% of a copy; its gradient 510) where 256 threads took 244, and the gradient of 3000 x 19999 bf16 388 where they took 373.
template <int N> struct Width { static constexpr int value = N; };
template <int W, typename F>
__device__ __forceinline__ void walk(long long cols, int head, F f) {          // f(Width, column)
    const long long packets = (cols - head) / W;
#pragma unroll 4
    for (long long p = threadIdx.x; p < packets; p += blockDim.x) f(Width<W>(), head + p * W);
    if (W > 1)
        for (int e = threadIdx.x; e < (int)(cols - packets * W); e += blockDim.x) f(Width<1>(), e < head ? e : e + packets * W);
}
template <int W, typename T>
__device__ __forceinline__ int head_of(const T* row, long long cols) {          // elements in front of the row's first packet
    return W == 1 ? 0 : (int)min((long long)((16 - (uintptr_t)row % 16) % 16 / sizeof(T)), cols);
}
template <int V, typename T, typename A>
__device__ __forceinline__ void read_cells(const T* from, A (&v)[V]) {
    if constexpr (V == 1) {
        v[0] = widen(*from);
    } else {
        const Packet<T> q = load_packet(from);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = widen(q.v[e]);
    }
}
template <int V, typename T, typename A>
__device__ __forceinline__ void write_cells(T* to, const A (&v)[V]) {
    if constexpr (V == 1) {
        *to = Narrow<T>::of(v[0]);
    } else {
        Packet<T> q;
#pragma unroll
        for (int e = 0; e < V; ++e) q.v[e] = Narrow<T>::of(v[e]);
        store_packet(to, q);
    }
}

template <typename T, typename P, int W>
__global__ void __launch_bounds__(1024) norm_rows_kernel(const T* x, long long ldx, const P* __restrict__ gamma, const P* __restrict__ beta,
                                                         T* y, long long ldy, long long rows, long long cols, double eps) {
    typedef typename AccOf<T>::type A;
    __shared__ A sm[32];
    dependent_prologue();
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* in = x + row * ldx;
        T* out = y + row * ldy;
        const int head = head_of<W>(in, cols);
        A s = 0;
        walk<W>(cols, head, [&](auto width, long long c) {
            A v[decltype(width)::value];
            read_cells(in + c, v);
            for (A e : v) s += e;
        });
        const A mean = block_sum(s, sm) / (A)cols;
        A q = 0;
        walk<W>(cols, head, [&](auto width, long long c) {
            A v[decltype(width)::value];
            read_cells(in + c, v);
            for (A e : v) q += (e - mean) * (e - mean);
        });
        const A r = (A)1 / root(block_sum(q, sm) / (A)cols + (A)eps);
        walk<W>(cols, head, [&](auto width, long long c) {
            constexpr int V = decltype(width)::value;
            A v[V];
            read_cells(in + c, v);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] = (v[e] - mean) * r;
                if (gamma) v[e] *= widen(gamma[c + e]);
                if (beta) v[e] += widen(beta[c + e]);
            }
            write_cells(out + c, v);
        });
    }
}

template <int V, typename A, typename P>
__device__ __forceinline__ void weigh_cells(A (&v)[V], const P* gamma, long long c) {
    if (gamma)
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] *= (A)widen(gamma[c + e]);
}
template <int W, typename T, typename P, typename A>
__device__ __forceinline__ void write_gradient(const T* up, const T* in, const P* gamma, T* out, long long cols, int head, A mean, A r, A mean_a,
                                               A k) {
    walk<W>(cols, head, [&](auto width, long long c) {
        constexpr int V = decltype(width)::value;
        A v[V], a[V];
        read_cells(in + c, v);
        read_cells(up + c, a);
        weigh_cells(a, gamma, c);
#pragma unroll
        for (int e = 0; e < V; ++e) a[e] = r * (a[e] - mean_a - (v[e] - mean) * k);
        write_cells(out + c, a);
    });
}

// Per row: mean, r, mean(a) and r^2 mean(a h / r), 4 values in `stats` where the columns are summed behind it, and dx where it is given: where the columns are summed from
// matrices that dx is written over, dx_kernel writes it behind that.
template <typename T, typename P, int W>
__global__ void __launch_bounds__(1024) row_stats_kernel(const T* dy, long long lddy, const T* x, long long ldx, const P* __restrict__ gamma, T* dx,
                                                         long long lddx, long long rows, long long cols, double eps,
                                                         typename AccOf<T>::type* __restrict__ stats) {
    typedef typename AccOf<T>::type A;
    __shared__ A sm[32];
    dependent_prologue();
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* in = x + row * ldx;
        const T* up = dy + row * lddy;
        const int head = head_of<W>(in, cols);
        A s = 0, sa = 0;
        walk<W>(cols, head, [&](auto width, long long c) {
            A v[decltype(width)::value], a[decltype(width)::value];
            read_cells(in + c, v);
            read_cells(up + c, a);
            weigh_cells(a, gamma, c);
            for (A e : v) s += e;
            for (A e : a) sa += e;
        });
        const A mean = block_sum(s, sm) / (A)cols;
        const A mean_a = block_sum(sa, sm) / (A)cols;
        A q = 0, qa = 0;
        walk<W>(cols, head, [&](auto width, long long c) {
            constexpr int V = decltype(width)::value;
            A v[V], a[V];
            read_cells(in + c, v);
            read_cells(up + c, a);
            weigh_cells(a, gamma, c);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] -= mean;
                q += v[e] * v[e];
                qa += v[e] * a[e];
            }
        });
        const A r = (A)1 / root(block_sum(q, sm) / (A)cols + (A)eps);
        const A k = r * (r * (block_sum(qa, sm) / (A)cols));
        if (threadIdx.x == 0 && stats) {
            stats[4 * row] = mean;
            stats[4 * row + 1] = r;
            stats[4 * row + 2] = mean_a;
            stats[4 * row + 3] = k;
        }
        if (dx) write_gradient<W>(up, in, gamma, dx + row * lddx, cols, head, mean, r, mean_a, k);
    }
}

// partial[slice][0 / 1][col] = sum over the slice's rows of dy h / of dy
template <typename T>
__global__ void __launch_bounds__(kThreads) column_sums_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x,
                                                               long long ldx, long long rows, long long cols,
                                                               const typename AccOf<T>::type* __restrict__ stats,
                                                               typename AccOf<T>::type* __restrict__ partial) {
    typedef typename AccOf<T>::type A;
    dependent_prologue();
    const long long c = (long long)blockIdx.x * kThreads + threadIdx.x;
    if (c >= cols) return;
    A g = 0, b = 0;
    for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
        const A up = widen(dy[row * lddy + c]);
        g += up * ((widen(x[row * ldx + c]) - stats[4 * row]) * stats[4 * row + 1]);
        b += up;
    }
    partial[(2 * (long long)blockIdx.y) * cols + c] = g;
    partial[(2 * (long long)blockIdx.y + 1) * cols + c] = b;
}

template <typename T, typename P, int W>
__global__ void __launch_bounds__(1024) dx_kernel(const T* dy, long long lddy, const T* x, long long ldx, const P* __restrict__ gamma, T* dx,
                                                  long long lddx, long long rows, long long cols,
                                                  const typename AccOf<T>::type* __restrict__ stats) {
    dependent_prologue();
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* in = x + row * ldx;
        write_gradient<W>(dy + row * lddy, in, gamma, dx + row * lddx, cols, head_of<W>(in, cols), stats[4 * row], stats[4 * row + 1],
                          stats[4 * row + 2], stats[4 * row + 3]);
    }
}

// dgamma / dbeta: the slices' sums in slice order.  A warp owns 32 columns of one of the two, its CTA's warps share the slices.
template <typename A, typename P>
__global__ void __launch_bounds__(kThreads) fold_columns_kernel(const A* __restrict__ partial, long long slices, long long cols,
                                                                P* __restrict__ dgamma, P* __restrict__ dbeta) {
    constexpr int W = kThreads / 32;
    __shared__ A sm[W][33];
    dependent_prologue();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    P* out = blockIdx.y ? dbeta : dgamma;
    if (!out) return;
    const long long c = (long long)blockIdx.x * 32 + lane;
    A v = 0;
    if (c < cols)
        for (long long s = warp; s < slices; s += W) v += partial[(2 * s + blockIdx.y) * cols + c];
    sm[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && c < cols) {
        v = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) v += sm[w][lane];
        out[c] = Narrow<P>::of(v);
    }
}

// ---------------------------------------------------------------------------------------------- rows held in registers
// f32 and bf16 rows that fit: some warps share a row, a thread keeps packets of it, so that every row is read once and written once.
// Statistics need one exchange between the warps: each warp takes its own mean first (shuffles), then
//   Q = sum (x - mean_w)^2,  A = sum a,  C = sum a (x - mean_w)
// about it, and the warps' values are moved to the row's mean as they are added:
//   sum (x - mean)^2 = sum_w Q_w + n_w (mean_w - mean)^2,   sum a (x - mean) = sum_w C_w + A_w (mean_w - mean).
// No squares of values far from zero are subtracted from one another, and the backward pass needs no more exchanges with
// recomputed statistics than it would with saved ones.
//
// What bounds them, beside the 6570 GB/s of a copy.  Forward: memory (16384 x 4096 bf16 with f32 weights 45 us, 91%; 4096 x 8192 f32
// 43 us, 95%), and for rows that end off the 16-byte grid the elements at their edges (33537 x 2001 bf16 58 us, 70%).  Backward, f32:
// memory (32768 x 1024 67 us, 91%).  Backward, bf16: no unit is full (45% of the issue slots taken, DRAM 57%); what is left open is the
// latency of a row's sums behind one another, with the 16 warps that 128 registers a thread leave an SM (16384 x 4096 83 to 88 us, 70 to
// 74%; 13104 x 5121 136 us, 45%).  There, more values a thread, rows read again from shared memory in place of registers (136 us) and fewer shuffles for the sums gained nothing.

// A thread holds C packets of W elements of a row, the row's WR warps side by side.  Packets come through a ring of DEPTH rows in
// shared memory that every thread fills and reads for itself (cp.async; no thread waits for another one's copies), so that the
// loads of the next rows are under way while a row is worked on.
// EDGE: rows that do not lie on the 16-byte grid.  Their packets do; the few elements in front of the first one and behind the last one
// are one more for each of the row's first threads.  A CTA's rows are a multiple of W apart, so that every thread holds the same
// columns of all of them.  (W = 1: matrices whose rows do not even lie alike on the grid.)
enum Rowfit { FULL, WHOLE, EDGE };          // every thread holds C packets; packets are there or not; EDGE
__host__ __device__ constexpr int lanes_of(int warps) {          // a lane for each of them: the power of two above
    int n = 1;
    while (n < warps) n *= 2;
    return n;
}
template <int W, int C, int WR, Rowfit FIT>
struct Held {
    uint32_t there;          // bit i: the thread's i-th packet is one of the row's
    int first;               // column of the first packet; the others lie 32 WR W columns apart
    int edge;                // column of the thread's edge element, -1: it has none
    int mine, its;           // elements that this warp holds, and the warp of the row whose sums this lane looks after
    // `off`: elements by which the rows lie behind the grid
    __device__ __forceinline__ Held(int t, int cols, int off) : there(0), edge(-1) {
        const int head = FIT == EDGE && off ? min(W - off, cols) : 0, packets = (cols - head) / W, edges = cols - packets * W;
        first = head + t * W;
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (t + i * 32 * WR < packets) there |= 1u << i;
        if (FIT == EDGE && t < edges) edge = t < head ? t : t + packets * W;
        mine = of_warp(t >> 5, packets, edges);
        const int w = t % lanes_of(WR);
        its = w < WR ? of_warp(w, packets, edges) : 0;
    }
    __device__ __forceinline__ int column(int i) const { return first + i * 32 * WR * W; }
    __device__ __forceinline__ bool has(int i) const { return FIT == FULL || (there >> i & 1); }
    __device__ __forceinline__ bool has_edge() const { return FIT == EDGE && edge >= 0; }
  private:
    static __device__ __forceinline__ int of_warp(int w, int packets, int edges) {
        if (FIT == FULL) return 32 * C * W;
        int n = FIT == EDGE && w == 0 ? edges : 0;
#pragma unroll
        for (int i = 0; i < C; ++i) n += min(max(packets - (i * WR + w) * 32, 0), 32) * W;
        return n;
    }
};
template <Rowfit FIT, typename T>
__device__ __forceinline__ int behind_grid(const T* row) { return FIT == EDGE ? (int)((uintptr_t)row % 16 / sizeof(T)) : 0; }

__device__ __forceinline__ void copy_async(uint4* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// W neighbouring values: pairs, which one instruction works on, or a single one.
template <int W>
struct Vals {
    Two p[W / 2];
    __device__ __forceinline__ void all(float a) {
#pragma unroll
        for (int e = 0; e < W / 2; ++e) p[e] = both(a);
    }
    __device__ __forceinline__ float sum() const {
        Two s = p[0];
#pragma unroll
        for (int e = 1; e < W / 2; ++e) s = s + p[e];
        return total(s);
    }
    __device__ __forceinline__ void add(float a) {
#pragma unroll
        for (int e = 0; e < W / 2; ++e) p[e] = p[e] + both(a);
    }
    __device__ __forceinline__ void add(const Vals& a) {
#pragma unroll
        for (int e = 0; e < W / 2; ++e) p[e] = p[e] + a.p[e];
    }
    __device__ __forceinline__ void mul(float a) {
#pragma unroll
        for (int e = 0; e < W / 2; ++e) p[e] = p[e] * both(a);
    }
    __device__ __forceinline__ void mul(const Vals& a) {
#pragma unroll
        for (int e = 0; e < W / 2; ++e) p[e] = p[e] * a.p[e];
    }
    __device__ __forceinline__ void fma(const Vals& a, const Vals& b, const Vals& c) {        // a b + c
#pragma unroll
        for (int e = 0; e < W / 2; ++e) p[e] = multiply_add(a.p[e], b.p[e], c.p[e]);
    }
    __device__ __forceinline__ void fma(const Vals& a, const Vals& b, float c) {
#pragma unroll
        for (int e = 0; e < W / 2; ++e) p[e] = multiply_add(a.p[e], b.p[e], both(c));
    }
    __device__ __forceinline__ void fma(const Vals& a, float b, const Vals& c) {
#pragma unroll
        for (int e = 0; e < W / 2; ++e) p[e] = multiply_add(a.p[e], both(b), c.p[e]);
    }
    __device__ __forceinline__ float value(int e) const {
        float a, b;
        parts(p[e / 2], a, b);
        return e & 1 ? b : a;
    }
    template <typename T> __device__ __forceinline__ void read(const T* from) { pairs_of(*reinterpret_cast<const uint4*>(from), p, from); }
    template <typename T> __device__ __forceinline__ void write(T* to) const { *reinterpret_cast<uint4*>(to) = packet_of(p, to); }
    // weights of W neighbouring columns; they lie on the 16-byte grid, or element by element
    template <bool GRID, typename P> __device__ __forceinline__ void weights(const P* w) {
        if constexpr (!GRID) {
#pragma unroll
            for (int e = 0; e < W; e += 2) p[e / 2] = two(widen(w[e]), widen(w[e + 1]));
        } else if constexpr (sizeof(P) == 2) {
            read(w);
        } else {
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                const float4 q = reinterpret_cast<const float4*>(w)[i];
                p[2 * i] = two(q.x, q.y);
                p[2 * i + 1] = two(q.z, q.w);
            }
        }
    }
};
template <>
struct Vals<1> {
    float f;
    __device__ __forceinline__ void all(float a) { f = a; }
    __device__ __forceinline__ float sum() const { return f; }
    __device__ __forceinline__ void add(float a) { f += a; }
    __device__ __forceinline__ void add(const Vals& a) { f += a.f; }
    __device__ __forceinline__ void mul(float a) { f *= a; }
    __device__ __forceinline__ void mul(const Vals& a) { f *= a.f; }
    __device__ __forceinline__ void fma(const Vals& a, const Vals& b, const Vals& c) { f = __fmaf_rn(a.f, b.f, c.f); }
    __device__ __forceinline__ void fma(const Vals& a, const Vals& b, float c) { f = __fmaf_rn(a.f, b.f, c); }
    __device__ __forceinline__ void fma(const Vals& a, float b, const Vals& c) { f = __fmaf_rn(a.f, b, c.f); }
    __device__ __forceinline__ float value(int) const { return f; }
    template <typename T> __device__ __forceinline__ void read(const T* from) { f = widen(*from); }
    template <typename T> __device__ __forceinline__ void write(T* to) const { *to = Narrow<T>::of(f); }
    template <bool GRID, typename P> __device__ __forceinline__ void weights(const P* w) { f = widen(*w); }
};

// over the lanes that stand for WR warps
template <int WR>
__device__ __forceinline__ float sum_of(float v) {
#pragma unroll
    for (int m = lanes_of(WR) / 2; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// s / n, from 1 / n and one correction
__device__ __forceinline__ float quotient(float s, int n, float per_n) {
    const float m = s * per_n;
    return __fmaf_rn(__fmaf_rn(-m, (float)n, s), per_n, m);
}

// The threads that share a row meet: the two groups of a CTA at a barrier each (one whose number is computed would count as all
// sixteen), more of them at one, and go from row to row together.
__host__ __device__ constexpr bool meet(int warps, int groups) { return warps > 1 && groups > 2; }
template <int WR, int GROUPS>
__device__ __forceinline__ void row_barrier(int group) {
    if (GROUPS != 2) __syncthreads();
    else if (group == 0) asm volatile("bar.sync 1, %0;" ::"n"(32 * WR) : "memory");
    else asm volatile("bar.sync 2, %0;" ::"n"(32 * WR) : "memory");
}

template <typename T, typename P, int W, int C, int WR, int GROUPS, int DEPTH, int CTAS, Rowfit FIT>
__global__ void __launch_bounds__(32 * WR * GROUPS, CTAS) norm_resident_kernel(const T* x, long long ldx, const P* __restrict__ gamma,
                                                                               const P* __restrict__ beta, T* y, long long ldy,
                                                                               long long rows, int cols, float eps) {
    constexpr int THREADS = 32 * WR * GROUPS;
    constexpr bool MEET = meet(WR, GROUPS);
    extern __shared__ uint4 ring[];          // [DEPTH][C][THREADS]
    __shared__ float2 sm[2][GROUPS * WR];
    dependent_prologue();
    const int lane = threadIdx.x & 31, group = threadIdx.x / (32 * WR), warp = threadIdx.x / 32 % WR;
    long long row = (long long)blockIdx.x * GROUPS + group;
    const int off = behind_grid<FIT>(x + row * ldx);
    const Held<W, C, WR, FIT> at(threadIdx.x % (32 * WR), cols, off);
    const float per_mine = at.mine ? 1.0f / at.mine : 0.0f, per_col = 1.0f / cols;
    const float its = at.its, per_its = at.its ? 1.0f / at.its : 0.0f;
    const long long step = (long long)gridDim.x * GROUPS;
    // The weights stay in registers where there are not too many of them: reading them again for every row, 32 bytes for each 16 of
    // a bf16 row, kept L1 85% busy at 40% of the memory's bandwidth (62 us instead of 43 for 16384 x 4096).
    constexpr bool HOLD = C * W <= 16;
    Vals<W> g[HOLD ? C : 1], b[HOLD ? C : 1];
    if (HOLD) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            g[i].all(1);
            b[i].all(0);
            if (gamma && at.has(i)) g[i].template weights<FIT != EDGE>(gamma + at.column(i));
            if (beta && at.has(i)) b[i].template weights<FIT != EDGE>(beta + at.column(i));
        }
    }
    const T *from = x + row * ldx, *ahead = from;          // the row, and the next one to be fetched
    T* to = y + row * ldy;
    long long fetched = row;
    auto fetch = [&](int stage) {
        if (fetched < rows) {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (at.has(i)) copy_async(ring + (stage * C + i) * THREADS + threadIdx.x, ahead + at.column(i));
        }
        copies_issued();
        fetched += step;
        ahead += step * ldx;
    };
    if (W > 1)
        for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
    int stage = 0, turn = 0;
    const float edge_g = gamma && at.has_edge() ? widen(gamma[at.edge]) : 1.0f, edge_b = beta && at.has_edge() ? widen(beta[at.edge]) : 0.0f;
    T edge_next = T();          // a row ahead, and as it was read: widened here, the thread would wait for it
    if (at.has_edge() && row < rows) edge_next = from[at.edge];
    for (; row - (MEET ? group : 0) < rows; row += step, from += step * ldx, to += step * ldy) {
        const bool live = !MEET || row < rows;
        if (W > 1) {
            fetch(stage ? stage - 1 : DEPTH - 1);
            copies_but<DEPTH - 1>();
        }
        Vals<W> v[C];
        const float edge = widen(edge_next);
        if (at.has_edge() && row + step < rows) edge_next = from[step * ldx + at.edge];
        float sum = edge;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            if (at.has(i) && (W > 1 || live)) v[i].read(W > 1 ? (const T*)(ring + (stage * C + i) * THREADS + threadIdx.x) : from + at.column(i));
            else v[i].all(0);
            sum += v[i].sum();
        }
        sum = warp_sum(sum);
        const float mean_w = sum * per_mine;
        Vals<W> squares;
        squares.all(0);
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (at.has(i)) {
                Vals<W> d = v[i];
                d.add(-mean_w);
                squares.fma(d, d, squares);
            }
        float q = squares.sum();
        if (at.has_edge()) q += (edge - mean_w) * (edge - mean_w);
        q = warp_sum(q);
        float mean = quotient(sum, cols, per_col);
        if (WR > 1) {
            float2* all = sm[turn] + group * WR;
            turn ^= 1;
            if (lane == 0) all[warp] = make_float2(sum, q);
            row_barrier<WR, GROUPS>(group);
            const int other = lane % lanes_of(WR);
            const float2 o = other < WR ? all[other] : make_float2(0, 0);
            mean = quotient(sum_of<WR>(o.x), cols, per_col);
            const float d = o.x * per_its - mean;
            q = sum_of<WR>(o.y + its * d * d);
        }
        const float r = rsqrtf(q * per_col + eps);
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (at.has(i) && live) {
                v[i].add(-mean);          // (exact for a row that does not vary, where r is largest)
                v[i].mul(r);
                if (HOLD) {
                    v[i].fma(v[i], g[i], b[i]);
                } else {
                    Vals<W> w;
                    if (gamma) {
                        w.template weights<FIT != EDGE>(gamma + at.column(i));
                        v[i].mul(w);
                    }
                    if (beta) {
                        w.template weights<FIT != EDGE>(beta + at.column(i));
                        v[i].add(w);
                    }
                }
                v[i].write(to + at.column(i));
            }
        if (at.has_edge() && live) to[at.edge] = Narrow<T>::of((edge - mean) * r * edge_g + edge_b);
        stage = stage + 1 == DEPTH ? 0 : stage + 1;
    }
}

// Every CTA takes rows gridDim.x * GROUPS apart, sums dy h and dy of its columns in registers and leaves them, its groups added in
// their order, in partial[CTA][0 / 1].
template <typename T, typename P, int W, int C, int WR, int GROUPS, int DEPTH, int CTAS, Rowfit FIT>
__global__ void __launch_bounds__(32 * WR * GROUPS, CTAS)
    norm_backward_resident_kernel(const T* dy, long long lddy, const T* x, long long ldx, const P* __restrict__ gamma, T* dx, long long lddx,
                                  long long rows, int cols, float eps, float* __restrict__ partial) {
    constexpr int THREADS = 32 * WR * GROUPS;
    constexpr bool MEET = meet(WR, GROUPS);
    extern __shared__ uint4 ring[];          // [DEPTH][2][C][THREADS]; in the end [2][cols] sums, where several groups have some to add
    __shared__ float4 sm[2][GROUPS * WR];
    dependent_prologue();
    const int lane = threadIdx.x & 31, group = threadIdx.x / (32 * WR), warp = threadIdx.x / 32 % WR;
    long long row = (long long)blockIdx.x * GROUPS + group;
    const int off = behind_grid<FIT>(x + row * ldx);
    const Held<W, C, WR, FIT> at(threadIdx.x % (32 * WR), cols, off);
    const float per_mine = at.mine ? 1.0f / at.mine : 0.0f, per_col = 1.0f / cols;
    const float its = at.its, per_its = at.its ? 1.0f / at.its : 0.0f;
    const long long step = (long long)gridDim.x * GROUPS;
    // Up to 16 values a thread, the row and its weights stay in registers across the exchange; above, they are read again behind it
    // (the row from the ring, the weights from L1), and the sums of the columns have the registers.
    constexpr bool HOLD = C * W <= 16;
    // 16-bit rows whose threads do not all hold the same stay in their packets between the two passes, half the registers for one
    // more unpacking (without it 13419 x 5001 spilled: 208 us, now 139; 67108 x 1000 took 98 us, now 93).  Where 8 or more warps
    // share a row on the grid, nothing spills, and unpacking costs 3%.
    constexpr bool PACKED = HOLD && W > 1 && sizeof(T) == 2 && (FIT == EDGE || (FIT == WHOLE && WR < 8));
    constexpr int H = HOLD ? C : 1, R = PACKED ? 1 : H, K = PACKED ? C : 1;
    Vals<W> g[H], dg[C], db[C];
    auto weigh = [&](int i) {
        g[HOLD ? i : 0].all(1);
        if (gamma && at.has(i)) g[HOLD ? i : 0].template weights<FIT != EDGE>(gamma + at.column(i));
    };
#pragma unroll
    for (int i = 0; i < C; ++i) {
        dg[i].all(0);
        db[i].all(0);
        if (HOLD) weigh(i);
    }
    auto slot = [&](int stage, int which, int i) { return ring + ((stage * 2 + which) * C + i) * THREADS + threadIdx.x; };
    const T *from_x = x + row * ldx, *from_dy = dy + row * lddy, *ahead_x = from_x, *ahead_dy = from_dy;
    T* to_dx = dx + row * lddx;
    long long fetched = row;
    auto fetch = [&](int stage) {
        if (fetched < rows) {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (at.has(i)) {
                    copy_async(slot(stage, 0, i), ahead_x + at.column(i));
                    copy_async(slot(stage, 1, i), ahead_dy + at.column(i));
                }
        }
        copies_issued();
        fetched += step;
        ahead_x += step * ldx;
        ahead_dy += step * lddy;
    };
    if (W > 1)
        for (int d = 0; d < DEPTH - 1; ++d) fetch(d);
    int stage = 0, turn = 0;
    const float edge_g = gamma && at.has_edge() ? widen(gamma[at.edge]) : 1.0f;
    float edge_dg = 0, edge_db = 0;
    T edge_x_next = T(), edge_dy_next = T();          // a row ahead
    if (at.has_edge() && row < rows) {
        edge_x_next = from_x[at.edge];
        edge_dy_next = from_dy[at.edge];
    }
    for (; row - (MEET ? group : 0) < rows; row += step, from_x += step * ldx, from_dy += step * lddy, to_dx += step * lddx) {
        const bool live = !MEET || row < rows;
        if (W > 1) {
            fetch(stage ? stage - 1 : DEPTH - 1);
            copies_but<DEPTH - 1>();
        }
        Vals<W> v[R], u[R];
        uint4 px[K], pdy[K];
        float edge_x = widen(edge_x_next), edge_dy = widen(edge_dy_next);
        if (at.has_edge() && row + step < rows) {
            edge_x_next = from_x[step * ldx + at.edge];
            edge_dy_next = from_dy[step * lddy + at.edge];
        }
        float sum = edge_x;
        auto read_x = [&](int i) {
            if constexpr (PACKED) v[0].read((const T*)&px[i]);
            else v[HOLD ? i : 0].read(W > 1 ? (const T*)slot(stage, 0, i) : from_x + at.column(i));
        };
        auto read_dy = [&](int i) {
            if constexpr (PACKED) u[0].read((const T*)&pdy[i]);
            else u[HOLD ? i : 0].read(W > 1 ? (const T*)slot(stage, 1, i) : from_dy + at.column(i));
        };
        auto again = [&] {          // the values are taken out of their packets anew
            if constexpr (PACKED) {
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    asm volatile("" : "+r"(px[i].x), "+r"(px[i].y), "+r"(px[i].z), "+r"(px[i].w));
                    asm volatile("" : "+r"(pdy[i].x), "+r"(pdy[i].y), "+r"(pdy[i].z), "+r"(pdy[i].w));
                }
            }
        };
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (at.has(i) && (W > 1 || live)) {
                if constexpr (PACKED) {
                    px[i] = *slot(stage, 0, i);
                    pdy[i] = *slot(stage, 1, i);
                }
                read_x(i);
                if (HOLD && !PACKED) read_dy(i);
                sum += v[R > 1 ? i : 0].sum();
            }
        again();
        sum = warp_sum(sum);
        const float mean_w = sum * per_mine;
        Vals<W> sq, sa, sc;
        sq.all(0);
        sa.all(0);
        sc.all(0);
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (at.has(i)) {
                const int k = R > 1 ? i : 0, w = HOLD ? i : 0;
                if ((!HOLD || PACKED) && (W > 1 || live)) {
                    read_x(i);
                    read_dy(i);
                }
                if (!HOLD) weigh(i);
                Vals<W> d = v[k], ae = u[k];
                d.add(-mean_w);
                ae.mul(g[w]);
                sq.fma(d, d, sq);
                sa.add(ae);
                sc.fma(ae, d, sc);
            }
        float q = sq.sum(), a = sa.sum(), c = sc.sum();
        if (at.has_edge()) {
            const float d = edge_x - mean_w, ae = edge_dy * edge_g;
            q += d * d;
            a += ae;
            c += ae * d;
        }
        q = warp_sum(q);
        a = warp_sum(a);
        c = warp_sum(c);
        float mean = quotient(sum, cols, per_col);
        if (WR > 1) {
            float4* all = sm[turn] + group * WR;
            turn ^= 1;
            if (lane == 0) all[warp] = make_float4(sum, q, a, c);
            row_barrier<WR, GROUPS>(group);
            const int other = lane % lanes_of(WR);
            const float4 o = other < WR ? all[other] : make_float4(0, 0, 0, 0);
            mean = quotient(sum_of<WR>(o.x), cols, per_col);
            const float d = o.x * per_its - mean;      // (a warp without elements has o.x = o.z = 0)
            q = sum_of<WR>(o.y + its * d * d);
            a = sum_of<WR>(o.z);
            c = sum_of<WR>(o.w + o.z * d);
        }
        again();
        const float r = rsqrtf(q * per_col + eps);
        const float c1 = -r * (a * per_col), c2 = -r * r * (r * (c * per_col));
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (at.has(i) && live) {
                const int k = R > 1 ? i : 0, w = HOLD ? i : 0;
                if (!HOLD || PACKED) {
                    read_x(i);
                    read_dy(i);
                }
                if (!HOLD) weigh(i);
                v[k].add(-mean);          // h / r
                db[i].add(u[k]);
                u[k].mul(r);
                dg[i].fma(u[k], v[k], dg[i]);
                u[k].fma(u[k], g[w], c1);
                u[k].fma(v[k], c2, u[k]);
                if (dx) u[k].write(to_dx + at.column(i));
            }
        if (at.has_edge() && live) {
            edge_x -= mean;
            edge_db += edge_dy;
            edge_dy *= r;
            edge_dg += edge_dy * edge_x;
            if (dx) to_dx[at.edge] = Narrow<T>::of(edge_dy * edge_g + c1 + edge_x * c2);
        }
        stage = stage + 1 == DEPTH ? 0 : stage + 1;
    }
    if (!partial) return;
    float* to = partial + 2 * (long long)blockIdx.x * cols;
    float* columns = reinterpret_cast<float*>(ring);
    if (GROUPS > 1) __syncthreads();          // the ring is done with
    for (int k = 0; k < GROUPS; ++k) {
        if (group == k) {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (at.has(i)) {
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        float *pg = (GROUPS == 1 ? to : columns) + at.column(i) + e, *pb = pg + cols;
                        *pg = k ? *pg + dg[i].value(e) : dg[i].value(e);
                        *pb = k ? *pb + db[i].value(e) : db[i].value(e);
                    }
                }
        }
        if (group == k && at.has_edge()) {
            float *pg = (GROUPS == 1 ? to : columns) + at.edge, *pb = pg + cols;
            *pg = k ? *pg + edge_dg : edge_dg;
            *pb = k ? *pb + edge_db : edge_db;
        }
        if (GROUPS > 1) __syncthreads();
    }
    if (GROUPS > 1)
        for (int i = threadIdx.x; i < 2 * cols; i += THREADS) to[i] = columns[i];
}

// How rows are held: `packets` a thread, `warps` a row (0: they are too long), rows a CTA at a time where a row has fewer than 8 warps.
struct Layout { int packets, warps; };
constexpr int groups_of(int warps) { return warps < 8 ? 8 / warps : 1; }

// The warps are as few as hold the row: a lane without packets costs as much as one with them (13107 x 5120 bf16: 48 us with 10
// warps, 74 with 16).
// Forward, measured at 2^26 elements: 16 values a thread (16384 x 4096 bf16: 43 us; 8 values 53, 32 values 58), 8 where a warp can hold
// the row with them (65536 x 256 f32: 23 us; two warps 23 to 29), 32 for bf16 rows that 32 warps cannot hold with 16.
Layout forward_layout(int size, int64_t cols) {
    const int64_t packets = (cols + 16 / size - 1) / (16 / size);
    Layout l = {size == 2 ? 2 : 4, 1};
    if (packets <= 32ll * l.packets / 2) l.packets /= 2;
    else if (size == 2 && packets > 32 * 32 * 2) l.packets = 4;
    for (int warps : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 32}) {
        l.warps = warps;
        if (32ll * l.packets * warps >= packets) return l;
    }
    l.warps = 0;
    return l;
}
// Backward: 16 values a thread for bf16 rows (16384 x 4096: 82 us; 8 values 103), 8 for f32 rows (65536 x 1024: 127 us; 16 values 144);
// 32 for rows that 16 warps cannot hold with these.  No 6, 10 or 12 warps: what they save on lanes, the SM loses with 12 or 10 warps
// in place of 16.
Layout backward_layout(int size, int64_t cols) {
    const int64_t packets = (cols + 16 / size - 1) / (16 / size);
    Layout l = {size == 2 && packets <= 32 ? 1 : 2, 1};
    const int most = size == 2 ? 16 : 32;
    for (int warps : {1, 2, 3, 4, 5, 8, 16, 32, 64}) {
        l.warps = warps;
        if (32ll * l.packets * warps >= packets) break;
    }
    if (l.warps > most) l = {size == 2 ? 4 : 8, 32ll * 16 * (size == 2 ? 4 : 8) < packets ? 0 : 16};
    return l;
}
// Do the rows of two matrices lie alike on the 16-byte grid?
bool alike(const Rows& a, const Rows& b) {
    return ((uintptr_t)a.data - (uintptr_t)b.data) % 16 == 0 && (a.rows < 2 || (a.stride - b.stride) * a.size % 16 == 0);
}
bool on_grid(const void* p) { return (uintptr_t)p % 16 == 0; }
bool on_grid(const Rows& m) { return (uintptr_t)m.data % 16 == 0 && (m.rows < 2 || m.stride * m.size % 16 == 0); }
// at most that many CTAs, a multiple of 8, so that the rows of one lie alike on the grid
long long capped_alike(long long want, long long most) { return want <= most ? std::max(want, 1ll) : most / 8 * 8; }

long long capped(long long want, long long most) { return std::max<long long>(1, std::min(want, most)); }

long long column_slices(long long rows, long long cols) {
    const long long tiles = (cols + kThreads - 1) / kThreads;
    return capped((kSms * 8 + tiles - 1) / tiles, std::max<long long>(1, rows / 4));
}

// 16 values a thread take 128 registers: 16 warps an SM, or 15.
constexpr int backward_groups_of(int warps) { return warps == 3 ? 5 : groups_of(warps); }
constexpr int backward_resident_ctas(int threads) { return threads > 256 ? 1 : threads > 160 ? 2 : 3; }
long long backward_ctas(const Layout& l, int64_t rows) {
    const int groups = backward_groups_of(l.warps);
    return capped_alike((rows + groups - 1) / groups, kSms * backward_resident_ctas(32 * groups * l.warps));
}

// What the sums over the rows hand from launch to launch; dx alone comes out of one launch that needs none of it.
struct BackwardSpace { size_t stats, partial, total; long long slices; };
BackwardSpace backward_space(int dtype, int64_t rows, int64_t cols) {
    const size_t a = dtype == DALIB200_F64 ? 8 : 4;
    BackwardSpace b;
    const Layout l = backward_layout(size_of(dtype), cols);
    if (dtype != DALIB200_F64 && l.warps) {
        b.slices = backward_ctas(l, rows);
        b.stats = 0;
    } else {
        b.slices = column_slices(rows, cols);
        b.stats = ((size_t)rows * 4 * a + 255) / 256 * 256;
    }
    b.partial = (size_t)b.slices * 2 * cols * a;
    b.total = b.stats + b.partial;
    return b;
}

// Lets the kernel take more shared memory than every kernel may; asked for once a device (`done`: a bit for each).
template <typename K>
cudaError_t allow_shared(K kernel, size_t bytes, std::atomic<unsigned long long>* done) {
    if (bytes <= 40 * 1024) return cudaSuccess;
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || done->load() >> (device & 63) & 1) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) done->fetch_or(1ull << (device & 63));
    return e;
}

constexpr int kDepth = 3;
template <typename T, typename P, int C, int WR>
cudaError_t forward_resident(cudaStream_t s, const Rows& x, const void* gamma, const void* beta, const Rows& y, double eps) {
    constexpr int N = Packet<T>::N, GROUPS = groups_of(WR), THREADS = 32 * WR * GROUPS;
    constexpr int CTAS = std::max(1, (C * N > 16 ? 512 : C * N > 8 ? 768 : 1024) / THREADS);          // (80 registers a thread hold 16 values)
    // (16 values and a thread's edge want some registers more; with two CTAs in place of three: 67041 x 1001 bf16 86 -> 59 us)
    constexpr int EC = C * N > 8 && THREADS <= 256 ? 512 / THREADS : CTAS;
    const bool vec = alike(x, y);
    const bool whole = vec && on_grid(x) && x.cols % N == 0 && on_grid(gamma) && on_grid(beta), full = whole && x.cols == (int64_t)32 * WR * C * N;
    auto kernel = full    ? norm_resident_kernel<T, P, N, C, WR, GROUPS, kDepth, CTAS, FULL>
                  : whole ? norm_resident_kernel<T, P, N, C, WR, GROUPS, kDepth, CTAS, WHOLE>
                  : vec   ? norm_resident_kernel<T, P, N, C, WR, GROUPS, kDepth, EC, EDGE>
                          : norm_resident_kernel<T, P, 1, C * N, WR, GROUPS, kDepth, CTAS, WHOLE>;
    const size_t smem = vec ? (size_t)kDepth * C * THREADS * 16 : 0;
    static std::atomic<unsigned long long> allowed[3];
    const cudaError_t e = allow_shared(kernel, smem, &allowed[full ? 0 : whole ? 1 : 2]);
    if (e != cudaSuccess) return e;
    const long long ctas = (x.rows + GROUPS - 1) / GROUPS;
    return launch(kernel, dim3((unsigned)capped_alike(ctas, kSms * (vec ? whole ? CTAS : EC : 32))), THREADS, smem, s, 1,
                  (const T*)x.data, (long long)x.stride, (const P*)gamma, (const P*)beta, (T*)y.data, (long long)y.stride,
                  (long long)x.rows, (int)x.cols, (float)eps);
}
template <typename T, typename P, int C>
cudaError_t forward_resident(cudaStream_t s, int warps, const Rows& x, const void* gamma, const void* beta, const Rows& y, double eps) {
    switch (warps) {
        case 1: return forward_resident<T, P, C, 1>(s, x, gamma, beta, y, eps);
        case 2: return forward_resident<T, P, C, 2>(s, x, gamma, beta, y, eps);
        case 3: return forward_resident<T, P, C, 3>(s, x, gamma, beta, y, eps);
        case 4: return forward_resident<T, P, C, 4>(s, x, gamma, beta, y, eps);
        case 5: return forward_resident<T, P, C, 5>(s, x, gamma, beta, y, eps);
        case 6: return forward_resident<T, P, C, 6>(s, x, gamma, beta, y, eps);
        case 10: return forward_resident<T, P, C, 10>(s, x, gamma, beta, y, eps);
        case 12: return forward_resident<T, P, C, 12>(s, x, gamma, beta, y, eps);
        case 8: return forward_resident<T, P, C, 8>(s, x, gamma, beta, y, eps);
        case 16: return forward_resident<T, P, C, 16>(s, x, gamma, beta, y, eps);
        default: return forward_resident<T, P, C, 32>(s, x, gamma, beta, y, eps);
    }
}

template <typename T> constexpr int packet_width() { return sizeof(T) == 8 ? 1 : Packet<T>::N; }
int row_threads(int64_t cols) { return cols > 4096 ? 1024 : kThreads; }

template <typename T, typename P>
cudaError_t forward(cudaStream_t s, const Rows& x, const void* gamma, const void* beta, const Rows& y, double eps) {
    if constexpr (sizeof(T) < 8) {
        const Layout l = forward_layout(sizeof(T), x.cols);
        constexpr int C = sizeof(T) == 2 ? 1 : 2;
        if (l.warps) {
            if (l.packets == C) return forward_resident<T, P, C, 1>(s, x, gamma, beta, y, eps);
            if constexpr (sizeof(T) == 2)
                if (l.packets == 4) return forward_resident<T, P, 4, 32>(s, x, gamma, beta, y, eps);          // (above 2048 packets a row)
            return forward_resident<T, P, 2 * C>(s, l.warps, x, gamma, beta, y, eps);
        }
    }
    auto kernel = sizeof(T) < 8 && alike(x, y) ? norm_rows_kernel<T, P, packet_width<T>()> : norm_rows_kernel<T, P, 1>;
    return launch(kernel, dim3((unsigned)capped(x.rows, kSms * 64)), row_threads(x.cols), 0, s, 1, (const T*)x.data, (long long)x.stride,
                  (const P*)gamma, (const P*)beta, (T*)y.data, (long long)y.stride, (long long)x.rows, (long long)x.cols, eps);
}

template <typename P, typename A>
cudaError_t fold_columns(cudaStream_t s, const A* partial, long long slices, long long cols, void* dgamma, void* dbeta) {
    return launch(fold_columns_kernel<A, P>, dim3((unsigned)((cols + 31) / 32), 2), kThreads, 0, s, 1, partial, slices, cols, (P*)dgamma,
                  (P*)dbeta);
}

template <typename T, typename P, int C, int WR>
cudaError_t backward_resident(cudaStream_t s, const BackwardSpace& b, const Rows& dy, const Rows& x, const void* gamma, const Rows& dx,
                              void* dgamma, void* dbeta, double eps, void* space) {
    constexpr int N = Packet<T>::N, GROUPS = backward_groups_of(WR), THREADS = 32 * WR * GROUPS;
    constexpr int CTAS = backward_resident_ctas(THREADS);
    constexpr int DEPTH = C * N > 16 ? (sizeof(T) == 2 ? 2 : 1) : kDepth;          // (what fits an SM's shared memory)
    const bool vec = alike(x, dy) && (!dx.data || alike(x, dx));
    const bool whole = vec && on_grid(x) && x.cols % N == 0 && on_grid(gamma), full = whole && x.cols == (int64_t)32 * WR * C * N;
    auto kernel = full    ? norm_backward_resident_kernel<T, P, N, C, WR, GROUPS, DEPTH, CTAS, FULL>
                  : whole ? norm_backward_resident_kernel<T, P, N, C, WR, GROUPS, DEPTH, CTAS, WHOLE>
                  : vec   ? norm_backward_resident_kernel<T, P, N, C, WR, GROUPS, DEPTH, CTAS, EDGE>
                          : norm_backward_resident_kernel<T, P, 1, C * N, WR, GROUPS, DEPTH, CTAS, WHOLE>;
    float* partial = dgamma || dbeta ? (float*)space : nullptr;
    const size_t smem = std::max<size_t>(vec ? (size_t)DEPTH * 2 * C * THREADS * 16 : 0, GROUPS > 1 ? 2 * x.cols * sizeof(float) : 0);
    static std::atomic<unsigned long long> allowed[3];
    cudaError_t e = allow_shared(kernel, smem, &allowed[full ? 0 : whole ? 1 : 2]);
    if (e != cudaSuccess) return e;
    e = launch(kernel, dim3((unsigned)b.slices), THREADS, smem, s, 1, (const T*)dy.data, (long long)dy.stride, (const T*)x.data,
               (long long)x.stride, (const P*)gamma, (T*)dx.data, (long long)dx.stride, (long long)x.rows, (int)x.cols, (float)eps, partial);
    return e == cudaSuccess && partial ? fold_columns<P>(s, (const float*)partial, b.slices, x.cols, dgamma, dbeta) : e;
}
template <typename T, typename P, int C, typename... R>
cudaError_t backward_resident_of(int warps, R... rest) {
    switch (warps) {
        case 1: return backward_resident<T, P, C, 1>(rest...);
        case 2: return backward_resident<T, P, C, 2>(rest...);
        case 3: return backward_resident<T, P, C, 3>(rest...);
        case 4: return backward_resident<T, P, C, 4>(rest...);
        case 5: return backward_resident<T, P, C, 5>(rest...);
        case 8: return backward_resident<T, P, C, 8>(rest...);
        case 16: return backward_resident<T, P, C, 16>(rest...);
        default:
            if constexpr (sizeof(T) == 4) return backward_resident<T, P, C, 32>(rest...);
            return cudaErrorInvalidValue;          // (no layout of 16-bit rows has more than 16 warps)
    }
}

template <typename T, typename P>
cudaError_t backward(cudaStream_t s, const Rows& dy, const Rows& x, const void* gamma, const Rows& dx, void* dgamma, void* dbeta,
                     double eps, void* space) {
    typedef typename AccOf<T>::type A;
    const BackwardSpace b = backward_space(sizeof(T) == 8 ? DALIB200_F64 : sizeof(T) == 2 ? DALIB200_BF16 : DALIB200_F32, x.rows, x.cols);
    if constexpr (sizeof(T) < 8) {
        const Layout l = backward_layout(sizeof(T), x.cols);
        if (l.warps) {
            if (l.packets == 2) return backward_resident_of<T, P, 2>(l.warps, s, b, dy, x, gamma, dx, dgamma, dbeta, eps, space);
            if constexpr (sizeof(T) == 2) {
                if (l.packets == 1) return backward_resident<T, P, 1, 1>(s, b, dy, x, gamma, dx, dgamma, dbeta, eps, space);
                return backward_resident<T, P, 4, 16>(s, b, dy, x, gamma, dx, dgamma, dbeta, eps, space);
            } else {
                return backward_resident<T, P, 8, 16>(s, b, dy, x, gamma, dx, dgamma, dbeta, eps, space);
            }
        }
    }
    A* stats = (A*)space;          // nullptr: no sums are asked for
    A* partial = (A*)((char*)space + b.stats);
    const bool packets = sizeof(T) < 8 && alike(x, dy) && (!dx.data || alike(x, dx)), sums = dgamma || dbeta;
    const bool late = sums && dx.data && (meets(dx.data, dx.end() - dx.begin(), x.data, x.end() - x.begin()) ||
                                          meets(dx.data, dx.end() - dx.begin(), dy.data, dy.end() - dy.begin()));
    const dim3 by_row((unsigned)capped(x.rows, kSms * 64));
    cudaError_t e = launch(packets ? row_stats_kernel<T, P, packet_width<T>()> : row_stats_kernel<T, P, 1>, by_row, row_threads(x.cols), 0, s, 1,
                           (const T*)dy.data, (long long)dy.stride, (const T*)x.data, (long long)x.stride, (const P*)gamma,
                           late ? nullptr : (T*)dx.data, (long long)dx.stride, (long long)x.rows, (long long)x.cols, eps, stats);
    if (e == cudaSuccess && sums) {
        e = launch(column_sums_kernel<T>, dim3((unsigned)((x.cols + kThreads - 1) / kThreads), (unsigned)b.slices), kThreads, 0, s, 1,
                   (const T*)dy.data, (long long)dy.stride, (const T*)x.data, (long long)x.stride, (long long)x.rows,
                   (long long)x.cols, (const A*)stats, partial);
        if (e == cudaSuccess) e = fold_columns<P>(s, (const A*)partial, b.slices, x.cols, dgamma, dbeta);
    }
    if (e == cudaSuccess && late)
        e = launch(packets ? dx_kernel<T, P, packet_width<T>()> : dx_kernel<T, P, 1>, by_row, row_threads(x.cols), 0, s, 1, (const T*)dy.data,
                   (long long)dy.stride, (const T*)x.data, (long long)x.stride, (const P*)gamma, (T*)dx.data, (long long)dx.stride,
                   (long long)x.rows, (long long)x.cols, (const A*)stats);
    return e;
}

// ---------------------------------------------------------------------------------------------- arguments
int check_types(const char* what, int dtype, int param_dtype) {
    if (!floating(dtype)) return refuse(std::string(what) + ": dtype must be f32, f64 or bf16");
    if (param_dtype != dtype && !(dtype == DALIB200_BF16 && param_dtype == DALIB200_F32))
        return refuse(std::string(what) + ": the weights have the rows' type, or f32 beside bf16 rows");
    return DALIB200_OK;
}

int check_weights(const char* what, const char* name, const void* p, int param_dtype) {
    if (p && (uintptr_t)p % size_of(param_dtype)) return refuse(std::string(what) + ": " + name + " is not aligned to its elements");
    return DALIB200_OK;
}

}  // namespace
}  // namespace dalib

using namespace dalib;

extern "C" int dalib200_layer_norm(int device, void* stream, int dtype, int param_dtype, int64_t rows, int64_t cols, const void* x,
                                   int64_t x_row_stride, const void* gamma, const void* beta, double eps, void* out,
                                   int64_t out_row_stride) {
    return guarded("dalib200_layer_norm", [&]() -> int {
        const char* what = "dalib200_layer_norm";
        int rc = check_types(what, dtype, param_dtype);
        if (rc != DALIB200_OK) return rc;
        if (rows < 0 || cols < 0) return refuse("dalib200_layer_norm: negative size");
        if (!(eps >= 0) || eps > 1e30) return refuse("dalib200_layer_norm: eps must be a number >= 0");
        if (rows == 0 || cols == 0) return OnDevice(device).status;
        const Rows mx = {"x", x, rows, cols, x_row_stride, size_of(dtype)}, my = {"out", out, rows, cols, out_row_stride, size_of(dtype)};
        for (const Rows* m : {&mx, &my}) {
            const std::string w = wrong(*m);
            if (!w.empty()) return refuse("dalib200_layer_norm: " + w);
        }
        if (clash(mx, my)) return refuse("dalib200_layer_norm: out overlaps x without being x");
        if ((rc = check_weights(what, "gamma", gamma, param_dtype)) != DALIB200_OK) return rc;
        if ((rc = check_weights(what, "beta", beta, param_dtype)) != DALIB200_OK) return rc;
        const size_t out_bytes = (size_t)(my.end() - my.begin()), w_bytes = (size_t)cols * size_of(param_dtype);
        if (meets(gamma, w_bytes, out, out_bytes) || meets(beta, w_bytes, out, out_bytes))
            return refuse("dalib200_layer_norm: out overlaps the weights");
        OnDevice on(device);
        if (on.status != DALIB200_OK) return on.status;
        cudaStream_t s = (cudaStream_t)stream;
        cudaError_t e;
        if (dtype == DALIB200_F32) e = forward<float, float>(s, mx, gamma, beta, my, eps);
        else if (dtype == DALIB200_F64) e = forward<double, double>(s, mx, gamma, beta, my, eps);
        else if (param_dtype == DALIB200_F32) e = forward<bf16_s, float>(s, mx, gamma, beta, my, eps);
        else e = forward<bf16_s, bf16_s>(s, mx, gamma, beta, my, eps);
        return launched(what, e);
    });
}

extern "C" size_t dalib200_layer_norm_backward_workspace(int dtype, int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return backward_space(dtype, rows, cols).total;
}

extern "C" int dalib200_layer_norm_backward(int device, void* stream, int dtype, int param_dtype, int64_t rows, int64_t cols,
                                            const void* dy, int64_t dy_row_stride, const void* x, int64_t x_row_stride,
                                            const void* gamma, double eps, void* dx, int64_t dx_row_stride, void* dgamma, void* dbeta,
                                            void* workspace, size_t workspace_bytes) {
    return guarded("dalib200_layer_norm_backward", [&]() -> int {
        const char* what = "dalib200_layer_norm_backward";
        int rc = check_types(what, dtype, param_dtype);
        if (rc != DALIB200_OK) return rc;
        if (rows < 0 || cols < 0) return refuse("dalib200_layer_norm_backward: negative size");
        if (!(eps >= 0) || eps > 1e30) return refuse("dalib200_layer_norm_backward: eps must be a number >= 0");
        if (cols == 0) return OnDevice(device).status;
        const int size = size_of(dtype), wsize = size_of(param_dtype);
        for (const void* p : {gamma, (const void*)dgamma, (const void*)dbeta})
            if ((rc = check_weights(what, "a weight or its gradient", p, param_dtype)) != DALIB200_OK) return rc;
        const size_t w_bytes = (size_t)cols * wsize;
        if (meets(dgamma, w_bytes, dbeta, w_bytes)) return refuse("dalib200_layer_norm_backward: dgamma overlaps dbeta");
        for (void* w : {dgamma, dbeta})
            if (meets(w, w_bytes, gamma, w_bytes)) return refuse("dalib200_layer_norm_backward: a weight's gradient overlaps the weight");
        cudaStream_t s = (cudaStream_t)stream;
        if (rows == 0) {      // sums over no rows
            OnDevice on(device);
            if (on.status != DALIB200_OK) return on.status;
            for (void* w : {dgamma, dbeta})
                if (w && (rc = launched(what, cudaMemsetAsync(w, 0, w_bytes, s))) != DALIB200_OK) return rc;
            return DALIB200_OK;
        }
        if (!dx && !dgamma && !dbeta) return refuse("dalib200_layer_norm_backward: no gradient is asked for");
        const Rows mdy = {"dy", dy, rows, cols, dy_row_stride, size}, mx = {"x", x, rows, cols, x_row_stride, size};
        const Rows mdx = {"dx", dx, rows, cols, dx ? dx_row_stride : cols, size};
        for (const Rows* m : {&mdy, &mx, &mdx}) {
            if (m == &mdx && !dx) continue;
            const std::string w = wrong(*m);
            if (!w.empty()) return refuse("dalib200_layer_norm_backward: " + w);
        }
        const size_t need = dgamma || dbeta ? backward_space(dtype, rows, cols).total : 0;
        if (dx) {
            if (clash(mdy, mdx)) return refuse("dalib200_layer_norm_backward: dx overlaps dy without being dy");
            if (clash(mx, mdx)) return refuse("dalib200_layer_norm_backward: dx overlaps x without being x");
            for (const void* w : {gamma, (const void*)dgamma, (const void*)dbeta})
                if (meets(w, w_bytes, dx, (size_t)(mdx.end() - mdx.begin())))
                    return refuse("dalib200_layer_norm_backward: dx overlaps a weight or its gradient");
        }
        for (const Rows* m : {&mdy, &mx})
            for (void* w : {dgamma, dbeta})
                if (meets(w, w_bytes, m->data, (size_t)(m->end() - m->begin())))
                    return refuse("dalib200_layer_norm_backward: a weight's gradient overlaps dy or x");
        if (need) {
            for (const Rows* m : {&mdy, &mx, &mdx})
                if (m->data && meets(workspace, need, m->data, (size_t)(m->end() - m->begin())))
                    return refuse(std::string("dalib200_layer_norm_backward: the workspace overlaps ") + m->name);
            for (const void* w : {gamma, (const void*)dgamma, (const void*)dbeta})
                if (meets(workspace, need, w, w_bytes))
                    return refuse("dalib200_layer_norm_backward: the workspace overlaps a weight or its gradient");
        }
        OnDevice on(device);
        if (on.status != DALIB200_OK) return on.status;
        std::unique_lock<std::mutex> together(launch_mutex(), std::defer_lock);
        void* space = nullptr;
        if (need) {
            if (!workspace) together.lock();
            if ((rc = workspace_for(device, stream, need, workspace, workspace_bytes, &space)) != DALIB200_OK) return rc;
        }
        cudaError_t e;
        if (dtype == DALIB200_F32) e = backward<float, float>(s, mdy, mx, gamma, mdx, dgamma, dbeta, eps, space);
        else if (dtype == DALIB200_F64) e = backward<double, double>(s, mdy, mx, gamma, mdx, dgamma, dbeta, eps, space);
        else if (param_dtype == DALIB200_F32) e = backward<bf16_s, float>(s, mdy, mx, gamma, mdx, dgamma, dbeta, eps, space);
        else e = backward<bf16_s, bf16_s>(s, mdy, mx, gamma, mdx, dgamma, dbeta, eps, space);
        return launched(what, e);
    });
}
