// The norm of a list of gradients taken as one vector, and the gradients scaled down to a largest norm:
// dalib200_sum_squares, dalib200_global_norm, dalib200_scale_to_norm, dalib200_clip_by_global_norm.
//
//   n = sqrt(sum over the tensors of sum g^2),   out = g max_norm / n  where n > max_norm, else g
//
// Squares are summed in fp64: a norm that fp32 can hold does not overflow on the way, and a list of billions of elements
// loses nothing.  A norm that is not finite as it is reported, in fp32 or in fp64, scales nothing: who steps over a list whose
// norm reads infinity finds it unchanged, in place too.
//
// The tensors of a list are cut into chunks; the kernels take the list by value (pointers, sizes and first chunk of each, up
// to kList tensors a launch).  Every CTA of the summing kernel writes one partial sum, and whoever needs the total folds the
// partials in their order, so results do not depend on scheduling and nothing waits.
//
// Bound by memory: the squares of 4e8 bf16 elements 126 us (a copy's rate over the bytes read: 97%; 181 us before a thread's next
// packets were under way while it worked on some), clipped 398 to 409 us.  The gradients are read twice, what is left of them in L2 apart:
// whether they have to be scaled is known when all of them have been read.  Short lists (six tensors
// of 1e6 elements together, 17 us a call) are bound by the host: the list, its checks and the launches.
#include <algorithm>
#include <cmath>
#include <vector>

#include "op_device.cuh"
#include "op_host.h"

namespace dalib {
namespace {

constexpr int kThreads = 256;
constexpr int kList = 96;                    // tensors a launch takes (a list of 96 stays within 4 KB of kernel parameters)
constexpr int kMinChunk = 2048, kMaxChunk = 65536;      // elements
constexpr int kMaxCtas = kSms * 8;

struct List {
    const void* in[kList];
    void* out[kList];
    long long numel[kList];
    long long first[kList + 1];              // chunk
    unsigned char dtype[kList];
    int n, chunk;
};

// the tensor that holds a chunk
__device__ __forceinline__ int tensor_of(const List& l, long long chunk) {
    int lo = 0, hi = l.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= chunk) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

constexpr int kBatch = 4;                    // packets a thread has under way

__device__ __forceinline__ double square(double s, float v) { const double d = (double)v; return fma(d, d, s); }
__device__ __forceinline__ double square(double s, double v) { return fma(v, v, s); }

// a thread's packets of a piece of memory: `head` elements up to the 16-byte grid, whole packets, the rest
template <typename T>
struct Piece {
    static constexpr int N = Packet<T>::N;
    const T* body;
    int head, packets, edges;
    __device__ __forceinline__ Piece(const T* x, int n) {
        head = min(n, (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T)));
        packets = (n - head) / N;
        edges = n - packets * N;
        body = x + head;
    }
    // place of the thread's edge element in the piece (threadIdx.x < edges)
    __device__ __forceinline__ int edge() const { return (int)threadIdx.x < head ? threadIdx.x : threadIdx.x + packets * N; }
    __device__ __forceinline__ Packet<T> packet(int p) const {
        Packet<T> q = {};
        if (p < packets) q = load_packet(body + p * N);
        return q;
    }
};

template <typename T>
__device__ __forceinline__ double sum_chunk(const T* x, int n) {
    constexpr int N = Packet<T>::N;
    const Piece<T> piece(x, n);
    double s = 0, s2 = 0;
    if ((int)threadIdx.x < piece.edges) s = square(s, widen(x[piece.edge()]));
    Packet<T> ahead[kBatch];          // the next packets are on their way while some are worked on (absent ones are zeros)
#pragma unroll
    for (int i = 0; i < kBatch; ++i) ahead[i] = piece.packet(threadIdx.x + i * kThreads);
    for (int p = threadIdx.x; p < piece.packets; p += kBatch * kThreads) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const Packet<T> q = ahead[i];
            ahead[i] = piece.packet(p + (kBatch + i) * kThreads);
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                s = square(s, widen(q.v[e]));
                s2 = square(s2, widen(q.v[e + 1]));
            }
        }
    }
    return s + s2;
}

__global__ void __launch_bounds__(kThreads, 4) squares_kernel(const __grid_constant__ List l, double* __restrict__ partial) {
    __shared__ double sm[kThreads / 32];
    dependent_prologue();
    double s = 0;
    for (long long c = blockIdx.x; c < l.first[l.n]; c += gridDim.x) {
        const int t = tensor_of(l, c);
        const long long at = (c - l.first[t]) * l.chunk;
        const int n = (int)min((long long)l.chunk, l.numel[t] - at);
        if (l.dtype[t] == DALIB200_F32) s += sum_chunk((const float*)l.in[t] + at, n);
        else if (l.dtype[t] == DALIB200_BF16) s += sum_chunk((const bf16_s*)l.in[t] + at, n);
        else s += sum_chunk((const double*)l.in[t] + at, n);
    }
    s = block_sum(s, sm);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ double fold_partials(const double* partial, int n, double* sm) {
    double s = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) s += partial[i];
    return block_sum(s, sm);
}

__device__ __forceinline__ void write_norm(double sum, void* norm, int norm_f64) {
    if (norm_f64) *(double*)norm = sqrt(sum);
    else *(float*)norm = (float)sqrt(sum);
}

// sum (its root with `rooted`) of the partials
__global__ void __launch_bounds__(kThreads) total_kernel(const double* __restrict__ partial, int n, int rooted, void* out, int out_f64) {
    __shared__ double sm[kThreads / 32];
    dependent_prologue();
    const double s = fold_partials(partial, n, sm);
    if (threadIdx.x == 0) {
        if (rooted) write_norm(s, out, out_f64);
        else *(double*)out = s;
    }
}

template <typename T, typename F>
__device__ __forceinline__ void scale_chunk(const T* x, T* y, int n, F f) {
    constexpr int N = Packet<T>::N;
    if (((uintptr_t)x - (uintptr_t)y) % 16 != 0) {          // no packet of one is a packet of the other
        for (int i = threadIdx.x; i < n; i += kThreads) y[i] = Narrow<T>::of(widen(x[i]) * f);
        return;
    }
    const Piece<T> piece(x, n);
    if ((int)threadIdx.x < piece.edges) y[piece.edge()] = Narrow<T>::of(widen(x[piece.edge()]) * f);
    for (int p = threadIdx.x; p < piece.packets; p += kBatch * kThreads) {
        Packet<T> q[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) q[i] = piece.packet(p + i * kThreads);
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
            if (p + i * kThreads < piece.packets) {
#pragma unroll
                for (int e = 0; e < N; ++e) q[i].v[e] = Narrow<T>::of(widen(q[i].v[e]) * f);
                // (streaming: what is written is not read here again, what is still in L2 of the first pass is)
                __stcs(reinterpret_cast<uint4*>(y + piece.head + (p + i * kThreads) * N), *reinterpret_cast<const uint4*>(&q[i]));
            }
    }
}

__global__ void __launch_bounds__(kThreads, 4) scale_kernel(const __grid_constant__ List l, const double* __restrict__ partial, int n_partial,
                                                         double max_norm, void* norm, int norm_f64) {
    __shared__ double sm[kThreads / 32];
    dependent_prologue();
    const double sum = fold_partials(partial, n_partial, sm);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) write_norm(sum, norm, norm_f64);
    const double n = sqrt(sum);
    const bool down = n > max_norm && (norm_f64 ? n <= DBL_MAX : (float)n <= FLT_MAX);
    const double f = down ? max_norm / n : 1.0;
    // from the end of the list: what has been read last for the sum is still in L2
    for (long long c = l.first[l.n] - 1 - blockIdx.x; c >= 0; c -= gridDim.x) {
        const int t = tensor_of(l, c);
        if (!down && l.in[t] == l.out[t]) continue;
        const long long at = (c - l.first[t]) * l.chunk;
        const int m = (int)min((long long)l.chunk, l.numel[t] - at);
        if (l.dtype[t] == DALIB200_F32) scale_chunk((const float*)l.in[t] + at, (float*)l.out[t] + at, m, (float)f);
        else if (l.dtype[t] == DALIB200_BF16) scale_chunk((const bf16_s*)l.in[t] + at, (bf16_s*)l.out[t] + at, m, (float)f);
        else scale_chunk((const double*)l.in[t] + at, (double*)l.out[t] + at, m, f);
    }
}

// ---------------------------------------------------------------------------------------------- the list
struct Tensors {
    std::vector<List> lists;
    int ctas(const List& l) const { return (int)std::min<long long>(l.first[l.n], kMaxCtas); }
    int partials() const {
        int n = 0;
        for (const List& l : lists) n += ctas(l);
        return n;
    }
};

size_t partial_bytes(int64_t tensors) { return ((size_t)(tensors + kList - 1) / kList + 1) * kMaxCtas * sizeof(double); }

struct Range { uintptr_t lo, hi; int tensor; bool written; };

// "" or what is wrong; fills `t`.  out == nullptr: the list is only read.
std::string gather_list(int n, const int* dtypes, const int64_t* numel, const void* const* in, void* const* out, Tensors* t) {
    if (n < 0) return "negative number of tensors";
    if (n > 0 && (!dtypes || !numel || !in)) return "the list's dtypes, numel or pointers are null";
    std::vector<Range> ranges;
    if (out) ranges.reserve(2 * (size_t)n);
    t->lists.reserve(((size_t)n + kList - 1) / kList);
    List* l = nullptr;
    // chunks of a size that gives every CTA several, and of one packet a thread at least
    int64_t all = 0;
    for (int i = 0; i < n; ++i) all += numel[i] > 0 ? std::min<int64_t>(numel[i], int64_t(1) << 40) : 0;
    int chunk = kMinChunk;
    while (chunk < kMaxChunk && (int64_t)chunk * kMaxCtas * 4 < all) chunk *= 2;
    for (int i = 0; i < n; ++i) {
        const auto who = [i] { return "tensor " + std::to_string(i); };
        if (!floating(dtypes[i])) return who() + ": dtype must be f32, f64 or bf16";
        if (numel[i] < 0 || numel[i] > (int64_t(1) << 48)) return who() + ": number of elements out of range";
        if (numel[i] == 0) continue;
        const int size = size_of(dtypes[i]);
        if (!in[i] || (out && !out[i])) return who() + " is a null pointer";
        if ((uintptr_t)in[i] % size || (out && (uintptr_t)out[i] % size)) return who() + " is not aligned to its elements";
        if (out) {
            const uintptr_t a = (uintptr_t)in[i], b = (uintptr_t)out[i], bytes = (uintptr_t)numel[i] * size;
            if (a != b) ranges.push_back({a, a + bytes, i, false});
            ranges.push_back({b, b + bytes, i, true});
        }
        if (!l || l->n == kList) {
            t->lists.emplace_back();
            l = &t->lists.back();
            l->n = 0;
            l->chunk = chunk;
            l->first[0] = 0;
        }
        const int k = l->n++;
        l->in[k] = in[i];
        l->out[k] = out ? out[i] : nullptr;
        l->numel[k] = numel[i];
        l->dtype[k] = (unsigned char)dtypes[i];
        l->first[k + 1] = l->first[k] + (numel[i] + chunk - 1) / chunk;
    }
    // what is written is read or written nowhere else in the list
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.lo < b.lo; });
    uintptr_t end_any = 0, end_written = 0;
    for (const Range& r : ranges) {
        if (r.lo < end_written || (r.written && r.lo < end_any)) return "tensor " + std::to_string(r.tensor) + ": a tensor that is written overlaps another one of the list";
        end_any = std::max(end_any, r.hi);
        if (r.written) end_written = std::max(end_written, r.hi);
    }
    return "";
}

cudaError_t queue_squares(cudaStream_t s, const Tensors& t, double* partial) {
    cudaError_t e = cudaSuccess;
    int at = 0;
    for (const List& l : t.lists) {
        if (e == cudaSuccess) e = launch(squares_kernel, dim3(t.ctas(l)), kThreads, 0, s, 1, l, partial + at);
        at += t.ctas(l);
    }
    return e;
}

cudaError_t queue_scale(cudaStream_t s, const Tensors& t, const double* partial, int n_partial, double max_norm, void* norm, int norm_f64) {
    cudaError_t e = cudaSuccess;
    for (size_t i = t.lists.size(); i-- > 0 && e == cudaSuccess;)
        e = launch(scale_kernel, dim3(t.ctas(t.lists[i])), kThreads, 0, s, 1, t.lists[i], partial, n_partial, max_norm,
                   i == 0 ? norm : nullptr, norm_f64);
    return e;
}

std::string wrong_norm(const void* norm, int norm_dtype, int n, const int64_t* numel, const int* dtypes, const void* const* in, void* const* out) {
    if (norm_dtype != DALIB200_F32 && norm_dtype != DALIB200_F64) return "the norm is f32 or f64";
    if (!norm) return "norm is a null pointer";
    const size_t size = size_of(norm_dtype);
    if ((uintptr_t)norm % size) return "norm is not aligned to its type";
    for (int i = 0; i < n; ++i) {
        const size_t bytes = (size_t)numel[i] * size_of(dtypes[i]);
        if (meets(norm, size, in[i], bytes) || (out && meets(norm, size, out[i], bytes))) return "norm overlaps tensor " + std::to_string(i);
    }
    return "";
}

std::string wrong_workspace(const void* workspace, const void* norm, int norm_dtype, int n, const int64_t* numel, const int* dtypes,
                            const void* const* in, void* const* out) {
    const size_t need = partial_bytes(n);
    if (meets(workspace, need, norm, size_of(norm_dtype))) return "the workspace overlaps the result";
    for (int i = 0; i < n; ++i) {
        const size_t bytes = (size_t)numel[i] * size_of(dtypes[i]);
        if (meets(workspace, need, in[i], bytes) || (out && meets(workspace, need, out[i], bytes)))
            return "the workspace overlaps tensor " + std::to_string(i);
    }
    return "";
}

}  // namespace
}  // namespace dalib

using namespace dalib;

extern "C" size_t dalib200_global_norm_workspace(int n_tensors) { return n_tensors < 0 ? 0 : partial_bytes(n_tensors); }

static int total_of(const char* name, int device, void* stream, int n, const int* dtypes, const int64_t* numel, const void* const* in, int rooted,
                    void* out, int out_dtype, void* workspace, size_t workspace_bytes) {
    return guarded(name, [&]() -> int {
        Tensors t;
        std::string w = gather_list(n, dtypes, numel, in, nullptr, &t);
        if (w.empty()) w = wrong_norm(out, out_dtype, n, numel, dtypes, in, nullptr);
        if (w.empty()) w = wrong_workspace(workspace, out, out_dtype, n, numel, dtypes, in, nullptr);
        if (!w.empty()) return refuse(std::string(name) + ": " + w);
        OnDevice on(device);
        if (on.status != DALIB200_OK) return on.status;
        std::unique_lock<std::mutex> together(launch_mutex(), std::defer_lock);
        if (!workspace) together.lock();
        void* space = nullptr;
        const int rc = workspace_for(device, stream, partial_bytes(n), workspace, workspace_bytes, &space);
        if (rc != DALIB200_OK) return rc;
        cudaError_t e = queue_squares((cudaStream_t)stream, t, (double*)space);
        if (e == cudaSuccess)
            e = launch(total_kernel, dim3(1), kThreads, 0, (cudaStream_t)stream, 1, (const double*)space, t.partials(), rooted, out,
                       (int)(out_dtype == DALIB200_F64));
        return launched(name, e);
    });
}

extern "C" int dalib200_sum_squares(int device, void* stream, int n_tensors, const int* dtypes, const int64_t* numel,
                                    const void* const* tensors, double* sum, void* workspace, size_t workspace_bytes) {
    return total_of("dalib200_sum_squares", device, stream, n_tensors, dtypes, numel, tensors, 0, sum, DALIB200_F64, workspace, workspace_bytes);
}

extern "C" int dalib200_global_norm(int device, void* stream, int n_tensors, const int* dtypes, const int64_t* numel,
                                    const void* const* tensors, int norm_dtype, void* norm, void* workspace, size_t workspace_bytes) {
    return total_of("dalib200_global_norm", device, stream, n_tensors, dtypes, numel, tensors, 1, norm, norm_dtype, workspace, workspace_bytes);
}

int dalib::scale_to_norm(int device, void* stream, int n_tensors, const int* dtypes, const int64_t* numel, const void* const* tensors,
                         void* const* outs, const double* sum_squares, double max_norm, int norm_dtype) {
    return guarded("dalib200_scale_to_norm", [&]() -> int {
        if (!(max_norm > 0)) return refuse("dalib200_scale_to_norm: max_norm must be a number > 0");
        Tensors t;
        std::string w = n_tensors > 0 && !outs ? "outs is a null pointer" : gather_list(n_tensors, dtypes, numel, tensors, outs, &t);
        if (w.empty()) w = wrong_norm(sum_squares, DALIB200_F64, n_tensors, numel, dtypes, outs, nullptr);
        if (!w.empty()) return refuse("dalib200_scale_to_norm: " + w);
        OnDevice on(device);
        if (on.status != DALIB200_OK) return on.status;
        return launched("dalib200_scale_to_norm", queue_scale((cudaStream_t)stream, t, sum_squares, 1, max_norm, nullptr,
                                                              norm_dtype == DALIB200_F64));
    });
}

extern "C" int dalib200_scale_to_norm(int device, void* stream, int n_tensors, const int* dtypes, const int64_t* numel,
                                      const void* const* tensors, void* const* outs, const double* sum_squares, double max_norm) {
    return scale_to_norm(device, stream, n_tensors, dtypes, numel, tensors, outs, sum_squares, max_norm, DALIB200_F64);
}

extern "C" int dalib200_clip_by_global_norm(int device, void* stream, int n_tensors, const int* dtypes, const int64_t* numel,
                                            const void* const* tensors, void* const* outs, double max_norm, int norm_dtype, void* norm,
                                            void* workspace, size_t workspace_bytes) {
    return guarded("dalib200_clip_by_global_norm", [&]() -> int {
        if (!(max_norm > 0)) return refuse("dalib200_clip_by_global_norm: max_norm must be a number > 0");
        Tensors t;
        std::string w = n_tensors > 0 && !outs ? "outs is a null pointer" : gather_list(n_tensors, dtypes, numel, tensors, outs, &t);
        if (w.empty()) w = wrong_norm(norm, norm_dtype, n_tensors, numel, dtypes, tensors, outs);
        if (w.empty()) w = wrong_workspace(workspace, norm, norm_dtype, n_tensors, numel, dtypes, tensors, outs);
        if (!w.empty()) return refuse("dalib200_clip_by_global_norm: " + w);
        OnDevice on(device);
        if (on.status != DALIB200_OK) return on.status;
        std::unique_lock<std::mutex> together(launch_mutex(), std::defer_lock);
        if (!workspace) together.lock();
        void* space = nullptr;
        const int rc = workspace_for(device, stream, partial_bytes(n_tensors), workspace, workspace_bytes, &space);
        if (rc != DALIB200_OK) return rc;
        cudaError_t e = queue_squares((cudaStream_t)stream, t, (double*)space);
        if (e == cudaSuccess && t.lists.empty())
            e = launch(total_kernel, dim3(1), kThreads, 0, (cudaStream_t)stream, 1, (const double*)space, 0, 1, norm, (int)(norm_dtype == DALIB200_F64));
        else if (e == cudaSuccess)
            e = queue_scale((cudaStream_t)stream, t, (const double*)space, t.partials(), max_norm, norm, norm_dtype == DALIB200_F64);
        return launched("dalib200_clip_by_global_norm", e);
    });
}
