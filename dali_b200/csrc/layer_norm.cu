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

#include "op_device.cuh"
#include "op_host.h"

namespace dalib {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------------------------- rows of any length
// A CTA walks a row element by element, once for the mean, once for the squared deviations (a row is read again from L2), and
// once to write it.
template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) norm_rows_kernel(const T* __restrict__ x, long long ldx, const P* __restrict__ gamma,
                                                             const P* __restrict__ beta, T* y, long long ldy, long long rows,
                                                             long long cols, double eps) {
    typedef typename AccOf<T>::type A;
    __shared__ A sm[kThreads / 32];
    dependent_prologue();
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* in = x + row * ldx;
        T* out = y + row * ldy;
        A s = 0;
        for (long long c = threadIdx.x; c < cols; c += kThreads) s += widen(in[c]);
        const A mean = block_sum(s, sm) / (A)cols;
        A q = 0;
        for (long long c = threadIdx.x; c < cols; c += kThreads) {
            const A d = widen(in[c]) - mean;
            q += d * d;
        }
        const A r = (A)1 / root(block_sum(q, sm) / (A)cols + (A)eps);
        for (long long c = threadIdx.x; c < cols; c += kThreads) {
            A v = (widen(in[c]) - mean) * r;
            if (gamma) v *= widen(gamma[c]);
            if (beta) v += widen(beta[c]);
            out[c] = Narrow<T>::of(v);
        }
    }
}

// Per row: mean, r, mean(a) and r mean(a h), 4 values in `stats`.  dx is written by dx_kernel after the columns have been
// summed, so that it may be written over x or dy.
template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) row_stats_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ x,
                                                             long long ldx, const P* __restrict__ gamma, long long rows,
                                                             long long cols, double eps, typename AccOf<T>::type* __restrict__ stats) {
    typedef typename AccOf<T>::type A;
    __shared__ A sm[kThreads / 32];
    dependent_prologue();
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T* in = x + row * ldx;
        const T* up = dy + row * lddy;
        A s = 0, sa = 0;
        for (long long c = threadIdx.x; c < cols; c += kThreads) {
            s += widen(in[c]);
            sa += gamma ? widen(up[c]) * (A)widen(gamma[c]) : (A)widen(up[c]);
        }
        const A mean = block_sum(s, sm) / (A)cols;
        const A mean_a = block_sum(sa, sm) / (A)cols;
        A q = 0, qa = 0;
        for (long long c = threadIdx.x; c < cols; c += kThreads) {
            const A d = widen(in[c]) - mean;
            q += d * d;
            qa += d * (gamma ? widen(up[c]) * (A)widen(gamma[c]) : (A)widen(up[c]));
        }
        const A r = (A)1 / root(block_sum(q, sm) / (A)cols + (A)eps);
        const A mean_ah = r * (block_sum(qa, sm) / (A)cols);
        if (threadIdx.x == 0) {
            stats[4 * row] = mean;
            stats[4 * row + 1] = r;
            stats[4 * row + 2] = mean_a;
            stats[4 * row + 3] = r * mean_ah;
        }
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

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) dx_kernel(const T* dy, long long lddy, const T* x, long long ldx,
                                                      const P* __restrict__ gamma, T* dx, long long lddx, long long rows,
                                                      long long cols, const typename AccOf<T>::type* __restrict__ stats) {
    typedef typename AccOf<T>::type A;
    dependent_prologue();
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const A mean = stats[4 * row], r = stats[4 * row + 1], mean_a = stats[4 * row + 2], k = stats[4 * row + 3];
        for (long long c = threadIdx.x; c < cols; c += kThreads) {
            const A a = gamma ? widen(dy[row * lddy + c]) * (A)widen(gamma[c]) : (A)widen(dy[row * lddy + c]);
            dx[row * lddx + c] = Narrow<T>::of(r * (a - mean_a - (widen(x[row * ldx + c]) - mean) * k));
        }
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

long long capped(long long want, long long most) { return std::max<long long>(1, std::min(want, most)); }

long long column_slices(long long rows, long long cols) {
    const long long tiles = (cols + kThreads - 1) / kThreads;
    return capped((kSms * 8 + tiles - 1) / tiles, std::max<long long>(1, rows / 4));
}

struct BackwardSpace { size_t stats, partial, total; long long slices; };
BackwardSpace backward_space(int dtype, int64_t rows, int64_t cols) {
    const size_t a = dtype == DALIB200_F64 ? 8 : 4;
    BackwardSpace b;
    b.slices = column_slices(rows, cols);
    b.stats = ((size_t)rows * 4 * a + 255) / 256 * 256;
    b.partial = (size_t)b.slices * 2 * cols * a;
    b.total = b.stats + b.partial;
    return b;
}

template <typename T, typename P>
cudaError_t forward(cudaStream_t s, const Rows& x, const void* gamma, const void* beta, const Rows& y, double eps) {
    return launch(norm_rows_kernel<T, P>, dim3((unsigned)capped(x.rows, kSms * 64)), kThreads, 0, s, 1, (const T*)x.data,
                  (long long)x.stride, (const P*)gamma, (const P*)beta, (T*)y.data, (long long)y.stride, (long long)x.rows,
                  (long long)x.cols, eps);
}

template <typename T, typename P>
cudaError_t backward(cudaStream_t s, const Rows& dy, const Rows& x, const void* gamma, const Rows& dx, void* dgamma, void* dbeta,
                     double eps, void* space) {
    typedef typename AccOf<T>::type A;
    const BackwardSpace b = backward_space(sizeof(T) == 8 ? DALIB200_F64 : DALIB200_F32, x.rows, x.cols);
    A* stats = (A*)space;
    A* partial = (A*)((char*)space + b.stats);
    const dim3 by_row((unsigned)capped(x.rows, kSms * 64));
    cudaError_t e = launch(row_stats_kernel<T, P>, by_row, kThreads, 0, s, 1, (const T*)dy.data, (long long)dy.stride, (const T*)x.data,
                           (long long)x.stride, (const P*)gamma, (long long)x.rows, (long long)x.cols, eps, stats);
    if (e == cudaSuccess && (dgamma || dbeta)) {
        e = launch(column_sums_kernel<T>, dim3((unsigned)((x.cols + kThreads - 1) / kThreads), (unsigned)b.slices), kThreads, 0, s, 1,
                   (const T*)dy.data, (long long)dy.stride, (const T*)x.data, (long long)x.stride, (long long)x.rows,
                   (long long)x.cols, (const A*)stats, partial);
        if (e == cudaSuccess)
            e = launch(fold_columns_kernel<A, P>, dim3((unsigned)((x.cols + 31) / 32), 2), kThreads, 0, s, 1, (const A*)partial, b.slices,
                       (long long)x.cols, (P*)dgamma, (P*)dbeta);
    }
    if (e == cudaSuccess && dx.data)
        e = launch(dx_kernel<T, P>, by_row, kThreads, 0, s, 1, (const T*)dy.data, (long long)dy.stride, (const T*)x.data,
                   (long long)x.stride, (const P*)gamma, (T*)dx.data, (long long)dx.stride, (long long)x.rows, (long long)x.cols,
                   (const A*)stats);
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
        const BackwardSpace need = backward_space(dtype, rows, cols);
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
        OnDevice on(device);
        if (on.status != DALIB200_OK) return on.status;
        std::unique_lock<std::mutex> together(launch_mutex(), std::defer_lock);
        if (!workspace) together.lock();
        void* space = nullptr;
        if ((rc = workspace_for(device, stream, need.total, workspace, workspace_bytes, &space)) != DALIB200_OK) return rc;
        cudaError_t e;
        if (dtype == DALIB200_F32) e = backward<float, float>(s, mdy, mx, gamma, mdx, dgamma, dbeta, eps, space);
        else if (dtype == DALIB200_F64) e = backward<double, double>(s, mdy, mx, gamma, mdx, dgamma, dbeta, eps, space);
        else if (param_dtype == DALIB200_F32) e = backward<bf16_s, float>(s, mdy, mx, gamma, mdx, dgamma, dbeta, eps, space);
        else e = backward<bf16_s, bf16_s>(s, mdy, mx, gamma, mdx, dgamma, dbeta, eps, space);
        return launched(what, e);
    });
}
