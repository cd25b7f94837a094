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

// ---------------------------------------------------------------------------------------------- simplest form
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

template <typename T>
__global__ void __launch_bounds__(kThreads) logprobs_backward_kernel(const T* logits, long long ld, long long rows, int vocab,
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

long long capped(long long want, long long most) { return std::max<long long>(1, std::min(want, most)); }

template <typename T>
cudaError_t forward(cudaStream_t s, const Rows& z, const int* tokens, void* logprob, void* entropy, void* lse, int top, void* top_logprobs,
                    int* top_tokens) {
    typedef typename AccOf<T>::type A;
    return launch(logprobs_rows_kernel<T>, dim3((unsigned)capped(z.rows, kSms * 64)), kThreads, 0, s, 1, (const T*)z.data,
                  (long long)z.stride, (long long)z.rows, (int)z.cols, tokens, (A*)logprob, (A*)entropy, (A*)lse, top, (A*)top_logprobs,
                  top_tokens);
}

template <typename T>
cudaError_t backward(cudaStream_t s, const Rows& z, const int* tokens, const void* lse, const void* entropy, const void* dlogprob,
                     const void* dentropy, const Rows& dz) {
    typedef typename AccOf<T>::type A;
    return launch(logprobs_backward_kernel<T>, dim3((unsigned)capped(z.rows, kSms * 64)), kThreads, 0, s, 1, (const T*)z.data,
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
