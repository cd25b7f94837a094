// Device helpers shared by the hand-written operators (layer_norm.cu, token_logprobs.cu, clip_norm.cu): element types and
// their accumulators, 16-byte packets, warp folds and the hand-over between dependent launches.
#ifndef DALI_B200_CSRC_OP_DEVICE_CUH
#define DALI_B200_CSRC_OP_DEVICE_CUH

#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

namespace dalib {

// bf16 is a storage type here as everywhere in the library: loads widen to fp32 exactly, stores round to nearest even.
struct bf16_s { uint16_t bits; };

template <typename T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ double widen(double x) { return x; }
__device__ __forceinline__ float widen(bf16_s x) { return __uint_as_float((uint32_t)x.bits << 16); }

template <typename T> struct Narrow;
template <> struct Narrow<float> { static __device__ __forceinline__ float of(float x) { return x; } };
template <> struct Narrow<double> { static __device__ __forceinline__ double of(double x) { return x; } };
template <> struct Narrow<bf16_s> {
    static __device__ __forceinline__ bf16_s of(float x) {
        bf16_s r;
        asm("cvt.rn.bf16.f32 %0, %1;" : "=h"(r.bits) : "f"(x));
        return r;
    }
};

// 16 bytes of T, loaded and stored as one 128-bit access
template <typename T> struct alignas(16) Packet {
    static constexpr int N = 16 / (int)sizeof(T);
    T v[N];
};
template <typename T> __device__ __forceinline__ Packet<T> load_packet(const T* p) {
    Packet<T> r;
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
    return r;
}
template <typename T> __device__ __forceinline__ void store_packet(T* p, const Packet<T>& v) {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&v);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// Sum over the threads of a CTA, the same bits in every thread (warps are folded in warp order).  `sm`: one value per warp;
// the leading barrier lets the caller use it again at once.
template <typename A>
__device__ __forceinline__ A block_sum(A v, A* sm) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = v;
    __syncthreads();
    A r = 0;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) r += sm[w];
    return r;
}

__device__ __forceinline__ float root(float x) { return sqrtf(x); }
__device__ __forceinline__ double root(double x) { return sqrt(x); }

// A kernel launched as the programmatic dependent of its predecessor in the stream must not touch global memory before the
// predecessor has finished; it lets its own successor be set up at once.
__device__ __forceinline__ void dependent_prologue() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

}  // namespace dalib
#endif
