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

// two fp32 values, one instruction
struct Two { unsigned long long v; };
__device__ __forceinline__ Two two(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void parts(Two x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v)); }
__device__ __forceinline__ Two operator+(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Two multiply_add(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

__device__ __forceinline__ Two both(float a) { return two(a, a); }
__device__ __forceinline__ float total(Two x) {
    float a, b;
    parts(x, a, b);
    return a + b;
}
// two bf16 values of one word
__device__ __forceinline__ Two widen_pair(uint32_t w) { return two(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t narrow_pair(Two x) {
    float a, b;
    parts(x, a, b);
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// a packet of 16 bytes as pairs, and back
__device__ __forceinline__ void pairs_of(uint4 q, Two (&z)[2], const float*) {
    z[0] = two(__uint_as_float(q.x), __uint_as_float(q.y));
    z[1] = two(__uint_as_float(q.z), __uint_as_float(q.w));
}
__device__ __forceinline__ void pairs_of(uint4 q, Two (&z)[4], const bf16_s*) {
    z[0] = widen_pair(q.x);
    z[1] = widen_pair(q.y);
    z[2] = widen_pair(q.z);
    z[3] = widen_pair(q.w);
}
__device__ __forceinline__ uint4 packet_of(const Two (&z)[2], const float*) {
    uint4 q;
    float a, b, c, d;
    parts(z[0], a, b);
    parts(z[1], c, d);
    q.x = __float_as_uint(a), q.y = __float_as_uint(b), q.z = __float_as_uint(c), q.w = __float_as_uint(d);
    return q;
}
__device__ __forceinline__ uint4 packet_of(const Two (&z)[4], const bf16_s*) {
    return make_uint4(narrow_pair(z[0]), narrow_pair(z[1]), narrow_pair(z[2]), narrow_pair(z[3]));
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
