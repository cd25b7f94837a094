// Host side shared by the entry points of the hand-written operators: argument checks, workspaces, launches.
#ifndef DALI_B200_CSRC_OP_HOST_H
#define DALI_B200_CSRC_OP_HOST_H

#include <cuda_runtime.h>

#include <cstdint>
#include <exception>
#include <mutex>
#include <string>

#include "../../include/dali_b200.h"
#include "runtime.h"

namespace dalib {

constexpr int kSms = 148;      // streaming multiprocessors of the one GPU this library is written for

inline int refuse(const std::string& what) {
    set_error(what);
    return DALIB200_ERR_INVALID;
}
inline int size_of(int dtype) { return dtype == DALIB200_F64 ? 8 : dtype == DALIB200_BF16 ? 2 : 4; }
inline bool floating(int dtype) { return dtype == DALIB200_F32 || dtype == DALIB200_F64 || dtype == DALIB200_BF16; }

// Makes `device` current for the duration of an entry point (the caller's current device comes back with `restore`).
struct OnDevice {
    DeviceRestore restore;
    int status;
    explicit OnDevice(int device) : status(DALIB200_OK) {
        const int ord = device_ordinal(device);
        if (ord < 0) {
            set_error("device index out of range");
            status = dalib200_device_count() ? DALIB200_ERR_INVALID : DALIB200_ERR_NO_DEVICE;
            return;
        }
        const cudaError_t e = cudaSetDevice(ord);
        if (e != cudaSuccess) { set_error(std::string("cudaSetDevice: ") + cudaGetErrorString(e)); status = DALIB200_ERR_CUDA; }
    }
};

// A row-major matrix as an entry point receives it.
struct Rows {
    const char* name;
    const void* data;
    int64_t rows, cols, stride;     // elements
    int size;                       // bytes of an element
    const char* begin() const { return static_cast<const char*>(data); }
    const char* end() const { return begin() + ((rows - 1) * stride + cols) * size; }
};

// "" or what is wrong with the matrix on its own
inline std::string wrong(const Rows& m) {
    if (!m.data) return std::string(m.name) + " is a null pointer";
    if ((uintptr_t)m.data % m.size) return std::string(m.name) + " is not aligned to its elements";
    if (m.rows > 1 && m.stride < m.cols) return std::string("the row stride of ") + m.name + " is shorter than a row";
    if (m.stride < 0 || m.stride > (int64_t(1) << 40)) return std::string("the row stride of ") + m.name + " is out of range";
    return "";
}

// Do a read and a written matrix of the same rows x cols share an element, other than by being the same matrix (which the
// operators allow: every element is read before the thread that read it writes it)?
inline bool clash(const Rows& in, const Rows& out) {
    if (in.rows == 0 || in.cols == 0 || in.end() <= out.begin() || out.end() <= in.begin()) return false;
    if (in.data == out.data && in.size == out.size && (in.rows == 1 || in.stride == out.stride)) return false;
    if (in.size == out.size && in.rows > 1 && in.stride == out.stride && (out.begin() - in.begin()) % in.size == 0) {
        // two column blocks of one wider matrix
        int64_t d = (out.begin() - in.begin()) / in.size % in.stride;
        if (d < 0) d += in.stride;
        if (d >= in.cols && d + in.cols <= in.stride) return false;
    }
    return true;
}

inline bool meets(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    const char *x = static_cast<const char*>(a), *y = static_cast<const char*>(b);
    return a && b && x < y + b_bytes && y < x + a_bytes;
}

// The caller's workspace, or space of the library's own for (device, stream), which operators that need more than one launch
// pass their partial results through (op_host.cc).  The latter is handed to the next call on that stream (and kept for it, up
// to 512 MB a device over all streams), so a captured
// call, whose graph may be replayed beside anything, has to bring its own, and so has one on the per-thread default stream,
// whose one handle stands for several streams.  Without a caller's workspace the launches of a call stay together under
// launch_mutex(), so that two threads that share a stream do not mix their partial results.
int workspace_for(int device, void* stream, size_t need, void* given, size_t given_bytes, void** out);
std::mutex& launch_mutex();

// Launches as the programmatic dependent of what precedes it in the stream (the kernel starts with dependent_prologue).
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, unsigned cluster, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (dependent_launch_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    if (e == cudaSuccess) count_launch();
    return e;
}

inline int launched(const char* what, cudaError_t e) {
    if (e == cudaSuccess) return DALIB200_OK;
    set_error(std::string(what) + ": " + cudaGetErrorString(e));
    return DALIB200_ERR_CUDA;
}

// dalib200_scale_to_norm for a norm that is reported in norm_dtype: one that is not finite there scales nothing (clip_norm.cu).
int scale_to_norm(int device, void* stream, int n_tensors, const int* dtypes, const int64_t* numel, const void* const* tensors,
                  void* const* outs, const double* sum_squares, double max_norm, int norm_dtype);

// No C++ exception leaves a C entry point.
template <typename F>
int guarded(const char* what, F f) {
    try {
        return f();
    } catch (const std::exception& e) {
        set_error(std::string(what) + ": " + e.what());
        return DALIB200_ERR_INVALID;
    } catch (...) {
        set_error(std::string(what) + ": unknown exception");
        return DALIB200_ERR_INVALID;
    }
}

}  // namespace dalib
#endif
