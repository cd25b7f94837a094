// Workspaces of the hand-written operators (op_host.h).
#include "op_host.h"

#include <algorithm>
#include <map>
#include <utility>

namespace dalib {

std::mutex& launch_mutex() {
    static std::mutex* m = new std::mutex();
    return *m;
}

namespace {
struct Space { void* data = nullptr; size_t bytes = 0; unsigned long long stream_id = 0, last_call = 0; };
// What a device's blocks may take together (128 streams of 4 MB).  Beyond that the one whose last call is the longest ago goes
// first: nothing says which of the streams are still there.
constexpr size_t kKept = 512u << 20;
// apart from the exchange space of generated kernels: those are queued without the launch mutex
std::map<std::pair<int, void*>, Space>& spaces() {
    static auto* m = new std::map<std::pair<int, void*>, Space>();
    return *m;
}

void drop_oldest(int device, const Space& but) {
    for (;;) {
        size_t bytes = 0;
        auto oldest = spaces().end();
        for (auto i = spaces().begin(); i != spaces().end(); ++i) {
            if (i->first.first != device) continue;
            bytes += i->second.bytes;
            if (&i->second != &but && (oldest == spaces().end() || i->second.last_call < oldest->second.last_call)) oldest = i;
        }
        if (bytes <= kKept || oldest == spaces().end()) return;
        if (oldest->second.data) cudaFree(oldest->second.data);          // (waits for the device)
        spaces().erase(oldest);
    }
}
}  // namespace

int workspace_for(int device, void* stream, size_t need, void* given, size_t given_bytes, void** out) {
    if (given) {
        if (given_bytes < need) return refuse("workspace of " + std::to_string(given_bytes) + " bytes, " + std::to_string(need) + " are needed");
        if ((uintptr_t)given % 16) return refuse("workspace is not 16-byte aligned");
        *out = given;
        return DALIB200_OK;
    }
    if ((cudaStream_t)stream == cudaStreamPerThread) return refuse("a call on the per-thread default stream needs a workspace of its own");
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    const cudaError_t asked = cudaStreamIsCapturing((cudaStream_t)stream, &st);
    if (asked != cudaSuccess || st != cudaStreamCaptureStatusNone) {
        cudaGetLastError();
        return refuse("a call that is captured into a graph needs a workspace of its own");
    }
    // a stream made where a destroyed one lay has another id, and kernels of the destroyed one may still be running
    unsigned long long id = 0;
    if (cudaStreamGetId((cudaStream_t)stream, &id) != cudaSuccess) cudaGetLastError();
    static unsigned long long calls = 0;
    Space& s = spaces()[std::make_pair(device, stream)];
    s.last_call = ++calls;
    if (s.bytes < need || s.stream_id != id) {
        // (kernels in flight may still use the old block: cudaFree waits for the device)
        const size_t bytes = std::max<size_t>(need, 4u << 20);
        void* fresh = nullptr;
        const cudaError_t e = cudaMalloc(&fresh, bytes);
        if (e != cudaSuccess) {
            cudaGetLastError();
            set_error(std::string("workspace: cudaMalloc: ") + cudaGetErrorString(e));
            return DALIB200_ERR_CUDA;
        }
        if (s.data) cudaFree(s.data);
        s.data = fresh;
        s.bytes = bytes;
        s.stream_id = id;
        drop_oldest(device, s);
    }
    *out = s.data;
    return DALIB200_OK;
}

}  // namespace dalib
