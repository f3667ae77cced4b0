// dev_entry.cuh — what the C entries of the operators on device tensors share: refusals, the device of a call, the choice among types.
#pragma once
#include "device_ops.h"

#include <algorithm>
#include <exception>
#include <string>

#include "dev_common.cuh"

namespace dev {

inline int bad(const char* op, const char* what) { return dev_fail(B200_ERR_INVALID_ARGUMENT, (std::string(op) + ": " + what).c_str()); }
inline int shape(const char* op, const char* what) { return dev_fail(B200_ERR_SHAPE_MISMATCH, (std::string(op) + ": " + what).c_str()); }
inline bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
// Whether rows of an output, hd elements each, may lie on one another: they do not where all heads of a token are between one token and the next, or all tokens of a head between one head and the next.
inline bool overlap(int64_t tokens, int64_t token, int64_t heads, int64_t head, int64_t hd) {
    if (tokens <= 1 || heads <= 1) return (tokens > 1 && token < hd) || (heads > 1 && head < hd);
    const int64_t n = token < head ? tokens : heads, inner = std::min(token, head), outer = std::max(token, head);
    return inner < hd || (outer - hd) / (n - 1) < inner;
}
inline int type_bytes(uint32_t t) { return t == B200_TYPE_F32 ? 4 : t == B200_TYPE_F16 || t == B200_TYPE_BF16 ? 2 : 0; }
inline int bad_type(const char* op, uint32_t t) {
    return dev_fail(B200_ERR_UNSUPPORTED_DTYPE, (std::string(op) + ": type " + std::to_string(t) + " (F32, F16 and BF16 only)").c_str());
}
constexpr int64_t kMost = (int64_t)1 << 31;      // grids and 32-bit counts
constexpr int64_t kMostTiled = kMost - (1 << 20);      // ... that a last tile may go beyond

// No exception crosses the C boundary.
template <typename F> int entry(const char* op, F&& body) {
    try {
        return body();
    } catch (const std::exception& e) {
        return dev_fail(B200_ERR_OPERATION_FAILED, e.what());
    } catch (...) {
        return dev_fail(B200_ERR_OPERATION_FAILED, op);
    }
}
// The work of a call on its device; the caller's current device comes back afterwards.
template <typename F> int on_device(const char* op, int device, F&& launch) {
    int n = 0, was = -1;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
        cudaGetLastError();
        return dev_fail(B200_ERR_NOT_AVAILABLE, "cuda-b200: no CUDA device (this backend has no CPU fallback)");
    }
    if (device < 0 || device >= n) return bad(op, "no such device");
    cudaError_t e = cudaGetDevice(&was);
    if (e == cudaSuccess && was != device) e = cudaSetDevice(device);
    if (e == cudaSuccess) e = launch();
    if (was >= 0 && was != device) cudaSetDevice(was);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return dev_fail(B200_ERR_OPERATION_FAILED, (std::string(op) + ": " + cudaGetErrorString(e)).c_str());
    }
    return B200_OK;
}
template <typename F> cudaError_t by_type(uint32_t t, F&& f) {
    return t == B200_TYPE_F32 ? f(float{}) : t == B200_TYPE_F16 ? f(__half{}) : f(__nv_bfloat16{});
}

}  // namespace dev
