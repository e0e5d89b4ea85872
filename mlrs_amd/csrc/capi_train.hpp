// What the entry points of the training operators share.
#pragma once
#include <hip/hip_runtime.h>

#include <initializer_list>

#include "../../include/mlrs_hip_knn.h"
#include "capi_shared.hpp"

namespace mlrs {
namespace train {

inline int32_t null_error(const char* operand) {
    return capi::error(MLRS_ERR_NULL_POINTER, operand, 0, 0, 0, "null pointer");
}

// Carves a call's scratch: first a pass that only adds up, then one that hands
// out addresses.
struct Scratch {
    char* base = nullptr;
    size_t used = 0;
    template <typename T>
    T* take(size_t n) {
        used = (used + 255) & ~(size_t)255;
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += n * sizeof(T);
        return p;
    }
};

// What a call writes may be no part of what it reads or else writes: workgroups
// read operands while others write results.
struct Span {
    const void* p;
    int64_t bytes;
    template <typename T>
    Span(const T* t, int64_t len) : p(t), bytes(t ? len * (int64_t)sizeof(T) : 0) {}
    bool meets(const Span& o) const {
        const uintptr_t a = (uintptr_t)p, b = (uintptr_t)o.p;
        return bytes > 0 && o.bytes > 0 && a < b + (uintptr_t)o.bytes && b < a + (uintptr_t)bytes;
    }
    bool meets(std::initializer_list<Span> others) const {
        for (const Span& o : others)
            if (meets(o)) return true;
        return false;
    }
};
inline int32_t overlap_error(const char* out) {
    return capi::error(MLRS_ERR_INVALID_PARAM, out, 0, 0, 0, "an output overlaps another operand");
}

// The workspace, of a call that is not being captured into a graph: the library's
// calls share it, in the order in which they are made, and a replay has no place
// in that order.
inline int32_t eager_scratch(size_t bytes, hipStream_t s, char** out, int* cus) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if (s && hipStreamIsCapturing(s, &status) == hipSuccess && status != hipStreamCaptureStatusNone)
        return capi::error(MLRS_ERR_UNSUPPORTED, "stream", 0, 0, (int64_t)bytes,
                           "a call that takes the library's workspace cannot be captured into a graph");
    return capi::scratch(bytes, s, out, cus);
}

}  // namespace train
}  // namespace mlrs

#define MLRS_TRY(call)                                      \
    do {                                                    \
        const hipError_t e_ = (call);                       \
        if (e_ != hipSuccess) return capi::hip_error(e_, where); \
    } while (0)
