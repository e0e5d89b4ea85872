// What capi.hip lends the entry points of other files: the process-wide call
// lock with the ordering of calls, errors, the cached workspace, timing.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace mlrs {
namespace capi {

// Runs body(ctx) as one entry-point call.
int32_t run_call(int32_t (*body)(void*), void* ctx);
template <typename F>
int32_t call(F&& f) {
    return run_call([](void* p) -> int32_t { return (*static_cast<F*>(p))(); }, &f);
}

int32_t error(int32_t code, const char* operand, int64_t rows, int64_t cols, int64_t len, const char* message);
int32_t shape_error(const char* operand, int64_t rows, int64_t cols, int64_t len);
int32_t hip_error(hipError_t e, const char* where);
// rows * cols == len without overflow
bool geometry(int64_t rows, int64_t cols, int64_t len);

// `bytes` of the device's cached workspace, after the last call's work on it.
int32_t scratch(size_t bytes, hipStream_t s, char** out, int* cus);
int32_t cu_count(int* cus);

// Events around a call's dominant launches (mlrs_timing_enable).
struct Timed {
    Timed(hipStream_t s, const char* name);
    ~Timed();
    Timed(const Timed&) = delete;
    Timed& operator=(const Timed&) = delete;
    alignas(16) char room[64];
};

}  // namespace capi
}  // namespace mlrs
