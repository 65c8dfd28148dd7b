// What the host sides of the 8-bit operators share: the handle, errors, checks of
// arguments, the workspace.
#pragma once

#include "q8_internal.hpp"
#include "sgemm_internal.hpp"

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <new>

struct q8_handle {
    struct Retired {
        void* memory;
        Retired* next;
    };
    int device = 0;
    hipStream_t stream = nullptr;
    hipStream_t own_stream = nullptr;
    char* workspace = nullptr;
    size_t workspace_bytes = 0;
    Retired* retired = nullptr;    // workspaces that captured calls may still use
    bool captured = false;         // a call that used the workspace was captured
    uint32_t* tickets = nullptr;   // kTickets zeros of device memory, zeros again after each launch that uses them
};

namespace q8 {

inline int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
inline int fail(int code, const char* fmt, ...) {
    char msg[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(msg, sizeof(msg), fmt, ap);
    va_end(ap);
    return sgemm_internal::set_error(code, msg);
}
inline int hip_fail(hipError_t e, const char* what) { return fail((int)e, "%s: %s (%d)", what, hipGetErrorString(e), (int)e); }
inline int launched(hipError_t e, const char* what) { return e == hipSuccess ? SGEMM_OK : hip_fail(e, what); }

#define HIP_TRY(call)                                      \
    do {                                                   \
        const hipError_t e_ = (call);                      \
        if (e_ != hipSuccess) return hip_fail(e_, #call);  \
    } while (0)
#define CHECK(call)                       \
    do {                                  \
        const int c_ = (call);            \
        if (c_ != SGEMM_OK) return c_;    \
    } while (0)

// The handle's device is current while a call runs.
class OnDevice {
public:
    explicit OnDevice(int device) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = device;
        if (before_ != device) status_ = hipSetDevice(device);
        device_ = device;
    }
    ~OnDevice() {
        if (before_ != device_) (void)hipSetDevice(before_);
    }
    hipError_t status() const { return status_; }

private:
    int before_ = 0, device_ = 0;
    hipError_t status_ = hipSuccess;
};

inline bool capturing(hipStream_t stream) {
    hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
    return hipStreamIsCapturing(stream, &s) != hipSuccess || s != hipStreamCaptureStatusNone;
}

// While it lives, this thread's allocations are none of other streams' captures, which they would end.
class BesideCaptures {
public:
    BesideCaptures() { (void)hipThreadExchangeStreamCaptureMode(&mode_); }
    ~BesideCaptures() { (void)hipThreadExchangeStreamCaptureMode(&mode_); }
    BesideCaptures(const BesideCaptures&) = delete;
    BesideCaptures& operator=(const BesideCaptures&) = delete;

private:
    hipStreamCaptureMode mode_ = hipStreamCaptureModeRelaxed;      // then the thread's own
};

inline bool is_type(int dtype) { return dtype == Q8_F32 || dtype == Q8_F16 || dtype == Q8_BF16; }

// A matrix argument: rows of cols values at ld, `bytes` each.
struct Span {
    const char* name;
    const void* p;
    uint64_t rows, cols, ld;
    uint32_t bytes;
};
inline int check(const Span& s) {
    if (!s.rows || !s.cols) return SGEMM_OK;
    if (!s.p) return fail(SGEMM_E_INVALID, "%s is null", s.name);
    if ((uintptr_t)s.p % s.bytes) return fail(SGEMM_E_INVALID, "%s is not aligned to its %u-byte values", s.name, s.bytes);
    if (s.ld < s.cols)
        return fail(SGEMM_E_SHAPE, "%s: leading dimension %llu below its %llu columns", s.name, (unsigned long long)s.ld,
                    (unsigned long long)s.cols);
    return SGEMM_OK;
}
// Whether two matrices share a byte.  Windows of different columns of one buffer
// (the same ld) do not.
inline bool overlap(const Span& a, const Span& b) {
    if (!a.p || !b.p || !a.rows || !a.cols || !b.rows || !b.cols) return false;
    const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
    const uint64_t la = a.ld * a.bytes, lb = b.ld * b.bytes;
    const uint64_t a1 = a0 + (a.rows - 1) * la + a.cols * a.bytes, b1 = b0 + (b.rows - 1) * lb + b.cols * b.bytes;
    if (a1 <= b0 || b1 <= a0) return false;
    if (la != lb) return true;
    const uint64_t d = a0 <= b0 ? (b0 - a0) % la : (la - (a0 - b0) % la) % la;   // b's first column in a's rows
    return d < a.cols * a.bytes || d + b.cols * b.bytes > la;
}
inline bool same(const Span& a, const Span& b) { return a.p == b.p && a.ld == b.ld && a.bytes == b.bytes; }
inline int check_apart(const Span& out, const Span& in, bool in_place = false) {
    if (in_place && same(out, in)) return SGEMM_OK;
    if (overlap(out, in)) return fail(SGEMM_E_INVALID, "%s overlaps %s", out.name, in.name);
    return SGEMM_OK;
}
inline Span vec(const char* name, const void* p, uint64_t count, uint32_t bytes) { return Span{name, p, 1, count, count, bytes}; }

inline int grow(q8_handle* h, size_t bytes) {
    if (bytes <= h->workspace_bytes) return SGEMM_OK;
    if (capturing(h->stream))
        return fail(SGEMM_E_SHAPE, "a workspace of %zu bytes is needed and %zu are there: under graph capture it cannot grow "
                                   "(q8_reserve beforehand)", bytes, h->workspace_bytes);
    constexpr size_t kStep = (size_t)2 << 20;
    if (bytes > SIZE_MAX - kStep) return hip_fail(hipErrorOutOfMemory, "workspace");    // rounded up it would pass 0
    const size_t want = (bytes + kStep - 1) / kStep * kStep;
    HIP_TRY(hipStreamSynchronize(h->stream));
    if (h->workspace && h->captured) {
        // a captured call may be replayed: its workspace stays until the handle goes
        q8_handle::Retired* r = new (std::nothrow) q8_handle::Retired{h->workspace, h->retired};
        if (!r) return fail(SGEMM_E_SHAPE, "out of host memory");
        h->retired = r;
    } else if (h->workspace) {
        HIP_TRY(hipFree(h->workspace));
    }
    h->workspace = nullptr;
    h->workspace_bytes = 0;
    void* p = nullptr;
    HIP_TRY(hipMalloc(&p, want));
    h->workspace = static_cast<char*>(p);
    h->workspace_bytes = want;
    return SGEMM_OK;
}
inline int take_workspace(q8_handle* h, size_t bytes) {
    if (!bytes) return SGEMM_OK;
    CHECK(grow(h, bytes));
    if (!h->captured && capturing(h->stream)) h->captured = true;
    return SGEMM_OK;
}

inline int check_handle(const q8_handle* h) { return h ? SGEMM_OK : fail(SGEMM_E_INVALID, "the handle is null"); }
inline int check_type(int dtype) { return is_type(dtype) ? SGEMM_OK : fail(SGEMM_E_INVALID, "%d is no type", dtype); }

}  // namespace q8
