// vs_host.h -- host helpers shared by the sources that hold entry points.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <new>
#include <vector>

#include "../../include/vs_hip.h"

namespace vs {

// Sets the calling thread's error text and returns `code`.
int report(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
// The same for a failed runtime call.
int report_hip(hipError_t e, const char *what);
// hipMalloc that takes idle row copies of indexes back when the device is full.
hipError_t device_alloc(void **p, size_t bytes);

// Restores the caller's current device on scope exit.
struct DeviceGuard {
    int prev = -1, dev;
    hipError_t err = hipSuccess;
    explicit DeviceGuard(int device) : dev(device) {
        if (hipGetDevice(&prev) != hipSuccess) prev = -1;
        if (prev != dev) err = hipSetDevice(dev);
    }
    ~DeviceGuard() {
        if (prev >= 0 && prev != dev) (void)hipSetDevice(prev);
    }
};

// A number of the calling thread's own, never given to another.
inline uint64_t thread_number() {
    static std::atomic<uint64_t> last{0};
    thread_local const uint64_t mine = ++last;
    return mine;
}

// Scratch memory of a handle, one buffer per stream, so that calls on
// different streams never share one.  hipStreamPerThread is one name for a
// stream of each thread's own, so there the thread counts too.  A buffer that
// is outgrown is kept until the handle ends: a recorded graph may still use it.
struct StreamScratch {
    struct Buf {
        hipStream_t st;
        uint64_t thread;  // 0: the stream is the same for all
        void *p;
        size_t bytes;
    };
    std::vector<Buf> bufs;

    int get(hipStream_t st, size_t need, void **out) {
        const uint64_t thread = st == hipStreamPerThread ? thread_number() : 0;
        for (auto it = bufs.rbegin(); it != bufs.rend(); ++it)
            if (it->st == st && it->thread == thread) {
                if (it->bytes < need) break;
                *out = it->p;
                return VS_OK;
            }
        hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
        if (hipStreamIsCapturing(st, &cap) != hipSuccess) {
            (void)hipGetLastError();
            cap = hipStreamCaptureStatusNone;
        }
        if (cap != hipStreamCaptureStatusNone)
            return report(VS_ERR_UNSUPPORTED,
                          "scratch memory has to grow: run this call once before recording it");
        size_t bytes = 1 << 16;
        while (bytes < need) bytes *= 2;
        void *p = nullptr;
        hipError_t e = device_alloc(&p, bytes);
        if (e != hipSuccess) return report_hip(e, "scratch memory");
        try {
            bufs.push_back({st, thread, p, bytes});
        } catch (const std::bad_alloc &) {
            (void)hipFree(p);
            return report(VS_ERR_OOM, "host allocation");
        }
        *out = p;
        return VS_OK;
    }
    void release() {
        for (auto &b : bufs) (void)hipFree(b.p);
        bufs.clear();
    }
};

// Whether [a, a + na) and [b, b + nb) share a byte.
inline bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    return a && b && (const char *)a < (const char *)b + nb && (const char *)b < (const char *)a + na;
}

// Rows of `heads` heads of dim elements of e bytes, wherever the strides (in
// elements) put them: the bytes from the first to the last, and what is between.
struct Extent {
    const char *low;
    int64_t bytes, width;  // width: of one head of one row
    int64_t n[2], s[2];    // how many rows and heads, and how far apart, upwards
    Extent(const void *p, int64_t row, int64_t head, int64_t nrows, int64_t heads, int64_t dim,
           int64_t e)
        : low((const char *)p), width(dim * e), n{nrows, heads}, s{row * e, head * e} {
        bytes = width;
        for (int i = 0; i < 2; ++i) {
            if (s[i] < 0) low += (n[i] - 1) * s[i], s[i] = -s[i];
            bytes += (n[i] - 1) * s[i];
        }
    }
    // Its bytes lie in the first span(period) of every `period` from low on.
    int64_t span(int64_t period) const {
        int64_t x = width;
        for (int i = 0; i < 2; ++i)
            if (s[i] % period) x += (n[i] - 1) * s[i];
        return x;
    }
};

// Whether they may share a byte.  Parts of one projection's output do not: what comes
// again after the same stretch, side by side within it, be it rows or heads, or the
// heads of rows that do.
inline bool meet(const Extent &a, const Extent &b) {
    if (!overlap(a.low, a.bytes, b.low, b.bytes)) return false;
    auto apart = [&](int64_t period) {
        const int64_t d = (int64_t)((uintptr_t)b.low - (uintptr_t)a.low) % period;
        return d < 0 ? d + period : d;
    };
    for (const Extent *x : {&a, &b})
        for (int i = 0; i < 2; ++i) {
            const int64_t period = x->s[i];
            if (x->n[i] < 2 || period == 0) continue;
            const int64_t d = apart(period);
            if (d >= a.span(period) && period - d >= b.span(period)) return false;
        }
    for (int i = 0; i < 2; ++i) {
        const int64_t period = a.s[i];
        if (a.n[i] < 2 || b.n[i] < 2 || period == 0 || b.s[i] != period) continue;
        Extent x = a, y = b;  // one of each, which no other repetition reaches into
        x.n[i] = y.n[i] = 1;
        x.bytes -= (a.n[i] - 1) * period;
        y.bytes -= (b.n[i] - 1) * period;
        if (x.bytes > period || y.bytes > period) continue;
        y.low = x.low + apart(period);
        if (meet(x, y)) return true;
        y.low -= period;
        return meet(x, y);
    }
    return true;
}

// A launch of so many workgroups: the runtime counts a grid's threads in 32 bits.
inline bool grid_ok(int64_t workgroups, int threads) { return workgroups <= UINT32_MAX / threads; }

// The device exists; VS_OK or the error.
inline int check_device(int device) {
    int count = 0;
    if (hipGetDeviceCount(&count) != hipSuccess || count <= 0)
        return report(VS_ERR_NO_DEVICE, "no HIP device visible");
    if (device < 0 || device >= count)
        return report(VS_ERR_INVALID, "device %d out of range [0, %d)", device, count);
    return VS_OK;
}

inline int cu_count(int device) {
    int n = 0;
    return hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) == hipSuccess &&
                   n > 0
               ? n
               : 256;
}

}  // namespace vs
