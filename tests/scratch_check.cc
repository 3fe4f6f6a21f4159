// Which buffers vs::StreamScratch hands out, with the runtime's calls replaced
// by the host's: 0 if a stream of each thread's own never shares one.
#include "../dart-pytorch_amd/csrc/vs_host.h"

#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <thread>

namespace vs {
int report(int code, const char *, ...) { return code; }
int report_hip(hipError_t, const char *) { return VS_ERR_OOM; }
hipError_t device_alloc(void **p, size_t bytes) {
    *p = std::malloc(bytes);
    return hipSuccess;
}
}  // namespace vs
extern "C" {
hipError_t hipFree(void *p) {
    std::free(p);
    return hipSuccess;
}
hipError_t hipGetLastError(void) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus *s) {
    *s = hipStreamCaptureStatusNone;
    return hipSuccess;
}
}

static void *take(vs::StreamScratch &s, hipStream_t st, size_t need) {
    void *p = nullptr;
    if (s.get(st, need, &p) != VS_OK) std::abort();
    return p;
}
static void *take_in_thread(vs::StreamScratch &s, hipStream_t st, size_t need) {
    void *p = nullptr;
    std::thread([&] { p = take(s, st, need); }).join();
    return p;
}

int main() {
    vs::StreamScratch s;
    int bad = 0;
    auto check = [&](bool ok, const char *what) {
        if (!ok) std::printf("%s\n", what), bad = 1;
    };
    const hipStream_t a = (hipStream_t)0x1000, b = (hipStream_t)0x2000;
    void *pa = take(s, a, 100), *pb = take(s, b, 100), *p0 = take(s, nullptr, 100);
    check(pa != pb && pa != p0 && pb != p0, "streams share a buffer");
    check(take(s, a, 100) == pa && take_in_thread(s, a, 100) == pa, "a stream's buffer changes");
    void *mine = take(s, hipStreamPerThread, 100);
    check(take(s, hipStreamPerThread, 100) == mine, "the thread's buffer changes");
    void *t1 = take_in_thread(s, hipStreamPerThread, 100);
    void *t2 = take_in_thread(s, hipStreamPerThread, 100);  // (the first thread is gone, its work may not be)
    check(t1 != mine && t2 != mine && t1 != t2, "threads' own streams share a buffer");
    void *big = take(s, a, 1 << 20);
    check(big != pa && take(s, a, 100) == big && take(s, b, 100) == pb, "growth");
    s.release();
    return bad;
}
