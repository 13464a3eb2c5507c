// State of libgen9blas_llm.so: errors, the stream of libgen9blas.so, operand checks, work buffers.
#include "llm.h"
#include <stdarg.h>
#include <stdio.h>

namespace g9llm {

static char errbuf[1200];
static int status;
hipStream_t stream;
int num_cus;
static int device = -1;

int fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(errbuf, sizeof errbuf, fmt, ap);
    va_end(ap);
    return status = code;
}

int hip_fail(hipError_t e, const char *what, const char *file, int line) {
    (void)hipGetLastError();
    return fail(e == hipErrorOutOfMemory ? GEN9BLAS_ERR_OUT_OF_MEMORY : GEN9BLAS_ERR, "%s: %s (%s:%d)", what, hipGetErrorString(e),
                file, line);
}

int begin() {
    status = 0;
    if (device < 0) {
        if (int r = gen9blas_init()) return fail(r, "%s", gen9blas_error());
        hipStream_t s = (hipStream_t)gen9blas_hip_stream();
        hipDevice_t d = 0;
        G9_HIP(hipStreamGetDevice(s, &d));
        G9_HIP(hipDeviceGetAttribute(&num_cus, hipDeviceAttributeMultiprocessorCount, d));
        stream = s;
        device = d;
    }
    int cur = -1;
    if (hipGetDevice(&cur) != hipSuccess || cur != device) G9_HIP(hipSetDevice(device));
    return 0;
}

int need_device(const void *p, size_t bytes, const char *what) {
    if (!p) G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "%s is NULL", what);
    if (!gen9blas_is_device(p, bytes))
        G9_FAIL(GEN9BLAS_ERR_INVALID_ARG, "%s (%zu bytes) is not device memory, or runs past the end of its allocation", what, bytes);
    return 0;
}

int scratch(int slot, size_t bytes, void **p) {
    static struct { void *p; size_t size; } buf[NSLOTS];
    if (buf[slot].size < bytes) {
        const size_t size = (bytes + (2u << 20) - 1) & ~(size_t)((2u << 20) - 1);
        G9_HIP(hipStreamSynchronize(stream));
        if (buf[slot].p) {
            void *old = buf[slot].p;
            buf[slot].p = nullptr;
            buf[slot].size = 0;
            G9_HIP(hipFree(old));
        }
        G9_HIP(hipMalloc(&buf[slot].p, size));
        buf[slot].size = size;
    }
    *p = buf[slot].p;
    return 0;
}

}  // namespace g9llm

extern "C" {
const char *gen9blas_llm_error(void) { return g9llm::errbuf; }
int gen9blas_llm_last_status(void) { return g9llm::status; }
}
