// What serving.cpp calls of the HIP runtime and of the kernels' launchers, on the host: memory
// from malloc, one call of a kind made to fail on request, launches recorded and not made.
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "ctx.hpp"
#include "paged.hpp"

static int g_fail_memset = 0;
static long g_live = 0, g_launches = 0;
static int g_sample_parts = 0;
static char g_message[512];

extern "C" {
hipError_t hipMalloc(void** p, size_t n) {
    *p = aligned_alloc(256, (n + 255) / 256 * 256);
    memset(*p, 0xAB, n);
    ++g_live;
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    if (p) --g_live;
    free(p);
    return hipSuccess;
}
hipError_t hipMemsetAsync(void* p, int v, size_t n, hipStream_t) {
    if (g_fail_memset > 0 && g_fail_memset-- == 1) return hipErrorUnknown;
    memset(p, v, n);
    return hipSuccess;
}
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t, hipStreamCaptureStatus* s) {
    *s = hipStreamCaptureStatusNone;
    return hipSuccess;
}
hipError_t hipSetDevice(int) { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return "made to fail"; }

m1moe_ctx_t stub_ctx(void) {
    m1moe_ctx* c = new m1moe_ctx();
    c->cus = 256;
    return c;
}
void stub_free(m1moe_ctx_t c) {
    for (void* p : {(void*)c->paged_part, (void*)c->paged_cnt, (void*)c->sample_part}) (void)hipFree(p);
    delete c;
}
void stub_fail_memset(int nth) { g_fail_memset = nth; }
long stub_live(void) { return g_live; }
long stub_launches(void) { return g_launches; }
int stub_sample_parts(void) { return g_sample_parts; }
const char* stub_message(void) { return g_message; }
}

namespace m1moe {
int32_t fail(int32_t code, const char* fmt, ...) {
    va_list a;
    va_start(a, fmt);
    vsnprintf(g_message, sizeof g_message, fmt, a);
    va_end(a);
    return code;
}
static int launch(const void* zeroed, size_t words) {
    for (size_t i = 0; i < words; ++i)
        if (static_cast<const uint32_t*>(zeroed)[i]) abort();   // counters that were never cleared
    ++g_launches;
    return 0;
}
int launch_kv_append(const AppendArgs&, int, void*) { return launch(nullptr, 0); }
int64_t paged_attention_plan(PagedAttnArgs& a, int cus, int64_t* own) {
    a.grid = 2 * cus;
    return *own = 1000;
}
int launch_paged_attention(const PagedAttnArgs& a, void*) { return launch(a.counters, a.grid); }
int sample_parts(int, int, int) { return 4; }
int64_t sample_part_words(int cus) { return (int64_t)cus * 7; }
int launch_sample(const SampleArgs& a, void*) {
    g_sample_parts = a.parts;
    return launch(a.counters, a.parts > 1 ? a.rows : 0);
}
}  // namespace m1moe
