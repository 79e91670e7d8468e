/* The calls of the HIP runtime that a context and the training operators make, without a GPU: two devices, streams and events as plain
 * numbers, launches and waits written into a log.  Loaded in front of the library (RTLD_GLOBAL), it takes the runtime's place. */
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

typedef struct { uint32_t x, y, z; } dim3;

static int device = 0;
static uintptr_t events = 0, capturing = 0, pushed = 0;
static char text[1 << 16];

static void note(const char* what, uintptr_t a, uintptr_t b) {
    size_t n = strlen(text);
    snprintf(text + n, sizeof text - n, "%s %lu %lu\n", what, (unsigned long)a, (unsigned long)b);
}
const char* fake_log(void) { return text; }
void fake_clear(void) { text[0] = 0; }
void fake_capture(uintptr_t stream) { capturing = stream; }
int fake_device(void) { return device; }

int hipGetDeviceCount(int* n) { *n = 2; return 0; }
int hipSetDevice(int d) { device = d; return 0; }
int hipGetDevice(int* d) { *d = device; return 0; }
int hipEventCreate(void** e) { *e = (void*)++events; return 0; }
int hipEventCreateWithFlags(void** e, unsigned flags) { (void)flags; *e = (void*)++events; return 0; }
int hipEventDestroy(void* e) { (void)e; return 0; }
int hipEventRecord(void* e, void* s) { (void)e; note("record", (uintptr_t)s, 0); return 0; }
int hipStreamWaitEvent(void* s, void* e, unsigned flags) { (void)e; (void)flags; note("wait", (uintptr_t)s, 0); return 0; }
int hipStreamIsCapturing(void* s, int* status) { *status = capturing && (uintptr_t)s == capturing; return 0; }
int hipStreamSynchronize(void* s) { (void)s; return 0; }
int hipDeviceSynchronize(void) { note("synchronize", 0, 0); return 0; }
int hipMalloc(void** p, size_t n) { *p = malloc(n); return 0; }
int hipFree(void* p) { free(p); return 0; }
int hipMemcpy(void* to, const void* from, size_t n, int kind) { (void)kind; memcpy(to, from, n); return 0; }
int hipGetLastError(void) { return 0; }
int __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, void* s) { (void)g; (void)b; (void)lds; pushed = (uintptr_t)s; return 0; }
int __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, void** s) {
    const dim3 one = {1, 1, 1};
    *g = *b = one, *lds = 0, *s = (void*)pushed;
    return 0;
}
int hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t lds, void* s) {
    (void)f; (void)g; (void)b; (void)args; (void)lds;
    note("launch", (uintptr_t)s, (uintptr_t)device);
    return 0;
}
