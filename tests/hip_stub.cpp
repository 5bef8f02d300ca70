// The HIP calls of the library on the host alone, for tests of what it refuses and of what it launches: memory is malloc's,
// nothing runs, and stub_launches lists the launches since the last call ("kernel gx gy gz block" a line).
#include <hip/hip_runtime.h>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <string>
#include "qp_scratch.h"

static std::string g_log;
static char g_fn[4096][64];
static int g_nfn;

extern "C" {
int stub_launches(char* out, size_t cap) {
    if (g_log.size() + 1 > cap) return -1;
    memcpy(out, g_log.c_str(), g_log.size() + 1);
    g_log.clear();
    return 0;
}
hipError_t hipGetDeviceCount(int* n) { *n = 1; return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetDeviceProperties(hipDeviceProp_t* p, int) {
    memset(p, 0, sizeof *p);
    strcpy(p->name, "stub");
    strcpy(p->gcnArchName, "gfx950");
    p->multiProcessorCount = 256;
    p->totalGlobalMem = 1ull << 38;
    return hipSuccess;
}
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned) { *s = nullptr; return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipStreamBeginCapture(hipStream_t, hipStreamCaptureMode) { return hipSuccess; }
hipError_t hipStreamEndCapture(hipStream_t, hipGraph_t* g) { *g = (hipGraph_t)8; return hipSuccess; }
hipError_t hipGraphInstantiate(hipGraphExec_t* e, hipGraph_t, hipGraphNode_t*, char*, size_t) { *e = (hipGraphExec_t)8; return hipSuccess; }
hipError_t hipGraphDestroy(hipGraph_t) { return hipSuccess; }
hipError_t hipGraphExecDestroy(hipGraphExec_t) { return hipSuccess; }
hipError_t hipGraphLaunch(hipGraphExec_t, hipStream_t) { return hipSuccess; }
hipError_t hipModuleLoad(hipModule_t* m, const char*) { *m = (hipModule_t)8; return hipSuccess; }
hipError_t hipModuleGetFunction(hipFunction_t* f, hipModule_t, const char* name) {
    if (g_nfn == 4096) return hipErrorOutOfMemory;
    snprintf(g_fn[g_nfn], 64, "%s", name);
    *f = (hipFunction_t)g_fn[g_nfn++];
    return hipSuccess;
}
hipError_t hipModuleGetGlobal(hipDeviceptr_t*, size_t*, hipModule_t, const char*) { return hipErrorNotFound; }
hipError_t hipModuleOccupancyMaxActiveBlocksPerMultiprocessor(int* n, hipFunction_t, int, size_t) { *n = 1; return hipSuccess; }
hipError_t hipModuleLaunchKernel(hipFunction_t f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned, unsigned, unsigned,
                                 hipStream_t, void**, void**) {
    char line[160];
    snprintf(line, sizeof line, "%s %u %u %u %u\n", (const char*)f, gx, gy, gz, bx);
    g_log += line;
    return hipSuccess;
}
hipError_t hipMalloc(void** p, size_t n) { *p = aligned_alloc(256, (n + 255) / 256 * 256); return *p ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipFree(void* p) { free(p); return hipSuccess; }
hipError_t hipMemcpy(void* d, const void* s, size_t n, hipMemcpyKind) { memcpy(d, s, n); return hipSuccess; }
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind, hipStream_t) { memcpy(d, s, n); return hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { *e = nullptr; return hipSuccess; }
hipError_t hipEventDestroy(hipEvent_t) { return hipSuccess; }
hipError_t hipEventRecord(hipEvent_t, hipStream_t) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t) { return hipSuccess; }
hipError_t hipEventElapsedTime(float* ms, hipEvent_t, hipEvent_t) { *ms = 0; return hipSuccess; }
const char* hipGetErrorName(hipError_t) { return "error"; }
const char* hipGetErrorString(hipError_t) { return "error"; }
}

namespace qp_scratch {
int lookup(int, uint64_t* ptr) {
    static void* p = aligned_alloc(256, QP_SCRATCH_BYTES);
    *ptr = (uint64_t)p;
    return 0;
}
}  // namespace qp_scratch
