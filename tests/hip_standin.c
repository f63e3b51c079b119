/* A stand-in for the HIP runtime, loaded in front of it by CPU tests of what the library's host code asks for: memory of a chosen size, no
 * kernel runs, every launch is written down.  Addresses that it gives out are numbers, nothing may read them. */
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>
#include <stdlib.h>
#include <string.h>

typedef struct { unsigned long grid[3], block[3]; } launch_t;
static launch_t* launches;
static size_t n_launches, room;
static size_t memory = (size_t)288 << 30, taken, largest, frees;
static uintptr_t next_at = 0x100000000000;
static struct { uintptr_t at; size_t bytes; } blocks[4096];
static int n_blocks, sticky, capturing, waits;

/* ---- what a test reads and sets */
void standin_memory(size_t bytes) { memory = bytes; }
void standin_capture(int on) { capturing = on; }
size_t standin_taken(void) { return taken; }
size_t standin_largest(void) { return largest; }
size_t standin_frees(void) { return frees; }
int standin_waits(void) { return waits; }   /* for a stream */
size_t standin_launches(void) { return n_launches; }
void standin_launch(size_t i, unsigned long* six) { memcpy(six, &launches[i], sizeof(launch_t)); }
void standin_forget(void) { n_launches = largest = 0; }

static hipError_t launch(dim3 g, dim3 b) {
    if (n_launches == room) launches = realloc(launches, (room = room ? 2 * room : 1024) * sizeof(launch_t));
    launches[n_launches++] = (launch_t){{g.x, g.y, g.z}, {b.x, b.y, b.z}};
    const int fits = g.x && g.y && g.z && (unsigned long)g.x * b.x < 1ul << 32 && (unsigned long)g.y * b.y < 1ul << 32 && (unsigned long)g.z * b.z < 1ul << 32 && g.y < 65536 && g.z < 65536;
    sticky = fits ? 0 : hipErrorInvalidConfiguration;
    return sticky;
}
hipError_t hipExtLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t lds, hipStream_t s, hipEvent_t e0, hipEvent_t e1, int flags) { return launch(g, b); }
hipError_t hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t lds, hipStream_t s) { return launch(g, b); }
hipError_t hipGetLastError(void) {
    const int e = sticky;
    sticky = 0;
    return e;
}
const char* hipGetErrorString(hipError_t e) { return "an error of the stand-in"; }

hipError_t hipMalloc(void** p, size_t bytes) {
    if (bytes > memory - taken || n_blocks == 4096) return sticky = hipErrorOutOfMemory;
    blocks[n_blocks].at = next_at;
    blocks[n_blocks++].bytes = bytes;
    *p = (void*)next_at;
    next_at += (bytes + 0xffffff) & ~(size_t)0xffffff;
    taken += bytes;
    if (bytes > largest) largest = bytes;
    return hipSuccess;
}
hipError_t hipFree(void* p) {
    if (!p) return hipSuccess;
    for (int i = 0; i < n_blocks; i++)
        if (blocks[i].at == (uintptr_t)p) {
            taken -= blocks[i].bytes;
            blocks[i] = blocks[--n_blocks];
            frees++;
            return hipSuccess;
        }
    return hipErrorInvalidValue;
}
hipError_t hipHostMalloc(void** p, size_t bytes, unsigned flags) { return (*p = malloc(bytes)) ? hipSuccess : hipErrorOutOfMemory; }
hipError_t hipHostFree(void* p) { return free(p), hipSuccess; }
hipError_t hipMemcpyAsync(void* d, const void* s, size_t n, hipMemcpyKind k, hipStream_t t) { return hipSuccess; }
hipError_t hipMemsetAsync(void* d, int v, size_t n, hipStream_t t) { return hipSuccess; }

hipError_t hipSetDevice(int d) { return hipSuccess; }
hipError_t hipGetDevice(int* d) { return *d = 0, hipSuccess; }
hipError_t hipGetDevicePropertiesR0600(hipDeviceProp_tR0600* p, int d) {
    memset(p, 0, sizeof *p);
    p->multiProcessorCount = 256;
    return hipSuccess;
}
hipError_t hipGetSymbolAddress(void** p, const void* symbol) { return *p = (void*)0x7000000, hipSuccess; }
hipError_t hipFuncSetAttribute(const void* f, hipFuncAttribute a, int v) { return hipSuccess; }
hipError_t hipStreamCreateWithFlags(hipStream_t* s, unsigned flags) { return *s = (hipStream_t)0x10, hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t s) { return waits++, capturing ? hipErrorStreamCaptureUnsupported : hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t s, hipStreamCaptureStatus* st) { return *st = capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone, hipSuccess; }
hipError_t hipEventCreate(hipEvent_t* e) { return *e = (hipEvent_t)0x20, hipSuccess; }
hipError_t hipEventCreateWithFlags(hipEvent_t* e, unsigned flags) { return *e = (hipEvent_t)0x20, hipSuccess; }
hipError_t hipEventRecord(hipEvent_t e, hipStream_t s) { return hipSuccess; }
hipError_t hipEventSynchronize(hipEvent_t e) { return hipSuccess; }
