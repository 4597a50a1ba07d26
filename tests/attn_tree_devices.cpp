// The tree attention's host side over a CUDA runtime of two devices that only keeps count: a launch with
// more than 48 KB of dynamic shared memory succeeds on a device where its kernel was allowed that much.
// Linked with the library's own objects in place of the CUDA runtime; run by test_attn_tree_devices.py.
#include <cuda_runtime_api.h>
#include <stdio.h>

#include <map>
#include <utility>

#include "slate_cuda.h"

static int device = 0, set_calls = 0, fail_sets = 0, launches = 0;
static cudaError_t pending = cudaSuccess;       // of some call before, of another library say
static std::map<std::pair<int, const void*>, size_t> allowed;

extern "C" {
void** __cudaRegisterFatBinary(void*) { static void* h; return &h; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, uint3*, uint3*, dim3*, dim3*, int*) {}
unsigned __cudaPushCallConfiguration(dim3, dim3, size_t, void*) { return 0; }
cudaError_t __cudaPopCallConfiguration(dim3*, dim3*, size_t*, void*) { return cudaSuccess; }
cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
cudaError_t cudaGetLastError(void) { const cudaError_t e = pending; pending = cudaSuccess; return e; }
cudaError_t cudaLaunchKernel(const void*, dim3, dim3, void**, size_t, cudaStream_t) { ++launches; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute a, int v) {
    ++set_calls;
    if (fail_sets) return --fail_sets, cudaErrorInvalidValue;
    if (a == cudaFuncAttributeMaxDynamicSharedMemorySize) allowed[{device, f}] = (size_t)v;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernelExC(const cudaLaunchConfig_t* c, const void* f, void**) {
    if (c->dynamicSmemBytes > 48 * 1024 && allowed[{device, f}] < c->dynamicSmemBytes) return cudaErrorInvalidValue;
    ++launches;
    return cudaSuccess;
}
void sb_set_error(const char*, ...) {}
int sb_cuda_check(cudaError_t e, const char*) { return e == cudaSuccess ? 0 : -5; }
}

static int call(int nodes, int kv, int hd) {
    alignas(16) static char pool[16], ws[16];
    static int32_t ints[4];
    static uint64_t mask[1];
    static float f[1];
    slate_kv_cache_t c = {};
    c.pool = pool, c.page_table = ints, c.n_pages = 4, c.n_slots = 1, c.max_pages = 4, c.n_layers = 1, c.n_kv_heads = 1;
    c.head_dim = hd, c.kv_dtype = kv;
    slate_tree_t t = {};
    t.n_seq = 1, t.rows = nodes, t.max_nodes = nodes, t.row_off = ints, t.slot = ints, t.ctx = ints, t.mask = mask;
    return slate_cuda_attention_tree(&c, 0, &t, 1, f, hd, f, hd, 1.f, ws, (size_t)1 << 40, nullptr);
}

int main() {
    // every kernel: 8, 16, 32, 64 and more rows (more than 16 heads' rows by nodes), each type and head_dim
    static const int rows[] = {1, 8, 9, 16, 17, 32, 33, 64};
    for (int pass = 0; pass < 2; ++pass)
        for (device = 0; device < 2; ++device) {
            int bad = 0, before = set_calls;
            for (int kv = 0; kv < 3; ++kv)
                for (int hd : {64, 128})
                    for (int n : rows) bad += call(n, kv, hd) != 0;
            printf("pass %d device %d: %d failed, %d set\n", pass, device, bad, set_calls - before);
        }
    device = 2;                                   // a failure is not remembered
    fail_sets = 1;
    const int first = call(1, 0, 64), second = call(1, 0, 64);
    printf("device 2: %d then %d\n", first, second);
    device = 70;                                  // an ordinal beyond the ones whose state is kept
    const int a = call(40, 1, 128), b = call(40, 1, 128);
    printf("device 70: %d %d\n", a, b);
    device = 0;
    pending = cudaErrorInvalidValue;
    const int c = call(3, 1, 64);
    pending = cudaErrorInvalidValue;
    const int d = call(3, 1, 24);
    printf("after an error of another call: %d %d\n", c, d);
    return 0;
}
