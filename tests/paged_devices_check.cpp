// Host-only check of the paged attention launchers on more than one device, built and run by tests/test_paged_devices_cpu.py
// from the library's own objects and the CUDA runtime below, a fake: a kernel may be launched with more than 48 KB of
// dynamic shared memory only where its limit was raised on the device that is current. No GPU is used.
#include <cuda_runtime.h>

#include <cstdio>
#include <map>
#include <stdexcept>
#include <string>
#include <utility>

#include "paged.h"

static int device = 0, launches = 0, refused = 0;
static bool fail_attributes = false;
static std::map<std::pair<int, const void*>, int> limit;
static struct { dim3 grid, block; size_t smem; cudaStream_t stream; } config;
static cudaError_t last = cudaSuccess;

extern "C" {
cudaError_t cudaGetDevice(int* d) { *d = device; return cudaSuccess; }
cudaError_t cudaFuncSetAttribute(const void* f, cudaFuncAttribute, int value) {
    if (fail_attributes) return cudaErrorUnknown;
    limit[{device, f}] = value;
    return cudaSuccess;
}
cudaError_t cudaLaunchKernel(const void* f, dim3, dim3, void**, size_t smem, cudaStream_t) {
    ++launches;
    if (smem > 48 * 1024 && limit[{device, f}] < int(smem)) {
        ++refused;
        return last = cudaErrorInvalidValue;
    }
    return cudaSuccess;
}
cudaError_t cudaGetLastError() { const cudaError_t e = last; last = cudaSuccess; return e; }
const char* cudaGetErrorString(cudaError_t) { return "an error"; }
unsigned __cudaPushCallConfiguration(dim3 g, dim3 b, size_t smem, cudaStream_t s) {
    config = {g, b, smem, s};
    return 0;
}
cudaError_t __cudaPopCallConfiguration(dim3* g, dim3* b, size_t* smem, void* s) {
    *g = config.grid;
    *b = config.block;
    *smem = config.smem;
    *static_cast<cudaStream_t*>(s) = config.stream;
    return cudaSuccess;
}
void** __cudaRegisterFatBinary(void*) { static void* p; return &p; }
void __cudaRegisterFatBinaryEnd(void**) {}
void __cudaUnregisterFatBinary(void**) {}
void __cudaRegisterFunction(void**, const char*, char*, const char*, int, void*, void*, void*, void*, int*) {}
}
namespace gpt {
int num_sms() { return 148; }
}

static bool attention(int dim, int new_tokens, int box_log) {
    gpt::KvMaps maps{};
    gpt::KvView c{};
    c.kv_heads = 1;
    c.dim = dim;
    c.page = gpt::FastDiv::of(16);
    c.num_pages = 1;
    c.box_log = box_log;
    gpt::KvBatch b{};
    b.seqs = 1;
    b.tokens = b.max_new = new_tokens;
    gpt::PagedAttnArgs a{};
    a.type = a.kv_type = gpt::kBF16;
    a.q_heads = 8;
    a.rows_to = 0x7fffffff;
    try {
        gpt::launch_paged_attention(maps, c, b, a, nullptr, nullptr);
        return true;
    } catch (const std::exception&) {
        return false;
    }
}

int main() {
    const int shapes[][3] = {{64, 1, 4}, {128, 1, 4}, {64, 500, 4}, {64, 500, 0}, {128, 500, 4}, {128, 500, 0}};
    int bad = 0;
    for (const auto& s : shapes)
        for (int d : {0, 1, 5, 0}) {
            device = d;
            if (!attention(s[0], s[1], s[2])) {
                std::printf("FAIL: dim %d, %d tokens, box %d refused on device %d\n", s[0], s[1], s[2], d);
                ++bad;
            }
        }
    // a failure to set a limit is reported, and not for good
    device = 9;
    fail_attributes = true;
    if (attention(64, 500, 4)) std::printf("FAIL: a failed attribute went unnoticed\n"), ++bad;
    fail_attributes = false;
    if (!attention(64, 500, 4)) std::printf("FAIL: a failed attribute is kept\n"), ++bad;
    if (launches == 0) std::printf("FAIL: nothing was launched\n"), ++bad;
    std::printf(bad ? "%d failures\n" : "OK\n", bad);
    return bad != 0;
}
