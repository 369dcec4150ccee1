// Stands in for the HIP calls that a launch makes and records them, on the CPU: a program that links librt4k.so with this
// finds these definitions before the runtime's, so no kernel starts and no device is needed.  The entry points at the end let
// a test choose the device and read what was asked for.
#include <hip/hip_runtime_api.h>

#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <utility>

#include "rt4k.h"

namespace {

int g_dev = 0, g_sets = 0, g_launches = 0;
std::map<std::pair<const void*, int>, size_t> g_limit;      // dynamic LDS of a kernel on a device
thread_local struct {
    dim3 grid, block;
    size_t lds;
    hipStream_t st;
} g_cfg;
size_t g_lds = 0;                                           // of the last launch
const void* g_fn = nullptr;

size_t limit() {
    const auto it = g_limit.find({g_fn, g_dev});
    return it == g_limit.end() ? 65536 : it->second;
}
void check(bool ok, const char* what) {
    if (ok) return;
    std::fprintf(stderr, "failed: %s\n", what);
    std::exit(1);
}

}  // namespace

extern "C" {
hipError_t hipGetDevice(int* d) { return *d = g_dev, hipSuccess; }
hipError_t hipDeviceGetAttribute(int* v, hipDeviceAttribute_t, int) { return *v = 256, hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
hipError_t hipFuncSetAttribute(const void* f, hipFuncAttribute, int v) { return g_sets++, g_limit[{f, g_dev}] = (size_t)v, hipSuccess; }
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t st) { return g_cfg = {g, b, lds, st}, hipSuccess; }
hipError_t __hipPopCallConfiguration(dim3* g, dim3* b, size_t* lds, hipStream_t* st) {
    return *g = g_cfg.grid, *b = g_cfg.block, *lds = g_cfg.lds, *st = g_cfg.st, hipSuccess;
}
hipError_t hipLaunchKernel(const void* f, dim3, dim3, void**, size_t lds, hipStream_t) { return g_fn = f, g_lds = lds, g_launches++, hipSuccess; }
}

namespace {

void* const kAt = reinterpret_cast<void*>(0x1000);

int gate4(int rows, int K) {
    return rt4_ffn_gate_w4a8((float*)kAt, (const uint32_t*)kAt, (const uint16_t*)kAt, (const uint32_t*)kAt, (const uint16_t*)kAt, (const int8_t*)kAt,
                             (const float*)kAt, rows, 70, K, RT4_SILU, nullptr);
}

// A launch that another thread has prepared stays within the limit whatever K the next call has, on each device.
void gate4_lds() {
    for (int rows = 2; rows <= 4; rows++)
        for (g_dev = 0; g_dev < 2; g_dev++) {
            const int sets = g_sets;
            check(gate4(rows, 38912) == RT4_OK, "the largest K");
            const size_t most = g_lds;
            check(most > 65536 && most <= limit(), "the largest K fits its limit");
            for (int K = 128; K <= 38912; K += 128) {
                check(gate4(rows, K) == RT4_OK && (g_lds <= 65536 || g_lds <= limit()), "a launch fits its limit");
                check(most <= limit(), "no call lowers the limit");
            }
            check(g_sets == sets + 1, "the limit is raised once");
        }
    check(gate4(1, 38912) == RT4_OK && g_lds <= 65536, "one row needs no limit");
}

int norm(void* h_out, int64_t ldho, const void* y) {
    return rt4_block_norm(h_out, ldho, kAt, 256, RT4_F32, y, 256, RT4_F32, nullptr, 0, nullptr, (const float*)kAt, 1.0, 1e-6, 0.0, (void*)0x9000, nullptr,
                          RT4_F32, 4, 256, nullptr);
}

// Without y nothing is written to h_out, so nothing is asked of it.
void norm_without_y() {
    check(norm(nullptr, 0, nullptr) == RT4_OK, "no h_out");
    check(norm(kAt, 0, nullptr) == RT4_OK, "h_out as h, any stride");
    check(norm((char*)kAt + 1, 3, nullptr) == RT4_OK, "h_out not aligned");
    check(norm(kAt, 300, kAt) == RT4_E_ARG && norm((char*)kAt + 1, 256, kAt) == RT4_E_ARG && norm(kAt, 256, kAt) == RT4_OK, "with y they count");
}

}  // namespace

int main(int argc, char** argv) {
    if (argc == 2 && !std::strcmp(argv[1], "gate4_lds")) gate4_lds();
    else if (argc == 2 && !std::strcmp(argv[1], "norm_without_y")) norm_without_y();
    else return 2;
    std::printf("launches %d\n", g_launches);
    return 0;
}
