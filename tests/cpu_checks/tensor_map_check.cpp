// Host threads that make their first tensor maps at once.
#include <cuda.h>
#include <cuda_runtime_api.h>
#include <stdio.h>

#include <atomic>
#include <thread>
#include <vector>

static std::atomic<int> made;
static CUresult encode_map(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                           CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill)
{
    made++;
    return CUDA_SUCCESS;
}
static cudaError_t get_entry(const char *, void **fn, unsigned long long, cudaDriverEntryPointQueryResult *q)
{
    *fn = (void *)encode_map;
    *q = cudaDriverEntryPointSuccess;
    return cudaSuccess;
}
#define cudaGetDriverEntryPoint get_entry
static int fail(const char *, ...) { return 1; }
#include "kernels.inc"

int main()
{
    std::vector<std::thread> t;
    std::atomic<int> ready{0}, bad{0};
    for (int i = 0; i < 8; i++)
        t.emplace_back([&] {
            CUtensorMap map;
            for (ready++; ready < 8;) {}
            bad += make_box_map("check", nullptr, true, 1, 64, 64, 64, &map);
        });
    for (auto &x : t) x.join();
    printf(made == 8 && !bad ? "ok\n" : "not made\n");
    return 0;
}
