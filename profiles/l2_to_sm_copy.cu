// How fast TMA brings the boxes of tree_attn_kernel out of L2 into all SMs when nothing else happens: one block per SM, a ring of 16 KiB slots, one thread
// that requests and one that takes.  A K slot is two boxes of 64 dims x 64 rows (two pages of 64), a V slot one box of 4 x 64 dims x 32 rows.
//
//   nvcc -gencode arch=compute_100a,code=sm_100a -O3 -std=c++17 -o /tmp/l2_to_sm_copy profiles/l2_to_sm_copy.cu && /tmp/l2_to_sm_copy
#include <cuda.h>
#include <cstdio>
#include "../qwen_tailor_b200/csrc/sm100_prims.cuh"
using namespace sm100;

constexpr int SLOT = 16384, RING = 10, SLOTS_PER_BLOCK = 4000;

template <bool V>
__global__ void __launch_bounds__(64, 1) copy_boxes(const __grid_constant__ CUtensorMap map, int region, int* failed, long long* cycles) {
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ uint64_t full[RING], empty[RING];
    const uint32_t sb = smem_addr(smem);
    if (threadIdx.x == 0) {
        for (int i = 0; i < RING; i++) { mbar_init(smem_addr(&full[i]), 1); mbar_init(smem_addr(&empty[i]), 1); }
        fence_barrier_init();
    }
    __syncthreads();
    const long long start = clock64();
    if (threadIdx.x == 0) {
        for (int i = 0; i < SLOTS_PER_BLOCK; i++) {
            const int s = i % RING;
            if (i >= RING && !mbar_wait(smem_addr(&empty[s]), (i / RING - 1) & 1)) { *failed = 1; break; }
            const uint32_t f = smem_addr(&full[s]), dst = sb + s * SLOT;
            const int c = (blockIdx.x * 37 + i) % region;            // slot of the region: a page pair has four slabs of two heads, a page two halves of two heads
            mbar_expect_tx(f, SLOT);
            for (int q = 0; q < (V ? 1 : 2); q++)
                asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
                             ::"r"(dst + q * 8192), "l"(&map), "r"(f), "r"(0), "r"(V ? (c & 1) * 32 : 0), "r"(V ? 0 : c & 3), "r"(V ? c >> 1 & 1 : c >> 2 & 1),
                               "r"(V ? c >> 2 : 2 * (c >> 3) + q) : "memory");
        }
    } else if (threadIdx.x == 32) {
        for (int i = 0; i < SLOTS_PER_BLOCK; i++) {
            if (!mbar_wait(smem_addr(&full[i % RING]), (i / RING) & 1)) { *failed = 1; break; }
            mbar_arrive(smem_addr(&empty[i % RING]));
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && blockIdx.x == 0) *cycles = clock64() - start;
}

typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                           CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int main() {
    const int region = 256;                                          // slots: 4 MiB, 64 pages [2 heads, 64 rows, 256] bf16
    const cuuint64_t pages = (cuuint64_t)region * SLOT / 65536;
    char* data;
    int* failed;
    long long* cycles;
    cudaMalloc(&data, (size_t)region * SLOT);
    cudaMemset(data, 0, (size_t)region * SLOT);
    cudaMallocManaged(&failed, sizeof(int));
    cudaMallocManaged(&cycles, sizeof(long long));
    *failed = 0;
    void* f = nullptr;
    cudaDriverEntryPointQueryResult qr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qr) != cudaSuccess || !f) return 1;
    for (int v = 0; v < 2; v++) {
        CUtensorMap map;
        const cuuint64_t dims[5] = {64, 64, 4, 2, pages}, strides[4] = {512, 128, 32768, 65536};
        const cuuint32_t box[5] = {64, v ? 32u : 64u, v ? 4u : 1u, 1, 1}, es[5] = {1, 1, 1, 1, 1};
        if (reinterpret_cast<Encode>(f)(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, data, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                        CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) return 1;
        auto kernel = v ? copy_boxes<true> : copy_boxes<false>;
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RING * SLOT);
        cudaEvent_t e0, e1;
        cudaEventCreate(&e0);
        cudaEventCreate(&e1);
        float ms = 0;
        for (int i = 0; i < 4; i++) {
            cudaEventRecord(e0);
            kernel<<<148, 64, RING * SLOT>>>(map, region, failed, cycles);
            cudaEventRecord(e1);
            if (cudaEventSynchronize(e1) != cudaSuccess) return 1;
            cudaEventElapsedTime(&ms, e0, e1);
        }
        printf("%s boxes: %.2f TB/s over 148 SMs, %.1f bytes a cycle and SM%s\n", v ? "V" : "K", 148. * SLOTS_PER_BLOCK * SLOT / ms / 1e9, (double)SLOTS_PER_BLOCK * SLOT / *cycles,
               *failed ? " (a wait gave up)" : "");
    }
    return *failed;
}
