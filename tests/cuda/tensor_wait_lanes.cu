// Test kernel for the answer that a warp gets from the product's bounded wait (gq_tcgen05.cuh:
// tc::wait).  Its lanes come to the wait one after another, on a phase that nothing completes (warp
// 0) and on one that a thread of warp 1 completes meanwhile; afterwards all lanes go through
// elect.sync and a barrier together, which they only can with one answer for all of them.
#include <cuda_runtime.h>
#include <stdint.h>

#include "gq_tcgen05.cuh"

__global__ void lanes(int* answers, int* elected) {
    __shared__ uint64_t bars[2];
    const uint32_t at = gq::smem_u32addr(bars);
    if (threadIdx.x == 0) {
        gq::tc::init(at, 1);
        gq::tc::init(at + 8, 1);
        gq::mbar_init_fence();
    }
    __syncthreads();
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    if (warp < 2) {
        const uint64_t t0 = gq::global_ns();
        while (gq::global_ns() - t0 < 1000ull * lane) {
        }
        const bool ok = gq::tc::wait(at + 8 * warp, 0);
        answers[threadIdx.x] = ok ? 1 : 0;
        if (gq::tc::elect()) atomicAdd(elected + warp, 1);
        __syncwarp();
    } else if (lane == 0) {
        const uint64_t t0 = gq::global_ns();
        while (gq::global_ns() - t0 < 16000ull) {
        }
        gq::tc::arrive(at + 8);
    }
    __syncthreads();
    if (gq::tc::elect()) atomicAdd(elected + 2, 1);
}

extern "C" int run_lanes(int* answers, int* elected) {
    int* d = nullptr;
    if (cudaMalloc(&d, 67 * sizeof(int)) != cudaSuccess) return -1;
    cudaError_t e = cudaMemset(d, 0, 67 * sizeof(int));
    if (e == cudaSuccess) {
        lanes<<<1, 96>>>(d, d + 64);
        e = cudaDeviceSynchronize();
    }
    if (e == cudaSuccess) e = cudaMemcpy(answers, d, 64 * sizeof(int), cudaMemcpyDeviceToHost);
    if (e == cudaSuccess) e = cudaMemcpy(elected, d + 64, 3 * sizeof(int), cudaMemcpyDeviceToHost);
    cudaFree(d);
    return static_cast<int>(e);
}
