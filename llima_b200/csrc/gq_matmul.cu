// out = a b^T (+ bias) for block-scaled e4m3 operands.
//
// One CTA per 64 x 64 tile of the output, 4 x 4 values per thread; 32 columns of both
// operands at a time are widened to f32 in shared memory.  Each 128-column block's products
// are summed on their own and join the total times both scales.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "gq_device.cuh"
#include "gq_internal.h"

namespace gq {
namespace {

template <class T>
__device__ __forceinline__ T out_cast(float x);
template <>
__device__ __forceinline__ float out_cast<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half out_cast<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 out_cast<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float e8m0_value(uint32_t b) {
    return b == 255u ? __uint_as_float(0x7FFFFFFFu) : __uint_as_float(b == 0 ? 0x00400000u : b << 23);
}

template <class T>
__global__ void __launch_bounds__(256) gq_matmul_kernel(const GqMatmul p) {
    __shared__ float sa[64][33], sb[64][33];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t tiles_n = (p.n + 63) / 64;
    const int64_t m0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * 64;
    float total[4][4] = {}, part[4][4] = {};
    for (int64_t k0 = 0; k0 < p.k; k0 += 32) {
        const int r = tid >> 2, c = 8 * (tid & 3);
        for (int i = 0; i < 8; ++i) {
            __nv_fp8_e4m3 x, y;
            x.__x = m0 + r < p.m ? p.a[(m0 + r) * p.ld_a + k0 + c + i] : 0;
            y.__x = n0 + r < p.n ? p.b[(n0 + r) * p.ld_b + k0 + c + i] : 0;
            sa[r][c + i] = static_cast<float>(x);
            sb[r][c + i] = static_cast<float>(y);
        }
        __syncthreads();
        for (int k = 0; k < 32; ++k)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) part[i][j] = __fmaf_rn(sa[4 * ty + i][k], sb[tx + 16 * j][k], part[i][j]);
        __syncthreads();
        if ((k0 & 127) == 96 || k0 + 32 >= p.k) {
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) {
                    const int64_t m = m0 + 4 * ty + i, n = n0 + tx + 16 * j;
                    if (m < p.m && n < p.n)
                        total[i][j] += part[i][j] * e8m0_value(p.a_scales[m * p.ld_a_scales + k0 / 128]) *
                                       e8m0_value(p.b_scales[n / 128 * p.ld_b_scales + k0 / 128]);
                    part[i][j] = 0.0f;
                }
        }
    }
    T* out = reinterpret_cast<T*>(p.out);
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const int64_t m = m0 + 4 * ty + i, n = n0 + tx + 16 * j;
            if (m < p.m && n < p.n) out[m * p.ld_out + n] = out_cast<T>(total[i][j] + (p.bias != nullptr ? p.bias[n] : 0.0f));
        }
}

template <class T>
int launch_t(const GqMatmul& p, cudaStream_t s) {
    const int64_t tiles = (p.m + 63) / 64 * ((p.n + 63) / 64);
    if (tiles > INT32_MAX) return static_cast<int>(cudaErrorInvalidValue);
    gq_matmul_kernel<T><<<static_cast<unsigned>(tiles), 256, 0, s>>>(p);
    return static_cast<int>(cudaGetLastError());
}

}  // namespace

int launch_matmul(int dtype, const GqMatmul& p, void* stream) {
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case GQ_TYPE_F32: return launch_t<float>(p, s);
        case GQ_TYPE_F16: return launch_t<__half>(p, s);
        case GQ_TYPE_BF16: return launch_t<__nv_bfloat16>(p, s);
        default: return static_cast<int>(cudaErrorInvalidValue);
    }
}

}  // namespace gq
