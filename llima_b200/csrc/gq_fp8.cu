// Block-scaled 8-bit floats: GGUF weights to e4m3 with one scale per 128 x 128 block, and
// activations to e4m3 with one scale per 1 x 128 block (after an RMS norm, after a gated
// activation, or as they are).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "gq_blocks.cuh"
#include "gq_fp8.cuh"
#include "gq_internal.h"

namespace gq {
namespace {

// ---------------------------------------------------------------------------------------
// Weights
// ---------------------------------------------------------------------------------------

// Source row of output row o (inverse of the llama q/k permutation: row 2a + t of a head
// moves to t * D/2 + a, gguf_conversion.py:314-332).
__device__ __forceinline__ int64_t fp8_src_row(int32_t head_dim, int64_t o) {
    if (head_dim == 0) return o;
    const int64_t h = o / head_dim;
    const int rem = static_cast<int>(o - h * head_dim), half = head_dim >> 1;
    const int t = rem >= half ? 1 : 0;
    return h * head_dim + 2 * (rem - t * half) + t;
}

// Shared bytes per row of a 256-column tile: the 16-byte-aligned window around the row's
// bytes, an odd number of 16-byte chunks so that lanes on neighbouring rows read different
// banks.
template <int TYPE>
struct Fp8Tile {
    static constexpr int kChunkBytes = 256 / BlockView<TYPE>::kUnitValues * BlockView<TYPE>::kUnitBytes;
    static constexpr int kChunks = ((kChunkBytes + 15 + 15) / 16) | 1;
    static constexpr int kPitch = 16 * kChunks;
    static constexpr int kSmem = 128 * kPitch + 64;
};

// One CTA per 128 rows x 256 columns (two scale blocks).  Thread t owns row t % 128 of block
// t / 128: 128 values, kept as their integer codes.  A value is a monotone function of its
// code, so a 16- or 32-value block's largest |x| is at its smallest or largest code.
template <int TYPE>
__global__ void __launch_bounds__(256) gq_fp8_weight_kernel(const GqFp8Weight p) {
    using V = BlockView<TYPE>;
    using T = Fp8Tile<TYPE>;
    constexpr int NB = 128 / V::BV;
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t* wmax = reinterpret_cast<uint32_t*>(smem + 128 * T::kPitch);
    const int tid = threadIdx.x;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / p.n_col_tiles) * 128;
    const int64_t col0 = static_cast<int64_t>(blockIdx.x % p.n_col_tiles) * 256;
    const int rows = static_cast<int>(min(static_cast<int64_t>(128), p.rows - row0));
    const int cols = static_cast<int>(min(static_cast<int64_t>(256), p.cols - col0));
    const int64_t at = col0 / V::kUnitValues * V::kUnitBytes;
    const int bytes = cols / V::kUnitValues * V::kUnitBytes;
    for (int i = tid; i < rows * T::kChunks; i += 256) {
        const int r = i / T::kChunks, c = i - r * T::kChunks;
        const int64_t start = fp8_src_row(p.head_dim, row0 + r) * p.row_bytes + at;
        const int64_t a = (start & ~int64_t(15)) + 16 * c;
        if (a < start + bytes)
            cp_async16(smem + r * T::kPitch + 16 * c, p.src + a, static_cast<int>(min(static_cast<int64_t>(16), p.src_bytes - a)));
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();

    const int r = tid & 127, half = tid >> 7;
    const int nb = r < rows ? max(0, min(NB, (cols - 128 * half) / V::BV)) : 0;
    const int64_t start = fp8_src_row(p.head_dim, row0 + r) * p.row_bytes + at;
    const uint8_t* row = smem + r * T::kPitch + static_cast<int>(start & 15);
    uint32_t w[NB][V::NW];
    float A[NB], B[NB];
    uint32_t amax = 0;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        if (i >= nb) continue;
        uint32_t words[8];
        decode_block<TYPE>(row, NB * half + i, words, A[i], B[i]);
#pragma unroll
        for (int j = 0; j < V::NW; ++j) w[i][j] = words[j];
        if ((__float_as_uint(A[i]) & 0x7FFFFFFFu) < kInfBits && (__float_as_uint(B[i]) & 0x7FFFFFFFu) < kInfBits) {
            uint32_t mn = 0xFFFFFFFFu, mx = 0u;
#pragma unroll
            for (int j = 0; j < V::NW; ++j) {
                const uint32_t e = words[j] & 0x00FF00FFu, o = (words[j] >> 8) & 0x00FF00FFu;
                mn = vmin16(mn, e, o);
                mx = vmax16(mx, e, o);
            }
            const int lo = static_cast<int>(min(mn & 0xFFFFu, mn >> 16)) - V::OFF;
            const int hi = static_cast<int>(max(mx & 0xFFFFu, mx >> 16)) - V::OFF;
            amax = max(amax, max(finite_abs(block_value<TYPE>(A[i], B[i], lo)), finite_abs(block_value<TYPE>(A[i], B[i], hi))));
        } else {
            finite = false;
            for (int j = 0; j < V::BV; ++j) {
                const int q = static_cast<int>(byte_of(words[j >> 2], j & 3)) - V::OFF;
                amax = max(amax, finite_abs(block_value<TYPE>(A[i], B[i], q)));
            }
        }
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((tid & 31) == 0) wmax[tid >> 5] = amax;
    __syncthreads();
    const uint32_t* m = wmax + 4 * half;
    const uint32_t byte = scale_byte(max(max(m[0], m[1]), max(m[2], m[3])));
    const float inv = inverse_scale(byte);
    if (r == 0 && 128 * half < cols)
        p.scales[(row0 >> 7) * p.scale_cols + (col0 >> 7) + half] = static_cast<uint8_t>(byte);
    uint8_t* out = p.codes + (row0 + r) * p.cols + col0 + 128 * half;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        if (i >= nb) continue;
        uint32_t c[V::NW];
#pragma unroll
        for (int j = 0; j < V::NW; ++j) {
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[k] = block_value<TYPE>(A[i], B[i], static_cast<int>(byte_of(w[i][j], k)) - V::OFF);
                if (!finite) x[k] = nan_unless_finite(x[k]);
                x[k] = __fmul_rn(x[k], inv);
            }
            c[j] = e4m3x2(x[0], x[1]) | (e4m3x2(x[2], x[3]) << 16);
        }
#pragma unroll
        for (int j = 0; j < V::NW; j += 4) stg128(out + V::BV * i + 4 * j, make_uint4(c[j], c[j + 1], c[j + 2], c[j + 3]));
    }
}

// ---- elements of the float types, eight at a time -----------------------------------------

struct F32 {};
struct F16 {};
struct BF16 {};

template <class T>
struct Elem;
template <>
struct Elem<F32> {
    static constexpr int kBytes = 4;
    static __device__ __forceinline__ void load8(const void* p, float (&x)[8]) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
    static __device__ __forceinline__ float round(float x) { return x; }
    static __device__ __forceinline__ void store8(void* p, const float (&x)[8]) {
        stg128f(reinterpret_cast<float*>(p), x[0], x[1], x[2], x[3]);
        stg128f(reinterpret_cast<float*>(p) + 4, x[4], x[5], x[6], x[7]);
    }
};
template <>
struct Elem<F16> {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ void load8(const void* p, float (&x)[8]) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = h2f(w[i]);
            x[2 * i + 1] = h2f(w[i] >> 16);
        }
    }
    static __device__ __forceinline__ float round(float x) { return __half2float(__float2half_rn(x)); }
    static __device__ __forceinline__ void store8(void* p, const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = __half_as_ushort(__float2half_rn(x[2 * i])) | (static_cast<uint32_t>(__half_as_ushort(__float2half_rn(x[2 * i + 1]))) << 16);
        stg128(p, make_uint4(w[0], w[1], w[2], w[3]));
    }
};
template <>
struct Elem<BF16> {
    static constexpr int kBytes = 2;
    static __device__ __forceinline__ void load8(const void* p, float (&x)[8]) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ float round(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }
    static __device__ __forceinline__ void store8(void* p, const float (&x)[8]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = __bfloat16_as_ushort(__float2bfloat16_rn(x[2 * i])) |
                   (static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(x[2 * i + 1]))) << 16);
        stg128(p, make_uint4(w[0], w[1], w[2], w[3]));
    }
};

// Eight values over the block scale to eight codes
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float inv) {
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __fmul_rn(nan_unless_finite(x[4 * i + k]), inv);
        c[i] = e4m3x2(v[0], v[1]) | (e4m3x2(v[2], v[3]) << 16);
    }
    return make_uint2(c[0], c[1]);
}
__device__ __forceinline__ uint32_t amax8(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, finite_abs(x[k]));
    return m;
}
// over the 16 lanes that hold one 128-value block
__device__ __forceinline__ uint32_t max16(uint32_t m) {
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    return m;
}

// Weights of a float type: one CTA per 128 x 128 block, thread t the 8 columns 8 (t % 16) of
// rows t / 16 + 16 i, held in registers between the block's maximum and the codes.
template <class T>
__global__ void __launch_bounds__(256) gq_fp8_float_weight_kernel(const GqFp8Weight p) {
    __shared__ uint32_t wmax[8];
    const int tid = threadIdx.x;
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / p.n_col_tiles) * 128;
    const int64_t col = static_cast<int64_t>(blockIdx.x % p.n_col_tiles) * 128 + 8 * (tid & 15);
    float x[8][8];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = row0 + (tid >> 4) + 16 * i;
        if (r < p.rows && col < p.cols) {
            Elem<T>::load8(p.src + fp8_src_row(p.head_dim, r) * p.row_bytes + col * Elem<T>::kBytes, x[i]);
            amax = max(amax, amax8(x[i]));
        }
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((tid & 31) == 0) wmax[tid >> 5] = amax;
    __syncthreads();
    amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max(amax, wmax[i]);
    const uint32_t byte = scale_byte(amax);
    const float inv = inverse_scale(byte);
    if (tid == 0) p.scales[(row0 >> 7) * p.scale_cols + blockIdx.x % p.n_col_tiles] = static_cast<uint8_t>(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = row0 + (tid >> 4) + 16 * i;
        if (r < p.rows && col < p.cols) st_global(reinterpret_cast<uint2*>(p.codes + r * p.cols + col), encode8(x[i], inv));
    }
}

template <int TYPE>
int launch_weight(GqFp8Weight& p, cudaStream_t s) {
    using T = Fp8Tile<TYPE>;
    auto kern = gq_fp8_weight_kernel<TYPE>;
    if (T::kSmem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem);
        if (e != cudaSuccess) return static_cast<int>(e);
    }
    p.n_col_tiles = static_cast<uint32_t>((p.cols + 255) / 256);
    const int64_t tiles = (p.rows + 127) / 128 * p.n_col_tiles;
    kern<<<static_cast<unsigned>(tiles), 256, T::kSmem, s>>>(p);
    return static_cast<int>(cudaGetLastError());
}
template <class T>
int launch_float_weight(GqFp8Weight& p, cudaStream_t s) {
    p.n_col_tiles = static_cast<uint32_t>((p.cols + 127) / 128);
    const int64_t tiles = (p.rows + 127) / 128 * p.n_col_tiles;
    gq_fp8_float_weight_kernel<T><<<static_cast<unsigned>(tiles), 256, 0, s>>>(p);
    return static_cast<int>(cudaGetLastError());
}

// ---------------------------------------------------------------------------------------
// Activations
// ---------------------------------------------------------------------------------------

// y = silu(g) * x = g / (1 + exp(-g)) * x, or x.  The reciprocal and the exponential are the
// hardware's approximations (a few ulp of f32, where a code keeps 4 bits); g = -inf gives NaN
// and a g whose exponential overflows gives -0, as the formula does.
template <bool GATED>
__device__ __forceinline__ void gate8(float (&x)[8], const float (&g)[8]) {
    if constexpr (GATED) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float r;
            asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.0f, __expf(-g[k]))));
            x[k] = __fmul_rn(__fmul_rn(g[k], r), x[k]);
        }
    }
}

// One 128-value block per 16 lanes and step.
template <class T, bool GATED>
__global__ void __launch_bounds__(256) gq_fp8_rows_kernel(const GqFp8Rows p) {
    const int64_t groups = p.rows * p.blocks;
    const int sub = threadIdx.x & 15;
    for (int64_t g0 = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 4;; g0 += static_cast<int64_t>(gridDim.x) * 16) {
        // both halves of a warp stay in the loop together (the shuffles name all lanes)
        if (__all_sync(0xffffffffu, g0 >= groups)) break;
        const bool on = g0 < groups;
        const int64_t row = on ? g0 / p.blocks : 0;
        const int64_t kb = on ? g0 - row * p.blocks : 0;
        const int64_t col = kb * 128 + 8 * sub;
        const bool in = on && col < p.cols;
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0}, g[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (in) {
            Elem<T>::load8(p.x + (row * p.ld_x + col) * Elem<T>::kBytes, x);
            if constexpr (GATED) Elem<T>::load8(p.gate + (row * p.ld_gate + col) * Elem<T>::kBytes, g);
        }
        gate8<GATED>(x, g);
        const uint32_t byte = scale_byte(max16(amax8(x)));
        if (in) st_global(reinterpret_cast<uint2*>(p.codes + row * p.ld_codes + col), encode8(x, inverse_scale(byte)));
        if (on && sub == 0) p.scales[row * p.ld_scales + kb] = static_cast<uint8_t>(byte);
    }
}

// RMS norm of a row (with the residual's addition), one CTA per row: pass 1 keeps the sum
// of squares, pass 2 normalizes and quantizes.  The sum x + r is rounded to the input type
// first: the norm is of what the next layer reads.
template <class T, bool RESIDUAL>
__global__ void __launch_bounds__(256) gq_fp8_norm_kernel(const GqFp8Rows p) {
    __shared__ float wsum[8];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const uint8_t* xr = p.x + row * p.ld_x * Elem<T>::kBytes;
    const uint8_t* rr = RESIDUAL ? p.residual + row * p.ld_residual * Elem<T>::kBytes : nullptr;
    uint8_t* hr = RESIDUAL ? p.sum + row * p.ld_sum * Elem<T>::kBytes : nullptr;
    float ss = 0.0f;
    for (int64_t c = 8 * tid; c < p.cols; c += 2048) {
        float h[8];
        Elem<T>::load8(xr + c * Elem<T>::kBytes, h);
        if constexpr (RESIDUAL) {
            float r[8];
            Elem<T>::load8(rr + c * Elem<T>::kBytes, r);
#pragma unroll
            for (int k = 0; k < 8; ++k) h[k] = Elem<T>::round(__fadd_rn(h[k], r[k]));
            Elem<T>::store8(hr + c * Elem<T>::kBytes, h);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) ss = __fmaf_rn(h[k], h[k], ss);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, d));
    if ((tid & 31) == 0) wsum[tid >> 5] = ss;
    __syncthreads();
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __fadd_rn(ss, wsum[i]);
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(p.cols)), p.eps)));
    const int64_t padded = p.blocks * 128;
    for (int64_t c0 = 0; c0 < padded; c0 += 2048) {
        const int64_t c = c0 + 8 * tid;
        float y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (c < p.cols) {
            float w[8];
            if constexpr (RESIDUAL) {
                Elem<T>::load8(hr + c * Elem<T>::kBytes, y);   // this thread wrote these values itself
            } else {
                Elem<T>::load8(xr + c * Elem<T>::kBytes, y);
            }
            Elem<F32>::load8(p.weight + c, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = __fmul_rn(__fmul_rn(y[k], rstd), w[k]);
        }
        const uint32_t byte = scale_byte(max16(amax8(y)));
        if (c < p.cols) st_global(reinterpret_cast<uint2*>(p.codes + row * p.ld_codes + c), encode8(y, inverse_scale(byte)));
        if (c < p.cols && (tid & 15) == 0) p.scales[row * p.ld_scales + (c >> 7)] = static_cast<uint8_t>(byte);
    }
}

template <class T>
int launch_rows(const GqFp8Rows& p, cudaStream_t s) {
    if (p.weight != nullptr) {
        if (p.residual != nullptr) gq_fp8_norm_kernel<T, true><<<static_cast<unsigned>(p.rows), 256, 0, s>>>(p);
        else gq_fp8_norm_kernel<T, false><<<static_cast<unsigned>(p.rows), 256, 0, s>>>(p);
    } else {
        const int64_t want = (p.rows * p.blocks + 15) / 16;
        const unsigned grid = static_cast<unsigned>(want < 65536 ? want : 65536);
        if (p.gate != nullptr) gq_fp8_rows_kernel<T, true><<<grid, 256, 0, s>>>(p);
        else gq_fp8_rows_kernel<T, false><<<grid, 256, 0, s>>>(p);
    }
    return static_cast<int>(cudaGetLastError());
}

}  // namespace

int launch_fp8_weight(int type, GqFp8Weight& p, void* stream) {
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (type) {
        case GQ_TYPE_F32: return launch_float_weight<F32>(p, s);
        case GQ_TYPE_F16: return launch_float_weight<F16>(p, s);
        case GQ_TYPE_BF16: return launch_float_weight<BF16>(p, s);
        case GQ_TYPE_Q8_0: return launch_weight<GQ_TYPE_Q8_0>(p, s);
        case GQ_TYPE_Q4_0: return launch_weight<GQ_TYPE_Q4_0>(p, s);
        case GQ_TYPE_Q4_1: return launch_weight<GQ_TYPE_Q4_1>(p, s);
        case GQ_TYPE_Q5_0: return launch_weight<GQ_TYPE_Q5_0>(p, s);
        case GQ_TYPE_Q5_1: return launch_weight<GQ_TYPE_Q5_1>(p, s);
        case GQ_TYPE_Q2_K: return launch_weight<GQ_TYPE_Q2_K>(p, s);
        case GQ_TYPE_Q3_K: return launch_weight<GQ_TYPE_Q3_K>(p, s);
        case GQ_TYPE_Q4_K: return launch_weight<GQ_TYPE_Q4_K>(p, s);
        case GQ_TYPE_Q5_K: return launch_weight<GQ_TYPE_Q5_K>(p, s);
        case GQ_TYPE_Q6_K: return launch_weight<GQ_TYPE_Q6_K>(p, s);
        default: return static_cast<int>(cudaErrorInvalidValue);
    }
}

int launch_fp8_rows(int dtype, const GqFp8Rows& p, void* stream) {
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case GQ_TYPE_F32: return launch_rows<F32>(p, s);
        case GQ_TYPE_F16: return launch_rows<F16>(p, s);
        case GQ_TYPE_BF16: return launch_rows<BF16>(p, s);
        default: return static_cast<int>(cudaErrorInvalidValue);
    }
}

}  // namespace gq
