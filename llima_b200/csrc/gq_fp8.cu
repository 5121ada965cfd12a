// Block-scaled 8-bit floats: GGUF weights to e4m3 with one scale per 128 x 128 block, and
// activations to e4m3 with one scale per 1 x 128 block (after an RMS norm, after a gated
// activation, or as they are).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

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

// Four codes (bytes of w, offset OFF) over the block scale as four e4m3 codes: A and B are the
// block's constants already divided by the scale (a power of two, so every product and
// difference rounds as before).  A byte becomes a float by placing it under the exponent of
// 2^23 and subtracting, both exact.
template <int TYPE>
__device__ __forceinline__ uint32_t encode_codes(uint32_t w, float A, float B) {
    using V = BlockView<TYPE>;
    const float2 a = make_float2(A, A), b = make_float2(-B, -B), off = make_float2(-8388608.0f - V::OFF, -8388608.0f - V::OFF);
    uint32_t c[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float2 q = make_float2(__uint_as_float(__byte_perm(w, 0x4B000000u, 0x7650 + 2 * h)),
                                     __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7651 + 2 * h)));
        float2 x = __fmul2_rn(a, __fadd2_rn(q, off));
        if constexpr (V::kSub) x = __fadd2_rn(x, b);
        c[h] = e4m3x2(x.x, x.y);
    }
    return c[0] | (c[1] << 16);
}

// One CTA per 128 rows x 256 columns (two scale blocks).  A lane owns 32 consecutive columns of
// four rows, eight lanes a row's 256: their integer codes stay in registers between the
// block's maximum and the encoding, and a warp stores whole rows of 256 bytes.  A value is a
// monotone function of its code, so a 16- or 32-value block's largest |x| is at its smallest or
// largest code.
template <int TYPE>
__global__ void __launch_bounds__(256) gq_fp8_weight_kernel(const GqFp8Weight p) {
    using V = BlockView<TYPE>;
    using T = Fp8Tile<TYPE>;
    constexpr int NP = 32 / V::BV;                                          // blocks per 32 columns
    constexpr bool kUnits16 = TYPE == GQ_TYPE_Q4_K || TYPE == GQ_TYPE_Q5_K;   // 9 and 11 times 16 bytes
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t* wmax = reinterpret_cast<uint32_t*>(smem + 128 * T::kPitch);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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

    const int sub = lane & 7;
    const bool col_in = 32 * sub < cols;
    uint32_t w[4][8];
    float A[4][NP], B[4][NP];
    uint32_t amax = 0;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 32 * i + 4 * warp + (lane >> 3);
        if (!col_in || r >= rows) continue;
        int skew = 0;
        if constexpr (!kUnits16) skew = static_cast<int>((fp8_src_row(p.head_dim, row0 + r) * p.row_bytes + at) & 15);
        const uint8_t* row = smem + r * T::kPitch + skew;
#pragma unroll
        for (int b = 0; b < NP; ++b) {
            uint32_t words[8];
            decode_block<TYPE, kUnits16>(row, NP * sub + b, words, A[i][b], B[i][b]);
#pragma unroll
            for (int j = 0; j < V::NW; ++j) w[i][V::NW * b + j] = words[j];
            if ((__float_as_uint(A[i][b]) & 0x7FFFFFFFu) < kInfBits && (__float_as_uint(B[i][b]) & 0x7FFFFFFFu) < kInfBits) {
                uint32_t mn = 0xFFFFFFFFu, mx = 0u;
#pragma unroll
                for (int j = 0; j < V::NW; ++j) {
                    const uint32_t e = words[j] & 0x00FF00FFu, o = (words[j] >> 8) & 0x00FF00FFu;
                    mn = vmin16(mn, e, o);
                    mx = vmax16(mx, e, o);
                }
                const int lo = static_cast<int>(min(mn & 0xFFFFu, mn >> 16)) - V::OFF;
                const int hi = static_cast<int>(max(mx & 0xFFFFu, mx >> 16)) - V::OFF;
                amax = max(amax, max(finite_abs(block_value<TYPE>(A[i][b], B[i][b], lo)),
                                     finite_abs(block_value<TYPE>(A[i][b], B[i][b], hi))));
            } else {
                finite = false;
                for (int j = 0; j < V::BV; ++j) {
                    const int q = static_cast<int>(byte_of(words[j >> 2], j & 3)) - V::OFF;
                    amax = max(amax, finite_abs(block_value<TYPE>(A[i][b], B[i][b], q)));
                }
            }
        }
    }
    // lanes with equal bit 2 hold the same block's columns
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 8));
    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
    const int half = (lane >> 2) & 1;
    if ((lane & 27) == 0) wmax[8 * half + warp] = amax;
    __syncthreads();
    const uint4 m0 = *reinterpret_cast<const uint4*>(wmax + 8 * half), m1 = *reinterpret_cast<const uint4*>(wmax + 8 * half + 4);
    const uint32_t byte = scale_byte(max(max(max(m0.x, m0.y), max(m0.z, m0.w)), max(max(m1.x, m1.y), max(m1.z, m1.w))));
    const float inv = inverse_scale(byte);
    if (warp == 0 && (lane & 27) == 0 && 128 * half < cols)
        p.scales[(row0 >> 7) * p.scale_cols + (col0 >> 7) + half] = static_cast<uint8_t>(byte);
    const bool sectors = (reinterpret_cast<uintptr_t>(p.codes) & 31) == 0;    // rows are multiples of 32 bytes
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 32 * i + 4 * warp + (lane >> 3);
        if (!col_in || r >= rows) continue;
        uint32_t c[8];
        if (finite) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                c[j] = encode_codes<TYPE>(w[i][j], __fmul_rn(A[i][j / V::NW], inv), V::kSub ? __fmul_rn(B[i][j / V::NW], inv) : 0.0f);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float x[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    x[k] = __fmul_rn(nan_unless_finite(block_value<TYPE>(A[i][j / V::NW], B[i][j / V::NW],
                                                                         static_cast<int>(byte_of(w[i][j], k)) - V::OFF)), inv);
                c[j] = e4m3x2(x[0], x[1]) | (e4m3x2(x[2], x[3]) << 16);
            }
        }
        uint8_t* out = p.codes + (row0 + r) * p.cols + col0 + 32 * sub;
        if (sectors) {
            stg256(out, c);
        } else {
            stg128(out, make_uint4(c[0], c[1], c[2], c[3]));
            stg128(out + 16, make_uint4(c[4], c[5], c[6], c[7]));
        }
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

// Eight values over the block scale to eight codes.  A NaN becomes the NaN code by itself; an
// infinity would saturate, so callers that may hold one make it a NaN first (SAFE).
template <bool SAFE>
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float inv) {
    uint32_t c[4];
    const float2 s = make_float2(inv, inv);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float u = SAFE ? x[2 * i] : nan_unless_finite(x[2 * i]), v = SAFE ? x[2 * i + 1] : nan_unless_finite(x[2 * i + 1]);
        const float2 y = __fmul2_rn(make_float2(u, v), s);
        c[i] = e4m3x2(y.x, y.y);
    }
    return make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
}
__device__ __forceinline__ uint32_t amax8(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, finite_abs(x[k]));
    return m;
}
// the largest |x| with NaN left out (fmaxf does) and infinities in
__device__ __forceinline__ float amax8_or_inf(const float (&x)[8]) {
    const float a = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    const float b = fmaxf(fmaxf(fabsf(x[4]), fabsf(x[5])), fmaxf(fabsf(x[6]), fabsf(x[7])));
    return fmaxf(a, b);
}
// over the 16 lanes that hold one 128-value block
__device__ __forceinline__ uint32_t max16(uint32_t m) {
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    return m;
}

// The codes and scale byte of one 128-value block by 16 lanes, eight values each; all lanes
// of the warp call it together.
__device__ __forceinline__ uint2 quantize_block(const float (&x)[8], uint32_t& byte) {
    uint32_t m = max16(__float_as_uint(amax8_or_inf(x)));   // non-negative floats order as their bits
    if (__any_sync(0xffffffffu, m >= kInfBits)) {
        byte = scale_byte(max16(amax8(x)));
        return encode8<false>(x, inverse_scale(byte));
    }
    byte = scale_byte(m);
    return encode8<true>(x, inverse_scale(byte));
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
        if (r < p.rows && col < p.cols) st_global(reinterpret_cast<uint2*>(p.codes + r * p.cols + col), encode8<false>(x[i], inv));
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

// Rows as they are or gated: a block per 16 lanes, kSteps blocks per lane with all their loads
// ahead of the arithmetic.  Blocks are numbered through the rows (fewer than 2^31 per launch).
constexpr int kSteps = 2;
template <class T, bool GATED>
__global__ void __launch_bounds__(256) gq_fp8_rows_kernel(const GqFp8Rows p, const uint32_t count, const uint32_t mul,
                                                          const uint32_t shift) {
    constexpr int E = Elem<T>::kBytes;
    const uint32_t sub = threadIdx.x & 15;
    const uint32_t first = blockIdx.x * (16 * kSteps) + (threadIdx.x >> 4);
    uint32_t row[kSteps], col[kSteps];
    bool in[kSteps];
    float x[kSteps][8], g[GATED ? kSteps : 1][8];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const uint32_t b = first + 16 * i;
        row[i] = fast_div(b, mul, shift);
        col[i] = 128 * (b - row[i] * static_cast<uint32_t>(p.blocks)) + 8 * sub;
        in[i] = b < count && col[i] < p.cols;
#pragma unroll
        for (int k = 0; k < 8; ++k) x[i][k] = 0.0f;
        if constexpr (GATED)
#pragma unroll
            for (int k = 0; k < 8; ++k) g[i][k] = 0.0f;
        if (in[i]) {
            Elem<T>::load8(p.x + (row[i] * p.ld_x + col[i]) * E, x[i]);
            if constexpr (GATED) Elem<T>::load8(p.gate + (row[i] * p.ld_gate + col[i]) * E, g[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        gate8<GATED>(x[i], g[GATED ? i : 0]);
        uint32_t byte;
        const uint2 c = quantize_block(x[i], byte);
        if (in[i]) {
            st_global(reinterpret_cast<uint2*>(p.codes + row[i] * p.ld_codes + col[i]), c);
            if (sub == 0) p.scales[row[i] * p.ld_scales + (col[i] >> 7)] = static_cast<uint8_t>(byte);
        }
    }
}

// RMS norm of a row (with the residual's addition), one CTA per row: h stays in registers
// between the sum of squares and the codes (VPT groups of eight values per thread; 0: rows too
// long for that are read again).  The sum x + r is rounded to the input type first: the norm
// is of what the next layer reads.
template <class T, bool RESIDUAL, int VPT>
__global__ void __launch_bounds__(1024) gq_fp8_norm_kernel(const GqFp8Rows p) {
    constexpr int E = Elem<T>::kBytes;
    __shared__ float wsum[32];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, threads = blockDim.x;
    const uint8_t* xr = p.x + row * p.ld_x * E;
    const uint8_t* rr = RESIDUAL ? p.residual + row * p.ld_residual * E : nullptr;
    uint8_t* hr = RESIDUAL ? p.sum + row * p.ld_sum * E : nullptr;
    const auto add = [&](float (&h)[8], const float (&r)[8], int64_t c) {
#pragma unroll
        for (int k = 0; k < 8; ++k) h[k] = Elem<T>::round(__fadd_rn(h[k], r[k]));
        Elem<T>::store8(hr + c * E, h);
    };
    const auto squares = [](const float (&h)[8], float s) {
#pragma unroll
        for (int k = 0; k < 8; ++k) s = __fmaf_rn(h[k], h[k], s);
        return s;
    };
    float h[VPT > 0 ? VPT : 1][8];
    float ss = 0.0f;
    if constexpr (VPT > 0) {
        float r[VPT][8];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = 8 * (tid + i * threads);
#pragma unroll
            for (int k = 0; k < 8; ++k) h[i][k] = 0.0f;
            if (c < p.cols) {
                Elem<T>::load8(xr + c * E, h[i]);
                if constexpr (RESIDUAL) Elem<T>::load8(rr + c * E, r[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int64_t c = 8 * (tid + i * threads);
            if constexpr (RESIDUAL)
                if (c < p.cols) add(h[i], r[i], c);
            ss = squares(h[i], ss);
        }
    } else {
        for (int64_t c = 8 * tid; c < p.cols; c += 8 * threads) {
            Elem<T>::load8(xr + c * E, h[0]);
            if constexpr (RESIDUAL) {
                float r[8];
                Elem<T>::load8(rr + c * E, r);
                add(h[0], r, c);
            }
            ss = squares(h[0], ss);
        }
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, d));
    if (threads > 32) {
        if ((tid & 31) == 0) wsum[tid >> 5] = ss;
        __syncthreads();
        ss = (tid & 31) < (threads >> 5) ? wsum[tid & 31] : 0.0f;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xffffffffu, ss, d));
    }
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, static_cast<float>(p.cols)), p.eps)));
    const auto finish = [&](float (&y)[8], int64_t c) {
        const bool in = c < p.cols;
        if (in) {
            float w[8];
            Elem<F32>::load8(p.weight + c, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = __fmul_rn(__fmul_rn(y[k], rstd), w[k]);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = 0.0f;
        }
        uint32_t byte;
        const uint2 codes = quantize_block(y, byte);
        if (in) {
            st_global(reinterpret_cast<uint2*>(p.codes + row * p.ld_codes + c), codes);
            if ((tid & 15) == 0) p.scales[row * p.ld_scales + (c >> 7)] = static_cast<uint8_t>(byte);
        }
    };
    if constexpr (VPT > 0) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) finish(h[i], 8 * (tid + i * threads));
    } else {
        for (int64_t c0 = 0; c0 < p.cols; c0 += 8 * threads) {   // all lanes together (quantize_block)
            const int64_t c = c0 + 8 * tid;
            if (c < p.cols) Elem<T>::load8((RESIDUAL ? hr : xr) + c * E, h[0]);   // this thread wrote these values itself
            finish(h[0], c);
        }
    }
}

template <class T, bool RESIDUAL>
void launch_norm(const GqFp8Rows& p, cudaStream_t s) {
    const int64_t eights = (p.cols + 7) / 8;
    const auto threads = [&](int vpt) { return static_cast<unsigned>((eights + 32 * vpt - 1) / (32 * vpt) * 32); };
    const unsigned rows = static_cast<unsigned>(p.rows);
    if (eights <= 512) gq_fp8_norm_kernel<T, RESIDUAL, 1><<<rows, threads(1), 0, s>>>(p);
    else if (eights <= 1024) gq_fp8_norm_kernel<T, RESIDUAL, 2><<<rows, threads(2), 0, s>>>(p);
    else if (eights <= 4096) gq_fp8_norm_kernel<T, RESIDUAL, 4><<<rows, threads(4), 0, s>>>(p);
    else gq_fp8_norm_kernel<T, RESIDUAL, 0><<<rows, 1024, 0, s>>>(p);
}

template <class T>
int launch_rows(GqFp8Rows p, cudaStream_t s) {
    if (p.weight != nullptr) {
        if (p.residual != nullptr) launch_norm<T, true>(p, s);
        else launch_norm<T, false>(p, s);
        return static_cast<int>(cudaGetLastError());
    }
    if (p.blocks > INT32_MAX) return static_cast<int>(cudaErrorInvalidValue);
    uint32_t mul, shift;
    fast_div_params(static_cast<uint32_t>(p.blocks), mul, shift);
    // rows in runs of fewer than 2^31 blocks
    const int64_t run = std::max<int64_t>(1, (int64_t(1) << 30) / p.blocks), all = p.rows;
    for (int64_t r = 0; r < all; r += run) {
        p.rows = std::min(run, all - r);
        const uint32_t count = static_cast<uint32_t>(p.rows * p.blocks);
        const unsigned grid = (count + 16 * kSteps - 1) / (16 * kSteps);
        if (p.gate != nullptr) gq_fp8_rows_kernel<T, true><<<grid, 256, 0, s>>>(p, count, mul, shift);
        else gq_fp8_rows_kernel<T, false><<<grid, 256, 0, s>>>(p, count, mul, shift);
        p.x += run * p.ld_x * Elem<T>::kBytes;
        if (p.gate != nullptr) p.gate += run * p.ld_gate * Elem<T>::kBytes;
        p.codes += run * p.ld_codes;
        p.scales += run * p.ld_scales;
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
