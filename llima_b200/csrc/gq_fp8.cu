// Block-scaled 8-bit floats: GGUF weights to e4m3 with one scale per 128 x 128 block, and
// activations to e4m3 with one scale per 1 x 128 block (after an RMS norm, after a gated
// activation, or as they are).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gq_blocks.cuh"
#include "gq_fp8.cuh"
#include "gq_internal.h"
#include "gq_launch.h"
#include "gq_tcgen05.cuh"

namespace gq {
namespace {

// Sticky error flags of this device's weight kernels (kErrWaitTimeout).
__device__ unsigned int gq_fp8_errors;

// ---------------------------------------------------------------------------------------
// Weights
// ---------------------------------------------------------------------------------------

// Source row of output row o (inverse of the llama q/k permutation: row 2a + t of a head
// moves to t * D/2 + a, gguf_conversion.py:314-332).
__device__ __forceinline__ int64_t fp8_src_row(uint32_t head_dim, uint32_t o) {
    if (head_dim == 0) return o;
    const uint32_t h = o / head_dim, rem = o - h * head_dim, half = head_dim >> 1;
    const uint32_t t = rem >= half ? 1u : 0u;
    return h * head_dim + 2 * (rem - t * half) + t;
}

// A tile is 128 rows x 256 columns, two scale blocks.  Shared bytes per row: the 16-byte-aligned
// window around the row's bytes, an odd number of 16-byte chunks so that lanes on neighbouring
// rows read different banks.
template <int TYPE>
struct Fp8Tile {
    static constexpr int kThreads = 512;
    static constexpr int kStages = 2;
    static constexpr int kChunkBytes = 256 / BlockView<TYPE>::kUnitValues * BlockView<TYPE>::kUnitBytes;
    static constexpr int kPitch = 16 * (((kChunkBytes + 15 + 15) / 16) | 1);
    static constexpr int kStageBytes = 128 * kPitch + 128;     // decoding may read a word past a row
    static constexpr int kSmem = kStages * kStageBytes + kStages * 8 + 3 * 2 * 4;
    static constexpr int kPerSm = 2;
};

// One 16- or 32-value block's codes as f16 pairs (exact) ...
template <int TYPE>
__device__ __forceinline__ void codes_to_half(const uint32_t* w, __half2* q) {
    using V = BlockView<TYPE>;
    // a byte under the exponent byte of 1024 is the f16 1024 + v
    const __half2 off = __float2half2_rn(-1024.0f - V::OFF);
#pragma unroll
    for (int j = 0; j < V::NW; ++j) {
        q[2 * j] = __hadd2_rn(u32_as_h2(__byte_perm(w[j], 0x64646464u, 0x4140)), off);
        q[2 * j + 1] = __hadd2_rn(u32_as_h2(__byte_perm(w[j], 0x64646464u, 0x4342)), off);
    }
}

// ... and its largest |x| as float bits: a value is a monotone function of its code, so it is at
// the smallest or the largest code.  At or above kInfBits where a constant is not finite.
template <int TYPE>
__device__ __forceinline__ uint32_t block_amax(const __half2* q, float A, float B) {
    using V = BlockView<TYPE>;
    if constexpr (V::kSub) {
        __half2 mn = q[0], mx = q[0];
#pragma unroll
        for (int j = 1; j < 2 * V::NW; ++j) {
            mn = __hmin2(mn, q[j]);
            mx = __hmax2(mx, q[j]);
        }
        const float lo = __half2float(__hmin(__low2half(mn), __high2half(mn)));
        const float hi = __half2float(__hmax(__low2half(mx), __high2half(mx)));
        return max(__float_as_uint(__fsub_rn(__fmul_rn(A, lo), B)) & 0x7FFFFFFFu,
                   __float_as_uint(__fsub_rn(__fmul_rn(A, hi), B)) & 0x7FFFFFFFu);
    } else {
        uint32_t m;
        memcpy(&m, &q[0], 4);
#pragma unroll
        for (int j = 1; j < 2 * V::NW; ++j) {
            uint32_t x;
            memcpy(&x, &q[j], 4);
            asm("max.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(m) : "r"(x));   // magnitudes; the signs mean nothing
        }
        const float hi = fmaxf(fabsf(h2f(m)), fabsf(h2f(m >> 16)));
        return __float_as_uint(__fmul_rn(A, hi)) & 0x7FFFFFFFu;
    }
}

// One x of a code's f16 value, as gguf-py computes it
template <int TYPE>
__device__ __forceinline__ float half_value(float A, float B, __half q) {
    const float x = __fmul_rn(A, __half2float(q));
    return BlockView<TYPE>::kSub ? __fsub_rn(x, B) : x;
}

// The largest finite |x| of a block whose constants are not all finite
template <int TYPE>
__device__ __forceinline__ uint32_t finite_amax(const __half2* q, float A, float B) {
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 2 * BlockView<TYPE>::NW; ++j)
        m = max(m, max(finite_abs(half_value<TYPE>(A, B, __low2half(q[j]))), finite_abs(half_value<TYPE>(A, B, __high2half(q[j])))));
    return m;
}

// 32 codes over the block scale as e4m3.  The constants are divided by the scale, a power of two,
// so that every product and difference rounds as before.
template <int TYPE, bool CHECK>
__device__ __forceinline__ void encode32(const __half2* q, const float* A, const float* B, float inv, uint32_t (&c)[8]) {
    using V = BlockView<TYPE>;
#pragma unroll
    for (int b = 0; b < 32 / V::BV; ++b) {
        const float a = __fmul_rn(A[b], inv), nb = V::kSub ? -__fmul_rn(B[b], inv) : 0.0f;
        const float2 a2 = make_float2(a, a), nb2 = make_float2(nb, nb);
#pragma unroll
        for (int j = V::NW * b; j < V::NW * (b + 1); ++j) {
            float2 x = __fmul2_rn(a2, __half22float2(q[2 * j])), y = __fmul2_rn(a2, __half22float2(q[2 * j + 1]));
            if constexpr (V::kSub) {
                x = __fadd2_rn(x, nb2);
                y = __fadd2_rn(y, nb2);
            }
            if constexpr (CHECK) {
                x = make_float2(nan_unless_finite(x.x), nan_unless_finite(x.y));
                y = make_float2(nan_unless_finite(y.x), nan_unless_finite(y.y));
            }
            c[j] = e4m3x4(x.x, x.y, y.x, y.y);
        }
    }
}

// A persistent grid of CTAs with a ring of two tiles each, loaded two tiles ahead.  BOXES: the
// rows' windows arrive as boxes of a tensor map (columns of 4 bytes, the two rows of a permuted
// pair, pairs), issued by one thread; p.box_rows rows to a box.  That takes rows of whole 16
// bytes, and heads whose half is 8, 16, 32 or 64 rows or a multiple of 128.  Otherwise every row's
// window is a bulk copy of its own, which costs a loop over lanes (28 against 26 us for Q6_K
// 4096 x 14336).  A lane owns 32 consecutive columns of two
// rows, eight lanes a row's 256: their codes stay in registers between the block's maximum and
// the encoding (and the stage is free for the next copy), and a warp stores whole rows of 256
// bytes.  The arithmetic is placed on the half-rate integer pipe as little as possible: codes
// become f16 pairs by one permute and one add, the maximum is taken two at a time.
template <int TYPE, bool BOXES>
__global__ void __launch_bounds__(Fp8Tile<TYPE>::kThreads, Fp8Tile<TYPE>::kPerSm) gq_fp8_weight_kernel(
    const __grid_constant__ CUtensorMap map, const GqFp8Weight p) {
    using V = BlockView<TYPE>;
    using T = Fp8Tile<TYPE>;
    constexpr int NP = 32 / V::BV, NR = 2;                                  // blocks per 32 columns, rows per lane
    constexpr uint32_t kGaveUp = 0xFFFFFFFFu;                               // above the bits of every finite magnitude
    constexpr bool kUnits16 = TYPE == GQ_TYPE_Q4_K || TYPE == GQ_TYPE_Q5_K;   // 9 and 11 times 16 bytes
    extern __shared__ __align__(128) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + T::kStages * T::kStageBytes);
    uint32_t* wmax = reinterpret_cast<uint32_t*>(bars + T::kStages);     // [turn % 3][half]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int s = 0; s < T::kStages; ++s) mbar_init(bars + s, BOXES ? 1 : 128);
        mbar_init_fence();
        for (int i = 0; i < 6; ++i) wmax[i] = 0;
    }
    __syncthreads();
    // no let_next(): the next kernel's CTAs would take the free halves of some SMs (1024 x 4096 3.5
    // against 4.8 us, back to back)
    after_previous();
    const uint32_t all_rows = static_cast<uint32_t>(p.rows), all_cols = static_cast<uint32_t>(p.cols);
    constexpr uint32_t kColBytes = T::kChunkBytes;         // of 256 columns
    const auto issue = [&](uint32_t t, int s) {
        const uint32_t tile_r = fast_div(t, p.ncol_mul, p.ncol_shift), tile_c = t - tile_r * p.n_col_tiles;
        if constexpr (BOXES) {
            if (warp == 0 && tc::elect()) {
                const uint32_t bar = smem_u32addr(bars + s), x = tile_c * kColBytes / 16 * 4;
                tc::arrive_expect(bar, 128 * T::kPitch);
                for (uint32_t r = 0; r < 128; r += p.box_rows) {
                    uint32_t o = tile_r * 128 + r, second = 0;
                    if (p.head_dim != 0) {
                        const uint32_t h = o / p.head_dim, rem = o - h * p.head_dim, hd = p.head_dim >> 1;
                        second = rem >= hd ? 1u : 0u;
                        o = h * hd + rem - second * hd;
                    }
                    tc::load_box(smem_u32addr(smem + s * T::kStageBytes + r * T::kPitch), &map, static_cast<int>(x),
                                 static_cast<int>(second), static_cast<int>(o), bar);
                }
            }
            return;
        }
        if (tid >= 128) return;                      // one row each
        const uint32_t bytes = min(256u, all_cols - 256 * tile_c) / V::kUnitValues * V::kUnitBytes;
        uint32_t whole = 0;
        const uint8_t* from = nullptr;
        uint8_t* to = smem + s * T::kStageBytes + tid * T::kPitch;
        if (tile_r * 128 + tid < all_rows) {
            const int64_t start = fp8_src_row(p.head_dim, tile_r * 128 + tid) * p.row_bytes + static_cast<int64_t>(tile_c) * kColBytes;
            const uint32_t skew = static_cast<uint32_t>(start) & 15u;
            from = p.src + (start - skew);
            whole = (skew + bytes + 15u) & ~15u;
            const int64_t left = p.src_bytes - (start - skew);
            if (whole > left) {
                // the tensor's last bytes, when they are no whole 16
                whole = static_cast<uint32_t>(left) & ~15u;
                for (int64_t i = whole; i < left; ++i) to[i] = from[i];
            }
        }
        mbar_arrive_expect_tx(bars + s, whole);
        if (whole != 0) bulk_load(to, from, whole, bars + s);
    };
    for (int s = 0; s < T::kStages; ++s)
        if (blockIdx.x + s * gridDim.x < p.n_tiles) issue(blockIdx.x + s * gridDim.x, s);

    const int sub = lane & 7, half = (lane >> 2) & 1;
    const bool sectors = (reinterpret_cast<uintptr_t>(p.codes) & 31) == 0;    // rows are multiples of 32 bytes
    // what does not change from tile to tile: this lane's first row and its place in the output
    const uint32_t my_row = 4 * warp + (lane >> 3);
    uint8_t* const my_out = p.codes + static_cast<int64_t>(my_row) * p.cols + 32 * sub;
    const uint8_t* const my_smem = smem + my_row * T::kPitch;
    const uint32_t row_bytes16 = static_cast<uint32_t>(p.row_bytes) & 15u;
    int s = 0;
    uint32_t parity = 0, turn = 0, t = blockIdx.x;
    for (; t < p.n_tiles; t += gridDim.x) {
        // a wait that gave up ends the loop for all threads together, at this tile's barrier
        if (!mbar_wait(bars + s, parity)) {
            atomicOr(&gq_fp8_errors, kErrWaitTimeout);
            atomicMax(wmax + 2 * turn, kGaveUp);
            atomicMax(wmax + 2 * turn + 1, kGaveUp);
        }
        const uint32_t tile_r = fast_div(t, p.ncol_mul, p.ncol_shift), tile_c = t - tile_r * p.n_col_tiles;
        const uint32_t row0 = tile_r * 128, rows = all_rows - row0, cols = all_cols - 256 * tile_c;    // left from here on
        const bool col_in = static_cast<uint32_t>(32 * sub) < cols;
        __half2 q[NR][16];
        float A[NR][NP], B[NR][NP];
        uint32_t amax = 0;
        bool finite = true;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            if (!col_in || my_row + 64 * i >= rows) continue;
            uint32_t skew = 0;
            if constexpr (!kUnits16)
                skew = (static_cast<uint32_t>(fp8_src_row(p.head_dim, row0 + my_row + 64 * i)) * row_bytes16 + tile_c * kColBytes) & 15u;
            uint32_t w[8];
            decode32<TYPE, kUnits16>(my_smem + s * T::kStageBytes + 64 * i * T::kPitch + skew, sub, w, A[i], B[i]);
#pragma unroll
            for (int b = 0; b < NP; ++b) {
                codes_to_half<TYPE>(w + V::NW * b, q[i] + 2 * V::NW * b);
                uint32_t m = block_amax<TYPE>(q[i] + 2 * V::NW * b, A[i][b], B[i][b]);
                if (m >= kInfBits) {
                    finite = false;
                    m = finite_amax<TYPE>(q[i] + 2 * V::NW * b, A[i][b], B[i][b]);
                }
                amax = max(amax, m);
            }
        }
        // lanes with equal bit 2 hold the same block's columns
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 8));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 16));
        // joined over the warps in one of three places in turn; the next turn's is cleared here,
        // after its last reading and before its next use
        uint32_t* const wm = wmax + 2 * turn + half;
        turn = turn == 2 ? 0 : turn + 1;
        if ((lane & 27) == 0) {
            atomicMax(wm, amax);
            if (warp == 0) wmax[2 * turn + half] = 0;
        }
        __syncthreads();
        const uint32_t block_amax_bits = *wm;
        if (block_amax_bits == kGaveUp) break;
        // every thread is done with the stage
        if (t + T::kStages * gridDim.x < p.n_tiles) issue(t + T::kStages * gridDim.x, s);
        if (++s == T::kStages) {
            s = 0;
            parity ^= 1;
        }
        const uint32_t byte = scale_byte(block_amax_bits);
        const float inv = inverse_scale(byte);
        if (warp == 0 && (lane & 27) == 0 && static_cast<uint32_t>(128 * half) < cols)
            p.scales[static_cast<int64_t>(tile_r) * p.scale_cols + 2 * tile_c + half] = static_cast<uint8_t>(byte);
        // a warp with a value that is not finite takes its own way
        const bool plain = __all_sync(0xffffffffu, finite);
        uint8_t* out = my_out + (static_cast<int64_t>(row0) * p.cols + 256 * tile_c);
#pragma unroll
        for (int i = 0; i < NR; ++i, out += 64 * p.cols) {
            if (!col_in || my_row + 64 * i >= rows) continue;
            uint32_t c[8];
            if (plain) encode32<TYPE, false>(q[i], A[i], B[i], inv, c);
            else encode32<TYPE, true>(q[i], A[i], B[i], inv, c);
            if (sectors) {
                stg256(out, c);
            } else {
                stg128(out, make_uint4(c[0], c[1], c[2], c[3]));
                stg128(out + 16, make_uint4(c[4], c[5], c[6], c[7]));
            }
        }
    }
    // After a wait that gave up, this CTA's copies have as long again to land before it ends (waiting
    // on their barriers keeps state in registers through the loop: up to 60 bytes of spills, 15%).
    if (t < p.n_tiles)
        for (const uint64_t t0 = global_ns(); global_ns() - t0 < kWaitLimitNs;) {
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
};

// Eight values over the block scale to eight codes
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float inv) {
    uint32_t c[2];
    const float2 s = make_float2(inv, inv);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 y = __fmul2_rn(make_float2(nan_unless_finite(x[4 * i]), nan_unless_finite(x[4 * i + 1])), s);
        const float2 z = __fmul2_rn(make_float2(nan_unless_finite(x[4 * i + 2]), nan_unless_finite(x[4 * i + 3])), s);
        c[i] = e4m3x4(y.x, y.y, z.x, z.y);
    }
    return make_uint2(c[0], c[1]);
}
__device__ __forceinline__ uint32_t amax8(const float (&x)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, finite_abs(x[k]));
    return m;
}

// Weights of a float type: one CTA per 128 x 128 block, thread t the 8 columns 8 (t % 16) of
// rows t / 16 + 16 i, held in registers between the block's maximum and the codes.
template <class T>
__global__ void __launch_bounds__(256) gq_fp8_float_weight_kernel(const GqFp8Weight p) {
    __shared__ uint32_t wmax[8];
    const int tid = threadIdx.x;
    let_next();
    after_previous();
    const int64_t row0 = static_cast<int64_t>(blockIdx.x / p.n_col_tiles) * 128;
    const int64_t col = static_cast<int64_t>(blockIdx.x % p.n_col_tiles) * 128 + 8 * (tid & 15);
    float x[8][8];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t r = row0 + (tid >> 4) + 16 * i;
        if (r < p.rows && col < p.cols) {
            Elem<T>::load8(p.src + fp8_src_row(p.head_dim, static_cast<uint32_t>(r)) * p.row_bytes + col * Elem<T>::kBytes, x[i]);
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
    static std::atomic<uint64_t> allowed[2]{};
    const int64_t hd = p.head_dim / 2;
    // boxes start on 128 bytes in shared memory: eight rows at least
    const bool boxes = p.row_bytes % 16 == 0 && (hd == 0 || (hd >= 8 && (128 % hd == 0 || hd % 128 == 0)));
    auto kern = boxes ? gq_fp8_weight_kernel<TYPE, true> : gq_fp8_weight_kernel<TYPE, false>;
    int sms = 0;
    cudaError_t e = sm_count(sms);
    if (e == cudaSuccess) e = allow_smem(kern, T::kSmem, allowed[boxes]);
    if (e != cudaSuccess) return static_cast<int>(e);
    CUtensorMap map{};
    if (boxes) {
        p.box_rows = static_cast<uint32_t>(hd == 0 ? 128 : std::min<int64_t>(hd, 128));
        const cuuint64_t per = hd == 0 ? 1 : 2;
        const cuuint64_t dims[3] = {static_cast<cuuint64_t>(p.row_bytes / 4), per, static_cast<cuuint64_t>(p.rows) / per};
        const cuuint64_t strides[2] = {static_cast<cuuint64_t>(p.row_bytes), per * static_cast<cuuint64_t>(p.row_bytes)};
        const cuuint32_t box[3] = {T::kPitch / 4, 1, p.box_rows};
        const int st = encode_map(&map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, p.src, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
        if (st != 0) return st;
    }
    p.n_col_tiles = static_cast<uint32_t>((p.cols + 255) / 256);
    p.n_tiles = static_cast<uint32_t>((p.rows + 127) / 128 * p.n_col_tiles);
    fast_div_params(p.n_col_tiles, p.ncol_mul, p.ncol_shift);
    const uint32_t most = static_cast<uint32_t>(sms * T::kPerSm);
    return launch_early(kern, std::min(p.n_tiles, most), T::kThreads, T::kSmem, s, 1, map, p);
}
template <class T>
int launch_float_weight(GqFp8Weight& p, cudaStream_t s) {
    p.n_col_tiles = static_cast<uint32_t>((p.cols + 127) / 128);
    const int64_t tiles = (p.rows + 127) / 128 * p.n_col_tiles;
    return launch_early(gq_fp8_float_weight_kernel<T>, static_cast<unsigned>(tiles), 256, 0, s, 1, p);
}

// ---------------------------------------------------------------------------------------
// Activations: 16 consecutive values per lane, eight lanes per 128-value block
// ---------------------------------------------------------------------------------------

// 16 values as they lie in memory.  Rows start on 16-byte boundaries; where they start on 32
// (WIDE, the same for a whole launch) one load takes 32 bytes.
template <class T>
struct Raw16 {
    static constexpr int kWords = 4 * Elem<T>::kBytes;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const uint8_t* p, bool wide) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < kWords; i += 8)
                asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]), "=r"(w[i + 5]),
                               "=r"(w[i + 6]), "=r"(w[i + 7])
                             : "l"(p + 4 * i));
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 4)
                asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3])
                             : "l"(p + 4 * i));
        }
    }
    __device__ __forceinline__ void store(uint8_t* p, bool wide) const {
#pragma unroll
        for (int i = 0; i < kWords; i += 8) {
            if (wide) {
                const uint32_t v[8] = {w[i], w[i + 1], w[i + 2], w[i + 3], w[i + 4], w[i + 5], w[i + 6], w[i + 7]};
                stg256(p + 4 * i, v);
            } else {
                stg128(p + 4 * i, make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]));
                stg128(p + 4 * i + 16, make_uint4(w[i + 4], w[i + 5], w[i + 6], w[i + 7]));
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    // value pair i of 8
    __device__ __forceinline__ float2 get(int i) const {
        if constexpr (std::is_same<T, F32>::value) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else return widen(w[i]);
    }
    static __device__ __forceinline__ float2 widen(uint32_t v) {
        if constexpr (std::is_same<T, F16>::value) return __half22float2(u32_as_h2(v));
        else return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    }
    // one pair on its own
    static __device__ __forceinline__ float2 load2(const uint8_t* p) {
        uint32_t a, b;
        if constexpr (std::is_same<T, F32>::value) {
            asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "l"(p));
            return make_float2(__uint_as_float(a), __uint_as_float(b));
        } else {
            asm volatile("ld.global.b32 %0, [%1];" : "=r"(a) : "l"(p));
            return widen(a);
        }
    }
    // rounds to the type
    __device__ __forceinline__ void set(int i, float2 v) {
        if constexpr (std::is_same<T, F32>::value) {
            w[2 * i] = __float_as_uint(v.x);
            w[2 * i + 1] = __float_as_uint(v.y);
        } else if constexpr (std::is_same<T, F16>::value) {
            const __half2 h = __float22half2_rn(v);
            memcpy(&w[i], &h, 4);
        } else {
            const __nv_bfloat162 h = __float22bfloat162_rn(v);
            memcpy(&w[i], &h, 4);
        }
    }
};

// over the eight lanes that hold one 128-value block
__device__ __forceinline__ uint32_t max8(uint32_t m) {
#pragma unroll
    for (int d = 4; d > 0; d >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, d));
    return m;
}

// The codes and scale byte of one 128-value block by eight lanes, 16 values each; all lanes of
// the warp call it together.  fmaxf leaves NaN out, and NaN becomes its code by itself; an
// infinity shows in the maximum, and then the values are looked at one by one.
__device__ __forceinline__ uint4 quantize_block(float2 (&y)[8], uint32_t& byte) {
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        m[i] = fmaxf(fmaxf(fabsf(y[2 * i].x), fabsf(y[2 * i].y)), fmaxf(fabsf(y[2 * i + 1].x), fabsf(y[2 * i + 1].y)));
    // non-negative floats order as their bits
    uint32_t amax = max8(__float_as_uint(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]))));
    if (__any_sync(0xffffffffu, amax >= kInfBits)) {
        amax = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            amax = max(amax, max(finite_abs(y[i].x), finite_abs(y[i].y)));
            y[i] = make_float2(nan_unless_finite(y[i].x), nan_unless_finite(y[i].y));
        }
        amax = max8(amax);
    }
    byte = scale_byte(amax);
    const float inv = inverse_scale(byte);
    const float2 s = make_float2(inv, inv);
    uint32_t c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 u = __fmul2_rn(y[2 * i], s), v = __fmul2_rn(y[2 * i + 1], s);
        c[i] = e4m3x4(u.x, u.y, v.x, v.y);
    }
    return make_uint4(c[0], c[1], c[2], c[3]);
}

// silu(g) * x = g / (1 + exp(-g)) * x of two values, and the least quotient so far.  The hardware's
// reciprocal gives 0 below the normal range, from g = -87.3 down; where a quotient is 0 the values
// are taken from far_silu_times.  Relative error of both: an exponent off by 1.25 * 2^-24 of itself
// (the product and the constant) shows as |g| 2^-23.7, the hardware's approximations are off by 2^-22
// for each exponential and 2^-23 for the quotient, each rounding by 2^-24: under |g| 2^-23 + 2^-20,
// where a code keeps four bits.  A g that is not finite gives NaN or an infinity.
__device__ __forceinline__ float2 silu_times(float2 g, float2 x, float& least) {
    constexpr float kC = -1.44269504f;      // -1 / ln 2
    const float2 t = __fmul2_rn(g, make_float2(kC, kC));
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    e = __fadd2_rn(e, make_float2(1.0f, 1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(e.y));
    least = fminf(fminf(r.x, r.y), least);
    return __fmul2_rn(__fmul2_rn(g, r), x);
}

// The same with u = exp(-|g| / 2): g / (1 + u^2) * x, for g < 0 times u^2, one u to each factor.
// Nothing overflows, and no factor leaves the normal range before |g| = 174.
__device__ __forceinline__ float2 far_silu_times(float2 g, float2 x) {
    constexpr float kC = -0.72134752f;      // -1 / (2 ln 2)
    float2 u, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(u.x) : "f"(__fmul_rn(fabsf(g.x), kC)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(u.y) : "f"(__fmul_rn(fabsf(g.y), kC)));
    const float2 s = __ffma2_rn(u, u, make_float2(1.0f, 1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(s.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(s.y));
    const float2 v = make_float2(g.x < 0.0f ? u.x : 1.0f, g.y < 0.0f ? u.y : 1.0f);
    return __fmul2_rn(__fmul2_rn(__fmul2_rn(g, r), v), __fmul2_rn(x, v));
}

// Rows as they are or gated, a block per eight lanes.  Blocks are numbered through the rows
// (fewer than 2^31 per launch).  Six CTAs to an SM for gated rows of 16-bit values: they
// need the loads of so many in flight (4096 x 14336 42.7 us; 43.6 with five, 51.6 with eight, whose
// 32 registers spill); the others as the compiler has them (0).
template <class T, bool GATED>
__global__ void __launch_bounds__(256, GATED && Elem<T>::kBytes == 2 ? 6 : 0) gq_fp8_rows_kernel(const GqFp8Rows p, const uint32_t count, const uint32_t mul,
                                                          const uint32_t shift, const bool wide) {
    constexpr int E = Elem<T>::kBytes;
    let_next();
    after_previous();
    const uint32_t sub = threadIdx.x & 7;
    const uint32_t b = blockIdx.x * 32 + (threadIdx.x >> 3);
    const uint32_t row = fast_div(b, mul, shift);
    const uint32_t kb = b - row * static_cast<uint32_t>(p.blocks), col = 128 * kb + 16 * sub;
    const bool in = b < count && col < p.cols;
    Raw16<T> x, g;
    x.clear();
    if constexpr (GATED) g.clear();
    if (in) {
        x.load(p.x + (row * p.ld_x + col) * E, wide);
        if constexpr (GATED) g.load(p.gate + (row * p.ld_gate + col) * E, wide);
    }
    float2 y[8];
    float least = 1.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = x.get(i);
        if constexpr (GATED) y[i] = silu_times(g.get(i), y[i], least);
    }
    if constexpr (GATED) {
        // loaded again, a pair at a time, so that this way costs no registers
        if (least == 0.0f) {
            const uint8_t* const from_x = p.x + (row * p.ld_x + col) * E;
            const uint8_t* const from_g = p.gate + (row * p.ld_gate + col) * E;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                y[i] = far_silu_times(Raw16<T>::load2(from_g + 2 * i * E), Raw16<T>::load2(from_x + 2 * i * E));
        }
    }
    uint32_t byte;
    const uint4 c = quantize_block(y, byte);
    if (in) {
        stg128(p.codes + row * p.ld_codes + col, c);
        if (sub == 0) p.scales[row * p.ld_scales + kb] = static_cast<uint8_t>(byte);
    }
}

// RMS norm of rows (with the residual's addition): a CTA takes rows one after another, each
// lane NV groups of 16 values of every row.  h stays in registers between the sum of squares
// and the codes; with one group per lane the weights stay there too and the next row's loads
// are issued before this row's sum is joined.  The sum x + r is rounded to the input type
// first: the norm is of what the next layer reads.
template <class T, bool RESIDUAL, int NV>
__global__ void __launch_bounds__(512) gq_fp8_norm_kernel(const GqFp8Rows p, const bool wide) {
    constexpr int E = Elem<T>::kBytes;
    __shared__ float wsum[2][16];
    const int tid = threadIdx.x, threads = blockDim.x;
    const auto column = [&](int i) { return 16 * (static_cast<int64_t>(tid) + static_cast<int64_t>(i) * threads); };
    const auto fetch = [&](int64_t row, int i, Raw16<T>& x, Raw16<T>& r) {
        const int64_t c = column(i);
        x.clear();
        if constexpr (RESIDUAL) r.clear();
        if (row < p.rows && c < p.cols) {
            x.load(p.x + (row * p.ld_x + c) * E, wide);
            if constexpr (RESIDUAL) r.load(p.residual + (row * p.ld_residual + c) * E, wide);
        }
    };
    let_next();
    after_previous();
    float4 weight[NV == 1 ? 4 : 1];
    if constexpr (NV == 1) {
        if (column(0) < p.cols)
#pragma unroll
            for (int j = 0; j < 4; ++j) weight[j] = reinterpret_cast<const float4*>(p.weight + column(0))[j];
    }
    Raw16<T> x[NV], r[RESIDUAL ? NV : 1];
#pragma unroll
    for (int i = 0; i < NV; ++i) fetch(blockIdx.x, i, x[i], r[RESIDUAL ? i : 0]);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        Raw16<T> h[NV];
        float2 ss = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if constexpr (RESIDUAL) h[i].set(k, __fadd2_rn(x[i].get(k), r[i].get(k)));
                const float2 v = RESIDUAL ? h[i].get(k) : x[i].get(k);
                ss = __ffma2_rn(v, v, ss);
            }
            if constexpr (RESIDUAL) {
                if (column(i) < p.cols) h[i].store(p.sum + (row * p.ld_sum + column(i)) * E, wide);
            } else {
                h[i] = x[i];
            }
        }
        if constexpr (NV == 1) fetch(row + gridDim.x, 0, x[0], r[0]);
        float s = __fadd_rn(ss.x, ss.y);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, d));
        if (threads > 32) {
            if ((tid & 31) == 0) wsum[turn][tid >> 5] = s;
            __syncthreads();
            s = (tid & 15) < (threads >> 5) ? wsum[turn][tid & 15] : 0.0f;
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, d));
        }
        const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(s, static_cast<float>(p.cols)), p.eps)));
        const float2 rs = make_float2(rstd, rstd);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = column(i);
            const bool in = c < p.cols;
            float2 y[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if constexpr (NV == 1) w = weight[j];
                else if (in) w = reinterpret_cast<const float4*>(p.weight + c)[j];
                y[2 * j] = __fmul2_rn(__fmul2_rn(h[i].get(2 * j), rs), make_float2(w.x, w.y));
                y[2 * j + 1] = __fmul2_rn(__fmul2_rn(h[i].get(2 * j + 1), rs), make_float2(w.z, w.w));
            }
            if (!in)
#pragma unroll
                for (int k = 0; k < 8; ++k) y[k] = make_float2(0.0f, 0.0f);
            uint32_t byte;
            const uint4 codes = quantize_block(y, byte);
            if (in) {
                stg128(p.codes + row * p.ld_codes + c, codes);
                if ((tid & 7) == 0) p.scales[row * p.ld_scales + (c >> 7)] = static_cast<uint8_t>(byte);
            }
        }
        if constexpr (NV > 1)
#pragma unroll
            for (int i = 0; i < NV; ++i) fetch(row + gridDim.x, i, x[i], r[RESIDUAL ? i : 0]);
    }
}

// Rows too long for registers: the sum of squares in one pass, the codes in another that reads
// h again.
template <class T, bool RESIDUAL>
__global__ void __launch_bounds__(512) gq_fp8_long_norm_kernel(const GqFp8Rows p, const bool wide) {
    constexpr int E = Elem<T>::kBytes;
    __shared__ float wsum[16];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    let_next();
    after_previous();
    const uint8_t* from = p.x + row * p.ld_x * E;
    float2 ss = make_float2(0.0f, 0.0f);
    for (int64_t c = 16 * tid; c < p.cols; c += 16 * 512) {
        Raw16<T> x;
        x.load(from + c * E, wide);
        if constexpr (RESIDUAL) {
            Raw16<T> r;
            r.load(p.residual + (row * p.ld_residual + c) * E, wide);
#pragma unroll
            for (int k = 0; k < 8; ++k) x.set(k, __fadd2_rn(x.get(k), r.get(k)));
            x.store(p.sum + (row * p.ld_sum + c) * E, wide);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) ss = __ffma2_rn(x.get(k), x.get(k), ss);
    }
    float s = __fadd_rn(ss.x, ss.y);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, d));
    if ((tid & 31) == 0) wsum[tid >> 5] = s;
    __syncthreads();
    s = wsum[tid & 15];
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, d));
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(s, static_cast<float>(p.cols)), p.eps)));
    if constexpr (RESIDUAL) from = p.sum + row * p.ld_sum * E;      // what this thread wrote itself
    for (int64_t c0 = 0; c0 < p.cols; c0 += 16 * 512) {           // all lanes together (quantize_block)
        const int64_t c = c0 + 16 * tid;
        const bool in = c < p.cols;
        float2 y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = make_float2(0.0f, 0.0f);
        if (in) {
            Raw16<T> h;
            h.load(from + c * E, wide);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float2 w = reinterpret_cast<const float2*>(p.weight + c)[k], v = h.get(k);
                y[k] = make_float2(__fmul_rn(__fmul_rn(v.x, rstd), w.x), __fmul_rn(__fmul_rn(v.y, rstd), w.y));
            }
        }
        uint32_t byte;
        const uint4 codes = quantize_block(y, byte);
        if (in) {
            stg128(p.codes + row * p.ld_codes + c, codes);
            if ((tid & 7) == 0) p.scales[row * p.ld_scales + (c >> 7)] = static_cast<uint8_t>(byte);
        }
    }
}

template <class T, bool RESIDUAL, int NV>
int launch_norm_rows(const GqFp8Rows& p, bool wide, cudaStream_t s) {
    auto kern = gq_fp8_norm_kernel<T, RESIDUAL, NV>;
    const int threads = static_cast<int>(((p.cols + 15) / 16 + 32 * NV - 1) / (32 * NV) * 32);
    int sms = 0, per = 0;
    const cudaError_t e = sm_count(sms);
    if (e != cudaSuccess) return static_cast<int>(e);
    int64_t grid = p.rows;
    if (grid > sms) {
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, threads, 0);
        grid = std::min<int64_t>(grid, static_cast<int64_t>(sms) * std::max(per, 1));
    }
    return launch_early(kern, static_cast<unsigned>(grid), threads, 0, s, 1, p, wide);
}

template <class T, bool RESIDUAL>
int launch_norm(const GqFp8Rows& p, bool wide, cudaStream_t s) {
    if (p.cols <= 8192) return launch_norm_rows<T, RESIDUAL, 1>(p, wide, s);
    if (p.cols <= 16384) return launch_norm_rows<T, RESIDUAL, 2>(p, wide, s);
    return launch_early(gq_fp8_long_norm_kernel<T, RESIDUAL>, static_cast<unsigned>(p.rows), 512, 0, s, 1, p, wide);
}

// every row starts on a 32-byte boundary
bool rows32(const void* p, int64_t ld, int64_t rows, int elem_bytes) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 31) == 0 && (rows <= 1 || (ld * elem_bytes) % 32 == 0));
}

template <class T>
int launch_rows(GqFp8Rows p, cudaStream_t s) {
    constexpr int E = Elem<T>::kBytes;
    const bool wide = rows32(p.x, p.ld_x, p.rows, E) && rows32(p.gate, p.ld_gate, p.rows, E) &&
                      rows32(p.residual, p.ld_residual, p.rows, E) && rows32(p.sum, p.ld_sum, p.rows, E);
    if (p.weight != nullptr) {
        return p.residual != nullptr ? launch_norm<T, true>(p, wide, s) : launch_norm<T, false>(p, wide, s);
    }
    uint32_t mul, shift;
    fast_div_params(static_cast<uint32_t>(p.blocks), mul, shift);
    // rows in runs of fewer than 2^31 blocks
    const int64_t run = std::max<int64_t>(1, (int64_t(1) << 30) / p.blocks), all = p.rows;
    for (int64_t r = 0; r < all; r += run) {
        p.rows = std::min(run, all - r);
        const uint32_t count = static_cast<uint32_t>(p.rows * p.blocks);
        auto kern = p.gate != nullptr ? gq_fp8_rows_kernel<T, true> : gq_fp8_rows_kernel<T, false>;
        const int e = launch_early(kern, (count + 31) / 32, 256, 0, s, 1, p, count, mul, shift, wide);
        if (e != 0) return e;
        p.x += run * p.ld_x * E;
        if (p.gate != nullptr) p.gate += run * p.ld_gate * E;
        p.codes += run * p.ld_codes;
        p.scales += run * p.ld_scales;
    }
    return 0;
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

int fp8_errors(bool clear, uint32_t* flags) {
    unsigned v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, gq_fp8_errors, sizeof(v));
    if (e == cudaSuccess && clear && v != 0) {
        const unsigned zero = 0;
        e = cudaMemcpyToSymbol(gq_fp8_errors, &zero, sizeof(zero));
    }
    *flags = v;
    return static_cast<int>(e);
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
