// out = a b^T (+ bias) for block-scaled e4m3 operands, on the tensor cores.
//
// The matrix instruction (tcgen05.mma, kind mxf8f6f4) takes one E8M0 scale per row and 32
// columns and multiplies by it itself, so a 1 x 128 or 128 x 128 block's scale is the same
// byte for four instructions and the sum over all of k stays in tensor memory.
//
// gq_matmul_narrow: the weights' 128 rows are the instruction's M and the tokens its N, so
// that a few tokens cost a narrow instruction and not a padded one.  What bounds it is the
// weights' traffic: a CTA streams its 128 rows through a ring of 128-column tiles.  Where
// there are too few row tiles for the SMs, a cluster of 2 to 8 CTAs splits k and adds the
// partial sums over distributed shared memory in a fixed order.  Measured: 1 x 28672 x 4096 in
// 20.1 us (5.8 TB/s, 89% of the copy rate), 1 x 4096 x 4096 in 5.8 us, of which the weights'
// bytes are 2.6 and the rest set-up, one round of loads and the join.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "gq_choose.h"
#include "gq_fp8.cuh"
#include "gq_internal.h"
#include "gq_launch.h"
#include "gq_tcgen05.cuh"

namespace gq {
namespace {

// Sticky error flags of this device's product kernels (kErrWaitTimeout).
__device__ unsigned int gq_matmul_errors;

template <class T>
__device__ __forceinline__ T out_cast(float x);
template <>
__device__ __forceinline__ float out_cast<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half out_cast<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 out_cast<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Four values to one row of the output, as one store where the address allows it
template <class T>
__device__ __forceinline__ void store4(T* out, const float (&v)[4], int64_t left) {
    if (left >= 4 && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0) {
        if constexpr (sizeof(T) == 4) {
            stg128f(reinterpret_cast<float*>(out), v[0], v[1], v[2], v[3]);
        } else {
            T c[4] = {out_cast<T>(v[0]), out_cast<T>(v[1]), out_cast<T>(v[2]), out_cast<T>(v[3])};
            uint2 w;
            memcpy(&w, c, sizeof(w));
            st_global(reinterpret_cast<uint2*>(out), w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) out[i] = out_cast<T>(v[i]);
    }
}

// Four consecutive scale bytes from block kb on as a word; blocks from `blocks` on read as 1
__device__ __forceinline__ uint32_t scale_word(const uint8_t* row, int64_t kb, int64_t blocks) {
    const uint8_t* s = row + kb;
    if (kb + 4 <= blocks && (reinterpret_cast<uintptr_t>(s) & 3) == 0) return *reinterpret_cast<const uint32_t*>(s);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (kb + i < blocks ? static_cast<uint32_t>(s[i]) : 127u) << (8 * i);
    return w;
}

constexpr int kTileK = 128;
constexpr int kSfSlots = 4;      // groups of four 128-column blocks whose scales are staged

template <int BN, class T>
struct Narrow {
    static constexpr int kThreads = 192;
    static constexpr int kStageBytes = 128 * kTileK + BN * kTileK;
    static constexpr int kStages = BN <= 32 ? 5 : BN == 64 ? 4 : 3;
    static constexpr int kSfBytes = 1024;                          // 512 for each operand
    static constexpr int kBars = 2 * kStages + 2 * kSfSlots + 1;
    static constexpr int kRing = kStages * kStageBytes;            // reused for the f32 sums
    static constexpr int kUsed = 1024 + kRing + kSfSlots * kSfBytes + 8 * kBars + 16;
    static constexpr int kPieces = narrow_pieces(BN, sizeof(T) == 4);      // accumulators
    static constexpr int kNeed = kPieces * BN + 8 * kSfSlots;
    static constexpr int kCols = kNeed <= 64 ? 64 : kNeed <= 128 ? 128 : 256;
    // CTAs that share an SM find room in its 512 columns of tensor memory together, so that none
    // waits for another's: shared memory is taken in the same proportion, 228 KB for 512 columns.
    static constexpr int kLeast = kCols * 228 * 2 - 1024;
    static constexpr int kSmem = kUsed > kLeast ? kUsed : kLeast;
    static_assert(kRing >= BN * 128 * 4, "the sums fit the ring");
    static_assert(kSmem <= 227 * 1024, "one CTA's shared memory");
};

template <int BN, class T>
__global__ void __launch_bounds__(Narrow<BN, T>::kThreads) gq_matmul_narrow(const __grid_constant__ CUtensorMap map_b,
                                                                         const __grid_constant__ CUtensorMap map_a,
                                                                         const GqMatmul p, const int split) {
    using C = Narrow<BN, T>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32addr(smem_raw) + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - smem_u32addr(smem_raw));
    const uint32_t sf = base + C::kRing, bars = sf + kSfSlots * C::kSfBytes, slot = bars + 8 * C::kBars;
    const auto full = [&](int s) { return bars + 8 * s; };
    const auto empty = [&](int s) { return bars + 8 * (C::kStages + s); };
    const auto sf_full = [&](int s) { return bars + 8 * (2 * C::kStages + s); };
    const auto sf_empty = [&](int s) { return bars + 8 * (2 * C::kStages + kSfSlots + s); };
    const uint32_t done = bars + 8 * (C::kBars - 1);
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   // uniform for the compiler

    const uint32_t rank = split > 1 ? tc::cluster_rank() : 0;
    const int64_t tile = blockIdx.x / split;
    const int64_t m_tiles = (p.m + BN - 1) / BN;
    const int64_t m0 = tile % m_tiles * BN, n0 = tile / m_tiles * 128;
    const int kb0 = static_cast<int>(p.kb * rank / split), kb1 = static_cast<int>(p.kb * (rank + 1) / split);
    const int blocks = kb1 - kb0;
    // pieces of whole groups of four blocks
    const int most = min(C::kPieces, (blocks + kPiece - 1) / kPiece), piece = ((blocks + most - 1) / most + 3) & ~3;
    const int pieces = (blocks + piece - 1) / piece;

    if (warp == 5) tc::tmem_alloc<C::kCols>(slot);
    if (warp == 4 && tc::elect()) {
        tc::prefetch_map(&map_b);
        tc::prefetch_map(&map_a);
    }
    if (tid == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            tc::init(full(s), 1);
            tc::init(empty(s), 1);
        }
        for (int s = 0; s < kSfSlots; ++s) {
            tc::init(sf_full(s), 1);
            tc::init(sf_empty(s), 1);
        }
        tc::init(done, 1);
        mbar_init_fence();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = lds_u32(slot);
    let_next();
    after_previous();

    bool ok = true;
    if (warp == 4) {
        int issued = 0;
        for (int i = 0; i < blocks; ++i) {
            const int s = i % C::kStages, round = i / C::kStages;
            if (round > 0 && !(ok = tc::wait(empty(s), (round - 1) & 1))) break;
            if (tc::elect()) {
                tc::arrive_expect(full(s), C::kStageBytes);
                const uint32_t at = base + s * C::kStageBytes;
                tc::load_tile(at, &map_b, (kb0 + i) * kTileK, static_cast<int>(n0), full(s));
                tc::load_tile(at + 128 * kTileK, &map_a, (kb0 + i) * kTileK, static_cast<int>(m0), full(s));
            }
            issued = i + 1;
        }
        // nothing of this CTA is in flight when it ends, also after a wait that gave up
        if (!ok)
            for (int i = max(0, issued - C::kStages); i < issued; ++i) tc::wait(full(i % C::kStages), (i / C::kStages) & 1);
    } else if (warp == 5) {
        // what changes from block to block changes by additions: the loop's own instructions, not
        // the matrix ones, set the pace of a narrow tile
        const uint64_t da0 = tc::operand_desc(base), db0 = tc::operand_desc(base + 128 * kTileK);
        uint64_t da = da0, db = db0;
        uint32_t parity = 0;
        int s = 0;
        for (int g = 0; 4 * g < blocks && ok; ++g) {
            const int q = g % kSfSlots;
            const uint32_t d = tmem + BN * (4 * g / piece), ta = tmem + C::kPieces * BN + 8 * q, tb = ta + 4;
            const bool first = 4 * g % piece == 0;
            if (!(ok = tc::wait(sf_full(q), (g / kSfSlots) & 1))) break;
            tc::fence_after();
            if (tc::elect()) {
                tc::copy_scales(ta, tc::scale_desc(sf + q * C::kSfBytes));
                tc::copy_scales(tb, tc::scale_desc(sf + q * C::kSfBytes + 512));
            }
            __syncwarp();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (4 * g + u >= blocks || !ok) continue;
                if (!(ok = tc::wait(full(s), parity))) continue;
                tc::fence_after();
                if (tc::elect()) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc::mma(d, da + 2 * k, db + 2 * k, tc::instruction<128, BN>(u), ta, tb, !first || u > 0 || k > 0);
                    tc::commit(empty(s));
                }
                __syncwarp();
                da += C::kStageBytes >> 4;
                db += C::kStageBytes >> 4;
                if (++s == C::kStages) {
                    s = 0;
                    parity ^= 1;
                    da = da0;
                    db = db0;
                }
            }
            if (ok && tc::elect()) tc::commit(sf_empty(q));
            __syncwarp();
        }
        if (tc::elect()) tc::commit(done);
    } else if (warp == 2) {
        // scales: the weights' byte is the same for all 128 rows of the tile
        const uint8_t* wrow = p.b_scales + (n0 >> 7) * p.ld_b_scales;
        for (int i = 0; i < blocks; i += 4) {
            const int g = i / 4, q = g % kSfSlots, round = g / kSfSlots;
            const uint32_t w = scale_word(wrow, kb0 + i, p.kb);
            uint32_t x[(BN + 31) / 32];
#pragma unroll
            for (int j = 0; j < (BN + 31) / 32; ++j) {
                const int64_t m = m0 + 32 * j + lane;
                x[j] = m < p.m ? scale_word(p.a_scales + m * p.ld_a_scales, kb0 + i, p.kb) : 0x7F7F7F7Fu;
            }
            if (round > 0 && !(ok = tc::wait(sf_empty(q), (round - 1) & 1))) break;
            sts(sf + q * C::kSfBytes + 16 * lane, make_uint4(w, w, w, w));
#pragma unroll
            for (int j = 0; j < (BN + 31) / 32; ++j) sts(sf + q * C::kSfBytes + 512 + 16 * lane + 4 * j, x[j]);
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::arrive(sf_full(q));
        }
    }
    if (warp < 4) {
        if (!tc::wait(done, 0)) ok = false;
        __syncwarp();
        tc::fence_after();
        // lane = weight row: the sums go to shared memory as (token, 128 rows)
        float* sums = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int c = 0; c < BN; c += 16) {
            uint32_t v[16];
            tc::tmem_load16(tmem + (static_cast<uint32_t>(32 * warp) << 16) + c, v);
            tc::tmem_wait();
            for (int k = 1; k < pieces; ++k) {
                uint32_t more[16];
                tc::tmem_load16(tmem + (static_cast<uint32_t>(32 * warp) << 16) + BN * k + c, more);
                tc::tmem_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __float_as_uint(__fadd_rn(__uint_as_float(v[j]), __uint_as_float(more[j])));
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) sums[(c + j) * 128 + 32 * warp + lane] = __uint_as_float(v[j]);
        }
        tc::fence_before();
        asm volatile("bar.arrive 1, 160;" ::: "memory");
    }
    if (!ok) atomicOr(&gq_matmul_errors, kErrWaitTimeout);
    __syncwarp();
    if (split > 1) tc::cluster_arrive();
    else __syncthreads();
    if (warp == 5) {
        // The tensor memory goes back before this CTA waits for another one of its cluster, which
        // may not have its own yet: a kernel of another stream that takes tensor memory by other
        // proportions may hold it there, and wait here for this CTA's.
        asm volatile("bar.sync 1, 160;" ::: "memory");
        tc::fence_after();
        tc::tmem_free<C::kCols>(tmem);
    }
    if (split > 1) tc::cluster_wait();

    T* const out = reinterpret_cast<T*>(p.out);
    const bool fours = ((reinterpret_cast<uintptr_t>(p.out) | static_cast<uintptr_t>(p.ld_out * sizeof(T))) & (4 * sizeof(T) - 1)) == 0;
    const int rows = static_cast<int>(min(static_cast<int64_t>(BN), p.m - m0));
    for (int u = static_cast<int>(rank) * C::kThreads + tid; u < 32 * rows; u += C::kThreads * split) {
        const int r = u >> 5, c = 4 * (u & 31);
        if (!fours) {
            // rows off the boundaries of four values: neighbouring lanes on neighbouring values
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = (u & 31) + 32 * i;
                if (n0 + n >= p.n) continue;
                const uint32_t at = base + (r * 128 + n) * 4;
                float x[8] = {*reinterpret_cast<const float*>(smem + (r * 128 + n) * 4), 0, 0, 0, 0, 0, 0, 0};
                if (split > 1)
#pragma unroll
                    for (int s = 0; s < 8; ++s)
                        if (s < split) x[s] = tc::load_cluster1(tc::map_shared(at, s));
                float v = x[0];
#pragma unroll
                for (int s = 1; s < 8; ++s)
                    if (s < split) v = __fadd_rn(v, x[s]);
                if (p.bias != nullptr) v = __fadd_rn(v, p.bias[n0 + n]);
                out[(m0 + r) * p.ld_out + n0 + n] = out_cast<T>(v);
            }
            continue;
        }
        if (n0 + c >= p.n) continue;
        const uint32_t at = base + (r * 128 + c) * 4;
        float4 x[8];
        x[0] = *reinterpret_cast<const float4*>(smem + (r * 128 + c) * 4);
        // all CTAs' parts on their way before the first addition
        if (split > 1)
#pragma unroll
            for (int s = 0; s < 8; ++s)
                if (s < split) x[s] = tc::load_cluster(tc::map_shared(at, s));
        float v[4] = {x[0].x, x[0].y, x[0].z, x[0].w};
#pragma unroll
        for (int s = 1; s < 8; ++s)
            if (s < split) {
                v[0] = __fadd_rn(v[0], x[s].x);
                v[1] = __fadd_rn(v[1], x[s].y);
                v[2] = __fadd_rn(v[2], x[s].z);
                v[3] = __fadd_rn(v[3], x[s].w);
            }
        if (p.bias != nullptr)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n0 + c + i < p.n) v[i] = __fadd_rn(v[i], p.bias[n0 + c + i]);
        store4(out + (m0 + r) * p.ld_out + n0 + c, v, p.n - n0 - c);
    }
    // the partial sums stay until every CTA of the cluster has read them
    if (split > 1) tc::cluster_sync();
}

// ---- wide products ----------------------------------------------------------------------------
//
// gq_matmul_wide: a persistent grid of CTA pairs (cta_group::2), each pair on a tile of 256
// tokens (128 per CTA) x BN output channels; every CTA loads its own tokens' rows and half of
// the weights' rows, so a pair reads as much from L2 as one CTA with a tile half as wide.
// The first 8 warps (16 for f32 outputs) drain the accumulators into registers, release them and
// then store; of the last three, one loads tiles, one (of the first CTA) issues the matrix
// instructions and one stages the scales.  Measured: 8192 x 28672 x 4096 in 650 us (2.9 PFLOP/s)
// in runs of a few ms; held for a second the board's 1000 W bring it to 760-780 us.

// A tile's scales as they lie in memory: 128 rows of the tokens' and two of the weights', for all
// of k.  They come by bulk copies, the next tile's as soon as this one's are read: the tile loads
// keep the SM's whole read path from L2 busy (64 bytes a cycle), and a plain load queues behind
// all of them (measured: 1000 to 3000 cycles for each group of scales).
constexpr int kRawA = 16384, kRawB = 512;

// A region of scale rows first..first + rows - 1 (those within `all`): from the 16-byte boundary
// before it to the one after it, or to the end of the tensor, whose last bytes are `tail`.
struct RawRegion {
    int64_t start;      // bytes from the tensor's first
    int skew, whole, tail;
};
__device__ __forceinline__ RawRegion raw_region(int64_t first, int rows, int64_t all, int64_t ld, int64_t blocks) {
    RawRegion r{0, 0, 0, 0};
    if (first >= all) return r;
    const int64_t begin = first * ld, end = (min(first + rows, all) - 1) * ld + blocks, last = (all - 1) * ld + blocks;
    r.start = begin & ~int64_t(15);
    r.skew = static_cast<int>(begin - r.start);
    const int64_t stop = (end + 15) & ~int64_t(15);
    r.whole = static_cast<int>((stop <= last ? stop : end & ~int64_t(15)) - r.start);
    r.tail = static_cast<int>(stop <= last ? 0 : end & 15);
    return r;
}
// Four scale bytes at shared address a
__device__ __forceinline__ uint32_t raw_word(uint32_t a, bool words) {
    if (words) return lds_u32(a);
    return __funnelshift_r(lds_u32(a & ~3u), lds_u32((a & ~3u) + 4), 8 * (a & 3u));
}

// They are staged for the copy to tensor memory in batches of kBatch groups (16 blocks of 128
// columns), two batches in turn: the fence and the remote arrival that a batch ends with take
// longer than the instructions of one group of a narrow tile.
constexpr int kBatch = 4;

// Outputs go out through shared memory, a few KB per warp, in the place of a stage of the ring
// (measured: the ring loses nothing by it): as boxes of a tensor map where the rows start and
// end on 16 bytes, or (PLAIN) by the warp's own stores, a row's values side by side from neighbouring
// lanes.  A lane that stores its own row directly touches 32 lines at a time (8192 x 28672 x 4096
// 689 us against 649 without stores; 440 us for 6482 x 12260 x 320, whose rows start off 16 bytes).
template <int BN, class T, bool PLAIN>
struct Wide {
    // warps that take the accumulators out: f32 outputs need room for a piece beside the sum
    static constexpr int kOut = sizeof(T) == 4 ? 16 : 8;
    static constexpr int kPieceBlocks = sizeof(T) == 4 ? kPiece : INT32_MAX;
    static constexpr int kThreads = 32 * (kOut + 3);
    static constexpr int kHalf = BN / 2;                       // weight rows per CTA
    static constexpr int kStageBytes = 128 * kTileK + kHalf * kTileK;
    static constexpr int kStages = BN == 256 ? 5 : PLAIN && sizeof(T) == 4 ? 6 : 7;
    static constexpr int kBox = sizeof(T) == 4 ? 64 : 128;     // bytes of a row that a warp stages at a time
    static constexpr int kOutBytes = PLAIN ? kOut * 32 * 17 * 4 : kOut * 32 * kBox;
    static constexpr int kSfBytes = 512 + 512 * (BN / 128);
    static constexpr int kSfCols = 4 + 4 * (BN / 128);
    static constexpr int kAcc = BN == 256 ? 1 : 2;             // accumulators in tensor memory
    static constexpr int kSlots = 2 * kBatch;
    static constexpr int kBars = 2 * kStages + 2 * 2 + 2 * kAcc + 1;
    static constexpr int kCols = 512;
    static constexpr int kSmem = 227 * 1024;                   // all of an SM's, as all of its tensor memory
    static_assert(1024 + kStages * kStageBytes + kSlots * kSfBytes + kRawA + kRawB + kOutBytes + 128 + 8 * kBars + 16 <= kSmem, "shared memory");
    static_assert(kAcc * BN + kSlots * kSfCols <= kCols, "tensor memory");
};

template <class T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    T c[2] = {out_cast<T>(x), out_cast<T>(y)};
    uint32_t w;
    memcpy(&w, c, sizeof(w));
    return w;
}

// Tile t of the order in which pairs take them: bands of `tall` row tiles, within a band column by
// column, so that the tiles in flight share rows of both operands in L2 and the band's tokens
// stay there while the weights pass.
struct Order {
    int tiles_m, tiles_n, tall;
};
__device__ __forceinline__ void tile_place(int t, const Order& o, int& tm, int& tn) {
    const int band = t / (o.tall * o.tiles_n), in = t - band * (o.tall * o.tiles_n);
    const int tall = min(o.tall, o.tiles_m - band * o.tall);
    tn = in / tall;
    tm = band * o.tall + in - tn * tall;
}

template <int BN, class T, bool PLAIN>
__global__ void __launch_bounds__(Wide<BN, T, PLAIN>::kThreads, 1)
    gq_matmul_wide(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_out, const GqMatmul p, const Order order, const bool use_raw) {
    using C = Wide<BN, T, PLAIN>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t out_stage = base + C::kStages * C::kStageBytes, sf = out_stage + (C::kOutBytes + 127) / 128 * 128;
    const uint32_t raw_a = sf + C::kSlots * C::kSfBytes, raw_b = raw_a + kRawA, bars = raw_b + kRawB, slot = bars + 8 * C::kBars;
    const auto full = [&](int s) { return bars + 8 * s; };
    const auto empty = [&](int s) { return bars + 8 * (C::kStages + s); };
    const auto sf_full = [&](int s) { return bars + 8 * (2 * C::kStages + s); };
    const auto sf_empty = [&](int s) { return bars + 8 * (2 * C::kStages + 2 + s); };
    const uint32_t raw_full = bars + 8 * (C::kBars - 1);
    const auto acc_full = [&](int s) { return bars + 8 * (2 * C::kStages + 4 + s); };
    const auto acc_empty = [&](int s) { return bars + 8 * (2 * C::kStages + 4 + C::kAcc + s); };
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);   // uniform for the compiler
    const uint32_t rank = tc::cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1, tiles = order.tiles_m * order.tiles_n;
    const int blocks = static_cast<int>(p.kb), groups = (blocks + 3) / 4;
    if (warp == C::kOut + 1) tc::tmem_alloc_pair<C::kCols>(slot);
    if (warp == C::kOut && tc::elect()) {
        tc::prefetch_map(&map_a);
        tc::prefetch_map(&map_b);
    }
    if (tid == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            tc::init(full(s), 1);        // the first CTA's: both CTAs' loads
            tc::init(empty(s), 1);
        }
        for (int s = 0; s < 2; ++s) {
            tc::init(sf_full(s), 2);
            tc::init(sf_empty(s), 1);
        }
        for (int s = 0; s < C::kAcc; ++s) {
            tc::init(acc_full(s), 1);
            tc::init(acc_empty(s), 2 * C::kOut);  // the first CTA's: both CTAs' warps
        }
        tc::init(raw_full, 1);
        mbar_init_fence();
    }
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();
    tc::fence_after();
    const uint32_t tmem = lds_u32(slot);
    let_next();
    after_previous();

    bool ok = true;
    if (warp == C::kOut) {
        int it = 0;
        asm volatile("bar.sync 1, 64;" ::: "memory");      // the scales' first request is out
        for (int t = pair; t < tiles && ok; t += pairs) {
            int tm, tn;
            tile_place(t, order, tm, tn);
            const int m0 = tm * 256 + 128 * static_cast<int>(rank), n0 = tn * BN + C::kHalf * static_cast<int>(rank);
            for (int i = 0; i < blocks; ++i, ++it) {
                const int s = it % C::kStages, round = it / C::kStages;
                if (round > 0 && !(ok = tc::wait(empty(s), (round - 1) & 1))) break;
                if (tc::elect()) {
                    const uint32_t bar = tc::map_shared(full(s), 0), at = base + s * C::kStageBytes;
                    // the first CTA expects both CTAs' bytes; the second's may land before: its
                    // loads wait for the instructions that used the stage, so for this phase
                    if (rank == 0) tc::arrive_expect(full(s), 2 * C::kStageBytes);
                    tc::load_tile_pair(at, &map_a, i * kTileK, m0, bar);
                    tc::load_tile_pair(at + 128 * kTileK, &map_b, i * kTileK, n0, bar);
                }
            }
        }
        // the instructions' arrivals on this CTA's barriers, before it may end
        for (int i = max(0, it - C::kStages); ok && i < it; ++i) ok = tc::wait(empty(i % C::kStages), (i / C::kStages) & 1);
        // after a wait that gave up, loads may be in flight whose barrier is the other CTA's:
        // they land long before these 10 ms are over
        if (!ok)
            for (const uint64_t t0 = global_ns(); global_ns() - t0 < 10000000ull;) {
            }
    } else if (warp == C::kOut + 1) {
        // what changes from block to block changes by additions: with divisions in it this loop
        // took longer than a 256 x 128 tile's instructions (512 x 4096 x 14336 35 us)
        constexpr int kPieceGroups = C::kPieceBlocks / 4;
        const uint64_t da0 = tc::operand_desc(base), db0 = tc::operand_desc(base + 128 * kTileK);
        uint64_t da = da0, db = db0;
        uint32_t parity = 0;
        int s = 0, bi = 0, n = 0;     // stage; batches and pieces so far
        for (int t = pair; rank == 0 && t < tiles && ok; t += pairs) {
            for (int g = 0; g < groups && ok; ++g) {
                const int b = n % C::kAcc, use = n / C::kAcc;
                const bool first = g % kPieceGroups == 0;
                if (first) {
                    if (use > 0 && !(ok = tc::wait(acc_empty(b), (use - 1) & 1))) break;
                    tc::fence_after();
                }
                if (g % kBatch == 0) {
                    if (!(ok = tc::wait(sf_full(bi & 1), (bi >> 1) & 1))) break;
                    tc::fence_after();
                }
                const int q = (bi & 1) * kBatch + g % kBatch;
                const uint32_t d = tmem + BN * b, ta = tmem + C::kAcc * BN + C::kSfCols * q, tb = ta + 4;
                if (tc::elect()) {
                    const uint32_t from = sf + q * C::kSfBytes;
                    tc::copy_scales_pair(ta, tc::scale_desc(from));
#pragma unroll
                    for (int j = 0; j < BN / 128; ++j) tc::copy_scales_pair(tb + 4 * j, tc::scale_desc(from + 512 + 512 * j));
                }
                __syncwarp();
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (4 * g + u >= blocks || !ok) continue;
                    if (!(ok = tc::wait(full(s), parity))) continue;
                    tc::fence_after();
                    if (tc::elect()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc::mma_pair(d, da + 2 * k, db + 2 * k, tc::instruction<256, BN>(u), ta, tb, !first || u > 0 || k > 0);
                        tc::commit_pair(empty(s));
                    }
                    __syncwarp();
                    da += C::kStageBytes >> 4;
                    db += C::kStageBytes >> 4;
                    if (++s == C::kStages) {
                        s = 0;
                        parity ^= 1;
                        da = da0;
                        db = db0;
                    }
                }
                if (!ok) break;
                const bool batch = g % kBatch == kBatch - 1 || g + 1 == groups;
                const bool piece = g % kPieceGroups == kPieceGroups - 1 || g + 1 == groups;
                if (tc::elect()) {
                    if (batch) tc::commit_pair(sf_empty(bi & 1));
                    if (piece) tc::commit_pair(acc_full(b));
                }
                __syncwarp();
                bi += batch;
                n += piece;
            }
            // after a wait that gave up: those who wait for this piece end sooner
            if (!ok && tc::elect()) tc::commit_pair(acc_full(n % C::kAcc));
            __syncwarp();
        }
    } else if (warp == C::kOut + 2) {
        constexpr int kB = BN / 128;
        int bi = 0;
        const int64_t nbs = (p.n + 127) >> 7;
        RawRegion ra{0, 0, 0, 0}, rb{0, 0, 0, 0};
        const bool words = ((p.ld_a_scales | p.ld_b_scales) & 3) == 0;
        int asked = 0, read = 0;      // requests made, and waited for
        const auto request = [&](int t) {
            ++asked;
            int tm, tn;
            tile_place(t, order, tm, tn);
            ra = raw_region(static_cast<int64_t>(tm) * 256 + 128 * rank, 128, p.m, p.ld_a_scales, p.kb);
            rb = raw_region(static_cast<int64_t>(tn) * kB, kB, nbs, p.ld_b_scales, p.kb);
            if (tc::elect()) {
                tc::arrive_expect(raw_full, static_cast<uint32_t>(ra.whole + rb.whole));
                if (ra.whole > 0) tc::bulk(raw_a, p.a_scales + ra.start, ra.whole, raw_full);
                if (rb.whole > 0) tc::bulk(raw_b, p.b_scales + rb.start, rb.whole, raw_full);
            }
            __syncwarp();
        };
        const auto direct = [&](int64_t m0, int64_t nb0, int g0, uint32_t (&x)[kBatch][4], uint32_t (&w)[kBatch][kB]) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int kb = 4 * (g0 + u);
                if (g0 + u >= groups) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int64_t m = m0 + 32 * j + lane;
                    x[u][j] = m < p.m ? scale_word(p.a_scales + m * p.ld_a_scales, kb, blocks) : 0x7F7F7F7Fu;
                }
#pragma unroll
                for (int j = 0; j < kB; ++j)
                    w[u][j] = nb0 + j < nbs ? scale_word(p.b_scales + (nb0 + j) * p.ld_b_scales, kb, blocks) : 0x7F7F7F7Fu;
            }
        };
        const auto stage = [&](int g0, const uint32_t (&x)[kBatch][4], const uint32_t (&w)[kBatch][kB]) {
            if (bi > 1 && !(ok = tc::wait(sf_empty(bi & 1), ((bi >> 1) - 1) & 1))) return;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                if (g0 + u >= groups) continue;
                const uint32_t to = sf + ((bi & 1) * kBatch + u) * C::kSfBytes + 16 * lane;
                sts(to, make_uint4(x[u][0], x[u][1], x[u][2], x[u][3]));
#pragma unroll
                for (int j = 0; j < kB; ++j) sts(to + 512 + 512 * j, make_uint4(w[u][j], w[u][j], w[u][j], w[u][j]));
            }
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::arrive_remote(tc::map_shared(sf_full(bi & 1), 0));
            ++bi;
        };
        uint32_t x[kBatch][4], w[kBatch][kB];
        // ahead of the first tile loads, which wait for this warp here (512 x 4096 x 4096 14.1 against
        // 14.6 us with the first batch by plain loads at the same time)
        if (use_raw && groups > kBatch) request(pair);
        asm volatile("bar.arrive 1, 64;" ::: "memory");
        if (groups <= kBatch) {
            // short sums: one batch per tile, the next tile's on its way in registers
            int tm, tn;
            tile_place(pair, order, tm, tn);
            direct(static_cast<int64_t>(tm) * 256 + 128 * rank, static_cast<int64_t>(tn) * kB, 0, x, w);
            for (int t = pair; t < tiles && ok; t += pairs) {
                stage(0, x, w);
                if (t + pairs < tiles) {
                    tile_place(t + pairs, order, tm, tn);
                    direct(static_cast<int64_t>(tm) * 256 + 128 * rank, static_cast<int64_t>(tn) * kB, 0, x, w);
                }
            }
        }
        for (int t = pair; groups > kBatch && t < tiles && ok; t += pairs) {
            int tm, tn;
            tile_place(t, order, tm, tn);
            const int64_t m0 = static_cast<int64_t>(tm) * 256 + 128 * rank, nb0 = static_cast<int64_t>(tn) * kB;
            uint32_t from_a[4] = {0, 0, 0, 0}, from_b[kB] = {};
            bool raw = false;
            for (int g0 = 0; g0 < groups; g0 += kBatch) {
                if (use_raw && !raw) {
                    if (!(ok = tc::wait(raw_full, read & 1))) break;
                    ++read;
                    raw = true;
                    if (lane < ra.tail) sts(raw_a + ra.whole + lane, p.a_scales[ra.start + ra.whole + lane]);
                    if (lane < rb.tail) sts(raw_b + rb.whole + lane, p.b_scales[rb.start + rb.whole + lane]);
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 4; ++j) from_a[j] = raw_a + ra.skew + static_cast<uint32_t>((32 * j + lane) * p.ld_a_scales);
#pragma unroll
                    for (int j = 0; j < kB; ++j) from_b[j] = raw_b + rb.skew + static_cast<uint32_t>(j * p.ld_b_scales);
                }
                if (raw) {
#pragma unroll
                    for (int u = 0; u < kBatch; ++u) {
                        if (g0 + u >= groups) continue;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            x[u][j] = m0 + 32 * j + lane < p.m ? raw_word(from_a[j] + 4 * (g0 + u), words) : 0x7F7F7F7Fu;
#pragma unroll
                        for (int j = 0; j < kB; ++j) w[u][j] = nb0 + j < nbs ? raw_word(from_b[j] + 4 * (g0 + u), words) : 0x7F7F7F7Fu;
                    }
                } else {
                    direct(m0, nb0, g0, x, w);
                }
                // this tile's are read: the next one's may overwrite them
                if (use_raw && g0 + kBatch >= groups && t + pairs < tiles) {
                    tc::fence_async_shared();
                    __syncwarp();
                    request(t + pairs);
                }
                stage(g0, x, w);
                if (!ok) break;
            }
        }
        // a request that nothing waited for, after a wait that gave up
        if (!ok && asked > read) tc::wait(raw_full, read & 1);
        for (int i = max(0, bi - 2); ok && i < bi; ++i) ok = tc::wait(sf_empty(i & 1), (i >> 1) & 1);
    } else {
        constexpr int kPart = BN / (C::kOut / 4);           // columns per warp
        int n = 0;
        for (int t = pair; t < tiles && ok; t += pairs) {
            int tm, tn;
            tile_place(t, order, tm, tn);
            const int64_t m = static_cast<int64_t>(tm) * 256 + 128 * rank + 32 * (warp & 3) + lane;
            const int64_t n0 = static_cast<int64_t>(tn) * BN + kPart * (warp >> 2);
            // the columns' bias, a value per lane and 32 columns, on its way while the sums are made
            float bias[kPart / 32] = {};
            if (p.bias != nullptr)
#pragma unroll
                for (int i = 0; i < kPart / 32; ++i)
                    if (n0 + 32 * i + lane < p.n) bias[i] = p.bias[n0 + 32 * i + lane];
            uint32_t v[kPart];
            for (int i = 0; i < blocks; i += min(C::kPieceBlocks, blocks), ++n) {
                const int b = n % C::kAcc, use = n / C::kAcc;
                if (!(ok = tc::wait(acc_full(b), use & 1))) break;
                __syncwarp();
                tc::fence_after();
                const uint32_t from = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + BN * b + kPart * (warp >> 2);
                if (sizeof(T) < 4 || i == 0) {
#pragma unroll
                    for (int c = 0; c < kPart; c += 32) tc::tmem_load32(from + c, v + c);
                    tc::tmem_wait();
                } else {
#pragma unroll
                    for (int c = 0; c < kPart; c += 16) {
                        uint32_t more[16];
                        tc::tmem_load16(from + c, more);
                        tc::tmem_wait();
#pragma unroll
                        for (int k = 0; k < 16; ++k) v[c + k] = __float_as_uint(__fadd_rn(__uint_as_float(v[c + k]), __uint_as_float(more[k])));
                    }
                }
                // the accumulators are free for the next piece once they are in registers
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::arrive_remote_relaxed(tc::map_shared(acc_empty(b), 0));
            }
            if (!ok) break;
            if (p.bias != nullptr) {
#pragma unroll
                for (int i = 0; i < kPart; ++i)
                    v[i] = __float_as_uint(__fadd_rn(__uint_as_float(v[i]), __shfl_sync(0xffffffffu, bias[i / 32], i % 32)));
            }
            if constexpr (PLAIN) {
                // 64 bytes of each of the warp's rows at a time, two rows to a store
                const uint32_t stage = out_stage + warp * (32 * 17 * 4);
                const int64_t top = m - lane;
#pragma unroll
                for (int c = 0; c < kPart; c += 64 / static_cast<int>(sizeof(T))) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        if constexpr (sizeof(T) == 4) sts(stage + 4 * (17 * lane + i), v[c + i]);
                        else sts(stage + 4 * (17 * lane + i), pack2<T>(__uint_as_float(v[c + 2 * i]), __uint_as_float(v[c + 2 * i + 1])));
                    }
                    __syncwarp();
                    const int word = lane & 15;
                    const int64_t col = n0 + c + word * static_cast<int>(4 / sizeof(T));
                    T* out = reinterpret_cast<T*>(p.out) + (top + (lane >> 4)) * p.ld_out + col;
#pragma unroll 4
                    for (int r = lane >> 4; r < 32; r += 2, out += 2 * p.ld_out) {
                        const uint32_t x = lds_u32(stage + 4 * (17 * r + word));
                        if (top + r >= p.m || col >= p.n) continue;
                        if (sizeof(T) == 4 || (col + 1 < p.n && (reinterpret_cast<uintptr_t>(out) & 3) == 0)) {
                            st_global(reinterpret_cast<uint32_t*>(out), x);
                        } else {
                            st_global(reinterpret_cast<uint16_t*>(out), static_cast<uint16_t>(x));
                            if (col + 1 < p.n) st_global(reinterpret_cast<uint16_t*>(out) + 1, static_cast<uint16_t>(x >> 16));
                        }
                    }
                    __syncwarp();
                }
            } else {
                // boxes of 32 rows x kBox bytes in the swizzle of that width: 16-byte piece j of
                // row r at j ^ (r % 8) (128 bytes) or j ^ (r / 2 % 4) (64)
                constexpr int kCols = C::kBox / static_cast<int>(sizeof(T));
                const uint32_t stage = out_stage + warp * (32 * C::kBox), row = stage + lane * C::kBox;
                const int turn = C::kBox == 128 ? lane & 7 : (lane >> 1) & 3;
                const int64_t top = m - lane;
#pragma unroll
                for (int c = 0; c < kPart; c += kCols) {
                    if (tc::elect()) tc::store_read();      // the box before this one
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < C::kBox / 16; ++j) {
                        uint32_t x[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if constexpr (sizeof(T) == 4) x[k] = v[c + 4 * j + k];
                            else x[k] = pack2<T>(__uint_as_float(v[c + 8 * j + 2 * k]), __uint_as_float(v[c + 8 * j + 2 * k + 1]));
                        }
                        sts(row + 16 * (j ^ turn), make_uint4(x[0], x[1], x[2], x[3]));
                    }
                    tc::fence_async_shared();
                    __syncwarp();
                    if (top < p.m && n0 + c < p.n && tc::elect())
                        tc::store_tile(&map_out, static_cast<int>(n0 + c), static_cast<int>(top), stage);
                }
            }
        }
        if (!PLAIN && tc::elect()) tc::store_done();
        __syncwarp();
    }
    if (!ok) atomicOr(&gq_matmul_errors, kErrWaitTimeout);
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();
    if (warp == C::kOut + 1) {
        tc::fence_after();
        tc::tmem_free_pair<C::kCols>(tmem);
    }
}

// ---- host side ------------------------------------------------------------------------------

// (rows, k) bytes with a row stride, in boxes of box_rows x 128 bytes laid out in the
// 128-byte swizzle
int tile_map(CUtensorMap* map, const uint8_t* p, int64_t rows, int64_t k, int64_t ld, int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2] = {kTileK, static_cast<cuuint32_t>(box_rows)};
    return encode_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

template <int BN, class T>
int launch_narrow(const GqMatmul& p, int sms, cudaStream_t s) {
    using C = Narrow<BN, T>;
    auto kern = gq_matmul_narrow<BN, T>;
    CUtensorMap map_b, map_a;
    int st = tile_map(&map_b, p.b, p.n, p.k, p.ld_b, 128);
    if (st == 0) st = tile_map(&map_a, p.a, p.m, p.k, p.ld_a, BN);
    if (st != 0) return st;
    static std::atomic<uint64_t> allowed{0};
    cudaError_t e = allow_smem(kern, C::kSmem, allowed);
    if (e != cudaSuccess) return static_cast<int>(e);
    const int64_t tiles = (p.m + BN - 1) / BN * ((p.n + 127) / 128);
    const int split = narrow_split({p.m, p.n, p.k, p.kb}, BN, sizeof(T) == 4, sms);
    if (tiles * split > INT32_MAX) return static_cast<int>(cudaErrorInvalidValue);
    return launch_early(kern, static_cast<unsigned>(tiles * split), C::kThreads, C::kSmem, s, static_cast<unsigned>(split), map_b,
                        map_a, p, split);
}

template <int BN, class T, bool PLAIN>
int launch_wide(const GqMatmul& p, int sms, cudaStream_t s) {
    using C = Wide<BN, T, PLAIN>;
    auto kern = gq_matmul_wide<BN, T, PLAIN>;
    CUtensorMap map_b, map_a, map_out{};
    int st = tile_map(&map_b, p.b, p.n, p.k, p.ld_b, C::kHalf);
    if (st == 0) st = tile_map(&map_a, p.a, p.m, p.k, p.ld_a, 128);
    if (!PLAIN && st == 0) {
        const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p.n), static_cast<cuuint64_t>(p.m)};
        const cuuint64_t strides[1] = {static_cast<cuuint64_t>(p.ld_out) * sizeof(T)};
        const cuuint32_t box[2] = {C::kBox / sizeof(T), 32};
        st = encode_map(&map_out, sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, p.out, dims, strides,
                        box, C::kBox == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
    }
    if (st != 0) return st;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(kern, C::kSmem, allowed);
    if (e != cudaSuccess) return static_cast<int>(e);
    const int64_t tiles_m = (p.m + 255) / 256, tiles_n = (p.n + BN - 1) / BN;
    if (tiles_m * tiles_n * p.kb > INT32_MAX) return static_cast<int>(cudaErrorInvalidValue);
    const bool use_raw = (reinterpret_cast<uintptr_t>(p.a_scales) & 15) == 0 && (reinterpret_cast<uintptr_t>(p.b_scales) & 15) == 0 &&
                         128 * p.ld_a_scales <= kRawA && BN / 128 * p.ld_b_scales + 32 <= kRawB;
    const int64_t pairs = sms / 2;
    const unsigned grid = static_cast<unsigned>(2 * (tiles_m * tiles_n < pairs ? tiles_m * tiles_n : pairs));
    // a band's tokens take about 37 MB (measured, held for a second: 8192 x 28672 x 4096 819 / 783 /
    // 756 / 756 us with bands of 4 / 8 / 16 / 32 tiles, 17 to 33 MB; 16384 x 8192 x 8192 857 / 852 / 866 /
    // 949 with 12 / 16 / 20 / 32, the last 67 MB; 8192 x 4096 x 14336 395 / 404 / 430 with 12 / 16 / 32)
    Order order{static_cast<int>(tiles_m), static_cast<int>(tiles_n), 0};
    order.tall = static_cast<int>(std::min<int64_t>(std::max<int64_t>((int64_t(37) << 20) / (256 * p.k), 8), 32));
    return launch_early(kern, grid, C::kThreads, C::kSmem, s, 2, map_a, map_b, map_out, p, order, use_raw);
}

// out = bias (or 0): a product over no columns
template <class T>
__global__ void gq_matmul_bias(const GqMatmul p) {
    let_next();
    after_previous();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < p.m * p.n;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t m = i / p.n, n = i - m * p.n;
        reinterpret_cast<T*>(p.out)[m * p.ld_out + n] = out_cast<T>(p.bias != nullptr ? p.bias[n] : 0.0f);
    }
}

template <class T>
int launch_t(const GqMatmul& p, cudaStream_t s) {
    if (p.k == 0) {
        return launch_early(gq_matmul_bias<T>, 1024, 256, 0, s, 1, p);
    }
    int sms = 0;
    const cudaError_t e = sm_count(sms);
    if (e != cudaSuccess) return static_cast<int>(e);
    // Boxes end on 16 bytes, not on an element: where a row of the output does not, its last box would
    // reach into what lies beside it.
    const bool plain = (reinterpret_cast<uintptr_t>(p.out) | static_cast<uintptr_t>(p.ld_out * sizeof(T)) |
                        static_cast<uintptr_t>(p.n * sizeof(T))) % 16 != 0;
    switch (choose({p.m, p.n, p.k, p.kb}, sizeof(T) == 4, sms)) {
        case 16: return launch_narrow<16, T>(p, sms, s);
        case 32: return launch_narrow<32, T>(p, sms, s);
        case 64: return launch_narrow<64, T>(p, sms, s);
        case 128: return launch_narrow<128, T>(p, sms, s);
        case 2 * 128: return plain ? launch_wide<128, T, true>(p, sms, s) : launch_wide<128, T, false>(p, sms, s);
        default: return plain ? launch_wide<256, T, true>(p, sms, s) : launch_wide<256, T, false>(p, sms, s);
    }
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

int matmul_errors(bool clear, uint32_t* flags) {
    unsigned v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, gq_matmul_errors, sizeof(v));
    if (e == cudaSuccess && clear && v != 0) {
        const unsigned zero = 0;
        e = cudaMemcpyToSymbol(gq_matmul_errors, &zero, sizeof(zero));
    }
    *flags = v;
    return static_cast<int>(e);
}

}  // namespace gq
