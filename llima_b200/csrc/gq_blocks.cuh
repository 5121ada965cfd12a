// Block view of GGUF rows: the codes and constants of one block, as gguf-py's dequantize
// uses them, for every block-quantized type.
//
// Block b of a row (16 values for Q6_K, Q2_K and Q3_K, 32 otherwise) as unsigned byte codes
// v (packed in words, value j in byte j % 4 of word j / 4), an offset (the code is
// q = v - OFF) and constants A, B: x = RN(A * q), or RN(RN(A * q) - B) where kSub (Q4_1 and
// Q5_1 store the minimum that is added, so B is its negative).
#pragma once

#include "gq_device.cuh"

namespace gq {

template <int TYPE>
struct BlockView {
    static constexpr int BV = TYPE == GQ_TYPE_Q6_K || TYPE == GQ_TYPE_Q2_K || TYPE == GQ_TYPE_Q3_K ? 16 : 32;
    static constexpr int NW = BV / 4;
    static constexpr int OFF = TYPE == GQ_TYPE_Q6_K   ? 32
                               : TYPE == GQ_TYPE_Q8_0 ? 128
                               : TYPE == GQ_TYPE_Q4_0 ? 8
                               : TYPE == GQ_TYPE_Q5_0 ? 16
                               : TYPE == GQ_TYPE_Q3_K ? 4
                                                      : 0;
    static constexpr bool kSub = TYPE == GQ_TYPE_Q4_K || TYPE == GQ_TYPE_Q5_K || TYPE == GQ_TYPE_Q4_1 ||
                                 TYPE == GQ_TYPE_Q5_1 || TYPE == GQ_TYPE_Q2_K;
    static constexpr int kUnitValues =
        TYPE == GQ_TYPE_Q8_0 || TYPE == GQ_TYPE_Q4_0 || TYPE == GQ_TYPE_Q4_1 || TYPE == GQ_TYPE_Q5_0 || TYPE == GQ_TYPE_Q5_1
            ? 32
            : 256;
    static constexpr int kUnitBytes = TYPE == GQ_TYPE_Q8_0   ? 34
                                      : TYPE == GQ_TYPE_Q4_0 ? 18
                                      : TYPE == GQ_TYPE_Q4_1 ? 20
                                      : TYPE == GQ_TYPE_Q5_0 ? 22
                                      : TYPE == GQ_TYPE_Q5_1 ? 24
                                      : TYPE == GQ_TYPE_Q2_K ? 84
                                      : TYPE == GQ_TYPE_Q3_K ? 110
                                      : TYPE == GQ_TYPE_Q4_K ? 144
                                      : TYPE == GQ_TYPE_Q5_K ? 176
                                                             : 210;
};

// 32 bytes as eight words from `bits` bits after (before, if negative) a shared address that is a
// multiple of 2: a shift that the fields of the words need costs nothing beside the one that the
// alignment needs.  Bits that come in from neighbouring bytes are the caller's to mask.
__device__ __forceinline__ void load32_bits(const uint8_t* p, int bits, uint32_t (&x)[8]) {
    const uint32_t a = 8u * smem_u32addr(p) + static_cast<uint32_t>(bits);     // shared addresses fit in 18 bits
    const uint32_t sh = a & 31u, w = (a >> 5) << 2;
    uint32_t prev = lds_u32(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t next = lds_u32(w + 4 * i + 4);
        x[i] = __funnelshift_r(prev, next, sh);
        prev = next;
    }
}

// 16 bytes of a unit: rows of 16-byte units at 16-byte addresses (UNITS16) in one load
template <bool UNITS16>
__device__ __forceinline__ uint4 unit_bytes16(const uint8_t* p) {
    if constexpr (UNITS16) return lds128(p);
    else return lds128_align2(p);
}

// UNITS16: the row starts at a 16-byte address (which Q4_K's and Q5_K's units then do as well)
template <int TYPE, bool UNITS16 = false>
__device__ __forceinline__ void decode_block(const uint8_t* row, int b, uint32_t (&w)[8], float& A, float& B) {
    B = 0.0f;
    if constexpr (TYPE == GQ_TYPE_Q6_K) {
        // ql[128] | qh[64] | scales int8[16] | d; value 128h + 32g + j (ggml_quant.py:274-308)
        const uint8_t* sp = row + 210 * (b >> 4);
        const int kb = b & 15, h = kb >> 3, g = (kb >> 1) & 3, j0 = 16 * (kb & 1);
        A = __fmul_rn(h2f(lds16(sp + 208)), static_cast<float>(static_cast<int8_t>(sp[192 + kb])));
        const uint4 l = lds128_align2(sp + 64 * h + 32 * (g & 1) + j0);
        const uint4 q = lds128_align2(sp + 128 + 32 * h + j0);
        const uint32_t lw[4] = {l.x, l.y, l.z, l.w}, hw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = ((lw[i] >> (4 * (g >> 1))) & 0x0F0F0F0Fu) | (((hw[i] >> (2 * g)) & 0x03030303u) << 4);
    } else if constexpr (TYPE == GQ_TYPE_Q4_K || TYPE == GQ_TYPE_Q5_K) {
        // d, dmin | scales[12] | (qh[32]) | qs[128]; block k: nibble k & 1 of qs[32(k/2) + j]
        constexpr bool Q5 = TYPE == GQ_TYPE_Q5_K;
        const uint8_t* sp = row + (Q5 ? 176 : 144) * (b >> 3);
        const int k = b & 7, g = k >> 1;
        int sc, mn;
        if (k < 4) {
            sc = sp[4 + k] & 63;
            mn = sp[8 + k] & 63;
        } else {
            sc = (sp[12 + k - 4] & 0xF) | ((sp[4 + k - 4] >> 6) << 4);
            mn = (sp[12 + k - 4] >> 4) | ((sp[8 + k - 4] >> 6) << 4);
        }
        A = __fmul_rn(h2f(lds16(sp)), static_cast<float>(sc));
        B = __fmul_rn(h2f(lds16(sp + 2)), static_cast<float>(mn));
        const uint8_t* qp = sp + (Q5 ? 48 : 16) + 32 * g;
        const uint4 a0 = unit_bytes16<UNITS16>(qp), a1 = unit_bytes16<UNITS16>(qp + 16);
        const uint32_t x[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = (x[i] >> (4 * (k & 1))) & 0x0F0F0F0Fu;
        if constexpr (Q5) {
            const uint4 c0 = unit_bytes16<UNITS16>(sp + 16), c1 = unit_bytes16<UNITS16>(sp + 32);
            const uint32_t hb[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] |= ((hb[i] >> k) & 0x01010101u) << 4;
        }
    } else if constexpr (TYPE == GQ_TYPE_Q8_0) {
        // d | int8[32]: the codes biased by 128 to unsigned bytes
        const uint8_t* bp = row + 34 * b;
        A = h2f(lds16(bp));
        const uint4 a0 = lds128_align2(bp + 2), a1 = lds128_align2(bp + 18);
        const uint32_t x[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = x[i] ^ 0x80808080u;
    } else if constexpr (TYPE == GQ_TYPE_Q4_1 || TYPE == GQ_TYPE_Q5_0 || TYPE == GQ_TYPE_Q5_1) {
        // d | (m) | (qh: bit j of the word is the fifth bit of value j) | nibbles[16]
        constexpr int UB = BlockView<TYPE>::kUnitBytes;
        const uint8_t* bp = row + UB * b;
        A = h2f(lds16(bp));
        if constexpr (TYPE != GQ_TYPE_Q5_0) B = -h2f(lds16(bp + 2));
        const uint4 a0 = lds128_align2(bp + UB - 16);
        const uint32_t x[4] = {a0.x, a0.y, a0.z, a0.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = x[i] & 0x0F0F0F0Fu;
            w[4 + i] = (x[i] >> 4) & 0x0F0F0F0Fu;
        }
        if constexpr (TYPE != GQ_TYPE_Q4_1) {
            const uint32_t qh = lds16(bp + UB - 20) | (lds16(bp + UB - 18) << 16);
            // four bits to bit 4 of four bytes: the products' copies of the bits do not overlap
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] |= ((((qh >> (4 * i)) & 0xFu) * 0x00204081u) & 0x01010101u) << 4;
        }
    } else if constexpr (TYPE == GQ_TYPE_Q2_K) {
        // scales[16] | qs[64] | d | dmin; value 128h + 32j + i = bits 2j..2j+1 of qs[32h + i]
        const uint8_t* sp = row + 84 * (b >> 4);
        const int kb = b & 15, h = kb >> 3, j = (kb >> 1) & 3;
        const int sc = sp[kb];
        A = __fmul_rn(h2f(lds16(sp + 80)), static_cast<float>(sc & 0xF));
        B = __fmul_rn(h2f(lds16(sp + 82)), static_cast<float>(sc >> 4));
        const uint4 x = lds128_align2(sp + 16 + 32 * h + 16 * (kb & 1));
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (xw[i] >> (2 * j)) & 0x03030303u;
    } else if constexpr (TYPE == GQ_TYPE_Q3_K) {
        // hmask[32] | qs[64] | scales[12] | d; third bit = bit 4h + j of hmask[i]; 6-bit scale
        // kb: low four bits of byte kb % 8 (its high nibble for kb >= 8), top two from bits
        // 2(kb/4).. of byte 8 + kb % 4, minus 32
        const uint8_t* sp = row + 110 * (b >> 4);
        const int kb = b & 15, h = kb >> 3, j = (kb >> 1) & 3, b0 = 16 * (kb & 1);
        const int low = kb < 8 ? (sp[96 + kb] & 0xF) : (sp[96 + kb - 8] >> 4);
        const int top = (sp[104 + (kb & 3)] >> (2 * (kb >> 2))) & 3;
        A = __fmul_rn(h2f(lds16(sp + 108)), static_cast<float>((low | (top << 4)) - 32));
        const uint4 x = lds128_align2(sp + 32 + 32 * h + b0);
        const uint4 m = lds128_align2(sp + b0);
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, mw[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = ((xw[i] >> (2 * j)) & 0x03030303u) | (((mw[i] >> (4 * h + j)) & 0x01010101u) << 2);
    } else {   // Q4_0: d | nibbles[16]; value j < 16 low nibble of byte j, else high of j - 16
        const uint8_t* bp = row + 18 * b;
        A = h2f(lds16(bp));
        const uint4 a0 = lds128_align2(bp + 2);
        const uint32_t x[4] = {a0.x, a0.y, a0.z, a0.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = x[i] & 0x0F0F0F0Fu;
            w[4 + i] = (x[i] >> 4) & 0x0F0F0F0Fu;
        }
    }
}

// 32 consecutive values (values 32 s on) of a row: one block, or two of 16 values
template <int TYPE, bool UNITS16 = false>
__device__ __forceinline__ void decode32(const uint8_t* row, int s, uint32_t (&w)[8], float (&A)[32 / BlockView<TYPE>::BV],
                                         float (&B)[32 / BlockView<TYPE>::BV]) {
    if constexpr (TYPE == GQ_TYPE_Q6_K) {
        const uint8_t* sp = row + 210 * (s >> 3);
        const int h = (s >> 2) & 1, g = s & 3;
        const float d = h2f(lds16(sp + 208));
        const uint32_t sc = lds16(sp + 192 + 2 * (s & 7));
        A[0] = __fmul_rn(d, static_cast<float>(static_cast<int8_t>(sc)));
        A[1] = __fmul_rn(d, static_cast<float>(static_cast<int8_t>(sc >> 8)));
        B[0] = B[1] = 0.0f;
        // low nibbles or high ones of 32 bytes, and bits 2g.. of 32 more moved to bits 4 and 5
        uint32_t q[8];
        load32_bits(sp + 64 * h + 32 * (g & 1), 4 * (g >> 1), w);
        load32_bits(sp + 128 + 32 * h, 2 * g - 4, q);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = (w[i] & 0x0F0F0F0Fu) | (q[i] & 0x30303030u);
    } else if constexpr (TYPE == GQ_TYPE_Q8_0) {
        const uint8_t* bp = row + 34 * s;
        A[0] = h2f(lds16(bp));
        B[0] = 0.0f;
        load32_bits(bp + 2, 0, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] ^= 0x80808080u;
    } else {
        constexpr int NP = 32 / BlockView<TYPE>::BV, NW = BlockView<TYPE>::NW;
#pragma unroll
        for (int b = 0; b < NP; ++b) {
            uint32_t x[8];
            decode_block<TYPE, UNITS16>(row, NP * s + b, x, A[b], B[b]);
#pragma unroll
            for (int i = 0; i < NW; ++i) w[NW * b + i] = x[i];
        }
    }
}

// x of code q, as gguf-py computes it (Q8_0: x * d, the same product)
template <int TYPE>
__device__ __forceinline__ float block_value(float A, float B, int q) {
    const float p = __fmul_rn(A, static_cast<float>(q));
    return BlockView<TYPE>::kSub ? __fsub_rn(p, B) : p;
}

}  // namespace gq
