// Which kernel and tile a matrix product takes (gq_matmul.cu).  Host arithmetic alone, so that it
// can be compiled and tested where there is no GPU.
#pragma once

#include <algorithm>
#include <cstdint>

namespace gq {

// The matrix instructions truncate as they add, so a sum's error grows with its length (1.7e-6 of
// the result's norm over 112 blocks of 128 columns).  Where the output keeps f32, a sum is taken in
// pieces of about kPiece blocks (half as many again at most) that are added in f32 with rounding
// (up to 3.5e-7 measured); 16-bit outputs lose nothing without.
constexpr int kPiece = 32;
constexpr int kLongestPiece = kPiece + kPiece / 2;

// Pieces that a narrow tile of bn tokens has accumulators for
constexpr int narrow_pieces(int bn, bool f32) { return !f32 || bn == 128 ? 1 : bn == 16 ? 4 : 3; }

struct ProductShape {
    int64_t m, n, k, kb;      // kb = ceil(k / 128)
};

// Whether a CTA's part of a narrow product's sums is too long for its accumulators
inline bool narrow_too_long(const ProductShape& p, int bn, int split, bool f32) {
    return f32 && p.kb > static_cast<int64_t>(kLongestPiece) * narrow_pieces(bn, f32) * split;
}

// How k is split: until about two CTAs per SM, with at least two 128-column blocks for each; and
// further where the pieces of a sum would be too long (3 x 19100 x 32768 to f32: 117 us, and 98 in
// pieces of 64 blocks, off by 8.4e-7).
inline int narrow_split(const ProductShape& p, int bn, bool f32, int sms) {
    const int64_t tiles = (p.m + bn - 1) / bn * ((p.n + 127) / 128);
    int split = 1;
    while (split < 8 && ((tiles * split <= sms && p.kb >= 4 * split) || narrow_too_long(p, bn, split, f32))) split *= 2;
    return split;
}

// Which kernel and tile: the least estimated time (us).  A narrow tile costs what its operands
// take through an SM's read path (133 KB a us), the busiest SM counts, and no less than reading
// the operands from HBM (6.3 MB a us); set-up and the sums' way out grow with the tile and come
// again with every round of CTAs.  A wide
// one costs its tiles (0.287 us per 256 x 256 x 128 on a pair, the matrix instructions' rate; 0.19 per
// 256 x 128 x 128, where the way from the L2 bounds it: 24 KB per SM) and a drain, in rounds over
// the pairs.  Measured against it (us, k = 4096 unless said; the best and the runner-up): 64 x 28672
// narrow 64 23.2, narrow 128 24.7; 96 x 28672 narrow 128 26.1, wide 256 30.3; 160 x 28672 wide 256
// 31.5, wide 128 33.8; 128 x 4096 narrow 64 9.0, wide 128 11.0; 512 x 4096 wide 128 12.0, narrow 64
// 14.6; 768 x 4096 wide 256 16.8, wide 128 17.5; 160 x 4096, k = 14336 narrow 128 20.4, narrow 64
// 24.0.  At most 1.11 times the best over 27 such shapes (512 x 4096, k = 512: 6.2 against 5.6).
// Returns the narrow tile's tokens, or twice the wide tile's output channels.
inline int choose(const ProductShape& p, bool f32, int sms) {
    const double hbm = static_cast<double>(p.m + p.n) * static_cast<double>(p.k) / 6.3e6;
    int best = 16;
    double least = 1e30;
    const auto take = [&](int what, double us) {
        if (us < least) {
            least = us;
            best = what;
        }
    };
    for (int bn : {16, 32, 64, 128}) {
        const int split = narrow_split(p, bn, f32, sms);
        if (narrow_too_long(p, bn, split, f32)) continue;
        const int64_t ctas = (p.m + bn - 1) / bn * ((p.n + 127) / 128) * split;
        const double bytes = static_cast<double>((ctas + sms - 1) / sms) * static_cast<double>((p.kb + split - 1) / split) * (128 + bn) * 128;
        const double rounds = static_cast<double>((ctas + 2 * sms - 1) / (2 * sms));      // two CTAs on an SM
        take(bn, rounds * (3.0 + 0.032 * bn) + (split > 1 ? 1.0 : 0.0) + std::max(bytes / 133e3, hbm));
    }
    for (int bn : {128, 256}) {
        const int64_t tiles = (p.m + 255) / 256 * ((p.n + bn - 1) / bn), pairs = sms / 2;
        const double each = bn == 128 ? 0.19 * static_cast<double>(p.kb) + 1.7 : 0.287 * static_cast<double>(p.kb) + 2.8;
        take(2 * bn, 5.0 + std::max(static_cast<double>((tiles + pairs - 1) / pairs) * each, hbm));
    }
    return best;
}

}  // namespace gq
