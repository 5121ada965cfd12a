// The matrix product's choice of kernel, for a test: lines of "m n k f32 sms" in, lines of
// "choice split longest" out, the choice as gq_choose.h has it (16, 32, 64, 128: a narrow tile's
// tokens; 256, 512: twice a wide tile's channels), split and longest (the blocks of 128 columns that
// one accumulator takes at most) of the narrow kernel or 1 and the wide one's piece.
#include <cstdio>

#include "gq_choose.h"

int main() {
    long long m, n, k;
    int f32, sms;
    while (std::scanf("%lld %lld %lld %d %d", &m, &n, &k, &f32, &sms) == 5) {
        const gq::ProductShape p{m, n, k, (k + 127) / 128};
        const int tile = gq::choose(p, f32 != 0, sms);
        int split = 1;
        long long longest = f32 ? std::min<long long>(gq::kPiece, p.kb) : p.kb;
        if (tile <= 128) {
            split = gq::narrow_split(p, tile, f32 != 0, sms);
            const long long blocks = (p.kb + split - 1) / split;
            const long long most = std::min<long long>(gq::narrow_pieces(tile, f32 != 0), (blocks + gq::kPiece - 1) / gq::kPiece);
            longest = (blocks + most - 1) / most;
        }
        std::printf("%d %d %lld\n", tile, split, longest);
    }
    return 0;
}
