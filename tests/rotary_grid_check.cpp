// The grid of a rotation: within the limits of a launch and over every token, column and head, up to the longest
// calls that are accepted.
#include <climits>
#include <cstdio>
#include <initializer_list>

#include "rotary_grid.cuh"

int main() {
    using namespace rkv;
    int bad = 0;
    for (int D : {8, 24, 64, 96, 128, 256})
        for (int pairs : {1, 3, 4, 8, 12, 24, 32, 48, 64, 128})
            for (int vec : {1, 2, 4, 8})
                for (int heads : {1, 2, 7, 32, 40, 1000, 0x7FFFFFF})
                    for (int rows : {1, 2, 255, 256, 4096, 1 << 30, INT_MAX - 256, INT_MAX - 255, INT_MAX - 63, INT_MAX - 1, INT_MAX})
                        for (int batch : {1, 3, 65535}) {
                            if (2 * pairs > D || pairs % vec || D % vec) continue;
                            const RotGrid g = rotary_grid(D, pairs, vec, heads, rows, batch);
                            const bool ok = g.tiles >= 1 && g.tiles <= INT_MAX && g.tiles * g.tile >= rows && (g.tiles - 1) * g.tile < rows &&
                                            g.split >= 1 && g.split <= 65535 && g.slots >= 1 && g.tile >= 1 &&
                                            g.chunks * g.tile * g.slots <= kRotThreads && g.chunks * 2 * vec >= D &&
                                            g.turned * vec == pairs && (long long)g.slots * g.split <= 2LL * heads;
                            if (!ok && bad++ < 20)
                                std::printf("D %d, pairs %d, vec %d, heads %d, rows %d, batch %d: tile %d, slots %d, tiles %lld, split %lld\n", D,
                                            pairs, vec, heads, rows, batch, g.tile, g.slots, g.tiles, g.split);
                        }
    return bad ? 1 : 0;
}
