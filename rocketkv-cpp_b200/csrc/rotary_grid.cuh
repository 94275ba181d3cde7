// rotary_grid.cuh -- how the rows of a rotation are laid over CTAs and threads.
// Plain integer arithmetic, compiled without CUDA too (tests/rotary_grid_check.cpp).
#pragma once

namespace rkv {

constexpr int kRotThreads = 256;
constexpr int kRotHeads = 8;         // heads of a thread at most, where there are tokens for all threads
constexpr int kRotBlocks = 148 * 2;  // CTAs that the heads are spread for

struct RotGrid {
    int chunks, turned;      // of a row (two vectors each), and those with pairs
    int tile, slots;         // tokens of a CTA, and its threads that share a token's chunk by heads
    long long tiles, split;  // CTAs along the tokens, and along the heads
};

// D columns of which 2 pairs are turned, vectors of vec elements; rows, heads and batch >= 1.
inline RotGrid rotary_grid(int D, int pairs, int vec, int heads, int rows, int batch) {
    RotGrid g{};
    g.turned = pairs / vec;
    g.chunks = g.turned + ((D - 2 * pairs) / vec + 1) / 2;  // at most 128
    g.slots = (int)(((long long)heads + kRotHeads - 1) / kRotHeads);
    if (g.slots > kRotThreads / g.chunks) g.slots = kRotThreads / g.chunks;
    g.tile = kRotThreads / (g.chunks * g.slots);
    if (g.tile > rows) g.tile = rows;
    g.slots = kRotThreads / (g.chunks * g.tile);
    if (g.slots > heads) g.slots = heads;
    g.tiles = ((long long)rows + g.tile - 1) / g.tile;
    g.split = (kRotBlocks + g.tiles * batch - 1) / (g.tiles * batch);
    const long long most = ((long long)heads + g.slots - 1) / g.slots;
    if (g.split > most) g.split = most;
    if (g.split > 65535) g.split = 65535;
    const long long each = (most + g.split - 1) / g.split;  // heads of a thread
    g.split = (most + each - 1) / each;
    return g;
}

}  // namespace rkv
