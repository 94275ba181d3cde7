// Which pairs (stretches that follow, row of the first of them) the joins of the shared-prefix decode take: every one
// that the tcgen05 kernel writes, and none that leads behind the buffer or to more parts than the joins have room for.
#include <climits>
#include <cstdio>

#include "prefix_parts.cuh"

int main() {
    using namespace rkv;
    int bad = 0;
    auto fail = [&](const char* what, int behind, int row) { bad += std::printf("%s: %d, %d\n", what, behind, row) > 0; };
    // CTA c leaves the first stretch of a unit; the next CTAs, up to the last one, have the others'
    for (int c = 0; c < kTcSms; ++c)
        for (int behind = 0; c + behind < kTcSms; ++behind)
            for (int r = 0; r < kTcRows; ++r)
                if (!parts_in_buffer(behind, (c + 1) * kTcRows + r)) fail("refused", behind, (c + 1) * kTcRows + r);
    const long long rows = (long long)kTcSms * kTcRows;
    const int values[] = {INT_MIN, INT_MIN + 1, -(1 << 24), -257, -256, -2, -1, 0, 1, 2, 146, 147, 148, 149, 152, 255, 256, 257, 1 << 16,
                          kTcSms * kTcRows - 1, kTcSms * kTcRows, 1 << 24, 0x7FC00000, INT_MAX - 1, INT_MAX};
    for (int behind : values)
        for (int row : values) {
            if (!parts_in_buffer(behind, row)) continue;
            if (behind < 0 || 1 + behind > kMaxShared) fail("more parts than there is room for", behind, row);
            for (int p = 1; p <= behind; ++p) {
                const long long at = row + (p - 1LL) * kTcRows;
                if (at < 0 || at >= rows) fail("behind the buffer", behind, row);
            }
        }
    // (56 + 200) * 256 registers are the 128 * 512 of an SM
    for (int regs = 0; regs <= 255; ++regs)
        if (split_fits(regs) != (regs >= 128)) fail("registers", regs, 0);
    return bad ? 1 : 0;
}
