// The listing rule of the weight selection over whole slices, as its warps walk them: every token that must be
// listed is listed exactly once, by the warp whose stretch holds it, and no other is.
#include <algorithm>
#include <cstdio>
#include <vector>

#include "weight_list.cuh"

namespace {

// A slice of ns tokens in stretches of `per`, of which [c0, c1) compete; marked(i): the token's key is at or
// above the threshold (the kernel marks 16 at a time where all do, and only tokens of the stretch otherwise).
template <typename F>
bool slice(int ns, int warps, int c0, int c1, bool all, F marked, const char* what) {
    const int per = ((ns + warps - 1) / warps + 31) / 32 * 32;
    std::vector<int> times(ns + 1024, 0);
    for (int w = 0; w < warps; ++w) {
        const int t0 = std::min(ns, w * per), t1 = std::min(ns, t0 + per);
        for (int g0 = t0; g0 < t1; g0 += 512)
            for (int lane = 0; lane < 32; ++lane) {
                const int i0 = g0 + lane * 16;
                unsigned f = 0;
                for (int e = 0; e < 16; ++e)
                    if (all || (i0 + e < t1 && marked(i0 + e))) f |= 1u << e;
                f = rkv::listed_tokens(f, i0, c0, c1, t1);
                for (int e = 0; e < 32; ++e)
                    if ((f >> e) & 1u) {
                        if (e >= 16 || i0 + e < t0 || i0 + e >= t1) {
                            std::printf("%s: ns %d, warp %d of stretch [%d, %d) lists token %d\n", what, ns, w, t0, t1, i0 + e);
                            return false;
                        }
                        ++times[i0 + e];
                    }
            }
    }
    for (int i = 0; i < ns; ++i) {
        const int want = i < c0 || i >= c1 || all || marked(i);
        if (times[i] != want) {
            std::printf("%s: ns %d, token %d listed %d times, %d wanted\n", what, ns, i, times[i], want);
            return false;
        }
    }
    return true;
}

}  // namespace

int main() {
    int bad = 0;
    for (int ns : {1, 15, 16, 17, 31, 33, 511, 512, 513, 1000, 2000, 8193, 16384, 17000, 20001, 40960})
        for (int sinks : {0, 1, 4, 17, 600})
            for (int recent : {0, 1, 32, 77, 700})
                for (int shift : {0, 5000}) {  // a slice that begins behind the list's first token, or ends before its last
                    const int c0 = std::max(0, sinks - shift), c1 = std::min(ns, ns - recent + (shift ? 300 : 0));
                    bad += !slice(ns, 32, c0, c1, true, [](int) { return true; }, "all");
                    bad += !slice(ns, 32, c0, c1, false, [](int) { return false; }, "none");
                    bad += !slice(ns, 32, c0, c1, false, [](int i) { return (i * 2654435761u >> 7) % 5 == 0; }, "some");
                }
    if (bad) std::printf("%d slices listed wrongly\n", bad);
    return bad ? 1 : 0;
}
