// prefix.cuh -- decode of a batch whose sequences share leading tokens: the groups, and the passes over them.
#pragma once

#include "paged.cuh"
#include "prefix_parts.cuh"

namespace rkv {

// Groups of sequences: group g is starts[g] .. starts[g + 1] - 1 and shares its first tokens[g] tokens.
struct Groups {
    const int* starts;  // [n + 1], ascending
    const int* tokens;  // [n]
    int n, batch, max_len;

    __device__ __forceinline__ int start(int g) const { return min(max(starts[g], 0), batch); }
    __device__ __forceinline__ int size(int g) const { return max(0, start(g + 1) - start(g)); }
    // Shared tokens of group g: at most what a sequence can hold.
    __device__ __forceinline__ int shared(const PagedView& c, int g) const {
        const long long cap = (long long)c.table_stride * c.page_size;
        const int n = min(tokens[g], max_len);
        return max(0, cap < n ? (int)cap : n);
    }
};

// Shared tokens that sequence b of n tokens takes from its group: all of the
// group's, or none where the sequence is shorter (it is attended on its own
// then, so that every row of a shared tile sees all of it).  A whole warp calls.
struct Member {
    int group, tokens;  // -1, 0: of none
};
__device__ __forceinline__ Member member_of(const Groups& gr, const PagedView& c, int b, int n) {
    const int lane = threadIdx.x & 31;
    Member m{-1, 0};
    for (int g0 = 0; g0 < gr.n; g0 += 32) {
        const int g = g0 + lane;
        const bool some = g < gr.n;
        const int lo = some ? gr.start(g) : 0, hi = some ? gr.start(g + 1) : 0, p = some ? gr.shared(c, g) : 0;
        const unsigned hits = __ballot_sync(0xffffffffu, lo <= b && b < hi);
        if (hits) {
            const int l = __ffs(hits) - 1;
            m.group = g0 + l;
            m.tokens = __shfl_sync(0xffffffffu, p, l);
            break;
        }
    }
    if (m.tokens > n) m.tokens = 0;
    return m;
}
// The sequence through whose table row a group's shared tokens are read: the first that holds them all.  A whole
// warp calls.
__device__ __forceinline__ int leader_of(const Groups& gr, const PagedView& c, int g, int shared) {
    const int lane = threadIdx.x & 31, s0 = gr.start(g), s1 = gr.start(g + 1);
    for (int b0 = s0; b0 < s1; b0 += 32) {
        const int b = b0 + lane;
        const unsigned hits = __ballot_sync(0xffffffffu, b < s1 && paged_len(c, b, gr.max_len) >= shared);
        if (hits) return b0 + __ffs(hits) - 1;
    }
    return s0;
}

// Tokens of a part (a multiple of 32) where `tokens` are taken in at most `splits` parts of kPartLeast tokens or so, as
// many as that allows, about the same for all.  6 sequences with up to 300 own tokens behind 4080, fp32: 15.6 us with
// parts of 128, 16.7 with 256.
constexpr int kPartLeast = 128;
__host__ __device__ __forceinline__ int part_tokens(int tokens, int splits) {
    int parts = (tokens + kPartLeast - 1) / kPartLeast;
    if (parts > splits) parts = splits;
    if (parts < 1) parts = 1;
    const int c = ((tokens + parts - 1) / parts + 31) / 32 * 32;
    return c < 32 ? 32 : c;
}

// What the passes leave: part s of row (sequence b, query head h) at ((b H + h) slots + s), o [D] not divided by l,
// and (m, l) in base 2.  Own tokens take the slots 0 .. own - 1, shared ones the others (where the matrix-instruction
// kernel of paged.cu attends them).  info[row]: its parts of own tokens, and of shared ones (tcgen05: 1 for any).
struct SharedArgs {
    PagedView c;
    Groups gr;
    const uint8_t* Q;
    long long q_stride;
    int dtype, H, HK, D, batch;
    int own, slots;
    float* part_o;
    float2* part_ml;
    int2* info;
};
// Rows of a group that one CTA of the matrix-instruction kernel takes.
int shared_rows(int dtype, int D, int H, int HK, int batch, int groups);
// Parts of every sequence's own tokens, and of every group's shared ones for the matrix-instruction kernel.
int shared_own_parts(int dtype, int H, int HK, int D, int max_len, int batch, int groups);
int shared_prefix_parts(int dtype, int H, int HK, int D, int max_len, int batch, int groups);
// The shared tokens on the tcgen05 tensor cores (prefix_tc.cu): 16-bit types.  A unit is up to 256 rows (128 above 128
// columns) of one group and KV head; the tiles of the units are cut into stretches, one or more per CTA.  A unit's
// first stretch leaves its rows in first (row b H + h), a stretch that begins inside a unit in later (256 rows per
// CTA).  first_later[row]: how many stretches follow the first one, and the row of the first of them in later; the
// others' are 256 further each.
struct TcParts {
    float* first_o;
    float2* first_ml;
    int2* first_later;
    float* later_o;
    float2* later_ml;
    int* err;
};
// first_later[row] for a row with a part of shared tokens (some: 1).  A pair that the kernel cannot have written, which
// is there where it gave up a wait: the row is joined without shared tokens, and the call's error stays recorded.
__device__ __forceinline__ int2 parts_behind(const TcParts& t, long long row, int some) {
    const int2 x = t.first_later[row];
    if (parts_in_buffer(x.x, x.y)) return x;
    atomicCAS(t.err, 0, (int)RKV_ERR_DEVICE_TIMEOUT);
    return make_int2(-some, 0);
}
// Part p of row's shared tokens, wherever the pass over them left it; x: parts_behind of row.
__device__ __forceinline__ float2 shared_ml(const SharedArgs& s, const TcParts& t, long long row, int2 x, int p) {
    return !t.first_o ? s.part_ml[row * s.slots + s.own + p] : p == 0 ? t.first_ml[row] : t.later_ml[x.y + (p - 1) * kTcRows];
}
__device__ __forceinline__ const float* shared_o(const SharedArgs& s, const TcParts& t, long long row, int2 x, int p) {
    return !t.first_o ? s.part_o + (row * s.slots + s.own + p) * s.D
           : p == 0   ? t.first_o + row * s.D
                      : t.later_o + (long long)(x.y + (p - 1) * kTcRows) * s.D;
}
// The error word of a workspace that may have held anything: an error stays until it is read, all else is none.
__device__ __forceinline__ void keep_error(int* err) {
    if (*err != (int)RKV_ERR_DEVICE_TIMEOUT) *err = RKV_OK;
}
// Where the last pass leaves its rows, and the error word, where no pass before it has looked at it.
struct Result {
    void* O;  // [batch][H][D] of the cache's type
    float* lse;
    int* err;
};

// Passes of the matrix-instruction kernel: the groups' shared tokens, every sequence's own, or both; or the own ones in
// one part, joined with the parts of the shared ones that the launch before has left.
enum SharedPass { SHARED_TOKENS, OWN_TOKENS, ALL_TOKENS, OWN_AND_JOIN };
// dependent: launched while the kernel before it still runs, which it waits for at its end only.
int launch_shared_pass(const SharedArgs& s, SharedPass pass, const TcParts& t, const Result& r, bool dependent, cudaStream_t st);
// Whether the tcgen05 kernel can run as compiled (also where that is not known: the launch says so then); where it
// cannot, the matrix-instruction kernel attends the shared tokens.
bool prefix_tc_usable(int dtype, int D);
// spare: CTAs of the kernel before that hold an SM each; dependent as above.
int launch_prefix_tc(const SharedArgs& s, const TcParts& p, int spare, bool dependent, cudaStream_t st);

}  // namespace rkv
