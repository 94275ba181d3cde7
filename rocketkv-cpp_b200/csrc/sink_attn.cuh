// sink_attn.cuh -- prefill attention with a sliding window and sinks: arguments.
#pragma once

#include "rkv_common.cuh"

namespace rkv {

struct SinkArgs {
    const uint8_t* Q;
    const uint8_t* K;
    const uint8_t* V;
    uint8_t* O;
    float* lse;
    const int* lens;
    rkv_row_strides qs, ks, os;  // bytes
    int batch, len_q, len_k, H, HK, G, D, sinks, window;
    int qtiles;
    float scale2;  // log2(e) / sqrt(D)
    int* err;
    // keys in parts, where there are too few queries to fill the GPU: each part's rows go to the workspace
    int parts;
    float* part_o;    // [parts][batch][H][len_q][D], not divided by l
    float2* part_ml;  // [parts][batch][H][len_q] (m, l), m in base 2
};

constexpr int kSinkSms = 148;
constexpr int kSinkTicket = 1;  // word of the workspace header from which CTAs draw their further items
constexpr int kSinkMaxParts = 16;
constexpr int kSinkPartTiles = 4;  // key tiles of a part at least
// Parts of the keys for `items` CTAs' worth of queries that visit at most `tiles` key tiles each.
inline int sink_parts(long long items, long long tiles) {
    if (items <= 0 || items * 2 > kSinkSms) return 1;
    long long p = kSinkSms / items;
    if (p > tiles / kSinkPartTiles) p = tiles / kSinkPartTiles;
    if (p > kSinkMaxParts) p = kSinkMaxParts;
    return p < 1 ? 1 : (int)p;
}
// The most tiles of bn keys that `rows` queries visit.
inline long long sink_tiles_max(long long len_k, long long sinks, long long window, int rows, int bn) {
    const long long all = (len_k + bn - 1) / bn;
    if (window <= 0) return all;
    const long long some = (sinks + bn - 1) / bn + (window + rows - 2) / bn + 2;
    return some < all ? some : all;
}

// Keys of item b, and the keys a tile of queries i0 .. i0 + rows - 1 visits:
// tiles of `bn` keys from 0 that hold a sink, then those from the oldest
// window start to the newest position.
struct SinkRange {
    int n, p0;          // valid keys; position of query i0
    int sink_tiles;     // tiles 0 .. sink_tiles - 1 first
    int first, end;     // then tiles first .. end - 1
    int begin;          // this part's first of all those
    __device__ int count() const { return sink_tiles + max(0, end - first); }
    __device__ int tile(int i) const { return begin + i < sink_tiles ? begin + i : first + (begin + i - sink_tiles); }
    // Restricts the range to one of `parts` parts; the tiles of it.
    __device__ int part(int k, int parts) {
        const int all = count();
        begin = (int)((long long)all * k / parts);
        return (int)((long long)all * (k + 1) / parts) - begin;
    }
};
__device__ __forceinline__ SinkRange sink_range(const SinkArgs& a, int b, int i0, int rows, int bn) {
    SinkRange r;
    r.begin = 0;
    r.n = a.lens ? min(max(a.lens[b], 0), a.len_k) : a.len_k;
    r.p0 = i0 + a.len_k - a.len_q;
    const int pmax = min(r.p0 + min(rows, a.len_q - i0) - 1, r.n - 1);  // newest position with a row to write
    if (pmax < r.p0) {
        r.sink_tiles = r.first = r.end = 0;
        return r;
    }
    r.end = pmax / bn + 1;
    const int oldest = a.window > 0 ? max(0, r.p0 - a.window + 1) : 0;
    r.first = oldest / bn;
    r.sink_tiles = min((min(a.sinks, pmax + 1) + bn - 1) / bn, r.first);
    return r;
}
__device__ __forceinline__ bool sink_sees(const SinkArgs& a, int n, int p, int j) {
    return j <= p && j < n && (a.window <= 0 || j < a.sinks || j > p - a.window);
}

// 16-bit inputs on the tcgen05 tensor cores (sink_attn_tc.cu)
int launch_sink_tc(SinkArgs a, int dtype, int batch, cudaStream_t st);
// CTAs' worth of queries of that kernel, and the rows and keys of one's tiles
long long sink_tc_items(const SinkArgs& a, int* rows, int* keys);

}  // namespace rkv
