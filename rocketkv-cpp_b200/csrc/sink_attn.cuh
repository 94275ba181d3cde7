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
};

// Keys of item b, and the keys a tile of queries i0 .. i0 + rows - 1 visits:
// tiles of `bn` keys from 0 that hold a sink, then those from the oldest
// window start to the newest position.
struct SinkRange {
    int n, p0;          // valid keys; position of query i0
    int sink_tiles;     // tiles 0 .. sink_tiles - 1 first
    int first, end;     // then tiles first .. end - 1
    __device__ int count() const { return sink_tiles + max(0, end - first); }
    __device__ int tile(int i) const { return i < sink_tiles ? i : first + (i - sink_tiles); }
};
__device__ __forceinline__ SinkRange sink_range(const SinkArgs& a, int b, int i0, int rows, int bn) {
    SinkRange r;
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

}  // namespace rkv
