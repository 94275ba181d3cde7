// paged_evict.cu -- eviction from a paged KV cache by accumulated attention
// weight: per (sequence, KV head) the sinks, the most recent tokens and the
// heaviest of the others stay, and their rows and weights move to the front.
//
// The selection finds the m-th largest weight by a radix select over
// order-preserving 32-bit keys (digits of 11, 11 and 10 bits, largest first);
// the tokens above it stay, and the first of those equal to it.  A cluster of
// CTAs shares one (sequence, head): each keeps a slice of the weights in its
// shared memory, so they are read once, and the digit counts meet through
// distributed shared memory.  Then the rows are copied, K and V by the same
// threads, or moved in place.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace rkv {
namespace {

constexpr int kSelNT = 512, kSelWarps = kSelNT / 32;
constexpr int kBins = 2048, kPasses = 3;
constexpr int kSliceMax = 49152;  // weights of a slice in shared memory (192 KB beside the counts)

struct WEvictArgs {
    PagedView c, o;  // source and destination
    float* w;
    float* wo;
    int w_stride, max_len, budget, sinks, recent;
    int HK, kept_stride, list;  // list: min(budget, max_len) entries of a kept row
    int* kept;
    int* new_lens;
    int vpr;      // 16-byte vectors of a row
    int slice;    // tokens of a CTA's slice
    int inplace;  // rows move within their own pages
};

// Larger weight, larger key; -0 ranks as 0, NaN below every number.
__device__ __forceinline__ uint32_t weight_key(float w) { return w != w ? 0u : float_key(w + 0.0f); }

struct SelShared {
    unsigned hist[kPasses][kBins];
    unsigned warp_sum[kSelWarps];
    unsigned digit, above;
    int count[2];               // tokens of the slice that stay outright, ties
    int wcount[2][kSelWarps];
};

// One cluster per (item, KV head).  RESIDENT: the slice stays in shared
// memory and the kept weights are written from there (so in place is safe:
// every slice has been read before the first cluster barrier); otherwise the
// weights are read again from global memory and moved by weight_shift_kernel.
template <bool RESIDENT>
__global__ void __launch_bounds__(kSelNT) weight_select_kernel(const WEvictArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    extern __shared__ __align__(16) uint8_t smem[];
    SelShared& S = *reinterpret_cast<SelShared*>(smem);
    float* sw = reinterpret_cast<float*>(smem + sizeof(SelShared));
    cg::cluster_group cl = cg::this_cluster();
    const int CS = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int unit = blockIdx.x / CS, hk = unit % a.HK, b = unit / a.HK;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = paged_len(a.c, b, a.max_len), keep = min(n, a.budget);
    int* kept = a.kept + (size_t)unit * a.kept_stride;
    const float* w = a.w + (size_t)unit * a.w_stride;
    float* wo = a.wo + (size_t)unit * a.w_stride;
    const int lo_t = min(n, rank * a.slice), hi_t = min(n, lo_t + a.slice), ns = hi_t - lo_t;  // this slice

    if (rank == 0 && hk == 0 && tid == 0) a.new_lens[b] = keep;
    for (int i = keep + rank * kSelNT + tid; i < a.list; i += CS * kSelNT) kept[i] = -1;
    if (n <= a.budget) {
        for (int i = rank * kSelNT + tid; i < n; i += CS * kSelNT) {
            kept[i] = i;
            if (RESIDENT && wo != w) wo[i] = w[i];
        }
        if (RESIDENT)
            for (int i = keep + rank * kSelNT + tid; i < a.max_len; i += CS * kSelNT) wo[i] = 0.0f;
        return;  // the same for every CTA of the cluster
    }
    const int first = a.sinks, last = n - a.recent;  // the tokens that compete: first .. last - 1, more than m
    const int m = a.budget - a.sinks - a.recent;
    for (int i = tid; i < kPasses * kBins; i += kSelNT) (&S.hist[0][0])[i] = 0;
    if (RESIDENT)
        for (int i = tid; i < ns; i += kSelNT) sw[i] = w[lo_t + i];
    __syncthreads();
    auto weight = [&](int i) { return RESIDENT ? sw[i] : w[lo_t + i]; };
    const int c0 = max(0, first - lo_t), c1 = min(ns, last - lo_t);  // competing part of the slice
    uint32_t prefix = 0;
    unsigned need = m;  // still to be taken among the keys that share the prefix
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        const uint32_t mask = pass == 0 ? 0u : 0xFFFFFFFFu << (shift + bits);
        for (int i = c0 + tid; i < c1; i += kSelNT) {
            const uint32_t k = weight_key(weight(i));
            if ((k & mask) == prefix) atomicAdd(&S.hist[pass][(k >> shift) & ((1 << bits) - 1)], 1u);
        }
        cl.sync();
        // thread i sums bins 4 i .. 4 i + 3 from the top over the cluster; a scan finds where `need` falls
        constexpr int BPT = kBins / kSelNT;
        unsigned v[BPT], sum = 0;
#pragma unroll
        for (int e = 0; e < BPT; ++e) v[e] = 0;
        for (int r = 0; r < CS; ++r) {
            const unsigned* h = cl.map_shared_rank(&S.hist[pass][0], r);
            const uint4 x = *reinterpret_cast<const uint4*>(h + kBins - BPT * (tid + 1));
            v[0] += x.w, v[1] += x.z, v[2] += x.y, v[3] += x.x;
        }
#pragma unroll
        for (int e = 0; e < BPT; ++e) sum += v[e];
        unsigned inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) S.warp_sum[warp] = inc;
        __syncthreads();
        unsigned before = inc - sum;
        for (int x = 0; x < warp; ++x) before += S.warp_sum[x];
        if (before < need && before + sum >= need) {  // one thread, unless need is 0
            int e = 0;
            while (before + v[e] < need) before += v[e++];
            S.digit = kBins - 1 - (BPT * tid + e);
            S.above = before;
        }
        if (need == 0 && tid == 0) S.digit = kBins - 1, S.above = 0;
        __syncthreads();
        prefix |= S.digit << shift;
        need -= S.above;
    }
    // what stays: sinks, recent, keys above prefix; of those equal to it the first `need`.  m == 0: nothing
    // competes (prefix is then the largest key, which no weight but a NaN with that sign has, and need is 0)
    auto flags = [&](int i, bool& stay, bool& tie) {
        const int t = lo_t + i;
        const bool forced = t < first || t >= last;
        const uint32_t k = weight_key(weight(i));
        stay = forced || (m > 0 && k > prefix);
        tie = !forced && m > 0 && k == prefix;
    };
    // every warp takes a stretch of the slice: counts, then the places
    const int per = ((ns + kSelWarps - 1) / kSelWarps + 31) / 32 * 32;
    const int w0 = min(ns, warp * per), w1 = min(ns, w0 + per);
    int cs = 0, ct = 0;
    for (int i0 = w0; i0 < w1; i0 += 32) {
        bool stay = false, tie = false;
        if (i0 + lane < w1) flags(i0 + lane, stay, tie);
        cs += __popc(__ballot_sync(0xffffffffu, stay));
        ct += __popc(__ballot_sync(0xffffffffu, tie));
    }
    if (lane == 0) S.wcount[0][warp] = cs, S.wcount[1][warp] = ct;
    __syncthreads();
    if (tid < 2) {
        int x = 0;
        for (int i = 0; i < kSelWarps; ++i) x += S.wcount[tid][i];
        S.count[tid] = x;
    }
    cl.sync();
    int bs = 0, bt = 0;  // stays and ties before this warp's stretch
    for (int r = 0; r < rank; ++r) {
        const int* c = cl.map_shared_rank(&S.count[0], r);
        bs += c[0], bt += c[1];
    }
    for (int i = 0; i < warp; ++i) bs += S.wcount[0][i], bt += S.wcount[1][i];
    const int nt = (int)need;
    for (int i0 = w0; i0 < w1; i0 += 32) {
        bool stay = false, tie = false;
        if (i0 + lane < w1) flags(i0 + lane, stay, tie);
        const unsigned ms = __ballot_sync(0xffffffffu, stay), mt = __ballot_sync(0xffffffffu, tie), lt = (1u << lane) - 1;
        const int tb = bt + __popc(mt & lt);
        if (stay || (tie && tb < nt)) {
            const int pos = bs + __popc(ms & lt) + min(tb, nt);
            kept[pos] = lo_t + i0 + lane;
            if (RESIDENT) wo[pos] = weight(i0 + lane);
        }
        bs += __popc(ms);
        bt += __popc(mt);
    }
    if (RESIDENT)
        for (int i = keep + rank * kSelNT + tid; i < a.max_len; i += CS * kSelNT) wo[i] = 0.0f;
    cl.sync();  // no CTA leaves while its counts are being read
}

// The kept weights to the front where the selection did not hold them (chunk
// by chunk in order, so in place is safe), zeros behind them up to max_len.
__global__ void __launch_bounds__(1024) weight_shift_kernel(const WEvictArgs a) {
    const int unit = blockIdx.x, b = unit / a.HK;
    const int keep = min(paged_len(a.c, b, a.max_len), a.budget);
    const int* kept = a.kept + (size_t)unit * a.kept_stride;
    const float* w = a.w + (size_t)unit * a.w_stride;
    float* wo = a.wo + (size_t)unit * a.w_stride;
    for (int i0 = 0; i0 < keep; i0 += 1024) {
        const int i = i0 + threadIdx.x;
        const float x = i < keep ? w[kept[i]] : 0.0f;
        __syncthreads();
        if (i < keep) wo[i] = x;
        __syncthreads();
    }
    for (int i = keep + threadIdx.x; i < a.max_len; i += 1024) wo[i] = 0.0f;
}

constexpr int kMoveNT = 256;

// Rows to other pages: 2^lg lanes per row (the row's vectors, rounded up),
// K and V by the same thread, kCopyRows rows in flight per thread.
constexpr int kCopyRows = 4;
__global__ void __launch_bounds__(kMoveNT) weight_copy_kernel(const WEvictArgs a, int lg) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int unit = blockIdx.y, hk = unit % a.HK, b = unit / a.HK;
    const int keep = min(paged_len(a.c, b, a.max_len), a.budget);
    const int* kept = a.kept + (size_t)unit * a.kept_stride;
    const int per = kMoveNT >> lg, vec = threadIdx.x & ((1 << lg) - 1);  // rows of the CTA at a time
    const int i0 = blockIdx.x * per * kCopyRows + (threadIdx.x >> lg);
    if (vec >= a.vpr) return;
    const long long cap = (long long)a.o.table_stride * a.o.page_size;
    long long from[kCopyRows], to[kCopyRows];
#pragma unroll
    for (int u = 0; u < kCopyRows; ++u) {
        const int i = i0 + u * per;
        from[u] = to[u] = -1;
        if (i < keep && i < cap) {
            from[u] = paged_offset(a.c, b, hk, kept[i]);
            to[u] = paged_offset(a.o, b, hk, i);
        }
    }
    uint4 k[kCopyRows], v[kCopyRows];
#pragma unroll
    for (int u = 0; u < kCopyRows; ++u)
        if (from[u] >= 0 && to[u] >= 0) {
            k[u] = *reinterpret_cast<const uint4*>(a.c.K + from[u] + vec * 16);
            v[u] = *reinterpret_cast<const uint4*>(a.c.V + from[u] + vec * 16);
        }
#pragma unroll
    for (int u = 0; u < kCopyRows; ++u)
        if (from[u] >= 0 && to[u] >= 0) {
            *reinterpret_cast<uint4*>(a.o.K + to[u] + vec * 16) = k[u];
            *reinterpret_cast<uint4*>(a.o.V + to[u] + vec * 16) = v[u];
        }
}

// Rows within their own pages.  A kept list ascends and kept[i] >= i, so a
// row is overwritten only by rows whose sources lie at or behind it: reading
// a chunk's sources before writing any of its destinations keeps every
// source.  One CTA walks the chunks of an (item, head) in order; the row is
// cut into slices of slice_v vectors, and K and V are apart, so that several
// CTAs share it.
constexpr int kMoveVPT = 8;
__global__ void __launch_bounds__(kMoveNT) weight_move_kernel(const WEvictArgs a, int slice_v) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int unit = blockIdx.y, hk = unit % a.HK, b = unit / a.HK;
    const int n = paged_len(a.c, b, a.max_len), keep = min(n, a.budget);
    if (keep == n) return;
    const int* kept = a.kept + (size_t)unit * a.kept_stride;
    uint8_t* base = (blockIdx.x & 1) ? a.c.V : a.c.K;
    const int v0 = (blockIdx.x >> 1) * slice_v, nv = min(slice_v, a.vpr - v0);
    const int rows = kMoveNT * kMoveVPT / nv;  // per chunk
    for (int r0 = 0; r0 < keep; r0 += rows) {
        uint4 x[kMoveVPT];
        long long to[kMoveVPT];
#pragma unroll
        for (int u = 0; u < kMoveVPT; ++u) {
            const int g = threadIdx.x + u * kMoveNT;
            const int r = g / nv, i = r0 + r, vec = v0 + g - r * nv;
            to[u] = -1;
            if (r < rows && i < keep) {
                const int t = kept[i];
                if (t != i) {
                    const long long from = paged_offset(a.c, b, hk, t);
                    if (from >= 0) to[u] = paged_offset(a.c, b, hk, i);
                    if (to[u] >= 0) {
                        to[u] += vec * 16;
                        x[u] = *reinterpret_cast<const uint4*>(base + from + vec * 16);
                    }
                }
            }
        }
        __syncthreads();  // every source of the chunk read before a destination is written
#pragma unroll
        for (int u = 0; u < kMoveVPT; ++u)
            if (to[u] >= 0) *reinterpret_cast<uint4*>(base + to[u]) = x[u];
        __syncthreads();
    }
}

template <bool RESIDENT>
int launch_select(const WEvictArgs& a, long long units, int CS, cudaStream_t st) {
    const size_t smem = sizeof(SelShared) + (RESIDENT ? (size_t)a.slice * sizeof(float) : 0);
    if (cudaFuncSetAttribute(weight_select_kernel<RESIDENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
        cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CS;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t lc{};
    lc.gridDim = dim3((unsigned)(units * CS));
    lc.blockDim = dim3(kSelNT);
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    lc.attrs = at;
    lc.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&lc, weight_select_kernel<RESIDENT>, a);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_weight_evict(const rkv_paged_cache* cache, float* weights, int weight_stride, int max_len, int batch,
                                int budget, int sinks, int recent, const rkv_paged_cache* out, float* weights_out,
                                int* kept, int kept_stride, int* new_lens, void* stream) {
    int rc = paged_check(cache, true);
    if (rc) return rc;
    if (max_len < 0 || batch < 0 || budget < 0 || sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
        return RKV_ERR_INVALID_ARG;
    if (max_len > kMaxLen) return RKV_ERR_UNSUPPORTED;
    if (out) {
        if ((rc = paged_check(out, false))) return rc;
        if (out->dtype != cache->dtype || out->num_heads_kv != cache->num_heads_kv || out->dim_head != cache->dim_head)
            return RKV_ERR_INVALID_ARG;
    }
    if (out && out->block_table == cache->block_table && (out->K == cache->K) != (out->V == cache->V))
        return RKV_ERR_INVALID_ARG;  // one of K and V would move in place, the other not
    if (batch == 0) return RKV_OK;
    const int list = budget < max_len ? budget : max_len;
    if (!weights || weight_stride < max_len || !new_lens || new_lens == cache->lens) return RKV_ERR_INVALID_ARG;
    if (kept_stride < list || (list > 0 && !kept)) return RKV_ERR_INVALID_ARG;
    const long long units = (long long)batch * cache->num_heads_kv;
    if (units > 65535) return RKV_ERR_UNSUPPORTED;
    WEvictArgs a{};
    a.c = paged_view(*cache);
    a.o = out ? paged_view(*out) : a.c;
    a.w = weights;
    a.wo = weights_out ? weights_out : weights;
    a.w_stride = weight_stride;
    a.max_len = max_len;
    a.budget = budget;
    a.sinks = sinks;
    a.recent = recent;
    a.HK = cache->num_heads_kv;
    a.kept_stride = kept_stride;
    a.list = list;
    a.kept = kept;
    a.new_lens = new_lens;
    a.vpr = cache->dim_head * elem_size(cache->dtype) / 16;
    a.inplace = !out || (out->block_table == cache->block_table && out->K == cache->K && out->V == cache->V);
    if (out && a.inplace &&
        (out->page_size != cache->page_size || out->page_stride != cache->page_stride ||
         out->head_stride != cache->head_stride || out->token_stride != cache->token_stride ||
         out->table_stride != cache->table_stride || out->num_pages != cache->num_pages))
        return RKV_ERR_INVALID_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // CTAs of a cluster: slices of about 4096 tokens (8 weights a thread), at most eight
    int CS = 1;
    while (CS < 8 && max_len > CS * 4096) CS *= 2;
    a.slice = (max_len + CS - 1) / CS;
    const bool resident = a.slice <= kSliceMax;
    rc = resident ? launch_select<true>(a, units, CS, st) : launch_select<false>(a, units, CS, st);
    if (rc) return rc;
    cudaError_t e = cudaSuccess;
    if (list == 0) {
        // no rows stay
    } else if (a.inplace) {
        int slices = 1, slice_v = a.vpr;
        while (slices < 4 && slice_v % 2 == 0 && slice_v >= 4) {
            slices *= 2;
            slice_v /= 2;
        }
        e = launch_pdl(weight_move_kernel, dim3(2 * slices, (unsigned)units), dim3(kMoveNT), 0, st, a, slice_v);
    } else {
        int lg = 0;
        while ((1 << lg) < a.vpr) ++lg;
        const int per = (kMoveNT >> lg) * kCopyRows;
        e = launch_pdl(weight_copy_kernel, dim3((unsigned)((list + per - 1) / per), (unsigned)units), dim3(kMoveNT), 0, st, a, lg);
    }
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    if (resident) return RKV_OK;
    weight_shift_kernel<<<(unsigned)units, 1024, 0, st>>>(a);
    return launched();
}
