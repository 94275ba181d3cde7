// paged_evict.cu -- eviction from a paged KV cache by accumulated attention
// weight: per (sequence, KV head) the sinks, the most recent tokens and the
// heaviest of the others stay, and their rows and weights move to the front.
//
// The selection is a radix select over order-preserving 32-bit keys of the
// weights (four 8-bit digits, largest first) followed by one ordered pass that
// lists the tokens above the threshold and the first ones equal to it.
#include "paged.cuh"

namespace rkv {
namespace {

constexpr int kSelNT = 1024;

struct WEvictArgs {
    PagedView c, o;  // source and destination
    float* w;
    float* wo;
    int w_stride, max_len, budget, sinks, recent;
    int HK, kept_stride, list;  // list: min(budget, max_len) entries of a kept row
    int* kept;
    int* new_lens;
    long long rowb;
    int vpr;      // vectors per row
    int inplace;  // rows move within their own pages
};

// Larger weight, larger key; -0 ranks as 0, NaN below every number.
__device__ __forceinline__ uint32_t weight_key(float w) { return w != w ? 0u : float_key(w + 0.0f); }

// One CTA per (item, KV head).
__global__ void __launch_bounds__(kSelNT) weight_select_kernel(const WEvictArgs a) {
    __shared__ unsigned hist[256];
    __shared__ int tmp[66];
    __shared__ unsigned s_digit, s_above;
    const int hk = blockIdx.x % a.HK, b = blockIdx.x / a.HK, tid = threadIdx.x;
    const int n = paged_len(a.c, b, a.max_len);
    int* kept = a.kept + ((size_t)b * a.HK + hk) * a.kept_stride;
    const float* w = a.w + ((size_t)b * a.HK + hk) * a.w_stride;
    const int keep = min(n, a.budget);
    if (hk == 0 && tid == 0) a.new_lens[b] = keep;
    for (int i = keep + tid; i < a.list; i += kSelNT) kept[i] = -1;
    if (n <= a.budget) {
        for (int i = tid; i < n; i += kSelNT) kept[i] = i;
        return;
    }
    const int lo = a.sinks, hi = n - a.recent;  // the tokens that compete: lo .. hi - 1, more than m of them
    const int m = a.budget - a.sinks - a.recent;
    for (int i = tid; i < lo; i += kSelNT) kept[i] = i;
    for (int i = tid; i < a.recent; i += kSelNT) kept[lo + m + i] = hi + i;
    if (m == 0) return;
    uint32_t prefix = 0;
    unsigned need = m;  // still to be taken among the keys that share the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (int t = lo + tid; t < hi; t += kSelNT) {
            const uint32_t k = weight_key(w[t]);
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            unsigned above = 0;
            int d = 255;
            while (d > 0 && above + hist[d] < need) above += hist[d--];
            s_digit = d;
            s_above = above;
        }
        __syncthreads();
        prefix |= s_digit << shift;
        need -= s_above;
    }
    // keys above prefix: all; equal to it: the first `need`
    int base = 0, ties = 0;
    for (int t0 = lo; t0 < hi; t0 += kSelNT) {
        const int t = t0 + tid;
        const uint32_t k = t < hi ? weight_key(w[t]) : 0u;
        const int gt = t < hi && k > prefix, eq = t < hi && k == prefix;
        int pe, tg, te;
        const int pg = block_exclusive_scan2(gt, eq, tmp, &pe, &tg, &te);
        // entries before this one: those above the threshold, and the ties among the first `need`
        const int tie_before = min(ties + pe, (int)need) - min(ties, (int)need);
        if (gt || (eq && ties + pe < (int)need)) kept[lo + base + pg + tie_before] = t;
        base += tg + min(ties + te, (int)need) - min(ties, (int)need);
        ties += te;
    }
}

constexpr int kMoveNT = 256, kMoveVPT = 4;

// Rows of K and V.  A kept list ascends and kept[i] >= i, so in place a row
// is overwritten only by rows whose sources lie at or behind it: reading a
// chunk's sources before writing any of its destinations keeps every source.
// In place one CTA walks the chunks of its (item, head) in order, and the row
// is cut into column slices so that several CTAs share it; otherwise the
// chunks spread over the grid.  slice_v: vectors of a slice.
__global__ void __launch_bounds__(kMoveNT) weight_move_kernel(const WEvictArgs a, int slices, int slice_v) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int hk = blockIdx.y % a.HK, b = blockIdx.y / a.HK;
    const int n = paged_len(a.c, b, a.max_len), keep = min(n, a.budget);
    if (a.inplace && keep == n) return;
    const int* kept = a.kept + ((size_t)b * a.HK + hk) * a.kept_stride;
    const bool isv = blockIdx.z & 1;
    const int v0 = (blockIdx.z >> 1) * slice_v, nv = min(slice_v, a.vpr - v0);
    const uint8_t* src = isv ? a.c.V : a.c.K;
    uint8_t* dst = isv ? a.o.V : a.o.K;
    const int rows = kMoveNT * kMoveVPT / nv;  // per chunk
    const int chunks = (keep + rows - 1) / rows;
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        uint4 x[kMoveVPT];
        long long to[kMoveVPT];
#pragma unroll
        for (int u = 0; u < kMoveVPT; ++u) {
            const int g = threadIdx.x + u * kMoveNT;
            const int r = g / nv, i = c * rows + r, vec = v0 + g - r * nv;
            to[u] = -1;
            if (r < rows && i < keep) {
                const int t = kept[i];
                if (!(a.inplace && t == i)) {
                    const long long from = paged_offset(a.c, b, hk, t);
                    if (from >= 0 && (long long)i < (long long)a.o.table_stride * a.o.page_size)
                        to[u] = paged_offset(a.o, b, hk, i);
                    if (to[u] >= 0) {
                        to[u] += vec * 16;
                        x[u] = *reinterpret_cast<const uint4*>(src + from + vec * 16);
                    }
                }
            }
        }
        if (a.inplace) __syncthreads();  // every source of the chunk read before a destination is written
#pragma unroll
        for (int u = 0; u < kMoveVPT; ++u)
            if (to[u] >= 0) *reinterpret_cast<uint4*>(dst + to[u]) = x[u];
        if (a.inplace) __syncthreads();
    }
}

// The kept weights to the front (in order, chunk by chunk, so in place is
// safe), zeros behind them up to max_len.
__global__ void __launch_bounds__(kSelNT) weight_shift_kernel(const WEvictArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int hk = blockIdx.x % a.HK, b = blockIdx.x / a.HK;
    const int keep = min(paged_len(a.c, b, a.max_len), a.budget);
    const int* kept = a.kept + ((size_t)b * a.HK + hk) * a.kept_stride;
    const float* w = a.w + ((size_t)b * a.HK + hk) * a.w_stride;
    float* wo = a.wo + ((size_t)b * a.HK + hk) * a.w_stride;
    for (int i0 = 0; i0 < keep; i0 += kSelNT) {
        const int i = i0 + threadIdx.x;
        const float x = i < keep ? w[kept[i]] : 0.0f;
        __syncthreads();
        if (i < keep) wo[i] = x;
        __syncthreads();
    }
    for (int i = keep + threadIdx.x; i < a.max_len; i += kSelNT) wo[i] = 0.0f;
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
    a.rowb = (long long)cache->dim_head * elem_size(cache->dtype);
    a.vpr = (int)(a.rowb / 16);
    a.inplace = !out || (out->block_table == cache->block_table && out->K == cache->K && out->V == cache->V);
    if (out && a.inplace &&
        (out->page_size != cache->page_size || out->page_stride != cache->page_stride ||
         out->head_stride != cache->head_stride || out->token_stride != cache->token_stride ||
         out->table_stride != cache->table_stride || out->num_pages != cache->num_pages))
        return RKV_ERR_INVALID_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    weight_select_kernel<<<(unsigned)units, kSelNT, 0, st>>>(a);
    if ((rc = launched())) return rc;
    int slices = 1, slice_v = a.vpr, split = 1;
    if (a.inplace) {
        while (slices < 4 && slice_v % 2 == 0 && slice_v >= 4) {
            slices *= 2;
            slice_v /= 2;
        }
    } else {
        const int rows = kMoveNT * kMoveVPT / slice_v;
        const int chunks = (list + rows - 1) / rows;
        split = chunks < 64 ? (chunks > 0 ? chunks : 1) : 64;
    }
    if (launch_pdl(weight_move_kernel, dim3(split, (unsigned)units, 2 * slices), dim3(kMoveNT), 0, st, a, slices, slice_v) !=
        cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    weight_shift_kernel<<<(unsigned)units, kSelNT, 0, st>>>(a);
    return launched();
}
