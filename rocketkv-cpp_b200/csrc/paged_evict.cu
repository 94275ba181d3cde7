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
//
// bf16, 8 KV heads of 128, to other pages, device time: 64 ragged sequences of
// up to 3717 tokens to 1024, 90 us (481 MB), of which the selection takes 16
// and the copy 74; 8 x 131072 tokens (fp16) to 4096, 88 us (337 MB), 37 and 42;
// one of 2112 tokens to 2048, 9.5 us.  Memory bounds the copies; chains of digit counts,
// barriers and scans bound the selections (a weight is read from memory once
// and, in a long cache, a second time from L2; the zeros behind the kept weights
// are written in between).
#include <cooperative_groups.h>

#include <type_traits>

#include "paged.cuh"
#include "weight_list.cuh"

namespace cg = cooperative_groups;

namespace rkv {
namespace {

constexpr int kBins = 2048, kPasses = 3;
constexpr int kSliceMax = 32768;  // tokens of a slice whose keys and lists are in shared memory (192 KB beside the counts)

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
    int list_cap; // entries of a warp's list where the slice is not in shared memory
    int inplace;  // rows move within their own pages
};

// Larger weight, larger key; -0 ranks as 0, NaN below every number.
__device__ __forceinline__ uint32_t weight_key(float w) {
    const int b = __float_as_int(w + 0.0f);
    return w != w ? 0u : (uint32_t)(b ^ ((b >> 31) | (int)0x80000000));
}
// The weight of a key (-0 has become 0, a NaN is the canonical one).
__device__ __forceinline__ float key_weight(uint32_t k) {
    return k == 0u ? __int_as_float(0x7FC00000) : __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

constexpr int kMaxCluster = 8;

struct SelShared {
    unsigned hist[kPasses][kBins];
    unsigned warp_sum[32];
    unsigned digit, above;
    int count[2];               // tokens of the slice that stay outright, ties
    int wcount[2][32];
};

static_assert(sizeof(SelShared) % 16 == 0, "keys behind it are 16-byte aligned");

// dst[i] = 0 for lo <= i < hi, the cluster's threads in turn.
__device__ __forceinline__ void zero_tail(float* dst, int lo, int hi, int thread, int threads) {
    const int mis = (int)((reinterpret_cast<uintptr_t>(dst + lo) >> 2) & 3);
    const int body = min(hi, lo + (mis ? 4 - mis : 0)), quads = (hi - body) / 4;
    if (thread < body - lo) dst[lo + thread] = 0.0f;
    for (int i = thread; i < quads; i += threads)
        *reinterpret_cast<float4*>(dst + body + 4 * i) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (thread < hi - body - 4 * quads) dst[body + 4 * quads + thread] = 0.0f;
}

// One cluster per (item, KV head); every CTA has a slice of the tokens, every
// warp a stretch of the slice.  All weights are looked at twice, for the first
// and the second digit; in the second look each warp of a CTA of 1024 threads
// lists, in order, the tokens whose first digit is at or above the threshold's
// (a few per cent of a long cache), and the third digit, the counts and the
// output work on those lists.  RESIDENT: the slice's keys stay in shared memory, lists always fit,
// and the kept weights are written from there (in place is safe: every slice
// has been read before the first cluster barrier).  Otherwise the second look
// reads L2, a list holds keys too, a warp whose list is full looks at its
// whole stretch again instead, and in place weight_shift_kernel moves the
// weights afterwards.
template <int NT, bool RESIDENT, bool CLUSTER>
__global__ void __launch_bounds__(NT) weight_select_kernel(const WEvictArgs a) {
    asm volatile("griddepcontrol.launch_dependents;");
    constexpr int W = NT / 32;
    constexpr bool LISTS = NT == 1024;  // short lists of tokens are looked at whole
    static_assert(LISTS || RESIDENT, "without lists the keys are in shared memory");
    constexpr int EB = 4;  // loads of four weights that a thread has on their way together
    extern __shared__ __align__(16) uint8_t smem[];
    SelShared& S = *reinterpret_cast<SelShared*>(smem);
    uint32_t* skey = reinterpret_cast<uint32_t*>(smem + sizeof(SelShared));  // [slice] keys, or [W][list_cap] of the lists
    uint16_t* sidx = reinterpret_cast<uint16_t*>(skey + (RESIDENT ? a.slice : W * a.list_cap));
    cg::cluster_group cl = cg::this_cluster();
    const int CS = CLUSTER ? (int)cl.num_blocks() : 1, rank = CLUSTER ? (int)cl.block_rank() : 0;
    auto sync_all = [&] {
        if (CLUSTER)
            cl.sync();
        else
            __syncthreads();
    };
    const int unit = blockIdx.x / CS, hk = unit % a.HK, b = unit / a.HK;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ct = rank * NT + tid, cthreads = CS * NT;  // thread of the cluster
    const int n = paged_len(a.c, b, a.max_len), keep = min(n, a.budget);
    int* kept = a.kept + (size_t)unit * a.kept_stride;
    const float* w = a.w + (size_t)unit * a.w_stride;
    float* wo = a.wo + (size_t)unit * a.w_stride;
    const bool write_w = RESIDENT || wo != w;

    if (rank == 0 && hk == 0 && tid == 0) a.new_lens[b] = keep;
    for (int i = keep + ct; i < a.list; i += cthreads) kept[i] = -1;
    if (n <= a.budget) {
        for (int i = ct; i < n; i += cthreads) {
            kept[i] = i;
            if (wo != w) wo[i] = w[i];
        }
        if (write_w) zero_tail(wo, keep, a.max_len, ct, cthreads);
        return;  // the same for every CTA of the cluster
    }
    for (int i = tid; i < kPasses * kBins / 4; i += NT) reinterpret_cast<uint4*>(S.hist)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const int lo_t = (int)min((long long)n, (long long)rank * a.slice);
    const int ns = min(n - lo_t, a.slice);  // this slice
    const float* ws = w + lo_t;
    // the part of the slice that competes: more than m tokens over all slices
    const int c0 = max(0, a.sinks - lo_t), c1 = min(ns, n - a.recent - lo_t);
    const int m = a.budget - a.sinks - a.recent;
    const int per = ((ns + W - 1) / W + 31) / 32 * 32;
    const int t0 = min(ns, warp * per), t1 = min(ns, t0 + per);  // this warp's stretch
    const int cap = RESIDENT ? per : a.list_cap;
    uint16_t* li = sidx + (RESIDENT ? t0 : warp * a.list_cap);
    uint32_t* lk = skey + warp * a.list_cap;  // keys of the list (not RESIDENT)
    int nlist = 0;
    bool dense = !LISTS || per > 65536;  // indices of a stretch have 16 bits

    uint32_t prefix = 0;
    unsigned need = m;  // still to be taken among the keys that share the prefix
    // the digit at which `need` falls, over the cluster's counts: thread i sums BPT bins from the top
    auto find_digit = [&](int pass, int shift) {
        sync_all();
        constexpr int BPT = kBins / NT;  // 2 or 4
        unsigned v[BPT], sum = 0;
#pragma unroll
        for (int e = 0; e < BPT; ++e) v[e] = 0;
#pragma unroll
        for (int r = 0; r < (CLUSTER ? kMaxCluster : 1); ++r)
            if (r < CS) {
                const unsigned* h = CLUSTER ? cl.map_shared_rank(&S.hist[pass][0], r) : &S.hist[pass][0];
                h += kBins - BPT * (tid + 1);
#pragma unroll
                for (int e = 0; e < BPT; e += 2) {
                    const uint2 x = *reinterpret_cast<const uint2*>(h + BPT - 2 - e);
                    v[e] += x.y, v[e + 1] += x.x;
                }
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
        unsigned before = __reduce_add_sync(0xffffffffu, lane < warp ? S.warp_sum[lane] : 0u) + inc - sum;
        if (before < need && before + sum >= need) {  // one thread, unless need is 0
            int e = 0;
            while (before + v[e] < need) before += v[e++];
            S.digit = kBins - 1 - (BPT * tid + e);
            S.above = before;
        }
        if (need == 0 && tid == 0) S.digit = 0, S.above = 0;
        __syncthreads();
        prefix |= S.digit << shift;
        need -= S.above;
    };

    // four weights at a time where the rows are 16-byte aligned (a.slice is a multiple of four)
    const bool vec4 = ((reinterpret_cast<uintptr_t>(ws)) & 15) == 0;
    const int qlo = t0 / 4, qfull = t1 / 4, qend = t1 > t0 ? (t1 + 3) / 4 : qfull;
    auto weights4 = [&](int q, auto vec, float (&x)[4]) {
        if (decltype(vec)::value) {
            const float4 y = q < qfull ? *reinterpret_cast<const float4*>(ws + 4 * q) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = q < qfull ? ws[4 * q + e] : 0.0f;
        }
    };
    auto tail4 = [&](float (&x)[4]) {  // the quad that the slice ends in
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = 4 * qfull + e < t1 ? ws[4 * qfull + e] : 0.0f;
    };
    // first digit
    auto count4 = [&](int q, const float (&x)[4]) {
        const int at = 4 * q;
        uint32_t k[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) k[e] = weight_key(x[e]);
        if (RESIDENT) *reinterpret_cast<uint4*>(skey + at) = make_uint4(k[0], k[1], k[2], k[3]);
        if (at >= c0 && at + 4 <= c1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) atomicAdd(&S.hist[0][k[e] >> 21], 1u);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (at + e >= c0 && at + e < c1) atomicAdd(&S.hist[0][k[e] >> 21], 1u);
        }
    };
    auto first_digit = [&](auto vec) {
        for (int q0 = qlo + lane; q0 < qfull; q0 += 32 * EB) {
            float x[EB][4];
#pragma unroll
            for (int u = 0; u < EB; ++u) weights4(q0 + 32 * u, vec, x[u]);
#pragma unroll
            for (int u = 0; u < EB; ++u)
                if (q0 + 32 * u < qfull) count4(q0 + 32 * u, x[u]);
        }
        if (qfull < qend && lane == 0) {
            float x[4];
            tail4(x);
            count4(qfull, x);
        }
    };
    if (vec4)
        first_digit(std::true_type{});
    else
        first_digit(std::false_type{});
    find_digit(0, 21);
    if (write_w) zero_tail(wo, keep, a.max_len, ct, cthreads);
    // Second digit, and the lists: tokens whose key is at or above the prefix.  A lane looks at 16 tokens in a
    // row, so one scan over the lanes places 512 tokens; what it marks is compared as floats where it comes
    // from global memory, and a prefix of -infinity's digit or below (3: keys there are no numbers) marks all.
    const bool all = (prefix >> 21) <= 3u;
    const float bar = key_weight(prefix);
    if (!LISTS)
        for (int i = t0 + lane; i < t1; i += 32) {
            const uint32_t k = skey[i];
            if ((k >> 21) == (prefix >> 21) && i >= c0 && i < c1) atomicAdd(&S.hist[1][(k >> 10) & 2047], 1u);
        }
    for (int g0 = t0; LISTS && g0 < t1; g0 += 512) {
        const int i0 = g0 + lane * 16;
        unsigned f = 0;
        if (i0 + 16 <= t1 && (RESIDENT || vec4)) {
            uint4 y[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                y[u] = RESIDENT ? *reinterpret_cast<const uint4*>(skey + i0 + 4 * u)
                                : *reinterpret_cast<const uint4*>(ws + i0 + 4 * u);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t k[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    f |= (RESIDENT ? k[e] >= prefix : __uint_as_float(k[e]) >= bar) ? 1u << (4 * u + e) : 0u;
            }
        } else {
            for (int e = 0; e < 16; ++e)
                if (i0 + e < t1) f |= (RESIDENT ? skey[i0 + e] >= prefix : ws[i0 + e] >= bar) ? 1u << e : 0u;
        }
        if (all) f = 0xFFFFu;
        if (m == 0) f = 0;
        f = listed_tokens(f, i0, c0, c1, t1);
        const int c = __popc(f);
        int inc = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        const int total = __shfl_sync(0xffffffffu, inc, 31);
        if (nlist + total > cap) dense = true;
        int to = nlist + inc - c;
        while (f) {
            const int i = i0 + __ffs(f) - 1;
            f &= f - 1;
            const uint32_t k = RESIDENT ? skey[i] : weight_key(ws[i]);
            if (!dense) {
                li[to] = (uint16_t)(i - t0);
                if (!RESIDENT) lk[to] = k;
                ++to;
            }
            if ((k >> 21) == (prefix >> 21) && i >= c0 && i < c1) atomicAdd(&S.hist[1][(k >> 10) & 2047], 1u);
        }
        __syncwarp();
        if (!dense) nlist += total;
    }
    __syncwarp();
    // entry j of the warp's list (of its stretch where that is dense): token and key
    const int items = dense ? t1 - t0 : nlist;
    auto entry = [&](int j, int& i, uint32_t& k) {
        i = t0 + (dense ? j : (int)li[j]);
        k = RESIDENT ? skey[i] : dense ? weight_key(ws[i]) : lk[j];
        return i >= c0 && i < c1;  // competes
    };
    find_digit(1, 10);
    for (int j = lane; j < items; j += 32) {
        int i;
        uint32_t k;
        if (entry(j, i, k) && (k >> 10) == (prefix >> 10)) atomicAdd(&S.hist[2][k & 1023], 1u);
    }
    find_digit(2, 0);
    // What stays: sinks, recent, keys above prefix; of those equal to it the first `need`.  Where nothing
    // competes (m == 0) no key may count: cut is out of reach then.
    const uint32_t cut = m > 0 ? prefix : 0xFFFFFFFFu;
    int stays = 0, ties = 0;
    for (int j = lane; j < items; j += 32) {
        int i;
        uint32_t k;
        const bool comp = entry(j, i, k);
        stays += !comp || k > cut;
        ties += comp && k == cut;
    }
    stays = __reduce_add_sync(0xffffffffu, stays);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane == 0) S.wcount[0][warp] = stays, S.wcount[1][warp] = ties;
    __syncthreads();
    // stays and ties before this warp's stretch
    int bs = __reduce_add_sync(0xffffffffu, lane < warp ? S.wcount[0][lane] : 0);
    int bt = __reduce_add_sync(0xffffffffu, lane < warp ? S.wcount[1][lane] : 0);
    if (CLUSTER) {
        if (warp == W - 1 && lane == 0) S.count[0] = bs + stays, S.count[1] = bt + ties;
        cl.sync();
#pragma unroll
        for (int r = 0; r < kMaxCluster; ++r)
            if (r < rank) {
                const int* c = cl.map_shared_rank(&S.count[0], r);
                bs += c[0], bt += c[1];
            }
    }
    const int nt = (int)need;
    const unsigned lt = (1u << lane) - 1;
    for (int j0 = 0; j0 < items; j0 += 32) {
        int i = 0;
        uint32_t k = 0;
        const bool in = j0 + lane < items, comp = in && entry(j0 + lane, i, k);
        const bool stay = in && (!comp || k > cut), tie = comp && k == cut;
        const unsigned ms = __ballot_sync(0xffffffffu, stay), mt = __ballot_sync(0xffffffffu, tie);
        const int tb = bt + __popc(mt & lt);
        if (stay || (tie && tb < nt)) {
            const int pos = bs + __popc(ms & lt) + min(tb, nt);
            kept[pos] = lo_t + i;
            if (write_w) wo[pos] = key_weight(k);
        }
        bs += __popc(ms);
        bt += __popc(mt);
    }
    if (CLUSTER) cl.sync();  // no CTA leaves while its counts are being read
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
    zero_tail(wo, keep, a.max_len, threadIdx.x, 1024);
}

constexpr int kMoveNT = 256;

// Rows to other pages: 2^lg lanes per row (the row's vectors, rounded up),
// K and V by the same thread, kCopyRows rows in flight per thread (64 ragged
// sequences / 8 x 131072 tokens, whole eviction: 102 / 90 us with 1, 90 / 89
// with 2, 100 / 97 with 4, 127 / 117 with 8).
constexpr int kCopyRows = 2;
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
// source, and later chunks may be read earlier still.  One CTA walks the
// chunks of an (item, head) in order, with the next kMoveAhead chunks' sources
// on their way to shared memory (each thread's own vectors); the row is cut
// into slices of slice_v vectors, and K and V are apart, so that several CTAs
// share it.  Memory latency bounds it, a chunk after the other: the whole
// eviction in place, bf16, 8 KV heads of 128: 64 x 3717 tokens to 1024 124 us,
// 8 x 131072 to 8192 185, one of 2112 tokens to 1024 17.  2 vectors a thread
// and 3 chunks ahead were best (64 / 8 sequences 138 / 185 us; 1 and 3 139 /
// 248, 4 and 3 181 / 204, 2 and 5 163 / 263), and slices to 296 CTAs (124 /
// 185 us; to 592 124 / 216, to 1184 132 / 216).
constexpr int kMoveVPT = 2, kMoveAhead = 3;
constexpr long long kMoveCTAs = 2 * 148;  // as many at least, if the row's slices allow it
constexpr int kMoveSmem = (kMoveAhead + 1) * kMoveVPT * kMoveNT * 16;
__global__ void __launch_bounds__(kMoveNT) weight_move_kernel(const WEvictArgs a, int slice_v) {
    constexpr int S = kMoveAhead + 1, U = kMoveVPT;
    extern __shared__ __align__(16) uint8_t smem[];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int unit = blockIdx.y, hk = unit % a.HK, b = unit / a.HK;
    const int n = paged_len(a.c, b, a.max_len), keep = min(n, a.budget);
    if (keep == n) return;
    const int* kept = a.kept + (size_t)unit * a.kept_stride;
    const int* table = a.c.table + (size_t)b * a.c.table_stride;
    const unsigned page = a.c.page_size;
    uint8_t* base = (blockIdx.x & 1) ? a.c.V : a.c.K;
    const int v0 = (blockIdx.x >> 1) * slice_v, nv = min(slice_v, a.vpr - v0);
    const int rows = kMoveNT * U / nv;  // per chunk
    const int chunks = (keep + rows - 1) / rows;
    uint8_t* mine = smem + threadIdx.x * 16;
    // A source's address takes two loads, its place in the list and its page; each is asked for a chunk before
    // the next step needs it.
    int row[U], vec[U];                 // of a chunk
    int t2[U], t1[U], pf[U], pt[U];     // tokens of the chunk after the next; of the next, and its pages
    long long to[S][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int g = threadIdx.x + u * kMoveNT;
        row[u] = g / nv;
        vec[u] = (v0 + g - row[u] * nv) * 16;
        if (row[u] >= rows) row[u] = 0x40000000;  // the chunk's remainder
    }
    auto place = [&](int c, int u) { return c < chunks && row[u] < keep - c * rows ? c * rows + row[u] : -1; };
    auto tokens = [&](int c) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = place(c, u);
            t2[u] = i >= 0 ? kept[i] : -1;
        }
    };
    auto pages = [&](int c) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = place(c, u);
            t1[u] = t2[u] == i ? -1 : t2[u];  // a row that is in its place stays
            pf[u] = pt[u] = -1;
            if (t1[u] >= 0) {
                pf[u] = table[(unsigned)t1[u] / page];
                pt[u] = table[(unsigned)i / page];
            }
        }
    };
    auto fetch = [&](int c, long long* dst, int s) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            dst[u] = -1;
            if ((unsigned)pf[u] < (unsigned)a.c.num_pages && (unsigned)pt[u] < (unsigned)a.c.num_pages) {
                const unsigned i = c * rows + row[u], t = t1[u];
                dst[u] = pt[u] * a.c.page_stride + hk * a.c.head_stride + (long long)(i % page) * a.c.token_stride + vec[u];
                const long long from = pf[u] * a.c.page_stride + hk * a.c.head_stride + (long long)(t % page) * a.c.token_stride + vec[u];
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(mine + (s * U + u) * kMoveNT * 16)),
                             "l"(base + from)
                             : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        pages(c + 1);
        tokens(c + 2);
    };
    tokens(0);
    pages(0);
    tokens(1);
#pragma unroll
    for (int s = 0; s < kMoveAhead; ++s) fetch(s, to[s], s);
    for (int c0 = 0; c0 < chunks; c0 += S) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (c0 + s >= chunks) break;
            fetch(c0 + s + kMoveAhead, to[(s + kMoveAhead) % S], (s + kMoveAhead) % S);
            asm volatile("cp.async.wait_group %0;" ::"n"(kMoveAhead) : "memory");
            __syncthreads();  // every source of the chunk read before a destination is written
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (to[s][u] >= 0)
                    *reinterpret_cast<uint4*>(base + to[s][u]) = *reinterpret_cast<const uint4*>(mine + (s * U + u) * kMoveNT * 16);
        }
    }
}

template <int NT, bool RESIDENT, bool CLUSTER>
int launch_select(const WEvictArgs& a, long long units, int CS, cudaStream_t st) {
    // keys, and 16-bit indices where there are lists
    const size_t smem = sizeof(SelShared) + (RESIDENT ? (size_t)a.slice : (size_t)(NT / 32) * a.list_cap) * (NT == 1024 ? 6 : 4);
    if (cudaFuncSetAttribute(weight_select_kernel<NT, RESIDENT, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
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
    lc.blockDim = dim3(NT);
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    lc.attrs = at;
    lc.numAttrs = CLUSTER ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&lc, weight_select_kernel<NT, RESIDENT, CLUSTER>, a);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_weight_evict(const rkv_paged_cache* cache, float* weights, int weight_stride, int max_len, int batch,
                                int budget, int sinks, int recent, const rkv_paged_cache* out, float* weights_out,
                                int* kept, int kept_stride, int* new_lens, void* stream) {
    int rc = paged_check(cache, true, batch);
    if (rc) return rc;
    if (max_len < 0 || batch < 0 || budget < 0 || sinks < 0 || recent < 0 || (long long)sinks + recent > budget)
        return RKV_ERR_INVALID_ARG;
    if (max_len > kMaxLen) return RKV_ERR_UNSUPPORTED;
    if (out) {
        if ((rc = paged_check(out, false, batch))) return rc;
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
    // the rows that any sequence can keep have a place
    const long long from = (long long)cache->table_stride * cache->page_size, most = list < from ? list : from;
    if ((long long)a.o.table_stride * a.o.page_size < most) return RKV_ERR_INVALID_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    // Short lists: a CTA of 512 threads each, four to an SM.  Longer ones: CTAs of 1024 threads, one to an SM,
    // as many to a list as give every SM one (a second wave costs more than a longer slice).
    int CS = 1;
    const bool small = max_len <= 8192;
    if (!small)
        while (CS < kMaxCluster && units * CS * 2 <= 148 && max_len > CS * 4096) CS *= 2;
    a.slice = ((max_len + CS - 1) / CS + 3) / 4 * 4;
    const bool resident = a.slice <= kSliceMax;
    a.list_cap = kSliceMax / 32;
    if (small)
        rc = launch_select<512, true, false>(a, units, 1, st);
    else if (resident)
        rc = CS > 1 ? launch_select<1024, true, true>(a, units, CS, st) : launch_select<1024, true, false>(a, units, 1, st);
    else
        rc = CS > 1 ? launch_select<1024, false, true>(a, units, CS, st) : launch_select<1024, false, false>(a, units, 1, st);
    if (rc) return rc;
    cudaError_t e = cudaSuccess;
    if (list == 0) {
        // no rows stay
    } else if (a.inplace) {
        int slices = 1, slice_v = a.vpr;
        while (units * 2 * slices < kMoveCTAs && slice_v % 2 == 0 && slice_v >= 4) {
            slices *= 2;
            slice_v /= 2;
        }
        e = cudaFuncSetAttribute(weight_move_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMoveSmem);
        if (e == cudaSuccess)
            e = launch_pdl(weight_move_kernel, dim3(2 * slices, (unsigned)units), dim3(kMoveNT), kMoveSmem, st, a, slice_v);
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
    if (resident || a.wo != a.w) return RKV_OK;
    weight_shift_kernel<<<(unsigned)units, 1024, 0, st>>>(a);
    return launched();
}
