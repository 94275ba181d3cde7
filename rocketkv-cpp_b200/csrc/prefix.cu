// prefix.cu -- one token per sequence attended over a paged cache whose
// sequences share leading tokens, group by group.
//
// The softmax of a row (sequence, query head) is split between the tokens that
// its group shares and its own: parts with disjoint tokens, each (m, l, o) =
// (largest score, sum 2^(x - m), sum 2^(x - m) v) with x = q k log2(e) / sqrt(D),
// join as (M, sum l 2^(m - M), sum o 2^(m - M)).  A group's shared rows of K and V
// meet the queries of all its sequences at once, so they are read once and
// not once per sequence.  Two or three kernels: every sequence's own tokens
// with the shared ones (paged.cu), or before them where these run on the
// tcgen05 tensor cores (prefix_tc.cu), then the join; or, where the sequences
// alone fill the GPU, the shared tokens, then the own ones with the join.  Each
// is begun while the one before still runs.
//
// 24/8 heads of 128, bf16: 2 sequences behind 1024 tokens 11.6 us, 64 behind 8192
// with up to 512 of their own 48 (244 without sharing), 8 behind 131072 121, 104 at
// full clock (0.69, 0.81 of a copy's rate; 640 without sharing).  Not kept: the
// shared tokens first where a join follows (45 us -> 47, when that took 45), and the
// last CTA to arrive as the join (34 -> 42 for 24 sequences, when they took 34).
#include "prefix.cuh"

namespace rkv {
namespace {

struct JoinArgs {
    SharedArgs s;
    TcParts tc;  // where the shared tokens' parts are those of the tcgen05 kernel
    Result r;
};

template <typename T>
__device__ __forceinline__ void put4(T* o, const float4& v);
template <>
__device__ __forceinline__ void put4(float* o, const float4& v) { *reinterpret_cast<float4*>(o) = v; }
template <>
__device__ __forceinline__ void put4(__nv_bfloat16* o, const float4& v) {
    reinterpret_cast<__nv_bfloat162*>(o)[0] = __floats2bfloat162_rn(v.x, v.y);
    reinterpret_cast<__nv_bfloat162*>(o)[1] = __floats2bfloat162_rn(v.z, v.w);
}
template <>
__device__ __forceinline__ void put4(__half* o, const float4& v) {
    reinterpret_cast<__half2*>(o)[0] = __floats2half2_rn(v.x, v.y);
    reinterpret_cast<__half2*>(o)[1] = __floats2half2_rn(v.z, v.w);
}

constexpr int kJoinWarps = 8;  // of a CTA, which joins one row
constexpr int kJoinAhead = 4;  // parts of a warp that are on their way together

// Joins the parts of a row: those of its own tokens, then those of the shared
// ones, in their order whatever the grid.  O is rounded to Q's type, once.
template <typename T, bool TC, bool WIDE>
__global__ void __launch_bounds__(kJoinWarps * 32) prefix_join_kernel(const JoinArgs a) {
    const SharedArgs& s = a.s;
    constexpr int W = kJoinWarps, U = kJoinAhead;
    __shared__ float4 sums[W][WIDE ? 64 : 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long row = blockIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int2 info = s.info[row];
    const int own = info.x;
    int shared = info.y;
    int2 x = make_int2(0, 0);
    if (TC && shared > 0) {
        x = parts_behind(a.tc, row, shared);
        shared += x.x;
    }
    // own parts, then shared ones
    const int parts = own + shared;
    auto ml_of = [&](int i) { return i < own ? s.part_ml[row * s.slots + i] : shared_ml(s, a.tc, row, x, i - own); };
    auto o_of = [&](int i) { return i < own ? s.part_o + (row * s.slots + i) * s.D : shared_o(s, a.tc, row, x, i - own); };
    // warp w takes the parts w, w + W, ...; its first rows are on their way while the weights are formed
    const int c0 = lane * 4, c1 = c0 + 128;
    float4 v0[U], v1[U];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * W;
            v0[u] = v1[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i < parts) {
                const float* p = o_of(i);
                if (c0 < s.D) v0[u] = *reinterpret_cast<const float4*>(p + c0);
                if (WIDE && c1 < s.D) v1[u] = *reinterpret_cast<const float4*>(p + c1);
            }
        }
    };
    fetch(warp);
    float top = -INFINITY;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, ml_of(i).x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float base = top == -INFINITY ? 0.0f : top;
    float l = 0.0f;
    for (int i = lane; i < parts; i += 32) {
        const float2 v = ml_of(i);
        l = fmaf(v.y, exp2f(v.x - base), l);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    float4 o0 = make_float4(0.0f, 0.0f, 0.0f, 0.0f), o1 = o0;
    for (int i0 = warp; i0 < parts; i0 += U * W) {
        if (i0 != warp) fetch(i0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * W;
            const float f = i < parts ? exp2f(ml_of(i).x - base) : 0.0f;
            o0 = make_float4(fmaf(v0[u].x, f, o0.x), fmaf(v0[u].y, f, o0.y), fmaf(v0[u].z, f, o0.z), fmaf(v0[u].w, f, o0.w));
            if (WIDE) o1 = make_float4(fmaf(v1[u].x, f, o1.x), fmaf(v1[u].y, f, o1.y), fmaf(v1[u].z, f, o1.z), fmaf(v1[u].w, f, o1.w));
        }
    }
    sums[warp][lane] = o0;
    if (WIDE) sums[warp][lane + 32] = o1;
    __syncthreads();
    const int c = threadIdx.x * 4;
    if (c < s.D) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float4 o = sums[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < W; ++w) {
            const float4 v = sums[w][threadIdx.x];
            o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
        }
        put4(static_cast<T*>(a.r.O) + row * s.D + c, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
    if (threadIdx.x == 0 && a.r.lse) a.r.lse[row] = l == 0.0f ? -INFINITY : (base + log2f(l)) * 0.693147180559945f;
    if (a.r.err && blockIdx.x == 0 && threadIdx.x == 0) keep_error(a.r.err);
}

template <typename T>
int launch_join(const JoinArgs& a, cudaStream_t st) {
    const dim3 grid((unsigned)(a.s.batch * a.s.H)), block(kJoinWarps * 32);
    const bool wide = a.s.D > 128;
    const cudaError_t e = a.tc.first_o && wide ? launch_pdl(prefix_join_kernel<T, true, true>, grid, block, 0, st, a)
                          : a.tc.first_o       ? launch_pdl(prefix_join_kernel<T, true, false>, grid, block, 0, st, a)
                          : wide               ? launch_pdl(prefix_join_kernel<T, false, true>, grid, block, 0, st, a)
                                               : launch_pdl(prefix_join_kernel<T, false, false>, grid, block, 0, st, a);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}

int prefix_check(int dtype, int H, int HK, int D, int max_len, int batch, int groups) {
    if (!paged_dtype(dtype) || H <= 0 || HK <= 0 || H % HK != 0 || D <= 0 || max_len < 0 || batch < 0 || groups < 0)
        return RKV_ERR_INVALID_ARG;
    if (D % 8 != 0 || D > 256 || H / HK > 1024 || max_len > kMaxLen) return RKV_ERR_UNSUPPORTED;
    if ((long long)batch * H > 0x3FFFFFFFLL || groups > (1 << 24)) return RKV_ERR_UNSUPPORTED;
    return RKV_OK;
}

// The shared tokens on the tcgen05 tensor cores: 16-bit types where a group of mean size has more than 16 rows of a KV
// head (one CTA of the matrix-instruction kernel takes up to 16 with 128 columns, 8 above).  The groups themselves are
// known on the device alone, and num_groups counts empty ones too.  24/8 heads of 128, bf16, 64 sequences: one group
// behind 8192 tokens 49 us on the tensor cores, 91 as one of 12 groups and 130 as one of 64 on the other kernel; 16
// groups of 4 behind 2048 tokens 55 on the latter and 65 on the tensor cores, 64 groups of one 104 and 139.
bool on_tc(int dtype, int H, int HK, int D, int max_len, int batch, int groups) {
    const double tiles = ((double)groups + (double)batch * (H / HK) / 128) * HK * ((double)max_len / 64 + 1);
    return dtype != RKV_F32 && (long long)batch * (H / HK) > 16LL * groups && tiles < 1e9;  // counted in 32 bits
}

struct PrefixPlan {
    bool tc;
    int own, slots;
    size_t off_ml, off_o, off_info, off_first, off_first_ml, off_first_o, off_later_ml, off_later_o, bytes;
};
PrefixPlan prefix_plan(bool tc, int dtype, int H, int HK, int D, int max_len, int batch, int groups) {
    PrefixPlan p{};
    const bool any = groups > 0 && batch > 0;
    p.tc = any && tc && on_tc(dtype, H, HK, D, max_len, batch, groups);
    p.own = shared_own_parts(dtype, H, HK, D, max_len, batch, groups);
    p.slots = p.own + (any && !p.tc ? shared_prefix_parts(dtype, H, HK, D, max_len, batch, groups) : 0);
    size_t off = kWorkspaceHeader;
    auto take = [&](size_t& ml, size_t& o, size_t rows) {
        ml = off;
        off = align_up(off + rows * sizeof(float2), kWorkspaceAlign);
        o = off;
        off = align_up(off + rows * D * sizeof(float), kWorkspaceAlign);
    };
    take(p.off_ml, p.off_o, (size_t)batch * H * p.slots);
    p.off_info = off;
    off = align_up(off + (size_t)batch * H * sizeof(int2), kWorkspaceAlign);
    if (p.tc) {
        p.off_first = off;
        off = align_up(off + (size_t)batch * H * sizeof(int2), kWorkspaceAlign);
        take(p.off_first_ml, p.off_first_o, (size_t)batch * H);
        take(p.off_later_ml, p.off_later_o, (size_t)kTcSms * kTcRows);
    }
    p.bytes = off;
    return p;
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_prefix_decode_workspace_size(int dtype, int num_heads, int num_heads_kv, int dim_head, int max_len, int batch,
                                                int num_groups, size_t* bytes) {
    const int rc = prefix_check(dtype, num_heads, num_heads_kv, dim_head, max_len, batch, num_groups);
    if (rc || !bytes) return rc ? rc : (int)RKV_ERR_INVALID_ARG;
    *bytes = 0;  // the larger of the plans with the tcgen05 kernel and without
    for (bool tc : {true, false}) {
        const size_t n = prefix_plan(tc, dtype, num_heads, num_heads_kv, dim_head, max_len, batch, num_groups).bytes;
        if (n > *bytes) *bytes = n;
    }
    return RKV_OK;
}

extern "C" int rkv_prefix_decode(const void* Q, long long q_item_stride, int num_heads, const rkv_paged_cache* cache, int max_len,
                                 int batch, const int* group_starts, const int* group_tokens, int num_groups, void* O, float* lse,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    int rc = paged_check(cache, true, batch);
    if (!rc) rc = prefix_check(cache->dtype, num_heads, cache->num_heads_kv, cache->dim_head, max_len, batch, num_groups);
    if (rc) return rc;
    if (batch == 0) return RKV_OK;
    const int D = cache->dim_head, es = elem_size(cache->dtype);
    if (!Q || !O || ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(O)) & 15)) return RKV_ERR_INVALID_ARG;
    if (batch > 1 && (q_item_stride < (long long)num_heads * D * es || (q_item_stride & 15))) return RKV_ERR_INVALID_ARG;
    if (num_groups > 0 && (!group_starts || !group_tokens)) return RKV_ERR_INVALID_ARG;
    const bool tc = on_tc(cache->dtype, num_heads, cache->num_heads_kv, D, max_len, batch, num_groups) && prefix_tc_usable(cache->dtype, D);
    const PrefixPlan p = prefix_plan(tc, cache->dtype, num_heads, cache->num_heads_kv, D, max_len, batch, num_groups);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < p.bytes) return RKV_ERR_WORKSPACE;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    JoinArgs a{};
    SharedArgs& s = a.s;
    s.c = paged_view(*cache);
    s.gr = Groups{group_starts, group_tokens, num_groups, batch, max_len};
    s.Q = static_cast<const uint8_t*>(Q);
    s.q_stride = q_item_stride;
    s.dtype = cache->dtype;
    s.H = num_heads;
    s.HK = cache->num_heads_kv;
    s.D = D;
    s.batch = batch;
    s.own = p.own;
    s.slots = p.slots;
    s.part_ml = reinterpret_cast<float2*>(ws + p.off_ml);
    s.part_o = reinterpret_cast<float*>(ws + p.off_o);
    s.info = reinterpret_cast<int2*>(ws + p.off_info);
    a.r = Result{O, lse, nullptr};
    if (p.tc) {
        a.tc.first_later = reinterpret_cast<int2*>(ws + p.off_first);
        a.tc.first_ml = reinterpret_cast<float2*>(ws + p.off_first_ml);
        a.tc.first_o = reinterpret_cast<float*>(ws + p.off_first_o);
        a.tc.later_ml = reinterpret_cast<float2*>(ws + p.off_later_ml);
        a.tc.later_o = reinterpret_cast<float*>(ws + p.off_later_o);
        a.tc.err = static_cast<int*>(workspace);
    } else {
        a.r.err = static_cast<int*>(workspace);
    }
    if (p.own == 1) {
        // as many sequences as there is room for CTAs: each takes its own tokens in one part and joins the others' to it
        if (p.tc) rc = launch_prefix_tc(s, a.tc, 0, false, st);
        else if (num_groups > 0) rc = launch_shared_pass(s, SHARED_TOKENS, a.tc, a.r, false, st);
        return rc ? rc : launch_shared_pass(s, OWN_AND_JOIN, a.tc, a.r, num_groups > 0, st);
    }
    // side by side in one launch where both take CTAs of few rows
    const bool few = num_groups > 0 && !p.tc && shared_rows(s.dtype, D, num_heads, s.HK, batch, num_groups) <= 16;
    rc = launch_shared_pass(s, few ? ALL_TOKENS : OWN_TOKENS, a.tc, a.r, false, st);
    if (!rc && num_groups > 0 && !p.tc && !few) rc = launch_shared_pass(s, SHARED_TOKENS, a.tc, a.r, true, st);
    if (!rc && p.tc) rc = launch_prefix_tc(s, a.tc, batch * s.HK, true, st);
    if (rc) return rc;
    return s.dtype == RKV_F32 ? launch_join<float>(a, st) : s.dtype == RKV_BF16 ? launch_join<__nv_bfloat16>(a, st) : launch_join<__half>(a, st);
}
