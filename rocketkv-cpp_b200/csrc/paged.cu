// paged.cu -- a paged KV cache on the device: rows appended to its pages, and
// the attention of one new token over it.
//
// The attention.  For query head h of KV head hk the scores of the visible
// tokens are x_t = (q . k_t) log2(e) / sqrt(D); with m the largest score seen
// and the running pair (l, o) = (sum 2^(x_t - m), sum 2^(x_t - m) v_t), a new
// token with a larger score rescales the pair by 2^(m_old - m_new), so K and V
// are read once.  Pairs of disjoint token sets join the same way, which is
// what splits the cache's length over CTAs: each CTA leaves (m, l, o) of its
// part and a second kernel joins the parts in order.  O = o / l,
// lse = (m + log2 l) ln 2.
//
// Memory bounds it: K and V are read once, 4 G flops per row of K and V of D
// 16-bit values for G heads that share it.  bf16, 24/8 heads of 128, device
// time: 8 x 131072 tokens 641 us (6.7 TB/s), 64 ragged sequences of up to 8192
// 182 us (6.3), 16 x 3717 with weights 50-55 us (5.0-4.5); fp32, 8 x 32768
// tokens, 327 us (6.6).  Where there is little to read it is two launches:
// 1 x 2048 tokens 7.3 us, an fp32 window of 1024 tokens 10-14 us.  Not kept: the
// parts of a head joined in a cluster's shared memory (64 ragged 201 us -> 301: parts
// without tokens hold their SM until the longest ends), and by the last CTA to
// arrive in place of the second kernel (182 -> 187, 1 x 2048 7.3 -> 8.4).
#include "paged.cuh"
#include "prefix.cuh"
#include "tf32.cuh"

namespace rkv {
namespace {

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendArgs {
    PagedView c;
    const uint8_t* k;
    const uint8_t* v;
    const int* n_new;
    long long item_stride, src_token, src_head;  // bytes
    int n_rows, HK, vpr;                         // vpr: vectors per row
};

// Consecutive threads take consecutive vectors of (row, head), so source rows
// that lie back to back are read in whole lines; kAppendVecs vectors of K and
// of V are on their way per thread before the first is stored.  Memory bounds
// it: 6 x 2048 rows (48 MB moved) 10.2 us, 4.7 TB/s, with 4 vectors (10.5 /
// 10.4 / 11.6 with 1 / 2 / 8); 64 rows 2.1 us, a launch.
constexpr int kAppendVecs = 4;
template <typename VT>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs a) {
    constexpr int U = kAppendVecs;
    const int b = blockIdx.y;
    const int n = a.n_new ? min(max(a.n_new[b], 0), a.n_rows) : a.n_rows;
    const int first = a.c.lens[b] - n;
    const long long cap = (long long)a.c.table_stride * a.c.page_size;
    const int per = a.HK * a.vpr;
    const long long total = (long long)n * per;
    for (long long e = (long long)blockIdx.x * (256 * U); e < total; e += (long long)gridDim.x * (256 * U)) {
        const int row = (int)(e / per);
        const unsigned rest = (unsigned)(e - (long long)row * per) + threadIdx.x;
        VT k[U], v[U];
        long long to[U];
        int vec[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const unsigned x = rest + u * 256;
            const int i = (int)(x / (unsigned)per), r = (int)(x - (unsigned)i * per), h = r / a.vpr;
            const long long t = (long long)first + row + i;
            vec[u] = r - h * a.vpr;
            to[u] = -1;
            if (i < n - row && t >= 0 && t < cap) {
                const size_t s = (size_t)b * a.item_stride + (size_t)(row + i) * a.src_token + (size_t)h * a.src_head;
                k[u] = reinterpret_cast<const VT*>(a.k + s)[vec[u]];
                v[u] = reinterpret_cast<const VT*>(a.v + s)[vec[u]];
                to[u] = paged_offset(a.c, b, h, (int)t);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (to[u] >= 0) {
                reinterpret_cast<VT*>(a.c.K + to[u])[vec[u]] = k[u];
                reinterpret_cast<VT*>(a.c.V + to[u])[vec[u]] = v[u];
            }
    }
}

// ---------------------------------------------------------------------------
// decode
// ---------------------------------------------------------------------------
constexpr int kTile = 32;       // parts are multiples of this many tokens
constexpr int kMinChunk = 128;  // visible tokens per CTA at least
constexpr int kMaxSplits = 1024;
constexpr int kSms = 148;
constexpr int kMaxWaves = 8;       // of CTAs that a cache is split into at most
constexpr int kJoinAhead = 16;     // parts of a column that the joins read before the shares are known
constexpr int kStartTokens = 128;  // what a CTA costs before and behind its tokens, in tokens

struct DecodeArgs {
    PagedView c;
    const uint8_t* Q;
    long long q_stride;
    int H, HK, G, D, max_len, sinks, window;
    int ngroups;         // groups of query heads per KV head
    int splits, chunk;   // parts of the visible tokens, tokens per part
    int vmax;            // row stride of the scores
    float scale2;        // log2(e) / sqrt(D)
    float* O;
    float* lse;
    float* weights;
    int weight_stride;
    float* part_o;       // [batch][H][splits][D]
    float2* part_ml;     // [batch][H][splits]
    float* scores;       // [batch][H][vmax], base-2 scores (with weights)
    long long o_blocks;  // join: CTAs that join O; the others add weights
    int w_blocks;        // join: CTAs per (item, KV head) that add weights
    // the passes of a batch that shares leading tokens
    SharedArgs sh;
    TcParts tc;
    Result res;
    int shared_blocks;  // CTAs of shared tokens, before those of own ones
    int units;         // shared tokens: row groups of all groups at most
    int prefix_parts;  // of the shared tokens at most, 0 where they are not this kernel's
};

// The visible tokens are numbered 0 .. nvis - 1: the sinks, then the window.
struct Visible {
    int n, sinks, gap, nvis;
    __device__ int token(int v) const { return v < sinks ? v : v + gap; }
};
__device__ __forceinline__ Visible visible(const DecodeArgs& a, int b) {
    Visible s;
    s.n = paged_len(a.c, b, a.max_len);
    const int w = a.window > 0 ? min(a.window, s.n) : s.n;
    const int start = s.n - w;
    s.sinks = min(a.sinks, start);
    s.gap = start - s.sinks;
    s.nvis = s.sinks + w;
    return s;
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
    return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// What a launch of the decode kernel attends: all tokens of every sequence; or, of a batch that shares leading tokens,
// parts of every group's shared ones with the rows of all its sequences, and of every sequence's own; or the own ones
// last, joined with the others' parts.
enum { PASS_ALL = 0, PASS_PARTS = 1, PASS_LAST = 2 };

enum { KIND_F16 = 0, KIND_BF16 = 1, KIND_F32 = 2 };

// 0 in place of -inf, so that a set with nothing in it subtracts no infinities.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

// Joins the warps' (m, l, o) of ng heads from shared memory (ms, ls [warps][rows], os [warps][rows][pitch])
// and writes the part, or the output where there is one part.
template <int W>
__device__ __forceinline__ void merge_warps(const DecodeArgs& a, size_t head0, int ng, int split, const float* ms,
                                            const float* ls, const float* os, int rows, int pitch) {
    const int D = a.D;
    for (int i = threadIdx.x; i < ng * D; i += W * 32) {
        const int g = i / D, d = i - g * D;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) mm = fmaxf(mm, ms[w * rows + g]);
        const float mf = finite_max(mm);
        float ll = 0.0f, oo = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float c = exp2f(ms[w * rows + g] - mf);
            ll = fmaf(ls[w * rows + g], c, ll);
            oo = fmaf(os[(w * rows + g) * pitch + d], c, oo);
        }
        const size_t head = head0 + g;
        if (a.splits == 1) {
            a.O[head * D + d] = ll == 0.0f ? 0.0f : oo / ll;
            if (d == 0 && a.lse) a.lse[head] = ll == 0.0f ? -INFINITY : (mf + log2f(ll)) * 0.693147180559945f;
        }
        if (a.part_o) {
            if (a.splits > 1) a.part_o[(head * a.splits + split) * D + d] = oo;
            if (d == 0) a.part_ml[head * a.splits + split] = make_float2(mm, ll);
        }
    }
}

// The same for a part of a pass: a warp's share of a row is formed once (in fs [warps][rows]), four columns at a time.
template <int W, typename Head>
__device__ __forceinline__ void merge_part(const DecodeArgs& a, Head head_of, int ng, int slot, const float* ms, const float* ls,
                                           const float* os, float* fs, int rows, int pitch) {
    for (int i = threadIdx.x; i < W * ng; i += W * 32) {
        const int w = i / ng, g = i - w * ng;
        float mm = -INFINITY;
#pragma unroll
        for (int v = 0; v < W; ++v) mm = fmaxf(mm, ms[v * rows + g]);
        fs[w * rows + g] = exp2f(ms[w * rows + g] - finite_max(mm));
        if (w == 0) {
            float ll = 0.0f;
#pragma unroll
            for (int v = 0; v < W; ++v) ll = fmaf(ls[v * rows + g], exp2f(ms[v * rows + g] - finite_max(mm)), ll);
            a.part_ml[head_of(g) * a.sh.slots + slot] = make_float2(mm, ll);
        }
    }
    __syncthreads();
    const int per = a.D / 4;
    for (int i = threadIdx.x; i < ng * per; i += W * 32) {
        const int g = i / per, d = (i - g * per) * 4;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float c = fs[w * rows + g];
            const float4 v = *reinterpret_cast<const float4*>(os + (w * rows + g) * pitch + d);
            o = make_float4(fmaf(v.x, c, o.x), fmaf(v.y, c, o.y), fmaf(v.z, c, o.z), fmaf(v.w, c, o.w));
        }
        *reinterpret_cast<float4*>(a.part_o + (head_of(g) * a.sh.slots + slot) * a.D + d) = o;
    }
}

// The two values as a 16-bit pair.
template <bool BF>
__device__ __forceinline__ uint32_t round2(float x, float y) {
    if (BF) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Parts of a sequence's shared tokens; the tcgen05 kernel's: 1 for any, whose number it leaves itself.
__device__ __forceinline__ int shared_parts(const DecodeArgs& a, int shared) {
    if (shared == 0 || a.prefix_parts == 0) return shared > 0;
    const int t = part_tokens(shared, a.prefix_parts);
    return (shared + t - 1) / t;
}

// The end of the last pass: the warps' (m, l, o) and the parts of the shared tokens, joined; o [warps][rows][pitch],
// then room for fs [warps][rows], [rows] 1 / l, [rows] where the parts are and their shares [rows][kMaxShared].  A
// thread's first part rows are on their way while half a warp per row forms the shares.
template <int KIND, int W, typename Head>
__device__ __forceinline__ void merge_last(const DecodeArgs& a, Head head_of, int ng, int shared, const float* ms, const float* ls,
                                           const float* os, float* fs, int rows, int pitch) {
    constexpr int U = 12;  // parts on their way together
    float* inv = fs + W * rows;
    int2* xs = reinterpret_cast<int2*>(inv + rows);
    float* share = inv + 3 * rows;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the shared tokens' parts are there
    const int some = shared_parts(a, shared);
    if ((int)threadIdx.x < ng) xs[threadIdx.x] = a.tc.first_o && some > 0 ? parts_behind(a.tc, (long long)head_of(threadIdx.x), some) : make_int2(0, 0);
    __syncthreads();
    const int per = a.D / 4;
    float4 v[U];
    auto load = [&](int i, int p0) {
        const int g = i / per, d = (i - g * per) * 4;
        const int2 x = xs[g];
        const size_t row = head_of(g);
#pragma unroll
        for (int p = 0; p < U; ++p)
            v[p] = p0 + p < some + x.x ? *reinterpret_cast<const float4*>(shared_o(a.sh, a.tc, row, x, p0 + p) + d) : make_float4(0, 0, 0, 0);
    };
    if ((int)threadIdx.x < ng * per) load(threadIdx.x, 0);
    const int l16 = threadIdx.x & 15;
    for (int g0 = 0; g0 < ng; g0 += W * 2) {
        const int g = g0 + (threadIdx.x >> 4);
        const bool have = g < ng;
        const int2 x = have ? xs[g] : make_int2(0, 0);
        const size_t row = have ? head_of(g) : 0;
        const int parts = have ? some + x.x : 0;
        const float2 none = make_float2(-INFINITY, 0.0f);
        const float2 own = have && l16 < W ? make_float2(ms[l16 * rows + g], ls[l16 * rows + g]) : none;
        float2 ml[2];  // the first 32 parts'
#pragma unroll
        for (int k = 0; k < 2; ++k) ml[k] = l16 + 16 * k < parts ? shared_ml(a.sh, a.tc, row, x, l16 + 16 * k) : none;
        float top = fmaxf(own.x, fmaxf(ml[0].x, ml[1].x));
        for (int p = l16 + 32; p < parts; p += 16) top = fmaxf(top, shared_ml(a.sh, a.tc, row, x, p).x);
#pragma unroll
        for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float base = finite_max(top);
        float l = 0.0f;
        if (have && l16 < W) {
            const float f = exp2f(own.x - base);
            fs[l16 * rows + g] = f;
            l = own.y * f;
        }
        for (int p = l16; p < parts; p += 16) {
            const float2 m = p == l16 ? ml[0] : p == l16 + 16 ? ml[1] : shared_ml(a.sh, a.tc, row, x, p);
            const float f = exp2f(m.x - base);
            share[g * kMaxShared + p] = f;
            l = fmaf(m.y, f, l);
        }
#pragma unroll
        for (int o = 8; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (have && l16 == 0) {
            inv[g] = l == 0.0f ? 0.0f : 1.0f / l;
            if (a.res.lse) a.res.lse[row] = l == 0.0f ? -INFINITY : (base + log2f(l)) * 0.693147180559945f;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < ng * per; i += W * 32) {
        const int g = i / per, d = (i - g * per) * 4, parts = some + xs[g].x;
        const size_t row = head_of(g);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](const float4& y, float c) {
            o = make_float4(fmaf(y.x, c, o.x), fmaf(y.y, c, o.y), fmaf(y.z, c, o.z), fmaf(y.w, c, o.w));
        };
        if (i != (int)threadIdx.x) load(i, 0);
#pragma unroll
        for (int w = 0; w < W; ++w) add(*reinterpret_cast<const float4*>(os + (w * rows + g) * pitch + d), fs[w * rows + g]);
        for (int p0 = 0; p0 < parts; p0 += U) {
            if (p0 > 0) load(i, p0);
#pragma unroll
            for (int p = 0; p < U; ++p)
                if (p0 + p < parts) add(v[p], share[g * kMaxShared + p0 + p]);
        }
        const float f = inv[g];
        o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
        if (KIND == KIND_F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(a.res.O) + row * a.D + d) = o;
        } else {
            *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.res.O) + (row * a.D + d) * 2) =
                make_uint2(round2<KIND == KIND_BF16>(o.x, o.y), round2<KIND == KIND_BF16>(o.z, o.w));
        }
    }
    if (a.res.err && blockIdx.x == 0 && threadIdx.x == 0) keep_error(a.res.err);
}

// ---------------------------------------------------------------------------
// The decode kernel: matrix instructions on tiles of 16 tokens
// ---------------------------------------------------------------------------
constexpr int kKeys = 16;  // tokens of a tile

template <int KIND>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (KIND == KIND_BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else if (KIND == KIND_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(addr)
                     : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// 16 bytes global -> shared, or zeros (nothing is read) where !real.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ float ex2(float t) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
    return y;
}
// The two values as 16-bit pair, and what the rounding left of them.
template <bool BF>
__device__ __forceinline__ uint32_t split2(float& x, float& y) {
    if (BF) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        const uint32_t u = *reinterpret_cast<const uint32_t*>(&v);
        x -= __uint_as_float(u << 16);
        y -= __uint_as_float(u & 0xFFFF0000u);
        return u;
    }
    const __half2 v = __floats2half2_rn(x, y);
    const float2 f = __half22float2(v);
    x -= f.x;
    y -= f.y;
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Shapes of the kernel: DP columns (dim_head rounded up), 8 NT query heads, W warps, ring slots of a warp,
// CTAs of an SM.  SHORT: for stretches of a few hundred tokens, whose begin and end take longer than their tokens: CTAs
// of half the warps and twice as many of them, so that some read while others begin or end.
template <int KIND_, int DP_, int NT_, bool SHORT = false>
struct Shape {
    static constexpr int KIND = KIND_, DP = DP_, NT = NT_;
    static constexpr int SIZE = KIND == KIND_F32 ? 4 : 2;
    static constexpr int ROW = DP * SIZE;             // bytes of a row in shared memory
    static constexpr int SLOT = kKeys * ROW;          // 16 rows of K or of V
    static constexpr int W = (ROW > 512 ? 4 : 8) / (SHORT ? 2 : 1);
    static constexpr int SLOTS = ROW > 128 ? 3 : 5;   // odd: K and V take the slots in turn
    static constexpr int CTAS = (ROW > 256 ? 1 : 2) * (SHORT ? 2 : 1);
    static constexpr bool QS = KIND == KIND_F32 || NT > 1;  // q in shared memory, else in registers
    static constexpr int QBYTES = !QS ? 0 : KIND == KIND_F32 ? DP / 8 * NT * 512 : DP / 16 * NT * 256;
    static constexpr int RING = W * SLOTS * SLOT;
    static constexpr int PITCH = DP + 4;
    static constexpr int MERGE = (int)sizeof(float) * W * 8 * NT * (2 + PITCH);
    static constexpr int SMEM = QBYTES + (RING > MERGE ? RING : MERGE);
};

// One CTA per (item, KV head, group of up to 8 NT query heads, part); every
// warp takes tiles of 16 tokens on its own.  K rows and V rows arrive in turn
// in the warp's ring by 16-byte asynchronous copies, SLOTS - 1 of them ahead;
// masked rows and the columns behind dim_head arrive as zeros.
//
// Scores: K (16 tokens x 16 or 8 columns per step) by q^T (8 heads); output:
// V^T (16 columns x 16 or 8 tokens) by P (8 heads).  The 16-byte chunks of a
// row are stored at other places of the row (swizzled by the row's number), so
// that what one matrix load or one 128-bit load of eight lanes touches lies in
// different banks.
//
// 16 bit: fragments by ldmatrix; P's fragment is the transpose of the scores'.
// P keeps 22 bits or more: it enters as a sum of 16-bit parts (three for bf16,
// two for fp16), one product each, which costs little here, since the kernel is
// bound by its reads.  fp32: tf32 products, each operand as its top
// 19 bits and the rest, three products (hi hi + lo hi + hi lo); the columns a
// lane needs for four steps are one 16-byte chunk, since the order in which a
// product sums its columns (or tokens) is free.
//
// A tile's products are summed by the matrix units from zero and then added to
// the running output: their sums cut instead of rounding, which over the
// thousands of tokens of a part would show (1.3e-6 against 5e-7).
//
// A row's maximum is raised only when a score exceeds it by more than 2^8
// (all types hold P then); fp16's P is kept 2^7 larger, away from the type's
// smallest numbers.
//
// For a batch that shares leading tokens (PASS) it differs in which rows and
// tokens a CTA has: own tokens begin behind the shared ones; a group's shared
// tokens take the rows (sequence, head) of all its sequences, 8 NT at a time,
// the row groups of one stretch of tokens side by side, so that the L2 cache
// serves all but the first.
template <typename S, int PASS>
__global__ void __launch_bounds__(S::W * 32, S::CTAS) paged_decode_kernel(const DecodeArgs a) {
    constexpr int KIND = S::KIND, DP = S::DP, NT = S::NT, W = S::W, SLOTS = S::SLOTS;
    constexpr bool F32 = KIND == KIND_F32, BF = KIND == KIND_BF16;
    constexpr int CH = S::ROW / 16;                       // 16-byte chunks of a row
    constexpr int LPR = CH < 32 ? CH : 32;                // lanes that copy a row
    constexpr int RPI = 32 / LPR, CPL = CH / LPR;         // rows per copy instruction, chunks of a lane
    constexpr int LEAD = (SLOTS - 1) / 2;                 // tiles that the copies are ahead
    constexpr int MT = DP / 16;                           // output tiles of 16 columns
    constexpr int PARTS = BF ? 3 : 2;
    constexpr float kLift = KIND == KIND_F16 ? 7.0f : 0.0f, kGrow = 8.0f;
    extern __shared__ __align__(128) uint8_t smem[];
    asm volatile("griddepcontrol.launch_dependents;");  // the join may be scheduled (it waits for this grid)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int D = a.D, chunks = D * S::SIZE / 16;

    long long id = blockIdx.x;
    int split, b, hk, h0, ng, first = 0, shared = 0;  // b: whose table row; first: the group's first sequence
    Visible vis;
    int chunk = a.chunk;
    bool rows_of_group = false;  // the CTA's rows are of a group's sequences, not of one
    int parts = a.splits;
    if (PASS == PASS_PARTS) {
        rows_of_group = id < a.shared_blocks;
        if (rows_of_group) parts = a.prefix_parts;
        else id -= a.shared_blocks;
    }
    if (PASS == PASS_PARTS && rows_of_group) {
        const int unit = (int)(id % a.units);
        id /= a.units;
        hk = (int)(id % a.HK);
        split = (int)(id / a.HK);
        // the group of this row group
        int g = -1, before = 0;
        for (int g0 = 0; g0 < a.sh.gr.n && g < 0; g0 += 32) {
            const int mine = g0 + lane < a.sh.gr.n ? (a.sh.gr.size(g0 + lane) * a.G + 8 * NT - 1) / (8 * NT) : 0;
            int sum = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += y;
            }
            const unsigned hits = __ballot_sync(0xffffffffu, unit < before + sum);
            if (hits) {
                const int l = __ffs(hits) - 1;
                g = g0 + l;
                before += __shfl_sync(0xffffffffu, sum - mine, l);
            } else {
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        vis.n = vis.nvis = g < 0 ? 0 : a.sh.gr.shared(a.c, g);
        vis.sinks = vis.gap = 0;
        first = g < 0 ? 0 : a.sh.gr.start(g);
        h0 = (unit - before) * 8 * NT;  // row of the group
        ng = g < 0 ? 0 : min(8 * NT, a.sh.gr.size(g) * a.G - h0);
        b = g < 0 ? 0 : leader_of(a.sh.gr, a.c, g, vis.n);
        chunk = part_tokens(vis.n, parts);
    } else {
        split = (int)(id % a.splits);
        id /= a.splits;
        const int grp = (int)(id % a.ngroups);
        id /= a.ngroups;
        hk = (int)(id % a.HK);
        b = (int)(id / a.HK);
        vis = visible(a, b);
        if (PASS != PASS_ALL) {
            shared = member_of(a.sh.gr, a.c, b, vis.n).tokens;
            vis.sinks = 0;
            vis.gap = shared;
            vis.nvis = vis.n - shared;
            chunk = PASS == PASS_LAST ? vis.nvis : part_tokens(vis.nvis, a.splits);
            if (PASS == PASS_PARTS && split == 0 && tid < min(8 * NT, a.G - grp * 8 * NT)) {
                a.sh.info[(size_t)b * a.H + hk * a.G + grp * 8 * NT + tid] =
                    make_int2((vis.nvis + chunk - 1) / chunk, shared_parts(a, shared));
            }
        }
        h0 = hk * a.G + grp * 8 * NT;
        ng = min(8 * NT, a.G - grp * 8 * NT);
    }
    const long long v_lo = (long long)split * chunk;
    if (PASS != PASS_LAST && (PASS != PASS_ALL || split > 0) && v_lo >= vis.nvis) {
        // the join takes the parts that hold tokens
        if (PASS != PASS_ALL) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const int v0 = (int)v_lo, v1 = (int)min((long long)vis.nvis, v_lo + chunk);
    // row i of the CTA: its query head among all sequences', and its query
    auto head_of = [&](int i) -> size_t {
        if (!(PASS == PASS_PARTS && rows_of_group)) return (size_t)b * a.H + h0 + i;
        const unsigned r = (unsigned)(h0 + i), s = r / (unsigned)a.G;
        return (size_t)(first + s) * a.H + hk * a.G + (r - s * a.G);
    };

    uint8_t* qsm = smem;
    const uint32_t ring = smem_u32(smem + S::QBYTES) + warp * SLOTS * S::SLOT;

    // the tile's tokens: lane i (and i + 16) has the row of token i
    const int ntiles = v1 > v0 ? (v1 - v0 + kKeys - 1) / kKeys : 0;
    auto row_of = [&](int tile) -> long long {
        const int v = v0 + tile * kKeys + (lane & 15);
        return tile < ntiles && v < v1 ? paged_offset(a.c, b, hk, vis.token(v)) : -1;
    };
    const int clane = lane % LPR, crow = lane / LPR;
    auto fetch = [&](const uint8_t* base, bool isv, int slot, long long off) {
#pragma unroll
        for (int i = 0; i < kKeys / RPI; ++i) {
            const int r = i * RPI + crow;
            const long long o = __shfl_sync(0xffffffffu, off, r);
            const int swz = !F32 || isv ? r & 7 : (r & 1) << 2;
#pragma unroll
            for (int c0 = 0; c0 < CPL; ++c0) {
                const int c = c0 * LPR + clane;
                const bool real = o >= 0 && c < chunks;
                copy16(ring + slot * S::SLOT + r * S::ROW + ((c ^ swz) << 4), real ? base + o + c * 16 : a.Q, real);
            }
        }
    };
    // copies are numbered K0 V0 K1 V1 ...: number f is in slot f % SLOTS
    long long off_next = row_of(warp), off = -1;
    uint32_t real[LEAD];  // which tokens there are, of this tile and the next
#pragma unroll
    for (int i = 0; i < LEAD; ++i) {
        const int tile = warp + i * W;
        off = off_next;
        off_next = row_of(tile + W);
        real[i] = __ballot_sync(0xffffffffu, off >= 0);
        if (tile < ntiles) fetch(a.c.K, false, 2 * i, off);
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (tile < ntiles) fetch(a.c.V, true, 2 * i + 1, off);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // q^T fragments
    const uint8_t* qb = a.Q + (size_t)b * a.q_stride;
    auto query_of = [&](int i) -> const uint8_t* {
        if (!(PASS == PASS_PARTS && rows_of_group)) return qb + (size_t)(h0 + i) * D * S::SIZE;
        const unsigned r = (unsigned)(h0 + i), s = r / (unsigned)a.G;
        return a.Q + (size_t)(first + s) * a.q_stride + (size_t)(hk * a.G + (r - s * a.G)) * D * S::SIZE;
    };
    uint32_t q[S::QS ? 1 : NT][S::QS ? 1 : DP / 16][2];
    if (F32) {
        // step (blk, e): columns 32 blk + 4 t + e and 16 further of head g, as hi, hi, lo, lo
        for (int i = warp; i < DP / 8 * NT; i += W) {
            const int n = i / (DP / 8), st = i % (DP / 8), d = (st >> 2) * 32 + 4 * t + (st & 3);
            const bool have = n * 8 + g < ng;
            const float* row = reinterpret_cast<const float*>(query_of(n * 8 + g));
            const uint32_t b0 = have && d < D ? __float_as_uint(__ldg(row + d)) : 0u;
            const uint32_t b1 = have && d + 16 < D ? __float_as_uint(__ldg(row + d + 16)) : 0u;
            uint4 f;
            tf32_split(b0, f.x, f.z);
            tf32_split(b1, f.y, f.w);
            reinterpret_cast<uint4*>(qsm)[i * 32 + lane] = f;
        }
        __syncthreads();
    } else {
        // step k: columns 16 k + 2 t, 2 t + 1 (and + 8) of head g
        auto frag = [&](int n, int k, int e) {
            const int d = k * 16 + e * 8 + 2 * t;
            return n * 8 + g < ng && d < D
                       ? __ldg(reinterpret_cast<const uint32_t*>(query_of(n * 8 + g) + d * 2))
                       : 0u;
        };
        if (S::QS) {
            for (int i = warp; i < DP / 16 * NT; i += W)
                reinterpret_cast<uint2*>(qsm)[i * 32 + lane] = make_uint2(frag(i % NT, i / NT, 0), frag(i % NT, i / NT, 1));
            __syncthreads();
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < DP / 16; ++k) {
                    q[S::QS ? 0 : n][S::QS ? 0 : k][0] = frag(n, k, 0);
                    q[S::QS ? 0 : n][S::QS ? 0 : k][1] = frag(n, k, 1);
                }
        }
    }
    float m[NT][2], l[NT][2], o[NT][MT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int k = 0; k < MT; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][k][e] = 0.0f;
    }

    int slot = 0;  // of this tile's K; its V is in the next
    auto after = [&](int s, int k) { return s + k >= SLOTS ? s + k - SLOTS : s + k; };
    for (int tile = warp; tile < ntiles; tile += W) {
        asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 2) : "memory");
        __syncwarp();
        const uint32_t here = real[0];
#pragma unroll
        for (int i = 0; i + 1 < LEAD; ++i) real[i] = real[i + 1];
        const bool more = tile + LEAD * W < ntiles;
        off = off_next;
        off_next = row_of(tile + (LEAD + 1) * W);
        real[LEAD - 1] = __ballot_sync(0xffffffffu, off >= 0);
        if (more) fetch(a.c.K, false, after(slot, SLOTS - 1), off);
        asm volatile("cp.async.commit_group;" ::: "memory");

        const uint32_t kb = ring + slot * S::SLOT;
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
        if (F32) {
#pragma unroll
            for (int blk = 0; blk < DP / 32; ++blk) {
                // rows g and g + 8 (one parity), chunks t and t + 4 of the 32 columns
                const int c = blk * 8 + t, swz = (g & 1) << 2;
                const uint4 x0 = lds16(kb + g * S::ROW + ((c ^ swz) << 4)), x1 = lds16(kb + (g + 8) * S::ROW + ((c ^ swz) << 4));
                const uint4 x2 = lds16(kb + g * S::ROW + (((c + 4) ^ swz) << 4)),
                            x3 = lds16(kb + (g + 8) * S::ROW + (((c + 4) ^ swz) << 4));
                const uint32_t k0[4] = {x0.x, x0.y, x0.z, x0.w}, k1[4] = {x1.x, x1.y, x1.z, x1.w};
                const uint32_t k2[4] = {x2.x, x2.y, x2.z, x2.w}, k3[4] = {x3.x, x3.y, x3.z, x3.w};
                float part[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) part[n][e] = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t hi[4], lo[4];
                    tf32_split(k0[e], hi[0], lo[0]);
                    tf32_split(k1[e], hi[1], lo[1]);
                    tf32_split(k2[e], hi[2], lo[2]);
                    tf32_split(k3[e], hi[3], lo[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint4 qq = reinterpret_cast<const uint4*>(qsm)[(n * (DP / 8) + blk * 4 + e) * 32 + lane];
                        mma16<KIND>(part[n], hi, qq.z, qq.w);
                        mma16<KIND>(part[n], lo, qq.x, qq.y);
                        mma16<KIND>(part[n], hi, qq.x, qq.y);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] += part[n][e];
            }
        } else {
            const int kr = lane & 15, kc = lane >> 4;  // lane i addresses row i % 8 of block i / 8: rows, then column halves
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
                uint32_t f[4];
                ldmatrix4<false>(f, kb + kr * S::ROW + (((2 * k + kc) ^ (kr & 7)) << 4));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (S::QS) {
                        const uint2 qq = reinterpret_cast<const uint2*>(qsm)[(k * NT + n) * 32 + lane];
                        mma16<KIND>(s[n], f, qq.x, qq.y);
                    } else {
                        mma16<KIND>(s[n], f, q[S::QS ? 0 : n][S::QS ? 0 : k][0], q[S::QS ? 0 : n][S::QS ? 0 : k][1]);
                    }
                }
            }
        }
        // scores of tokens g and g + 8, heads 2 t and 2 t + 1
        const bool r0 = (here >> g) & 1, r1 = (here >> (g + 8)) & 1;
        bool need = false;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            s[n][0] = r0 ? s[n][0] * a.scale2 : -INFINITY;
            s[n][1] = r0 ? s[n][1] * a.scale2 : -INFINITY;
            s[n][2] = r1 ? s[n][2] * a.scale2 : -INFINITY;
            s[n][3] = r1 ? s[n][3] * a.scale2 : -INFINITY;
            need |= fmaxf(s[n][0], s[n][2]) > m[n][0] + kGrow || fmaxf(s[n][1], s[n][3]) > m[n][1] + kGrow;
            if (PASS == PASS_ALL && a.scores) {
                const int v = v0 + tile * kKeys + g;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int h = n * 8 + 2 * t + (e & 1), ve = v + (e >> 1) * 8;
                    if (h < ng && ve < v1) a.scores[((size_t)b * a.H + h0 + h) * a.vmax + ve] = s[n][e];
                }
            }
        }
        if (__any_sync(0xffffffffu, need)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
                    x = fmaxf(m[n][e], x);
                    const float corr = ex2(m[n][e] - finite_max(x));
                    m[n][e] = x;
                    l[n][e] *= corr;
#pragma unroll
                    for (int k = 0; k < MT; ++k) {
                        o[n][k][e] *= corr;
                        o[n][k][e + 2] *= corr;
                    }
                }
        }
        // P's fragments: 16 bit [part][tokens 0-7, 8-15], fp32 [tokens 0-7, 8-15][token 2 t, 2 t + 1]
        uint32_t p[NT][F32 ? 2 : PARTS][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float m0 = finite_max(m[n][0]) - kLift, m1 = finite_max(m[n][1]) - kLift;
            float x[4] = {ex2(s[n][0] - m0), ex2(s[n][1] - m1), ex2(s[n][2] - m0), ex2(s[n][3] - m1)};
            l[n][0] += x[0] + x[2];
            l[n][1] += x[1] + x[3];
            if (F32) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int from = (2 * t + e) * 4 + (g >> 1);  // the lane with token 2 t + e, head g
                        const float y0 = __shfl_sync(0xffffffffu, x[2 * h], from), y1 = __shfl_sync(0xffffffffu, x[2 * h + 1], from);
                        p[n][h][e] = __float_as_uint((g & 1) ? y1 : y0);
                    }
            } else {
#pragma unroll
                for (int i = 0; i < PARTS; ++i) {
                    p[n][i][0] = transpose8x8(split2<BF>(x[0], x[1]));
                    p[n][i][1] = transpose8x8(split2<BF>(x[2], x[3]));
                }
            }
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 2) : "memory");
        __syncwarp();
        if (more) fetch(a.c.V, true, slot, off);
        asm volatile("cp.async.commit_group;" ::: "memory");

        const uint32_t vb = ring + after(slot, 1) * S::SLOT;
        if (F32) {
            // output tile 2 j + h: rows g and g + 8 are columns 4 (g + 8 j) + 2 h and + 1
            uint32_t ph[NT][2][2], pl[NT][2][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) tf32_split(p[n][i >> 1][i & 1], ph[n][i >> 1][i & 1], pl[n][i >> 1][i & 1]);
#pragma unroll
            for (int j = 0; j < DP / 32; ++j) {
                float part[NT][2][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 8; ++e) part[n][e >> 2][e & 3] = 0.0f;
#pragma unroll
                for (int h8 = 0; h8 < 2; ++h8) {
                    const int row0 = h8 * 8 + 2 * t, c = g + 8 * j;  // this lane's tokens: row0, row0 + 1
                    const uint4 u = lds16(vb + row0 * S::ROW + ((c ^ (row0 & 7)) << 4));
                    const uint4 w = lds16(vb + (row0 + 1) * S::ROW + ((c ^ ((row0 + 1) & 7)) << 4));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t hi[4], lo[4];
                        tf32_split(h ? u.z : u.x, hi[0], lo[0]);
                        tf32_split(h ? u.w : u.y, hi[1], lo[1]);
                        tf32_split(h ? w.z : w.x, hi[2], lo[2]);
                        tf32_split(h ? w.w : w.y, hi[3], lo[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma16<KIND>(part[n][h], hi, pl[n][h8][0], pl[n][h8][1]);
                            mma16<KIND>(part[n][h], lo, ph[n][h8][0], ph[n][h8][1]);
                            mma16<KIND>(part[n][h], hi, ph[n][h8][0], ph[n][h8][1]);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[n][2 * j + (e >> 2)][e & 3] += part[n][e >> 2][e & 3];
            }
        } else {
            const int vr = (lane & 7) + ((lane >> 4) << 3), vc = (lane >> 3) & 1;  // blocks: column halves first, then rows
#pragma unroll
            for (int k = 0; k < MT; ++k) {
                uint32_t f[4];
                ldmatrix4<true>(f, vb + vr * S::ROW + (((2 * k + vc) ^ (vr & 7)) << 4));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = PARTS - 1; i >= 0; --i) mma16<KIND>(part, f, p[n][F32 ? 0 : i][0], p[n][F32 ? 0 : i][1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][k][e] += part[e];
                }
            }
        }
        slot = after(slot, 2);
    }
    // the warps' (m, l, o) meet in shared memory, over the ring
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    float* ms = reinterpret_cast<float*>(smem + S::QBYTES);  // [warps][8 NT]
    float* ls = ms + W * 8 * NT;
    float* os = ls + W * 8 * NT;                             // [warps][8 NT][PITCH]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float x = l[n][e];
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
            const int h = warp * 8 * NT + n * 8 + 2 * t + e;
            if (g == 0) {
                ms[h] = m[n][e] - kLift;
                ls[h] = x;
            }
#pragma unroll
            for (int k = 0; k < MT; ++k) {
                const int d0 = F32 ? 4 * (g + 8 * (k >> 1)) + 2 * (k & 1) : k * 16 + g, d1 = F32 ? d0 + 1 : d0 + 8;
                os[h * S::PITCH + d0] = o[n][k][e];
                os[h * S::PITCH + d1] = o[n][k][e + 2];
            }
        }
    __syncthreads();
    if constexpr (PASS == PASS_ALL) {
        merge_warps<W>(a, (size_t)b * a.H + h0, ng, split, ms, ls, os, 8 * NT, S::PITCH);
    } else if constexpr (PASS == PASS_LAST) {
        static_assert(S::MERGE + (W + 3 + kMaxShared) * 8 * NT * 4 <= S::RING, "the shares lie in the ring too");
        merge_last<KIND, W>(a, head_of, ng, shared, ms, ls, os, os + W * 8 * NT * S::PITCH, 8 * NT, S::PITCH);
    } else {
        merge_part<W>(a, head_of, ng, rows_of_group ? a.sh.own + split : split, ms, ls, os, os + W * 8 * NT * S::PITCH, 8 * NT, S::PITCH);
        asm volatile("griddepcontrol.wait;" ::: "memory");
    }
}

// m and l of all parts of a head (one warp): the same order whatever the grid.
__device__ __forceinline__ float2 join_ml(const float2* ml, int parts, int lane) {
    float m = -INFINITY;
    for (int s = lane; s < parts; s += 32) m = fmaxf(m, ml[s].x);
    m = finite_max(warp_max(m));
    float l = 0.0f;
    for (int s = lane; s < parts; s += 32) {
        const float2 x = ml[s];
        l = fmaf(x.y, exp2f(x.x - m), l);
    }
    return make_float2(m, warp_sum(l));
}

constexpr int kJoinTokens = 512;  // tokens whose weights one CTA of the join adds

// Joins the parts.  The first o_blocks CTAs take one query head each; the
// others add the weights of a stretch of tokens of one KV head.  Launched
// while the parts are still being made: what they do not write is read before
// the wait.
__global__ void __launch_bounds__(128) paged_join_kernel(const DecodeArgs a) {
    extern __shared__ __align__(16) float sm[];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long long id = blockIdx.x;
    if (id < a.o_blocks) {
        const int b = (int)(id / a.H);
        const int nvis = visible(a, b).nvis;
        const int parts = max(1, (nvis + a.chunk - 1) / a.chunk);
        const float2* ml = a.part_ml + id * a.splits;
        const float* po = a.part_o + (size_t)id * a.splits * a.D;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        float x[kJoinAhead];
#pragma unroll
        for (int s = 0; s < kJoinAhead; ++s) x[s] = s < parts && tid < a.D ? po[(size_t)s * a.D + tid] : 0.0f;
        if (warp == 0) {
            const float2 j = join_ml(ml, parts, lane);
            const float inv = j.y == 0.0f ? 0.0f : 1.0f / j.y;
            for (int s = lane; s < parts; s += 32) sm[s] = exp2f(ml[s].x - j.x) * inv;
            if (lane == 0 && a.lse) a.lse[id] = j.y == 0.0f ? -INFINITY : (j.x + log2f(j.y)) * 0.693147180559945f;
        }
        __syncthreads();
        for (int d = tid; d < a.D; d += 128) {
            float o = 0.0f;
#pragma unroll
            for (int s = 0; s < kJoinAhead; ++s)
                if (s < parts) o = fmaf(d == tid ? x[s] : po[(size_t)s * a.D + d], sm[s], o);
#pragma unroll 8
            for (int s = kJoinAhead; s < parts; ++s) o = fmaf(po[(size_t)s * a.D + d], sm[s], o);
            a.O[id * a.D + d] = o;
        }
        return;
    }
    id -= a.o_blocks;
    const int blk = (int)(id % a.w_blocks);
    id /= a.w_blocks;
    const int hk = (int)(id % a.HK), b = (int)(id / a.HK);
    const Visible vis = visible(a, b);
    const int parts = max(1, (vis.nvis + a.chunk - 1) / a.chunk);
    const int v0 = blk * kJoinTokens, v1 = min(vis.nvis, v0 + kJoinTokens);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (v0 >= vis.nvis) return;
    float2* st = reinterpret_cast<float2*>(sm);  // [G] (m, 1 / l)
    for (int g = warp; g < a.G; g += 4) {
        const float2 j = join_ml(a.part_ml + ((size_t)b * a.H + hk * a.G + g) * a.splits, parts, lane);
        if (lane == 0) st[g] = make_float2(j.x, j.y == 0.0f ? 0.0f : 1.0f / j.y);
    }
    __syncthreads();
    const float* x = a.scores + ((size_t)b * a.H + hk * a.G) * a.vmax + v0;
    float* w = a.weights + ((size_t)b * a.HK + hk) * a.weight_stride;
    constexpr int U = kJoinTokens / 128;  // tokens of a thread, all on their way together
    float old[U], sum[U];
    int t[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int v = v0 + tid + u * 128;
        t[u] = v < v1 ? vis.token(v) : -1;
        old[u] = t[u] >= 0 ? w[t[u]] : 0.0f;
        sum[u] = 0.0f;
    }
    for (int g = 0; g < a.G; ++g) {
        const float2 j = st[g];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (t[u] >= 0) sum[u] = fmaf(exp2f(x[(size_t)g * a.vmax + tid + u * 128] - j.x), j.y, sum[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (t[u] >= 0) w[t[u]] = old[u] + sum[u];
}

struct DecodePlan {
    int gt, ngroups, splits, chunk, vmax;
    size_t off_ml, off_o, off_scores, bytes;
};

// Query heads of a KV head that one CTA takes: 16 where more than 8 share a KV head of 16-bit rows of at
// most 128 columns, else 8 (more would not fit in registers).
int head_group(int dtype, int G, int D) { return dtype != RKV_F32 && G > 8 && D <= 128 ? 16 : 8; }
// CTAs that run at a time (Shape::CTAS of an SM).
int decode_slots(int dtype, int D) {
    const int row = (D <= 64 ? 64 : D <= 128 ? 128 : 256) * (dtype == RKV_F32 ? 4 : 2);
    return kSms * (row > 256 ? 1 : 2);
}
long long decode_units(int dtype, int H, int HK, int D, int batch) {
    const int G = H / HK, gt = head_group(dtype, G, D);
    return (long long)batch * HK * ((G + gt - 1) / gt);
}
// The most parts that decode_parts gives up to visible_max, which it grows with.
long long decode_parts_bound(int dtype, int H, int HK, int D, long long visible_max, int batch) {
    const long long units = decode_units(dtype, H, HK, D, batch);
    const long long slots = decode_slots(dtype, D);
    long long p = units > 0 ? kMaxWaves * slots / units : 1;
    const long long most = (visible_max + kMinChunk - 1) / kMinChunk;
    if (p > most) p = most;
    if (p > kMaxSplits) p = kMaxSplits;
    return p < 1 ? 1 : p;
}
// Parts of the visible tokens.  With w waves of CTAs as full as they get, a
// wave takes the time of a part and of about kStartTokens tokens more (start,
// first reads, join); the w with the least time in all.  Measured: 16 x 3717
// tokens with weights in 2 / 4 / 6 / 9 / 10 parts (0.9 / 1.7 / 2.6 / 3.9 / 4.3
// waves) 50 / 54 / 56 / 59 / 62 us; 8 x 131072 in 4 / 9 / 19 / 23 parts (0.9 /
// 1.9 / 4.1 / 5.0 waves) 686 / 650 / 705 / 654 us.  (One wave with equal
// stretches of all sequences' tokens, balanced on the device, was slower: 64
// ragged sequences 247 us against 198; the SMs do not stream at one rate.)
long long decode_parts(int dtype, int H, int HK, int D, long long visible_max, int batch) {
    const long long units = decode_units(dtype, H, HK, D, batch), bound = decode_parts_bound(dtype, H, HK, D, visible_max, batch);
    const long long slots = decode_slots(dtype, D);
    long long best = 1, best_cost = -1;
    for (int w = 0; w <= kMaxWaves; ++w) {
        long long p = w == 0 || units == 0 ? 1 : w * slots / units;
        if (p < 1) p = 1;
        if (p > bound) p = bound;
        const long long cost = ((units * p + slots - 1) / slots) * (kStartTokens + (visible_max + p - 1) / p);
        if (best_cost < 0 || cost < best_cost) best = p, best_cost = cost;
    }
    return best;
}

DecodePlan decode_plan(int dtype, int H, int HK, int D, long long visible_max, int max_len, int batch, bool weights) {
    DecodePlan p{};
    const int G = H / HK;
    p.gt = head_group(dtype, G, D);
    p.ngroups = (G + p.gt - 1) / p.gt;
    const long long parts = decode_parts(dtype, H, HK, D, visible_max, batch);
    long long chunk = (visible_max + parts - 1) / parts;
    chunk = (chunk + kTile - 1) / kTile * kTile;
    if (chunk < kTile) chunk = kTile;
    p.chunk = (int)chunk;
    const long long splits = (visible_max + chunk - 1) / chunk;
    p.splits = splits < 1 ? 1 : (int)splits;
    p.vmax = (max_len + 3) / 4 * 4;
    // the bound, not the parts, gives the layout: it grows with visible_max, so the workspace of max_len
    // serves every window
    const size_t heads = (size_t)batch * H, bound = (size_t)decode_parts_bound(dtype, H, HK, D, visible_max, batch);
    size_t off = kWorkspaceHeader;
    p.off_ml = off;
    off = align_up(off + heads * bound * sizeof(float2), kWorkspaceAlign);
    p.off_o = off;
    if (bound > 1) off = align_up(off + heads * bound * D * sizeof(float), kWorkspaceAlign);
    p.off_scores = off;
    if (weights) off = align_up(off + heads * (size_t)p.vmax * sizeof(float), kWorkspaceAlign);
    p.bytes = off;
    return p;
}

template <int KIND, int DP, int NT, int PASS>
int launch_shape(const DecodeArgs& a, long long blocks, bool dependent, cudaStream_t st) {
    using S = Shape<KIND, DP, NT, PASS != PASS_ALL && NT < 4>;
    static_assert(S::SMEM * S::CTAS + 1024 * S::CTAS <= 228 * 1024, "the CTAs of an SM fit in its shared memory");
    if (cudaFuncSetAttribute(paged_decode_kernel<S, PASS>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM) != cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    if (PASS != PASS_ALL && dependent) {
        const cudaError_t e = launch_pdl(paged_decode_kernel<S, PASS>, dim3((unsigned)blocks), dim3(S::W * 32), S::SMEM, st, a);
        if (e != cudaSuccess) (void)cudaGetLastError();
        return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
    }
    paged_decode_kernel<S, PASS><<<(unsigned)blocks, S::W * 32, S::SMEM, st>>>(a);
    return launched();
}
template <int KIND, int PASS>
int launch_kind(const DecodeArgs& a, int gt, long long blocks, bool dependent, cudaStream_t st) {
    if constexpr (KIND != KIND_F32) {
        if (gt == 16)
            return a.D <= 64 ? launch_shape<KIND, 64, 2, PASS>(a, blocks, dependent, st) : launch_shape<KIND, 128, 2, PASS>(a, blocks, dependent, st);
    } else if constexpr (PASS == PASS_PARTS) {
        if (gt == 32)
            return launch_shape<KIND, 128, 4, PASS>(a, blocks, dependent, st);
    }
    if (a.D <= 64) return launch_shape<KIND, 64, 1, PASS>(a, blocks, dependent, st);
    if (a.D <= 128) return launch_shape<KIND, 128, 1, PASS>(a, blocks, dependent, st);
    return launch_shape<KIND, 256, 1, PASS>(a, blocks, dependent, st);
}
template <int PASS>
int launch_pass(const DecodeArgs& a, int dtype, int gt, long long blocks, bool dependent, cudaStream_t st) {
    if (blocks > 0x7FFFFFFFLL) return RKV_ERR_UNSUPPORTED;
    switch (dtype) {
        case RKV_F32: return launch_kind<KIND_F32, PASS>(a, gt, blocks, dependent, st);
        case RKV_BF16: return launch_kind<KIND_BF16, PASS>(a, gt, blocks, dependent, st);
        default: return launch_kind<KIND_F16, PASS>(a, gt, blocks, dependent, st);
    }
}
}  // namespace
// Rows of a group that one CTA takes: as many as a group of mean size has, up to what fits in the registers.  fp32's
// operands are split once for all of them: 20 sequences behind 56208 tokens, 24/8 heads of 128, 395 us with 32 rows and
// 503 with 8; with 64 columns 42 and 36, with 256 columns there is room for 8 alone.
int shared_rows(int dtype, int D, int H, int HK, int batch, int groups) {
    const long long rows = ((long long)batch * (H / HK) + groups - 1) / groups;
    if (dtype == RKV_F32) return rows > 16 && D > 64 && D <= 128 ? 32 : 8;
    return head_group(dtype, rows > 8 ? 9 : 1, D);
}
namespace {
long long shared_units(int rows, int H, int HK, int batch, int groups) { return groups + (long long)batch * (H / HK) / rows; }

}  // namespace

// How many own tokens there are is known on the device alone, and they are few beside the shared ones as a rule;
// sequences with few leave their CTAs behind the first without work, so that these are one wave at most, but for
// kOwnMost tokens of max_len each: one of 64 sequences with 65536 own tokens (8 KV heads of 128, bf16) would take one CTA
// 1745 us.  Where nothing is shared, as many as the decode of all tokens takes.
constexpr int kOwnMost = 12288;
int shared_own_parts(int dtype, int H, int HK, int D, int max_len, int batch, int groups) {
    const long long units = decode_units(dtype, H, HK, D, batch), most = ((long long)max_len + kPartLeast - 1) / kPartLeast;
    long long p = units > 0 ? 2 * decode_slots(dtype, D) / units : 1;
    const long long many = ((long long)max_len + kOwnMost - 1) / kOwnMost;
    if (p < many) p = many < 64 ? many : 64;  // the workspace holds them all
    if (groups == 0) p = decode_parts(dtype, H, HK, D, max_len, batch);
    if (p > most) p = most;
    if (p > kMaxSplits) p = kMaxSplits;
    return p < 1 ? 1 : (int)p;
}
// As many as give two waves of CTAs, each of 128 tokens or more.
int shared_prefix_parts(int dtype, int H, int HK, int D, int max_len, int batch, int groups) {
    const int rows = shared_rows(dtype, D, H, HK, batch, groups);
    const long long each = ((long long)batch * (H / HK) + groups * (long long)rows - 1) / (groups * (long long)rows);  // of a group of mean size
    long long p = 2LL * 2 * decode_slots(dtype, D) / (each * groups * HK);
    const long long most = ((long long)max_len + kPartLeast - 1) / kPartLeast;
    if (p > most) p = most;
    if (p > 128) p = 128;  // of kMaxShared
    return p < 1 ? 1 : (int)p;
}
int launch_shared_pass(const SharedArgs& s, SharedPass pass, const TcParts& t, const Result& r, bool dependent, cudaStream_t st) {
    DecodeArgs a{};
    a.c = s.c;
    a.Q = s.Q;
    a.q_stride = s.q_stride;
    a.H = s.H;
    a.HK = s.HK;
    a.G = s.H / s.HK;
    a.D = s.D;
    a.max_len = s.gr.max_len;
    a.scale2 = 1.4426950408889634f / sqrtf((float)s.D);
    a.part_o = s.part_o;
    a.part_ml = s.part_ml;
    a.sh = s;
    a.tc = t;
    a.res = r;
    a.prefix_parts = s.slots - s.own;
    const bool shared = pass == SHARED_TOKENS || pass == ALL_TOKENS, own = pass != SHARED_TOKENS;
    int gt = 8;
    if (own) gt = head_group(s.dtype, a.G, s.D);
    if (shared) {
        const int rows = shared_rows(s.dtype, s.D, s.H, s.HK, s.batch, s.gr.n);
        if (rows > gt) gt = rows;
        const long long units = shared_units(gt, s.H, s.HK, s.batch, s.gr.n), blocks = units * s.HK * a.prefix_parts;
        if (blocks > 0x3FFFFFFF) return RKV_ERR_UNSUPPORTED;
        a.units = (int)units;
        a.shared_blocks = (int)blocks;
    }
    a.ngroups = (a.G + gt - 1) / gt;
    a.splits = pass == OWN_AND_JOIN ? 1 : s.own;
    const long long blocks = a.shared_blocks + (own ? (long long)s.batch * s.HK * a.ngroups * a.splits : 0);
    return pass == OWN_AND_JOIN ? launch_pass<PASS_LAST>(a, s.dtype, gt, blocks, dependent, st)
                                : launch_pass<PASS_PARTS>(a, s.dtype, gt, blocks, dependent, st);
}

}  // namespace rkv

using namespace rkv;

extern "C" int rkv_paged_append(const rkv_paged_cache* cache, const void* k, const void* v, int n_rows, int batch,
                                long long src_item_stride, long long src_token_stride, long long src_head_stride,
                                const int* n_new, void* stream) {
    const int rc = paged_check(cache, true, batch);
    if (rc) return rc;
    if (n_rows < 0 || batch < 0) return RKV_ERR_INVALID_ARG;
    if (n_rows == 0 || batch == 0 || cache->num_pages == 0 || cache->table_stride == 0) return RKV_OK;
    if (batch > 65535) return RKV_ERR_UNSUPPORTED;
    const int es = elem_size(cache->dtype);
    const long long rowb = (long long)cache->dim_head * es;
    if (!k || !v || src_item_stride < 0 || src_token_stride < 0 || src_head_stride < 0) return RKV_ERR_INVALID_ARG;
    uintptr_t al = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | (uintptr_t)rowb;
    if (batch > 1) al |= (uintptr_t)src_item_stride;
    if (n_rows > 1) al |= (uintptr_t)src_token_stride;
    if (cache->num_heads_kv > 1) al |= (uintptr_t)src_head_stride;
    if (al & (es - 1)) return RKV_ERR_INVALID_ARG;
    const int vb = (al & 15) == 0 ? 16 : (al & 7) == 0 ? 8 : (al & 3) == 0 ? 4 : 2;
    AppendArgs a{};
    a.c = paged_view(*cache);
    a.k = static_cast<const uint8_t*>(k);
    a.v = static_cast<const uint8_t*>(v);
    a.n_new = n_new;
    a.item_stride = src_item_stride;
    a.src_token = src_token_stride;
    a.src_head = src_head_stride;
    a.n_rows = n_rows;
    a.HK = cache->num_heads_kv;
    a.vpr = (int)(rowb / vb);
    if ((long long)a.HK * a.vpr > 0x7FFFFFFFLL) return RKV_ERR_UNSUPPORTED;
    const long long total = (long long)n_rows * a.HK * a.vpr;
    long long gx = (total + 256 * kAppendVecs - 1) / (256 * kAppendVecs);
    const long long most = 148 * 16 / batch + 1;
    if (gx > most) gx = most;
    const dim3 grid((unsigned)gx, batch);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (vb) {
        case 16: paged_append_kernel<uint4><<<grid, 256, 0, st>>>(a); break;
        case 8: paged_append_kernel<uint2><<<grid, 256, 0, st>>>(a); break;
        case 4: paged_append_kernel<uint32_t><<<grid, 256, 0, st>>>(a); break;
        default: paged_append_kernel<uint16_t><<<grid, 256, 0, st>>>(a); break;
    }
    return launched();
}

static int decode_shape_check(int H, int HK, int D, int max_len, int batch) {
    if (H <= 0 || HK <= 0 || H % HK != 0 || D <= 0 || max_len < 0 || batch < 0) return RKV_ERR_INVALID_ARG;
    if (D % 8 != 0 || D > 256) return RKV_ERR_UNSUPPORTED;
    if (H / HK > 1024 || max_len > kMaxLen) return RKV_ERR_UNSUPPORTED;
    return RKV_OK;
}

extern "C" int rkv_paged_decode_workspace_size(int num_heads, int num_heads_kv, int dim_head, int max_len, int batch,
                                               int with_weights, size_t* bytes) {
    const int rc = decode_shape_check(num_heads, num_heads_kv, dim_head, max_len, batch);
    if (rc || !bytes) return rc ? rc : (int)RKV_ERR_INVALID_ARG;
    *bytes = 0;  // the largest over the types
    for (int dtype : {RKV_F32, RKV_BF16}) {
        const size_t n = decode_plan(dtype, num_heads, num_heads_kv, dim_head, max_len, max_len, batch, with_weights != 0).bytes;
        if (n > *bytes) *bytes = n;
    }
    return RKV_OK;
}

extern "C" int rkv_paged_decode(const void* Q, long long q_item_stride, int num_heads, const rkv_paged_cache* cache,
                                int max_len, int batch, int sinks, int window, float* O, float* lse, float* weights,
                                int weight_stride, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = paged_check(cache, true, batch);
    if (!rc) rc = decode_shape_check(num_heads, cache->num_heads_kv, cache->dim_head, max_len, batch);
    if (rc) return rc;
    if (sinks < 0 || window < 0) return RKV_ERR_INVALID_ARG;
    if (batch == 0) return RKV_OK;
    const int D = cache->dim_head;
    const long long q_bytes = (long long)num_heads * D * elem_size(cache->dtype);
    if (!Q || !O || (reinterpret_cast<uintptr_t>(Q) & 15)) return RKV_ERR_INVALID_ARG;
    if (batch > 1 && (q_item_stride < q_bytes || (q_item_stride & 15))) return RKV_ERR_INVALID_ARG;
    if (weights && weight_stride < max_len) return RKV_ERR_INVALID_ARG;
    long long vis = max_len;
    if (window > 0 && (long long)sinks + window < vis) vis = (long long)sinks + window;
    const DecodePlan p = decode_plan(cache->dtype, num_heads, cache->num_heads_kv, D, vis, max_len, batch, weights != nullptr);
    if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < p.bytes) return RKV_ERR_WORKSPACE;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    DecodeArgs a{};
    a.c = paged_view(*cache);
    a.Q = static_cast<const uint8_t*>(Q);
    a.q_stride = q_item_stride;
    a.H = num_heads;
    a.HK = cache->num_heads_kv;
    a.G = num_heads / cache->num_heads_kv;
    a.D = D;
    a.max_len = max_len;
    a.sinks = sinks;
    a.window = window;
    a.ngroups = p.ngroups;
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.vmax = p.vmax;
    a.scale2 = 1.4426950408889634f / sqrtf((float)D);
    a.O = O;
    a.lse = lse;
    a.weights = weights;
    a.weight_stride = weight_stride;
    const bool join = p.splits > 1 || weights;
    if (join) {
        a.part_ml = reinterpret_cast<float2*>(ws + p.off_ml);
        a.part_o = reinterpret_cast<float*>(ws + p.off_o);
    }
    if (weights) a.scores = reinterpret_cast<float*>(ws + p.off_scores);
    const long long blocks = (long long)batch * a.HK * p.ngroups * p.splits;
    a.o_blocks = p.splits > 1 ? (long long)batch * a.H : 0;
    a.w_blocks = weights ? (int)((vis + kJoinTokens - 1) / kJoinTokens) : 0;
    const long long jblocks = a.o_blocks + (long long)batch * a.HK * a.w_blocks;
    if (blocks > 0x7FFFFFFFLL || jblocks > 0x7FFFFFFFLL) return RKV_ERR_UNSUPPORTED;
    rc = launch_pass<PASS_ALL>(a, cache->dtype, p.gt, blocks, false, st);
    if (rc || !join || jblocks == 0) return rc;
    size_t smem = (size_t)p.splits * sizeof(float);
    if (weights && smem < (size_t)a.G * sizeof(float2)) smem = (size_t)a.G * sizeof(float2);
    const cudaError_t e = launch_pdl(paged_join_kernel, dim3((unsigned)jblocks), dim3(128), smem, st, a);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}
