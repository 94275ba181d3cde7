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
#include "paged.cuh"

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
// that lie back to back are read in whole lines.
template <typename VT>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs a) {
    const int b = blockIdx.y;
    const int n = a.n_new ? min(max(a.n_new[b], 0), a.n_rows) : a.n_rows;
    const int first = a.c.lens[b] - n;
    const long long cap = (long long)a.c.table_stride * a.c.page_size;
    const int per = a.HK * a.vpr;
    const long long total = (long long)n * per;
    for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += (long long)gridDim.x * blockDim.x) {
        const int i = (int)(e / per), r = (int)(e - (long long)i * per);
        const int h = r / a.vpr, vec = r - h * a.vpr;
        const long long t = (long long)first + i;
        if (t < 0 || t >= cap) continue;
        const long long off = paged_offset(a.c, b, h, (int)t);
        if (off < 0) continue;
        const size_t s = (size_t)b * a.item_stride + (size_t)i * a.src_token + (size_t)h * a.src_head;
        reinterpret_cast<VT*>(a.c.K + off)[vec] = reinterpret_cast<const VT*>(a.k + s)[vec];
        reinterpret_cast<VT*>(a.c.V + off)[vec] = reinterpret_cast<const VT*>(a.v + s)[vec];
    }
}

// ---------------------------------------------------------------------------
// decode
// ---------------------------------------------------------------------------
constexpr int kWarps = 4;
constexpr int kTile = 32;       // tokens a warp takes at a time
constexpr int kMinChunk = 128;  // visible tokens per CTA at least
constexpr int kMaxSplits = 1024;
constexpr int kSms = 148;
constexpr int kMaxWaves = 8;       // of CTAs that a cache is split into at most
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

__device__ __forceinline__ float4 load16(const uint8_t* p) { return __ldg(reinterpret_cast<const float4*>(p)); }

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
// 0 in place of -inf, so that a set with nothing in it subtracts no infinities.
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

// Joins the warps' (m, l, o) of ng heads from shared memory (ms, ls [warps][rows], os [warps][rows][pitch])
// and writes the part, or the output where there is one part.
__device__ __forceinline__ void merge_warps(const DecodeArgs& a, size_t head0, int ng, int split, const float* ms,
                                            const float* ls, const float* os, int rows, int pitch) {
    const int D = a.D;
    for (int i = threadIdx.x; i < ng * D; i += kWarps * 32) {
        const int g = i / D, d = i - g * D;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, ms[w * rows + g]);
        const float mf = finite_max(mm);
        float ll = 0.0f, oo = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
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

size_t simt_smem(int GT, int D) { return sizeof(float) * ((size_t)GT * D + kWarps * GT * kTile + 2 * kWarps * GT + (size_t)kWarps * GT * D); }

// fp32 caches, fused multiply-adds on the CUDA cores: one CTA per (item, KV
// head, group of up to GT query heads, part).  Every warp takes 32 tokens at a
// time on its own: 8 lanes form the scores of a token, a lane per token forms the weights, and LR lanes of 16 bytes add
// up a V row.  VL: 16-byte vectors of a V row per lane.
template <int GT, int VL>
__global__ void __launch_bounds__(kWarps * 32) paged_decode_simt_kernel(const DecodeArgs a) {
    constexpr int N = 4;                // floats of a 16-byte vector
    constexpr int J = GT <= 2 ? 8 : 4;  // tokens whose scores a lane forms together
    constexpr int UV = GT <= 2 ? 16 : 4;  // V rows a lane has on their way together
    extern __shared__ __align__(16) float sm[];
    asm volatile("griddepcontrol.launch_dependents;");  // the join may be scheduled (it waits for this grid)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int D = a.D, VPR = D / N;
    float* qs = sm;                                         // [GT][D]
    float* pw = qs + GT * D + warp * GT * kTile;            // [GT][32] of this warp
    float* ms = qs + GT * D + kWarps * GT * kTile;          // [warps][GT]
    float* ls = ms + kWarps * GT;                           // [warps][GT]
    float* os = ls + kWarps * GT;                           // [warps][GT][D]

    long long id = blockIdx.x;
    const int split = (int)(id % a.splits);
    id /= a.splits;
    const int grp = (int)(id % a.ngroups);
    id /= a.ngroups;
    const int hk = (int)(id % a.HK), b = (int)(id / a.HK);
    const Visible vis = visible(a, b);
    const long long v_lo = (long long)split * a.chunk;
    if (split > 0 && v_lo >= vis.nvis) return;  // the join takes the parts that hold tokens
    const int v0 = (int)v_lo, v1 = (int)min((long long)vis.nvis, v_lo + a.chunk);
    const int h0 = hk * a.G + grp * GT, ng = min(GT, a.G - grp * GT);

    const float* q = reinterpret_cast<const float*>(a.Q + (size_t)b * a.q_stride);
    for (int i = tid; i < GT * D; i += kWarps * 32) {
        const int g = i / D;
        qs[i] = g < ng ? q[(h0 + g) * D + (i - g * D)] * a.scale2 : 0.0f;
    }
    __syncthreads();

    int LR = 1;
    while (LR < VPR && LR < 32) LR <<= 1;
    const int TPS = 32 / LR, vl0 = lane & (LR - 1), tsub = lane / LR;
    float m[GT], l[GT], acc[VL][N][GT];
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        m[g] = -INFINITY;
        l[g] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < VL; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e)
#pragma unroll
            for (int g = 0; g < GT; ++g) acc[i][e][g] = 0.0f;

    for (int t0 = v0 + warp * kTile; t0 < v1; t0 += kWarps * kTile) {
        const int v = t0 + lane;
        const long long off = v < v1 ? paged_offset(a.c, b, hk, vis.token(v)) : -1;
#pragma unroll
        for (int pass = 0; pass < 8 / J; ++pass) {
            long long o[J];
            float s[J][GT];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                o[j] = __shfl_sync(0xffffffffu, off, (pass * J + j) * 4 + (lane >> 3));
#pragma unroll
                for (int g = 0; g < GT; ++g) s[j][g] = 0.0f;
            }
#pragma unroll 2
            for (int vec = lane & 7; vec < VPR; vec += 8) {
                float4 x[J];
#pragma unroll
                for (int j = 0; j < J; ++j)
                    x[j] = o[j] >= 0 ? load16(a.c.K + o[j] + vec * 16) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const float f[N] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
                    for (int g = 0; g < GT; ++g)
#pragma unroll
                        for (int e = 0; e < N; ++e) s[j][g] = fmaf(f[e], qs[g * D + vec * N + e], s[j][g]);
                }
            }
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int g = 0; g < GT; ++g) {
                    float x = s[j][g];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    x += __shfl_xor_sync(0xffffffffu, x, 2);
                    x += __shfl_xor_sync(0xffffffffu, x, 4);
                    if ((lane & 7) == g) pw[g * kTile + (pass * J + j) * 4 + (lane >> 3)] = x;
                }
        }
        __syncwarp();
#pragma unroll
        for (int g = 0; g < GT; ++g) {
            const float x = off >= 0 ? pw[g * kTile + lane] : -INFINITY;
            if (a.scores && v < v1 && g < ng) a.scores[((size_t)b * a.H + h0 + g) * a.vmax + v] = x;
            const float mn = fmaxf(m[g], warp_max(x)), mf = finite_max(mn);
            const float corr = exp2f(m[g] - mf), p = exp2f(x - mf);
            m[g] = mn;
            l[g] = l[g] * corr + p;
            pw[g * kTile + lane] = p;
#pragma unroll
            for (int i = 0; i < VL; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) acc[i][e][g] *= corr;
        }
        __syncwarp();
#pragma unroll UV
        for (int s0 = 0; s0 < kTile; s0 += TPS) {
            const int t = s0 + tsub;
            const long long o = __shfl_sync(0xffffffffu, off, t);
#pragma unroll
            for (int i = 0; i < VL; ++i) {
                const int vec = vl0 + i * 32;
                const float4 x = o >= 0 && vec < VPR ? load16(a.c.V + o + vec * 16) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const float f[N] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int g = 0; g < GT; ++g) {
                    const float p = pw[g * kTile + t];
#pragma unroll
                    for (int e = 0; e < N; ++e) acc[i][e][g] = fmaf(p, f[e], acc[i][e][g]);
                }
            }
        }
        __syncwarp();
    }
    // the token groups of a warp, then the warps
#pragma unroll
    for (int g = 0; g < GT; ++g) {
        l[g] = warp_sum(l[g]);
        if (lane == 0) {
            ms[warp * GT + g] = m[g];
            ls[warp * GT + g] = l[g];
        }
#pragma unroll
        for (int i = 0; i < VL; ++i)
#pragma unroll
            for (int e = 0; e < N; ++e) {
                float x = acc[i][e][g];
                for (int o = LR; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                const int vec = vl0 + i * 32;
                if (tsub == 0 && vec < VPR) os[(warp * GT + g) * D + vec * N + e] = x;
            }
    }
    __syncthreads();
    merge_warps(a, (size_t)b * a.H + h0, ng, split, ms, ls, os, GT, D);
}

// ---------------------------------------------------------------------------
// 16-bit caches: matrix instructions on tiles of 16 tokens
// ---------------------------------------------------------------------------
constexpr int kKeys = 16;     // tokens of a tile
constexpr int kMmaStages = 3; // tiles of a warp in shared memory, one in use and the others on their way

template <bool BF>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
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

__host__ __device__ constexpr int mma_stage_bytes(int DP) { return kKeys * DP * 2 * 2; }  // K rows, V rows
constexpr size_t mma_smem(int DP, int NT) {
    const size_t ring = (size_t)kWarps * kMmaStages * mma_stage_bytes(DP);
    const size_t merge = sizeof(float) * kWarps * 8 * NT * (2 + DP + 4);
    return ring > merge ? ring : merge;
}

// One CTA per (item, KV head, group of up to 8 NT query heads, part); every
// warp takes tiles of 16 tokens on its own.  The tile's K and V rows arrive in
// the warp's ring by 16-byte asynchronous copies, rows of DP columns with the
// 16-byte chunk c of row r at c ^ (r % 8), so that the eight rows of a matrix
// load lie in different banks.  Scores: K (16 tokens x 16 columns per step) by
// q^T (8 heads); output: V^T (16 columns x 16 tokens) by P (8 heads), whose
// fragment is the transpose of the scores'.  P keeps fp32's precision: it
// enters as a sum of 16-bit parts (three for bf16, two for fp16), one product
// each, which costs nothing here, since the kernel is bound by its reads.
// A row's maximum is raised only when a score exceeds it by more than 2^8
// (both types hold P then); fp16's P is kept 2^7 larger, away from the type's
// smallest numbers.
template <bool BF, int DP, int NT>
__global__ void __launch_bounds__(kWarps * 32) paged_decode_mma_kernel(const DecodeArgs a) {
    constexpr int kStage = mma_stage_bytes(DP), CH = DP / 8;  // 16-byte chunks of a row
    constexpr int PARTS = BF ? 3 : 2;
    constexpr float kLift = BF ? 0.0f : 7.0f, kGrow = 8.0f;
    constexpr int RPI = 32 / CH;                              // rows a warp copies per instruction
    extern __shared__ __align__(128) uint8_t smem[];
    asm volatile("griddepcontrol.launch_dependents;");  // the join may be scheduled (it waits for this grid)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int D = a.D;

    long long id = blockIdx.x;
    const int split = (int)(id % a.splits);
    id /= a.splits;
    const int grp = (int)(id % a.ngroups);
    id /= a.ngroups;
    const int hk = (int)(id % a.HK), b = (int)(id / a.HK);
    const Visible vis = visible(a, b);
    const long long v_lo = (long long)split * a.chunk;
    if (split > 0 && v_lo >= vis.nvis) return;  // the join takes the parts that hold tokens
    const int v0 = (int)v_lo, v1 = (int)min((long long)vis.nvis, v_lo + a.chunk);
    const int h0 = hk * a.G + grp * 8 * NT, ng = min(8 * NT, a.G - grp * 8 * NT);

    uint8_t* ring = smem + warp * kMmaStages * kStage;
    const uint32_t ring_u = smem_u32(ring);
    if (D < DP)  // the columns behind D count as zeros and are never copied
        for (int e = lane; e < kMmaStages * 2 * kKeys * CH; e += 32) {
            const int row = e / CH, c = e % CH;
            if ((c ^ (row & 7)) >= D / 8) *reinterpret_cast<uint4*>(ring + row * DP * 2 + c * 16) = make_uint4(0, 0, 0, 0);
        }

    // the tile's tokens: lane i (and i + 16) has the row of token i
    const int ntiles = v1 > v0 ? (v1 - v0 + kKeys - 1) / kKeys : 0;
    auto row_of = [&](int tile) -> long long {
        const int v = v0 + tile * kKeys + (lane & 15);
        return tile < ntiles && v < v1 ? paged_offset(a.c, b, hk, vis.token(v)) : -1;
    };
    const int cchunk = lane % CH, crow = lane / CH;
    auto fetch = [&](int slot, long long off) {
#pragma unroll
        for (int i = 0; i < kKeys / RPI; ++i) {
            const int r = i * RPI + crow;
            const long long o = __shfl_sync(0xffffffffu, off, r);
            if (cchunk < D / 8) {
                const uint32_t dst = ring_u + slot * kStage + r * DP * 2 + ((cchunk ^ (r & 7)) << 4);
                copy16(dst, o >= 0 ? a.c.K + o + cchunk * 16 : a.Q, o >= 0);
                copy16(dst + kKeys * DP * 2, o >= 0 ? a.c.V + o + cchunk * 16 : a.Q, o >= 0);
            }
        }
    };
    long long off_next = row_of(warp);
    uint32_t real[kMmaStages];  // which of the tile's tokens there are
#pragma unroll
    for (int s = 0; s < kMmaStages - 1; ++s) {
        const long long off = off_next;
        off_next = row_of(warp + (s + 1) * kWarps);
        real[s] = __ballot_sync(0xffffffffu, off >= 0);
        if (warp + s * kWarps < ntiles) fetch(s, off);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // q^T fragments: columns 2 t, 2 t + 1 (and + 8) of head g
    uint32_t q[NT][DP / 16][2];
    const uint8_t* qb = a.Q + (size_t)b * a.q_stride;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = k * 16 + e * 8 + 2 * t;
                q[n][k][e] = n * 8 + g < ng && d < D
                                 ? __ldg(reinterpret_cast<const uint32_t*>(qb + ((size_t)(h0 + n * 8 + g) * D + d) * 2))
                                 : 0u;
            }
    float m[NT][2], l[NT][2], o[NT][DP / 16][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][k][e] = 0.0f;
    }
    // matrix loads: lane i gives the address of row i % 8 of block i / 8
    const int kr = lane & 15, kc = lane >> 4;                       // K: rows 0-15, column halves
    const int vr = (lane & 7) + ((lane >> 4) << 3), vc = (lane >> 3) & 1;  // V^T: column halves first, then rows

    int slot = 0;
    for (int tile = warp; tile < ntiles; tile += kWarps) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kMmaStages - 2) : "memory");
        __syncwarp();
        const uint32_t here = real[0];
#pragma unroll
        for (int s = 0; s + 1 < kMmaStages - 1; ++s) real[s] = real[s + 1];
        {
            const int ahead = tile + (kMmaStages - 1) * kWarps;
            const long long off = off_next;
            off_next = row_of(ahead + kWarps);
            real[kMmaStages - 2] = __ballot_sync(0xffffffffu, off >= 0);
            int fs = slot + kMmaStages - 1;
            if (fs >= kMmaStages) fs -= kMmaStages;
            if (ahead < ntiles) fetch(fs, off);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        const uint32_t kb = ring_u + slot * kStage, vb = kb + kKeys * DP * 2;
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            uint32_t f[4];
            ldmatrix4<false>(f, kb + kr * DP * 2 + (((2 * k + kc) ^ (kr & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816<BF>(s[n], f, q[n][k][0], q[n][k][1]);
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
            if (a.scores) {
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
                    for (int k = 0; k < DP / 16; ++k) {
                        o[n][k][e] *= corr;
                        o[n][k][e + 2] *= corr;
                    }
                }
        }
        uint32_t p[NT][PARTS][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float m0 = finite_max(m[n][0]) - kLift, m1 = finite_max(m[n][1]) - kLift;
            float x[4] = {ex2(s[n][0] - m0), ex2(s[n][1] - m1), ex2(s[n][2] - m0), ex2(s[n][3] - m1)};
            l[n][0] += x[0] + x[2];
            l[n][1] += x[1] + x[3];
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
                p[n][i][0] = transpose8x8(split2<BF>(x[0], x[1]));
                p[n][i][1] = transpose8x8(split2<BF>(x[2], x[3]));
            }
        }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            uint32_t f[4];
            ldmatrix4<true>(f, vb + vr * DP * 2 + (((2 * k + vc) ^ (vr & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < PARTS; ++i) mma16816<BF>(o[n][k], f, p[n][i][0], p[n][i][1]);
        }
        if (++slot == kMmaStages) slot = 0;
    }
    // the warps' (m, l, o) meet in shared memory, over the ring
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    float* ms = reinterpret_cast<float*>(smem);  // [warps][8 NT]
    float* ls = ms + kWarps * 8 * NT;
    float* os = ls + kWarps * 8 * NT;            // [warps][8 NT][DP + 4]
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
            for (int k = 0; k < DP / 16; ++k) {
                os[h * (DP + 4) + k * 16 + g] = o[n][k][e];
                os[h * (DP + 4) + k * 16 + g + 8] = o[n][k][e + 2];
            }
        }
    __syncthreads();
    merge_warps(a, (size_t)b * a.H + h0, ng, split, ms, ls, os, 8 * NT, DP + 4);
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
constexpr int kJoinAhead = 16;    // parts of a column read before the shares are known

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

// Query heads of a KV head that one CTA takes: up to 8 by fused multiply-adds (fp32); 8 or 16 by matrix
// instructions, 8 where 16 heads of 256 columns would not fit in registers.
int head_group(int dtype, int G, int D) {
    if (dtype == RKV_F32) return G >= 5 ? 8 : G >= 3 ? 4 : G;
    return G > 8 && D <= 128 ? 16 : 8;
}

// CTAs that run at a time: what shared memory (16-bit) or registers (fp32) let the SMs hold.
int decode_slots(int dtype, int gt, int D) {
    if (dtype == RKV_F32) return kSms * (gt <= 4 ? 4 : 3);
    return kSms * (D <= 64 ? 4 : D <= 128 ? 2 : 1);
}
long long decode_units(int dtype, int H, int HK, int D, int batch) {
    const int G = H / HK, gt = head_group(dtype, G, D);
    return (long long)batch * HK * ((G + gt - 1) / gt);
}
// The most parts that decode_parts gives up to visible_max, which it grows with.
long long decode_parts_bound(int dtype, int H, int HK, int D, long long visible_max, int batch) {
    const long long units = decode_units(dtype, H, HK, D, batch);
    const long long slots = decode_slots(dtype, head_group(dtype, H / HK, D), D);
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
    const long long slots = decode_slots(dtype, head_group(dtype, H / HK, D), D);
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

template <int GT>
int launch_simt(const DecodeArgs& a, long long blocks, cudaStream_t st) {
    const int vpr = a.D / 4;
    const size_t smem = simt_smem(GT, a.D);
    if (vpr > 32)
        paged_decode_simt_kernel<GT, 2><<<(unsigned)blocks, kWarps * 32, smem, st>>>(a);
    else
        paged_decode_simt_kernel<GT, 1><<<(unsigned)blocks, kWarps * 32, smem, st>>>(a);
    return launched();
}

int launch_f32(const DecodeArgs& a, int gt, long long blocks, cudaStream_t st) {
    switch (gt) {
        case 1: return launch_simt<1>(a, blocks, st);
        case 2: return launch_simt<2>(a, blocks, st);
        case 4: return launch_simt<4>(a, blocks, st);
        default: return launch_simt<8>(a, blocks, st);
    }
}

template <bool BF, int DP, int NT>
int launch_mma(const DecodeArgs& a, long long blocks, cudaStream_t st) {
    constexpr size_t smem = mma_smem(DP, NT);
    if (cudaFuncSetAttribute(paged_decode_mma_kernel<BF, DP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) !=
        cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    paged_decode_mma_kernel<BF, DP, NT><<<(unsigned)blocks, kWarps * 32, smem, st>>>(a);
    return launched();
}
template <bool BF>
int launch_16(const DecodeArgs& a, int gt, long long blocks, cudaStream_t st) {
    if (a.D <= 64) return gt == 16 ? launch_mma<BF, 64, 2>(a, blocks, st) : launch_mma<BF, 64, 1>(a, blocks, st);
    if (a.D <= 128) return gt == 16 ? launch_mma<BF, 128, 2>(a, blocks, st) : launch_mma<BF, 128, 1>(a, blocks, st);
    return launch_mma<BF, 256, 1>(a, blocks, st);
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_paged_append(const rkv_paged_cache* cache, const void* k, const void* v, int n_rows, int batch,
                                long long src_item_stride, long long src_token_stride, long long src_head_stride,
                                const int* n_new, void* stream) {
    const int rc = paged_check(cache, true);
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
    long long gx = (total + 255) / 256;
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
    int rc = paged_check(cache, true);
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
    switch (cache->dtype) {
        case RKV_F32: rc = launch_f32(a, p.gt, blocks, st); break;
        case RKV_BF16: rc = launch_16<true>(a, p.gt, blocks, st); break;
        default: rc = launch_16<false>(a, p.gt, blocks, st); break;
    }
    if (rc || !join || jblocks == 0) return rc;
    size_t smem = (size_t)p.splits * sizeof(float);
    if (weights && smem < (size_t)a.G * sizeof(float2)) smem = (size_t)a.G * sizeof(float2);
    const cudaError_t e = launch_pdl(paged_join_kernel, dim3((unsigned)jblocks), dim3(128), smem, st, a);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}
