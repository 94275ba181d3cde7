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

// ---------------------------------------------------------------------------
// The decode kernel: matrix instructions on tiles of 16 tokens
// ---------------------------------------------------------------------------
constexpr int kKeys = 16;  // tokens of a tile

enum { KIND_F16 = 0, KIND_BF16 = 1, KIND_F32 = 2 };

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
// CTAs of an SM.
template <int KIND_, int DP_, int NT_>
struct Shape {
    static constexpr int KIND = KIND_, DP = DP_, NT = NT_;
    static constexpr int SIZE = KIND == KIND_F32 ? 4 : 2;
    static constexpr int ROW = DP * SIZE;             // bytes of a row in shared memory
    static constexpr int SLOT = kKeys * ROW;          // 16 rows of K or of V
    static constexpr int W = ROW > 512 ? 4 : 8;
    static constexpr int SLOTS = ROW > 128 ? 3 : 5;   // odd: K and V take the slots in turn
    static constexpr int CTAS = ROW > 256 ? 1 : 2;
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
template <typename S>
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
    uint32_t q[S::QS ? 1 : NT][S::QS ? 1 : DP / 16][2];
    if (F32) {
        // step (blk, e): columns 32 blk + 4 t + e and 16 further of head g, as hi, hi, lo, lo
        for (int i = warp; i < DP / 8 * NT; i += W) {
            const int n = i / (DP / 8), st = i % (DP / 8), d = (st >> 2) * 32 + 4 * t + (st & 3);
            const bool have = n * 8 + g < ng;
            const float* row = reinterpret_cast<const float*>(qb) + (size_t)(h0 + n * 8 + g) * D;
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
                       ? __ldg(reinterpret_cast<const uint32_t*>(qb + ((size_t)(h0 + n * 8 + g) * D + d) * 2))
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
    merge_warps<W>(a, (size_t)b * a.H + h0, ng, split, ms, ls, os, 8 * NT, S::PITCH);
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

template <int KIND, int DP, int NT>
int launch_shape(const DecodeArgs& a, long long blocks, cudaStream_t st) {
    using S = Shape<KIND, DP, NT>;
    static_assert(S::SMEM * S::CTAS + 1024 * S::CTAS <= 228 * 1024, "the CTAs of an SM fit in its shared memory");
    if (cudaFuncSetAttribute(paged_decode_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM) != cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    paged_decode_kernel<S><<<(unsigned)blocks, S::W * 32, S::SMEM, st>>>(a);
    return launched();
}
template <int KIND>
int launch_kind(const DecodeArgs& a, int gt, long long blocks, cudaStream_t st) {
    if constexpr (KIND != KIND_F32) {
        if (gt == 16) return a.D <= 64 ? launch_shape<KIND, 64, 2>(a, blocks, st) : launch_shape<KIND, 128, 2>(a, blocks, st);
    }
    if (a.D <= 64) return launch_shape<KIND, 64, 1>(a, blocks, st);
    if (a.D <= 128) return launch_shape<KIND, 128, 1>(a, blocks, st);
    return launch_shape<KIND, 256, 1>(a, blocks, st);
}

}  // namespace
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
    switch (cache->dtype) {
        case RKV_F32: rc = launch_kind<KIND_F32>(a, p.gt, blocks, st); break;
        case RKV_BF16: rc = launch_kind<KIND_BF16>(a, p.gt, blocks, st); break;
        default: rc = launch_kind<KIND_F16>(a, p.gt, blocks, st); break;
    }
    if (rc || !join || jblocks == 0) return rc;
    size_t smem = (size_t)p.splits * sizeof(float);
    if (weights && smem < (size_t)a.G * sizeof(float2)) smem = (size_t)a.G * sizeof(float2);
    const cudaError_t e = launch_pdl(paged_join_kernel, dim3((unsigned)jblocks), dim3(128), smem, st, a);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}
