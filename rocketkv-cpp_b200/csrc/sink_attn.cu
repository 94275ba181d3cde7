// sink_attn.cu -- causal prefill attention with a sliding window and a few
// first tokens that stay visible.
//
// For a tile of queries the keys are taken tile by tile with the running
// (m, l, o) of a softmax: x = q k^T log2(e) / sqrt(D), m the row's largest x,
// l = sum 2^(x - m), o = sum 2^(x - m) v; tiles that neither hold a sink nor
// meet the window of any row are not visited.  O = o / l, lse = (m + log2 l) ln 2.
#include "sink_attn.cuh"
#include "tf32.cuh"

namespace rkv {
namespace {

constexpr int kBN = 64;  // keys of a tile

// fp32 inputs: tf32 products of each operand as its top 19 bits and the rest,
// three per product (hi hi + lo hi + hi lo), summed by the matrix units over a
// tile or less and then added (their sums cut instead of rounding).  The rate
// of mma.sync bounds it: 24/8 heads of 128, 2048 tokens, causal, 642 us, 40
// TFLOP/s, which is 120 of products (tcgen05 would allow some 275; not built).
// Spills at 128 and 256 columns: 56 and 248 bytes a thread.  One CTA per BM
// queries of a head, a warp per 16 of them, 64 keys at a time; V arrives under the scores
// and the next K under the output's products.
//
// S = Q K^T has the queries on the rows; its fragment is P's fragment for
// O += P V when the keys 2 t and 2 t + 1 of eight count as steps t and t + 4,
// and the order of a product's steps is free.  Likewise a lane's 16-byte chunk
// of a K row gives four steps of columns, and one of a V row four columns of
// the output.  Chunks are stored at other places of their rows (c ^ 4 (r % 2)
// for Q and K, c ^ (r % 8) for V), so that eight lanes' loads lie in different
// banks.
template <int DP>
struct F32Shape {
    static constexpr int BM = DP <= 128 ? 128 : 64;
    static constexpr int NT = BM * 2;             // threads: a warp per 16 queries
    static constexpr int ROW = DP * 4;            // bytes
    static constexpr int SMEM = (BM + 2 * kBN) * ROW;
};

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t word(const uint4& v, int e) { return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w; }

template <int DP>
__global__ void __launch_bounds__(F32Shape<DP>::NT) sink_f32_kernel(const SinkArgs a) {
    using S = F32Shape<DP>;
    constexpr int CH = DP / 4;  // 16-byte chunks of a row
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t qs = smem_u32(smem), ks = qs + S::BM * S::ROW, vs = ks + kBN * S::ROW;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    if (blockIdx.x == 0 && tid == 0) *a.err = 0;  // nothing here waits
    long long id = blockIdx.x;
    const int part = (int)(id % a.parts);
    id /= a.parts;
    const int rest = (int)(id % ((long long)a.H * a.batch));
    const int qt = a.qtiles - 1 - (int)(id / ((long long)a.H * a.batch));  // the longest rows first
    const int h = rest % a.H, b = rest / a.H, hk = h / a.G, i0 = qt * S::BM;
    SinkRange rg = sink_range(a, b, i0, S::BM, kBN);
    const int tiles = rg.part(part, a.parts);
    const size_t prow0 = (((size_t)part * a.batch + b) * a.H + h) * a.len_q + i0;  // the first row of the part
    asm volatile("griddepcontrol.launch_dependents;");  // a join may be scheduled (it waits for this grid)
    if (tiles == 0) {
        if (a.parts > 1)
            for (int i = tid; i < min(min(S::BM, a.len_q - i0), rg.n - rg.p0); i += S::NT)
                a.part_ml[prow0 + i] = make_float2(-INFINITY, 0.0f);
        return;
    }
    const uint8_t* K = a.K + (size_t)b * a.ks.item + (size_t)hk * a.ks.head;
    const uint8_t* V = a.V + (size_t)b * a.ks.item + (size_t)hk * a.ks.head;
    const uint8_t* Q = a.Q + (size_t)b * a.qs.item + (size_t)h * a.qs.head + (size_t)i0 * a.qs.token;
    const int qrows = min(min(S::BM, a.len_q - i0), rg.n - rg.p0);  // rows that are written
    const int chunks = a.D / 4;
    // rows of a tile, zeros (nothing is read) behind `valid` rows and behind dim_head
    auto fetch = [&](uint32_t dst, const uint8_t* src, long long stride, int rows, int valid, bool isv) {
        for (int e = tid; e < rows * CH; e += S::NT) {
            const int r = e / CH, c = e % CH;
            const bool real = r < valid && c < chunks;
            copy16(dst + r * S::ROW + ((c ^ (isv ? r & 7 : (r & 1) << 2)) << 4), real ? src + r * stride + c * 16 : a.Q, real);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto key_tile = [&](int it, bool isv) {
        const int j0 = rg.tile(it) * kBN;
        fetch(isv ? vs : ks, (isv ? V : K) + (size_t)j0 * a.ks.token, a.ks.token, kBN, min(kBN, rg.n - j0), isv);
    };
    fetch(qs, Q, a.qs.token, S::BM, qrows, false);
    key_tile(0, false);

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};  // rows g and g + 8 of the warp's 16
    float o[DP / 8][4];
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;
    const uint32_t qw = qs + warp * 16 * S::ROW;
    const int pg = rg.p0 + warp * 16 + g;  // position of row g
    for (int it = 0; it < tiles; ++it) {
        key_tile(it, true);
        asm volatile("cp.async.wait_group 1;" ::: "memory");  // K (and Q) are here, V is on its way
        __syncthreads();
        float s[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.0f;
        const int swz = (g & 1) << 2;
#pragma unroll 1
        for (int blk = 0; blk < DP / 32; ++blk) {
            // rows g and g + 8, chunks t and t + 4 of 32 columns
            const int c = blk * 8 + t;
            const uint4 x0 = lds16(qw + g * S::ROW + ((c ^ swz) << 4)), x1 = lds16(qw + (g + 8) * S::ROW + ((c ^ swz) << 4));
            const uint4 x2 = lds16(qw + g * S::ROW + (((c + 4) ^ swz) << 4)), x3 = lds16(qw + (g + 8) * S::ROW + (((c + 4) ^ swz) << 4));
            uint32_t qh[4][4], ql[4][4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                tf32_split(word(x0, e), qh[e][0], ql[e][0]);
                tf32_split(word(x1, e), qh[e][1], ql[e][1]);
                tf32_split(word(x2, e), qh[e][2], ql[e][2]);
                tf32_split(word(x3, e), qh[e][3], ql[e][3]);
            }
#pragma unroll
            for (int n0 = 0; n0 < 8; n0 += 4) {  // products into four accumulators in turn: one alone waits for itself
                uint4 y0[4], y1[4];
                float part[4][4];
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const uint32_t kr = ks + ((n0 + n) * 8 + g) * S::ROW;
                    y0[n] = lds16(kr + ((c ^ swz) << 4));
                    y1[n] = lds16(kr + (((c + 4) ^ swz) << 4));
#pragma unroll
                    for (int e = 0; e < 4; ++e) part[n][e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t h0[4], h1[4], l0[4], l1[4];
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        tf32_split(word(y0[n], e), h0[n], l0[n]);
                        tf32_split(word(y1[n], e), h1[n], l1[n]);
                    }
#pragma unroll
                    for (int n = 0; n < 4; ++n) mma_tf32(part[n], qh[e], l0[n], l1[n]);
#pragma unroll
                    for (int n = 0; n < 4; ++n) mma_tf32(part[n], ql[e], h0[n], h1[n]);
#pragma unroll
                    for (int n = 0; n < 4; ++n) mma_tf32(part[n], qh[e], h0[n], h1[n]);
                }
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n0 + n][e] += part[n][e];
            }
        }
        // columns 8 n + 2 t and + 1 of rows g (s[n][0], s[n][1]) and g + 8
        const int j0 = rg.tile(it) * kBN, pw = pg - g;  // the warp's rows are at positions pw .. pw + 15
        const bool whole = j0 + kBN - 1 <= pw && j0 + kBN <= rg.n && (a.window <= 0 || j0 > pw + 15 - a.window || j0 + kBN <= a.sinks);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int p = pg + 8 * r;
            float mt = -INFINITY;
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float& x = s[n][2 * r + e];
                    x = whole || sink_sees(a, rg.n, p, j0 + n * 8 + 2 * t + e) ? x * a.scale2 : -INFINITY;
                    mt = fmaxf(mt, x);
                }
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
            const float mn = fmaxf(m[r], mt), mf = mn == -INFINITY ? 0.0f : mn;
            const float corr = exp2f(m[r] - mf);
            m[r] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < 8; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    s[n][2 * r + e] = exp2f(s[n][2 * r + e] - mf);
                    sum += s[n][2 * r + e];
                }
            l[r] = l[r] * corr + sum;
#pragma unroll
            for (int n = 0; n < DP / 8; ++n) {
                o[n][2 * r] *= corr;
                o[n][2 * r + 1] *= corr;
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // V is here, and every warp is done with K
        if (it + 1 < tiles) key_tile(it + 1, false);
#pragma unroll
        for (int j = 0; j < DP / 32; ++j) {
            float part[4][4];
#pragma unroll
            for (int e = 0; e < 16; ++e) part[e >> 2][e & 3] = 0.0f;
#pragma unroll
            for (int n8 = 0; n8 < 8; ++n8) {
                // keys 8 n8 + 2 t and + 1 are steps t and t + 4
                uint32_t ph[4], pl[4], h0[4], h1[4], l0[4], l1[4];
                tf32_split(__float_as_uint(s[n8][0]), ph[0], pl[0]);
                tf32_split(__float_as_uint(s[n8][2]), ph[1], pl[1]);
                tf32_split(__float_as_uint(s[n8][1]), ph[2], pl[2]);
                tf32_split(__float_as_uint(s[n8][3]), ph[3], pl[3]);
                const int r0 = n8 * 8 + 2 * t, c = g + 8 * j;
                const uint4 u = lds16(vs + r0 * S::ROW + ((c ^ (r0 & 7)) << 4));
                const uint4 w = lds16(vs + (r0 + 1) * S::ROW + ((c ^ ((r0 + 1) & 7)) << 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    tf32_split(word(u, e), h0[e], l0[e]);
                    tf32_split(word(w, e), h1[e], l1[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) mma_tf32(part[e], ph, l0[e], l1[e]);
#pragma unroll
                for (int e = 0; e < 4; ++e) mma_tf32(part[e], pl, h0[e], h1[e]);
#pragma unroll
                for (int e = 0; e < 4; ++e) mma_tf32(part[e], ph, h0[e], h1[e]);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) o[4 * j + (e >> 2)][e & 3] += part[e >> 2][e & 3];
        }
        __syncthreads();  // every warp is done with V
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        const int row = warp * 16 + g + 8 * r;
        if (row >= qrows) continue;
        const float inv = a.parts > 1 ? 1.0f : l[r] == 0.0f ? 0.0f : 1.0f / l[r];
        float* po = a.parts > 1 ? a.part_o + (prow0 + row) * a.D
                                : reinterpret_cast<float*>(a.O + (size_t)b * a.os.item + (size_t)h * a.os.head +
                                                           (size_t)(i0 + row) * a.os.token);
        // output column 4 (i + 8 j) + e is column i of tile 4 j + e; this lane has i = 2 t and 2 t + 1
#pragma unroll
        for (int j = 0; j < DP / 32; ++j)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int d = 4 * (2 * t + x + 8 * j);
                if (d < a.D)
                    *reinterpret_cast<float4*>(po + d) = make_float4(o[4 * j][2 * r + x] * inv, o[4 * j + 1][2 * r + x] * inv,
                                                                     o[4 * j + 2][2 * r + x] * inv, o[4 * j + 3][2 * r + x] * inv);
            }
        if (a.parts > 1) {
            if (t == 0) a.part_ml[prow0 + row] = make_float2(m[r] == -INFINITY ? 0.0f : m[r], l[r]);
        } else if (a.lse && t == 0)
            a.lse[((size_t)b * a.H + h) * a.len_q + i0 + row] =
                l[r] == 0.0f ? -INFINITY : ((m[r] == -INFINITY ? 0.0f : m[r]) + log2f(l[r])) * 0.693147180559945f;
    }
}

// Joins the parts of the keys: a warp per row.  m and l of a part that saw no key are -inf (or 0) and 0.
template <typename T>
__device__ __forceinline__ void store4(uint8_t* p, const float4& v);
template <>
__device__ __forceinline__ void store4<float>(uint8_t* p, const float4& v) { *reinterpret_cast<float4*>(p) = v; }
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(uint8_t* p, const float4& v) {
    __nv_bfloat162 x[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(x);
}
template <>
__device__ __forceinline__ void store4<__half>(uint8_t* p, const float4& v) {
    __half2 x[2] = {__floats2half2_rn(v.x, v.y), __floats2half2_rn(v.z, v.w)};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(x);
}
template <typename T>
__global__ void __launch_bounds__(256) sink_join_kernel(const SinkArgs a) {
    const long long rows = (long long)a.batch * a.H * a.len_q;
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    const int i = (int)(row % a.len_q), h = (int)(row / a.len_q % a.H), b = (int)(row / a.len_q / a.H);
    const int n = a.lens && row < rows ? min(max(a.lens[b], 0), a.len_k) : a.len_k;
    // Every thread waits, also those without a row: where no row exists the join would otherwise end before the
    // attention, and the stream's next work would not be ordered behind that.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (row >= rows || i + a.len_k - a.len_q >= n) return;  // or behind the sequence's end
    const float2 ml = lane < a.parts ? a.part_ml[lane * rows + row] : make_float2(-INFINITY, 0.0f);
    // a part without a visible key has l = 0, whatever its m
    float m = ml.y == 0.0f ? -INFINITY : ml.x;
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float mf = m == -INFINITY ? 0.0f : m;
    const float w = ml.y == 0.0f ? 0.0f : exp2f(ml.x - mf);
    float l = ml.y * w;
#pragma unroll
    for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint8_t* po = a.O + (size_t)b * a.os.item + (size_t)h * a.os.head + (size_t)i * a.os.token;
    for (int c0 = 0; c0 < a.D / 4; c0 += 32) {
        const int c = c0 + lane;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int p = 0; p < a.parts; ++p) {
            const float wp = __shfl_sync(0xffffffffu, w, p);
            if (wp != 0.0f && c < a.D / 4) {  // (a NaN weight counts)
                const float4 x = *reinterpret_cast<const float4*>(a.part_o + (p * rows + row) * a.D + 4 * c);
                o.x = fmaf(x.x, wp, o.x), o.y = fmaf(x.y, wp, o.y), o.z = fmaf(x.z, wp, o.z), o.w = fmaf(x.w, wp, o.w);
            }
        }
        if (c < a.D / 4) store4<T>(po + c * 4 * sizeof(T), make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    }
    if (lane == 0 && a.lse) a.lse[row] = l == 0.0f ? -INFINITY : (mf + log2f(l)) * 0.693147180559945f;
}
template <typename T>
int launch_join(const SinkArgs& a, cudaStream_t st) {
    const long long rows = (long long)a.batch * a.H * a.len_q;
    const cudaError_t e = launch_pdl(sink_join_kernel<T>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, a);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}

// CTAs' worth of queries, and the rows and keys of one's tiles.
long long sink_items(const SinkArgs& a, int dtype, int* rows, int* keys) {
    if (dtype != RKV_F32) return sink_tc_items(a, rows, keys);
    *rows = a.D <= 128 ? F32Shape<128>::BM : F32Shape<256>::BM;
    *keys = kBN;
    return (long long)((a.len_q + *rows - 1) / *rows) * a.batch * a.H;
}
struct SinkPlan {
    int parts;
    size_t off_ml, off_o, bytes;
};
// window 0: the most parts of any window.
SinkPlan sink_plan(const SinkArgs& a, int dtype, int sinks, int window) {
    int rows, keys;
    const long long items = sink_items(a, dtype, &rows, &keys);
    SinkPlan p{};
    p.parts = sink_parts(items, sink_tiles_max(a.len_k, sinks, window, rows, keys));
    p.off_ml = p.off_o = p.bytes = kWorkspaceHeader;
    if (p.parts > 1) {
        const size_t n = (size_t)p.parts * a.batch * a.H * a.len_q;
        p.off_o = align_up(p.off_ml + n * sizeof(float2), kWorkspaceAlign);
        p.bytes = align_up(p.off_o + n * a.D * sizeof(float), kWorkspaceAlign);
    }
    return p;
}

template <int DP>
int launch_f32(SinkArgs a, cudaStream_t st) {
    using S = F32Shape<DP>;
    a.qtiles = (a.len_q + S::BM - 1) / S::BM;
    const long long blocks = (long long)a.qtiles * a.H * a.batch * a.parts;
    if (blocks > 0x7FFFFFFFLL) return RKV_ERR_UNSUPPORTED;
    if (cudaFuncSetAttribute(sink_f32_kernel<DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM) != cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    sink_f32_kernel<DP><<<(unsigned)blocks, S::NT, S::SMEM, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}

}  // namespace
}  // namespace rkv

using namespace rkv;

static int sink_shape_check(int dtype, int len_q, int len_k, int batch, int num_heads, int num_heads_kv, int dim_head) {
    if (dtype != RKV_F32 && dtype != RKV_BF16 && dtype != RKV_F16) return RKV_ERR_INVALID_ARG;
    if (len_q < 0 || len_k < len_q || batch < 0 || num_heads <= 0 || num_heads_kv <= 0 || num_heads % num_heads_kv != 0 ||
        dim_head <= 0)
        return RKV_ERR_INVALID_ARG;
    if (dim_head % 8 != 0 || dim_head > 256 || len_k > (1 << 30)) return RKV_ERR_UNSUPPORTED;
    return RKV_OK;
}

extern "C" int rkv_sink_attention_workspace_size(int dtype, int len_q, int len_k, int batch, int num_heads, int num_heads_kv,
                                                 int dim_head, size_t* bytes) {
    const int rc = sink_shape_check(dtype, len_q, len_k, batch, num_heads, num_heads_kv, dim_head);
    if (rc || !bytes) return rc ? rc : (int)RKV_ERR_INVALID_ARG;
    SinkArgs a{};
    a.batch = batch;
    a.len_q = len_q;
    a.len_k = len_k;
    a.H = num_heads;
    a.HK = num_heads_kv;
    a.G = num_heads / num_heads_kv;
    a.D = dim_head;
    *bytes = sink_plan(a, dtype, 0, 0).bytes;
    return RKV_OK;
}

extern "C" int rkv_sink_attention(const void* Q, const void* K, const void* V, int dtype, int len_q, int len_k, int batch,
                                  int num_heads, int num_heads_kv, int dim_head, const rkv_row_strides* q_strides,
                                  const rkv_row_strides* kv_strides, const int* lens, int sinks, int window, void* O,
                                  const rkv_row_strides* o_strides, float* lse, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    const int rc = sink_shape_check(dtype, len_q, len_k, batch, num_heads, num_heads_kv, dim_head);
    if (rc) return rc;
    if (sinks < 0 || window < 0) return RKV_ERR_INVALID_ARG;
    if (batch == 0 || len_q == 0) return RKV_OK;
    const long long rowb = (long long)dim_head * (dtype == RKV_F32 ? 4 : 2);
    SinkArgs a{};
    a.qs = rkv_row_strides{(long long)num_heads * len_q * rowb, (long long)len_q * rowb, rowb};
    a.os = a.qs;
    a.ks = rkv_row_strides{(long long)num_heads_kv * len_k * rowb, (long long)len_k * rowb, rowb};
    if (q_strides) a.qs = *q_strides;
    if (kv_strides) a.ks = *kv_strides;
    if (o_strides) a.os = *o_strides;
    for (const rkv_row_strides* s : {&a.qs, &a.ks, &a.os}) {
        const bool kv = s == &a.ks;
        if ((s->item | s->head | s->token) & 15) return RKV_ERR_INVALID_ARG;
        if ((batch > 1 && s->item < rowb) || ((kv ? num_heads_kv : num_heads) > 1 && s->head < rowb) ||
            ((kv ? len_k : len_q) > 1 && s->token < rowb))
            return RKV_ERR_INVALID_ARG;
    }
    if (!Q || !K || !V || !O) return RKV_ERR_INVALID_ARG;
    if ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V) |
         reinterpret_cast<uintptr_t>(O)) & 15)
        return RKV_ERR_INVALID_ARG;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    a.Q = static_cast<const uint8_t*>(Q);
    a.K = static_cast<const uint8_t*>(K);
    a.V = static_cast<const uint8_t*>(V);
    a.O = static_cast<uint8_t*>(O);
    a.lse = lse;
    a.lens = lens;
    a.len_q = len_q;
    a.len_k = len_k;
    a.batch = batch;
    a.H = num_heads;
    a.HK = num_heads_kv;
    a.G = num_heads / num_heads_kv;
    a.D = dim_head;
    a.sinks = sinks < len_k ? sinks : len_k;      // no key lies behind len_k, so larger values
    a.window = window < len_k ? window : len_k;   // mean the same and could overflow below
    a.scale2 = 1.4426950408889634f / sqrtf((float)dim_head);
    a.err = static_cast<int*>(workspace);
    const SinkPlan plan = sink_plan(a, dtype, a.sinks, a.window);
    if (!workspace || workspace_bytes < plan.bytes || (reinterpret_cast<uintptr_t>(workspace) & 15)) return RKV_ERR_WORKSPACE;
    a.parts = plan.parts;
    a.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + plan.off_ml);
    a.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.off_o);
    int done;
    if (dtype != RKV_F32)
        done = launch_sink_tc(a, dtype, batch, st);
    else
        done = dim_head <= 64 ? launch_f32<64>(a, st) : dim_head <= 128 ? launch_f32<128>(a, st) : launch_f32<256>(a, st);
    if (done || a.parts == 1) return done;
    return dtype == RKV_F32 ? launch_join<float>(a, st)
           : dtype == RKV_BF16 ? launch_join<__nv_bfloat16>(a, st) : launch_join<__half>(a, st);
}
