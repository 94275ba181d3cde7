// sink_attn.cu -- causal prefill attention with a sliding window and a few
// first tokens that stay visible.
//
// For a tile of queries the keys are taken tile by tile with the running
// (m, l, o) of a softmax: x = q k^T log2(e) / sqrt(D), m the row's largest x,
// l = sum 2^(x - m), o = sum 2^(x - m) v; tiles that neither hold a sink nor
// meet the window of any row are not visited.  O = o / l, lse = (m + log2 l) ln 2.
#include "sink_attn.cuh"

namespace rkv {
namespace {

constexpr int kBM = 64, kBN = 64, kNT = 256;
constexpr int kPad = 4;  // floats behind each row of a transposed tile

template <typename T>
__device__ __forceinline__ void load4(const uint8_t* p, float* f);
template <>
__device__ __forceinline__ void load4<float>(const uint8_t* p, float* f) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const uint8_t* p, float* f) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xFFFF0000u);
    f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xFFFF0000u);
}
template <>
__device__ __forceinline__ void load4<__half>(const uint8_t* p, float* f) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}
template <typename T>
__device__ __forceinline__ void store4(uint8_t* p, const float* f);
template <>
__device__ __forceinline__ void store4<float>(uint8_t* p, const float* f) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
}
template <>
__device__ __forceinline__ void store4<__nv_bfloat16>(uint8_t* p, const float* f) {
    __nv_bfloat162 v[2] = {__floats2bfloat162_rn(f[0], f[1]), __floats2bfloat162_rn(f[2], f[3])};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v);
}
template <>
__device__ __forceinline__ void store4<__half>(uint8_t* p, const float* f) {
    __half2 v[2] = {__floats2half2_rn(f[0], f[1]), __floats2half2_rn(f[2], f[3])};
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(v);
}

// rows x D values of a tile into dst[d][row] (transposed) or dst[row][d];
// rows from `valid` on become zero and are not read.
template <typename T, bool TR>
__device__ __forceinline__ void stage(const uint8_t* src, long long stride, int valid, int D, float* dst, int pitch) {
    const int q4 = D / 4;
    for (int e = threadIdx.x; e < 64 * q4; e += kNT) {
        const int r = TR ? (e & 63) : e / q4, d = 4 * (TR ? (e >> 6) : e - r * q4);
        float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < valid) load4<T>(src + r * stride + d * (int)sizeof(T), f);
        if (TR) {
#pragma unroll
            for (int i = 0; i < 4; ++i) dst[(d + i) * pitch + r] = f[i];
        } else {
            *reinterpret_cast<float4*>(dst + r * pitch + d) = make_float4(f[0], f[1], f[2], f[3]);
        }
    }
}

__host__ __device__ constexpr size_t simt_floats(int D) {
    return (size_t)D * (kBM + kPad) + (size_t)(D * (kBN + kPad) > kBN * (D + kPad) ? D * (kBN + kPad) : kBN * (D + kPad)) +
           (size_t)kBN * (kBM + kPad);
}

// fp32 multiply-adds on the CUDA cores, any type: one CTA of 16 x 16 threads
// per 64 queries of a head, 64 keys at a time; a thread holds 4 x 4 scores and
// 4 rows x 4 NC columns of the output.
template <typename T, int NC>
__global__ void __launch_bounds__(kNT) sink_simt_kernel(const SinkArgs a) {
    extern __shared__ __align__(16) float sm[];
    const int D = a.D, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    float* Qs = sm;                                  // [D][64 + pad]
    float* KV = Qs + D * (kBM + kPad);               // K [D][64 + pad], then V [64][D + pad]
    float* Ps = KV + (simt_floats(D) - (size_t)D * (kBM + kPad) - (size_t)kBN * (kBM + kPad));  // [64 keys][64 + pad]
    long long id = blockIdx.x;
    const int qt = a.qtiles - 1 - (int)(id % a.qtiles);  // the longest rows first
    id /= a.qtiles;
    const int h = (int)(id % a.H), b = (int)(id / a.H), hk = h / a.G;
    const int i0 = qt * kBM;
    const SinkRange rg = sink_range(a, b, i0, kBM, kBN);
    const int tiles = rg.count();
    if (tiles == 0) return;
    const uint8_t* K = a.K + (size_t)b * a.ks.item + (size_t)hk * a.ks.head;
    const uint8_t* V = a.V + (size_t)b * a.ks.item + (size_t)hk * a.ks.head;
    const int qrows = min(min(kBM, a.len_q - i0), rg.n - rg.p0);
    stage<T, true>(a.Q + (size_t)b * a.qs.item + (size_t)h * a.qs.head + (size_t)i0 * a.qs.token, a.qs.token, qrows, D, Qs,
                   kBM + kPad);
    float m[4], l[4], o[4][NC][4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][c][e] = 0.0f;
    }
    for (int it = 0; it < tiles; ++it) {
        const int j0 = rg.tile(it) * kBN, valid = min(kBN, rg.n - j0);
        __syncthreads();
        stage<T, true>(K + (size_t)j0 * a.ks.token, a.ks.token, valid, D, KV, kBN + kPad);
        __syncthreads();
        float s[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[r][c] = 0.0f;
#pragma unroll 4
        for (int d = 0; d < D; ++d) {
            const float4 q = *reinterpret_cast<const float4*>(Qs + d * (kBM + kPad) + ty * 4);
            const float4 k = *reinterpret_cast<const float4*>(KV + d * (kBN + kPad) + tx * 4);
            const float qv[4] = {q.x, q.y, q.z, q.w}, kv[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[r][c] = fmaf(qv[r], kv[c], s[r][c]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int p = rg.p0 + ty * 4 + r;
            float mt = -INFINITY;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = sink_sees(a, rg.n, p, j0 + tx * 4 + c) ? s[r][c] * a.scale2 : -INFINITY;
                mt = fmaxf(mt, s[r][c]);
            }
#pragma unroll
            for (int x = 1; x < 16; x <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, x));
            const float mn = fmaxf(m[r], mt), mf = mn == -INFINITY ? 0.0f : mn;
            const float corr = exp2f(m[r] - mf);
            m[r] = mn;
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = exp2f(s[r][c] - mf);
                sum += s[r][c];
            }
            l[r] = l[r] * corr + sum;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[r][c][e] *= corr;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<float4*>(Ps + (tx * 4 + c) * (kBM + kPad) + ty * 4) =
                make_float4(s[0][c], s[1][c], s[2][c], s[3][c]);
        __syncthreads();  // the scores are done with K; P is written
        stage<T, false>(V + (size_t)j0 * a.ks.token, a.ks.token, valid, D, KV, D + kPad);
        __syncthreads();
#pragma unroll 2
        for (int k = 0; k < kBN; ++k) {
            const float4 p4 = *reinterpret_cast<const float4*>(Ps + k * (kBM + kPad) + ty * 4);
            const float p[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if (tx * 4 + c * 64 < D) {
                    const float4 v = *reinterpret_cast<const float4*>(KV + k * (D + kPad) + tx * 4 + c * 64);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        o[r][c][0] = fmaf(p[r], v.x, o[r][c][0]);
                        o[r][c][1] = fmaf(p[r], v.y, o[r][c][1]);
                        o[r][c][2] = fmaf(p[r], v.z, o[r][c][2]);
                        o[r][c][3] = fmaf(p[r], v.w, o[r][c][3]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int x = 1; x < 16; x <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], x);
        const int row = ty * 4 + r;
        if (row >= qrows) continue;
        const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
        uint8_t* po = a.O + (size_t)b * a.os.item + (size_t)h * a.os.head + (size_t)(i0 + row) * a.os.token;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = tx * 4 + c * 64;
            if (d < D) {
                const float f[4] = {o[r][c][0] * inv, o[r][c][1] * inv, o[r][c][2] * inv, o[r][c][3] * inv};
                store4<T>(po + d * (int)sizeof(T), f);
            }
        }
        if (a.lse && tx == 0)
            a.lse[((size_t)b * a.H + h) * a.len_q + i0 + row] =
                l[r] == 0.0f ? -INFINITY : ((m[r] == -INFINITY ? 0.0f : m[r]) + log2f(l[r])) * 0.693147180559945f;
    }
}

template <typename T, int NC>
int launch_simt(const SinkArgs& a, long long blocks, cudaStream_t st) {
    const size_t smem = simt_floats(a.D) * sizeof(float);
    if (cudaFuncSetAttribute(sink_simt_kernel<T, NC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    sink_simt_kernel<T, NC><<<(unsigned)blocks, kNT, smem, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}
template <typename T>
int launch_simt_d(const SinkArgs& a, long long blocks, cudaStream_t st) {
    if (a.D <= 64) return launch_simt<T, 1>(a, blocks, st);
    if (a.D <= 128) return launch_simt<T, 2>(a, blocks, st);
    return launch_simt<T, 4>(a, blocks, st);
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_sink_attention_workspace_size(size_t* bytes) {
    if (!bytes) return RKV_ERR_INVALID_ARG;
    *bytes = kWorkspaceHeader;
    return RKV_OK;
}

extern "C" int rkv_sink_attention(const void* Q, const void* K, const void* V, int dtype, int len_q, int len_k, int batch,
                                  int num_heads, int num_heads_kv, int dim_head, const rkv_row_strides* q_strides,
                                  const rkv_row_strides* kv_strides, const int* lens, int sinks, int window, void* O,
                                  const rkv_row_strides* o_strides, float* lse, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    if (dtype != RKV_F32 && dtype != RKV_BF16 && dtype != RKV_F16) return RKV_ERR_INVALID_ARG;
    if (len_q < 0 || len_k < len_q || batch < 0 || num_heads <= 0 || num_heads_kv <= 0 || num_heads % num_heads_kv != 0 ||
        dim_head <= 0 || sinks < 0 || window < 0)
        return RKV_ERR_INVALID_ARG;
    if (dim_head % 8 != 0 || dim_head > 256 || len_k > (1 << 30)) return RKV_ERR_UNSUPPORTED;
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
    if (!workspace || workspace_bytes < kWorkspaceHeader || (reinterpret_cast<uintptr_t>(workspace) & 15))
        return RKV_ERR_WORKSPACE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    a.Q = static_cast<const uint8_t*>(Q);
    a.K = static_cast<const uint8_t*>(K);
    a.V = static_cast<const uint8_t*>(V);
    a.O = static_cast<uint8_t*>(O);
    a.lse = lse;
    a.lens = lens;
    a.len_q = len_q;
    a.len_k = len_k;
    a.H = num_heads;
    a.HK = num_heads_kv;
    a.G = num_heads / num_heads_kv;
    a.D = dim_head;
    a.sinks = sinks < len_k ? sinks : len_k;      // no key lies behind len_k, so larger values
    a.window = window < len_k ? window : len_k;   // mean the same and could overflow below
    a.scale2 = 1.4426950408889634f / sqrtf((float)dim_head);
    a.err = static_cast<int*>(workspace);
    if (cudaMemsetAsync(a.err, 0, sizeof(int), st) != cudaSuccess) return RKV_ERR_CUDA;
    if (sink_tc_supported(dtype)) return launch_sink_tc(a, dtype, batch, st);
    a.qtiles = (len_q + kBM - 1) / kBM;
    const long long blocks = (long long)a.qtiles * num_heads * batch;
    if (blocks > 0x7FFFFFFFLL) return RKV_ERR_UNSUPPORTED;
    switch (dtype) {
        case RKV_F32: return launch_simt_d<float>(a, blocks, st);
        case RKV_BF16: return launch_simt_d<__nv_bfloat16>(a, blocks, st);
        default: return launch_simt_d<__half>(a, blocks, st);
    }
}
