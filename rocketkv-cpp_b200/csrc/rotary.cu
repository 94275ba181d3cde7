// rotary.cu -- rotary positions on rows of Q and K, and the paged append that
// applies them on the way.
//
// Pair i of a row, the columns (i, i + pairs) or (2 i, 2 i + 1), holds (x, y)
// and becomes (x cos t - y sin t, x sin t + y cos t) with t = f_i p, p the
// row's position on the pair's axis; columns from 2 pairs on are copied.
//
// The angle.  f_i is kept as turns per position in units of 2^-64, so that the
// 64-bit product with p wraps as the angle does: what is left is the fraction
// of a turn, exact for every 32-bit position but for f_i's own rounding
// (2^-65 |p| turns).  Its top 32 bits become the fp32 argument of sincospif: off
// by 2^-25 half turns for the rounding to fp32, 2^-31 for the bits below, 2^-33
// for f_i at most.  Products and sums are fp32 with one rounding to the rows'
// type at the end.
//
// Memory bounds it: every row is read and written once, six operations per
// pair.  A CTA has a tile of tokens; its threads ask for their first rows, form
// the tile's sines and cosines in shared memory meanwhile (one after the other:
// the code of eight side by side took longer to fetch than to run in small
// calls), then each takes a chunk (a vector of each half of the pairs) of one
// token and goes through the heads, so that a sine and a cosine serve up to 8 of
// them.  Where there are few tokens the heads are spread over more threads and
// CTAs.  bf16, 24/8 heads of 128: 4 x 4096 tokens on three axes (268 MB moved)
// 47.5 us, 5.6 TB/s, 0.86 of a copy; 512 tokens 4.5 us; the step of 64 sequences
// with its append 3.8 us.  Measured at 4 x 4096 tokens: sines and cosines in
// each thread's registers 78 us, all heads in one thread 61, products one by one
// in place of two 73; 2 heads ahead 50 and with the next two behind them 61.
#include <cmath>

#include "paged.cuh"
#include "rotary_grid.cuh"

namespace rkv {
namespace {

constexpr int kRotAhead = 4;  // heads whose rows are on their way per thread

// Rows of one tensor: element (b, h, i, d) at b item + h head + i token + d elements.
struct Rows {
    const uint8_t* src;
    uint8_t* dst;
    rkv_row_strides in, out;
};
struct RotArgs {
    const unsigned long long* freqs;
    const unsigned char* axes;
    const int* positions;  // [num_axes][batch][rows]
    int pairs, num_axes, D;
    int rows, batch;
    int H, HK, heads;      // heads of q, of k, and in all (with v's in the paged form)
    int tile, slots;       // tokens of a CTA, and its threads that share a token's chunk by heads
    int chunks, turned;    // of a row, and those with pairs
    Rows q, k, v;
    PagedView c;           // paged form: where k's and v's rows go
    const int* n_new;
};

// Two neighbouring elements in fp32, and back.
template <typename T>
__device__ __forceinline__ float2 widen(const T* e);
template <>
__device__ __forceinline__ float2 widen(const float* e) { return make_float2(e[0], e[1]); }
template <>
__device__ __forceinline__ float2 widen(const __nv_bfloat16* e) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(e);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <>
__device__ __forceinline__ float2 widen(const __half* e) { return __half22float2(*reinterpret_cast<const __half2*>(e)); }
template <typename T>
__device__ __forceinline__ void narrow(T* e, float2 x);
template <>
__device__ __forceinline__ void narrow(float* e, float2 x) { e[0] = x.x, e[1] = x.y; }
template <>
__device__ __forceinline__ void narrow(__nv_bfloat16* e, float2 x) { *reinterpret_cast<__nv_bfloat162*>(e) = __floats2bfloat162_rn(x.x, x.y); }
template <>
__device__ __forceinline__ void narrow(__half* e, float2 x) { *reinterpret_cast<__half2*>(e) = __floats2half2_rn(x.x, x.y); }
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void set(float& y, float x) { y = x; }
__device__ __forceinline__ void set(__nv_bfloat16& y, float x) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void set(__half& y, float x) { y = __float2half_rn(x); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
    T e[VEC];
};

// (x, y) to (x c - y s, x s + y c): two pairs of two vectors, one pair of neighbours, or one of single elements.
template <typename T, int VEC, bool INTER>
__device__ __forceinline__ void turn_chunk(Vec<T, VEC>& l, Vec<T, VEC>& h, const float (&cs)[VEC], const float (&sn)[VEC]) {
    if constexpr (VEC == 1) {
        const float x = to_f32(l.e[0]), y = to_f32(h.e[0]);
        set(l.e[0], fmaf(x, cs[0], -(y * sn[0])));
        set(h.e[0], fmaf(x, sn[0], y * cs[0]));
    } else if constexpr (INTER) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            T* p = (e < VEC / 2 ? l.e : h.e) + 2 * (e % (VEC / 2));
            const float2 v = widen(p);
            narrow(p, __ffma2_rn(make_float2(v.x, v.x), make_float2(cs[e], sn[e]),
                                 __fmul2_rn(make_float2(v.y, v.y), make_float2(-sn[e], cs[e]))));
        }
    } else {
#pragma unroll
        for (int e = 0; e < VEC; e += 2) {
            const float2 x = widen(l.e + e), y = widen(h.e + e), c = make_float2(cs[e], cs[e + 1]), s = make_float2(sn[e], sn[e + 1]);
            narrow(l.e + e, __ffma2_rn(x, c, __fmul2_rn(y, make_float2(-s.x, -s.y))));
            narrow(h.e + e, __ffma2_rn(x, s, __fmul2_rn(y, c)));
        }
    }
}

template <typename T, int VEC, bool INTER, bool PAGED>
__global__ void __launch_bounds__(kRotThreads, 3) rotary_kernel(const RotArgs a) {
    using V = Vec<T, VEC>;
    constexpr int U = kRotAhead;
    extern __shared__ float2 table[];  // [tile][pairs], cosine and sine
    const int b = blockIdx.z, tid = threadIdx.x;
    const long long i0 = (long long)blockIdx.x * a.tile;
    int n = a.rows, first = 0;  // rows of this item; token of row 0
    if (PAGED) {
        if (a.n_new) n = min(max(a.n_new[b], 0), n);
        if (i0 >= n) return;
        first = a.c.lens[b] - n;
    }
    const int chunk = tid % a.chunks, rest = tid / a.chunks;
    const long long i = i0 + rest % a.tile;
    const int step = a.slots * gridDim.y, slot = blockIdx.y * a.slots + rest / a.tile;
    const bool have = rest / a.tile < a.slots && i < n;
    // columns of the chunk's two vectors, and the pairs that they begin with; past the pairs the vectors that are
    // copied, the second of a chunk where there is one
    const bool turn = chunk < a.turned;
    const int rest_vecs = (a.D - 2 * a.pairs) / VEC, j = chunk - a.turned, half = (rest_vecs + 1) / 2;
    const int lo = turn ? (INTER && VEC == 1 ? 2 * chunk : chunk * VEC) : 2 * a.pairs + j * VEC;
    const int hi = turn ? (INTER && VEC == 1 ? lo + 1 : lo + a.pairs) : lo + half * VEC;
    const bool two = turn || j + half < rest_vecs;

    V l[U], h[U];
    const uint8_t* qs = a.q.src + b * a.q.in.item + i * a.q.in.token;
    const long long kv = b * a.k.in.item + i * a.k.in.token;
    auto fetch = [&](int h0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int g = h0 + u * step;
            if (!have || g >= a.heads) continue;
            const uint8_t* s = qs + g * a.q.in.head;
            if (g >= a.H) {
                g -= a.H;
                const bool isv = PAGED && g >= a.HK;
                s = (isv ? a.v.src : a.k.src) + kv + (isv ? g - a.HK : g) * a.k.in.head;
            }
            l[u] = *reinterpret_cast<const V*>(reinterpret_cast<const T*>(s) + lo);
            if (two) h[u] = *reinterpret_cast<const V*>(reinterpret_cast<const T*>(s) + hi);
        }
    };
    fetch(slot);
    long long page = -1;  // paged form: this row's place in K and V, head 0
    if (PAGED && have) {
        const long long t = first + i;
        if (t >= 0 && t < (long long)a.c.table_stride * a.c.page_size) page = paged_offset(a.c, b, 0, (int)t);
    }
#pragma unroll 2
    for (int x = tid; x < a.tile * a.pairs; x += kRotThreads) {
        const int row = x / a.pairs, pair = x - row * a.pairs;
        const int axis = a.axes ? a.axes[pair] : 0;
        float2 t = make_float2(1.0f, 0.0f);
        if (i0 + row < n && axis < a.num_axes) {
            const int p = PAGED && !a.positions ? (int)(first + i0 + row) : a.positions[((size_t)axis * a.batch + b) * a.rows + i0 + row];
            const unsigned long long ph = (unsigned long long)(long long)p * a.freqs[pair];
            sincospif((float)(int)(ph >> 32) * 0x1p-31f, &t.y, &t.x);
        }
        table[x] = t;
    }
    __syncthreads();
    if (!have) return;
    float cs[VEC], sn[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        // neighbouring columns: half of a chunk's pairs lie in each vector
        const int pair = INTER && VEC > 1 ? (e < VEC / 2 ? lo / 2 + e : hi / 2 + e - VEC / 2) : chunk * VEC + e;
        const float2 t = turn ? table[(int)(i - i0) * a.pairs + pair] : make_float2(1.0f, 0.0f);
        cs[e] = t.x;
        sn[e] = t.y;
    }
    uint8_t* qd = a.q.dst + b * a.q.out.item + i * a.q.out.token;
    uint8_t* kd = PAGED ? a.c.K + page : a.k.dst + b * a.k.out.item + i * a.k.out.token;
    const long long ks = PAGED ? a.c.head_stride : a.k.out.head;
    for (int h0 = slot;;) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int g = h0 + u * step;
            if (g >= a.heads) break;
            uint8_t* d = qd + g * a.q.out.head;
            bool isv = false;
            if (g >= a.H) {
                if (PAGED && page < 0) continue;
                g -= a.H;
                isv = PAGED && g >= a.HK;
                d = (isv ? a.c.V + page : kd) + (isv ? g - a.HK : g) * ks;
            }
            if (turn && !isv) turn_chunk<T, VEC, INTER>(l[u], h[u], cs, sn);
            *reinterpret_cast<V*>(reinterpret_cast<T*>(d) + lo) = l[u];
            if (two) *reinterpret_cast<V*>(reinterpret_cast<T*>(d) + hi) = h[u];
        }
        h0 += U * step;
        if (h0 >= a.heads) break;
        fetch(h0);
    }
}

template <typename T, int VEC, bool PAGED>
void launch_vec(const RotArgs& a, bool inter, dim3 grid, cudaStream_t st) {
    const size_t smem = sizeof(float2) * a.tile * a.pairs;  // at most 256 / chunks rows of pairs: 256 VEC entries, 16 KB
    if (inter) rotary_kernel<T, VEC, true, PAGED><<<grid, kRotThreads, smem, st>>>(a);
    else rotary_kernel<T, VEC, false, PAGED><<<grid, kRotThreads, smem, st>>>(a);
}
// Vectors of 16 or 8 bytes where the pairs and the addresses allow it, else single elements.
template <typename T, bool PAGED>
void launch_type(const RotArgs& a, int bytes, bool inter, dim3 grid, cudaStream_t st) {
    constexpr int E = 16 / (int)sizeof(T);
    if (bytes == 16) launch_vec<T, E, PAGED>(a, inter, grid, st);
    else if (bytes == 8) launch_vec<T, E / 2, PAGED>(a, inter, grid, st);
    else launch_vec<T, 1, PAGED>(a, inter, grid, st);
}

int rotary_check(const rkv_rotary* r, int dim_head) {
    if (!r || r->pairs <= 0 || r->num_axes <= 0 || dim_head <= 0) return RKV_ERR_INVALID_ARG;
    if (r->pairs > dim_head / 2 || !r->freqs || (reinterpret_cast<uintptr_t>(r->freqs) & 7)) return RKV_ERR_INVALID_ARG;
    if (dim_head % 8 != 0 || dim_head > 256 || r->num_axes > 256) return RKV_ERR_UNSUPPORTED;
    return RKV_OK;
}

// Strides as given, or rows, heads and items back to back; those of a dimension of one entry are not used and
// become 0.  Rows that are written must not meet (own).  al gathers what the alignment depends on.
bool set_strides(rkv_row_strides& out, const rkv_row_strides* s, long long rowb, int rows, int heads, int batch, bool own, uintptr_t& al) {
    out = s ? *s : rkv_row_strides{rowb * rows * heads, rowb * rows, rowb};
    if (batch <= 1) out.item = 0;
    if (heads <= 1) out.head = 0;
    if (rows <= 1) out.token = 0;
    if (out.item < 0 || out.head < 0 || out.token < 0) return false;
    if (own && ((batch > 1 && out.item < rowb) || (heads > 1 && out.head < rowb) || (rows > 1 && out.token < rowb))) return false;
    al |= (uintptr_t)out.item | (uintptr_t)out.head | (uintptr_t)out.token;
    return true;
}

template <bool PAGED>
int launch(RotArgs& a, const rkv_rotary* r, int dtype, uintptr_t al, cudaStream_t st) {
    const int es = elem_size(dtype);
    if (al & (es - 1)) return RKV_ERR_INVALID_ARG;
    a.freqs = r->freqs;
    a.axes = r->axes;
    a.pairs = r->pairs;
    a.num_axes = r->num_axes;
    const uintptr_t all = al | (uintptr_t)(r->pairs * es);
    const int bytes = (all & 15) == 0 ? 16 : (all & 7) == 0 ? 8 : es, vec = bytes / es;
    const RotGrid g = rotary_grid(a.D, a.pairs, vec, a.heads, a.rows, a.batch);
    a.turned = g.turned;
    a.chunks = g.chunks;
    a.slots = g.slots;
    a.tile = g.tile;
    const dim3 grid((unsigned)g.tiles, (unsigned)g.split, a.batch);
    switch (dtype) {
        case RKV_F32: launch_type<float, PAGED>(a, bytes, r->interleaved != 0, grid, st); break;
        case RKV_BF16: launch_type<__nv_bfloat16, PAGED>(a, bytes, r->interleaved != 0, grid, st); break;
        default: launch_type<__half, PAGED>(a, bytes, r->interleaved != 0, grid, st); break;
    }
    return launched();
}

}  // namespace
}  // namespace rkv

using namespace rkv;

extern "C" int rkv_rotary_frequencies(const double* radians, int pairs, unsigned long long* freqs) {
    if (!radians || !freqs || pairs < 0) return RKV_ERR_INVALID_ARG;
    for (int i = 0; i < pairs; ++i)
        if (!(radians[i] > -0x1p64 && radians[i] < 0x1p64)) return RKV_ERR_INVALID_ARG;
    // floor(2^192 / 2 pi), low word first.  A double is an integer m < 2^53 times 2^e, e <= 11; the product of m with
    // these 192 bits is off by m at most, and its bits from 128 - e on (117 or more) are the steps of 2^-64 turns.
    constexpr unsigned long long inv[3] = {0x36d8a5664f10e410ull, 0x7f09d5f47d4d3770ull, 0x28be60db9391054aull};
    for (int i = 0; i < pairs; ++i) {
        int e = 0;
        const double x = frexp(radians[i] < 0 ? -radians[i] : radians[i], &e);
        const unsigned long long m = (unsigned long long)ldexp(x, 53);
        unsigned long long p[5] = {};
        for (int k = 0; k < 3; ++k) {
            const unsigned __int128 y = (unsigned __int128)m * inv[k] + p[k];
            p[k] = (unsigned long long)y;
            p[k + 1] = (unsigned long long)(y >> 64);
        }
        auto word = [&](int at) {  // 64 bits from bit `at` on; those from 256 on are 0
            const int w = at / 64, r = at % 64;
            return w > 3 ? 0ull : r ? p[w] >> r | p[w + 1] << (64 - r) : p[w];
        };
        const int at = 128 - (e - 53);
        const unsigned long long f = word(at) + (word(at - 1) & 1);  // rounded; a whole turn is none
        freqs[i] = radians[i] < 0 ? 0 - f : f;
    }
    return RKV_OK;
}

extern "C" int rkv_rotate(const rkv_rotary* rotary, const int* positions, const void* q, void* q_out, int num_heads, const void* k,
                          void* k_out, int num_heads_kv, int dtype, int dim_head, int len, int batch, const rkv_row_strides* q_strides,
                          const rkv_row_strides* q_out_strides, const rkv_row_strides* k_strides, const rkv_row_strides* k_out_strides,
                          void* stream) {
    const int rc = rotary_check(rotary, dim_head);
    if (rc) return rc;
    if (!paged_dtype(dtype) || num_heads < 0 || num_heads_kv < 0 || len < 0 || batch < 0) return RKV_ERR_INVALID_ARG;
    const long long heads = (long long)num_heads + num_heads_kv;
    if (heads > 0x7FFFFFF) return RKV_ERR_UNSUPPORTED;
    if (heads == 0 || len == 0 || batch == 0) return RKV_OK;
    if (batch > 65535) return RKV_ERR_UNSUPPORTED;
    if (!positions || (num_heads > 0 && (!q || !q_out)) || (num_heads_kv > 0 && (!k || !k_out))) return RKV_ERR_INVALID_ARG;
    RotArgs a{};
    a.positions = positions;
    a.D = dim_head;
    a.rows = len;
    a.batch = batch;
    a.H = num_heads;
    a.HK = num_heads_kv;
    a.heads = (int)heads;
    a.q.src = static_cast<const uint8_t*>(q);
    a.q.dst = static_cast<uint8_t*>(q_out);
    a.k.src = static_cast<const uint8_t*>(k);
    a.k.dst = static_cast<uint8_t*>(k_out);
    const long long rowb = (long long)dim_head * elem_size(dtype);
    uintptr_t al = 0;
    if (num_heads > 0) {
        al |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out);
        if (!set_strides(a.q.in, q_strides, rowb, len, num_heads, batch, false, al) ||
            !set_strides(a.q.out, q_out_strides, rowb, len, num_heads, batch, true, al))
            return RKV_ERR_INVALID_ARG;
    }
    if (num_heads_kv > 0) {
        al |= reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out);
        if (!set_strides(a.k.in, k_strides, rowb, len, num_heads_kv, batch, false, al) ||
            !set_strides(a.k.out, k_out_strides, rowb, len, num_heads_kv, batch, true, al))
            return RKV_ERR_INVALID_ARG;
    }
    return launch<false>(a, rotary, dtype, al, static_cast<cudaStream_t>(stream));
}

extern "C" int rkv_paged_append_rotated(const rkv_paged_cache* cache, const rkv_rotary* rotary, const int* positions, const void* k,
                                        const void* v, const rkv_row_strides* kv_strides, int n_rows, int batch, const int* n_new,
                                        const void* q, const rkv_row_strides* q_strides, void* q_out,
                                        const rkv_row_strides* q_out_strides, int num_heads, void* stream) {
    int rc = paged_check(cache, true, batch);
    if (!rc) rc = rotary_check(rotary, cache->dim_head);
    if (rc) return rc;
    if (n_rows < 0 || batch < 0 || num_heads < 0) return RKV_ERR_INVALID_ARG;
    if (num_heads > 0x3FFFFFF || cache->num_heads_kv > 0x3FFFFFF) return RKV_ERR_UNSUPPORTED;
    if (n_rows == 0 || batch == 0) return RKV_OK;
    if (batch > 65535) return RKV_ERR_UNSUPPORTED;
    if (!k || !v || (num_heads > 0 && (!q || !q_out))) return RKV_ERR_INVALID_ARG;
    RotArgs a{};
    a.positions = positions;
    a.D = cache->dim_head;
    a.rows = n_rows;
    a.batch = batch;
    a.H = num_heads;
    a.HK = cache->num_heads_kv;
    a.heads = a.H + 2 * a.HK;
    a.n_new = n_new;
    a.c = paged_view(*cache);  // 16-byte aligned throughout
    a.q.src = static_cast<const uint8_t*>(q);
    a.q.dst = static_cast<uint8_t*>(q_out);
    a.k.src = static_cast<const uint8_t*>(k);
    a.v.src = static_cast<const uint8_t*>(v);
    const long long rowb = (long long)a.D * elem_size(cache->dtype);
    uintptr_t al = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
    if (!set_strides(a.k.in, kv_strides, rowb, n_rows, a.HK, batch, false, al)) return RKV_ERR_INVALID_ARG;
    if (num_heads > 0) {
        al |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out);
        if (!set_strides(a.q.in, q_strides, rowb, n_rows, num_heads, batch, false, al) ||
            !set_strides(a.q.out, q_out_strides, rowb, n_rows, num_heads, batch, true, al))
            return RKV_ERR_INVALID_ARG;
    }
    return launch<true>(a, rotary, cache->dtype, al, static_cast<cudaStream_t>(stream));
}
