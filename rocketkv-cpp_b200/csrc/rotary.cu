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
// (2^-65 |p| turns).  Its top 32 bits become the fp32 argument of sincospif (off
// by 2^-25 half turns at most).  Products and sums are fp32 with one rounding
// to the rows' type at the end.
//
// Memory bounds it: every row is read and written once, six operations per
// pair.  A thread has one chunk (a vector of each half of the pairs) of one
// token and goes through the heads, so that a sine and a cosine serve all of
// them; where there are few tokens the heads are spread over more threads.
#include "paged.cuh"

namespace rkv {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotHeads = 4;                    // heads whose rows are on their way per thread
constexpr long long kRotFull = 148LL * 1024;    // threads that the heads are spread for

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
    int slots;             // threads that share a token's chunk, by heads
    int chunks, turned;    // of a row, and those with pairs
    Rows q, k, v;
    PagedView c;           // paged form: where k's and v's rows go
    const int* n_new;
};

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
    T e[VEC];
};

template <typename T, int VEC, bool INTER, bool PAGED>
__global__ void __launch_bounds__(kRotThreads) rotary_kernel(const RotArgs a) {
    using V = Vec<T, VEC>;
    constexpr int U = kRotHeads;
    const int b = blockIdx.y;
    const unsigned x = blockIdx.x * kRotThreads + threadIdx.x;
    const unsigned rest = x / (unsigned)a.chunks, chunk = x - rest * a.chunks;
    const int slot = (int)(rest / (unsigned)a.rows), i = (int)(rest - (unsigned)slot * a.rows);
    if (slot >= a.slots) return;
    int first = 0;          // token of row 0
    long long page = -1;    // paged form: this row's place in K and V, head 0
    if (PAGED) {
        const int n = a.n_new ? min(max(a.n_new[b], 0), a.rows) : a.rows;
        if (i >= n) return;
        first = a.c.lens[b] - n;
        const long long t = (long long)first + i;
        if (t >= 0 && t < (long long)a.c.table_stride * a.c.page_size) page = paged_offset(a.c, b, 0, (int)t);
    }
    // columns of the chunk's two vectors; one vector where nothing is turned
    const bool turn = (int)chunk < a.turned;
    const int tail = 2 * a.pairs + ((int)chunk - a.turned) * VEC;
    const int lo = !turn ? tail : INTER ? 2 * (int)chunk * VEC : (int)chunk * VEC;
    const int hi = INTER ? lo + VEC : lo + a.pairs;

    V xl[U], xh[U];
    T* to[U];
    auto fetch = [&](int h0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int h = h0 + u * a.slots;
            to[u] = nullptr;
            if (h >= a.heads) continue;
            const bool isq = h < a.H;
            if (!isq) h -= a.H;
            const bool isv = PAGED && !isq && h >= a.HK;
            if (isv) h -= a.HK;
            const Rows& r = isq ? a.q : a.k;
            const uint8_t* src = isv ? a.v.src : r.src;
            if (PAGED && !isq) {
                if (page < 0) continue;
                to[u] = reinterpret_cast<T*>((isv ? a.c.V : a.c.K) + page + (long long)h * a.c.head_stride);
            } else {
                to[u] = reinterpret_cast<T*>(r.dst + (long long)b * r.out.item + (long long)h * r.out.head + (long long)i * r.out.token);
            }
            const T* s = reinterpret_cast<const T*>(src + (long long)b * r.in.item + (long long)h * r.in.head + (long long)i * r.in.token);
            xl[u] = *reinterpret_cast<const V*>(s + lo);
            if (turn) xh[u] = *reinterpret_cast<const V*>(s + hi);
        }
    };
    fetch(slot);
    float cs[VEC], sn[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        cs[e] = 1.0f;
        sn[e] = 0.0f;
        if (turn) {
            const int pair = (int)chunk * VEC + e;
            const int axis = a.axes ? a.axes[pair] : 0;
            if (axis < a.num_axes) {
                const int p = PAGED && !a.positions ? first + i : a.positions[((size_t)axis * a.batch + b) * a.rows + i];
                const unsigned long long ph = (unsigned long long)(long long)p * a.freqs[pair];
                sincospif((float)(int)(ph >> 32) * 0x1p-31f, &sn[e], &cs[e]);
            }
        }
    }
    for (int h0 = slot; h0 < a.heads; h0 += U * a.slots) {
        if (h0 != slot) fetch(h0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (!to[u]) continue;
            if (turn && !(PAGED && h0 + u * a.slots >= a.H + a.HK)) {
                V yl, yh;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    // pair e of the chunk: element e of both vectors, or two neighbours of one
                    const bool up = INTER && VEC > 1 && e >= VEC / 2;
                    const int j = INTER && VEC > 1 ? 2 * (e % (VEC / 2 > 0 ? VEC / 2 : 1)) : e;
                    const float p = to_f32(up ? xh[u].e[j] : xl[u].e[j]);
                    const float q = to_f32(INTER && VEC > 1 ? (up ? xh[u].e[j + (VEC > 1)] : xl[u].e[j + (VEC > 1)]) : xh[u].e[j]);
                    const T r = from_f32<T>(fmaf(p, cs[e], -q * sn[e])), s = from_f32<T>(fmaf(p, sn[e], q * cs[e]));
                    if (INTER && VEC > 1) {
                        if (up) yh.e[j] = r, yh.e[j + (VEC > 1)] = s;
                        else yl.e[j] = r, yl.e[j + (VEC > 1)] = s;
                    } else {
                        yl.e[j] = r;
                        yh.e[j] = s;
                    }
                }
                xl[u] = yl;
                xh[u] = yh;
            }
            *reinterpret_cast<V*>(to[u] + lo) = xl[u];
            if (turn) *reinterpret_cast<V*>(to[u] + hi) = xh[u];
        }
    }
}

template <typename T, int VEC, bool PAGED>
void launch_vec(const RotArgs& a, bool inter, dim3 grid, cudaStream_t st) {
    if (inter) rotary_kernel<T, VEC, true, PAGED><<<grid, kRotThreads, 0, st>>>(a);
    else rotary_kernel<T, VEC, false, PAGED><<<grid, kRotThreads, 0, st>>>(a);
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
    a.turned = a.pairs / vec;
    a.chunks = a.turned + (a.D - 2 * a.pairs) / vec;
    const long long per = (long long)a.rows * a.chunks;
    long long slots = (kRotFull + per * a.batch - 1) / (per * a.batch);
    if (slots > a.heads) slots = a.heads;
    const long long each = (a.heads + slots - 1) / slots;
    slots = (a.heads + each - 1) / each;
    a.slots = (int)slots;
    const long long threads = per * slots;
    if (threads > 0x7FFFFFFFLL - kRotThreads) return RKV_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)((threads + kRotThreads - 1) / kRotThreads), a.batch);
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
        if (!(radians[i] >= -1e300 && radians[i] <= 1e300)) return RKV_ERR_INVALID_ARG;
    for (int i = 0; i < pairs; ++i) {
        long double t = (long double)radians[i] / 6.283185307179586476925286766559006L;
        t -= __builtin_floorl(t);
        const long double s = __builtin_rintl(t * 18446744073709551616.0L);
        freqs[i] = s >= 18446744073709551616.0L ? 0ull : (unsigned long long)s;  // a whole turn
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
