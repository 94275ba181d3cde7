// sink_attn_tc.cu -- the sink-window prefill attention of 16-bit inputs on the
// tcgen05 tensor cores: sink_tc_kernel for dim_head <= 128, sink_wide_kernel
// for up to 256.
//
// A CTA takes two units -- a unit is 128 queries of one query head -- of one
// KV head, so that both use every K and V tile that is loaded: 128 keys at a
// time, S = Q K^T into tensor memory, P = 2^(S - m) rounded to the inputs'
// type back into tensor memory in S's place, O += P V.  While one unit's
// softmax runs on its four warps (a thread per query row), the tensor cores
// work on the other unit.
//
//   warp 0       copies Q and the K, V tiles (one TMA box per 64 columns) into
//                shared memory; a stage of the ring holds the V of a tile and
//                the K of the next, which the products take one after the other
//   warp 1       issues the products: per tile and unit P V, then the next S
//   warps 4-7, 8-11   softmax of unit 0, 1, and their output rows
//
// Two roundings to 16 bits: P (relative half a step of the type, as the
// products take both operands in one type; two parts of P would double P V) and
// the output.  Error against 64 bits, bf16: 2.1e-3, 1.6e-3 with the output's
// rounding alone.  Scores, m, l and the accumulator are fp32.  The accumulator
// is rescaled only when a row's largest score has grown by more than 2^8 since
// its last rescale: P stays below 2^8 then (2^15 in fp16, see kLift), which both
// types hold, and O and l carry the same factor.
//
// What bounds it.  24/8 heads of 128, causal: 4096 tokens 104 us (994
// TFLOP/s), 8192 tokens under a window of 2048 185-200 us (900-970) cold and
// 213 in loops of seconds.  A pair of tiles takes 3300 cycles, 2048 of them
// products at their full rate: a unit's chain is 2100 of softmax, then 1200 of
// its last products with P and its next scores, and the two units fill each
// other's gaps only in part (the tensor and the exponentials' pipe are both
// active 55 % of the time).  Power comes on top: some milliseconds of it bring
// the GPU to its 1000 W cap (1.74 GHz sampled, of 1.97).  Shortening one part
// of the chain gives little: leaving out the maximum or the exponentials (wrong
// results, to see) makes it 3 and 9 % faster.  With 128 columns the kernel
// spills 76 bytes a thread.  Measured and not kept, beside 186 us: 64 keys a
// tile with two score buffers 237 (200 with a second issuing warp for P V); one
// thread that issues everything 224; two issuing warps 213; 16 softmax warps
// 197; P handed over whole 197; the maximum taken under the first half's
// exponentials 203.
#include "attn_tc.cuh"
#include "sink_attn.cuh"

namespace rkv {
namespace {

constexpr int kTile = 128;            // queries of a unit, keys of a tile
constexpr int kThreads = 384;
constexpr int kBlk = kTile * 128;     // bytes of a 128-row block of 64 columns

__host__ __device__ constexpr int stages(int kb) { return kb == 1 ? 4 : 2; }  // of a V and a K tile

// 64 columns of a warp's 32 output rows (a row per lane in o) times inv, through 4 KB of shared memory, so that
// eight lanes write 128 bytes of a row (a lane per row wrote half sectors); chunk c of row r is kept at c ^ (r % 8).
template <bool BF>
__device__ __forceinline__ void write_rows(uint8_t* so, const uint32_t* o, float inv, uint32_t rows_ok, uint8_t* po, int row0,
                                           long long stride, int col0, int D, int lane) {
#pragma unroll
    for (int v = 0; v < 8; ++v) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            w[e] = pack2<BF>(__uint_as_float(o[v * 8 + 2 * e]) * inv, __uint_as_float(o[v * 8 + 2 * e + 1]) * inv);
        *reinterpret_cast<uint4*>(so + lane * 128 + ((v ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const int r = x * 4 + (lane >> 3), v = lane & 7;
        const uint4 y = *reinterpret_cast<const uint4*>(so + r * 128 + ((v ^ (r & 7)) << 4));
        if (((rows_ok >> r) & 1u) && col0 + v * 8 < D)
            *reinterpret_cast<uint4*>(po + (size_t)(row0 + r) * stride + (col0 + v * 8) * 2) = y;
    }
    __syncwarp();
}

// The same for 32 columns in fp32, of a part's rows (back to back).
__device__ __forceinline__ void write_part(uint8_t* so, const uint32_t* o, uint32_t rows_ok, float* po, int col0, int D, int lane) {
#pragma unroll
    for (int v = 0; v < 8; ++v)
        *reinterpret_cast<uint4*>(so + lane * 128 + ((v ^ (lane & 7)) << 4)) = make_uint4(o[v * 4], o[v * 4 + 1], o[v * 4 + 2], o[v * 4 + 3]);
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const int r = x * 4 + (lane >> 3), v = lane & 7;
        const uint4 y = *reinterpret_cast<const uint4*>(so + r * 128 + ((v ^ (r & 7)) << 4));
        if (((rows_ok >> r) & 1u) && col0 + v * 4 < D) *reinterpret_cast<uint4*>(po + (size_t)r * D + col0 + v * 4) = y;
    }
    __syncwarp();
}

// A pair of units: (query tile, head of the group) numbers u0 and u0 + 1 of one KV head.
struct Pair {
    int b, hk, u0, nu;
    SinkRange rg;
    int tiles, part;
};
// Item i of the list, the latest queries (the longest rows) first, the parts of their keys side by side.
__device__ __forceinline__ Pair pair_of(const SinkArgs& a, int i, int per) {
    const int units = a.G * a.qtiles, pairs = (units + 1) / 2;
    Pair p;
    p.part = i % a.parts;
    i /= a.parts;
    p.u0 = 2 * (pairs - 1 - i / per);
    const int bh = i % per;
    p.b = bh / a.HK;
    p.hk = bh - p.b * a.HK;
    p.nu = min(2, units - p.u0);
    const int qt0 = p.u0 / a.G, qt1 = (p.u0 + p.nu - 1) / a.G;
    p.rg = sink_range(a, p.b, qt0 * kTile, (qt1 - qt0 + 1) * kTile, kTile);
    p.tiles = p.rg.part(p.part, a.parts);
    return p;
}
// A CTA's items: the first by its number, then the next that no CTA has taken, so that CTAs with short ones take
// more (causal, 4096 tokens: 104 us, 107 with a fixed order to and fro).  The copying warp draws them and hands them to the other roles through two places in shared memory.
struct Items {
    uint64_t full[2], empty[2];
    volatile int at[2];
    __device__ void init(int readers) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], readers);
        }
    }
    // the copying warp's
    __device__ int draw(int items, int* err, int lane) {
        int n = 0;
        if (items > (int)gridDim.x && lane == 0) n = (int)atomicAdd(reinterpret_cast<unsigned*>(err) + kSinkTicket, 1u);
        return items > (int)gridDim.x ? (int)gridDim.x + __shfl_sync(0xffffffffu, n, 0) : items;
    }
    __device__ bool put(int k, int item, int* err, volatile int* abort, int lane) {
        if (k >= 2 && !warp_wait(&empty[k & 1], (uint32_t)(((k >> 1) - 1) & 1), err, abort)) return false;
        if (lane == 0) {
            at[k & 1] = item;
            mbar_arrive1(&full[k & 1]);
        }
        __syncwarp();
        return true;
    }
    // a reading warp's k-th item; past every item where the wait gave up
    __device__ int get(int k, int* err, volatile int* abort, int lane) {
        if (!warp_wait(&full[k & 1], (uint32_t)((k >> 1) & 1), err, abort)) return 0x7FFFFFFF;
        const int item = at[k & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive1(&empty[k & 1]);
        return item;
    }
};

struct TcBars {
    uint64_t q_full, q_empty, o_full, drained;
    uint64_t s_full[2], p_half[2], p_ready[2], o_empty[2];  // of a unit
    uint64_t full[4], empty[4];
    Items items;
    uint32_t tmem;
    int abort;
};

// KB: blocks of 64 columns (dim_head <= 64 KB; columns behind dim_head are
// filled with zeros by the copies).  One CTA per SM goes through its items
// (pairs of units); every role keeps its own count of barrier phases over all
// of them, so the copies, and the first scores, of an item run under the end
// of the one before.
template <int KB, bool BF>
__global__ void __launch_bounds__(kThreads, 1)
    sink_tc_kernel(const SinkArgs a, const int items, const int per, const __grid_constant__ CUtensorMap tq,
                   const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv) {
    constexpr int NS = stages(KB);
    constexpr uint32_t kOne = KB * kBlk, kStage = 2 * kOne;  // a tile of Q, V or K; the V of a tile, then the K of the next
    constexpr uint32_t kColO = 256;  // tensor memory: S0, S1 (128 columns each), O0, O1 (64 KB each)
    extern __shared__ uint8_t smem_raw[];
    asm volatile("griddepcontrol.launch_dependents;");  // a join may be scheduled (it waits for this grid)
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    TcBars& B = *reinterpret_cast<TcBars*>(sm);
    volatile int* abort_flag = &B.abort;
    uint8_t* sq = sm + 1024;
    uint8_t* ring = sq + 2 * kOne;
    uint8_t* stage_o = ring + NS * kStage;  // 4 KB per softmax warp
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        mbar_init(&B.q_full, 1);
        mbar_init(&B.q_empty, 1);
        mbar_init(&B.o_full, 1);
        mbar_init(&B.drained, 1);
        B.items.init(9);
        if (blockIdx.x == 0 && items <= (int)gridDim.x) *a.err = 0;
        for (int u = 0; u < 2; ++u) {
            mbar_init(&B.s_full[u], 1);
            mbar_init(&B.p_half[u], 4);
            mbar_init(&B.p_ready[u], 4);
            mbar_init(&B.o_empty[u], 4);
        }
        for (int i = 0; i < NS; ++i) {
            mbar_init(&B.full[i], 1);
            mbar_init(&B.empty[i], 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(&B.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = B.tmem;

    if (warp < 4) {
        // 88 * 128 + 208 * 256 registers are the 168 * 384 of the launch
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == 0) {
            // stage number q of the ring: an item of t tiles takes t + 1, V of tile j - 1 and K of tile j in stage j
            int q = 0, nq = 0;
            bool ok = true;
            auto copy = [&](const Pair& P, int j) {
                const int s = q % NS;
                if (q >= NS && !(ok = warp_wait(&B.empty[s], (uint32_t)((q / NS - 1) & 1), a.err, abort_flag))) return;
                mbar_arrive_expect_tx_w(&B.full[s], j == 0 || j == P.tiles ? kOne : kStage);
                for (int kb = 0; kb < KB && j < P.tiles; ++kb)
                    tma_load_4d_w(ring + s * kStage + kOne + kb * kBlk, &tk, kb * 64, P.rg.tile(j) * kTile, P.hk, P.b, &B.full[s]);
                for (int kb = 0; kb < KB && j > 0; ++kb)
                    tma_load_4d_w(ring + s * kStage + kb * kBlk, &tv, kb * 64, P.rg.tile(j - 1) * kTile, P.hk, P.b, &B.full[s]);
                ++q;
            };
            int it = blockIdx.x;
            for (int k = 0; ok; ++k, it = B.items.draw(items, a.err, lane)) {
                if (!B.items.put(k, it, a.err, abort_flag, lane)) break;
                if (it >= items) break;
                const Pair P = pair_of(a, it, per);
                if (P.tiles == 0) continue;
                copy(P, 0);
                if (!ok || (nq > 0 && !(ok = warp_wait(&B.q_empty, (uint32_t)((nq - 1) & 1), a.err, abort_flag)))) break;
                mbar_arrive_expect_tx_w(&B.q_full, P.nu * kOne);
                for (int u = 0; u < P.nu; ++u)
                    for (int kb = 0; kb < KB; ++kb)
                        tma_load_4d_w(sq + u * kOne + kb * kBlk, &tq, kb * 64, (P.u0 + u) / a.G * kTile,
                                      P.hk * a.G + (P.u0 + u) % a.G, P.b, &B.q_full);
                ++nq;
                for (int j = 1; j <= P.tiles && ok; ++j) copy(P, j);
            }
            // every copy has landed before the CTA may end
            if (nq > 0) mbar_wait_bounded(&B.q_full, (uint32_t)((nq - 1) & 1), a.err);
            for (int s = 0; s < min(q, NS); ++s) mbar_wait_bounded(&B.full[s], (uint32_t)(((q - 1 - s) / NS) & 1), a.err);
        } else if (warp == 1) {
            const uint32_t ids = mma_idesc(BF ? 1u : 0u, kTile);
            const uint32_t idv = mma_idesc(BF ? 1u : 0u, KB * 64) | (1u << 16);  // B with N contiguous
            const uint64_t qd = mma_desc_sw128(smem_u32(sq)), kd = mma_desc_sw128(smem_u32(ring) + kOne);
            const uint64_t vd = v_desc(smem_u32(ring), kBlk);
            auto scores = [&](int u, int slot) {
                const uint64_t da = qd + (uint32_t)(u * (kOne >> 4)), db = kd + (uint32_t)(slot * (kStage >> 4));
#pragma unroll
                for (int ks = 0; ks < KB * 4; ++ks) {
                    const uint32_t o = ((ks >> 2) * kBlk + (ks & 3) * 32) >> 4;
                    mma_ss(tbase + u * 128, da + o, db + o, ids, ks > 0);
                }
                mma_commit_w(&B.s_full[u]);
            };
            int q = 0, nq = 0;                  // stages, items
            uint32_t tiles_ph = 0, out_ph = 0;  // a bit per unit: parity of its tiles and of its items
            uint32_t used = 0;                  // the unit's output columns have been written before
            bool ok = true;
            auto wait = [&](uint64_t* bar, int n) { return ok = warp_wait(bar, (uint32_t)(n & 1), a.err, abort_flag); };
            for (int k = 0; ok; ++k) {
                const int it = B.items.get(k, a.err, abort_flag, lane);
                if (it >= items) break;
                const Pair P = pair_of(a, it, per);
                if (P.tiles == 0) continue;
                if (!wait(&B.q_full, nq) || !wait(&B.full[q % NS], q / NS)) break;
                ++nq;
                tc_fence_after();
                scores(0, q % NS);
                if (P.nu > 1) scores(1, q % NS);
                mma_commit_w(&B.empty[q % NS]);
                if (P.tiles == 1) mma_commit_w(&B.q_empty);
                ++q;
                for (int j = 0; j < P.tiles && ok; ++j, ++q) {
                    const int slot = q % NS;
                    const uint64_t vdj = vd + (uint32_t)(slot * (kStage >> 4));
                    if (!wait(&B.full[slot], q / NS)) break;
                    const int behind = P.rg.n - P.rg.tile(j) * kTile;  // keys of the tile that exist
                    if (behind < kTile && P.rg.n < a.len_k) {
                        // the padding behind a sequence's end may hold anything, and 0 * NaN is NaN
                        uint8_t* vt = ring + slot * kStage;
                        for (int e = lane; e < (kTile - behind) * 8; e += 32)
#pragma unroll
                            for (int kb = 0; kb < KB; ++kb)
                                *reinterpret_cast<uint4*>(vt + kb * kBlk + behind * 128 + e * 16) = make_uint4(0, 0, 0, 0);
                        fence_proxy_async();
                        __syncwarp();
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u >= P.nu) break;
                        if (j == 0) {  // the output rows of the unit before have been read
                            if ((used >> u) & 1u) {
                                if (!wait(&B.o_empty[u], out_ph >> u)) break;
                                out_ph ^= 1u << u;
                            }
                            used |= 1u << u;
                        }
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            if (!wait(half ? &B.p_ready[u] : &B.p_half[u], tiles_ph >> u)) break;
                            tc_fence_after();
#pragma unroll
                            for (int ks = half * 4; ks < half * 4 + 4; ++ks)
                                mma_ts(tbase + kColO + u * (KB * 64), tbase + u * 128 + ks * 8, vdj + ks * 128, idv,
                                       (j | ks) > 0);
                        }
                        if (!ok) break;
                        tiles_ph ^= 1u << u;
                        if (j + 1 < P.tiles) scores(u, slot);
                    }
                    mma_commit_w(&B.empty[slot]);
                    if (j + 2 == P.tiles) mma_commit_w(&B.q_empty);
                }
                if (ok) mma_commit_w(&B.o_full);
            }
            // the products have ended before the tensor memory is freed
            mma_commit_w(&B.drained);
            mbar_wait_bounded(&B.drained, 0, a.err);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int u = (warp >> 2) - 1, q4 = warp & 3, row = q4 * 32 + lane;
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        const uint32_t ts = tbase + u * 128 + lane_off, to = tbase + kColO + u * (KB * 64) + lane_off;
        const float2 sc = make_float2(a.scale2, a.scale2);
        int nt = 0, ni = 0;  // tiles of this unit, items
        bool ok = true;
        for (int k = 0; ok; ++k) {
            const int it = B.items.get(k, a.err, abort_flag, lane);
            if (it >= items) break;
            const Pair P = pair_of(a, it, per);
            if (P.tiles > 0) ++ni;
            if (u >= P.nu) continue;
            const int qt = (P.u0 + u) / a.G, h = P.hk * a.G + (P.u0 + u) % a.G;
            const int p0 = qt * kTile + a.len_k - a.len_q, p = p0 + row, n = P.rg.n;
            const int i = qt * kTile + row;
            const bool real = i < a.len_q && p < n;
            const size_t prow = (((size_t)P.part * a.batch + P.b) * a.H + h) * a.len_q + i;  // this row of the part
            if (P.tiles == 0) {
                if (a.parts > 1 && real) a.part_ml[prow] = make_float2(-INFINITY, 0.0f);
                continue;
            }
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < P.tiles; ++j, ++nt) {
                if (!(ok = warp_wait(&B.s_full[u], (uint32_t)(nt & 1), a.err, abort_flag))) break;
                tc_fence_after();
                uint32_t r[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) ld32_async(ts + c * 32, r + c * 32);
                wait_ld();
#pragma unroll
                for (int c = 0; c < 4; ++c) pin32(r + c * 32);
                const int j0 = P.rg.tile(j) * kTile;
                const bool whole = j0 + kTile - 1 <= p0 && j0 + kTile <= n &&
                                   (a.window <= 0 || j0 > p0 + kTile - 1 - a.window || j0 + kTile <= a.sinks);
                if (!whole) {
                    const int hi = min(p, n - 1) - j0 + 1, lo = a.window > 0 ? p - a.window + 1 - j0 : 0, sk = a.sinks - j0;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {  // a bit per column
                        const uint32_t see = below(hi - 32 * w) & (~below(lo - 32 * w) | below(sk - 32 * w));
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!(see & (1u << c))) r[32 * w + c] = 0xFF800000u;  // -inf
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 128; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(r[c]), __uint_as_float(r[c + 1]));
                const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                const bool need = (mt - m) * a.scale2 > kGrow;  // true for a row's first key, false while it has none
                if (__any_sync(0xffffffffu, need)) {
                    const float corr = need ? ex2_approx((m - mt) * a.scale2) : 1.0f;
                    l *= corr;
                    if (need) m = mt;
                    if (j > 0) {  // the products up to here are complete: this tile's scores were issued behind them
#pragma unroll 1
                        for (int c = 0; c < KB * 2; ++c) {
                            uint32_t o[32];
                            ld32_async(to + c * 32, o);
                            wait_ld();
                            pin32(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                            st32(to + c * 32, o);
                        }
                    }
                }
                const float ms = (m == -INFINITY ? 0.0f : m) * a.scale2 - kLift<BF>;
                const float2 nm = make_float2(-ms, -ms);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int half = 0; half < 2; ++half) {  // the products of the first 64 keys start under the second's exponentials
#pragma unroll
                    for (int c = half * 32; c < half * 32 + 32; ++c) {
                        float2 x = __ffma2_rn(make_float2(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1])), sc, nm);
                        x.x = ex2_approx(x.x);
                        x.y = ex2_approx(x.y);
                        sum[c & 1] = __fadd2_rn(sum[c & 1], x);
                        r[c] = pack2<BF>(x.x, x.y);
                    }
                    st32(ts + half * 32, r + half * 32);
                    wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive1(half ? &B.p_ready[u] : &B.p_half[u]);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            if (!ok || !(ok = warp_wait(&B.o_full, (uint32_t)((ni - 1) & 1), a.err, abort_flag))) break;
            tc_fence_after();
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint8_t* po = a.O + (size_t)P.b * a.os.item + (size_t)h * a.os.head;
            uint32_t o[KB * 64];
#pragma unroll
            for (int c = 0; c < KB * 2; ++c) ld32_async(to + c * 32, o + c * 32);
            wait_ld();
#pragma unroll
            for (int c = 0; c < KB * 2; ++c) pin32(o + c * 32);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive1(&B.o_empty[u]);
            uint8_t* so = stage_o + (warp - 4) * 4096;
            const uint32_t rows_ok = __ballot_sync(0xffffffffu, real);
            if (a.parts > 1) {
                if (real) a.part_ml[prow] = make_float2((m == -INFINITY ? 0.0f : m) * a.scale2 - kLift<BF>, l);
#pragma unroll
                for (int kb = 0; kb < KB * 2; ++kb)
                    write_part(so, o + kb * 32, rows_ok, a.part_o + (prow - lane) * a.D, kb * 32, a.D, lane);
                continue;
            }
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
                write_rows<BF>(so, o + kb * 64, inv, rows_ok, po, qt * kTile + q4 * 32, a.os.token, kb * 64, a.D, lane);
            if (real && a.lse)
                a.lse[((size_t)P.b * a.H + h) * a.len_q + i] =
                    l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m) * a.scale2 - kLift<BF> + log2f(l)) * 0.693147180559945f;
        }
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tbase, 512);
}

// dim_head 129 .. 256: the output of one unit takes 256 columns of tensor
// memory, so a CTA has one unit, tiles of 64 keys, and two score buffers that
// the tiles take in turn: the scores of the next tile are formed under this
// tile's softmax.  Warp 0 copies, warp 1 issues, warps 4-7 are the softmax.
// 24/8 heads of 256, 2048 tokens, causal: 64-66 us (790-800 TFLOP/s); with one
// unit there is nothing to fill the gaps of its chain.
constexpr int kWideKB = 4, kWideKeys = 64, kWideSlots = 4;
constexpr int kWideThreads = 256;
constexpr int kWideBlk = kWideKeys * 128;        // bytes of 64 rows of 64 columns
constexpr int kWideSlot = kWideKB * kWideBlk;
constexpr int kWideSmem = 2048 + kWideKB * kBlk + kWideSlots * kWideSlot + 4 * 4096;
struct WideBars {
    uint64_t q_full, q_empty, o_full, o_empty, pv_done, drained;
    uint64_t s_full[2], p_ready[2];
    uint64_t full[kWideSlots], empty[kWideSlots];
    Items items;
    uint32_t tmem;
    int abort;
};
struct WideItem {
    int b, h, qt;
    SinkRange rg;
    int tiles, part;
};
__device__ __forceinline__ WideItem wide_item(const SinkArgs& a, int i, int per) {
    WideItem w;
    w.part = i % a.parts;
    i /= a.parts;
    w.qt = a.qtiles - 1 - i / per;  // the longest rows first
    const int bh = i % per;
    w.b = bh / a.H;
    w.h = bh - w.b * a.H;
    w.rg = sink_range(a, w.b, w.qt * kTile, kTile, kWideKeys);
    w.tiles = w.rg.part(w.part, a.parts);
    return w;
}

template <bool BF>
__global__ void __launch_bounds__(kWideThreads, 1)
    sink_wide_kernel(const SinkArgs a, const int items, const int per, const __grid_constant__ CUtensorMap tq,
                     const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv) {
    constexpr int KB = kWideKB, NS = kWideSlots;
    extern __shared__ uint8_t smem_raw[];
    asm volatile("griddepcontrol.launch_dependents;");  // a join may be scheduled (it waits for this grid)
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    WideBars& B = *reinterpret_cast<WideBars*>(sm);
    volatile int* abort_flag = &B.abort;
    uint8_t* sq = sm + 1024;
    uint8_t* ring = sq + KB * kBlk;
    uint8_t* stage_o = ring + NS * kWideSlot;  // 4 KB per softmax warp
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        mbar_init(&B.q_full, 1);
        mbar_init(&B.q_empty, 1);
        mbar_init(&B.o_full, 1);
        mbar_init(&B.o_empty, 4);
        mbar_init(&B.pv_done, 1);
        mbar_init(&B.drained, 1);
        B.items.init(5);
        if (blockIdx.x == 0 && items <= (int)gridDim.x) *a.err = 0;
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.s_full[i], 1);
            mbar_init(&B.p_ready[i], 4);
        }
        for (int i = 0; i < NS; ++i) {
            mbar_init(&B.full[i], 1);
            mbar_init(&B.empty[i], 1);
        }
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 1) tmem_alloc(&B.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = B.tmem;  // output: columns 0-255, scores: 64 columns from 256 and from 384

    if (warp == 0) {
        int q = 0, nq = 0;
        bool ok = true;
        auto copy = [&](const WideItem& P, int j, bool v) {
            const int s = q % NS;
            if (q >= NS && !(ok = warp_wait(&B.empty[s], (uint32_t)((q / NS - 1) & 1), a.err, abort_flag))) return;
            mbar_arrive_expect_tx_w(&B.full[s], kWideSlot);
            for (int kb = 0; kb < KB; ++kb)
                tma_load_4d_w(ring + s * kWideSlot + kb * kWideBlk, v ? &tv : &tk, kb * 64, P.rg.tile(j) * kWideKeys, P.h / a.G, P.b,
                              &B.full[s]);
            ++q;
        };
        int it = blockIdx.x;
        for (int k = 0; ok; ++k, it = B.items.draw(items, a.err, lane)) {
            if (!B.items.put(k, it, a.err, abort_flag, lane)) break;
            if (it >= items) break;
            const WideItem P = wide_item(a, it, per);
            if (P.tiles == 0) continue;
            copy(P, 0, false);
            if (!ok || (nq > 0 && !(ok = warp_wait(&B.q_empty, (uint32_t)((nq - 1) & 1), a.err, abort_flag)))) break;
            mbar_arrive_expect_tx_w(&B.q_full, KB * kBlk);
            for (int kb = 0; kb < KB; ++kb) tma_load_4d_w(sq + kb * kBlk, &tq, kb * 64, P.qt * kTile, P.h, P.b, &B.q_full);
            ++nq;
            for (int j = 0; j < P.tiles && ok; ++j) {  // the scores run a tile ahead: K1 before V0
                if (j + 1 < P.tiles) copy(P, j + 1, false);
                if (ok) copy(P, j, true);
            }
        }
        // every copy has landed before the CTA may end
        if (nq > 0) mbar_wait_bounded(&B.q_full, (uint32_t)((nq - 1) & 1), a.err);
        for (int s = 0; s < min(q, NS); ++s) mbar_wait_bounded(&B.full[s], (uint32_t)(((q - 1 - s) / NS) & 1), a.err);
    } else if (warp == 1) {
        const uint32_t ids = mma_idesc(BF ? 1u : 0u, kWideKeys);
        const uint32_t idv = mma_idesc(BF ? 1u : 0u, KB * 64) | (1u << 16);  // B with N contiguous
        const uint64_t qd = mma_desc_sw128(smem_u32(sq)), kd = mma_desc_sw128(smem_u32(ring));
        const uint64_t vd = v_desc(smem_u32(ring), kWideBlk);
        int q = 0, nq = 0, nt = 0, no = 0;  // ring copies, items, tiles, items whose output was begun
        bool ok = true;
        auto wait = [&](uint64_t* bar, int n) { return ok = warp_wait(bar, (uint32_t)(n & 1), a.err, abort_flag); };
        auto scores = [&](int t, int slot) {  // of tile number t of all
            const uint64_t d = kd + (uint32_t)(slot * (kWideSlot >> 4));
#pragma unroll
            for (int ks = 0; ks < KB * 4; ++ks)
                mma_ss(tbase + 256 + (t & 1) * 128, qd + (((ks >> 2) * kBlk + (ks & 3) * 32) >> 4),
                       d + (((ks >> 2) * kWideBlk + (ks & 3) * 32) >> 4), ids, ks > 0);
            mma_commit_w(&B.s_full[t & 1]);
            mma_commit_w(&B.empty[slot]);
        };
        for (int k = 0; ok; ++k) {
            const int it = B.items.get(k, a.err, abort_flag, lane);
            if (it >= items) break;
            const WideItem P = wide_item(a, it, per);
            if (P.tiles == 0) continue;
            if (!wait(&B.q_full, nq) || !wait(&B.full[q % NS], q / NS)) break;
            ++nq;
            tc_fence_after();
            scores(nt, q % NS);
            if (P.tiles == 1) mma_commit_w(&B.q_empty);
            ++q;
            for (int j = 0; j < P.tiles; ++j, ++nt) {
                if (j + 1 < P.tiles) {
                    // its buffer held the P of the tile before, whose products are issued already
                    if (!wait(&B.full[q % NS], q / NS)) break;
                    tc_fence_after();
                    scores(nt + 1, q % NS);
                    if (j + 2 == P.tiles) mma_commit_w(&B.q_empty);
                    ++q;
                }
                const int sv = q % NS;
                if (!wait(&B.full[sv], q / NS)) break;
                ++q;
                const int behind = P.rg.n - P.rg.tile(j) * kWideKeys;  // keys of the tile that exist
                if (behind < kWideKeys && P.rg.n < a.len_k) {
                    // the padding behind a sequence's end may hold anything, and 0 * NaN is NaN
                    uint8_t* vt = ring + sv * kWideSlot;
                    for (int e = lane; e < (kWideKeys - behind) * 8; e += 32)
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb)
                            *reinterpret_cast<uint4*>(vt + kb * kWideBlk + behind * 128 + e * 16) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();
                    __syncwarp();
                }
                if (j == 0 && no++ > 0 && !wait(&B.o_empty, no)) break;  // the output rows before have been read
                if (!wait(&B.p_ready[nt & 1], nt >> 1)) break;
                tc_fence_after();
                const uint64_t d = vd + (uint32_t)(sv * (kWideSlot >> 4));
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) mma_ts(tbase, tbase + 256 + (nt & 1) * 128 + ks * 8, d + ks * 128, idv, (j | ks) > 0);
                mma_commit_w(&B.empty[sv]);
                mma_commit_w(&B.pv_done);
            }
            if (ok) mma_commit_w(&B.o_full);
        }
        // the products have ended before the tensor memory is freed
        mma_commit_w(&B.drained);
        mbar_wait_bounded(&B.drained, 0, a.err);
    } else if (warp >= 4) {
        const int q4 = warp & 3, row = q4 * 32 + lane;
        const uint32_t to = tbase + ((uint32_t)(q4 * 32) << 16);
        uint8_t* so = stage_o + q4 * 4096;
        const float2 sc = make_float2(a.scale2, a.scale2);
        int nt = 0, ni = 0;
        bool ok = true;
        for (int k = 0; ok; ++k) {
            const int it = B.items.get(k, a.err, abort_flag, lane);
            if (it >= items) break;
            const WideItem P = wide_item(a, it, per);
            const int p0 = P.qt * kTile + a.len_k - a.len_q, p = p0 + row, n = P.rg.n;
            const int i = P.qt * kTile + row;
            const bool real = i < a.len_q && p < n;
            const size_t prow = (((size_t)P.part * a.batch + P.b) * a.H + P.h) * a.len_q + i;  // this row of the part
            if (P.tiles == 0) {
                if (a.parts > 1 && real) a.part_ml[prow] = make_float2(-INFINITY, 0.0f);
                continue;
            }
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < P.tiles; ++j, ++nt) {
                const uint32_t ts = to + 256 + (nt & 1) * 128;
                if (!(ok = warp_wait(&B.s_full[nt & 1], (uint32_t)((nt >> 1) & 1), a.err, abort_flag))) break;
                tc_fence_after();
                uint32_t r[64];
                ld32_async(ts, r);
                ld32_async(ts + 32, r + 32);
                wait_ld();
                pin32(r);
                pin32(r + 32);
                const int j0 = P.rg.tile(j) * kWideKeys;
                const bool whole = j0 + kWideKeys - 1 <= p0 && j0 + kWideKeys <= n &&
                                   (a.window <= 0 || j0 > p0 + kTile - 1 - a.window || j0 + kWideKeys <= a.sinks);
                if (!whole) {
                    const int hi = min(p, n - 1) - j0 + 1, lo = a.window > 0 ? p - a.window + 1 - j0 : 0, sk = a.sinks - j0;
#pragma unroll
                    for (int w = 0; w < 2; ++w) {  // a bit per column
                        const uint32_t see = below(hi - 32 * w) & (~below(lo - 32 * w) | below(sk - 32 * w));
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!(see & (1u << c))) r[32 * w + c] = 0xFF800000u;  // -inf
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 64; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(r[c]), __uint_as_float(r[c + 1]));
                const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                const bool need = (mt - m) * a.scale2 > kGrow;  // true for a row's first key, false while it has none
                if (__any_sync(0xffffffffu, need)) {
                    const float corr = need ? ex2_approx((m - mt) * a.scale2) : 1.0f;
                    l *= corr;
                    if (need) m = mt;
                    if (j > 0) {  // behind the products of the tile before
                        if (!(ok = warp_wait(&B.pv_done, (uint32_t)((nt - 1) & 1), a.err, abort_flag))) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < KB * 2; ++c) {
                            uint32_t o[32];
                            ld32_async(to + c * 32, o);
                            wait_ld();
                            pin32(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                            st32(to + c * 32, o);
                        }
                    }
                }
                const float ms = (m == -INFINITY ? 0.0f : m) * a.scale2 - kLift<BF>;
                const float2 nm = make_float2(-ms, -ms);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                    float2 x = __ffma2_rn(make_float2(__uint_as_float(r[2 * c]), __uint_as_float(r[2 * c + 1])), sc, nm);
                    x.x = ex2_approx(x.x);
                    x.y = ex2_approx(x.y);
                    sum[c & 1] = __fadd2_rn(sum[c & 1], x);
                    r[c] = pack2<BF>(x.x, x.y);
                }
                st32(ts, r);
                wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive1(&B.p_ready[nt & 1]);
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            if (!ok || !(ok = warp_wait(&B.o_full, (uint32_t)(ni++ & 1), a.err, abort_flag))) break;
            tc_fence_after();
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            uint8_t* po = a.O + (size_t)P.b * a.os.item + (size_t)P.h * a.os.head;
            const uint32_t rows_ok = __ballot_sync(0xffffffffu, real);
#pragma unroll 1
            for (int kb = 0; kb < KB; ++kb) {
                uint32_t o[64];
                ld32_async(to + kb * 64, o);
                ld32_async(to + kb * 64 + 32, o + 32);
                wait_ld();
                pin32(o);
                pin32(o + 32);
                if (kb == KB - 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive1(&B.o_empty);
                }
                if (a.parts > 1) {
                    write_part(so, o, rows_ok, a.part_o + (prow - lane) * a.D, kb * 64, a.D, lane);
                    write_part(so, o + 32, rows_ok, a.part_o + (prow - lane) * a.D, kb * 64 + 32, a.D, lane);
                } else {
                    write_rows<BF>(so, o, inv, rows_ok, po, P.qt * kTile + q4 * 32, a.os.token, kb * 64, a.D, lane);
                }
            }
            if (a.parts > 1) {
                if (real) a.part_ml[prow] = make_float2((m == -INFINITY ? 0.0f : m) * a.scale2 - kLift<BF>, l);
                continue;
            }
            if (real && a.lse)
                a.lse[((size_t)P.b * a.H + P.h) * a.len_q + i] =
                    l == 0.0f ? -INFINITY : ((m == -INFINITY ? 0.0f : m) * a.scale2 - kLift<BF> + log2f(l)) * 0.693147180559945f;
        }
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 1) tmem_dealloc(tbase, 512);
}

// [batch][heads][rows][D] with byte strides; boxes of 64 columns x box_rows rows, 128-byte swizzle, zeros
// outside.  A stride of a dimension of one entry is not used and set to a valid value.
bool encode(CUtensorMap* m, const void* base, bool bf, int D, int rows, int heads, int batch, const rkv_row_strides& s,
            int box_rows) {
    auto enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t rowb = (cuuint64_t)D * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batch};
    const cuuint64_t st[3] = {rows > 1 ? (cuuint64_t)s.token : rowb, heads > 1 ? (cuuint64_t)s.head : rowb,
                              batch > 1 ? (cuuint64_t)s.item : rowb};
    const cuuint32_t box[4] = {64u, (cuuint32_t)box_rows, 1u, 1u}, one[4] = {1u, 1u, 1u, 1u};
    return enc(m, bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, st,
               box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Error word and ticket.  Where no ticket is drawn the kernel clears the error word itself: a wait gives up after
// two seconds at the soonest, long after the first CTA's first instructions, and a memset costs a launch.
bool clear_header(const SinkArgs& a, int items, cudaStream_t st) {
    return items <= kSinkSms || cudaMemsetAsync(a.err, 0, (kSinkTicket + 1) * sizeof(int), st) == cudaSuccess;
}

template <int KB, bool BF>
int launch_kb(const SinkArgs& a, int items, int per, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
              cudaStream_t st) {
    if (!clear_header(a, items, st)) return RKV_ERR_CUDA;
    // the barriers, and up to 1023 bytes of alignment; Q and the ring; the output rows' stage
    const int smem = 2048 + (2 + 2 * stages(KB)) * KB * kBlk + 8 * 4096;
    if (cudaFuncSetAttribute(sink_tc_kernel<KB, BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    sink_tc_kernel<KB, BF><<<items < kSinkSms ? items : kSinkSms, kThreads, smem, st>>>(a, items, per, tq, tk, tv);
    return cudaGetLastError() == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}

template <bool BF>
int launch_wide(const SinkArgs& a, int items, int per, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                cudaStream_t st) {
    if (!clear_header(a, items, st)) return RKV_ERR_CUDA;
    if (cudaFuncSetAttribute(sink_wide_kernel<BF>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideSmem) != cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    sink_wide_kernel<BF><<<items < kSinkSms ? items : kSinkSms, kWideThreads, kWideSmem, st>>>(a, items, per, tq, tk, tv);
    return cudaGetLastError() == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}

}  // namespace

int launch_sink_tc(SinkArgs a, int dtype, int batch, cudaStream_t st) {
    const bool bf = dtype == RKV_BF16;
    CUtensorMap tq, tk, tv;
    const int keys = a.D <= 128 ? kTile : kWideKeys;
    if (!encode(&tq, a.Q, bf, a.D, a.len_q, a.H, batch, a.qs, kTile) || !encode(&tk, a.K, bf, a.D, a.len_k, a.HK, batch, a.ks, keys) ||
        !encode(&tv, a.V, bf, a.D, a.len_k, a.HK, batch, a.ks, keys))
        return RKV_ERR_CUDA;
    a.qtiles = (a.len_q + kTile - 1) / kTile;
    if (a.D > 128) {
        const long long per = (long long)batch * a.H, items = (long long)a.qtiles * per * a.parts;
        if (items > (1 << 30)) return RKV_ERR_UNSUPPORTED;
        return bf ? launch_wide<true>(a, (int)items, (int)per, tq, tk, tv, st)
                  : launch_wide<false>(a, (int)items, (int)per, tq, tk, tv, st);
    }
    const long long units = (long long)a.G * a.qtiles, per = (long long)batch * a.HK, items = (units + 1) / 2 * per * a.parts;
    if (units > 0x7FFFFFFELL || items > (1 << 30)) return RKV_ERR_UNSUPPORTED;
    const int n = (int)items, p = (int)per;
    if (a.D <= 64) return bf ? launch_kb<1, true>(a, n, p, tq, tk, tv, st) : launch_kb<1, false>(a, n, p, tq, tk, tv, st);
    return bf ? launch_kb<2, true>(a, n, p, tq, tk, tv, st) : launch_kb<2, false>(a, n, p, tq, tk, tv, st);
}

long long sink_tc_items(const SinkArgs& a, int* rows, int* keys) {
    const long long qtiles = (a.len_q + kTile - 1) / kTile;
    *keys = a.D <= 128 ? kTile : kWideKeys;
    if (a.D > 128) {
        *rows = kTile;
        return qtiles * a.batch * a.H;
    }
    *rows = 2 * kTile;  // two units of different query tiles at most
    return (a.G * qtiles + 1) / 2 * a.batch * a.HK;
}

}  // namespace rkv
