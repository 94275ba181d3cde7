// prefix_tc.cu -- the shared tokens of a group of sequences against all of the
// group's queries on the tcgen05 tensor cores: 16-bit types.
//
// Rows are (sequence, query head of the KV head), 128 to an accumulator; a unit
// is up to 256 of them, two accumulators, so that both use every K and V tile
// that is loaded.  A unit of 128 rows or fewer takes the tiles in turn
// instead, the even ones to the first accumulator and the odd ones to the
// second, and joins the two at the end: either way one accumulator's softmax
// runs while the tensor cores work on the other's products.  128 keys at a
// time: S = Q K^T into tensor memory, P = 2^(S - m) as a sum of two 16-bit parts
// back into tensor memory in S's place, O += P V, a product for each part.
//
// Above 128 columns the accumulator of 128 rows takes half of the tensor memory:
// a unit is 128 rows then, tiles are 64 keys, and two score buffers take the
// tiles in turn, so that the next scores are formed under this tile's softmax.
//
//   warps 0-3    copy Q's rows by 16-byte asynchronous copies into the swizzled tiles; also K's and V's, in
//                pages of any size, unless these are multiples of 8 tokens
//   warp 5       has K's and V's copied as boxes of a tensor map where they are
//   warp 4       issues the products
//   warp 6       tells the others which rows and tiles are next
//   warps 8-11, 12-15   softmax of the first accumulator, of the second, and their rows (above 128 columns the
//                latter only write half of them)
//
// The tiles of the units are cut into stretches so that, whatever the groups'
// sizes and lengths, every SM has about the same work.
// Each stretch leaves (m, l, O) of its rows, not divided by l, for the join.
//
// The products take both operands in one type, so P enters as its value rounded
// to the type and what that rounding left, rounded: 16 bits of a weight in bf16,
// 22 in fp16 (2^-32 of the row's largest at least), as many as the two parts have
// columns in S's place.  One part alone (8 and 11 bits) made a sequence's weights
// depend on how many others share its tokens, and where values of opposite signs
// meet its output was up to 35 times further off than a decode of its own may be;
// it took 43 us in place of 48 for 64 sequences behind 8192 tokens, 99 in place of
// 103 for 8 behind 131072.  Scores, m, l and the accumulators are fp32.  Every
// row of a tile sees all of its keys, but for those behind the shared tokens
// and on pages outside the pool, which a mask of a bit per key leaves out.
//
// What bounds it.  Many rows: a pair of tiles takes 3.2 us, of which the products
// are 1.7 at their full rate and the exponentials 1.1 at theirs; an accumulator's
// chain of scores, softmax and products is covered by the other's in part.  Long
// prefixes and few rows: the same chain with one warp of each softmax at work, and
// behind it HBM: 8 sequences behind 131072 tokens (24/8 heads of 128, bf16) 104 us
// a call, 5.3 TB/s, at full clock, 115-121 where the power cap lowers it.  Short
// ones: begin and end, 64 sequences behind 8192 tokens 25 us, 4 until the first
// scores, 4 tiles, 2 for the rows.  Not kept, measured with P in one part: a wait
// of the copying warps before each hand-over (a call at 131072 tokens 103 us ->
// 119), K and V by 16-byte copies where boxes can be (its kernel 97 us with boxes,
// 111 with copies, at a time when it took more than at the end).
#include <atomic>

#include "attn_tc.cuh"
#include "prefix.cuh"

namespace rkv {
namespace {

constexpr int kThreads = kTcThreads;
constexpr int kBlk = 128 * 128;  // bytes of a 128-row block of 64 columns
constexpr int kMasks = 16;       // tiles whose masks are kept: more than the copies are ahead of the softmax

// By blocks of 64 columns: slots of the ring (each a K or a V tile), keys of a tile, rows of a unit.
__host__ __device__ constexpr int ring_slots(int kb) { return kb == 1 ? 8 : 5; }
__host__ __device__ constexpr int tile_keys(int kb) { return kb > 2 ? 64 : 128; }
__host__ __device__ constexpr int unit_rows(int kb) { return kb > 2 ? 128 : 256; }

struct Args {
    SharedArgs s;
    TcParts p;
    int G;
    int box;       // tokens of a box, a power of two that divides the page size; 0: none, copies by 16 bytes
    int spare;     // SMs that may be left to the kernel before, at most half of all
    float scale2;  // log2(e) / sqrt(D)
};

// A CTA's part of a unit: rows row0 .. row0 + rows - 1 of group g (whose first sequence is s0) and KV head hk, and
// `tiles` tiles (0: there is no more to do) from tile j0 on of its `shared` tokens; from tile 0: how many CTAs behind
// this one have the others.
struct Stretch {
    int g, hk, s0, row0, rows, shared, j0, tiles, behind;
};
// The stretches on their way from the warp that finds them to the others, through two places.
struct Stretches {
    uint64_t full[2], empty[2];
    Stretch at[2];
    __device__ void init(int readers) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], readers);
        }
    }
    __device__ __forceinline__ bool put(int k, const Stretch& x, int* err, volatile int* abort, int lane) {
        if (k >= 2 && !warp_wait(&empty[k & 1], (uint32_t)(((k >> 1) - 1) & 1), err, abort)) return false;
        if (lane == 0) {
            at[k & 1] = x;
            mbar_arrive1(&full[k & 1]);
        }
        __syncwarp();
        return x.tiles > 0;
    }
    // A reading warp's k-th; false behind the last and where the wait gave up.
    __device__ __forceinline__ bool get(int k, Stretch& x, int* err, volatile int* abort, int lane) {
        if (!warp_wait(&full[k & 1], (uint32_t)((k >> 1) & 1), err, abort)) return false;
        x = at[k & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive1(&empty[k & 1]);
        return x.tiles > 0;
    }
};

struct Bars {
    uint64_t q_full, o_full, o_empty, written, drained;
    uint64_t s_full[2], p_half[2], p_ready[2], pv_done;  // of an accumulator (above 128 columns: of a score buffer)
    uint64_t full[8], empty[8];
    uint64_t pair[4];  // of the two softmax warps that hold the same rows
    Stretches next;
    alignas(16) uint32_t mask[kMasks][4];
    uint32_t tmem;
    int abort;
};
static_assert(sizeof(Bars) <= 1024, "the barriers' part of shared memory");

// Rows of a group and KV head, the group's units (of all KV heads) and the tiles of one.
struct Group {
    int start, rows, per_head, units, shared, tiles;
};
template <int KB>
__device__ __forceinline__ Group group_of(const Args& a, int g) {
    Group t{0, 0, 0, 0, 0, 0};
    if (g < a.s.gr.n) {
        t.start = a.s.gr.start(g);
        t.rows = max(0, a.s.gr.start(g + 1) - t.start) * a.G;
        t.per_head = (t.rows + unit_rows(KB) - 1) / unit_rows(KB);
        t.units = t.per_head * a.s.HK;
        t.shared = a.s.gr.shared(a.s.c, g);
        t.tiles = (t.shared + tile_keys(KB) - 1) / tile_keys(KB);
    }
    return t;
}
// The stretches of this CTA (a warp walks them).  Either each unit is cut into as many equal stretches as its share of
// the tiles is worth CTAs, one per CTA; or, where that needs more CTAs than there are or leaves one kAligned tiles
// more to do than an equal share, the tiles of all units are one list that is cut into equal stretches: a CTA whose
// stretch spans two units pays the ends of a unit (4 us) twice.
constexpr int kAligned = 3;
constexpr int kSpare = 4;  // tiles more of a CTA at most for SMs that are left to the own tokens' CTAs
__host__ __device__ constexpr int min_tiles(int kb) { return 128 / tile_keys(kb); }  // of a stretch
template <int KB>
struct Walk {
    int total, ctas;  // tiles, CTAs that take them
    int at, end;      // this CTA's; aligned: one stretch
    bool aligned;
    Group mine;       // group number `lane`

    __device__ __forceinline__ Group group(const Args& a, int g0, int lane) const { return g0 == 0 ? mine : group_of<KB>(a, g0 + lane); }
    __device__ __forceinline__ int parts(const Group& t) const {  // aligned: of a unit
        return max(1, min((int)((unsigned)ctas * t.tiles / (unsigned)total), t.tiles / min_tiles(KB)));
    }
    __device__ __forceinline__ void begin_walk(const Args& a, int lane) {
        mine = group_of<KB>(a, lane);
        int n = 0;
        for (int g0 = 0; g0 < a.s.gr.n; g0 += 32) {
            const Group t = group(a, g0, lane);
            n += t.units * t.tiles;
        }
        total = __reduce_add_sync(0xffffffffu, n);
        // the own tokens' CTAs, begun before, hold their SMs for about as long as four tiles take
        const int all = gridDim.x, few = all - a.spare;
        ctas = (total + few - 1) / few <= (total + all - 1) / all + kSpare ? few : all;
        at = end = 0;
        aligned = true;
        if (total > 0) {
            int need = 0, most = 0;
            for (int g0 = 0; g0 < a.s.gr.n; g0 += 32) {
                const Group t = group(a, g0, lane);
                if (t.units > 0 && t.tiles > 0) {
                    const int p = parts(t);
                    need += t.units * p;
                    most = max(most, (t.tiles + p - 1) / p);
                }
            }
            need = __reduce_add_sync(0xffffffffu, need);
            most = __reduce_max_sync(0xffffffffu, most);
            aligned = need <= ctas && (most <= min_tiles(KB) + 1 || most <= (total + ctas - 1) / ctas + kAligned);
            const int c = blockIdx.x;
            if (aligned) {
                end = c < need;
            } else {
                ctas = min(ctas, (total + min_tiles(KB) - 1) / min_tiles(KB));
                if (c < ctas) at = begin(c), end = begin(c + 1);
            }
        }
    }
    // One list: the first total % ctas CTAs have a tile more than the others.
    __device__ __forceinline__ int begin(int c) const { return total / ctas * c + min(c, total % ctas); }
    __device__ __forceinline__ int cta_of(int tile) const {
        const int q = total / ctas, r = total % ctas, cut = (q + 1) * r;
        return tile < cut ? tile / (q + 1) : r + (tile - cut) / q;
    }
    __device__ __forceinline__ Stretch next(const Args& a, int lane) {
        Stretch x{0, 0, 0, 0, 0, 0, 0, 0, 0};
        if (at >= end) return x;
        const int want = aligned ? (int)blockIdx.x : at;
        int base = 0;
        for (int g0 = 0; g0 < a.s.gr.n; g0 += 32) {
            const Group t = group(a, g0, lane);
            const int p = aligned && t.units > 0 && t.tiles > 0 ? parts(t) : 0;
            const int here = t.units * (aligned ? p : t.tiles);
            int sum = here;
            if (a.s.gr.n > 1) {
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o) sum += y;
                }
            }
            const unsigned hits = __ballot_sync(0xffffffffu, want < base + sum);
            if (hits) {
                const int l = __ffs(hits) - 1;
                auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, l); };
                const int off = want - base - of(sum - here), per_head = of(t.per_head), tiles = of(t.tiles), n = of(p);
                const int unit = off / (aligned ? n : tiles);  // the units of a KV head side by side: they read the same tiles
                const int in = off - unit * (aligned ? n : tiles);
                x.g = g0 + l;
                x.hk = unit / per_head;
                x.row0 = (unit - x.hk * per_head) * unit_rows(KB);
                x.rows = min(unit_rows(KB), of(t.rows) - x.row0);
                x.s0 = of(t.start);
                x.shared = of(t.shared);
                if (aligned) {
                    x.j0 = (int)((unsigned)tiles * in / (unsigned)n);
                    x.tiles = (int)((unsigned)tiles * (in + 1) / (unsigned)n) - x.j0;
                    x.behind = n - 1;
                    at = end;
                } else {
                    x.j0 = in;
                    x.tiles = min(tiles - in, end - at);
                    x.behind = in == 0 ? cta_of(at + tiles - 1) - (int)blockIdx.x : 0;
                    at += x.tiles;
                }
                return x;
            }
            base += __shfl_sync(0xffffffffu, sum, 31);
        }
        return x;
    }
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
// Arrives on `bar` once the copies that this thread has begun have landed.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A warp's ROWS rows of KB blocks of 64 columns (of BLK bytes each) into a swizzled tile at dst (this warp's first
// row): off is this lane's row's offset from src, or -1 for a row of zeros; columns from `chunks` 16-byte chunks on
// are zeros.
template <int KB, int ROWS, int BLK>
__device__ __forceinline__ void copy_rows(uint32_t dst, const uint8_t* src, long long off, int chunks, int lane) {
    constexpr int LPR = KB * 8, RPI = 32 / LPR;  // lanes of a row, rows of an instruction
    const int c = lane % LPR, r0 = lane / LPR;
    constexpr int U = 8;  // rows whose places are asked for together
    src += c * 16;
    dst += (c >> 3) * BLK + r0 * 128;
#pragma unroll
    for (int i0 = 0; i0 < ROWS / RPI; i0 += U) {
        long long o[U];
#pragma unroll
        for (int i = 0; i < U; ++i) o[i] = __shfl_sync(0xffffffffu, off, (i0 + i) * RPI + r0);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int r = (i0 + i) * RPI;
            const bool real = o[i] >= 0 && c < chunks;
            copy16(dst + r * 128 + (((c & 7) ^ ((r + r0) & 7)) << 4), src + (real ? o[i] : -16 * c), real);
        }
    }
}

// 32 fp32 columns of a warp's 32 rows (a row per lane in o) to the rows' places (place: this lane's row's, in
// floats, or -1), through 4 KB of shared memory so that eight lanes write 128 bytes of a row.
__device__ __forceinline__ void write_cols(uint8_t* so, const uint32_t* o, float* dst, long long place, int col0, int D, int lane) {
#pragma unroll
    for (int v = 0; v < 8; ++v)
        *reinterpret_cast<uint4*>(so + lane * 128 + ((v ^ (lane & 7)) << 4)) = make_uint4(o[v * 4], o[v * 4 + 1], o[v * 4 + 2], o[v * 4 + 3]);
    __syncwarp();
#pragma unroll
    for (int x = 0; x < 8; ++x) {
        const int r = x * 4 + (lane >> 3), v = lane & 7;
        const uint4 y = *reinterpret_cast<const uint4*>(so + r * 128 + ((v ^ (r & 7)) << 4));
        const long long at = __shfl_sync(0xffffffffu, place, r);
        if (at >= 0 && col0 + v * 4 < D) *reinterpret_cast<uint4*>(dst + at + col0 + v * 4) = y;
    }
    __syncwarp();
}

template <int KB, bool BF, bool BOXES>
__global__ void __launch_bounds__(kThreads, 1)
    prefix_tc_kernel(const Args a, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv) {
    constexpr bool WIDE = KB > 2;
    constexpr int NS = ring_slots(KB), KEYS = tile_keys(KB), WORDS = KEYS / 32;
    constexpr uint32_t kTileBlk = KEYS * 128, kSlot = KB * kTileBlk;  // bytes of a tile's 64 columns, of a tile
    constexpr uint32_t kRows = KB * kBlk;                             // bytes of 128 rows of Q
    // tensor memory: S0, S1 (KEYS columns each), O0, O1 (64 KB columns each); above 128 columns O, then S0, S1
    constexpr uint32_t kColS = WIDE ? 256 : 0, kColO = WIDE ? 0 : 256, kStepO = WIDE ? 0 : KB * 64;
    extern __shared__ uint8_t smem_raw[];
    asm volatile("griddepcontrol.launch_dependents;");  // the kernel behind may be scheduled (it waits for this grid)
    uint8_t* sm = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    Bars& B = *reinterpret_cast<Bars*>(sm);
    volatile int* abort_flag = &B.abort;
    int* err = a.p.err;
    uint8_t* sq = sm + 1024;
    uint8_t* ring = sq + unit_rows(KB) / 128 * kRows;
    uint8_t* stage = ring - 8 * 4096;  // 4 KB per softmax warp, in Q's place once its products have ended
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    Walk<KB> walk;
    Stretch x;
    if (warp == 6) {
        walk.begin_walk(a, lane);
        x = walk.next(a, lane);
    }
    if (tid == 0) {
        mbar_init(&B.q_full, 128);
        mbar_init(&B.o_full, 1);
        mbar_init(&B.o_empty, 8);
        mbar_init(&B.written, 8);
        mbar_init(&B.drained, 1);
        mbar_init(&B.pv_done, 1);
        for (int u = 0; u < 2; ++u) {
            mbar_init(&B.s_full[u], 1);
            mbar_init(&B.p_half[u], 4);
            mbar_init(&B.p_ready[u], 4);
        }
        for (int i = 0; i < NS; ++i) {
            mbar_init(&B.full[i], BOXES ? 1 : 4 * 33);  // 33: a copying warp's lanes' copies, and its part of the mask
            mbar_init(&B.empty[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&B.pair[i], 2);
        B.next.init(BOXES ? 14 : 13);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 4) tmem_alloc(&B.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = B.tmem;

    // split_fits: together as many registers as the launch has
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTcFewRegs));
        const int chunks = a.s.D / 8;
        int q = 0, nk = 0;  // slots, tiles
        bool ok = true;
        auto slot = [&](const uint8_t* base, long long off) {
            const int s = q % NS;
            if (q >= NS) ok = warp_wait(&B.empty[s], (uint32_t)((q / NS - 1) & 1), err, abort_flag);
            if (ok) {
                copy_rows<KB, KEYS / 4, kTileBlk>(smem_u32(ring) + s * kSlot + warp * (KEYS / 4 * 128), base, off, chunks, lane);
                copies_arrive(&B.full[s]);
                if (lane == 0) mbar_arrive1(&B.full[s]);
                ++q;
            }
        };
        for (int nq = 0; ok && B.next.get(nq, x, err, abort_flag, lane); ++nq) {
            if (nq > 0 && !(ok = warp_wait(&B.written, (uint32_t)((nq - 1) & 1), err, abort_flag))) break;
            for (int u = 0; u < (x.rows > 128 ? 2 : 1); ++u) {
                const int r = u * 128 + warp * 32 + lane;
                const unsigned row = x.row0 + r, sq_ = row / (unsigned)a.G;
                const long long off = r < x.rows ? (long long)(x.s0 + (int)sq_) * a.s.q_stride +
                                                       (long long)(x.hk * a.G + (int)(row - sq_ * a.G)) * a.s.D * 2
                                                 : -1;
                copy_rows<KB, 32, kBlk>(smem_u32(sq) + u * kRows + warp * 4096, a.s.Q, off, chunks, lane);
            }
            copies_arrive(&B.q_full);
            if (!BOXES) {
                const int leader = leader_of(a.s.gr, a.s.c, x.g, x.shared);
                for (int j = x.j0; j < x.j0 + x.tiles && ok; ++j, ++nk) {
                    const int t = j * KEYS + warp * (KEYS / 4) + lane;
                    const long long off = lane < KEYS / 4 && t < x.shared ? paged_offset(a.s.c, leader, x.hk, t) : -1;
                    const uint32_t mask = __ballot_sync(0xffffffffu, off >= 0);
                    if (lane == 0) {
                        if (WIDE) reinterpret_cast<uint16_t*>(B.mask[nk % kMasks])[warp] = (uint16_t)mask;
                        else B.mask[nk % kMasks][warp] = mask;
                    }
                    slot(a.s.c.K, off);
                    if (ok) slot(a.s.c.V, off);
                }
            }
        }
        // every copy has landed before the CTA may end
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp < 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTcFewRegs));
        if (warp == 4) {
            const uint32_t ids = mma_idesc(BF ? 1u : 0u, KEYS);
            const uint32_t idv = mma_idesc(BF ? 1u : 0u, KB * 64) | (1u << 16);  // B with N contiguous
            const uint64_t qd = mma_desc_sw128(smem_u32(sq)), kd = mma_desc_sw128(smem_u32(ring));
            const uint64_t vd = v_desc(smem_u32(ring), kTileBlk);
            int q = 0;
            uint32_t steps = 0;  // a bit per accumulator: parity of its steps
            bool ok = true;
            auto wait = [&](uint64_t* bar, int n) { ok = ok && warp_wait(bar, (uint32_t)(n & 1), err, abort_flag); };
            for (int nq = 0; ok && B.next.get(nq, x, err, abort_flag, lane); ++nq) {
                // step k: accumulator k & 1 and the next tile, or both accumulators one after the other with each tile
                const bool both = !WIDE && x.rows > 128;
                const int n = both ? 2 * x.tiles : x.tiles;
                auto scores = [&](int k) {
                    const int u = k & 1, at = q + 2 * (both ? k >> 1 : k), s = at % NS;
                    if (!(both && u)) {
                        wait(&B.full[s], at / NS);
                        if (!BOXES) fence_proxy_async();  // what 16-byte copies wrote is read through another proxy
                    }
                    if (ok) {
                        tc_fence_after();
                        const uint64_t da = qd + (uint32_t)((both ? u : 0) * (kRows >> 4)), db = kd + (uint32_t)(s * (kSlot >> 4));
#pragma unroll
                        for (int ks = 0; ks < KB * 4; ++ks)
                            mma_ss(tbase + kColS + u * KEYS, da + (((ks >> 2) * kBlk + (ks & 3) * 32) >> 4),
                                   db + (((ks >> 2) * kTileBlk + (ks & 3) * 32) >> 4), ids, ks > 0);
                        mma_commit_w(&B.s_full[u]);
                        if (!both || u) mma_commit_w(&B.empty[s]);
                    }
                };
                wait(&B.q_full, nq);
                fence_proxy_async();
                scores(0);
                if (ok && n > 1) scores(1);
                if (ok && nq > 0) wait(&B.o_empty, nq - 1);  // the rows of the stretch before have been read
                for (int k = 0; k < n && ok; ++k) {
                    const int u = k & 1, at = q + 2 * (both ? k >> 1 : k) + 1, s = at % NS;
                    if (!(both && u)) {
                        wait(&B.full[s], at / NS);
                        if (!BOXES) fence_proxy_async();
                    }
                    const int real = x.shared - (x.j0 + (both ? k >> 1 : k)) * KEYS;  // of the tile's rows
                    if (BOXES && ok && real < KEYS && !(both && u)) {
                        // a box holds what lies behind the shared tokens too, which may be anything, and 0 * NaN is NaN
                        for (int e = lane; e < (KEYS - real) * 8; e += 32)
#pragma unroll
                            for (int kb = 0; kb < KB; ++kb)
                                *reinterpret_cast<uint4*>(ring + s * kSlot + kb * kTileBlk + real * 128 + e * 16) = make_uint4(0, 0, 0, 0);
                        fence_proxy_async();
                        __syncwarp();
                    }
                    const uint64_t db = vd + (uint32_t)(s * (kSlot >> 4));
#pragma unroll
                    for (int half = WIDE ? 1 : 0; half < 2; ++half) {
                        wait(half ? &B.p_ready[u] : &B.p_half[u], (int)(steps >> u));
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int ks = WIDE ? 0 : half * 4; ks < half * 4 + 4 && ks < KEYS / 16; ++ks)
#pragma unroll
                            for (int part = 0; part < 2; ++part)
                                mma_ts(tbase + kColO + u * kStepO, tbase + kColS + u * KEYS + part * (KEYS / 2) + ks * 8, db + ks * 128, idv,
                                       k > (WIDE ? 0 : 1) || ks > 0 || part > 0);
                    }
                    if (!ok) break;
                    steps ^= 1u << u;
                    if (!both || u) mma_commit_w(&B.empty[s]);
                    if (WIDE) mma_commit_w(&B.pv_done);
                    if (k + 2 < n) scores(k + 2);
                }
                if (ok) mma_commit_w(&B.o_full);
                q += 2 * x.tiles;
            }
            // the products have ended before the tensor memory is freed
            mma_commit_w(&B.drained);
            mbar_wait_bounded(&B.drained, 0, err);
        } else if (BOXES && warp == 5) {
            int q = 0, nk = 0;  // slots, tiles
            bool ok = true;
            for (int nq = 0; ok && B.next.get(nq, x, err, abort_flag, lane); ++nq) {
                const int leader = leader_of(a.s.gr, a.s.c, x.g, x.shared);
                for (int j = x.j0; j < x.j0 + x.tiles && ok; ++j, ++nk) {
                    // lane i has box i; one of a page outside the pool begins behind it and is filled with zeros
                    const int t = j * KEYS + lane * a.box;
                    int page = a.s.c.num_pages, row = 0;
                    if (lane * a.box < KEYS && t < x.shared) {
                        const unsigned n = (unsigned)t / (unsigned)a.s.c.page_size;
                        const int p = a.s.c.table[(size_t)leader * a.s.c.table_stride + n];
                        if ((unsigned)p < (unsigned)page) page = p, row = t - (int)n * a.s.c.page_size;
                    }
                    const uint32_t have = __ballot_sync(0xffffffffu, page < a.s.c.num_pages);
                    uint32_t mask[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int w = 0; w < WORDS; ++w) {
                        const int k = w * 32 + lane;
                        mask[w] = __ballot_sync(0xffffffffu, ((have >> (k / a.box)) & 1u) && j * KEYS + k < x.shared);
                    }
                    if (lane == 0) *reinterpret_cast<uint4*>(B.mask[nk % kMasks]) = make_uint4(mask[0], mask[1], mask[2], mask[3]);
                    for (int v = 0; v < 2 && ok; ++v) {
                        const int s = q % NS;
                        if (q >= NS) ok = warp_wait(&B.empty[s], (uint32_t)((q / NS - 1) & 1), err, abort_flag);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&B.full[s], kSlot);
                        __syncwarp();
                        if (lane * a.box < KEYS)
                            for (int kb = 0; kb < KB; ++kb)
                                tma_load_4d(ring + s * kSlot + kb * kTileBlk + lane * a.box * 128, v ? &tv : &tk, kb * 64, row, x.hk, page,
                                            &B.full[s]);
                        ++q;
                    }
                }
            }
            // every copy has landed before the CTA may end
            for (int s = 0; s < min(q, NS); ++s) mbar_wait_bounded(&B.full[s], (uint32_t)(((q - 1 - s) / NS) & 1), err);
        } else if (warp == 6) {
            for (int k = 0; B.next.put(k, x, err, abort_flag, lane); ++k) x = walk.next(a, lane);
        } else if (warp == 7 && blockIdx.x == 0 && lane == 0) {
            keep_error(err);  // a wait gives up after two seconds at the soonest, long after this
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTcManyRegs));
        const int u = (warp >> 2) - 2, q4 = warp & 3, row = q4 * 32 + lane;
        const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
        const uint32_t to = tbase + kColO + lane_off;
        uint8_t* so = stage + (warp - 8) * 4096;
        const float2 sc = make_float2(a.scale2, a.scale2);
        int nt = 0, nk = 0;     // steps of this accumulator; tiles
        uint32_t buffers = 0;  // above 128 columns: a bit per score buffer, parity of its steps
        bool ok = true;
        for (int nq = 0; ok && B.next.get(nq, x, err, abort_flag, lane); ++nq) {
            const bool both = !WIDE && x.rows > 128;
            const int n = WIDE ? (u ? 0 : x.tiles) : both ? x.tiles : (x.tiles + 1 - u) >> 1;
            const int r = (both ? u * 128 : 0) + row;
            const bool some = (both ? u * 128 : 0) + q4 * 32 < x.rows;  // this warp has rows
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < n; ++j, ++nt) {
                const int v = WIDE ? j & 1 : u;  // the score buffer
                if (!(ok = warp_wait(&B.s_full[v], (WIDE ? buffers >> v : (uint32_t)nt) & 1u, err, abort_flag))) break;
                buffers ^= 1u << v;
                if (!some) {
                    if (lane == 0) {
                        mbar_arrive1(&B.p_half[v]);
                        mbar_arrive1(&B.p_ready[v]);
                    }
                    continue;
                }
                const uint32_t ts = tbase + kColS + v * KEYS + lane_off;
                tc_fence_after();
                uint32_t s[KEYS];
#pragma unroll
                for (int c = 0; c < WORDS; ++c) ld32_async(ts + c * 32, s + c * 32);
                const uint4 mask = *reinterpret_cast<const uint4*>(B.mask[(nk + (both || WIDE ? j : 2 * j + u)) % kMasks]);
                wait_ld();
#pragma unroll
                for (int c = 0; c < WORDS; ++c) pin32(s + c * 32);
                if ((WIDE ? mask.x & mask.y : mask.x & mask.y & mask.z & mask.w) != 0xFFFFFFFFu) {
                    const uint32_t see[4] = {mask.x, mask.y, mask.z, mask.w};
#pragma unroll
                    for (int w = 0; w < WORDS; ++w)
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!(see[w] & (1u << c))) s[32 * w + c] = 0xFF800000u;  // -inf
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < KEYS; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                const bool need = (mt - m) * a.scale2 > kGrow;  // true for a row's first key, false while it has none
                if (__any_sync(0xffffffffu, need)) {
                    const float corr = need ? ex2_approx((m - mt) * a.scale2) : 1.0f;
                    l *= corr;
                    if (need) m = mt;
                    if (j > 0) {
                        // the products up to here are complete: this tile's scores were issued behind them, but for
                        // those above 128 columns
                        if (WIDE && !(ok = warp_wait(&B.pv_done, (uint32_t)((nt - 1) & 1), err, abort_flag))) break;
                        if (WIDE) tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < KB * 2; ++c) {
                            uint32_t o[32];
                            ld32_async(to + u * kStepO + c * 32, o);
                            wait_ld();
                            pin32(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                            st32(to + u * kStepO + c * 32, o);
                        }
                    }
                }
                const float ms = (m == -INFINITY ? 0.0f : m) * a.scale2 - kLift<BF>;
                const float2 nm = make_float2(-ms, -ms);
                float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
                for (int half = WIDE ? 1 : 0; half < 2; ++half) {  // the products of the first 64 keys start under the second's exponentials
                    constexpr int H = 32;  // pairs of keys
                    const int c0 = WIDE ? 0 : half * H;
                    uint32_t rest[H];
#pragma unroll
                    for (int i = 0; i < H; ++i) {
                        const int c = c0 + i;
                        float2 e = __ffma2_rn(make_float2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), sc, nm);
                        e.x = ex2_approx(e.x);
                        e.y = ex2_approx(e.y);
                        sum[c & 1] = __fadd2_rn(sum[c & 1], e);
                        s[c] = pack2<BF>(e.x, e.y);
                        const float2 r = minus2<BF>(e, s[c]);  // exact
                        rest[i] = pack2<BF>(r.x, r.y);
                    }
                    st32(ts + c0, s + c0);
                    st32(ts + KEYS / 2 + c0, rest);
                    wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive1(half ? &B.p_ready[v] : &B.p_half[v]);
                }
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            }
            if (!ok || !(ok = warp_wait(&B.o_full, (uint32_t)(nq & 1), err, abort_flag))) break;
            tc_fence_after();
            const bool first = x.j0 == 0;
            if (first && r < x.rows && (both || u == 0)) {
                const unsigned of = x.row0 + r, sq_ = of / (unsigned)a.G;
                a.p.first_later[(long long)(x.s0 + (int)sq_) * a.s.H + x.hk * a.G + (int)(of - sq_ * a.G)] =
                    make_int2(x.behind, (int)(blockIdx.x + 1) * kTcRows + r);
            }
            nk += x.tiles;
            if (!some) {
                tc_fence_before();
                if (lane == 0) {
                    mbar_arrive1(&B.o_empty);
                    mbar_arrive1(&B.written);
                }
                continue;
            }
            // this row's place
            long long at = -1;
            if (r < x.rows) {
                const unsigned of = x.row0 + r, sq_ = of / (unsigned)a.G;
                at = first ? (long long)(x.s0 + (int)sq_) * a.s.H + x.hk * a.G + (int)(of - sq_ * a.G) : (long long)blockIdx.x * kTcRows + r;
            }
            float* po = first ? a.p.first_o : a.p.later_o;
            float2* pml = first ? a.p.first_ml : a.p.later_ml;
            float2 ml = make_float2(m == -INFINITY ? -INFINITY : m * a.scale2 - kLift<BF>, l);
            if (both || WIDE) {
                // an accumulator each, or half of the columns of one
                constexpr int N = WIDE ? 4 : KB * 2;
                const int col0 = WIDE ? u * 128 : 0;
                uint32_t o[N * 32];
#pragma unroll
                for (int c = 0; c < N; ++c) ld32_async(to + u * kStepO + col0 + c * 32, o + c * 32);
                wait_ld();
#pragma unroll
                for (int c = 0; c < N; ++c) pin32(o + c * 32);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive1(&B.o_empty);
                if (at >= 0 && (both || u == 0)) pml[at] = ml;
                const long long place = at >= 0 ? at * a.s.D : -1;
#pragma unroll
                for (int c = 0; c < N; ++c) write_cols(so, o + c * 32, po, place, col0 + c * 32, a.s.D, lane);
                if (lane == 0) mbar_arrive1(&B.written);
                continue;
            }
            // the two accumulators hold the same rows: each softmax takes half of the columns of their sum.  The
            // warps meet by a wait with a limit: one of them may have given up the wait before that the other did not
            float2* mine = reinterpret_cast<float2*>(so);
            const float2* others = reinterpret_cast<const float2*>(stage + ((warp - 8) ^ 4) * 4096);
            mine[lane] = ml;
            __syncwarp();
            if (lane == 0) mbar_arrive1(&B.pair[q4]);
            if (!(ok = warp_wait(&B.pair[q4], 0, err, abort_flag))) break;
            const float2 ot = others[lane];
            __syncwarp();
            if (lane == 0) mbar_arrive1(&B.pair[q4]);
            if (!(ok = warp_wait(&B.pair[q4], 1, err, abort_flag))) break;  // the stage's other use begins
            const float top = fmaxf(ml.x, ot.x), base = top == -INFINITY ? 0.0f : top;
            const float fm = exp2f(ml.x - base), fo = exp2f(ot.x - base);
            const float f0 = u ? fo : fm, f1 = u ? fm : fo;
            if (u == 0 && at >= 0) pml[at] = make_float2(top, ml.y * fm + ot.y * fo);
            const long long place = at >= 0 ? at * a.s.D : -1;
#pragma unroll
            for (int c = 0; c < KB; ++c) {
                const int col = (u * KB + c) * 32;
                uint32_t o[32], p[32];
                ld32_async(to + col, o);
                ld32_async(to + kStepO + col, p);
                wait_ld();
                pin32(o);
                pin32(p);
                if (c == KB - 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive1(&B.o_empty);
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    // an accumulator without a tile holds anything
                    const float y = x.tiles > 1 ? __uint_as_float(p[i]) * f1 : 0.0f;
                    o[i] = __float_as_uint(fmaf(__uint_as_float(o[i]), f0, y));
                }
                write_cols(so, o, po, place, col, a.s.D, lane);
            }
            if (lane == 0) mbar_arrive1(&B.written);
        }
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (warp == 4) tmem_dealloc(tbase, 512);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the pass before, where there is one, has ended too once this one has
}

// [pages][heads][tokens of a page][D] with the cache's strides; boxes of 64 columns x box tokens of a page and
// head, 128-byte swizzle, zeros outside.  A stride of a dimension of one entry is not used and set to a valid value.
bool encode(CUtensorMap* m, const uint8_t* base, const SharedArgs& s, int box) {
    auto enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t rowb = (cuuint64_t)s.D * 2;
    const cuuint64_t dims[4] = {(cuuint64_t)s.D, (cuuint64_t)s.c.page_size, (cuuint64_t)s.HK, (cuuint64_t)s.c.num_pages};
    const cuuint64_t st[3] = {s.c.page_size > 1 ? (cuuint64_t)s.c.token_stride : rowb, s.HK > 1 ? (cuuint64_t)s.c.head_stride : rowb,
                              s.c.num_pages > 1 ? (cuuint64_t)s.c.page_stride : rowb};
    const cuuint32_t sizes[4] = {64u, (cuuint32_t)box, 1u, 1u}, one[4] = {1u, 1u, 1u, 1u};
    return enc(m, s.dtype == RKV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<uint8_t*>(base),
               dims, st, sizes, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// What the kernel was compiled to, asked for until there is an answer; 0: none.
template <int KB, bool BF, bool BOXES>
int registers_of() {
    static std::atomic<int> regs{0};
    if (regs == 0) {
        cudaFuncAttributes f;
        if (cudaFuncGetAttributes(&f, prefix_tc_kernel<KB, BF, BOXES>) == cudaSuccess) regs = f.numRegs;
        else (void)cudaGetLastError();
    }
    return regs;
}
template <int KB, bool BF>
bool usable() {
    const int boxes = registers_of<KB, BF, true>(), rows = registers_of<KB, BF, false>();
    return (boxes == 0 || split_fits(boxes)) && (rows == 0 || split_fits(rows));
}

template <int KB, bool BF, bool BOXES>
int launch_kernel(const Args& a, const CUtensorMap& tk, const CUtensorMap& tv, bool dependent, cudaStream_t st) {
    // the barriers, and up to 1023 bytes of alignment; Q and the ring
    const int smem = 2048 + unit_rows(KB) / 128 * KB * kBlk + ring_slots(KB) * KB * tile_keys(KB) * 128;
    if (!split_fits(registers_of<KB, BF, BOXES>())) return RKV_ERR_CUDA;  // not known
    if (cudaFuncSetAttribute(prefix_tc_kernel<KB, BF, BOXES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
        (void)cudaGetLastError();
        return RKV_ERR_CUDA;
    }
    if (!dependent) {
        prefix_tc_kernel<KB, BF, BOXES><<<kTcSms, kThreads, smem, st>>>(a, tk, tv);
        return launched();
    }
    const cudaError_t e = launch_pdl(prefix_tc_kernel<KB, BF, BOXES>, dim3(kTcSms), dim3(kThreads), smem, st, a, tk, tv);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? RKV_OK : RKV_ERR_CUDA;
}
template <int KB, bool BF>
int launch(Args& a, bool dependent, cudaStream_t st) {
    CUtensorMap tk{}, tv{};
    const int page = a.s.c.page_size & -a.s.c.page_size;  // the largest power of two that divides it
    a.box = page < 8 ? 0 : page < tile_keys(KB) ? page : tile_keys(KB);
    // strides and sizes of a tensor map are bounded; where it cannot be made the copies need none
    if (a.box && a.s.c.num_pages > 0 && encode(&tk, a.s.c.K, a.s, a.box) && encode(&tv, a.s.c.V, a.s, a.box))
        return launch_kernel<KB, BF, true>(a, tk, tv, dependent, st);
    return launch_kernel<KB, BF, false>(a, tk, tv, dependent, st);
}

}  // namespace

bool prefix_tc_usable(int dtype, int D) {
    const bool bf = dtype == RKV_BF16;
    if (D <= 64) return bf ? usable<1, true>() : usable<1, false>();
    if (D <= 128) return bf ? usable<2, true>() : usable<2, false>();
    return bf ? usable<4, true>() : usable<4, false>();
}

int launch_prefix_tc(const SharedArgs& s, const TcParts& p, int spare, bool dependent, cudaStream_t st) {
    Args a{};
    a.s = s;
    a.p = p;
    a.G = s.H / s.HK;
    a.spare = spare < kTcSms / 2 ? spare : kTcSms / 2;
    a.scale2 = 1.4426950408889634f / sqrtf((float)s.D);
    const bool bf = s.dtype == RKV_BF16;
    if (s.D <= 64) return bf ? launch<1, true>(a, dependent, st) : launch<1, false>(a, dependent, st);
    if (s.D <= 128) return bf ? launch<2, true>(a, dependent, st) : launch<2, false>(a, dependent, st);
    return bf ? launch<4, true>(a, dependent, st) : launch<4, false>(a, dependent, st);
}

}  // namespace rkv
