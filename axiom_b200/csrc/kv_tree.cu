// kv_tree.cu — attention of the newest tokens of a ragged batch over its KV cache, fp32 in / fp32 out.  Sequence b holds
// lens[b] cached rows and, behind them, the rows of its n new tokens (drafted for verification: a chain, or a tree given
// by ancestor bits).  For query head h of token t, on key head h / (H / Hkv):
//     out = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale * Q.K_j - max),  j over the cached rows and the new rows t sees.
// A row that sees nothing gives 0.  The tokens and heads that share a key head are the rows of one small product, so K
// and V are read once for all of them: HBM-bound while those rows are few, bound by the tensor cores when they are many.
//
// Both products run as three tf32 products over hi/lo parts (lo.hi + hi.lo + hi.hi, fp32-accurate; hi is the value as it
// lies, of which the tensor core reads the tf32 part, lo the exact remainder) with warp-level mma.m16n8k8: 16 query
// rows fit decode far better than the 128 rows of a tcgen05 tile.  Measured rate of that instruction: 512 multiply-adds
// a clock and SM, so three products of 16 rows need 0.55 of the time in which HBM delivers the keys, of 32 rows 1.1.
// Its layouts cost nothing here:
//   * the contraction index is free, so a lane's 16-byte load of a K row (elements 4t .. 4t+3 of 16) serves two k steps;
//   * the accumulator of Q.K^T (row g, key columns 2t, 2t+1) IS the A operand of P.V with keys 2t, 2t+1 as k = t, t+4;
//   * tiles lie as TMA leaves them (128-byte rows, 16-byte chunks XOR-ed with the row's low bits); key column c of an
//     8-key group is row perm(c) = {0,5,2,7,4,1,6,3}, which makes both the K loads (two rows a phase, their halves
//     of the 128 bytes swapped by bit 2) and the V loads (four rows a phase, two chunks each) conflict-free.
// The tensor core's truncating accumulation never spans more than a tile: every tile's P.V starts from zero and is folded
// into fp32 registers with the online-softmax factor in the same multiply-add.
//
// Work split: the tiles of 64 keys of all (sequence, key head, row block) items form one line, cut into equal pieces,
// one per SM — lengths differ by orders of magnitude in a batch, and the device knows them, not the host.  A piece that
// does not hold an item's whole line leaves (max, sum, unnormalised output) in its workspace slot; the CTA that
// arrives last at the item's counter adds the pieces in line order (nobody waits; the result does not depend on who was
// last) and clears the counter.
//
// One CTA per SM: warp 8 feeds K and V tiles through separate rings; warps 0-7 each own 16 rows x a slice of a tile's
// keys with a running softmax of their own, merged through shared memory at the end of a piece.
#include "kv_tree.cuh"

#include "errors.cuh"
#include "gemm_tc.cuh"
#include "ptx.cuh"
#include "rope.cuh"

#include <cuda.h>
#include <math.h>

namespace axb {

static constexpr int KT_KEYS = 64, KT_CONSUMERS = 8, KT_THREADS = (KT_CONSUMERS + 1) * 32;
static constexpr int KT_MAX_ROWS = 64;   // query rows of an item
enum { TERR_PRODUCER = 91, TERR_CONSUMER = 92 };

// DKP: head dim rounded up to 32 (the tiles' columns beyond dk read as zero).  MT: 16-row tiles of an item.
template <int DKP, int MT>
struct TreeCfg {
    static constexpr int KEYS_WARP = MT == 4 ? 32 : 16;              // keys of a tile that one warp takes
    static constexpr int SLICES = KT_KEYS / KEYS_WARP;               // warps side by side on a tile's keys
    static constexpr int GROUPS = KT_CONSUMERS / (MT * SLICES);      // tiles in work at the same time (2 for one row tile)
    static constexpr int PARTS = SLICES * GROUPS;                    // partial results of a row tile
    static constexpr int NT = KEYS_WARP / 8;
    static constexpr int TILE = KT_KEYS * DKP * 4;                   // bytes of a K or V tile
    static constexpr int MERGE = PARTS * MT * 16 * (DKP + 4 + 2) * 4;
    static constexpr int STAGES = (220 * 1024 - MERGE) / (2 * TILE) < 6 ? (220 * 1024 - MERGE) / (2 * TILE) : 6;
    static constexpr int SMEM = 1024 + STAGES * 2 * TILE + MERGE;
};

struct TreeMaps {
    CUtensorMap k, v;   // [B*Hkv][max_seq][dk], boxes of 32 columns x 64 rows
};

struct TreeSeq {
    int len, n, rows, blocks, tiles;   // cached rows, new tokens, query rows of a key head, row blocks, key tiles
};

__device__ __forceinline__ TreeSeq tree_seq(const KvTreeArgs &a, int b, int block_rows, bool *bad = nullptr)
{
    TreeSeq s;
    s.len = __ldg(a.lens + b);
    s.n = a.n_new ? __ldg(a.n_new + b) : a.T;
    const bool off = s.len < 0 || s.n < 0 || s.n > a.T || (int64_t)s.len + s.n > a.max_seq;
    if (bad) *bad = off;
    if (off) s.len = s.n = 0;   // refused whole: its output rows are left alone
    s.rows = s.n * (a.H / a.Hkv);
    s.blocks = (s.rows + block_rows - 1) / block_rows;
    s.tiles = s.n ? (int)(((int64_t)s.len + s.n + KT_KEYS - 1) / KT_KEYS) : 0;
    return s;
}

__device__ __forceinline__ int64_t tree_tiles(const KvTreeArgs &a, const TreeSeq &s) { return (int64_t)a.Hkv * s.blocks * s.tiles; }

// a CTA's place in the line of tiles
struct TreeCursor {
    int b;
    int64_t off;        // tile inside sequence b's part of the line
    int64_t pos, end;   // tile inside the whole line
};

// one piece: consecutive tiles of one item
struct TreePiece {
    TreeSeq s;
    int b, hk, block, t0, count;
    int64_t item_pos;   // where the item's line starts
};

__device__ __forceinline__ bool next_piece(const KvTreeArgs &a, TreeCursor &c, int block_rows, TreePiece &p)
{
    while (c.pos < c.end) {
        p.s = tree_seq(a, c.b, block_rows);
        const int64_t total = tree_tiles(a, p.s);
        if (c.off >= total) {
            c.off -= total;
            ++c.b;
            continue;
        }
        const int64_t item = c.off / p.s.tiles;
        p.b = c.b;
        p.t0 = (int)(c.off - item * p.s.tiles);
        p.hk = (int)(item / p.s.blocks);
        p.block = (int)(item - (int64_t)p.hk * p.s.blocks);
        const int64_t left = c.end - c.pos;
        p.count = p.s.tiles - p.t0 < left ? p.s.tiles - p.t0 : (int)left;
        p.item_pos = c.pos - p.t0;
        c.off += p.count;
        c.pos += p.count;
        return true;
    }
    return false;
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// what the tensor core does not read of x, exactly
__device__ __forceinline__ uint32_t tf32_rest(float x)
{
    return __float_as_uint(x - __uint_as_float(__float_as_uint(x) & 0xffffe000u));
}

__device__ __forceinline__ float4 lds128(const uint8_t *p) { return *reinterpret_cast<const float4 *>(p); }

// byte offset of 16-byte chunk `chunk` (0..7) of 32-column slab `slab` of row `row` of a tile
__device__ __forceinline__ uint32_t tile_at(int row, int slab, int chunk)
{
    return (uint32_t)(slab * (KT_KEYS * 128) + row * 128 + ((chunk ^ (row & 7)) << 4));
}

// row of an 8-key group behind key column c
__device__ __forceinline__ int key_perm(int c) { return c & 1 ? (c - 1) ^ 5 : c; }

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(KT_CONSUMERS * 32) : "memory"); }

__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// whether token t sees new token j
__device__ __forceinline__ bool tree_sees(const KvTreeArgs &a, int b, int t, int j)
{
    if (!a.mask) return j <= t;
    return (__ldg(a.mask + b * a.mask_stride + (int64_t)t * a.words + (j >> 6)) >> (j & 63)) & 1;
}

template <int DKP, int MT>
struct TreeWarp {
    using C = TreeCfg<DKP, MT>;
    float o[DKP / 32][4][4];    // [slab][e]: rows g, g+8 x columns 32*slab + 8t + e and + 4
    float m[2], l[2];           // running maximum (log2 domain) and this lane's part of the sum
};

// One tile for one warp: its 16 rows against KEYS_WARP keys.  TAIL: the tile holds rows behind the cached ones.
template <int DKP, int MT, bool TAIL>
__device__ __forceinline__ void tree_tile(const KvTreeArgs &a, TreeWarp<DKP, MT> &w, const uint8_t *qbase, const uint8_t *kbase, const uint8_t *vbase, int key0, const TreeSeq &s,
                                          int b, int tok_a, int tok_b, uint32_t v_full, uint32_t v_parity, bool &ok)
{
    using C = TreeCfg<DKP, MT>;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int slice = (threadIdx.x >> 5) / MT % C::SLICES, row0 = slice * C::KEYS_WARP;
    float sc[C::NT][4];
#pragma unroll
    for (int i = 0; i < C::NT; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
    const int krow = row0 + key_perm(g);
#pragma unroll
    for (int j = 0; j < DKP / 16; ++j) {
        const float4 qa = lds128(qbase + (2 * j) * 512), qb = lds128(qbase + (2 * j + 1) * 512);   // rows g, g+8: elements 16j + 4t .. +3
        // [k step]: rows g, g+8 at k = t, then at k = t + 4
        const float x[2][4] = { { qa.x, qb.x, qa.y, qb.y }, { qa.z, qb.z, qa.w, qb.w } };
        uint32_t hi[2][4], lo[2][4];
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[st][e] = __float_as_uint(x[st][e]);
                lo[st][e] = tf32_rest(x[st][e]);
            }
#pragma unroll
        for (int i = 0; i < C::NT; ++i) {
            const float4 k4 = lds128(kbase + tile_at(krow + 8 * i, j >> 1, 4 * (j & 1) + t));
            const uint32_t h[4] = { __float_as_uint(k4.x), __float_as_uint(k4.y), __float_as_uint(k4.z), __float_as_uint(k4.w) };
            const uint32_t r[4] = { tf32_rest(k4.x), tf32_rest(k4.y), tf32_rest(k4.z), tf32_rest(k4.w) };
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                mma_tf32(sc[i], lo[st], h[2 * st], h[2 * st + 1]);
                mma_tf32(sc[i], hi[st], r[2 * st], r[2 * st + 1]);
                mma_tf32(sc[i], hi[st], h[2 * st], h[2 * st + 1]);
            }
        }
    }
    // scores in the log2 domain, the row maxima, the factor on what was summed before
    float mx[2] = { -INFINITY, -INFINITY };
#pragma unroll
    for (int i = 0; i < C::NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = sc[i][e] * a.c_log2;
            if (TAIL) {
                const int j = key0 + row0 + 8 * i + key_perm(2 * t + (e & 1)) - s.len;   // < 0: a cached row
                if (j >= 0 && (j >= s.n || !tree_sees(a, b, e < 2 ? tok_a : tok_b, j))) x = -INFINITY;
            }
            sc[i][e] = x;
            mx[e >> 1] = fmaxf(mx[e >> 1], x);
        }
    float corr[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
        const float m_new = fmaxf(w.m[r], mx[r]);
        const float base = m_new == -INFINITY ? 0.f : m_new;   // nothing seen so far: every p below is 2^-inf = 0
        corr[r] = ex2_approx(w.m[r] - base);
        w.m[r] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < C::NT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float p = ex2_approx(sc[i][2 * r + e] - base);
                sc[i][2 * r + e] = p;
                sum += p;
            }
        w.l[r] = w.l[r] * corr[r] + sum;
    }
    if (ok && !__all_sync(0xffffffffu, mbar_wait_bounded(v_full, v_parity))) ok = false;
    if (!ok) return;
    // O = O * corr + P.V, the tile's product from zero
    bool odd = false;   // a value behind the cached rows that is not finite
#pragma unroll
    for (int sl = 0; sl < DKP / 32; ++sl) {
        float acc[4][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e][0] = acc[e][1] = acc[e][2] = acc[e][3] = 0.f;
#pragma unroll
        for (int i = 0; i < C::NT; ++i) {
            const int ra = row0 + 8 * i + key_perm(2 * t), rb = row0 + 8 * i + key_perm(2 * t + 1);
            float4 va = lds128(vbase + tile_at(ra, sl, g)), vb = lds128(vbase + tile_at(rb, sl, g));
            if (TAIL) {
                // rows behind the last one hold anything, and rows that only some tokens see must not reach the others
                // through 0 * inf: such values leave the product and are added below
                float *x = &va.x, *y = &vb.x;
                const int ja = key0 + ra - s.len, jb = key0 + rb - s.len;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (ja >= 0 && !(ja < s.n && finite_f(x[e]))) { odd = odd || ja < s.n; x[e] = 0.f; }
                    if (jb >= 0 && !(jb < s.n && finite_f(y[e]))) { odd = odd || jb < s.n; y[e] = 0.f; }
                }
            }
            const uint32_t phi[4] = { __float_as_uint(sc[i][0]), __float_as_uint(sc[i][2]), __float_as_uint(sc[i][1]), __float_as_uint(sc[i][3]) };
            const uint32_t plo[4] = { tf32_rest(sc[i][0]), tf32_rest(sc[i][2]), tf32_rest(sc[i][1]), tf32_rest(sc[i][3]) };
            const float *x = &va.x, *y = &vb.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t h0 = __float_as_uint(x[e]), h1 = __float_as_uint(y[e]);
                mma_tf32(acc[e], plo, h0, h1);
                mma_tf32(acc[e], phi, tf32_rest(x[e]), tf32_rest(y[e]));
                mma_tf32(acc[e], phi, h0, h1);
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w.o[sl][e][0] = fmaf(w.o[sl][e][0], corr[0], acc[e][0]);
            w.o[sl][e][1] = fmaf(w.o[sl][e][1], corr[0], acc[e][1]);
            w.o[sl][e][2] = fmaf(w.o[sl][e][2], corr[1], acc[e][2]);
            w.o[sl][e][3] = fmaf(w.o[sl][e][3], corr[1], acc[e][3]);
        }
    }
    if (TAIL && __any_sync(0xffffffffu, odd)) {
        // rare: an infinity or a NaN among the new rows' values goes to the rows that see it, and to no others
#pragma unroll 1
        for (int key = 0; key < C::KEYS_WARP; ++key) {
            const int j = key0 + row0 + key - s.len;
            if (j < 0 || j >= s.n) continue;
            const bool see_a = tree_sees(a, b, tok_a, j), see_b = tree_sees(a, b, tok_b, j);
#pragma unroll
            for (int sl = 0; sl < DKP / 32; ++sl)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 v4 = lds128(vbase + tile_at(row0 + key, sl, 2 * t + h));
                    const float *x = &v4.x;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!finite_f(x[e])) {
                            if (see_a) w.o[sl][e][h] += x[e];
                            if (see_b) w.o[sl][e][2 + h] += x[e];
                        }
                }
        }
    }
}

// slot of the workspace: [rows][DKP] outputs, then [rows] maxima and [rows] sums
template <int DKP, int MT>
__device__ __forceinline__ float *tree_slot(const KvTreeArgs &a, int slot)
{
    return a.slots + (size_t)slot * (MT * 16) * (DKP + 2);
}

template <int DKP, int MT>
__global__ void __launch_bounds__(KT_THREADS, 1) kv_tree_kernel(const __grid_constant__ KvTreeArgs a, const __grid_constant__ TreeMaps tm, int tma)
{
    using C = TreeCfg<DKP, MT>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(8) uint64_t bars[4 * C::STAGES];
    __shared__ unsigned long long s_total;
    __shared__ int s_b, s_last;
    __shared__ long long s_off;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t *const tiles = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);   // the swizzle is a function of the address
    float *merge = reinterpret_cast<float *>(tiles + C::STAGES * 2 * C::TILE);
    const uint32_t bar0 = smem_u32(bars);
    auto bar = [&](int kind, int stage) { return bar0 + 8u * (kind * C::STAGES + stage); };   // 0 K full, 1 K empty, 2 V full, 3 V empty
    auto ktile = [&](int stage) { return tiles + stage * 2 * C::TILE; };
    if (tid == 0) {
        s_total = 0;
        for (int s = 0; s < C::STAGES; ++s)
            for (int k = 0; k < 4; ++k) mbar_init(bar(k, s), k & 1 ? MT * C::SLICES : (tma ? 1 : 32));
        mbar_fence_init();
    }
    __syncthreads();

    // the line of tiles, this CTA's part of it, and the sequence that part starts in
    constexpr int ROWS = MT * 16;
    {
        unsigned long long sum = 0;
        for (int b = tid; b < a.B; b += KT_THREADS) {
            bool bad;
            const TreeSeq s = tree_seq(a, b, ROWS, &bad);
            sum += (unsigned long long)tree_tiles(a, s);
            if (bad && blockIdx.x == 0 && a.err) atomicCAS(a.err, 0, (int)AXB_DEVERR_ROWS);
        }
        if (sum) atomicAdd(&s_total, sum);
        __syncthreads();
    }
    const int64_t total = (int64_t)s_total, per = (total + gridDim.x - 1) / gridDim.x;
    TreeCursor cur;
    cur.pos = per * blockIdx.x;
    cur.end = cur.pos + per < total ? cur.pos + per : total;
    if (cur.pos >= cur.end) return;
    if (warp == 0) {
        int64_t before = 0;
        for (int b0 = 0; b0 < a.B; b0 += 32) {
            const int64_t mine = b0 + lane < a.B ? tree_tiles(a, tree_seq(a, b0 + lane, ROWS)) : 0;
            int64_t upto = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + upto > cur.pos);
            if (past) {
                const int k = __ffs(past) - 1;
                if (lane == k) {
                    s_b = b0 + k;
                    s_off = cur.pos - (before + upto - mine);
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
    }
    __syncthreads();
    cur.b = s_b;
    cur.off = s_off;
    TreePiece p;
    bool ok = true;
    uint32_t it = 0;   // tiles since the start: ring stage it % STAGES, phase it / STAGES

    if (warp == KT_CONSUMERS) {
        // ---- producer
        while (ok && next_piece(a, cur, ROWS, p)) {
            const int head = p.b * a.Hkv + p.hk;
            for (int i = 0; ok && i < p.count; ++i, ++it) {
                const int s = it % C::STAGES, row = (p.t0 + i) * KT_KEYS;
                const uint32_t ph = (it / C::STAGES) & 1;
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    if (it >= C::STAGES && !__all_sync(0xffffffffu, mbar_wait_bounded(bar(2 * v + 1, s), ph ^ 1))) { ok = false; break; }
                    const uint32_t full = bar(2 * v, s), dst = smem_u32(ktile(s)) + v * C::TILE;
                    if (tma) {
                        if (lane == 0) {
                            mbar_arrive_expect_tx(full, C::TILE);
#pragma unroll
                            for (int sl = 0; sl < DKP / 32; ++sl) tma_load_3d(dst + sl * (KT_KEYS * 128), v ? &tm.v : &tm.k, full, 32 * sl, row, head);
                        }
                    } else {
                        // tensors that a tensor map cannot describe: the same layout, four bytes at a time
                        const float *src = (v ? a.V : a.K) + (int64_t)head * a.max_seq * a.dk;
                        for (int r = 0; r < KT_KEYS; ++r) {
                            const bool in = (int64_t)row + r < a.max_seq;
#pragma unroll
                            for (int sl = 0; sl < DKP / 32; ++sl) {
                                const int c = 32 * sl + lane;
                                const bool get = in && c < a.dk;
                                const float *from = get ? src + ((int64_t)row + r) * a.dk + c : src;
                                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + tile_at(r, sl, lane >> 2) + 4 * (lane & 3)),
                                             "l"(from), "r"(get ? 4 : 0)
                                             : "memory");
                            }
                        }
                        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full) : "memory");
                    }
                }
            }
        }
        if (!ok) {
            if (lane == 0 && a.err) atomicCAS(a.err, 0, (int)TERR_PRODUCER);
            // copies in flight land before the CTA's memory goes away
            for (int s = 0; s < C::STAGES; ++s)
                for (int k = 0; k <= 2; k += 2) mbar_wait_bounded(bar(k, s), ((it >= (uint32_t)s ? it - s : 0) / C::STAGES) & 1);
        }
        return;
    }

    // ---- consumers
    const int g = lane >> 2, t = lane & 3, rt = warp % MT, part = warp / MT, grp = part / C::SLICES;
    const int heads_per = a.H / a.Hkv;
    TreeWarp<DKP, MT> w;
    while (next_piece(a, cur, ROWS, p)) {
        const int r0 = p.block * ROWS + rt * 16;
        // query row r: head r / n of the group, token r % n
        const int ra = r0 + g, rb = r0 + g + 8;
        const int ga = ra / p.s.n, gb = rb / p.s.n, tok_a = ra < p.s.rows ? ra - ga * p.s.n : 0, tok_b = rb < p.s.rows ? rb - gb * p.s.n : 0;
        const bool idle = r0 >= p.s.rows;
        // the rows' Q as the lanes will read it, in the merge area: [row tile][16-column group][rows g | g + 8][lane]
        for (int i = tid; i < ROWS * (DKP / 4); i += KT_CONSUMERS * 32) {
            const int r = i / (DKP / 4), c = i - r * (DKP / 4), row = p.block * ROWS + r;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (row < p.s.rows) {
                const int gh = row / p.s.n;
                const float *src = a.Q + (((int64_t)p.b * a.H + p.hk * heads_per + gh) * a.T + (row - gh * p.s.n)) * a.dk + 4 * c;
                if (tma) {   // rows are whole 16-byte pieces
                    if (4 * c < a.dk) x = __ldg(reinterpret_cast<const float4 *>(src));
                } else {
                    if (4 * c < a.dk) x.x = __ldg(src);
                    if (4 * c + 1 < a.dk) x.y = __ldg(src + 1);
                    if (4 * c + 2 < a.dk) x.z = __ldg(src + 2);
                    if (4 * c + 3 < a.dk) x.w = __ldg(src + 3);
                }
            }
            reinterpret_cast<float4 *>(merge)[((r >> 4) * (DKP / 16) + (c >> 2)) * 64 + ((r >> 3) & 1) * 32 + (r & 7) * 4 + (c & 3)] = x;
        }
        const uint8_t *qbase = reinterpret_cast<const uint8_t *>(merge) + rt * (DKP / 16) * 1024 + lane * 16;
        w.m[0] = w.m[1] = -INFINITY;
        w.l[0] = w.l[1] = 0.f;
#pragma unroll
        for (int sl = 0; sl < DKP / 32; ++sl)
#pragma unroll
            for (int e = 0; e < 4; ++e) w.o[sl][e][0] = w.o[sl][e][1] = w.o[sl][e][2] = w.o[sl][e][3] = 0.f;
        consumers_sync();

        for (int i = 0; i < p.count; ++i, ++it) {
            if (C::GROUPS > 1 && (int)(it % C::GROUPS) != grp) continue;
            const int s = it % C::STAGES;
            const uint32_t ph = (it / C::STAGES) & 1;
            const int key0 = (p.t0 + i) * KT_KEYS;
            if (ok && !__all_sync(0xffffffffu, mbar_wait_bounded(bar(0, s), ph))) ok = false;
            if (ok && !idle) {
                // (the last column of a 32-bit key index: key0 <= max_seq < 2^31)
                if (key0 + KT_KEYS > p.s.len)
                    tree_tile<DKP, MT, true>(a, w, qbase, ktile(s), ktile(s) + C::TILE, key0, p.s, p.b, tok_a, tok_b, bar(2, s), ph, ok);
                else
                    tree_tile<DKP, MT, false>(a, w, qbase, ktile(s), ktile(s) + C::TILE, key0, p.s, p.b, tok_a, tok_b, bar(2, s), ph, ok);
            } else if (ok) {
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar(2, s), ph))) ok = false;
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bar(1, s));
                mbar_arrive(bar(3, s));
            }
        }

        consumers_sync();   // Q has been read
        // ---- merge the warps' parts: [part][row][DKP + 4] outputs, then [part][row] maxima and sums
        float *mo = merge, *mm = merge + C::PARTS * ROWS * (DKP + 4), *ml = mm + C::PARTS * ROWS;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float sum = w.l[h];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const int row = part * ROWS + rt * 16 + g + 8 * h;
            if (t == 0) {
                mm[row] = w.m[h];
                ml[row] = sum;
            }
#pragma unroll
            for (int sl = 0; sl < DKP / 32; ++sl)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    *reinterpret_cast<float4 *>(mo + row * (DKP + 4) + 32 * sl + 8 * t + 4 * c) =
                        make_float4(w.o[sl][0][2 * h + c], w.o[sl][1][2 * h + c], w.o[sl][2][2 * h + c], w.o[sl][3][2 * h + c]);
        }
        consumers_sync();
        const int rows_here = p.s.rows - p.block * ROWS < ROWS ? p.s.rows - p.block * ROWS : ROWS;
        const bool whole = p.count == p.s.tiles;
        // the item's pieces belong to consecutive CTAs; the first one's index names its counter
        const int first = (int)(p.item_pos / per), pieces = (int)((p.item_pos + p.s.tiles - 1) / per) - first + 1;
        float *slot = tree_slot<DKP, MT>(a, 2 * (int)blockIdx.x + (p.t0 == 0 ? 1 : 0));
        auto store_out = [&](int r, int c, float4 y) {
            const int row = p.block * ROWS + r, gh = row / p.s.n, tok = row - gh * p.s.n;
            float *dst = a.out + (((int64_t)p.b * a.H + p.hk * heads_per + gh) * a.T + tok) * a.dk + c;
            if (tma) {
                *reinterpret_cast<float4 *>(dst) = y;
            } else {
                const float *v = &y.x;
                for (int e = 0; e < 4; ++e)
                    if (c + e < a.dk) dst[e] = v[e];
            }
        };
        for (int i = tid; i < rows_here * (DKP / 4); i += KT_CONSUMERS * 32) {
            const int r = i / (DKP / 4), c = (i - r * (DKP / 4)) * 4;
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int k = 0; k < C::PARTS; ++k) M = fmaxf(M, mm[k * ROWS + r]);
            const float base = M == -INFINITY ? 0.f : M;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < C::PARTS; ++k) {
                const float f = ex2_approx(mm[k * ROWS + r] - base);
                const float4 v = *reinterpret_cast<const float4 *>(mo + (k * ROWS + r) * (DKP + 4) + c);
                L = fmaf(f, ml[k * ROWS + r], L);
                y.x = fmaf(f, v.x, y.x); y.y = fmaf(f, v.y, y.y); y.z = fmaf(f, v.z, y.z); y.w = fmaf(f, v.w, y.w);
            }
            if (whole) {
                if (c >= a.dk) continue;
                const float inv = L == 0.f ? 0.f : 1.0f / L;   // nothing seen: 0
                store_out(r, c, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
            } else {
                *reinterpret_cast<float4 *>(slot + r * DKP + c) = y;
                if (c == 0) {
                    slot[ROWS * DKP + r] = M;
                    slot[ROWS * DKP + ROWS + r] = L;
                }
            }
        }
        if (!whole) {
            __threadfence();
            consumers_sync();
            if (tid == 0) s_last = atomicAdd(a.counters + first, 1) == pieces - 1;
            consumers_sync();
            if (s_last) {
                __threadfence();
                for (int i = tid; i < rows_here * (DKP / 4); i += KT_CONSUMERS * 32) {
                    const int r = i / (DKP / 4), c = (i - r * (DKP / 4)) * 4;
                    if (c >= a.dk) continue;
                    float M = -INFINITY, L = 0.f;
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                    for (int k = 0; k < pieces; ++k) {
                        const float *src = tree_slot<DKP, MT>(a, 2 * (first + k) + (k == 0 ? 1 : 0));
                        const float mk = __ldcg(src + ROWS * DKP + r), lk = __ldcg(src + ROWS * DKP + ROWS + r);
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(src + r * DKP + c));
                        const float m_new = fmaxf(M, mk), base = m_new == -INFINITY ? 0.f : m_new;
                        const float f0 = ex2_approx(M - base), f1 = ex2_approx(mk - base);
                        M = m_new;
                        L = L * f0 + lk * f1;
                        y.x = y.x * f0 + v.x * f1; y.y = y.y * f0 + v.y * f1; y.z = y.z * f0 + v.z * f1; y.w = y.w * f0 + v.w * f1;
                    }
                    const float inv = L == 0.f ? 0.f : 1.0f / L;
                    store_out(r, c, make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv));
                }
                if (tid == 0) a.counters[first] = 0;
            }
        }
        consumers_sync();   // the merge area is free again
    }
    if (!ok && lane == 0 && a.err) atomicCAS(a.err, 0, (int)TERR_CONSUMER);
}

template <int VEC>
struct Vec;
template <>
struct Vec<4> {
    float4 v;
};
template <>
struct Vec<1> {
    float v;
};

// Accepted rows: a thread owns one 16-byte (or 4-byte) column piece of one head of one cache and walks the list in order;
// the list ascends, so a row is read before the walk overwrites it and no thread meets another.
template <int VEC>
__global__ void __launch_bounds__(256) kv_compact_kernel(float *K, float *V, const int32_t *keep, const int32_t *n_keep, const int32_t *lens,
                                                         int32_t *lens_out, int Hkv, int T, int64_t max_seq, int dk, int *err)
{
    const int b = blockIdx.x;
    const int len = lens[b], n = n_keep[b];
    keep += (int64_t)b * T;
    bool bad = len < 0 || n < 0 || n > T;
    if (!bad)
        for (int i = threadIdx.x; i < n; i += 256) {
            const int k = keep[i], prev = i ? keep[i - 1] : -1;
            bad = bad || k <= prev || k >= T || (int64_t)len + k >= max_seq;
        }
    bad = __syncthreads_or(bad);
    if (blockIdx.y == 0 && threadIdx.x == 0) {
        if (bad && err) atomicCAS(err, 0, (int)AXB_DEVERR_KEEP);
        if (lens_out) lens_out[b] = bad ? len : len + n;
    }
    if (bad) return;   // refused whole
    const int pieces = dk / VEC, per_cache = Hkv * pieces;
    for (int i = blockIdx.y * 256 + threadIdx.x; i < 2 * per_cache; i += gridDim.y * 256) {
        const int c = i < per_cache ? i : i - per_cache, h = c / pieces;
        float *base = (i < per_cache ? K : V) + (((int64_t)b * Hkv + h) * max_seq + len) * dk + (c - h * pieces) * VEC;
        constexpr int UN = 8;
        for (int j = 0; j < n; j += UN) {
            Vec<VEC> x[UN];
            int from[UN];
#pragma unroll
            for (int k = 0; k < UN; ++k) from[k] = j + k < n ? __ldg(keep + j + k) : -1;
#pragma unroll
            for (int k = 0; k < UN; ++k)
                if (from[k] > j + k) x[k] = *reinterpret_cast<const Vec<VEC> *>(base + (int64_t)from[k] * dk);
#pragma unroll
            for (int k = 0; k < UN; ++k)
                if (from[k] > j + k) *reinterpret_cast<Vec<VEC> *>(base + (int64_t)(j + k) * dk) = x[k];
        }
    }
}

// ---------------------------------------------------------------------- host

static inline bool kt_aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

size_t kv_tree_workspace_bytes(int sm_count)
{
    return (size_t)sm_count * 2 * KT_MAX_ROWS * (128 + 2) * sizeof(float);
}

template <int DKP, int MT>
static int launch_tree(const KvTreeArgs &a, const TreeMaps &tm, int tma, int sm_count, cudaStream_t st)
{
    using C = TreeCfg<DKP, MT>;
    static_assert(C::STAGES >= 2 && C::SMEM <= 227 * 1024, "shared memory");
    static_assert(MT * 16 <= KT_MAX_ROWS && DKP <= 128, "workspace slots");
    static PerDeviceOnce once;
    if (once.first()) {
        cudaError_t e = cudaFuncSetAttribute(kv_tree_kernel<DKP, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
    }
    kv_tree_kernel<DKP, MT><<<sm_count, KT_THREADS, C::SMEM, st>>>(a, tm, tma);
    return (int)cudaGetLastError();
}

template <int MT>
static int launch_tree_mt(const KvTreeArgs &a, const TreeMaps &tm, int tma, int sm_count, cudaStream_t st)
{
    if (a.dk <= 32) return launch_tree<32, MT>(a, tm, tma, sm_count, st);
    if (a.dk <= 64) return launch_tree<64, MT>(a, tm, tma, sm_count, st);
    if (a.dk <= 96) return launch_tree<96, MT>(a, tm, tma, sm_count, st);
    return launch_tree<128, MT>(a, tm, tma, sm_count, st);
}

int launch_kv_cache_attend_tree(const KvTreeArgs &a, int sm_count, cudaStream_t st)
{
    const int tma = a.dk % 4 == 0 && kt_aligned16(a.K) && kt_aligned16(a.V) && kt_aligned16(a.Q) && kt_aligned16(a.out);
    TreeMaps tm = {};
    if (tma) {
        int e = encode_f32_batched_tmap(&tm.k, a.K, (int64_t)a.B * a.Hkv, a.max_seq, a.dk, a.dk, KT_KEYS, false);
        if (!e) e = encode_f32_batched_tmap(&tm.v, a.V, (int64_t)a.B * a.Hkv, a.max_seq, a.dk, a.dk, KT_KEYS, false);
        if (e) return e;
    }
    const int64_t rows = (int64_t)(a.H / a.Hkv) * a.T;   // of a key head, if every token is there
    if (rows <= 16) return launch_tree_mt<1>(a, tm, tma, sm_count, st);
    if (rows <= 32) return launch_tree_mt<2>(a, tm, tma, sm_count, st);
    return launch_tree_mt<4>(a, tm, tma, sm_count, st);
}

int launch_kv_cache_compact(float *K, float *V, const int32_t *keep, const int32_t *n_keep, const int32_t *lens, int32_t *lens_out,
                            int64_t B, int64_t Hkv, int64_t T, int64_t max_seq, int64_t dk, int *err, cudaStream_t st)
{
    const bool vec = dk % 4 == 0 && kt_aligned16(K) && kt_aligned16(V);
    const int64_t items = 2 * Hkv * (vec ? dk / 4 : dk);
    int64_t y = (items + 255) / 256;
    if (y > 64) y = 64;
    const dim3 grid((unsigned)B, (unsigned)y);
    if (vec) kv_compact_kernel<4><<<grid, 256, 0, st>>>(K, V, keep, n_keep, lens, lens_out, (int)Hkv, (int)T, max_seq, (int)dk, err);
    else kv_compact_kernel<1><<<grid, 256, 0, st>>>(K, V, keep, n_keep, lens, lens_out, (int)Hkv, (int)T, max_seq, (int)dk, err);
    return (int)cudaGetLastError();
}

}  // namespace axb
