// kv_tree.cu — attention of the newest tokens of a ragged batch over its KV cache, fp32 in / fp32 out.  Sequence b holds
// lens[b] cached rows and, behind them, the rows of its n new tokens (drafted for verification: a chain, or a tree given
// by ancestor bits).  For query head h of token t, on key head h / (H / Hkv):
//     out = sum_j p_j V_j / sum_j p_j,  p_j = exp(scale * Q.K_j - max),  j over the cached rows and the new rows t sees.
// A row that sees nothing gives 0.  The tokens and heads that share a key head are the rows of one small product, so K
// and V are read once for all of them: HBM-bound while those rows are few, bound by the tensor cores when they are many.
//
// Both products run transposed, S^T = K.Q^T and O^T = V^T.P^T, as three tf32 products over hi/lo parts (lo.hi + hi.lo +
// hi.hi, fp32-accurate) with warp-level mma.m16n8k8: keys (and head dims) fill the 16 side, query rows come in eights —
// a decode step has 1 to 32 of them, far from the 128 rows of a tcgen05 tile.  Measured rate of that instruction: 512
// multiply-adds a clock and SM, so three products of 8 rows take 0.27 of the time in which HBM delivers the keys, of 32
// rows 1.1.  Every element of K and V is split once for all rows of the warp.  The layouts cost nothing:
//   * the contraction index is free, so a lane's 16-byte load of a K row (elements 4t .. 4t+3 of 16) serves two k steps, and
//     that of a V row (columns 4g .. 4g+3 of 32) serves rows g and g+8 of two 16-column tiles;
//   * tiles lie as TMA leaves them (128-byte rows, 16-byte chunks XOR-ed with the row's low bits).  Row g of an 8-key
//     group is key perm(g) = {0,5,2,7,4,1,6,3}: the two rows of a load phase then differ in bit 2 and take the two halves
//     of the 128 bytes; V is read in key order (2t, 2t+1 as k = t, t+4), four rows a phase, two chunks each.  Neither
//     meets a bank twice;
//   * P^T changes from accumulator to operand layout with two shuffles a value inside the warp.
// The tensor core's truncating accumulation never spans more than 16 keys: P.V starts from zero every time and is folded
// into fp32 registers with the online-softmax factor in the same multiply-add.
//
// Work split: the tiles of 32 keys of all (sequence, key head, row block) items form one line, cut into equal pieces,
// one per SM (kv_tree_line.cuh) — lengths differ by orders of magnitude in a batch, and the device knows them, not the
// host.  A piece that does not hold an item's whole line leaves (max, sum, unnormalised output) in its workspace slot; the
// CTA that arrives last at the item's counter adds the pieces in line order (nobody waits; the result does not depend on
// who was last) and clears the counter.
//
// One CTA per SM: two producer warps feed K and V tiles through a ring; eight warps each take 16 keys of a tile with
// a running softmax of their own, added up at the end of a piece — up to 8 rows (16 of narrower heads) by a merger warp
// while the eight are at the next piece, which a scout warp has prepared.  32 sequences of 400 to 4100 rows, 8 key heads of 128
// (592 MB): 98 us, 6.0 TB/s, 0.92 of the copy bandwidth; without scout and merger 117.
#include "kv_tree.cuh"

#include "errors.cuh"
#include "gemm_tc.cuh"
#include "kv_tree_line.cuh"
#include "ptx.cuh"

#include <cuda.h>
#include <math.h>

namespace axb {

static constexpr int KT_KEYS = 32, KT_CONSUMERS = 8;
enum { TERR_PRODUCER = 91, TERR_CONSUMER = 92 };

// DKP: head dim rounded up to 32 (the tiles' columns beyond dk read as zero).  NR: query rows of an item, in eights.
template <int DKP, int NR>
struct TreeCfg {
    static constexpr int ROWS = 8 * NR;                          // query rows of an item
    static constexpr int SLICES = KT_KEYS / 16;                       // warps side by side on a tile's keys
    static constexpr int GROUPS = KT_CONSUMERS / SLICES;              // tiles in work at the same time
    static constexpr int FRAGS = DKP / 16 * NR;                       // float4 of a lane's O^T
    // Decode and small trees (ASYNC): a scout warp prepares the next piece (its place in the batch, its Q) and a merger warp
    // adds up and writes the finished one while the consumers go on; otherwise the consumers do both themselves, between
    // barriers (each costs a piece some 7,000 cycles, in which the ring stands still).
    static constexpr bool ASYNC = NR == 1 || (NR == 2 && DKP <= 96);
    // From one item to the next a CTA takes the time of several tiles (256 sequences of 280 rows, 8 key heads of 128, 599 MB: no
    // room for it on the line 173 us, 3 tiles 154, 5 140, 8 139; of 64: 97, -, 80, 80).
    static constexpr int GAP = ASYNC ? 5 : 8;
    static constexpr bool SPLIT_Q = NR < 4;                           // Q lies in shared memory as hi and lo
    static constexpr int TILE = KT_KEYS * DKP * 4;                    // bytes of a K or V tile
    static constexpr int Q_BYTES = ROWS * DKP * 4 * (SPLIT_Q ? 2 : 1);
    static constexpr int PART_BYTES = 32 * (FRAGS + NR) * 16;         // a warp's partial result
    static constexpr int MERGE_BYTES = KT_CONSUMERS / (ASYNC ? 1 : 2) * PART_BYTES;
    static constexpr int AREA = ASYNC ? 2 * Q_BYTES + MERGE_BYTES : Q_BYTES > MERGE_BYTES ? Q_BYTES : MERGE_BYTES;   // else first Q, then the merge
    // A stage always belongs to the same group of warps: a barrier's phases are then waited for in order by the same threads.
    // (Four stages carry HBM's rate, six were slower: 90 against 95 us for 537 MB.)
    static constexpr int ROOM = (224 * 1024 - AREA) / (2 * TILE) / GROUPS * GROUPS;
    static constexpr int STAGES = ROOM < 2 * GROUPS && ROOM > 0 ? ROOM : TILE <= 8192 ? 2 * GROUPS : GROUPS;
    static_assert(STAGES % GROUPS == 0 && STAGES <= ROOM, "ring");
    static constexpr int SMEM = 1024 + STAGES * 2 * TILE + AREA;
    // four rows in eights and 128 columns need more than the 168 registers that twelve warps leave a thread: the four
    // others hand theirs to the consumers
    static constexpr bool SHIFT_REGS = !ASYNC;
    static constexpr int THREADS = (KT_CONSUMERS + 4) * 32;
};

struct TreeMaps {
    CUtensorMap k, v;   // [B*Hkv][max_seq][dk], boxes of 32 columns x 32 rows
};

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float4 lds128(const uint8_t *p) { return *reinterpret_cast<const float4 *>(p); }

// byte offset of 16-byte chunk `chunk` (0..7) of 32-column slab `slab` of row `row` of a tile
__device__ __forceinline__ uint32_t tile_at(int row, int slab, int chunk)
{
    return (uint32_t)(slab * (KT_KEYS * 128) + row * 128 + ((chunk ^ (row & 7)) << 4));
}

// key behind row g of an 8-key group of S^T
__device__ __forceinline__ int key_perm(int g) { return g & 1 ? g ^ 4 : g; }

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(KT_CONSUMERS * 32) : "memory"); }

// What a lane (g = lane / 4, t = lane % 4) holds of its warp's query rows.  o[i][n]: columns 32*(i/2) + 4g + 2*(i%2) (elements
// 0: row 8n + 2t, 1: row 8n + 2t + 1) and the column behind it (elements 2, 3).
template <int DKP, int NR>
struct TreeWarp {
    float o[DKP / 16][NR][4];
    float m[NR][2], l[NR][2];   // running maximum (log2 domain) and sum of rows 8n + 2t, 8n + 2t + 1; l of this lane's keys
};

// One warp, 16 keys.  TAIL: some of them lie behind the cached rows.  toks: the token of each of the warp's query rows.
template <int DKP, int NR, bool TAIL>
__device__ __forceinline__ void tree_tile(const KvTreeArgs &a, TreeWarp<DKP, NR> &w, const uint8_t *qbase, const uint8_t *kbase, const uint8_t *vbase,
                                          int key0, int row0, const TreeSeq &s, int b, const int *toks, uint32_t k_empty, uint32_t v_full,
                                          uint32_t v_parity, bool &ok)
{
    using C = TreeCfg<DKP, NR>;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    // S^T: rows g, g+8 = keys row0 + perm(g) (+ 8), columns 2t, 2t+1 of each eight query rows; the cross products in chains of
    // their own, which shortens the dependent chain
    // (and the sum of the large ones in two: every accumulation cuts its sum off)
    constexpr int CH = NR <= 2 ? 2 : 1;
    float sc[NR][4], sc1[CH == 2 ? NR : 1][4], x1[NR][4], x2[NR == 1 ? NR : 1][4];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sc[n][e] = x1[n][e] = 0.f;
            if (CH == 2) sc1[CH == 2 ? n : 0][e] = 0.f;
            if (NR == 1) x2[0][e] = 0.f;
        }
    const int krow = row0 + key_perm(g);
#pragma unroll 2
    for (int j = 0; j < DKP / 16; ++j) {
        const float4 ka = lds128(kbase + tile_at(krow, j >> 1, 4 * (j & 1) + t)), kb = lds128(kbase + tile_at(krow + 8, j >> 1, 4 * (j & 1) + t));
        // [k step]: rows g, g+8 at k = t, then at k = t + 4
        const float kx[2][4] = { { ka.x, kb.x, ka.y, kb.y }, { ka.z, kb.z, ka.w, kb.w } };
        uint32_t hi[2][4], lo[2][4];
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[st][e] = __float_as_uint(kx[st][e]);
                lo[st][e] = tf32_lo(kx[st][e]);
            }
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const uint8_t *qp = qbase + (n * (DKP / 16) + j) * (C::SPLIT_Q ? 1024 : 512);
            const float4 q = lds128(qp);
            float4 r;
            if (C::SPLIT_Q) r = lds128(qp + 512);
            else r = make_float4(__uint_as_float(tf32_lo(q.x)), __uint_as_float(tf32_lo(q.y)), __uint_as_float(tf32_lo(q.z)), __uint_as_float(tf32_lo(q.w)));
            mma_tf32(x1[n], lo[0], __float_as_uint(q.x), __float_as_uint(q.y));
            mma_tf32(sc[n], hi[0], __float_as_uint(q.x), __float_as_uint(q.y));
            mma_tf32(NR == 1 ? x2[0] : x1[n], hi[0], __float_as_uint(r.x), __float_as_uint(r.y));
            mma_tf32(x1[n], lo[1], __float_as_uint(q.z), __float_as_uint(q.w));
            mma_tf32(CH == 2 ? sc1[CH == 2 ? n : 0] : sc[n], hi[1], __float_as_uint(q.z), __float_as_uint(q.w));
            mma_tf32(NR == 1 ? x2[0] : x1[n], hi[1], __float_as_uint(r.z), __float_as_uint(r.w));
        }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(k_empty);
    // Scores in the log2 domain.  The reference that is taken off in the exponent need not be the maximum: while no score
    // is more than 2^8 above it (one vote), it stays and nothing summed before needs a factor.
    bool above = false;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float top = CH == 2 ? sc[n][e] + sc1[CH == 2 ? n : 0][e] : sc[n][e];
            float x = (top + (NR == 1 ? x1[n][e] + x2[0][e] : x1[n][e])) * a.c_log2;
            if (TAIL) {
                const int j = key0 + krow + 8 * (e >> 1) - s.len;   // < 0: a cached row
                if (j >= 0 && (j >= s.n || !tree_sees(a, b, toks[8 * n + 2 * t + (e & 1)], j))) x = -INFINITY;
            }
            sc[n][e] = x;
            above = above || x > w.m[n][e & 1] + 8.f;
        }
    float corr[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) corr[n][0] = corr[n][1] = 1.f;
    if (__any_sync(0xffffffffu, above)) {
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float top = fmaxf(sc[n][r], sc[n][2 + r]);
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const float m_new = fmaxf(w.m[n][r], top);
                corr[n][r] = ex2_approx(w.m[n][r] - (m_new == -INFINITY ? 0.f : m_new));
                w.m[n][r] = m_new;
            }
    }
    // P^T as operand B (k = t, t+4: keys 2t, 2t+1 of each eight; column g: query row 8n + g)
    uint32_t phi[NR][4], plo[NR][4];
    const int from = 8 * t + (g >> 1);               // lane that holds key 2t (row 2t of S^T) and query row g; key 2t+1: row (2t+1)^4
    const int from1 = 4 * ((2 * t + 1) ^ 4) + (g >> 1);
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float base = w.m[n][r] == -INFINITY ? 0.f : w.m[n][r];   // nothing seen so far: p = 2^-inf = 0
            sc[n][r] = ex2_approx(sc[n][r] - base);
            sc[n][2 + r] = ex2_approx(sc[n][2 + r] - base);
            w.l[n][r] = fmaf(w.l[n][r], corr[n][r], sc[n][r] + sc[n][2 + r]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {   // key 2t, 2t+1 of the first eight, then of the second
            const int src = e & 1 ? from1 : from;
            const float even = __shfl_sync(0xffffffffu, sc[n][e & 2], src), oddv = __shfl_sync(0xffffffffu, sc[n][(e & 2) + 1], src);
            const float p = g & 1 ? oddv : even;
            phi[n][e] = __float_as_uint(p);
            plo[n][e] = tf32_lo(p);
        }
    }
    if (ok && !__all_sync(0xffffffffu, mbar_wait_bounded(v_full, v_parity))) ok = false;
    if (!ok) return;
    // O^T = O^T * corr + V^T.P^T
    bool odd = false;   // a value behind the cached rows that is not finite
#pragma unroll
    for (int sl = 0; sl < DKP / 32; ++sl) {
        float acc[2][NR][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NR; ++n) acc[h][n][0] = acc[h][n][1] = acc[h][n][2] = acc[h][n][3] = 0.f;
#pragma unroll
        for (int k8 = 0; k8 < 2; ++k8) {
            const int ra = row0 + 8 * k8 + 2 * t, rb = ra + 1;
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
            // rows g: columns 4g and 4g + 2; rows g+8: 4g + 1 and 4g + 3
            const float vx[2][4] = { { va.x, va.y, vb.x, vb.y }, { va.z, va.w, vb.z, vb.w } };
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    hi[e] = __float_as_uint(vx[h][e]);
                    lo[e] = tf32_lo(vx[h][e]);
                }
#pragma unroll
                for (int n = 0; n < NR; ++n) mma_tf32(acc[h][n], lo, phi[n][2 * k8], phi[n][2 * k8 + 1]);
#pragma unroll
                for (int n = 0; n < NR; ++n) mma_tf32(acc[h][n], hi, plo[n][2 * k8], plo[n][2 * k8 + 1]);
#pragma unroll
                for (int n = 0; n < NR; ++n) mma_tf32(acc[h][n], hi, phi[n][2 * k8], phi[n][2 * k8 + 1]);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) w.o[2 * sl + h][n][e] = fmaf(w.o[2 * sl + h][n][e], corr[n][e & 1], acc[h][n][e]);
    }
    if (TAIL && __any_sync(0xffffffffu, odd)) {
        // rare: an infinity or a NaN among the new rows' values goes to the rows that see it, and to no others
#pragma unroll 1
        for (int key = 0; key < 16; ++key) {
            const int j = key0 + row0 + key - s.len;
            if (j < 0 || j >= s.n) continue;
#pragma unroll
            for (int sl = 0; sl < DKP / 32; ++sl) {
                const float4 v4 = lds128(vbase + tile_at(row0 + key, sl, g));
                const float *x = &v4.x;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!finite_f(x[e]))
#pragma unroll
                        for (int n = 0; n < NR; ++n)
#pragma unroll
                            for (int r = 0; r < 2; ++r)
                                if (tree_sees(a, b, toks[8 * n + 2 * t + r], j)) w.o[2 * sl + (e >> 1)][n][2 * (e & 1) + r] += x[e];
            }
        }
    }
}

// (m, l, o) of a warp plus another part of the same rows
template <int DKP, int NR>
__device__ __forceinline__ void tree_add(TreeWarp<DKP, NR> &w, const float4 *frag, const float4 *ml, int stride)
{
    float f0[NR][2], f1[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const float4 v = ml[n * stride];   // maxima of the two rows, then sums
        const float m2[2] = { v.x, v.y }, l2[2] = { v.z, v.w };
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float m_new = fmaxf(w.m[n][r], m2[r]), base = m_new == -INFINITY ? 0.f : m_new;
            f0[n][r] = ex2_approx(w.m[n][r] - base);
            f1[n][r] = ex2_approx(m2[r] - base);
            w.m[n][r] = m_new;
            w.l[n][r] = w.l[n][r] * f0[n][r] + l2[r] * f1[n][r];
        }
    }
#pragma unroll
    for (int i = 0; i < DKP / 16; ++i)
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const float4 v = frag[(i * NR + n) * stride];
            const float *x = &v.x;
#pragma unroll
            for (int e = 0; e < 4; ++e) w.o[i][n][e] = w.o[i][n][e] * f0[n][e & 1] + x[e] * f1[n][e & 1];
        }
}

template <int DKP, int NR>
__device__ __forceinline__ void tree_put(const TreeWarp<DKP, NR> &w, float4 *frag, float4 *ml, int stride)
{
#pragma unroll
    for (int n = 0; n < NR; ++n) ml[n * stride] = make_float4(w.m[n][0], w.m[n][1], w.l[n][0], w.l[n][1]);
#pragma unroll
    for (int i = 0; i < DKP / 16; ++i)
#pragma unroll
        for (int n = 0; n < NR; ++n) frag[(i * NR + n) * stride] = make_float4(w.o[i][n][0], w.o[i][n][1], w.o[i][n][2], w.o[i][n][3]);
}

// all warps' parts into warp 0's: halves, quarters, ...; every consumer warp takes part
template <int DKP, int NR>
__device__ __forceinline__ void tree_merge(TreeWarp<DKP, NR> &w, float4 *area, int part)
{
    using C = TreeCfg<DKP, NR>;
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int half = KT_CONSUMERS / 2; half >= 1; half >>= 1) {
        float4 *frag = area + (size_t)(part >= half ? part - half : part) * 32 * (C::FRAGS + NR) + lane;
        if (part >= half && part < 2 * half) tree_put<DKP, NR>(w, frag, frag + C::FRAGS * 32, 32);
        consumers_sync();
        if (part < half) tree_add<DKP, NR>(w, frag, frag + C::FRAGS * 32, 32);
        consumers_sync();
    }
}

template <int DKP, int NR>
__global__ void __launch_bounds__(TreeCfg<DKP, NR>::THREADS, 1)
kv_tree_kernel(const __grid_constant__ KvTreeArgs a, const __grid_constant__ TreeMaps tm, int tma)
{
    using C = TreeCfg<DKP, NR>;
    constexpr int ROWS = C::ROWS;
    extern __shared__ uint8_t smem_raw[];
    __shared__ alignas(8) uint64_t bars[4 * C::STAGES + 6];
    __shared__ TreePiece s_piece[2];
    __shared__ int s_line[3], s_last, s_toks[2][ROWS];
    __shared__ volatile int s_gave_up;   // a consumer's wait ran out: its arrivals no longer mean free stages
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t *const tiles = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);   // the swizzle is a function of the address
    float4 *const area = reinterpret_cast<float4 *>(tiles + C::STAGES * 2 * C::TILE);
    const uint32_t bar0 = smem_u32(bars);
    auto empty_bar = [&](int v, int stage) { return bar0 + 8u * (v * C::STAGES + stage); };
    auto full_bar = [&](int v, int stage) { return bar0 + 8u * ((2 + v) * C::STAGES + stage); };
    // pieces (ASYNC): prepared, done with; partial results: all there, taken
    const uint32_t piece_full = bar0 + 8u * (4 * C::STAGES), piece_empty = piece_full + 16, merge_full = piece_full + 32, merge_empty = piece_full + 40;
    auto ktile = [&](int stage) { return tiles + stage * 2 * C::TILE; };
    // a call of a few microseconds: a thread a barrier, the descriptors on their way
    static_assert(4 * C::STAGES + 6 <= KT_CONSUMERS * 32, "barriers");
    if (tid < 4 * C::STAGES + 6) {
        const int k = tid - 4 * C::STAGES;
        mbar_init(bar0 + 8u * tid, k < -2 * C::STAGES ? C::SLICES : k < 0 ? (tma ? 1 : 32) : k == 2 || k == 3 ? KT_CONSUMERS + 1 : k == 4 ? KT_CONSUMERS : 1);
        mbar_fence_init();
    }
    if (tid == 0) s_gave_up = 0;
    if (tma && lane == 0 && (warp == KT_CONSUMERS || warp == KT_CONSUMERS + 1)) tma_prefetch_desc(warp == KT_CONSUMERS ? &tm.k : &tm.v);
    constexpr TreeLine line = { ROWS, KT_KEYS, C::GROUPS, C::GAP };
    TreeCursor cur;
    if (!tree_start(a, line, s_line, cur)) return;   // (its barriers make the initialised ones above visible)
    TreePiece p;
    bool ok = true;
    uint32_t it = 0;   // tiles since the start: ring stage it % STAGES, its use number it / STAGES

    const int heads_per = a.H / a.Hkv;
    // Query row r of a key head: head r / n, token r % n.  A piece's Q as the lanes will read it, [eight rows][16-column group]
    // [(hi, lo)][lane], and the rows' tokens, by `threads` threads.
    auto stage_q = [&](const TreePiece &pc, float4 *to, int *toks, int thread, int threads) {
#pragma unroll 4
        for (int i = thread; i < ROWS * (DKP / 4); i += threads) {
            const int r = i / (DKP / 4), c = i - r * (DKP / 4), row = pc.block * ROWS + r;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            int tok = 0;
            if (row < pc.s.rows) {
                const int gh = row / pc.s.n;
                tok = row - gh * pc.s.n;
                const float *src = a.Q + (((int64_t)pc.b * a.H + pc.hk * heads_per + gh) * a.T + tok) * a.dk + 4 * c;
                if (tma) {   // rows are whole 16-byte pieces
                    if (4 * c < a.dk) x = __ldg(reinterpret_cast<const float4 *>(src));
                } else {
                    if (4 * c < a.dk) x.x = __ldg(src);
                    if (4 * c + 1 < a.dk) x.y = __ldg(src + 1);
                    if (4 * c + 2 < a.dk) x.z = __ldg(src + 2);
                    if (4 * c + 3 < a.dk) x.w = __ldg(src + 3);
                }
            }
            if (c == 0) toks[r] = tok;
            const int at = ((r >> 3) * (DKP / 16) + (c >> 2)) * (C::SPLIT_Q ? 64 : 32) + (r & 7) * 4 + (c & 3);
            to[at] = x;
            if (C::SPLIT_Q)
                to[at + 32] = make_float4(__uint_as_float(tf32_lo(x.x)), __uint_as_float(tf32_lo(x.y)), __uint_as_float(tf32_lo(x.z)), __uint_as_float(tf32_lo(x.w)));
        }
    };
    TreeWarp<DKP, NR> w;
    auto clear = [&] {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            w.m[n][0] = w.m[n][1] = -INFINITY;
            w.l[n][0] = w.l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < DKP / 16; ++i) w.o[i][n][0] = w.o[i][n][1] = w.o[i][n][2] = w.o[i][n][3] = 0.f;
        }
    };
    // the workspace slots of an item's pieces, in lane order
    auto slot = [&](int k) { return reinterpret_cast<float4 *>(a.slots) + (size_t)k * (C::PART_BYTES / 16) + lane; };
    // a piece's tiles, by one consumer warp
    auto consume = [&](const TreePiece &pc, const float4 *q, const int *toks) {
        const uint8_t *qbase = reinterpret_cast<const uint8_t *>(q) + lane * 16;
        const int grp = warp / C::SLICES, row0 = warp % C::SLICES * 16;
        for (int i = 0; i < pc.count; ++i, ++it) {
            if (C::GROUPS > 1 && (int)(it % C::GROUPS) != grp) continue;
            const int s = it % C::STAGES;
            const uint32_t ph = (it / C::STAGES) & 1;
            const int key0 = (pc.t0 + i) * KT_KEYS;
            if (ok && !__all_sync(0xffffffffu, mbar_wait_bounded(full_bar(0, s), ph))) ok = false;
            const bool work = ok;
            if (work) {
                const uint8_t *kt = ktile(s);
                if (key0 + row0 + 16 > pc.s.len)
                    tree_tile<DKP, NR, true>(a, w, qbase, kt, kt + C::TILE, key0, row0, pc.s, pc.b, toks, empty_bar(0, s), full_bar(1, s), ph, ok);
                else
                    tree_tile<DKP, NR, false>(a, w, qbase, kt, kt + C::TILE, key0, row0, pc.s, pc.b, toks, empty_bar(0, s), full_bar(1, s), ph, ok);
            }
            if (!ok) {
                s_gave_up = 1;
                __threadfence_block();
            }
            __syncwarp();
            if (lane == 0) {
                if (!work) mbar_arrive(empty_bar(0, s));
                mbar_arrive(empty_bar(1, s));
            }
        }
        // the lanes' sums become the rows'
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) w.l[n][r] += __shfl_xor_sync(0xffffffffu, w.l[n][r], o);
    };
    // an item's result, by the warp that holds it
    auto write_out = [&](const TreePiece &pc) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = pc.block * ROWS + n * 8 + 2 * t + r;
                if (row >= pc.s.rows) continue;
                const int gh = row / pc.s.n, tok = row - gh * pc.s.n;
                float *dst = a.out + (((int64_t)pc.b * a.H + pc.hk * heads_per + gh) * a.T + tok) * a.dk;
                const float inv = w.l[n][r] == 0.f ? 0.f : 1.0f / w.l[n][r];   // nothing seen: 0
#pragma unroll
                for (int sl = 0; sl < DKP / 32; ++sl) {
                    const int c = 32 * sl + 4 * g;
                    const float4 y = make_float4(w.o[2 * sl][n][r] * inv, w.o[2 * sl][n][2 + r] * inv, w.o[2 * sl + 1][n][r] * inv,
                                                 w.o[2 * sl + 1][n][2 + r] * inv);
                    if (tma) {
                        if (c < a.dk) *reinterpret_cast<float4 *>(dst + c) = y;
                    } else {
                        const float *v = &y.x;
                        for (int e = 0; e < 4; ++e)
                            if (c + e < a.dk) dst[c + e] = v[e];
                    }
                }
            }
    };

    if (warp >= KT_CONSUMERS) {
        // ---- producers: warp 8 the K tiles, warp 9 the V tiles (one issuing thread turns a 16 KB tile around in some 700
        // cycles, which HBM's share of an SM would just about saturate)
        if (C::SHIFT_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (!C::ASYNC && warp > KT_CONSUMERS + 1) return;
        if (C::ASYNC && warp == KT_CONSUMERS + 2) {
            // ---- scout
            for (uint32_t k = 0;; ++k) {
                const bool more = next_piece(a, line, cur, p);
                if (k >= 2 && !__all_sync(0xffffffffu, mbar_wait_bounded(piece_empty + 8 * (k & 1), (k / 2 - 1) & 1))) return;
                if (!more) p.count = 0;
                if (lane == 0) s_piece[k & 1] = p;
                if (more) stage_q(p, area + (k & 1) * (C::Q_BYTES / 16), s_toks[k & 1], lane, 32);
                __syncwarp();
                if (lane == 0) mbar_arrive(piece_full + 8 * (k & 1));
                if (!more) return;
            }
        }
        if (C::ASYNC && warp == KT_CONSUMERS + 3) {
            // ---- merger
            float4 *const parts = area + 2 * (C::Q_BYTES / 16) + lane;
            uint32_t k = 0;
            for (;; ++k) {
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(piece_full + 8 * (k & 1), (k / 2) & 1))) break;
                p = s_piece[k & 1];
                if (p.count == 0) return;
                if (!__all_sync(0xffffffffu, mbar_wait_bounded(merge_full, k & 1))) break;
                clear();
#pragma unroll 1
                for (int i = 0; i < KT_CONSUMERS; ++i) tree_add<DKP, NR>(w, parts + i * (C::PART_BYTES / 16), parts + i * (C::PART_BYTES / 16) + C::FRAGS * 32, 32);
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(merge_empty);
                    mbar_arrive(piece_empty + 8 * (k & 1));
                }
                bool write = p.pieces == 1;
                if (!write) {
                    float4 *f = slot(tree_slot(blockIdx.x, p.t0 == 0));
                    tree_put<DKP, NR>(w, f, f + C::FRAGS * 32, 32);
                    __threadfence();
                    __syncwarp();
                    int last = 0;
                    if (lane == 0) last = tree_arrive(a, p);
                    write = __shfl_sync(0xffffffffu, last, 0) != 0;
                    if (write) {
                        __threadfence();
                        clear();
#pragma unroll 3
                        for (int i = 0; i < p.pieces; ++i) {   // (several pieces' loads in flight: a lone warp's time is their latency)
                            const float4 *s = slot(tree_slot(p.first + i, i == 0));
                            tree_add<DKP, NR>(w, s, s + C::FRAGS * 32, 32);
                        }
                        if (lane == 0) tree_clear(a, p);
                    }
                }
                if (write) write_out(p);
            }
            if (lane == 0) tree_leave(a, line, cur, k);
            return;
        }
        const int v = warp - KT_CONSUMERS;
        const float *const cache = v ? a.V : a.K;
        while (ok && next_piece(a, line, cur, p)) {
            const int head = p.b * a.Hkv + p.hk;
            for (int i = 0; ok && i < p.count; ++i, ++it) {
                const int s = it % C::STAGES, row = (p.t0 + i) * KT_KEYS;
                const uint32_t use = it / C::STAGES;
                if (use && !__all_sync(0xffffffffu, mbar_wait_bounded(empty_bar(v, s), (use - 1) & 1))) { ok = false; break; }
                if (s_gave_up) { ok = false; break; }
                const uint32_t full = full_bar(v, s), dst = smem_u32(ktile(s)) + v * C::TILE;
                if (tma) {
                    if (lane == 0) {
                        mbar_arrive_expect_tx(full, C::TILE);
#pragma unroll
                        for (int sl = 0; sl < DKP / 32; ++sl) tma_load_3d(dst + sl * (KT_KEYS * 128), v ? &tm.v : &tm.k, full, 32 * sl, row, head);
                    }
                } else {
                    // tensors that a tensor map cannot describe: the same layout, four bytes at a time
                    const float *src = cache + (int64_t)head * a.max_seq * a.dk;
#pragma unroll 1
                    for (int r = 0; r < KT_KEYS; ++r) {
                        const bool in = (int64_t)row + r < a.max_seq;
#pragma unroll 1
                        for (int sl = 0; sl < DKP / 32; ++sl) {
                            const int c = 32 * sl + lane;
                            const bool get = in && c < a.dk;
                            const float *get_from = get ? src + ((int64_t)row + r) * a.dk + c : src;
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + tile_at(r, sl, lane >> 2) + 4 * (lane & 3)),
                                         "l"(get_from), "r"(get ? 4 : 0)
                                         : "memory");
                        }
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full) : "memory");
                }
            }
        }
        if (!ok) {
            if (lane == 0 && a.err) atomicCAS(a.err + ERR_GAVE_UP, 0, (int)TERR_PRODUCER);
            // copies in flight land before the CTA's memory goes away
            for (uint32_t i = it > C::STAGES ? it - C::STAGES : 0; i < it; ++i) mbar_wait_bounded(full_bar(v, i % C::STAGES), (i / C::STAGES) & 1);
        }
        return;
    }

    // ---- consumers
    if (C::SHIFT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    if (C::ASYNC) {
        float4 *const mine = area + 2 * (C::Q_BYTES / 16) + warp * (C::PART_BYTES / 16) + lane;
        for (uint32_t k = 0;; ++k) {
            if (!ok || !__all_sync(0xffffffffu, mbar_wait_bounded(piece_full + 8 * (k & 1), (k / 2) & 1))) { ok = false; break; }
            p = s_piece[k & 1];
            if (p.count == 0) break;
            clear();
            consume(p, area + (k & 1) * (C::Q_BYTES / 16), s_toks[k & 1]);
            if (!ok || (k && !__all_sync(0xffffffffu, mbar_wait_bounded(merge_empty, (k - 1) & 1)))) { ok = false; break; }
            tree_put<DKP, NR>(w, mine, mine + C::FRAGS * 32, 32);
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(merge_full);
                mbar_arrive(piece_empty + 8 * (k & 1));
            }
        }
    } else {
        while (next_piece(a, line, cur, p)) {   // (to the end also after a wait that ran out: the items' counters need every arrival)
            stage_q(p, area, s_toks[0], tid, KT_CONSUMERS * 32);
            clear();
            consumers_sync();
            consume(p, area, s_toks[0]);
            consumers_sync();   // Q has been read
            tree_merge<DKP, NR>(w, area, warp);
            bool write = p.pieces == 1;
            if (!write) {
                if (warp == 0) {
                    float4 *f = slot(tree_slot(blockIdx.x, p.t0 == 0));
                    tree_put<DKP, NR>(w, f, f + C::FRAGS * 32, 32);
                    __threadfence();
                }
                consumers_sync();
                if (tid == 0) s_last = tree_arrive(a, p);
                consumers_sync();
                write = s_last != 0;
                if (write) {
                    __threadfence();
                    clear();
#pragma unroll 1
                    for (int k = warp; k < p.pieces; k += KT_CONSUMERS) {
                        const float4 *f = slot(tree_slot(p.first + k, k == 0));
                        tree_add<DKP, NR>(w, f, f + C::FRAGS * 32, 32);
                    }
                    tree_merge<DKP, NR>(w, area, warp);
                    if (tid == 0) tree_clear(a, p);
                }
            }
            if (write && warp == 0) write_out(p);
            consumers_sync();   // the merge area and the tokens are free again
        }
    }
    if (!ok && lane == 0 && a.err) atomicCAS(a.err + ERR_GAVE_UP, 0, (int)TERR_CONSUMER);
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
        if (bad && err) atomicCAS(err + ERR_KEEP, 0, (int)AXB_DEVERR_KEEP);
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
    return KT_SHARED_BYTES + (size_t)sm_count * 2 * KT_SLOT_BYTES;
}

template <int DKP, int NR>
static int launch_tree(const KvTreeArgs &a, const TreeMaps &tm, int tma, int sm_count, cudaStream_t st)
{
    using C = TreeCfg<DKP, NR>;
    static_assert(C::SMEM <= 227 * 1024 - 2048, "shared memory");
    static_assert((size_t)C::PART_BYTES <= KT_SLOT_BYTES, "workspace slots");
    static PerDeviceOnce once;
    if (once.first()) {
        cudaError_t e = cudaFuncSetAttribute(kv_tree_kernel<DKP, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
    }
    kv_tree_kernel<DKP, NR><<<sm_count, C::THREADS, C::SMEM, st>>>(a, tm, tma);
    return (int)cudaGetLastError();
}

template <int NR>
static int launch_tree_rows(const KvTreeArgs &a, const TreeMaps &tm, int tma, int sm_count, cudaStream_t st)
{
    if (a.dk <= 32) return launch_tree<32, NR>(a, tm, tma, sm_count, st);
    if (a.dk <= 64) return launch_tree<64, NR>(a, tm, tma, sm_count, st);
    if (a.dk <= 96) return launch_tree<96, NR>(a, tm, tma, sm_count, st);
    return launch_tree<128, NR>(a, tm, tma, sm_count, st);
}

int launch_kv_cache_attend_tree(const KvTreeArgs &a, int sm_count, cudaStream_t st, int *launches)
{
    *launches = 1;
    const int tma = a.dk % 4 == 0 && kt_aligned16(a.K) && kt_aligned16(a.V) && kt_aligned16(a.Q) && kt_aligned16(a.out);
    const int64_t rows = (int64_t)(a.H / a.Hkv) * a.T;   // of a key head, if every token is there
    if (tma && rows > kt_warp_rows(a.dk)) return launch_kv_tree_tc(a, sm_count, st, launches);
    TreeMaps tm = {};
    if (tma) {
        int e = encode_f32_batched_tmap(&tm.k, a.K, (int64_t)a.B * a.Hkv, a.max_seq, a.dk, a.dk, KT_KEYS, false);
        if (!e) e = encode_f32_batched_tmap(&tm.v, a.V, (int64_t)a.B * a.Hkv, a.max_seq, a.dk, a.dk, KT_KEYS, false);
        if (e) return e;
    }
    if (rows <= 8) return launch_tree_rows<1>(a, tm, tma, sm_count, st);
    if (rows <= 16) return launch_tree_rows<2>(a, tm, tma, sm_count, st);
    return launch_tree_rows<4>(a, tm, tma, sm_count, st);
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
