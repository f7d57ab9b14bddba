// kv_tree_tc.cu — kv_cache_attend_tree when many query rows share a key head (wide trees, grouped heads, chunks of a
// prompt): the same result as kv_tree.cu on tcgen05, 64 or 128 query rows of a key head at a time, head dim <= 128.
//     S = Q.K^T, O = P.V as three tf32 products each over hi/lo parts; the value as it lies is the hi operand (the tensor
//     core reads its tf32 part), the remainder rounded to tf32 the lo operand.
// The work line of kv_tree_line.cuh, cut into one stretch per CTA, replaces the grid over query tiles; key blocks of 128
// (head dim <= 64) or 64 keys.  Twenty warps:
//   0-7   softmax: two threads per query row, half the block's columns each (they swap maxima through shared memory).  Scores
//         leave tensor memory once and stay in registers; P hi and lo go to columns of their own, the A operands of P.V as
//         they lie, when the block before has read its own.  The exponent's reference stays until a score passes it by
//         2^8; every block's P.V starts from zero and is folded into fp32 registers, so the tensor core's truncating
//         accumulation never spans more than a block.
//   8-15  Q of a piece (gathered rows -> swizzled shared memory, lo part there or, for head dims above 64, in tensor
//         memory), the lo parts of the K and V blocks, and what must not reach the V product: rows behind the last token,
//         and infinities or NaN in new rows (those are added row by row);
//   16, 17  TMA of K and V (with 128 rows one operand has two raw buffers, the one whose chain is the longer: V for head dims up
//         to 64, K above; with 64 both do);
//   18, 19  one thread each issues the score and the P.V products.
// Shared memory is full either way (224 KB): Q, K and V and their lo parts, seven tiles of 32 KB.
//
// What bounds it: 128 rows a product whatever the query rows, so a block of 64 keys of head dim 128 costs the pipe 3,840 cycles
// (48 products of 48 cycles, 24 of 64) and its operands 4,100 cycles of shared memory, against 2,800 in which HBM brings its
// keys; 4,500 to 5,900 were measured, the softmax threads' 3,500 to 4,500 among them, at a clock that the power limit holds at
// 1.77 GHz.  8 sequences, 8 key heads of 128 with 64 rows, 41000 cached rows (338 MB): 120 us; with P over the scores, where
// a block's scores had to wait for the products of the last but one, 162.  6 key heads of 64 with 256 rows: 72 us, 112 TFLOP/s
// of the three products' 273.
#include "errors.cuh"
#include "gemm_tc.cuh"
#include "kv_tree_line.cuh"
#include "ptx.cuh"

#include <cuda.h>
#include <math.h>

namespace axb {

static constexpr int TT_THREADS = 640;
enum { CERR_LOAD = 94, CERR_CONVERT = 95, CERR_MMA = 96, CERR_SOFTMAX = 97 };

template <int NSLAB, bool FEW>
struct TreeTc {
    static constexpr bool WIDE = NSLAB > 2;
    static constexpr int ROWS = FEW ? 64 : 128;                // query rows (a product has 128 either way)
    static constexpr int SOFTMAX = 2 * ROWS;                   // threads at work on them
    static constexpr int DKP = 32 * NSLAB;
    static constexpr int KB = WIDE ? 64 : 128;                 // keys of a block
    static constexpr int QSLAB = ROWS * 128, SLAB = KB * 128;   // bytes of 32 columns
    static constexpr int QPLANE = NSLAB * QSLAB, PLANE = NSLAB * SLAB;
    static constexpr int KS = WIDE || FEW ? 2 : 1, VS = WIDE && !FEW ? 1 : 2; // raw buffers
    static constexpr int OB = WIDE ? 1 : 2;                    // accumulators of P.V
    static constexpr int SB = WIDE ? 2 : 1;                    // score buffers
    // tensor memory columns
    static constexpr int T_S = 0, T_P = SB * KB, T_PLO = T_P + KB, T_O = T_PLO + KB, T_QLO = T_O + OB * DKP;
    static constexpr int COLS = 512;
    static_assert(T_QLO + (WIDE ? DKP : 0) <= COLS, "tensor memory");
    static constexpr int HEADER = 3 * 1024;   // barriers, words, then the softmax threads' maxima
    static constexpr int Q_AT = HEADER, K_AT = Q_AT + QPLANE * (WIDE ? 1 : 2), KLO_AT = K_AT + KS * PLANE, V_AT = KLO_AT + PLANE,
                         VLO_AT = V_AT + VS * PLANE, SMEM = VLO_AT + PLANE;
    static_assert(SMEM <= 227 * 1024, "shared memory");   // all of it: the kernel has no static shared memory
};

enum {
    TB_Q_FULL, TB_Q_EMPTY, TB_K_RAW, TB_K_FULL = TB_K_RAW + 2, TB_K_EMPTY, TB_V_RAW = TB_K_EMPTY + 2, TB_V_FULL = TB_V_RAW + 2, TB_V_EMPTY,
    TB_S_FULL = TB_V_EMPTY + 2, TB_S_EMPTY = TB_S_FULL + 2, TB_P_FULL = TB_S_EMPTY + 2, TB_PLO_FULL, TB_KLO_EMPTY, TB_VLO_EMPTY, TB_O_FULL,
    TB_O_EMPTY, TB_DRAIN = TB_O_EMPTY + 2,
    TB_COUNT = TB_DRAIN + 2
};

struct TreeTcMaps {
    CUtensorMap k, v;   // [B*Hkv][max_seq][dk], boxes of 32 columns x KB rows (v: 32-byte swizzle atoms)
};

__device__ __forceinline__ uint32_t lo_bits(uint32_t x) { return tf32_lo(__uint_as_float(x)); }

// The three products of a block's scores / outputs, issued by one thread: four steps of eight at a time, in loops.  Unrolled whole
// the thread takes 55 cycles a product instead of 70 to 100, but the kernel's roles share the SM's instruction cache, and the call
// took 129 us instead of 120 (64 rows of 128), 73 instead of 72 (256 rows of 64); with a copy for each of six buffer turns 177.
template <int NSLAB, bool FEW>
__device__ __forceinline__ void issue_scores(uint32_t base, uint32_t tmem, uint32_t it, uint32_t idesc, uint32_t klo_empty)
{
    using C = TreeTc<NSLAB, FEW>;
    const uint64_t dk = smem_desc_kmajor(base, 128);   // (every offset below stays inside the CTA's 256 KB window)
    const uint32_t d = tmem + C::T_S + it % C::SB * C::KB, khi = C::K_AT + it % C::KS * C::PLANE;
#pragma unroll
    for (int pr = 0; pr < 3; ++pr) {   // hi.lo, whose lo tile the next block waits for, lo.hi, hi.hi
        uint64_t kd = dk + ((pr == 0 ? C::KLO_AT : khi) >> 4), qd = dk + ((C::Q_AT + (pr == 1 && !C::WIDE ? C::QPLANE : 0)) >> 4);
        uint32_t qt = tmem + C::T_QLO;
#pragma unroll 1
        for (int sl = 0; sl < NSLAB; ++sl, kd += C::SLAB >> 4, qd += C::QSLAB >> 4, qt += 32) {   // (columns from dk on are zero)
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                if (C::WIDE && pr == 1) tc_mma_ts_tf32(d, qt + ks * 8, kd + ks * 2, idesc, 1);
                else tc_mma<KIND_TF32>(d, qd + ks * 2, kd + ks * 2, idesc, pr | sl | ks);
            }
        }
        if (pr == 0) tc_commit(klo_empty);
    }
}

// Part 0: P hi . V lo, whose tile the next block waits for; part 1: P lo . V hi, whose operand comes last, and P hi . V hi: an
// accumulation cuts its sum off, so the small products go first (with P lo . V hi last the error was 1.2e-6, so 0.65e-6).
template <int NSLAB, bool FEW, int PART>
__device__ __forceinline__ void issue_outputs(uint32_t base, uint32_t tmem, uint32_t it, uint32_t idesc, uint32_t vlo_empty)
{
    using C = TreeTc<NSLAB, FEW>;
    const uint64_t dm = smem_desc_mnmajor_sw128_32b(base, C::SLAB, 512);
    const uint32_t d = tmem + C::T_O + it % C::OB * C::DKP, vhi = C::V_AT + it % C::VS * C::PLANE;
#pragma unroll
    for (int pr = PART ? 1 : 0; pr < (PART ? 3 : 1); ++pr) {
        uint64_t vd = dm + ((pr == 0 ? C::VLO_AT : vhi) >> 4);
        uint32_t pt = tmem + (pr == 1 ? C::T_PLO : C::T_P);
#pragma unroll 1
        for (int k0 = 0; k0 < C::KB / 32; ++k0, vd += 4 * 64, pt += 32) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) tc_mma_ts_tf32(d, pt + ks * 8, vd + ks * 64, idesc, pr | k0 | ks);
        }
        if (pr == 0) tc_commit(vlo_empty);
    }
}

// which of the 32 keys from new-token index `base` (negative: cached rows) token t sees
__device__ __forceinline__ uint32_t seen_bits(const KvTreeArgs &a, int b, int t, int n, int base)
{
    if (base <= -32) return 0xFFFFFFFFu;
    const int j0 = base > 0 ? base : 0, skip = j0 - base;   // skip cached rows come first
    uint32_t bits = 0;
    if (j0 < n) {
        if (!a.mask) {
            const int last = t < n - 1 ? t : n - 1;
            bits = last - j0 >= 31 ? 0xFFFFFFFFu : last < j0 ? 0u : (2u << (last - j0)) - 1u;
        } else {
            const uint64_t *m = a.mask + b * a.mask_stride + (int64_t)t * a.words + (j0 >> 6);
            const int sh = j0 & 63;
            uint64_t w = __ldg(m) >> sh;
            if (sh && (j0 >> 6) + 1 < a.words) w |= __ldg(m + 1) << (64 - sh);
            bits = (uint32_t)w;
            if (n - j0 < 32) bits &= (1u << (n - j0)) - 1u;
        }
    }
    return skip ? (bits << skip) | ((1u << skip) - 1u) : bits;
}

template <int NSLAB, bool FEW>
__global__ void __launch_bounds__(TT_THREADS, 1) kv_tree_tc_kernel(const __grid_constant__ KvTreeArgs a, const __grid_constant__ TreeTcMaps tm)
{
    using C = TreeTc<NSLAB, FEW>;
    // (GAP, blocks of room for the way to the next item: none 123 and 78 us for the two batches above, 2 120 and 72, 4 122 and 76)
    constexpr int GAP = 2, ROWS = C::ROWS, KB = C::KB, OH = C::DKP / 2, FOLD = OH % 32 || C::WIDE ? 16 : 32;   // OH: output columns of a softmax thread
    extern __shared__ __align__(1024) uint8_t sm[];
    const uint32_t base = smem_u32(sm);
    auto bar = [&](int i) -> uint32_t { return base + 8u * (uint32_t)i; };
    int *s_line = reinterpret_cast<int *>(sm + 256);
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(sm + 288);
    volatile int *words = reinterpret_cast<volatile int *>(sm + 304);
    volatile int &s_gave_up = words[0], *s_odd = words + 2;   // s_odd: block it + 1 holds non-finite new values
    int *s_row = reinterpret_cast<int *>(sm + 512);   // [ROWS]
    float (*s_max)[2][ROWS] = reinterpret_cast<float (*)[2][ROWS]>(sm + 1024);   // [block parity][half][row]
    if (threadIdx.x == 0) a.shared[blockIdx.x] = KvTreeShared{ 0, 0, 0, 0, 0, 0 };   // (this thread replaces it where the CTA begins a shared item)
    if (base & 1023) {   // the swizzles are functions of the address (it starts at a multiple of 1 KB; refused, should it ever not)
        if (threadIdx.x == 0 && a.err) atomicCAS(a.err + ERR_GAVE_UP, 0, (int)CERR_LOAD);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    static_assert(8 * TB_COUNT <= 256, "barriers");

    if (threadIdx.x < TB_COUNT) {   // a thread a barrier
        const int i = threadIdx.x;
        const bool conv = i == TB_Q_FULL || i == TB_K_FULL || i == TB_V_FULL;
        const bool soft = i == TB_P_FULL || i == TB_PLO_FULL || (i >= TB_S_EMPTY && i < TB_S_EMPTY + 2) || (i >= TB_O_EMPTY && i < TB_O_EMPTY + 2);
        mbar_init(bar(i), conv ? 256 : soft ? C::SOFTMAX : 1);
        mbar_fence_init();
    }
    if (lane == 0 && (warp == 16 || warp == 17)) tma_prefetch_desc(warp == 17 ? &tm.v : &tm.k);
    if (threadIdx.x == 0) {
        s_gave_up = 0;
        for (int i = 0; i < 4; ++i) s_odd[i] = 0;
    }
    constexpr TreeLine line = { ROWS, KB, 1, GAP };
    TreeCursor cur;
    if (!tree_start(a, line, s_line, cur)) return;
    if (warp == 19) {
        tmem_alloc(base + 288, C::COLS);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;

    // a wait that ran out anywhere stops every role: nobody loads or multiplies on arrivals that no longer mean anything
    auto wait = [&](int i, uint32_t parity) -> bool { return mbar_wait_bounded(bar(i), parity) && !s_gave_up; };
    auto wait_all = [&](int i, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait(i, parity) ? 1 : 0) != 0;
    };
    auto give_up = [&](int code) {
        s_gave_up = 1;
        if (a.err) atomicCAS(a.err + ERR_GAVE_UP, 0, code);
    };
    TreePiece p;
    uint32_t it = 0;      // key blocks since the start
    uint32_t np = 0;      // pieces since the start
    const int heads_per = a.H / a.Hkv;
    bool ok = true;

    // registers: 640 threads x 96 at launch = 256 x 144 (softmax) + 384 x 64
    if (warp >= 16) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp < 18 && lane == 0) {
            // -------------------------------------------------------- loads
            const bool v = warp == 17;
            const int stages = v ? C::VS : C::KS, b_raw = v ? TB_V_RAW : TB_K_RAW, b_empty = v ? TB_V_EMPTY : TB_K_EMPTY;
            const void *map = v ? &tm.v : &tm.k;
            while (ok && next_piece(a, line, cur, p)) {
                const int head = p.b * a.Hkv + p.hk;
                for (int i = 0; i < p.count; ++i, ++it) {
                    const uint32_t s = it % stages, use = it / stages;
                    if (use && !wait(b_empty + s, (use - 1) & 1)) { ok = false; break; }
                    if (s_gave_up) { ok = false; break; }
                    const int row = (p.t0 + i) * KB;
                    const uint32_t dst = base + (v ? C::V_AT : C::K_AT) + s * C::PLANE;
                    mbar_arrive_expect_tx(bar(b_raw + s), C::PLANE);
#pragma unroll
                    for (int sl = 0; sl < NSLAB; ++sl) tma_load_3d(dst + sl * C::SLAB, map, bar(b_raw + s), 32 * sl, row, head);
                    if (i + stages < p.count) {   // the block that waits for a buffer: into L2 meanwhile
#pragma unroll
                        for (int sl = 0; sl < NSLAB; ++sl) tma_prefetch_3d(map, 32 * sl, row + stages * KB, head);
                    }
                }
            }
            if (!ok) {
                give_up(CERR_LOAD);
                for (uint32_t i = it > (uint32_t)stages ? it - stages : 0; i < it; ++i) mbar_wait_bounded(bar(b_raw + i % stages), (i / stages) & 1);
            }
        } else if (warp == 18 && lane == 0) {
            // ----------------------------------------------------- scores
            const uint32_t idesc = make_idesc<KIND_TF32>(128, KB);
            while (ok && next_piece(a, line, cur, p)) {
                if (!wait(TB_Q_FULL, np & 1)) { ok = false; break; }
                ++np;
                for (int i = 0; i < p.count; ++i, ++it) {
                    // the softmax threads have the scores of block it - SB in registers
                    if (it >= C::SB && !wait(TB_S_EMPTY + it % C::SB, (it / C::SB - 1) & 1)) { ok = false; break; }
                    if (!wait(TB_K_FULL, it & 1)) { ok = false; break; }
                    tc_fence_after_sync();
                    issue_scores<NSLAB, FEW>(base, tmem, it, idesc, bar(TB_KLO_EMPTY));
                    tc_commit(bar(TB_S_FULL + it % C::SB));
                    tc_commit(bar(TB_K_EMPTY + it % C::KS));
                    if (i == p.count - 1) tc_commit(bar(TB_Q_EMPTY));
                }
            }
        } else if (warp == 19 && lane == 0) {
            // ----------------------------------------------------- outputs
            const uint32_t idesc = make_idesc<KIND_TF32>(128, (a.dk + 15) / 16 * 16) | (1u << 16);   // B is MN-major
            while (ok && next_piece(a, line, cur, p)) {
                for (int i = 0; i < p.count; ++i, ++it) {
                    if (!wait(TB_P_FULL, it & 1)) { ok = false; break; }
                    if (!wait(TB_V_FULL, it & 1)) { ok = false; break; }
                    if (it >= C::OB && !wait(TB_O_EMPTY + it % C::OB, (it / C::OB - 1) & 1)) { ok = false; break; }
                    tc_fence_after_sync();
                    issue_outputs<NSLAB, FEW, 0>(base, tmem, it, idesc, bar(TB_VLO_EMPTY));
                    if (!wait(TB_PLO_FULL, it & 1)) { ok = false; break; }
                    tc_fence_after_sync();
                    issue_outputs<NSLAB, FEW, 1>(base, tmem, it, idesc, 0);
                    tc_commit(bar(TB_O_FULL));
                    tc_commit(bar(TB_V_EMPTY + it % C::VS));
                }
            }
        }
        if (!ok && warp >= 18) {
            give_up(CERR_MMA);
            tc_commit(bar(TB_DRAIN + warp - 18));   // products in flight end before the tensor memory goes
            mbar_wait_bounded(bar(TB_DRAIN + warp - 18), 0);
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // ------------------------------------------------- Q, and the lo parts of K and V
        const int ct = threadIdx.x - 256;   // 0..255
        auto conv_sync = [] { asm volatile("bar.sync 6, 256;" ::: "memory"); };
        auto split = [&](const uint4 *src, uint4 *lo) {
            constexpr int PART = C::PLANE / 16 % (4 * 256) ? 2 : 4;
            static_assert(C::PLANE / 16 % (PART * 256) == 0, "whole batches");
#pragma unroll 1
            for (int c = ct; c < C::PLANE / 16; c += PART * 256) {
                uint4 x[PART];
#pragma unroll
                for (int e = 0; e < PART; ++e) x[e] = src[c + e * 256];
#pragma unroll
                for (int e = 0; e < PART; ++e) lo[c + e * 256] = make_uint4(lo_bits(x[e].x), lo_bits(x[e].y), lo_bits(x[e].z), lo_bits(x[e].w));
            }
        };
        // the lo tiles are single: the product of the block before that reads them (the first of its three) must be done
        auto ready = [&](int i, uint32_t parity) -> bool { return __all_sync(0xffffffffu, mbar_test_wait(bar(i), parity) ? 1 : 0) != 0; };
        auto do_k = [&](uint32_t jt) {
            split(reinterpret_cast<const uint4 *>(sm + C::K_AT + (jt % C::KS) * C::PLANE), reinterpret_cast<uint4 *>(sm + C::KLO_AT));
            fence_proxy_async_smem();
            mbar_arrive(bar(TB_K_FULL));
        };
        auto do_v = [&](uint32_t jt, int key0) {
            uint4 *tile = reinterpret_cast<uint4 *>(sm + C::V_AT + (jt % C::VS) * C::PLANE);
            bool odd = false;
            if (key0 + KB > p.s.len) {
                // rows behind the last one hold anything, and rows that only some tokens see must not reach the others through
                // 0 * inf: such values leave the product
#pragma unroll 1
                for (int c = ct; c < C::PLANE / 16; c += 256) {
                    const int j = key0 + (c >> 3) % KB - p.s.len;   // rows are 128 bytes whatever the swizzle
                    if (j < 0) continue;
                    uint4 x = tile[c];
                    uint32_t *w = &x.x;
                    bool change = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (j >= p.s.n || !finite_f(__uint_as_float(w[e]))) {
                            odd = odd || j < p.s.n;
                            change = true;
                            w[e] = 0;
                        }
                    if (change) tile[c] = x;
                }
            }
            split(tile, reinterpret_cast<uint4 *>(sm + C::VLO_AT));   // (a thread meets the pieces it changed)
            // (the word's last reader folded block jt - 4: the product of block jt - 1, which has begun, had to wait for the
            // accumulator of block jt - 2 or jt - 3)
            if (odd) s_odd[jt & 3] = (int)jt + 1;
            fence_proxy_async_smem();
            mbar_arrive(bar(TB_V_FULL));
        };
        while (ok && next_piece(a, line, cur, p)) {
            if (np && !wait_all(TB_Q_EMPTY, (np - 1) & 1)) { ok = false; break; }
            ++np;
            // the piece's query rows: row r of the key head is head r / n, token r % n.  s_row: rows of Q from the key head's first
            if (ct < ROWS) {
                const int r = p.block * ROWS + ct, gh = r / p.s.n;
                s_row[ct] = r < p.s.rows ? gh * a.T + (r - gh * p.s.n) : -1;
            }
            conv_sync();
            const float *q0 = a.Q + ((int64_t)p.b * a.H + p.hk * heads_per) * a.T * a.dk;
#pragma unroll 4
            for (int i = ct; i < ROWS * (C::DKP / 4); i += 256) {
                const int r = i / (C::DKP / 4), c = i - r * (C::DKP / 4), row = s_row[r];
                const bool get = row >= 0 && 4 * c < a.dk;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + C::Q_AT + (c >> 3) * C::QSLAB + r * 128 + (((c & 7) ^ (r & 7)) << 4)),
                             "l"(get ? q0 + (int64_t)row * a.dk + 4 * c : a.Q), "r"(get ? 16 : 0)
                             : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (C::WIDE) {
                conv_sync();
                if (ct < ROWS) {   // thread = row: lane of tensor memory
                    const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16) + C::T_QLO;
#pragma unroll 1
                    for (int sl = 0; sl < NSLAB; ++sl) {
                        uint32_t r32[32];
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const uint4 x = *reinterpret_cast<const uint4 *>(sm + C::Q_AT + sl * C::QSLAB + ct * 128 + ((c ^ (ct & 7)) << 4));
                            r32[4 * c] = lo_bits(x.x); r32[4 * c + 1] = lo_bits(x.y); r32[4 * c + 2] = lo_bits(x.z); r32[4 * c + 3] = lo_bits(x.w);
                        }
                        tmem_st_32x32(at + 32 * sl, r32);
                    }
                    tmem_st_wait();
                    tc_fence_before_sync();
                }
            } else {
#pragma unroll 4
                for (int i = ct; i < ROWS * (C::DKP / 4); i += 256) {   // (the pieces this thread brought)
                    const int r = i / (C::DKP / 4), c = i - r * (C::DKP / 4);
                    uint8_t *at = sm + C::Q_AT + (c >> 3) * C::QSLAB + r * 128 + (((c & 7) ^ (r & 7)) << 4);
                    const uint4 x = *reinterpret_cast<const uint4 *>(at);
                    *reinterpret_cast<uint4 *>(at + C::QPLANE) = make_uint4(lo_bits(x.x), lo_bits(x.y), lo_bits(x.z), lo_bits(x.w));
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(bar(TB_Q_FULL));
            {   // the next piece's rows into L2: there is one Q buffer, and the scores wait for it
                TreeCursor ahead = cur;
                TreePiece pn;
                if (next_piece(a, line, ahead, pn)) {
                    const int r = pn.block * ROWS + (ct >> 2) % ROWS, gh = r / pn.s.n;
                    if (r < pn.s.rows && (ct & 3) * 32 < a.dk && ct < 4 * ROWS) {
                        const float *src = a.Q + (((int64_t)pn.b * a.H + pn.hk * heads_per + gh) * a.T + r - gh * pn.s.n) * a.dk + (ct & 3) * 32;
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(src));
                    }
                }
            }
            // K and V blocks in whichever order they can be taken (every warp for itself: its part of a tile is its own)
            uint32_t kt = it, vt = it;
            const uint32_t end = it + p.count;
            for (uint32_t idle = 0; ok && (kt < end || vt < end);) {
                if (kt < end && ready(TB_K_RAW + kt % C::KS, (kt / C::KS) & 1) && (!kt || ready(TB_KLO_EMPTY, (kt - 1) & 1))) {
                    do_k(kt++);
                    idle = 0;
                } else if (vt < end && ready(TB_V_RAW + vt % C::VS, (vt / C::VS) & 1) && (!vt || ready(TB_VLO_EMPTY, (vt - 1) & 1))) {
                    do_v(vt, (p.t0 + (int)(vt - it)) * KB);
                    ++vt;
                    idle = 0;
                } else {
                    __nanosleep(20);
                    ok = ++idle < (1u << 24) && !s_gave_up;
                    ok = __all_sync(0xffffffffu, ok);
                }
            }
            it = end;
        }
        if (!ok && lane == 0) give_up(CERR_CONVERT);
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
        // ---------------------------------------------------------- softmax
        if (FEW && (warp & 3) >= 2) {
            // The products' rows 64 to 127 come from nowhere and go nowhere; zeros take the least power (at full rate the chip's
            // limit sets the clock).
            uint32_t zero[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) zero[c] = 0;
            const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16);
            if (warp < 4) {
#pragma unroll 1
                for (int c = 0; c < 2 * KB; c += 32) tmem_st_32x32(at + C::T_P + c, zero);
            } else if (C::WIDE) {
#pragma unroll 1
                for (int c = 0; c < C::DKP; c += 32) tmem_st_32x32(at + C::T_QLO + c, zero);
            }
            tmem_st_wait();
        }
        const int half = warp >> 2, row = (warp & 3) * 32 + lane;   // row = lane of tensor memory
        const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp & 3)) : "memory"); };   // the two warps of 32 rows
        float o[OH], m, l;
        while ((warp & 3) * 32 < ROWS && next_piece(a, line, cur, p)) {   // (with 64 rows the warps of lanes 64 to 127 have none)
            const int r = p.block * ROWS + row, gh = r / p.s.n, tok = r < p.s.rows ? r - gh * p.s.n : 0;
            const bool mine = r < p.s.rows;
            m = -INFINITY;
            l = 0.f;
#pragma unroll
            for (int c = 0; c < OH; ++c) o[c] = 0.f;
            // o = (o + O of block jt) * f, jt the block before `it`
            auto fold = [&](uint32_t jt, int key0, float f) {
                tc_fence_after_sync();
                const bool odd = s_odd[jt & 3] == (int)jt + 1;
#pragma unroll
                for (int h = 0; h < OH / FOLD; ++h) {
                    uint32_t x[FOLD];
                    const uint32_t at = lane_base + C::T_O + (jt % C::OB) * C::DKP + half * OH + FOLD * h;
                    if constexpr (FOLD == 32) tmem_ld_32x32(at, x);
                    else tmem_ld_32x32_x16(at, x);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < FOLD; ++c) o[FOLD * h + c] += __uint_as_float(x[c]);
                }
                tc_fence_before_sync();
                mbar_arrive(bar(TB_O_EMPTY + jt % C::OB));
                if (odd && mine) {
                    // rare: an infinity or a NaN among the new rows' values goes to the rows that see it, and to no others
#pragma unroll 1
                    for (int key = key0; key < key0 + KB; ++key) {
                        const int j = key - p.s.len;
                        if (j < 0 || j >= p.s.n || !tree_sees(a, p.b, tok, j)) continue;
                        const float *src = a.V + (((int64_t)p.b * a.Hkv + p.hk) * a.max_seq + key) * a.dk + half * OH;
#pragma unroll
                        for (int c = 0; c < OH; c += 4) {   // (dk is a multiple of 4)
                            if (half * OH + c >= a.dk) continue;
                            float4 v;   // (volatile: not all of the row's loads at once, o has the registers)
                            asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(src + c));
                            if (!finite_f(v.x)) o[c] += v.x;
                            if (!finite_f(v.y)) o[c + 1] += v.y;
                            if (!finite_f(v.z)) o[c + 2] += v.z;
                            if (!finite_f(v.w)) o[c + 3] += v.w;
                        }
                    }
                }
                if (__any_sync(0xffffffffu, f != 1.f)) {
#pragma unroll
                    for (int c = 0; c < OH; ++c) o[c] *= f;
                }
            };
            for (int i = 0; i < p.count; ++i, ++it) {
                const uint32_t b = it & 1;
                const int key0 = (p.t0 + i) * KB;
                constexpr int NCH = KB / 64;   // a thread's columns, 32 at a time
                const int first = key0 + half * (KB / 2) - p.s.len;   // new-token index of its first column
                const bool tail = first + KB / 2 > 0;
                if (ok && !wait_all(TB_S_FULL + it % C::SB, (it / C::SB) & 1)) ok = false;
                float mx = -INFINITY;
                uint32_t x[NCH][32], see[NCH];
                if (ok) {
                    tc_fence_after_sync();
#pragma unroll
                    for (int c0 = 0; c0 < NCH; ++c0) tmem_ld_32x32(lane_base + C::T_S + (it % C::SB) * KB + half * (KB / 2) + 32 * c0, x[c0]);
                    tmem_ld_wait();
                    tc_fence_before_sync();
                    mbar_arrive(bar(TB_S_EMPTY + it % C::SB));
                    // the largest of c * score: of the scores themselves, or the smallest where c is negative
                    const uint32_t flip = a.c_log2 < 0.f ? 0x80000000u : 0u;
                    float t4[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
                    for (int c0 = 0; c0 < NCH; ++c0) {
                        see[c0] = tail ? seen_bits(a, p.b, tok, p.s.n, first + 32 * c0) : 0xFFFFFFFFu;
                        if (tail || flip) {
#pragma unroll
                            for (int c = 0; c < 32; ++c)
                                if (see[c0] >> c & 1) t4[c & 3] = fmaxf(t4[c & 3], __uint_as_float(x[c0][c] ^ flip));
                        } else {
#pragma unroll
                            for (int c = 0; c < 32; c += 8)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    t4[e] = fmaxf(t4[e], fmaxf(__uint_as_float(x[c0][c + 2 * e]), __uint_as_float(x[c0][c + 2 * e + 1])));
                        }
                    }
                    mx = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3]));
                    if (mx != -INFINITY) mx *= fabsf(a.c_log2);   // (nothing seen: as it is, 0 * -inf would be NaN)
                }
                s_max[b][half][row] = mx;
                pair_sync();
                if (!ok) continue;
                mx = fmaxf(mx, s_max[b][half ^ 1][row]);
                float corr = 1.f;
                if (mx > m + 8.f) {
                    corr = ex2_approx(m - mx);   // 0 the first time
                    m = mx;
                }
                const float neg = m == -INFINITY ? 0.f : -m;
                float sum[4] = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
                for (int c0 = 0; c0 < NCH; ++c0) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) x[c0][c] = __float_as_uint(ex2_approx(fmaf(__uint_as_float(x[c0][c]), a.c_log2, neg)));
                    if (tail) {
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (!(see[c0] >> c & 1)) x[c0][c] = 0;
                    }
#pragma unroll
                    for (int c = 0; c < 32; ++c) sum[c & 3] += __uint_as_float(x[c0][c]);
                }
                l = l * corr + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                // P is single: the product of the block before must have read it
                if (i > 0 && !wait_all(TB_O_FULL, (it - 1) & 1)) { ok = false; continue; }
                tc_fence_after_sync();
                const uint32_t p_at = lane_base + C::T_P + half * (KB / 2);
#pragma unroll
                for (int c0 = 0; c0 < NCH; ++c0) tmem_st_32x32(p_at + 32 * c0, x[c0]);
                tmem_st_wait();
                tc_fence_before_sync();
                mbar_arrive(bar(TB_P_FULL));   // P hi: the first product can start (with one accumulator: once it is folded)
                if (i > 0 && C::OB == 1) fold(it - 1, key0 - KB, corr);
#pragma unroll
                for (int c0 = 0; c0 < NCH; ++c0) {
#pragma unroll
                    for (int c = 0; c < 32; ++c) x[c0][c] = lo_bits(x[c0][c]);
                    tmem_st_32x32(p_at + (C::T_PLO - C::T_P) + 32 * c0, x[c0]);
                }
                tmem_st_wait();
                tc_fence_before_sync();
                mbar_arrive(bar(TB_PLO_FULL));
                if (i > 0 && C::OB == 2) fold(it - 1, key0 - KB, corr);
            }
            if (ok) {
                if (wait_all(TB_O_FULL, (it - 1) & 1)) fold(it - 1, (p.t0 + p.count - 1) * KB, 1.f);
                else ok = false;
            }
            s_max[(it - 1) & 1][half][row] = l;   // (the last block's maxima have been read: its product had to wait for that)
            pair_sync();
            l += s_max[(it - 1) & 1][half ^ 1][row];

            if (p.pieces > 1) {
                // a piece of a shared item: [16-byte column][row] outputs, then [row] (maximum, sum), for the kernel behind this one
                float4 *s = reinterpret_cast<float4 *>(a.slots) + (size_t)tree_slot(blockIdx.x, p.t0 == 0) * (KT_SLOT_BYTES / 16);
#pragma unroll
                for (int c = 0; c < OH / 4; ++c)
                    s[(half * (OH / 4) + c) * ROWS + row] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
                if (half == 0) reinterpret_cast<float2 *>(s + C::DKP / 4 * ROWS)[row] = make_float2(m, l);
                if (p.t0 == 0 && threadIdx.x == 0) a.shared[blockIdx.x] = KvTreeShared{ p.pieces, p.b, p.hk, p.block, p.s.n, p.s.rows };
            }
            if (p.pieces == 1 && mine) {
                float *dst = a.out + (((int64_t)p.b * a.H + p.hk * heads_per + gh) * a.T + tok) * a.dk + half * OH;
                const float inv = l == 0.f ? 0.f : 1.0f / l;   // nothing seen: 0
#pragma unroll
                for (int c = 0; c < OH; c += 4)
                    if (half * OH + c < a.dk)
                        *reinterpret_cast<float4 *>(dst + c) = make_float4(o[c] * inv, o[c + 1] * inv, o[c + 2] * inv, o[c + 3] * inv);
            }
        }
        if (!ok && lane == 0) give_up(CERR_SOFTMAX);
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == 19) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, C::COLS);
    }
}

// The shared items' pieces added up, in line order within each of a unit's groups of threads and then over the groups.  A unit is
// a few rows of an item: fewer where more pieces want more groups.  (The CTA that arrived last used to do it, one piece after the
// other on one SM and with a counter's round trip for every piece: 30 us for 148 pieces of 128 rows.)
template <int DKP>
struct TreeJoin {
    static constexpr int COLS = DKP / 4, RG = COLS > 16 ? 16 : COLS > 8 ? 32 : 64, THREADS = RG * COLS;   // rows x groups of a unit
    // as many groups as leave each four pieces, and two rows to a unit (the rows of a 16-byte column then fill a 32-byte sector)
    static __device__ __forceinline__ int groups(int pieces)
    {
        int g = 1;
        while (g < RG / 2 && 8 * g <= pieces) g <<= 1;
        return g;
    }
};

template <int DKP, int ROWS>
__global__ void __launch_bounds__(TreeJoin<DKP>::THREADS, 2) kv_tree_join_kernel(const KvTreeArgs a, int ctas)
{
    using J = TreeJoin<DKP>;
    __shared__ float4 s_o[J::THREADS];
    __shared__ float2 s_ml[J::RG];
    __shared__ int s_upto[256], s_warp[8], s_unit[2];
    __shared__ KvTreeShared s_item[256];
    const int tid = threadIdx.x, lane = tid & 31;
    // units up to and including CTA tid's item
    if (tid < 256) {
        int units = 0;
        if (tid < ctas) {
            const KvTreeShared it = a.shared[tid];
            s_item[tid] = it;
            const int rows = it.rows - it.block * ROWS < ROWS ? it.rows - it.block * ROWS : ROWS, per = J::RG / J::groups(it.pieces);
            if (it.pieces) units = (rows + per - 1) / per;
        }
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, units, o);
            if (lane >= o) units += v;
        }
        s_upto[tid] = units;
        if (lane == 31) s_warp[tid >> 5] = units;
    }
    __syncthreads();
    if (tid < 256)
        for (int w = 0; w < tid >> 5; ++w) s_upto[tid] += s_warp[w];
    __syncthreads();
    for (int unit = blockIdx.x; unit < s_upto[255]; unit += gridDim.x) {
        if (tid < 256) {
            const int before = tid ? s_upto[tid - 1] : 0;
            if (unit >= before && unit < s_upto[tid]) {
                s_unit[0] = tid;
                s_unit[1] = unit - before;
            }
        }
        __syncthreads();
        const int first = s_unit[0];
        const KvTreeShared it = s_item[first];
        const int groups = J::groups(it.pieces), per = J::RG / groups;
        const int r = tid % per, c = tid / per % J::COLS, g = tid / (per * J::COLS), row = s_unit[1] * per + r;
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float2 ml, float4 x) {
            const float m_new = fmaxf(m, ml.x), ref = m_new == -INFINITY ? 0.f : m_new;
            const float f0 = ex2_approx(m - ref), f1 = ex2_approx(ml.x - ref);
            m = m_new;
            l = l * f0 + ml.y * f1;
            o.x = o.x * f0 + x.x * f1;
            o.y = o.y * f0 + x.y * f1;
            o.z = o.z * f0 + x.z * f1;
            o.w = o.w * f0 + x.w * f1;
        };
        constexpr int UN = 4;   // pieces on their way at a time
        for (int k0 = g; k0 < it.pieces; k0 += UN * groups) {
            float2 ml[UN];
            float4 x[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int k = k0 + u * groups;
                const float4 *s = reinterpret_cast<const float4 *>(a.slots) + (size_t)tree_slot(first + k, k == 0) * (KT_SLOT_BYTES / 16);
                const bool has = k < it.pieces && row < ROWS;
                ml[u] = has ? __ldcg(reinterpret_cast<const float2 *>(s + J::COLS * ROWS) + row) : make_float2(-INFINITY, 0.f);
                x[u] = has ? __ldcg(s + c * ROWS + row) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) add(ml[u], x[u]);
        }
        s_o[tid] = o;
        if (c == 0) s_ml[g * per + r] = make_float2(m, l);
        __syncthreads();
        if (g == 0) {
            for (int k = 1; k < groups; ++k) add(s_ml[k * per + r], s_o[tid + k * per * J::COLS]);
            const int at = it.block * ROWS + row, gh = at / it.n, heads_per = a.H / a.Hkv;
            if (row < ROWS && at < it.rows && 4 * c < a.dk) {
                const float inv = l == 0.f ? 0.f : 1.0f / l;   // nothing seen: 0
                *reinterpret_cast<float4 *>(a.out + (((int64_t)it.b * a.H + it.hk * heads_per + gh) * a.T + at - gh * it.n) * a.dk + 4 * c) =
                    make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
            }
        }
    }
}

// ---------------------------------------------------------------------- host

template <int NSLAB, bool FEW>
static int launch_tc(const KvTreeArgs &a, int sm_count, cudaStream_t st)
{
    using C = TreeTc<NSLAB, FEW>;
    static PerDeviceOnce once;
    if (once.first()) {
        cudaError_t e = cudaFuncSetAttribute(kv_tree_tc_kernel<NSLAB, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return (int)e;
    }
    TreeTcMaps tm;
    int e = encode_f32_batched_tmap(&tm.k, a.K, (int64_t)a.B * a.Hkv, a.max_seq, a.dk, a.dk, C::KB, false);
    if (!e) e = encode_f32_batched_tmap(&tm.v, a.V, (int64_t)a.B * a.Hkv, a.max_seq, a.dk, a.dk, C::KB, true);
    if (e) return e;
    kv_tree_tc_kernel<NSLAB, FEW><<<sm_count, TT_THREADS, C::SMEM, st>>>(a, tm);
    if ((e = (int)cudaGetLastError()) != 0) return e;
    using J = TreeJoin<C::DKP>;
    kv_tree_join_kernel<C::DKP, C::ROWS><<<2 * sm_count, J::THREADS, 0, st>>>(a, sm_count);
    return (int)cudaGetLastError();
}

int launch_kv_tree_tc(const KvTreeArgs &a, int sm_count, cudaStream_t st, int *launches)
{
    *launches = 2;
    if (a.H / a.Hkv <= 64 / a.T) {
        if (a.dk <= 32) return launch_tc<1, true>(a, sm_count, st);
        if (a.dk <= 64) return launch_tc<2, true>(a, sm_count, st);
        if (a.dk <= 96) return launch_tc<3, true>(a, sm_count, st);
        return launch_tc<4, true>(a, sm_count, st);
    }
    if (a.dk <= 32) return launch_tc<1, false>(a, sm_count, st);
    if (a.dk <= 64) return launch_tc<2, false>(a, sm_count, st);
    if (a.dk <= 96) return launch_tc<3, false>(a, sm_count, st);
    return launch_tc<4, false>(a, sm_count, st);
}

}  // namespace axb
