// kv_tree_line.cuh — how the kernels of kv_cache_attend_tree divide a ragged batch between their CTAs, on the device.
// The key tiles of all (sequence, key head, row block) items form one line, cut into equal stretches, one a CTA; the
// CTAs that share an item are consecutive and each holds a tile of it.  And the few device functions that they share.
#pragma once
#include "../../include/axiom_b200.h"
#include "device_error.cuh"
#include "kv_tree.cuh"

namespace axb {

// query rows of an item; keys of a tile; tiles that a CTA works on side by side (a shorter stretch takes as long, and an item
// cut into fewer pieces is added up sooner); the tiles in whose time a CTA gets from one item to the next: room for them is
// left on the line behind every item
struct TreeLine {
    int block_rows, tile_keys, min_stretch, gap;
};

struct TreeSeq {
    int len, n, rows, blocks, tiles;   // cached rows, new tokens, query rows of a key head, row blocks, key tiles
    int room;                          // of an item on the line
};

__device__ __forceinline__ TreeSeq tree_seq(const KvTreeArgs &a, const TreeLine &ln, int b, bool *bad = nullptr)
{
    TreeSeq s;
    s.len = __ldg(a.lens + b);
    s.n = a.n_new ? __ldg(a.n_new + b) : a.T;
    const bool off = s.len < 0 || s.n < 0 || s.n > a.T || (int64_t)s.len + s.n > a.max_seq;   // (max_seq <= 2^30)
    if (bad) *bad = off;
    if (off) s.len = s.n = 0;   // refused whole: its output rows are left alone
    s.rows = s.n * (a.H / a.Hkv);
    s.blocks = (s.rows + ln.block_rows - 1) / ln.block_rows;
    s.tiles = s.n ? (s.len + s.n + ln.tile_keys - 1) / ln.tile_keys : 0;
    s.room = s.n ? s.tiles + ln.gap : 0;
    return s;
}

// (the launcher refuses batches whose line could pass 2^31 tiles)
__device__ __forceinline__ int tree_tiles(const KvTreeArgs &a, const TreeSeq &s) { return a.Hkv * s.blocks * s.room; }

struct TreeCursor {
    int b;
    int base;      // where sequence b's part of the line begins
    int pos, end;  // what is left of this CTA's stretch
    int per;       // a stretch
};

// one piece: consecutive tiles of one item
struct TreePiece {
    TreeSeq s;
    int b, hk, block, t0, count;
    int first, pieces;   // the CTA that holds the item's first tile, and how many CTAs hold some
};

// Every thread of the CTA; shared: 3 words.  False: nothing for this CTA (for all its threads).
__device__ __forceinline__ bool tree_start(const KvTreeArgs &a, const TreeLine &ln, int *shared, TreeCursor &c)
{
    const int lane = threadIdx.x & 31;
    auto tiles_of = [&](int b) -> int {
        if (b >= a.B) return 0;
        bool bad;
        const TreeSeq s = tree_seq(a, ln, b, &bad);
        if (bad && blockIdx.x == 0 && a.err) atomicCAS(a.err + ERR_ROWS, 0, (int)AXB_DEVERR_ROWS);
        return tree_tiles(a, s);
    };
    int mine = 0;
    if (a.B > 32) {
        if (threadIdx.x == 0) shared[0] = 0;
        __syncthreads();
        int sum = 0;
        for (int b = threadIdx.x; b < a.B; b += blockDim.x) sum += tiles_of(b);
        sum = __reduce_add_sync(0xffffffffu, sum);
        if (lane == 0 && sum) atomicAdd(shared, sum);
        __syncthreads();
    }
    if (threadIdx.x < 32) {
        // one warp finds the total (of up to 32 sequences) and the sequence in which the stretch begins
        int total = shared[0];
        if (a.B <= 32) {
            mine = tiles_of(lane);
            total = __reduce_add_sync(0xffffffffu, mine);
        }
        const int per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, ln.min_stretch), pos = min(per * (int)blockIdx.x, total);
        int before = 0;
        for (int b0 = 0; pos < total && b0 < a.B; b0 += 32) {
            if (a.B > 32) mine = tiles_of(b0 + lane);
            int upto = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, before + upto > pos);
            if (past) {
                const int k = __ffs(past) - 1;
                if (lane == k) {
                    shared[1] = b0 + k;
                    shared[2] = before + upto - mine;
                }
                break;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        __syncwarp();
        if (lane == 0) shared[0] = total;
    }
    __syncthreads();
    const int total = shared[0];
    c.per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, ln.min_stretch);
    c.pos = min(c.per * (int)blockIdx.x, total);
    c.end = min(c.pos + c.per, total);
    c.b = shared[1];
    c.base = shared[2];
    return c.pos < c.end;
}

__device__ __forceinline__ bool next_piece(const KvTreeArgs &a, const TreeLine &ln, TreeCursor &c, TreePiece &p)
{
    while (c.pos < c.end) {
        p.s = tree_seq(a, ln, c.b);
        const int total = tree_tiles(a, p.s);
        if (c.pos - c.base >= total) {
            c.base += total;
            ++c.b;
            continue;
        }
        const int item = (c.pos - c.base) / p.s.room, item_pos = c.base + item * p.s.room;
        p.b = c.b;
        p.t0 = c.pos - item_pos;
        if (p.t0 >= p.s.tiles) {   // the gap behind an item
            c.pos = item_pos + p.s.room;
            continue;
        }
        p.hk = item / p.s.blocks;
        p.block = item - p.hk * p.s.blocks;
        p.count = min(p.s.tiles - p.t0, c.end - c.pos);
        p.first = item_pos / c.per;
        p.pieces = (item_pos + p.s.tiles - 1) / c.per - p.first + 1;
        c.pos += p.count;
        return true;
    }
    return false;
}

// A CTA holds at most one piece that continues an item (its first) and one that begins an item it does not finish (its
// last): two workspace slots a CTA are enough.
__device__ __forceinline__ int tree_slot(int cta, bool begins) { return 2 * cta + (begins ? 1 : 0); }

// A CTA is done with its piece of a shared item (one thread; what it leaves in its slot is visible by now).  True for the last of
// the item's CTAs, which adds the pieces and clears the counter for the next call.  The item's first CTA names the counter.
__device__ __forceinline__ bool tree_arrive(const KvTreeArgs &a, const TreePiece &p)
{
    return atomicAdd(a.counters + p.first, 1) == p.pieces - 1;
}

// (behind the sum: a store before it is one more thing that the fence in front of the slots' loads waits for, 0.3 us)
__device__ __forceinline__ void tree_clear(const KvTreeArgs &a, const TreePiece &p) { a.counters[p.first] = 0; }

// One thread of a CTA that gave up before its piece number `done`, c as tree_start left it: it arrives for the rest all the same,
// so that every launch leaves the counters at zero, whatever became of its results.
__device__ __forceinline__ void tree_leave(const KvTreeArgs &a, const TreeLine &ln, TreeCursor c, uint32_t done)
{
    TreePiece p;
    for (uint32_t k = 0; next_piece(a, ln, c, p); ++k)
        if (k >= done && p.pieces > 1 && tree_arrive(a, p)) tree_clear(a, p);
}

// whether token t sees new token j
__device__ __forceinline__ bool tree_sees(const KvTreeArgs &a, int b, int t, int j)
{
    if (!a.mask) return j <= t;
    return (__ldg(a.mask + b * a.mask_stride + (int64_t)t * a.words + (j >> 6)) >> (j & 63)) & 1;
}

// The lo part of x: what the tensor core, which reads the upper 19 bits of an operand, leaves of x as a hi operand; rounded
// to the bits it will read (cut, it would keep the sign of x — a bias that the sums over columns and keys add up).
__device__ __forceinline__ uint32_t tf32_lo(float x)
{
    return __float_as_uint(x - __uint_as_float(__float_as_uint(x) & 0xffffe000u)) + 0x1000u;
}

__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

}  // namespace axb
