// rope.cu — the pass between a QKV projection and the attention kernels, and its gradient.  For the token at position
// p and one of its heads x[dk] (q and k heads; v heads are moved as they are):
//     x += bias;   y = x * r * g,  r = 1 / sqrt(mean(x^2) + eps)                     (where a norm weight g is given)
//     (y_a, y_b) -> amplitude * (y_a cos t - y_b sin t, y_b cos t + y_a sin t),  t = p * f_i     for every pair i,
// the pair being elements (i, i + pairs) or (2i, 2i + 1) of the head's first 2*pairs elements.  Backward, with d the
// gradient after the transposed rotation and u = x * r:
//     dg += sum over tokens and heads of d * u;   dx = r * (d*g - u * mean(d*g*u)).
// Rows of dk floats go from the flat [B*T, (H + 2*Hkv)*dk] matrix to head-major buffers — or to the rows lens[b] + t
// of a cache — like the layout pass (head_layout.cu), whose place this takes: one read and one write of every element
// (the backward reads x too where there is a norm).  HBM-bound.
//
// The tokens lie on a line, each of them a number of steps long: a warp step takes as many head rows, all q, all k or all v,
// as fit its lanes.  Every warp gets a stretch of the line of the same length to within a step, and the next step's rows are
// on their way while it works on this one's; where a warp meets a token it forms that token's angles, each pair's once by one
// lane, for all its heads: p * f in turns in 64 bits (a position of 10^6 times a frequency of 1 has lost five of fp32's
// seven digits), the whole turns dropped, and the remainder's sine and cosine in fp32.  No barrier of the CTA is met: with
// CTAs that took four tokens at a time (angles behind a barrier, no row ahead) the backward of 8192 tokens of 16 + 2*8 heads
// of 128 (369 MB) took 113 us, so 70; the forward of 16384 tokens of 32 + 2*8 heads (805 MB) 143 and 135.  The backward's
// instructions, not its bytes, set its time: rows of one kind a step, instead of q, k and v rows side by side with selects,
// made 78 us 70.
//
// A group of lanes owns a head row (any number of lanes up to 32: a head of 80 takes 10, three rows a warp); a lane owns two
// 16-byte pieces of it that hold both partners of its pairs (piece c and c + pairs/4 of the half-split layout; the
// interleaved pairs lie inside a piece), so the rotation needs no exchange and the norm one shuffle tree.  Head dims and
// rotated parts that do not cut into 16-byte pieces, and unaligned tensors, take the same kernel with single floats in the
// place of the pieces.
#include "rope.cuh"

#include "device_error.cuh"

#include <math.h>

namespace axb {

static constexpr int RP_THREADS = 128, RP_WARPS = RP_THREADS / 32, RP_FWD_CTAS = 8, RP_BWD_CTAS = 5, RP_BWD_SETS = 8;
static constexpr double RP_INV_2PI = 0.15915494309189533577;

// which pieces (VEC floats each) of a head row unit u of a lane covers, and whether they form rotated pairs
template <int VEC>
struct RopeUnit {
    int v0, v1;      // piece indices, -1: none
    int p0, p1;      // first pair of the rotation of piece 0 (of both, unless whole pairs lie in a piece; -1: not rotated)
};

template <int VEC, bool INTER>
__device__ __forceinline__ RopeUnit<VEC> rope_unit(int u, int dk, int pairs)
{
    const int nv = dk / VEC;
    RopeUnit<VEC> r;
    if (INTER && VEC == 4) {
        const int h = (nv + 1) / 2, rv = pairs / 2;   // rotated pieces: two pairs each
        r.v0 = u < h ? u : -1;
        r.v1 = u + h < nv && u < h ? u + h : -1;
        r.p0 = r.v0 >= 0 && r.v0 < rv ? 2 * r.v0 : -1;
        r.p1 = r.v1 >= 0 && r.v1 < rv ? 2 * r.v1 : -1;
        return r;
    }
    const int pu = pairs / VEC;
    if (u < pu) {
        r.v0 = INTER ? 2 * u : u;
        r.v1 = INTER ? 2 * u + 1 : u + pu;
        r.p0 = u * VEC;
        r.p1 = -1;
    } else {
        const int t = u - pu, tail = nv - 2 * pu, tu = (tail + 1) / 2;
        r.v0 = t < tu ? 2 * pu + t : -1;
        r.v1 = t < tu && t + tu < tail ? 2 * pu + t + tu : -1;
        r.p0 = r.p1 = -1;
    }
    return r;
}

template <int VEC>
struct Piece {
    float x[VEC];
};

// (16-byte pieces: a lane without a second piece reads its first again, and its caller leaves it out of the sums)
template <int VEC>
__device__ __forceinline__ Piece<VEC> load_piece(const float *row, int v, int else_v)
{
    Piece<VEC> p;
    if (VEC == 4) {
        const float4 t = *reinterpret_cast<const float4 *>(row + 4 * (v < 0 ? else_v : v));
        p.x[0] = t.x; p.x[1 % VEC] = t.y; p.x[2 % VEC] = t.z; p.x[3 % VEC] = t.w;
    } else {
        p.x[0] = v < 0 ? 0.f : row[v];
    }
    return p;
}

template <int VEC>
__device__ __forceinline__ void store_piece(float *row, int v, const Piece<VEC> &p)
{
    if (v < 0) return;
    if (VEC == 4) *reinterpret_cast<float4 *>(row + 4 * v) = make_float4(p.x[0], p.x[1 % VEC], p.x[2 % VEC], p.x[3 % VEC]);
    else row[v] = p.x[0];
}

// rotates a lane's two pieces by its angles (cosines and sines times the amplitude); BACK turns the other way (the transpose)
template <int VEC, bool INTER, bool BACK>
__device__ __forceinline__ void rotate_unit(const RopeUnit<VEC> &u, const float *cs, const float *sn, Piece<VEC> &a, Piece<VEC> &b)
{
    if (!(INTER && VEC == 4)) {
        if (u.p0 < 0) return;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float c = cs[i], s = BACK ? -sn[i] : sn[i];
            const float x = a.x[i], y = b.x[i];
            a.x[i] = x * c - y * s;
            b.x[i] = y * c + x * s;
        }
        return;
    }
    auto turn = [&](Piece<VEC> &p, int at) {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
            const float c = cs[(at + i / 2) % VEC], s = BACK ? -sn[(at + i / 2) % VEC] : sn[(at + i / 2) % VEC];
            const float x = p.x[i], y = p.x[(i + 1) % VEC];
            p.x[i] = x * c - y * s;
            p.x[(i + 1) % VEC] = y * c + x * s;
        }
    };
    if (u.p0 >= 0) turn(a, 0);
    if (u.p1 >= 0) turn(b, 2);
}

// the sums of N numbers over a row's `width` lanes, in each of them (li: the lane's place in the row; lanes past the last
// row get what nobody uses)
template <int N>
__device__ __forceinline__ void lanes_sum(float *v, int li, int width)
{
    if ((width & (width - 1)) == 0) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            if (o < width) {
#pragma unroll
                for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
            }
        return;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float t = __shfl_down_sync(0xffffffffu, v[n], o);
            if (li + o < width) v[n] += t;
        }
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = __shfl_sync(0xffffffffu, v[n], (int)(threadIdx.x & 31) - li);
}

struct RopePlan {
    int lpr, rpw;   // lanes of a head row, head rows a warp takes at a time
    int sq, sk;     // steps of a token's q heads and of its k or v heads (a step's rows are of one kind: the code of a step
    int steps;      // is then the same for the whole warp); steps of a token: sq + 2*sk
    int blocks;
};

// A token: number s of sequence b (b < 0: not wanted), its row among the sequence's keys, its position.
struct RopeToken {
    int tok, b, s, kv, p;
};

__device__ __forceinline__ RopeToken rope_token(const RopeArgs &a, int tok)
{
    RopeToken t;
    t.tok = tok;
    t.b = tok / a.T;
    t.s = t.kv = tok - t.b * a.T;
    bool valid = true;
    if (a.lens) {
        const int len = a.lens[t.b], n = a.n_new ? a.n_new[t.b] : a.T;
        // a sequence that does not fit its rows is refused whole: nothing of it is read or written
        const bool bad = len < 0 || n < 0 || n > a.T || (int64_t)len + n > a.kv_rows;
        if (bad && a.err && (threadIdx.x & 31) == 0) atomicCAS(a.err + ERR_ROWS, 0, (int)AXB_DEVERR_ROWS);
        valid = !bad && t.s < n;
        if (valid) t.kv += len;
    }
    t.p = !valid ? 0 : a.pos ? a.pos[tok] : t.kv;
    if (!valid) t.b = -1;
    return t;
}

// A warp's stretch of the work line (all tokens in order, each `steps` long), and its place in it.
struct RopeCursor {
    int left;   // steps from here to the stretch's end
    int step;   // of the token
    RopeToken t;
};

__device__ __forceinline__ void rope_seek(RopeCursor &c, const RopeArgs &a, const RopePlan &p)
{
    while (c.left > 0 && c.t.b < 0) {   // the rest of a token that is not wanted
        c.left -= p.steps - c.step;
        c.step = 0;
        if (c.left > 0) c.t = rope_token(a, c.t.tok + 1);
    }
}

__device__ __forceinline__ RopeCursor rope_start(const RopeArgs &a, const RopePlan &p)
{
    RopeCursor c;
    const int64_t total = (int64_t)a.B * a.T * p.steps, warps = (int64_t)gridDim.x * RP_WARPS;
    const int64_t w = (int64_t)blockIdx.x * RP_WARPS + (threadIdx.x >> 5), each = total / warps, more = total % warps;
    const int64_t first = w * each + (w < more ? w : more);
    c.left = (int)each + (w < more);
    c.step = 0;
    c.t = RopeToken{ 0, -1, 0, 0, 0 };
    if (c.left == 0) return c;
    c.step = (int)(first % p.steps);
    c.t = rope_token(a, (int)(first / p.steps));
    rope_seek(c, a, p);
    return c;
}

__device__ __forceinline__ void rope_next(RopeCursor &c, const RopeArgs &a, const RopePlan &p)
{
    --c.left;
    if (++c.step < p.steps || c.left <= 0) return;
    c.step = 0;
    c.t = rope_token(a, c.t.tok + 1);
    rope_seek(c, a, p);
}

// The angles of position pos: each pair's once, by one lane, through the warp's 2*pairs words of shared memory.
template <int VEC, bool INTER, int NU>
__device__ __forceinline__ void rope_angles(const RopeArgs &a, int pos, float *table, const RopeUnit<VEC> *u, float *cs, float *sn)
{
    __syncwarp();   // the words before are read
    for (int i = threadIdx.x & 31; i < a.pairs; i += 32) {
        const double turns = (double)pos * (a.freq[i] * RP_INV_2PI);
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        table[i] = c * a.amplitude;
        table[a.pairs + i] = s * a.amplitude;
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < NU; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int at = INTER && VEC == 4 ? (i < 2 ? u[j].p0 + i : u[j].p1 + i - 2) : u[j].p0 + i;
            const bool has = INTER && VEC == 4 && i >= 2 ? u[j].p1 >= 0 : u[j].p0 >= 0;
            cs[j * VEC + i] = has ? table[at] : 1.f;
            sn[j * VEC + i] = has ? table[a.pairs + at] : 0.f;
        }
}

// A step's rows: which kind, the lane's head of that kind (none past the last: `on` false, the row then read is another
// one's), where it stands in qkv and in the head-major buffer.
enum RopeKind { ROPE_Q, ROPE_K, ROPE_V };

struct RopeRow {
    int kind;
    bool on;
    int64_t flat, head;   // element offsets
};

__device__ __forceinline__ RopeRow rope_row(const RopeArgs &a, const RopePlan &p, const RopeCursor &c, int row)
{
    RopeRow r;
    const int kv = c.step - p.sq;
    r.kind = kv < 0 ? ROPE_Q : kv < p.sk ? ROPE_K : ROPE_V;
    const int count = kv < 0 ? a.H : a.Hkv, at = kv < 0 ? c.step : kv < p.sk ? kv : kv - p.sk;
    int h = at * p.rpw + row;
    r.on = row < p.rpw && h < count;
    h = r.on ? h : at * p.rpw;
    r.flat = ((int64_t)c.t.tok * (a.H + 2 * a.Hkv) + (kv < 0 ? 0 : kv < p.sk ? a.H : a.H + a.Hkv) + h) * a.dk;
    r.head = kv < 0 ? (((int64_t)c.t.b * a.H + h) * a.T + c.t.s) * a.dk : (((int64_t)c.t.b * a.Hkv + h) * a.kv_rows + c.t.kv) * a.dk;
    return r;
}

template <int VEC, bool INTER>
__global__ void __launch_bounds__(RP_THREADS, RP_FWD_CTAS) qkv_norm_rope_kernel(const RopeArgs a, const RopePlan p)
{
    constexpr int NU = VEC == 4 ? 1 : 4;   // units a lane covers: 32 lanes hold 256 floats either way
    extern __shared__ float smem[];
    float *table = smem + (threadIdx.x >> 5) * 2 * a.pairs;
    const int lane = threadIdx.x & 31, row = lane / p.lpr, li = lane - row * p.lpr;
    RopeUnit<VEC> u[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) u[j] = rope_unit<VEC, INTER>(li + 32 * j, a.dk, a.pairs);
    const float inv_dk = 1.0f / (float)a.dk;
    float cs[NU * VEC], sn[NU * VEC];
    int angles_of = -1;

    RopeCursor c = rope_start(a, p);
    RopeRow nr;
    Piece<VEC> n0[NU], n1[NU];   // the next step's rows, on their way while this step's are worked on
    auto load = [&]() {
        nr = rope_row(a, p, c, row);
        const float *src = a.qkv + nr.flat;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            n0[j] = load_piece<VEC>(src, u[j].v0, 0);
            n1[j] = load_piece<VEC>(src, u[j].v1, u[j].v0);
        }
    };
    if (c.left > 0) load();
    while (c.left > 0) {   // (the same for all lanes of a warp: the norm's shuffles need every one)
        Piece<VEC> x0[NU], x1[NU];
#pragma unroll
        for (int j = 0; j < NU; ++j) { x0[j] = n0[j]; x1[j] = n1[j]; }
        const RopeRow r = nr;
        const int tok = c.t.tok, pos = c.t.p;
        rope_next(c, a, p);
        if (c.left > 0) load();
        if (a.bias) {
            const float *bias = a.bias + (r.flat - (int64_t)tok * (a.H + 2 * a.Hkv) * a.dk);
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                const Piece<VEC> b0 = load_piece<VEC>(bias, u[j].v0, 0), b1 = load_piece<VEC>(bias, u[j].v1, u[j].v0);
#pragma unroll
                for (int i = 0; i < VEC; ++i) { x0[j].x[i] += b0.x[i]; x1[j].x[i] += b1.x[i]; }
            }
        }
        if (r.kind != ROPE_V) {
            if (tok != angles_of) {
                rope_angles<VEC, INTER, NU>(a, pos, table, u, cs, sn);
                angles_of = tok;
            }
            if (const float *g = r.kind == ROPE_Q ? a.gq : a.gk) {
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < NU; ++j) {
                    float s0 = 0.f, s1 = 0.f;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) { s0 += x0[j].x[i] * x0[j].x[i]; s1 += x1[j].x[i] * x1[j].x[i]; }
                    ss += s0 + (u[j].v1 >= 0 ? s1 : 0.f);
                }
                lanes_sum<1>(&ss, li, p.lpr);
                const float rs = rsqrtf(ss * inv_dk + a.eps);
#pragma unroll
                for (int j = 0; j < NU; ++j) {
                    const Piece<VEC> g0 = load_piece<VEC>(g, u[j].v0, 0), g1 = load_piece<VEC>(g, u[j].v1, u[j].v0);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        x0[j].x[i] = x0[j].x[i] * rs * g0.x[i];
                        x1[j].x[i] = x1[j].x[i] * rs * g1.x[i];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NU; ++j) rotate_unit<VEC, INTER, false>(u[j], cs + j * VEC, sn + j * VEC, x0[j], x1[j]);
        }
        if (r.on) {
            float *dst = (r.kind == ROPE_Q ? a.q : r.kind == ROPE_K ? a.k : a.v) + r.head;
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                store_piece<VEC>(dst, u[j].v0, x0[j]);
                store_piece<VEC>(dst, u[j].v1, x1[j]);
            }
        }
    }
}

// A step of the backward's rows that have a norm weight: d (rotated back) becomes dx, d*u is added to acc.
template <int VEC, int NU>
__device__ __forceinline__ void norm_back(const RopeArgs &a, const float *g, const RopeUnit<VEC> *u, int li, int lpr, float inv_dk, bool on,
                                          Piece<VEC> *d0, Piece<VEC> *d1, const Piece<VEC> *x0, const Piece<VEC> *x1,
                                          float (&acc)[2][NU][VEC])
{
    float sum[2] = { 0.f, 0.f };   // x^2, d*g*x
    Piece<VEC> g0[NU], g1[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) {
        g0[j] = load_piece<VEC>(g, u[j].v0, 0);
        g1[j] = load_piece<VEC>(g, u[j].v1, u[j].v0);
        float s0 = 0.f, s1 = 0.f, e0 = 0.f, e1 = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            g0[j].x[i] *= d0[j].x[i];
            g1[j].x[i] *= d1[j].x[i];
            s0 += x0[j].x[i] * x0[j].x[i];
            s1 += x1[j].x[i] * x1[j].x[i];
            e0 += g0[j].x[i] * x0[j].x[i];
            e1 += g1[j].x[i] * x1[j].x[i];
        }
        sum[0] += s0 + (u[j].v1 >= 0 ? s1 : 0.f);
        sum[1] += e0 + (u[j].v1 >= 0 ? e1 : 0.f);
    }
    lanes_sum<2>(sum, li, lpr);
    const float rs = rsqrtf(sum[0] * inv_dk + a.eps), mean = sum[1] * rs * inv_dk;   // mean(d*g*u)
#pragma unroll
    for (int j = 0; j < NU; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float u0 = x0[j].x[i] * rs, u1 = x1[j].x[i] * rs;
            if (on) {
                acc[0][j][i] += d0[j].x[i] * u0;
                acc[1][j][i] += d1[j].x[i] * u1;
            }
            d0[j].x[i] = rs * (g0[j].x[i] - u0 * mean);
            d1[j].x[i] = rs * (g1[j].x[i] - u1 * mean);
        }
}

// The gradient: the same ownership the other way.  A lane meets the same head elements in every row, so the norm weights'
// gradients collect in its registers; rows are added in shared memory, CTAs by rope_dgamma_kernel, each in a fixed order.
template <int VEC, bool INTER>
__global__ void __launch_bounds__(RP_THREADS, RP_BWD_CTAS) qkv_norm_rope_bwd_kernel(const RopeArgs a, const RopePlan p)
{
    constexpr int NU = VEC == 4 ? 1 : 4;
    extern __shared__ float smem[];
    float *table = smem + (threadIdx.x >> 5) * 2 * a.pairs;
    const int lane = threadIdx.x & 31, row = lane / p.lpr, li = lane - row * p.lpr;
    RopeUnit<VEC> u[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) u[j] = rope_unit<VEC, INTER>(li + 32 * j, a.dk, a.pairs);
    const float inv_dk = 1.0f / (float)a.dk;
    float cs[NU * VEC], sn[NU * VEC];
    int angles_of = -1;
    float acc[2][2][NU][VEC];   // [q, k][piece][unit]
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < NU; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[w][e][j][i] = 0.f;

    RopeCursor c = rope_start(a, p);
    RopeRow nr;
    Piece<VEC> nd0[NU], nd1[NU], nx0[NU], nx1[NU];
    auto load = [&]() {
        nr = rope_row(a, p, c, row);
        const float *src = (nr.kind == ROPE_Q ? a.q : nr.kind == ROPE_K ? a.k : a.v) + nr.head;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            nd0[j] = load_piece<VEC>(src, u[j].v0, 0);
            nd1[j] = load_piece<VEC>(src, u[j].v1, u[j].v0);
        }
        if (nr.kind == ROPE_Q ? a.gq : nr.kind == ROPE_K ? a.gk : nullptr) {
            const float *in = a.qkv + nr.flat;
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                nx0[j] = load_piece<VEC>(in, u[j].v0, 0);
                nx1[j] = load_piece<VEC>(in, u[j].v1, u[j].v0);
            }
        }
    };
    if (c.left > 0) load();
    while (c.left > 0) {
        Piece<VEC> d0[NU], d1[NU], x0[NU], x1[NU];
#pragma unroll
        for (int j = 0; j < NU; ++j) { d0[j] = nd0[j]; d1[j] = nd1[j]; x0[j] = nx0[j]; x1[j] = nx1[j]; }
        const RopeRow r = nr;
        const int tok = c.t.tok, pos = c.t.p;
        rope_next(c, a, p);
        if (c.left > 0) load();
        if (r.kind != ROPE_V) {
            if (tok != angles_of) {
                rope_angles<VEC, INTER, NU>(a, pos, table, u, cs, sn);
                angles_of = tok;
            }
#pragma unroll
            for (int j = 0; j < NU; ++j) rotate_unit<VEC, INTER, true>(u[j], cs + j * VEC, sn + j * VEC, d0[j], d1[j]);
            if (const float *g = r.kind == ROPE_Q ? a.gq : a.gk) {
                if (a.bias) {
                    const float *bias = a.bias + (r.flat - (int64_t)tok * (a.H + 2 * a.Hkv) * a.dk);
#pragma unroll
                    for (int j = 0; j < NU; ++j) {
                        const Piece<VEC> b0 = load_piece<VEC>(bias, u[j].v0, 0), b1 = load_piece<VEC>(bias, u[j].v1, u[j].v0);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) { x0[j].x[i] += b0.x[i]; x1[j].x[i] += b1.x[i]; }
                    }
                }
                if (r.kind == ROPE_Q) norm_back<VEC, NU>(a, g, u, li, p.lpr, inv_dk, r.on, d0, d1, x0, x1, acc[0]);
                else norm_back<VEC, NU>(a, g, u, li, p.lpr, inv_dk, r.on, d0, d1, x0, x1, acc[1]);
            }
        }
        if (r.on) {
            float *dst = a.dqkv + r.flat;
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                store_piece<VEC>(dst, u[j].v0, d0[j]);
                store_piece<VEC>(dst, u[j].v1, d1[j]);
            }
        }
    }
    if (!a.partial) return;
    // [row][dk] per norm weight, then one thread per element adds the rows in order
    const int rows = RP_WARPS * p.rpw, mine = (threadIdx.x >> 5) * p.rpw + row;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        __syncthreads();
        if (row < p.rpw) {
#pragma unroll
            for (int j = 0; j < NU; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    if (u[j].v0 >= 0) smem[mine * a.dk + u[j].v0 * VEC + i] = acc[w][0][j][i];
                    if (u[j].v1 >= 0) smem[mine * a.dk + u[j].v1 * VEC + i] = acc[w][1][j][i];
                }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < a.dk; d += RP_THREADS) {
            float s = 0.f;
            for (int k = 0; k < rows; ++k) s += smem[k * a.dk + d];
            a.partial[((int64_t)blockIdx.x * 2 + w) * a.dk + d] = s;
        }
    }
}

// dg[w][d] += sum over blocks of partial[block][w][d], in 64 bits: 64 strands, each in block order, then in strand order.
// dgq == dgk (one weight for queries and keys): its element is one thread's, which adds both sums.
__global__ void __launch_bounds__(512) rope_dgamma_kernel(const float *partial, int blocks, int dk, float *dgq, float *dgk)
{
    __shared__ double red[64][9];
    const bool tied = dgq == dgk;
    const int x = threadIdx.x & 7, c = blockIdx.x * 8 + x, strand = threadIdx.x >> 3, columns = tied ? dk : 2 * dk;
    double s = 0.0;
    if (c < columns) {
#pragma unroll 8
        for (int b = strand; b < blocks; b += 64) s += (double)partial[(int64_t)b * 2 * dk + c];
        if (tied) {
#pragma unroll 8
            for (int b = strand; b < blocks; b += 64) s += (double)partial[((int64_t)b * 2 + 1) * dk + c];
        }
    }
    red[strand][x] = s;
    __syncthreads();
    if (strand == 0 && c < columns) {
        for (int k = 1; k < 64; ++k) s += red[k][x];
        float *dst = c < dk ? dgq : dgk;
        const int d = c < dk ? c : c - dk;
        if (dst) dst[d] = (float)((double)dst[d] + s);
    }
}

// ---------------------------------------------------------------------- host

static bool rope_vec(const RopeArgs &a)
{
    uintptr_t m = 0;
    for (const void *p : { (const void *)a.qkv, (const void *)a.bias, (const void *)a.gq, (const void *)a.gk, (const void *)a.q,
                           (const void *)a.k, (const void *)a.v, (const void *)a.dqkv })
        m |= reinterpret_cast<uintptr_t>(p);
    // whole 16-byte pieces on either side of every pair: half split 2*pairs floats cut in two, interleaved two pairs a piece
    return (m & 15) == 0 && a.dk % 4 == 0 && a.pairs % (a.interleaved ? 2 : 4) == 0;
}

static RopePlan rope_plan(const RopeArgs &a, bool vec, int sm_count, bool backward)
{
    RopePlan p;
    p.lpr = 32;
    if (vec) p.lpr = a.interleaved ? (a.dk / 4 + 1) / 2 : a.pairs / 4 + (a.dk / 4 - a.pairs / 2 + 1) / 2;
    p.rpw = 32 / p.lpr;
    p.sq = (a.H + p.rpw - 1) / p.rpw;
    p.sk = (a.Hkv + p.rpw - 1) / p.rpw;
    p.steps = p.sq + 2 * p.sk;
    const int64_t steps = (int64_t)a.B * a.T * p.steps, need = (steps + RP_WARPS - 1) / RP_WARPS;
    // One set of resident CTAs; where that leaves a warp more than 16 steps, up to four sets, so that an SM that is done early
    // takes more (the forward of 16384 tokens above: one set 148 us, two 136, four 134; 768 tokens: 7.8, 8.6 and 11.1).  The
    // backward, every CTA of it being a term of the norm weights' sums, keeps to one up to 256 steps a warp and to stretches of no
    // more than some 256 from there, up to eight sets: a lane adds in 32 bits, and the error of its sum grows with the root of its
    // terms (262,144 tokens of 16 + 2*8 heads of 128: 4.6e-7 of the gradient's norm with one set, 2100 us; 64 steps 1.7e-7, but 1 to
    // 2 per cent slower from 32,768 tokens on).
    int64_t most = (int64_t)sm_count * (backward ? RP_BWD_CTAS : RP_FWD_CTAS);
    const int64_t sets = need / ((backward ? 256 : 16) * most), limit = backward ? RP_BWD_SETS : 4;
    most *= sets < 1 ? 1 : sets > limit ? limit : sets;
    p.blocks = (int)(need < most ? need : most);
    return p;
}

static size_t rope_smem(const RopeArgs &a, const RopePlan &p, bool backward)
{
    const size_t n = RP_WARPS * 2 * (size_t)a.pairs * sizeof(float);
    const size_t red = backward ? RP_WARPS * (size_t)p.rpw * a.dk * sizeof(float) : 0;
    return n > red ? n : red;   // at most 8 KB
}

int launch_qkv_norm_rope(const RopeArgs &a, int sm_count, cudaStream_t st)
{
    const bool vec = rope_vec(a);
    const RopePlan p = rope_plan(a, vec, sm_count, false);
    const int grid = p.blocks;
    const size_t smem = rope_smem(a, p, false);
    if (vec && a.interleaved) qkv_norm_rope_kernel<4, true><<<grid, RP_THREADS, smem, st>>>(a, p);
    else if (vec) qkv_norm_rope_kernel<4, false><<<grid, RP_THREADS, smem, st>>>(a, p);
    else if (a.interleaved) qkv_norm_rope_kernel<1, true><<<grid, RP_THREADS, smem, st>>>(a, p);
    else qkv_norm_rope_kernel<1, false><<<grid, RP_THREADS, smem, st>>>(a, p);
    return (int)cudaGetLastError();
}

size_t qkv_norm_rope_bwd_bytes(int sm_count)
{
    return (size_t)sm_count * RP_BWD_CTAS * RP_BWD_SETS * 2 * 256 * sizeof(float);
}

int launch_qkv_norm_rope_bwd(const RopeArgs &a, float *dgq, float *dgk, int sm_count, cudaStream_t st, int *launches)
{
    const bool vec = rope_vec(a);
    const RopePlan p = rope_plan(a, vec, sm_count, true);
    const int grid = p.blocks;
    const size_t smem = rope_smem(a, p, true);
    if (vec && a.interleaved) qkv_norm_rope_bwd_kernel<4, true><<<grid, RP_THREADS, smem, st>>>(a, p);
    else if (vec) qkv_norm_rope_bwd_kernel<4, false><<<grid, RP_THREADS, smem, st>>>(a, p);
    else if (a.interleaved) qkv_norm_rope_bwd_kernel<1, true><<<grid, RP_THREADS, smem, st>>>(a, p);
    else qkv_norm_rope_bwd_kernel<1, false><<<grid, RP_THREADS, smem, st>>>(a, p);
    *launches = 1;
    int e = (int)cudaGetLastError();
    if (e || !a.partial) return e;
    rope_dgamma_kernel<<<((dgq == dgk ? 1 : 2) * a.dk + 7) / 8, 512, 0, st>>>(a.partial, grid, a.dk, dgq, dgk);
    *launches = 2;
    return (int)cudaGetLastError();
}

}  // namespace axb
