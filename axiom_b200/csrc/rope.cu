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
// A CTA takes a few tokens.  Their angles are formed once, for all heads: p * f in turns in 64 bits (a position of
// 10^6 times a frequency of 1 has lost five of fp32's seven digits), the whole turns dropped, and the remainder's sine
// and cosine in fp32.  A group of lanes owns a head row; a lane owns two 16-byte pieces of it that hold both partners of
// its pairs (piece c and c + pairs/4 of the half-split layout; the interleaved pairs lie inside a piece), so the rotation
// needs no exchange and the norm one shuffle tree.  Head dims and rotated parts that do not cut into 16-byte pieces,
// and unaligned tensors, take the same kernel with single floats in the place of the pieces.
#include "rope.cuh"

#include <math.h>

namespace axb {

static constexpr int RP_THREADS = 256;
static constexpr double RP_INV_2PI = 0.15915494309189533577;

// which pieces (VEC floats each) of a head row unit u of a lane covers, and whether they form rotated pairs
template <int VEC>
struct RopeUnit {
    int v0, v1;      // piece indices, -1: none
    int p0, p1;      // first pair of the rotation of piece 0 (half split: of both pieces; -1: not rotated)
    bool half;
};

template <int VEC, bool INTER>
__device__ __forceinline__ RopeUnit<VEC> rope_unit(int u, int dk, int pairs)
{
    const int nv = dk / VEC;
    RopeUnit<VEC> r;
    r.half = false;
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
        r.half = true;
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

template <int VEC>
__device__ __forceinline__ Piece<VEC> load_piece(const float *row, int v)
{
    Piece<VEC> p;
    if (v < 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p.x[i] = 0.f;
    } else if (VEC == 4) {
        const float4 t = *reinterpret_cast<const float4 *>(row + 4 * v);
        p.x[0] = t.x; p.x[1 % VEC] = t.y; p.x[2 % VEC] = t.z; p.x[3 % VEC] = t.w;
    } else {
        p.x[0] = row[v];
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

// rotates a lane's two pieces by the angles whose cosines and sines (times the amplitude) lie at cs, sn; BACK turns the
// other way (the transpose)
template <int VEC, bool BACK>
__device__ __forceinline__ void rotate_unit(const RopeUnit<VEC> &u, const float *cs, const float *sn, Piece<VEC> &a, Piece<VEC> &b)
{
    if (u.half) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float c = cs[u.p0 + i], s = BACK ? -sn[u.p0 + i] : sn[u.p0 + i];
            const float x = a.x[i], y = b.x[i];
            a.x[i] = x * c - y * s;
            b.x[i] = y * c + x * s;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i + 1 < VEC; i += 2) {
        if (u.p0 >= 0) {
            const float c = cs[u.p0 + i / 2], s = BACK ? -sn[u.p0 + i / 2] : sn[u.p0 + i / 2];
            const float x = a.x[i], y = a.x[(i + 1) % VEC];
            a.x[i] = x * c - y * s;
            a.x[(i + 1) % VEC] = y * c + x * s;
        }
        if (u.p1 >= 0) {
            const float c = cs[u.p1 + i / 2], s = BACK ? -sn[u.p1 + i / 2] : sn[u.p1 + i / 2];
            const float x = b.x[i], y = b.x[(i + 1) % VEC];
            b.x[i] = x * c - y * s;
            b.x[(i + 1) % VEC] = y * c + x * s;
        }
    }
}

__device__ __forceinline__ float lanes_sum(float v, int width)
{
    for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct RopePlan {
    int lpr;        // lanes per head row (power of two)
    int tok_cta;    // tokens a CTA takes at a time
    int heads_cta;  // head rows (of H + 2*Hkv) of a token that one CTA takes
};

// Places and angles of a CTA's tokens, in shared memory.  q_row / kv_row: the row index of head 0 (-1: not written).
struct RopeTokens {
    float *cs, *sn;            // [tok_cta][pairs]
    int64_t *q_row, *kv_row;   // [tok_cta]
};

__device__ __forceinline__ RopeTokens rope_tokens(void *smem, const RopePlan &p, int pairs)
{
    RopeTokens t;
    t.q_row = reinterpret_cast<int64_t *>(smem);
    t.kv_row = t.q_row + p.tok_cta;
    t.cs = reinterpret_cast<float *>(t.kv_row + p.tok_cta);
    t.sn = t.cs + (size_t)p.tok_cta * pairs;
    return t;
}

__device__ __forceinline__ void rope_place(const RopeArgs &a, const RopeTokens &t, int64_t tok0, int ntok, int64_t seq_rows)
{
    for (int i = threadIdx.x; i < ntok; i += RP_THREADS) {
        const int64_t tok = tok0 + i;
        const int b = (int)(tok / a.T), s = (int)(tok - (int64_t)b * a.T);
        int64_t first = 0;
        bool valid = true;
        if (a.lens) {
            const int len = a.lens[b], n = a.n_new ? a.n_new[b] : a.T;
            // a sequence that does not fit its rows is refused whole: nothing of it is read or written
            const bool bad = len < 0 || n < 0 || n > a.T || (int64_t)len + n > a.kv_rows;
            if (bad && a.err) atomicCAS(a.err, 0, (int)AXB_DEVERR_ROWS);
            valid = !bad && s < n;
            first = len;
        }
        t.q_row[i] = valid ? (int64_t)b * a.H * a.T + s : -1;
        t.kv_row[i] = valid ? (int64_t)b * a.Hkv * seq_rows + first + s : -1;
    }
    for (int i = threadIdx.x; i < ntok * a.pairs; i += RP_THREADS) {
        const int k = i / a.pairs;
        const int64_t tok = tok0 + k;
        const int b = (int)(tok / a.T);
        const int p = a.pos ? a.pos[tok] : (int)(tok - (int64_t)b * a.T) + (a.lens ? a.lens[b] : 0);
        const double turns = (double)p * (a.freq[i - k * a.pairs] * RP_INV_2PI);
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        t.cs[i] = c * a.amplitude;
        t.sn[i] = s * a.amplitude;
    }
}

template <int VEC, bool INTER>
__global__ void __launch_bounds__(RP_THREADS) qkv_norm_rope_kernel(const RopeArgs a, const RopePlan p)
{
    constexpr int NU = VEC == 4 ? 1 : 4;   // units a lane covers: 32 lanes hold 256 floats either way
    extern __shared__ double smem[];
    const RopeTokens tk = rope_tokens(smem, p, a.pairs);
    const int64_t tokens = (int64_t)a.B * a.T, tok0 = (int64_t)blockIdx.x * p.tok_cta;
    const int ntok = (int)(tokens - tok0 < p.tok_cta ? tokens - tok0 : p.tok_cta);
    rope_place(a, tk, tok0, ntok, a.kv_rows);
    __syncthreads();

    const int heads = a.H + 2 * a.Hkv, h0 = blockIdx.y * p.heads_cta;
    const int nh = heads - h0 < p.heads_cta ? heads - h0 : p.heads_cta;
    const int lane = threadIdx.x & 31, li = lane & (p.lpr - 1), rpw = 32 / p.lpr;
    const int step = (RP_THREADS / 32) * rpw, rows = ntok * nh;
    RopeUnit<VEC> u[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) u[j] = rope_unit<VEC, INTER>(li + 32 * j, a.dk, a.pairs);
    const float inv_dk = 1.0f / (float)a.dk;

    // (warp-uniform bounds: the norm's shuffles need every lane)
    for (int w0 = (threadIdx.x >> 5) * rpw; w0 < rows; w0 += step) {
        const int r = w0 + lane / p.lpr;
        const int t = r < rows ? r / nh : 0, h = h0 + (r < rows ? r - t * nh : 0);
        const int64_t qr = tk.q_row[t];
        const bool on = r < rows && qr >= 0;
        const float *src = a.qkv + ((tok0 + t) * heads + h) * a.dk;
        Piece<VEC> x0[NU], x1[NU];
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            x0[j] = load_piece<VEC>(src, on ? u[j].v0 : -1);
            x1[j] = load_piece<VEC>(src, on ? u[j].v1 : -1);
        }
        if (a.bias) {
            const float *bias = a.bias + (int64_t)h * a.dk;
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                const Piece<VEC> b0 = load_piece<VEC>(bias, u[j].v0), b1 = load_piece<VEC>(bias, u[j].v1);
#pragma unroll
                for (int i = 0; i < VEC; ++i) { x0[j].x[i] += b0.x[i]; x1[j].x[i] += b1.x[i]; }
            }
        }
        const float *g = h < a.H ? a.gq : h < a.H + a.Hkv ? a.gk : nullptr;
        if (a.gq || a.gk) {
#pragma unroll
            for (int j = 0; j < NU; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) ss += x0[j].x[i] * x0[j].x[i] + x1[j].x[i] * x1[j].x[i];
            ss = lanes_sum(ss, p.lpr);
        }
        if (g) {
            const float rs = rsqrtf(ss * inv_dk + a.eps);
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                const Piece<VEC> g0 = load_piece<VEC>(g, u[j].v0), g1 = load_piece<VEC>(g, u[j].v1);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    x0[j].x[i] = x0[j].x[i] * rs * g0.x[i];
                    x1[j].x[i] = x1[j].x[i] * rs * g1.x[i];
                }
            }
        }
        if (!on) continue;   // (no shuffle follows; lanes without a row meet the loop's bound with the others)
        if (h < a.H + a.Hkv) {
#pragma unroll
            for (int j = 0; j < NU; ++j) rotate_unit<VEC, false>(u[j], tk.cs + t * a.pairs, tk.sn + t * a.pairs, x0[j], x1[j]);
        }
        float *dst = h < a.H               ? a.q + (qr + (int64_t)h * a.T) * a.dk
                     : h < a.H + a.Hkv     ? a.k + (tk.kv_row[t] + (int64_t)(h - a.H) * a.kv_rows) * a.dk
                                           : a.v + (tk.kv_row[t] + (int64_t)(h - a.H - a.Hkv) * a.kv_rows) * a.dk;
#pragma unroll
        for (int j = 0; j < NU; ++j) {
            store_piece<VEC>(dst, u[j].v0, x0[j]);
            store_piece<VEC>(dst, u[j].v1, x1[j]);
        }
    }
}

// The gradient: the same ownership the other way, persistent CTAs.  A lane meets the same head elements in every row, so
// the norm weights' gradients collect in its registers; groups are added in shared memory, CTAs by rope_dgamma_kernel,
// each in a fixed order.
template <int VEC, bool INTER>
__global__ void __launch_bounds__(RP_THREADS) qkv_norm_rope_bwd_kernel(const RopeArgs a, const RopePlan p)
{
    constexpr int NU = VEC == 4 ? 1 : 4;
    extern __shared__ double smem[];
    const RopeTokens tk = rope_tokens(smem, p, a.pairs);
    const int64_t tokens = (int64_t)a.B * a.T, blocks = (tokens + p.tok_cta - 1) / p.tok_cta;
    const int nh = a.H + 2 * a.Hkv;
    const int lane = threadIdx.x & 31, li = lane & (p.lpr - 1), rpw = 32 / p.lpr, step = (RP_THREADS / 32) * rpw;
    RopeUnit<VEC> u[NU];
#pragma unroll
    for (int j = 0; j < NU; ++j) u[j] = rope_unit<VEC, INTER>(li + 32 * j, a.dk, a.pairs);
    const float inv_dk = 1.0f / (float)a.dk;
    float acc[2][2][NU][VEC];   // [q, k][piece][unit]
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < NU; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[w][e][j][i] = 0.f;

    for (int64_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
        const int64_t tok0 = blk * p.tok_cta;
        const int ntok = (int)(tokens - tok0 < p.tok_cta ? tokens - tok0 : p.tok_cta), rows = ntok * nh;
        __syncthreads();   // the previous block's angles are still being read
        rope_place(a, tk, tok0, ntok, a.T);
        __syncthreads();
        for (int w0 = (threadIdx.x >> 5) * rpw; w0 < rows; w0 += step) {
            const int r = w0 + lane / p.lpr;
            const bool on = r < rows;
            const int t = on ? r / nh : 0, h = on ? r - t * nh : 0;
            const float *src = h < a.H           ? a.q + (tk.q_row[t] + (int64_t)h * a.T) * a.dk
                               : h < a.H + a.Hkv ? a.k + (tk.kv_row[t] + (int64_t)(h - a.H) * a.T) * a.dk
                                                 : a.v + (tk.kv_row[t] + (int64_t)(h - a.H - a.Hkv) * a.T) * a.dk;
            const int64_t at = ((tok0 + t) * nh + h) * a.dk;
            const float *g = h < a.H ? a.gq : h < a.H + a.Hkv ? a.gk : nullptr;
            Piece<VEC> d0[NU], d1[NU], x0[NU], x1[NU];
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                d0[j] = load_piece<VEC>(src, on ? u[j].v0 : -1);
                d1[j] = load_piece<VEC>(src, on ? u[j].v1 : -1);
                x0[j] = load_piece<VEC>(a.qkv + at, on && g ? u[j].v0 : -1);
                x1[j] = load_piece<VEC>(a.qkv + at, on && g ? u[j].v1 : -1);
            }
            if (h < a.H + a.Hkv) {
#pragma unroll
                for (int j = 0; j < NU; ++j) rotate_unit<VEC, true>(u[j], tk.cs + t * a.pairs, tk.sn + t * a.pairs, d0[j], d1[j]);
            }
            if (a.gq || a.gk) {
                if (g && a.bias) {
                    const float *bias = a.bias + (int64_t)h * a.dk;
#pragma unroll
                    for (int j = 0; j < NU; ++j) {
                        const Piece<VEC> b0 = load_piece<VEC>(bias, on ? u[j].v0 : -1), b1 = load_piece<VEC>(bias, on ? u[j].v1 : -1);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) { x0[j].x[i] += b0.x[i]; x1[j].x[i] += b1.x[i]; }
                    }
                }
                Piece<VEC> g0[NU], g1[NU];
                float ss = 0.f, sd = 0.f;   // sum x^2, sum d*g*x
#pragma unroll
                for (int j = 0; j < NU; ++j) {
                    g0[j] = load_piece<VEC>(g, g ? u[j].v0 : -1);
                    g1[j] = load_piece<VEC>(g, g ? u[j].v1 : -1);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        ss += x0[j].x[i] * x0[j].x[i] + x1[j].x[i] * x1[j].x[i];
                        sd += d0[j].x[i] * g0[j].x[i] * x0[j].x[i] + d1[j].x[i] * g1[j].x[i] * x1[j].x[i];
                    }
                }
                ss = lanes_sum(ss, p.lpr);
                sd = lanes_sum(sd, p.lpr);
                if (g) {
                    const float rs = rsqrtf(ss * inv_dk + a.eps), mean = sd * rs * inv_dk;   // mean(d*g*u)
                    const bool is_q = h < a.H;
#pragma unroll
                    for (int j = 0; j < NU; ++j)
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            const float u0 = x0[j].x[i] * rs, u1 = x1[j].x[i] * rs;
                            const float e0 = d0[j].x[i] * u0, e1 = d1[j].x[i] * u1;
                            acc[0][0][j][i] += is_q ? e0 : 0.f;
                            acc[0][1][j][i] += is_q ? e1 : 0.f;
                            acc[1][0][j][i] += is_q ? 0.f : e0;
                            acc[1][1][j][i] += is_q ? 0.f : e1;
                            d0[j].x[i] = rs * (d0[j].x[i] * g0[j].x[i] - u0 * mean);
                            d1[j].x[i] = rs * (d1[j].x[i] * g1[j].x[i] - u1 * mean);
                        }
                }
            }
            if (!on) continue;
#pragma unroll
            for (int j = 0; j < NU; ++j) {
                store_piece<VEC>(a.dqkv + at, u[j].v0, d0[j]);
                store_piece<VEC>(a.dqkv + at, u[j].v1, d1[j]);
            }
        }
    }
    if (!a.partial) return;
    // [group][dk] per norm weight, then one thread per element adds the groups in order
    float *red = reinterpret_cast<float *>(smem);
    const int groups = RP_THREADS / p.lpr, group = threadIdx.x / p.lpr;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NU; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (u[j].v0 >= 0) red[group * a.dk + u[j].v0 * VEC + i] = acc[w][0][j][i];
                if (u[j].v1 >= 0) red[group * a.dk + u[j].v1 * VEC + i] = acc[w][1][j][i];
            }
        __syncthreads();
        if (threadIdx.x < a.dk) {
            float s = 0.f;
            for (int k = 0; k < groups; ++k) s += red[k * a.dk + threadIdx.x];
            a.partial[((int64_t)blockIdx.x * 2 + w) * a.dk + threadIdx.x] = s;
        }
    }
}

// dg[w][d] += sum over blocks of partial[block][w][d], in 64 bits and in block order within each of 32 strands
__global__ void __launch_bounds__(1024) rope_dgamma_kernel(const float *partial, int blocks, int dk, float *dgq, float *dgk)
{
    __shared__ double red[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), strand = threadIdx.x >> 5;
    double s = 0.0;
    if (c < 2 * dk)
        for (int b = strand; b < blocks; b += 32) s += (double)partial[(int64_t)b * 2 * dk + c];
    red[strand][threadIdx.x & 31] = s;
    __syncthreads();
    if (strand == 0 && c < 2 * dk) {
        for (int k = 1; k < 32; ++k) s += red[k][threadIdx.x];
        float *dst = c < dk ? dgq : dgk;
        const int d = c < dk ? c : c - dk;
        if (dst) dst[d] = (float)((double)dst[d] + s);
    }
}

// ---------------------------------------------------------------------- host

static bool rope_vec(const RopeArgs &a, const float *dgq, const float *dgk)
{
    uintptr_t m = 0;
    for (const void *p : { (const void *)a.qkv, (const void *)a.bias, (const void *)a.gq, (const void *)a.gk, (const void *)a.q,
                           (const void *)a.k, (const void *)a.v, (const void *)a.dqkv, (const void *)dgq, (const void *)dgk })
        m |= reinterpret_cast<uintptr_t>(p);
    // whole 16-byte pieces on either side of every pair: half split 2*pairs floats cut in two, interleaved two pairs a piece
    return (m & 15) == 0 && a.dk % 4 == 0 && a.pairs % (a.interleaved ? 2 : 4) == 0;
}

static RopePlan rope_plan(const RopeArgs &a, bool vec, int sm_count, bool backward)
{
    RopePlan p;
    const int heads = a.H + 2 * a.Hkv;
    p.lpr = 32;
    if (vec) {
        const int units = a.interleaved ? (a.dk / 4 + 1) / 2 : a.pairs / 4 + (a.dk / 4 - a.pairs / 2 + 1) / 2;
        p.lpr = 1;
        while (p.lpr < units) p.lpr <<= 1;
    }
    const int groups = RP_THREADS / p.lpr;
    const int64_t tokens = (int64_t)a.B * a.T;
    // Tokens per CTA: eight rows a group at least (the angles and the tokens' places cost a barrier), while every SM keeps
    // eight CTAs' worth of rows.
    p.tok_cta = 1;
    while (p.tok_cta < 16 && p.tok_cta * heads < 8 * groups && tokens >= (int64_t)2 * p.tok_cta * 8 * sm_count) p.tok_cta *= 2;
    p.heads_cta = heads;
    if (!backward) {
        // few tokens: the heads of a token are dealt out too, down to one row a group
        while (p.heads_cta > groups && (tokens + p.tok_cta - 1) / p.tok_cta * ((heads + p.heads_cta - 1) / p.heads_cta) < 4 * sm_count)
            p.heads_cta = (p.heads_cta + 1) / 2;
    }
    return p;
}

static size_t rope_smem(const RopeArgs &a, const RopePlan &p, bool backward)
{
    size_t n = (size_t)p.tok_cta * (2 * sizeof(int64_t) + 2 * (size_t)a.pairs * sizeof(float));
    const size_t red = backward ? (size_t)(RP_THREADS / p.lpr) * a.dk * sizeof(float) : 0;
    return n > red ? n : red;   // at most 33 KB (16 tokens of 128 pairs)
}

int launch_qkv_norm_rope(const RopeArgs &a, int sm_count, cudaStream_t st)
{
    const bool vec = rope_vec(a, nullptr, nullptr);
    const RopePlan p = rope_plan(a, vec, sm_count, false);
    const int64_t blocks = ((int64_t)a.B * a.T + p.tok_cta - 1) / p.tok_cta;
    const dim3 grid((unsigned)blocks, (unsigned)((a.H + 2 * a.Hkv + p.heads_cta - 1) / p.heads_cta));
    const size_t smem = rope_smem(a, p, false);
    if (vec && a.interleaved) qkv_norm_rope_kernel<4, true><<<grid, RP_THREADS, smem, st>>>(a, p);
    else if (vec) qkv_norm_rope_kernel<4, false><<<grid, RP_THREADS, smem, st>>>(a, p);
    else if (a.interleaved) qkv_norm_rope_kernel<1, true><<<grid, RP_THREADS, smem, st>>>(a, p);
    else qkv_norm_rope_kernel<1, false><<<grid, RP_THREADS, smem, st>>>(a, p);
    return (int)cudaGetLastError();
}

static int bwd_blocks(const RopeArgs &a, const RopePlan &p, int sm_count)
{
    const int64_t blocks = ((int64_t)a.B * a.T + p.tok_cta - 1) / p.tok_cta;
    const int64_t most = (int64_t)sm_count * 4;
    return (int)(blocks < most ? blocks : most);
}

int qkv_norm_rope_bwd_blocks(const RopeArgs &a, int sm_count)
{
    return bwd_blocks(a, rope_plan(a, rope_vec(a, nullptr, nullptr), sm_count, true), sm_count);
}

int launch_qkv_norm_rope_bwd(const RopeArgs &a, float *dgq, float *dgk, int sm_count, cudaStream_t st, int *launches)
{
    const bool vec = rope_vec(a, nullptr, nullptr);
    const RopePlan p = rope_plan(a, vec, sm_count, true);
    const int grid = bwd_blocks(a, p, sm_count);
    const size_t smem = rope_smem(a, p, true);
    if (vec && a.interleaved) qkv_norm_rope_bwd_kernel<4, true><<<grid, RP_THREADS, smem, st>>>(a, p);
    else if (vec) qkv_norm_rope_bwd_kernel<4, false><<<grid, RP_THREADS, smem, st>>>(a, p);
    else if (a.interleaved) qkv_norm_rope_bwd_kernel<1, true><<<grid, RP_THREADS, smem, st>>>(a, p);
    else qkv_norm_rope_bwd_kernel<1, false><<<grid, RP_THREADS, smem, st>>>(a, p);
    *launches = 1;
    int e = (int)cudaGetLastError();
    if (e || !a.partial) return e;
    rope_dgamma_kernel<<<(2 * a.dk + 31) / 32, 1024, 0, st>>>(a.partial, grid, a.dk, dgq, dgk);
    *launches = 2;
    return (int)cudaGetLastError();
}

}  // namespace axb
