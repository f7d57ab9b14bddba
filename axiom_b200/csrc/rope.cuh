// rope.cuh — launchers of the pass between a projection and the attention (rope.cu): head layout, bias, per-head RMS
// norm, position rotation; forward, into the rows of a KV cache, and backward.  dk <= 256.
#pragma once
#include "../../include/axiom_b200.h"

#include <cuda_runtime.h>
#include <stdint.h>

namespace axb {

struct RopeArgs {
    const float *qkv;            // [B*T, (H + 2*Hkv)*dk]
    const float *bias;           // [(H + 2*Hkv)*dk] or nullptr
    const float *gq, *gk;        // [dk] norm weights or nullptr (no norm)
    const double *freq;          // [pairs] radians per position
    const int32_t *pos;          // [B*T] or nullptr: lens[b] + t, or t without lens
    const int32_t *lens, *n_new; // cache form only: [B]; n_new nullptr = T for every sequence
    float *q, *k, *v;            // head-major [B*H, T, dk], [B*Hkv, kv_rows, dk] twice (read by the backward)
    float *dqkv;                 // backward: the gradient of qkv
    float *partial;              // backward, qkv_norm_rope_bwd_bytes(): [grid][2*dk] partial sums of the norm weights' gradients
    int64_t kv_rows;             // T, or the rows of a cache
    int *err;                    // the words of device_error.cuh
    float eps, amplitude;
    int B, T, H, Hkv, dk, pairs, interleaved;
};

int launch_qkv_norm_rope(const RopeArgs &a, int sm_count, cudaStream_t st);
// the most that the backward's partial sums take, whatever the shape
size_t qkv_norm_rope_bwd_bytes(int sm_count);
// dgq / dgk [dk] are added to (nullptr: not wanted; the same buffer twice: it receives both); *launches receives the number of kernels enqueued
int launch_qkv_norm_rope_bwd(const RopeArgs &a, float *dgq, float *dgk, int sm_count, cudaStream_t st, int *launches);

}  // namespace axb
