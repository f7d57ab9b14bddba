// kv_tree.cuh — launchers of the ragged-batch KV-cache kernels (kv_tree.cu, kv_tree_tc.cu): attention of T new tokens of every sequence
// over its cached rows and over one another (a chain or a drafted tree), and the move of accepted rows.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace axb {

// what the kernel that adds up an item's pieces has to know of it; it stands at the CTA that holds the item's first key tile
struct KvTreeShared {
    int pieces, b, hk, block, n, rows;   // pieces 0: none; n, rows: the sequence's new tokens and query rows of a key head
};

struct KvTreeArgs {
    const float *K, *V;          // [B*Hkv, max_seq, dk]
    const float *Q;              // [B*H, T, dk]
    const uint64_t *mask;        // [B or 1][T][words] bit j of token t: t attends to new token j; nullptr: j <= t
    const int32_t *lens, *n_new; // [B]; n_new nullptr: T for every sequence
    float *out;                  // [B*H, T, dk]
    int *counters;               // one per SM, zero on entry and on exit, of a launch that gave up too (the warp-level kernel's)
    KvTreeShared *shared;        // kv_tree_workspace_bytes(): one per SM, then
    float *slots;                // partial results, two slots per SM
    int64_t max_seq, mask_stride;
    int *err;                    // the words of device_error.cuh
    float c_log2;                // scale * log2(e)
    int B, H, Hkv, T, dk, words;
};

constexpr size_t KT_SHARED_BYTES = 256 * sizeof(KvTreeShared);   // (whole lines: the slots behind it begin one)
constexpr size_t KT_SLOT_BYTES = 128 * (128 + 2) * sizeof(float);   // the largest variant's partial result
size_t kv_tree_workspace_bytes(int sm_count);
// query rows of a key head up to which the warp-level kernel is at least as fast as the tensor-memory one (kv_tree_tc.cu), which
// costs the same for one row or 64.  8 sequences, 8 key heads, 41000 cached rows, warp-level against tensor memory: 16 rows of
// 128 75 / 120 us, 24 rows 141 / 119, 32 rows of 96 107 / 96, of 64 82 / 82, of 32 53 / 69.
constexpr int kt_warp_rows(int dk) { return dk > 64 ? 16 : 32; }
// *launches receives the number of kernels enqueued
int launch_kv_tree_tc(const KvTreeArgs &a, int sm_count, cudaStream_t st, int *launches);
int launch_kv_cache_attend_tree(const KvTreeArgs &a, int sm_count, cudaStream_t st, int *launches);

// rows lens[b] + keep[b][i] -> lens[b] + i for i < n_keep[b] in both caches; lens_out[b] = lens[b] + n_keep[b] (or nullptr)
int launch_kv_cache_compact(float *K, float *V, const int32_t *keep, const int32_t *n_keep, const int32_t *lens, int32_t *lens_out,
                            int64_t B, int64_t Hkv, int64_t T, int64_t max_seq, int64_t dk, int *err, cudaStream_t st);

}  // namespace axb
