// The few CUDA names that kv_tree_line.cuh uses, for a compiler of the host: one thread stands for a block.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>

#define __device__
#define __forceinline__ inline
using std::max;
using std::min;

typedef struct CUstream_st *cudaStream_t;
struct Dim3 {
    unsigned x = 0, y = 0, z = 0;
};
static Dim3 threadIdx, blockIdx, gridDim, blockDim;

template <typename T>
static T __ldg(const T *p) { return *p; }
static int atomicAdd(int *p, int v) { const int old = *p; *p += v; return old; }
static int atomicCAS(int *p, int cmp, int v) { const int old = *p; if (old == cmp) *p = v; return old; }
static float __uint_as_float(unsigned u) { float x; std::memcpy(&x, &u, 4); return x; }
static unsigned __float_as_uint(float x) { unsigned u; std::memcpy(&u, &x, 4); return u; }
// the search of tree_start, a whole warp's work: never called here
template <typename T>
static T __reduce_add_sync(unsigned, T v) { return v; }
template <typename T>
static T __shfl_up_sync(unsigned, T v, int) { return v; }
template <typename T>
static T __shfl_sync(unsigned, T v, int) { return v; }
static unsigned __ballot_sync(unsigned, bool v) { return v; }
static int __ffs(unsigned v) { return __builtin_ffs((int)v); }
static void __syncthreads() {}
static void __syncwarp() {}
