// Host launchers of the decode-step kernels: the paged key/value cache (paged_cache.cu), attention of one new token per
// sequence over it (paged_attention.cu), and products of few rows with a 4-bit weight (weight_only.cu).
#pragma once
#include <cuda_runtime.h>

#include "../../include/sharq_b200.h"

namespace sharq {

constexpr int kBadCacheIndex = 0x402;  // error code: a position, length, sequence or page outside the cache or its tables

constexpr int kAttentionTimeout = 0x403;  // error code: a wait for a copy ran out
constexpr int kWeightOnlyTimeout = 0x404;

// A position of a sequence in the cache; also what the kernels check before every access.
struct PagedCache {
  char *k, *v;
  const int *page_table;
  long long table_stride, page_stride, head_stride, token_stride;  // strides of the cache in bytes
  const float *k_scale, *v_scale;
  int seqs, max_pages, pages, page_size, kv_heads, head_dim;
};

// Tokens that a row of the page table can hold, within an int, and so far from its end that the tokens of a few tiles beyond are too.
__host__ __device__ inline int paged_capacity(const PagedCache &c) {
  const long long n = (long long)c.max_pages * c.page_size;
  return n > 0x7fff0000LL ? 0x7fff0000 : (int)n;
}

cudaError_t run_rope_append_paged(const void *qkv, long long row_stride, int rows, int heads, const void *cos_t, const void *sin_t,
                                  int table_rows, const int *positions, const int *sequences, const PagedCache &cache, bool fp8,
                                  void *q_out, void *k_out, int *error_flag, cudaStream_t stream);

// One query row per sequence of the cache's page table (cache.head_dim 64 or 128, heads a multiple of cache.kv_heads).
size_t paged_attention_workspace_bytes(int heads, const PagedCache &cache, bool fp8);
cudaError_t run_paged_attention(const void *q, long long q_row, long long q_head, int heads, const PagedCache &cache, bool fp8,
                                const int *lengths, float scale, void *out, void *workspace, int *error_flag, cudaStream_t stream);

// y[m, n] = bf16(scale * x . W^T + bias), m rows (1..16) of bf16 against a 4-bit weight with dense scale factors, k % 64 == 0.
constexpr int kWeightOnlyMaxRows = 16;
cudaError_t run_weight_only(const void *x, long long x_row, int m, int n, int k, const void *qw, const void *sf, const float *scale_dev,
                            float scale, const void *bias, void *y, int *error_flag, cudaStream_t stream);

// Leave for `bytes` of shared memory, asked for once per kernel and device (ready: a static array per kernel).
template <typename Kernel>
cudaError_t allow_smem(Kernel kernel, int bytes, bool (&ready)[64]) {
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess || (dev >= 0 && dev < 64 && ready[dev])) return err;
  err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == cudaSuccess && dev >= 0 && dev < 64) ready[dev] = true;
  return err;
}

}  // namespace sharq
