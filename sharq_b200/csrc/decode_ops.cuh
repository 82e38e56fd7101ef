// Host launchers of the decode-step kernels: the paged key/value cache (paged_cache.cu), attention of one new token per
// sequence over it (paged_attention.cu), products of few rows with a 4-bit weight (weight_only.cu), pages and places of a step's tokens
// (step_plan.cu), penalties, biases and masks on logits (logit_rules.cu), and attention of ragged prompts (prompt_attention.cu).
#pragma once
#include <cuda_runtime.h>

#include "../../include/sharq_b200.h"

namespace sharq {

constexpr int kBadCacheIndex = 0x402;  // error code: a position, length, sequence or page outside the cache or its tables

constexpr int kAttentionTimeout = 0x403;  // error code: a wait for a copy ran out
constexpr int kWeightOnlyTimeout = 0x404;
constexpr int kBadStepPlan = 0x405;     // error code: a length, count or number of free pages that the cache cannot have
constexpr int kBadLogitRules = 0x406;   // error code: a token, length or offset outside its range
constexpr int kBadOffsets = 0x407;      // error code: offsets of prompts that go back, or beyond the rows
constexpr int kPromptTimeout = 0x408;   // error code: a wait inside the attention of prompts ran out
constexpr int kPagesShort = 0x409;      // error code: pages that did not suffice for a step's tokens

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
// window: tokens that are seen from the last one back, with the first `sinks`; 0: all.
size_t paged_attention_workspace_bytes(int heads, const PagedCache &cache, bool fp8, int window, int sinks);
cudaError_t run_paged_attention(const void *q, long long q_row, long long q_head, int heads, const PagedCache &cache, bool fp8,
                                const int *lengths, float scale, int window, int sinks, void *out, void *workspace, int *error_flag,
                                cudaStream_t stream);

// y[m, n] = bf16(scale * x . W^T + bias), m rows (1..16) of bf16 against a 4-bit weight with dense scale factors, k % 64 == 0.
constexpr int kWeightOnlyMaxRows = 16;
cudaError_t run_weight_only(const void *x, long long x_row, int m, int n, int k, const void *qw, const void *sf, const float *scale_dev,
                            float scale, const void *bias, void *y, int *error_flag, cudaStream_t stream);

// Pages and places of a step's tokens (step_plan.cu); the fields as sharq_plan_paged_step has them.
struct StepPlan {
  int *table;
  long long table_stride;
  int sequences, max_pages, page_size, max_tokens;
  int *lengths;
  const int *counts;
  const unsigned char *released;
  int *stack;
  int stack_size;
  int *free_count;
  int rows;
  int *offsets, *positions, *row_sequences;
  int *error_flag;
  bool strict;  // pages that do not suffice are an error
};
cudaError_t run_step_plan(const StepPlan &plan, cudaStream_t stream);

// Penalties, biases and masks on logits (logit_rules.cu); the fields as sharq_logit_rules has them.
struct LogitRules {
  const void *logits;
  void *out;
  long long logits_stride, out_stride;
  int rows, vocab;
  const void *tokens;
  long long tokens_stride;
  int width;
  const int *lengths, *prompt_lengths;
  const float *repetition, *presence, *frequency;
  const int *bias_offsets, *bias_ids;
  const float *bias_values;
  int biases;
  const unsigned *mask;
  long long mask_stride;
  int *error_flag;
  int slice;  // tokens of a CTA, the launcher's choice
};
cudaError_t run_logit_rules(const LogitRules &rules, bool bf16, bool wide_ids, cudaStream_t stream);

// Attention of ragged prompts (prompt_attention.cu); the fields as sharq_prompt_attention has them, strides in elements.
struct PromptAttention {
  const void *q, *k, *v;
  long long q_row, q_head, k_row, k_head, v_row, v_head;
  int rows, k_rows, heads, kv_heads, head_dim;
  const int *offsets, *k_offsets;
  int seqs, window, sinks;
  float scale;
  void *out;
  bool fill;
  void *workspace;
  int *error_flag;
};
size_t prompt_attention_workspace_bytes(const PromptAttention &p);  // from the sizes alone
cudaError_t run_prompt_attention(const PromptAttention &p, cudaStream_t stream);
// Clock cycles that a wait inside it may take, of launches from now on; 0: the default, which no other setting exceeds.
void set_prompt_attention_wait_limit(long long cycles);

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
