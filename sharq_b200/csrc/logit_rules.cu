// Penalties for repeated tokens, biases and masks on logits, in one launch.  256 rows of 152064 with histories of up to 6000 tokens: 137 us, 2.3 TB/s; one
// row of 128256: 6.0 us.
//
//   x' = x > 0 ? x / r : x r   (tokens of the history),   x' - f n - p [n > 0]   (n: how often the answer so far has the token),   + biases,   -inf where masked
//
// Bound by reading and writing the logits once.  What touches a logit is known by token, not by place, so a CTA takes a slice of a row, counts the
// history's tokens that fall into it in a table in shared memory (whole numbers: the order of the atomics does not matter), and passes over its slice once.  A
// history is read by every CTA of its row, from L2, which is what a wider slice saves.
//
// A penalty or a bias may leave little of a logit, so what they touch is computed in double and rounded once; that is a token in hundreds.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "decode_ops.cuh"
#include "sm100_ptx.cuh"

namespace sharq {

namespace {

constexpr unsigned kSeen = 1u << 31, kBiased = 1u << 30, kTwice = 1u << 29, kCount = kTwice - 1;  // of a token's word; the rest counts

__device__ __forceinline__ float minus_inf() { return __int_as_float(0xff800000); }

struct Penalty {
  double repetition, presence, frequency;
};
__device__ __forceinline__ double penalised(double x, unsigned word, const Penalty &p) {
  const unsigned n = word & kCount;
  if (n != 0 || (word & kSeen) != 0) x = x > 0 ? x / p.repetition : x * p.repetition;
  if (n != 0) x = x - p.frequency * n - p.presence;
  return x;
}

template <typename T>
__device__ __forceinline__ T rounded(double x) {
  if constexpr (std::is_same<T, float>::value)
    return (float)x;
  else
    return __double2bfloat16(x);
}
template <typename T>
__device__ __forceinline__ double widened(T x) {
  if constexpr (std::is_same<T, float>::value)
    return (double)x;
  else
    return (double)__bfloat162float(x);
}

// T: type of the logits; Id: of the history's tokens; kVec: logits of a 16-byte access, or 1
template <typename T, typename Id, int kVec>
__global__ void __launch_bounds__(512) logit_rules_kernel(const __grid_constant__ LogitRules a) {
  extern __shared__ __align__(16) unsigned words[];
  const int row = blockIdx.y, tid = threadIdx.x, threads = blockDim.x;
  const int first = blockIdx.x * a.slice, size = min(a.slice, a.vocab - first);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  bool bad = false;
  int length = 0, prompt = 0;
  if (a.lengths != nullptr) {
    length = a.lengths[row];
    if (length < 0 || length > a.width) bad = true;
    length = min(max(length, 0), a.width);
    prompt = a.prompt_lengths == nullptr ? 0 : a.prompt_lengths[row];
  }
  int bias0 = 0, bias1 = 0;
  if (a.bias_offsets != nullptr) {
    bias0 = a.bias_offsets[row];
    bias1 = a.bias_offsets[row + 1];
    if (bias0 < 0 || bias1 < bias0 || bias1 > a.biases) bad = true, bias0 = bias1 = 0;
  }
  const Penalty penalty = {a.repetition == nullptr ? 1.0 : (double)a.repetition[row], a.presence == nullptr ? 0.0 : (double)a.presence[row],
                           a.frequency == nullptr ? 0.0 : (double)a.frequency[row]};
  const bool marked = length > 0 || bias1 > bias0;  // the table is in use
  if (marked) {
    for (int i = tid * 4; i < a.slice; i += threads * 4) *reinterpret_cast<uint4 *>(words + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
    const Id *tokens = static_cast<const Id *>(a.tokens) + row * a.tokens_stride;
#pragma unroll 4
    for (int j = tid; j < length; j += threads) {
      const Id id = tokens[j];
      const long long at = (long long)id - first;
      if (at >= 0 && at < size) {
        if (j < prompt)
          atomicOr(words + at, kSeen);
        else
          atomicAdd(words + at, 1u);
      } else if ((long long)id >= a.vocab) {
        bad = true;
      }
    }
    for (int j = bias0 + tid; j < bias1; j += threads) {
      const long long at = (long long)a.bias_ids[j] - first;
      if (at >= 0 && at < size) {
        if (atomicOr(words + at, kBiased) & kBiased) atomicOr(words + at, kTwice);
      } else if (at + first < 0 || at + first >= a.vocab) {
        bad = true;
      }
    }
    __syncthreads();
  }

  const T *in = static_cast<const T *>(a.logits) + row * a.logits_stride + first;
  T *out = static_cast<T *>(a.out) + row * a.out_stride + first;
  const unsigned *mask = a.mask == nullptr ? nullptr : a.mask + row * a.mask_stride + first / 32;
  const bool in_place = static_cast<const void *>(in) == static_cast<const void *>(out);
  struct __align__(kVec * sizeof(T)) Vec {
    T x[kVec];
  };
#pragma unroll 4
  for (int i = tid * kVec; i < size; i += threads * kVec) {
    const unsigned keep = mask == nullptr ? ~0u : mask[i >> 5] >> (i & 31);
    Vec v;
    if (kVec > 1 && i + kVec <= size)
      v = *reinterpret_cast<const Vec *>(in + i);
    else
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j < size) v.x[j] = in[i + j];
    unsigned any = 0, word[kVec];
    if (marked) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        word[j] = words[i + j];  // the table ends at a multiple of a vector
        any |= word[j];
      }
      if (any != 0) {
#pragma unroll
        for (int j = 0; j < kVec; ++j)
          if (word[j] != 0) v.x[j] = rounded<T>(penalised(widened<T>(v.x[j]), word[j], penalty));
      }
    }
    constexpr unsigned kAll = (1u << kVec) - 1;
    if ((keep & kAll) != kAll) {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if ((keep >> j & 1) == 0) v.x[j] = rounded<T>((double)minus_inf());
    } else if (in_place && any == 0) {
      continue;
    }
    if (kVec > 1 && i + kVec <= size && (any & kBiased) == 0)
      *reinterpret_cast<Vec *>(out + i) = v;
    else
#pragma unroll
      for (int j = 0; j < kVec; ++j)  // a biased one comes below, from the logit as it was
        if (i + j < size && !(marked && (word[j] & kBiased) != 0)) out[i + j] = v.x[j];
  }
  if (bias1 > bias0) {
    __syncthreads();
    for (int j = bias0 + tid; j < bias1; j += threads) {
      const long long at = (long long)a.bias_ids[j] - first;
      if (at < 0 || at >= size) continue;
      const unsigned word = atomicAnd(words + at, ~kBiased);
      if ((word & kBiased) == 0) continue;  // another thread has this token
      double x = penalised(widened<T>(in[at]), word & ~(kBiased | kTwice), penalty);
      if ((word & kTwice) == 0) {
        x += (double)a.bias_values[j];
      } else {  // a token with several biases: in the order of the list, whoever came first
        for (int k = bias0; k < bias1; ++k)
          if ((long long)a.bias_ids[k] - first == at) x += (double)a.bias_values[k];
      }
      const bool keeps = mask == nullptr || (mask[at >> 5] >> (at & 31) & 1) != 0;
      out[at] = keeps ? rounded<T>(x) : rounded<T>((double)minus_inf());
    }
  }
  if (bad && a.error_flag != nullptr) atomicCAS(a.error_flag, 0, kBadLogitRules);
}

template <typename T, typename Id, int kVec>
cudaError_t launch(LogitRules a, cudaStream_t stream) {
  int dev = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return err;
  // slices as wide as shared memory lets three CTAs share an SM, but two CTAs for every SM
  a.slice = 16384;
  while (a.slice > 1024 && (long long)a.rows * ((a.vocab + a.slice - 1) / a.slice) < 2 * sms) a.slice /= 2;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((a.vocab + a.slice - 1) / a.slice), (unsigned)a.rows);
  cfg.blockDim = dim3(a.slice >= 8192 ? 512 : 256);
  cfg.dynamicSmemBytes = (size_t)a.slice * sizeof(unsigned);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static bool ready[64] = {};
  err = allow_smem(logit_rules_kernel<T, Id, kVec>, 16384 * (int)sizeof(unsigned), ready);
  if (err != cudaSuccess) return err;
  return cudaLaunchKernelEx(&cfg, logit_rules_kernel<T, Id, kVec>, a);
}

}  // namespace

cudaError_t run_logit_rules(const LogitRules &a, bool bf16, bool wide_ids, cudaStream_t stream) {
  const int size = bf16 ? 2 : 4;
  const bool vec = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0 &&
                   (a.rows == 1 || (a.logits_stride * size % 16 == 0 && a.out_stride * size % 16 == 0));
#define SHARQ_RULES(BF16, WIDE, VEC, T, ID, N) \
  if (bf16 == BF16 && wide_ids == WIDE && vec == VEC) return launch<T, ID, N>(a, stream);
  SHARQ_RULES(false, false, true, float, int, 4)
  SHARQ_RULES(false, true, true, float, int64_t, 4)
  SHARQ_RULES(true, false, true, __nv_bfloat16, int, 8)
  SHARQ_RULES(true, true, true, __nv_bfloat16, int64_t, 8)
  SHARQ_RULES(false, false, false, float, int, 1)
  SHARQ_RULES(false, true, false, float, int64_t, 1)
  SHARQ_RULES(true, false, false, __nv_bfloat16, int, 1)
  SHARQ_RULES(true, true, false, __nv_bfloat16, int64_t, 1)
#undef SHARQ_RULES
  return cudaErrorInvalidValue;
}

}  // namespace sharq
