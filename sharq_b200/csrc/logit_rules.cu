// Penalties for repeated tokens, biases and masks on logits, in one launch.  256 rows of 152064 with histories of up to 6000 tokens: 78.5 us, 4.1 TB/s; one
// row of 128256: 3.4 us (a call takes 5.6 on the host).
//
//   x' = x > 0 ? x / r : x r   (tokens of the history),   x' - f n - p [n > 0]   (n: how often the answer so far has the token),   + biases,   -inf where masked
//
// Bound by reading and writing the logits once.  What touches a logit is known by token, not by place, so a CTA takes a slice of a row, counts the
// history's tokens that fall into it in a table in shared memory (whole numbers: the order of the atomics does not matter), and passes over its slice once.  A
// history is read by every CTA of its row, from L2, which is what a wider slice saves; what it concerns becomes a list, so that the few logits that take
// arithmetic are dealt out evenly, and goes over what the pass has written.  The logits are on their way while the tokens are counted.  (With the arithmetic in the
// pass, where a warp waits for its few lanes, 182 us; slices of half the width in CTAs of half the size 86; the list's and the biases' logits fetched ahead
// of the pass 92; the first tokens ahead of the logits 99; the pass alone 47.5, as a copy.)
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

constexpr unsigned kSeen = 1u << 31, kCount = kSeen - 1;  // of a token's word; the rest counts

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

constexpr int kThreads = 512, kSliceMost = 16384;

// Tokens with several biases, a lane each: the warp goes through the list for 32 neighbours at a time, and each lane adds up its token's in their order.  The list
// is read as often as there are such neighbours, 32 times per warp at most, however many biases a token has.  several: of the 32 neighbours that
// begin at 32 * (warp + 16 * lane), those that are such tokens and are not masked.
template <typename T>
__device__ __forceinline__ void add_several(const int *ids, const float *values, int biases, int first, unsigned several, const unsigned *words, const T *in, T *out,
                                            double repetition, double presence, double frequency) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (unsigned left = __ballot_sync(0xffffffffu, several != 0); left != 0; left &= left - 1) {
    const int from = __ffs(left) - 1, word = warp + from * (kThreads / 32);
    const unsigned these = __shfl_sync(0xffffffffu, several, from);
    double bias = -0.0;  // which changes no number that it is added to
    for (int j0 = 0; j0 < biases; j0 += 32) {
      const unsigned at = j0 + lane < biases ? (unsigned)ids[j0 + lane] - (unsigned)first : ~0u;
      const bool mine = (int)(at >> 5) == word && (these >> (at & 31) & 1) != 0;
      unsigned hits = __ballot_sync(0xffffffffu, mine);
      if (hits == 0) continue;
      const float value = mine ? values[j0 + lane] : 0.0f;
      for (; hits != 0; hits &= hits - 1) {
        const int of = __ffs(hits) - 1;
        const unsigned whose = __shfl_sync(0xffffffffu, at, of) & 31;
        const float x = __shfl_sync(0xffffffffu, value, of);
        if (whose == (unsigned)lane) bias += (double)x;
      }
      __syncwarp();
    }
    if ((these >> lane & 1) != 0) {
      const int at = word * 32 + lane;
      out[at] = rounded<T>(penalised(widened<T>(in[at]), words[at], {repetition, presence, frequency}) + bias);
    }
    __syncwarp();
  }
}

// T: type of the logits; Id: of the history's tokens; kVec: logits of a 16-byte access, or 1
template <typename T, typename Id, int kVec>
__global__ void __launch_bounds__(kThreads, 2) logit_rules_kernel(const __grid_constant__ LogitRules a) {
  constexpr int kPer = kSliceMost / (kThreads * kVec);  // accesses of a thread
  // for every token of the slice how often the history has it, and two bits: it has a bias, it has several; then the history's tokens, each once, in any order
  extern __shared__ __align__(16) unsigned words[];
  __shared__ int listed, repeated;  // repeated: some token has several biases
  unsigned *biased = words + a.slice, *twice = biased + a.slice / 32, *kept = twice + a.slice / 32;  // kept: the mask
  unsigned short *list = reinterpret_cast<unsigned short *>(kept + a.slice / 32);
  const int row = blockIdx.y, tid = threadIdx.x;
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
  const T *in = static_cast<const T *>(a.logits) + row * a.logits_stride + first;
  T *out = static_cast<T *>(a.out) + row * a.out_stride + first;
  static_assert(kThreads * 32 >= kSliceMost, "a word of the mask per thread");
  const unsigned mask = a.mask != nullptr && tid * 32 < size ? a.mask[row * a.mask_stride + first / 32 + tid] : ~0u;
  const float repetition = a.repetition == nullptr ? 1.0f : a.repetition[row], presence = a.presence == nullptr ? 0.0f : a.presence[row],
              frequency = a.frequency == nullptr ? 0.0f : a.frequency[row];
  struct __align__(kVec * sizeof(T)) Vec {
    T x[kVec];
  };
  Vec held[kPer];  // on their way while the history is counted
#pragma unroll
  for (int n = 0; n < kPer; ++n) {
    const int i = (n * kThreads + tid) * kVec;
    if (i + kVec <= size)
      held[n] = *reinterpret_cast<const Vec *>(in + i);
    else
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j < size) held[n].x[j] = in[i + j];
  }

  for (int i = tid * 4; i < a.slice + a.slice / 16; i += kThreads * 4) *reinterpret_cast<uint4 *>(words + i) = make_uint4(0, 0, 0, 0);
  if (tid == 0) listed = repeated = 0;
  __syncthreads();
  const Id *tokens = static_cast<const Id *>(a.tokens) + row * a.tokens_stride;
  auto place = [&](Id id, int *at) {  // in the slice
    if constexpr (sizeof(Id) == 4) {
      *at = (int)((unsigned)id - (unsigned)first);
      return (unsigned)*at < (unsigned)size;
    } else {
      *at = (int)(id - first);
      return id >= first && id - first < size;
    }
  };
  constexpr int kBatch = 32 / sizeof(Id);  // a thread's tokens that are on their way together
  for (int j0 = tid; j0 < length; j0 += kBatch * kThreads) {
    Id ids[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) ids[u] = j0 + u * kThreads < length ? tokens[j0 + u * kThreads] : (Id)-1;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      int at;
      if (place(ids[u], &at)) {
        const unsigned old = j0 + u * kThreads < prompt ? atomicOr(words + at, kSeen) : atomicAdd(words + at, 1u);
        if (old == 0) list[atomicAdd(&listed, 1)] = (unsigned short)at;
      } else if (ids[u] >= a.vocab) {
        bad = true;
      }
    }
  }
  auto mark = [&](int at) {
    const unsigned bit = 1u << (at & 31);
    if ((atomicOr(biased + (at >> 5), bit) & bit) != 0) atomicOr(twice + (at >> 5), bit), repeated = 1;
  };
  for (int j = bias0 + tid; j < bias1; j += kThreads) {
    const long long at = (long long)a.bias_ids[j] - first;
    if (at >= 0 && at < size)
      mark((int)at);
    else if (at + first < 0 || at + first >= a.vocab)
      bad = true;
  }
  if (tid * 32 < size) kept[tid] = mask;
  __syncthreads();

  // the logits as they are, or -inf
  const bool in_place = static_cast<const void *>(in) == static_cast<const void *>(out);
#pragma unroll
  for (int n = 0; n < kPer; ++n) {
    const int i = (n * kThreads + tid) * kVec;
    if (i >= size) break;
    constexpr unsigned kAll = (1u << kVec) - 1;
    const unsigned keep = kept[i >> 5] >> (i & 31) & kAll;
    if (in_place && keep == kAll) continue;
#pragma unroll
    for (int j = 0; j < kVec; ++j)
      if ((keep >> j & 1) == 0) held[n].x[j] = rounded<T>((double)minus_inf());
    if (i + kVec <= size)
      *reinterpret_cast<Vec *>(out + i) = held[n];
    else
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j < size) out[i + j] = held[n].x[j];
  }
  __syncthreads();

  // those that something concerns, from the logits as they were, over what has just been written (few turns of these loops: unrolled, 79.1 us)
  const Penalty penalty = {repetition, presence, frequency};
  auto stays = [&](int at) { return (kept[at >> 5] >> (at & 31) & 1) != 0; };
  const int concerned = listed;
#pragma unroll 1
  for (int j = tid; j < concerned; j += kThreads) {
    const int at = list[j];
    if ((biased[at >> 5] >> (at & 31) & 1) == 0 && stays(at)) out[at] = rounded<T>(penalised(widened<T>(in[at]), words[at], penalty));
  }
  // a token with one bias, by the bias's thread
  auto add = [&](int at, T x, float value) {
    if (stays(at) && (twice[at >> 5] >> (at & 31) & 1) == 0) out[at] = rounded<T>(penalised(widened<T>(x), words[at], penalty) + (double)value);
  };
#pragma unroll 1
  for (int j = bias0 + tid; j < bias1; j += kThreads) {
    const long long at = (long long)a.bias_ids[j] - first;
    if (at >= 0 && at < size) add((int)at, in[at], a.bias_values[j]);
  }
  if (repeated != 0) {
    static_assert(kThreads >= kSliceMost / 32, "32 neighbours per thread, of which its warp looks after all");
    const int word = (tid >> 5) + (tid & 31) * (kThreads / 32);
    const unsigned several = word < a.slice / 32 ? twice[word] & kept[word] : 0;
    add_several<T>(a.bias_ids + bias0, a.bias_values + bias0, bias1 - bias0, first, several, words, in, out, penalty.repetition, penalty.presence, penalty.frequency);
  }
  if (bad && a.error_flag != nullptr) atomicCAS(a.error_flag, 0, kBadLogitRules);
}

template <typename T, typename Id, int kVec>
cudaError_t launch(LogitRules a, cudaStream_t stream) {
  static int counts[64] = {};  // SMs of a device
  int dev = 0, sms = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err == cudaSuccess && dev < 64) sms = counts[dev];
  if (err == cudaSuccess && sms == 0) err = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (err != cudaSuccess) return err;
  if (dev < 64) counts[dev] = sms;
  // Equal slices of a row, as many as its tokens need, or as give every SM a CTA, but of 1024 tokens at least
  const int most = (a.vocab + 1023) / 1024, enough = (a.vocab + kSliceMost - 1) / kSliceMost, wanted = (sms + a.rows - 1) / a.rows;
  const int slices = wanted > most ? most : wanted > enough ? wanted : enough;
  a.slice = ((a.vocab + slices - 1) / slices + 127) / 128 * 128;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((a.vocab + a.slice - 1) / a.slice), (unsigned)a.rows);
  cfg.blockDim = dim3(kThreads);
  const long long concerned = (long long)a.width + a.biases;
  const int entries = concerned < a.slice ? (int)concerned : a.slice;  // of the list, at most
  cfg.dynamicSmemBytes = (size_t)(a.slice + a.slice / 32 * 3) * sizeof(unsigned) + (size_t)entries * sizeof(unsigned short);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  static bool ready[64] = {};
  err = allow_smem(logit_rules_kernel<T, Id, kVec>, (kSliceMost + kSliceMost / 32 * 3) * (int)sizeof(unsigned) + kSliceMost * (int)sizeof(unsigned short), ready);
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
