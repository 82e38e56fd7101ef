// Attention of one new token per sequence over a paged key/value cache.
//
//   out[b, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[b, h] . k_j - max),   j < lengths[b]
//
// One pass over the cache with a running maximum and sum.  A query group (the query heads that share a key/value head) is the 16-row operand of
// mma.sync.m16n8k16, in chunks of 16 heads; a warp streams tiles of keys and values through a ring of its own in shared memory (cp.async,
// no barrier between the warps of a CTA), multiplies, and keeps maximum, sum and the output rows in float registers.  The work is
// bound by reading the cache: 4 flop per byte and query head of the group, far below what even this tensor path gives, and a legacy MMA
// takes its operands from registers in the layout in which ldmatrix delivers cache rows, without a trip through tensor memory.
//
// The tiles of all sequences and heads are one list, and every CTA takes an equal stretch of it, whatever the lengths: a CTA joins the
// warps' parts of each (sequence, head) in shared memory and writes the finished row, or, where the stretch begins or ends inside a
// (sequence, head), a float part with its maximum and sum; a second kernel, which starts early and waits, joins those parts in the
// order of the list.  So the result does not depend on timing.
//
// e4m3 caches go through f16: their values are exact in it, queries are scaled to it by a power of two per head (a value below 2^-39 of its
// head's largest is lost), and probabilities carry a factor of 2^10, so that those down to 2^-24 of the largest keep f16's full precision.  For bf16
// caches the probabilities are rounded to bf16 for the product with the values (half a unit in the 8th bit, as the output itself); their sum is
// taken before that rounding, in float.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "decode_ops.cuh"
#include "sm100_ptx.cuh"

namespace sharq {

namespace {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr int kAttnStages = 3;
constexpr uint32_t kNaNWord = 0x7FFF7FFFu;  // NaN as two bf16 and as four e4m3
constexpr float kF16Lift = 10.0f;

__device__ __forceinline__ void cp_async16(uint32_t smem, const void *gmem, bool valid) {
  const int bytes = valid ? 16 : 0;  // 0: nothing is read, zeros are written
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t smem, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(smem), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t smem) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem) : "memory");
  return v;
}
__device__ __forceinline__ uint2 ld_shared8(uint32_t smem) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(smem) : "memory");
  return v;
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t smem) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t smem) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem)
               : "memory");
}

template <bool kF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_approx(float x) {  // 2 units in the last place; 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t *>(&v);
}
// the e4m3 values in the low / high half of a word as two f16
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
  return r;
}

struct AttnArgs {
  const __nv_bfloat16 *q;
  long long q_row, q_head;
  const int *lengths;
  __nv_bfloat16 *out;
  float *parts;  // [2 * gridDim.x][kRows][D] unnormalised rows, then their [maximum, sum]
  int *splits;   // [gridDim.x][2]: (sequence, head chunk) whose last tile lies in a later CTA and how many CTAs follow; 0 followers: none
  int seqs, heads, group, chunks;  // chunks: pieces of 16 query heads of a group
  float scale_log2;                // scale * log2(e)
  int *error_flag;
};

// Sizes that follow from the head and the type of the cache.  A tile holds 8 KB of keys and values (4 KB for e4m3 heads of 64).
template <int D, bool kFp8>
struct Tile {
  static constexpr int kSize = kFp8 ? 1 : 2;
  static constexpr int kTokens = D == 128 && !kFp8 ? 16 : 32;
  static constexpr int kChunks = D * kSize / 16;                // 16-byte pieces of a row
  static constexpr int kBytes = kTokens * D * kSize;            // of keys, or of values
  static constexpr int kStage = 2 * kBytes;
  static constexpr int kLoads = kTokens * kChunks / 32;         // per lane, for the keys and for the values
  // byte of piece `c` of row `r`: pieces are permuted so that the 8 rows of an ldmatrix, or the rows and pieces that a quarter of a warp
  // reads at once from an e4m3 tile, lie in different banks
  static __device__ __forceinline__ uint32_t at(int r, int c) {
    if (!kFp8) return (uint32_t)(r * kChunks + (c ^ (r & 7))) * 16;
    const int f = (r & 6) ^ ((r & 1) << 2);
    if (kChunks == 8) return (uint32_t)(r * 8 + (c ^ f)) * 16;
    return (uint32_t)((r >> 1) * 8 + ((((r & 1) << 2) | c) ^ (r & 6))) * 16;
  }
};

template <int D, int kRows>
constexpr int join_floats() {
  return kAttnWarps * 8 * (D + 4) + kAttnWarps * 16 * 2;  // eight rows at a time, and maximum and sum of all
}

template <int D, bool kFp8, int kRows>
constexpr int attn_smem_bytes() {
  return kAttnWarps * kAttnStages * Tile<D, kFp8>::kStage + join_floats<D, kRows>() * 4;
}

// A length as the kernel uses it: one that the page table cannot hold counts as an empty sequence whose rows come out as NaN.
struct Length {
  int tokens;
  bool bad;
};
__device__ __forceinline__ Length length_of(const AttnArgs &a, const PagedCache &c, int seq) {
  const int n = a.lengths[seq];
  const bool bad = n < 0 || n > paged_capacity(c);
  return {bad ? 0 : n, bad};
}
template <int kTokens>
__device__ __forceinline__ int tiles_of(int tokens) {  // an empty sequence has one tile, without tokens
  return tokens <= kTokens ? 1 : (tokens - 1) / kTokens + 1;
}

// kRows: rows of the 16-row operand that hold query heads (8 or 16)
template <int D, bool kFp8, int kRows>
__global__ void __launch_bounds__(kAttnThreads, 2) paged_attention_kernel(AttnArgs a, PagedCache c) {
  using T = Tile<D, kFp8>;
  constexpr int kTokens = T::kTokens;
  extern __shared__ __align__(128) unsigned char smem[];
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = ptx::smem_u32(smem) + warp * kAttnStages * T::kStage;
  float *join_o = reinterpret_cast<float *>(smem + kAttnWarps * kAttnStages * T::kStage);
  float *join_ml = join_o + kAttnWarps * 8 * (D + 4);
  const int items = c.kv_heads * a.chunks;  // (head, chunk) pairs of a sequence

  // this CTA's stretch [u0, u1) of the list of tiles
  long long total = 0;
  for (int b = lane; b < a.seqs; b += 32) total += tiles_of<kTokens>(length_of(a, c, b).tokens);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
  total *= items;
  long long per = (total + gridDim.x - 1) / gridDim.x;
  if (per < kAttnWarps) per = kAttnWarps;
  const long long u0 = blockIdx.x * per, u1 = min(u0 + per, total);
  if (threadIdx.x == 0) a.splits[2 * blockIdx.x + 1] = 0;
  if (u0 >= u1) return;
  int seq = 0, item = 0, first = 0;  // sequence, (head, chunk) and tile at u0
  {
    long long before = 0;
    for (int b0 = 0; b0 < a.seqs; b0 += 32) {
      const int b = b0 + lane;
      long long n = b < a.seqs ? (long long)items * tiles_of<kTokens>(length_of(a, c, b).tokens) : 0;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, n, off);
        if (lane >= off) n += up;
      }
      const unsigned over = __ballot_sync(0xffffffffu, before + n > u0);
      if (over != 0) {
        const int at = __ffs(over) - 1;
        const long long upto = __shfl_sync(0xffffffffu, n, at > 0 ? at - 1 : 0);
        seq = b0 + at;
        const long long rest = u0 - before - (at > 0 ? upto : 0);
        const int n_tiles = tiles_of<kTokens>(length_of(a, c, seq).tokens);
        item = (int)(rest / n_tiles);
        first = (int)(rest % n_tiles);
        break;
      }
      before += __shfl_sync(0xffffffffu, n, 31);
    }
  }

  // the next tile that this warp loads: tile `p_tile` < p_end of (p_seq, p_item), with p_left tiles of the stretch from p_tile's item on
  int p_seq = seq, p_item = item, p_tile = first + warp, p_tokens = length_of(a, c, seq).tokens;
  long long p_left = u1 - u0;
  int p_end = (int)min((long long)tiles_of<kTokens>(p_tokens), first + p_left);
  int p_first = first;
  int p_page = 0;  // lane j: page of the tile's token j
  auto settle = [&]() {  // moves on to the next item with a tile for this warp, and looks up the tile's pages
    while (p_tile >= p_end && p_left > 0) {
      p_left -= p_end - p_first;
      if (p_left <= 0) break;
      if (++p_item == items) {
        p_item = 0;
        ++p_seq;
        p_tokens = length_of(a, c, p_seq).tokens;
      }
      p_first = 0;
      p_tile = warp;
      p_end = (int)min((long long)tiles_of<kTokens>(p_tokens), p_left);
    }
    const int token = p_tile * kTokens + lane;
    p_page = p_left > 0 && lane < kTokens && token < p_tokens ? c.page_table[p_seq * c.table_stride + token / c.page_size] : 0;
  };
  int put = 0;  // stage that is filled next
  auto load = [&]() {
    if (p_left > 0) {
      const uint32_t stage = ring + put * T::kStage;
      const int token0 = p_tile * kTokens, row0 = lane / T::kChunks, piece = lane % T::kChunks;
      const long long in_page = (p_item / a.chunks) * c.head_stride + piece * 16;
      const int slot0 = (token0 + lane) % c.page_size;  // lane j: slot of token j
#pragma unroll
      for (int i = 0; i < T::kLoads; ++i) {
        const int row = row0 + i * (32 / T::kChunks);
        const int page = __shfl_sync(0xffffffffu, p_page, row), slot = __shfl_sync(0xffffffffu, slot0, row);
        const bool live = token0 + row < p_tokens;
        const bool bad = live && (unsigned)page >= (unsigned)c.pages;
        const long long from = bad || !live ? 0 : page * c.page_stride + slot * c.token_stride + in_page;
        const uint32_t to = stage + T::at(row, piece);
        if (bad) {
          st_shared16(to, kNaNWord);
          if (a.error_flag != nullptr) atomicExch(a.error_flag, kBadCacheIndex);
        } else {
          cp_async16(to, c.k + from, live);
        }
        cp_async16(to + T::kBytes, c.v + from, live && !bad);
      }
      p_tile += kAttnWarps;
    }
    cp_async_commit();
    put = put + 1 == kAttnStages ? 0 : put + 1;
    settle();
  };
  settle();
  for (int i = 0; i < kAttnStages - 1; ++i) load();

  int take = 0;  // stage that is used next
  long long left = u1 - u0;
  while (left > 0) {
    const Length len = length_of(a, c, seq);
    const int n_tiles = tiles_of<kTokens>(len.tokens);
    const int last = (int)min((long long)n_tiles, first + left);
    const int kv = item / a.chunks, chunk = item % a.chunks;
    const int rows = min(16, a.group - chunk * 16);  // query heads of the chunk
    const int head0 = kv * a.group + chunk * 16;

    // queries: rows g and g + 8 of the operand, zeros behind the group's heads
    uint32_t qa[D / 16][4];
    float sl[2] = {a.scale_log2, a.scale_log2};
    if (!kFp8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = g + 8 * h;
        const __nv_bfloat16 *q = a.q + seq * a.q_row + (head0 + row) * a.q_head + 2 * t;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const bool live = h < kRows / 8 && row < rows;
          qa[k][h] = live ? *reinterpret_cast<const uint32_t *>(q + 16 * k) : 0;
          qa[k][h + 2] = live ? *reinterpret_cast<const uint32_t *>(q + 16 * k + 8) : 0;
        }
      }
    } else {
      // step k of a span of 64 elements takes the elements 16 t + 4 (k % 4) + {0, 1, 2, 3} of the span from lane t, as the keys do
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = g + 8 * h;
        const bool live = h < kRows / 8 && row < rows;
        const __nv_bfloat16 *q = a.q + seq * a.q_row + (head0 + row) * a.q_head + 16 * t;
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint2 w = live ? *reinterpret_cast<const uint2 *>(q + (k / 4) * 64 + (k % 4) * 4) : make_uint2(0, 0);
          qa[k][h] = w.x;
          qa[k][h + 2] = w.y;
          top = __vmaxu2(top, __vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu));
        }
        top = max(top & 0xFFFFu, top >> 16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the largest value to [2^14, 2^15); a row with infinities or NaN as it is
        const int e = (int)(top >> 7), shift = e == 255 ? 0 : 141 - max(e, 1);
        // in two factors, each a normal float
        const int s1 = shift / 2, s2 = shift - s1;
        const float f1 = __int_as_float((127 + s1) << 23), f2 = __int_as_float((127 + s2) << 23);
        sl[h] = a.scale_log2 * c.k_scale[kv] * __int_as_float((127 - s1) << 23) * __int_as_float((127 - s2) << 23);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            const uint32_t w = qa[k][h + j];
            qa[k][h + j] = pack_f16(__uint_as_float(w << 16) * f1 * f2, __uint_as_float(w & 0xFFFF0000u) * f1 * f2);
          }
        }
      }
    }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    // maximum (of the scores, in units of log 2) and sum of rows g and g + 8
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int tile = first + warp; tile < last; tile += kAttnWarps) {
      load();
      cp_async_wait<kAttnStages - 1>();
      __syncwarp();
      const uint32_t keys = ring + take * T::kStage, values = keys + T::kBytes;

      float s[kTokens / 8][4];
#pragma unroll
      for (int n = 0; n < kTokens / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
      if (!kFp8) {
#pragma unroll
        for (int n = 0; n < kTokens / 16; ++n)
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];
            ldmatrix4(b, keys + T::at(n * 16 + (lane >> 4) * 8 + (lane & 7), 2 * k + ((lane >> 3) & 1)));
            mma16816<kFp8>(s[2 * n], qa[k], b[0], b[1]);
            mma16816<kFp8>(s[2 * n + 1], qa[k], b[2], b[3]);
          }
      } else {
#pragma unroll
        for (int n = 0; n < kTokens / 8; ++n)
#pragma unroll
          for (int span = 0; span < D / 64; ++span) {
            const uint4 w = ld_shared16(keys + T::at(n * 8 + g, span * 4 + t));
            mma16816<kFp8>(s[n], qa[span * 4 + 0], e4m3_lo(w.x), e4m3_hi(w.x));
            mma16816<kFp8>(s[n], qa[span * 4 + 1], e4m3_lo(w.y), e4m3_hi(w.y));
            mma16816<kFp8>(s[n], qa[span * 4 + 2], e4m3_lo(w.z), e4m3_hi(w.z));
            mma16816<kFp8>(s[n], qa[span * 4 + 3], e4m3_lo(w.w), e4m3_hi(w.w));
          }
      }

#pragma unroll
      for (int n = 0; n < kTokens / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] *= sl[j >> 1];
      const int live = len.tokens - tile * kTokens;  // tokens of the tile
      if (live < kTokens) {
#pragma unroll
        for (int n = 0; n < kTokens / 8; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n * 8 + 2 * t + (j & 1) >= live) s[n][j] = -INFINITY;
      }
      float top[2] = {m[0], m[1]};
#pragma unroll
      for (int h = 0; h < kRows / 8; ++h) {
#pragma unroll
        for (int n = 0; n < kTokens / 8; ++n) top[h] = fmaxf(top[h], fmaxf(s[n][2 * h], s[n][2 * h + 1]));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
        top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
        for (int h = 0; h < kRows / 8; ++h) {
          const float f = top[h] > m[h] ? exp2_approx(m[h] - top[h]) : 1.0f;  // m = -inf: 0, and nothing to keep
          m[h] = top[h];
          l[h] *= f;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][2 * h] *= f;
            o[i][2 * h + 1] *= f;
          }
        }
      }
      uint32_t p[kTokens / 8][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h >= kRows / 8) {
#pragma unroll
          for (int n = 0; n < kTokens / 8; ++n) p[n][h] = 0;
          continue;
        }
        // a row with no finite score so far has maximum -inf: its probabilities are 0, not exp(-inf + inf)
        const float base = (m[h] == -INFINITY ? 0.0f : m[h]) - (kFp8 ? kF16Lift : 0.0f);
#pragma unroll
        for (int n = 0; n < kTokens / 8; ++n) {
          const float p0 = exp2_approx(s[n][2 * h] - base), p1 = exp2_approx(s[n][2 * h + 1] - base);
          l[h] += p0 + p1;
          p[n][h] = kFp8 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
        }
      }

#pragma unroll
      for (int k = 0; k < kTokens / 16; ++k) {
        const uint32_t pa[4] = {p[2 * k][0], p[2 * k][1], p[2 * k + 1][0], p[2 * k + 1][1]};
        if (!kFp8) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t b[4];
            ldmatrix4_trans(b, values + T::at(k * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), 2 * i + (lane >> 4)));
            mma16816<kFp8>(o[2 * i], pa, b[0], b[1]);
            mma16816<kFp8>(o[2 * i + 1], pa, b[2], b[3]);
          }
        } else {
          // lane (g, t) takes the elements g * (D / 8) + i of four tokens; column g of output tile i is element g * (D / 8) + i
          constexpr int kWords = D / 32;
          uint32_t w[4][kWords];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = k * 16 + 2 * t + (j & 1) + (j >> 1) * 8;
            if (D == 128) {
              const uint4 v = ld_shared16(values + T::at(row, g));
              w[j][0] = v.x, w[j][1] = v.y, w[j][kWords - 2] = v.z, w[j][kWords - 1] = v.w;
            } else {
              const uint2 v = ld_shared8(values + T::at(row, g >> 1) + (g & 1) * 8);
              w[j][0] = v.x, w[j][1] = v.y;
            }
          }
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            const uint32_t a0 = __byte_perm(w[0][i], w[1][i], 0x5140), a1 = __byte_perm(w[0][i], w[1][i], 0x7362);
            const uint32_t b0 = __byte_perm(w[2][i], w[3][i], 0x5140), b1 = __byte_perm(w[2][i], w[3][i], 0x7362);
            mma16816<kFp8>(o[4 * i + 0], pa, e4m3_lo(a0), e4m3_lo(b0));
            mma16816<kFp8>(o[4 * i + 1], pa, e4m3_hi(a0), e4m3_hi(b0));
            mma16816<kFp8>(o[4 * i + 2], pa, e4m3_lo(a1), e4m3_lo(b1));
            mma16816<kFp8>(o[4 * i + 3], pa, e4m3_hi(a1), e4m3_hi(b1));
          }
        }
      }
      __syncwarp();  // the stage may be filled again
      take = take + 1 == kAttnStages ? 0 : take + 1;
    }

    // join the warps' parts
#pragma unroll
    for (int h = 0; h < kRows / 8; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    const bool whole = first == 0 && last == n_tiles;
    // the part of an item that began in an earlier CTA goes to this CTA's first place, of one that goes on in a later CTA to the second
    const long long place = 2LL * blockIdx.x + (first == 0 ? 1 : 0);
    float *part = a.parts + place * kRows * D;
    float *part_ml = a.parts + 2LL * gridDim.x * kRows * D + place * kRows * 2;
#pragma unroll
    for (int h = 0; h < kRows / 8; ++h) {
      __syncthreads();  // the space is free
      if (t == 0) {
        join_ml[(warp * 8 + g) * 2] = m[h];
        join_ml[(warp * 8 + g) * 2 + 1] = l[h];
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        float *to = join_o + (warp * 8 + g) * (D + 4);
        if (!kFp8) {
          *reinterpret_cast<float2 *>(to + 8 * i + 2 * t) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
        } else {
          to[2 * t * (D / 8) + i] = o[i][2 * h];
          to[(2 * t + 1) * (D / 8) + i] = o[i][2 * h + 1];
        }
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 8 * D; i += kAttnThreads) {
        const int row = i / D, d = i % D;
        if (8 * h + row >= rows) break;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) top = fmaxf(top, join_ml[(w * 8 + row) * 2]);
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
          const float mw = join_ml[(w * 8 + row) * 2];
          const float f = mw == top ? 1.0f : exp2_approx(mw - top);  // also where all are -inf
          sum += join_ml[(w * 8 + row) * 2 + 1] * f;
          acc += join_o[(w * 8 + row) * (D + 4) + d] * f;
        }
        if (whole) {
          float y = len.tokens == 0 ? 0.0f : acc / sum * (kFp8 ? c.v_scale[kv] : 1.0f);
          if (len.bad) y = __int_as_float(0x7fffffff);
          a.out[((long long)seq * a.heads + head0 + 8 * h + row) * D + d] = __float2bfloat16_rn(y);
        } else {
          part[(8 * h + row) * D + d] = acc;
          if (d == 0) {
            part_ml[(8 * h + row) * 2] = top;
            part_ml[(8 * h + row) * 2 + 1] = sum;
          }
        }
      }
    }
    if (threadIdx.x == 0) {
      if (len.bad && a.error_flag != nullptr) atomicExch(a.error_flag, kBadCacheIndex);
      if (first == 0 && !whole) {  // goes on in the next CTAs
        a.splits[2 * blockIdx.x] = seq * items + item;
        a.splits[2 * blockIdx.x + 1] = (int)((n_tiles - last + per - 1) / per);
      }
    }
    left -= last - first;
    first = 0;
    if (++item == items) {
      item = 0;
      ++seq;
    }
  }
  cp_async_wait<0>();
}

// The row blockIdx.y of the item that begins in CTA blockIdx.x of the kernel above and goes on in the next ones.
template <int D, int kRows, bool kFp8>
__global__ void __launch_bounds__(D) paged_attention_join_kernel(AttnArgs a, PagedCache c, int ctas) {
  ptx::grid_dependency_wait();
  const int followers = a.splits[2 * blockIdx.x + 1];
  if (followers == 0) return;
  const int at = a.splits[2 * blockIdx.x], items = c.kv_heads * a.chunks;
  const int seq = at / items, kv = at % items / a.chunks, chunk = at % items % a.chunks, row = blockIdx.y;
  if (row >= min(16, a.group - chunk * 16)) return;
  const float *ml = a.parts + 2LL * ctas * kRows * D;
  // part 0: the second place of this CTA, part i: the first place of the i-th CTA behind it
  auto place = [&](int i) { return i == 0 ? 2LL * blockIdx.x + 1 : 2LL * (blockIdx.x + i); };
  float top = -INFINITY;
  for (int i = 0; i <= followers; ++i) top = fmaxf(top, ml[(place(i) * kRows + row) * 2]);
  float sum = 0.0f, acc = 0.0f;
  for (int i = 0; i <= followers; ++i) {
    const float mi = ml[(place(i) * kRows + row) * 2];
    const float f = mi == top ? 1.0f : exp2_approx(mi - top);
    sum += ml[(place(i) * kRows + row) * 2 + 1] * f;
    acc += a.parts[(place(i) * kRows + row) * D + threadIdx.x] * f;
  }
  const float y = acc / sum * (kFp8 ? c.v_scale[kv] : 1.0f);
  a.out[((long long)seq * a.heads + kv * a.group + chunk * 16 + row) * D + threadIdx.x] = __float2bfloat16_rn(y);
}

int attn_sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0 && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 148;
  return sms[dev];
}

template <int D, bool kFp8, int kRows>
cudaError_t launch(const AttnArgs &a, const PagedCache &c, int ctas, cudaStream_t stream) {
  constexpr int kSmem = attn_smem_bytes<D, kFp8, kRows>();
  const auto kernel = paged_attention_kernel<D, kFp8, kRows>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kAttnThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, kernel, a, c);
  if (err != cudaSuccess) return err;
  cfg.gridDim = dim3((unsigned)ctas, (unsigned)(a.group < 16 ? a.group : 16));
  cfg.blockDim = dim3(D);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<D, kRows, kFp8>, a, c, ctas);
}

int attn_ctas() { return 2 * attn_sm_count(); }

}  // namespace

size_t paged_attention_workspace_bytes(int heads, int kv_heads, int head_dim) {
  const size_t rows = heads / kv_heads <= 8 ? 8 : 16, places = 2 * (size_t)attn_ctas();
  return places * rows * (head_dim + 2) * sizeof(float) + places * sizeof(int);
}

cudaError_t run_paged_attention(const void *q, long long q_row, long long q_head, int heads, const PagedCache &cache, bool fp8,
                                const int *lengths, float scale, void *out, void *workspace, int *error_flag, cudaStream_t stream) {
  const int ctas = attn_ctas(), group = heads / cache.kv_heads, rows = group <= 8 ? 8 : 16, d = cache.head_dim;
  AttnArgs a;
  a.q = static_cast<const __nv_bfloat16 *>(q);
  a.q_row = q_row;
  a.q_head = q_head;
  a.lengths = lengths;
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.parts = static_cast<float *>(workspace);
  a.splits = reinterpret_cast<int *>(a.parts + 2LL * ctas * rows * (d + 2));
  a.seqs = cache.seqs;
  a.heads = heads;
  a.group = group;
  a.chunks = (group + 15) / 16;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.error_flag = error_flag;
#define SHARQ_ATTN(D, FP8, ROWS) \
  if (d == D && fp8 == FP8 && rows == ROWS) return launch<D, FP8, ROWS>(a, cache, ctas, stream);
  SHARQ_ATTN(128, false, 8)
  SHARQ_ATTN(128, false, 16)
  SHARQ_ATTN(128, true, 8)
  SHARQ_ATTN(128, true, 16)
  SHARQ_ATTN(64, false, 8)
  SHARQ_ATTN(64, false, 16)
  SHARQ_ATTN(64, true, 8)
  SHARQ_ATTN(64, true, 16)
#undef SHARQ_ATTN
  return cudaErrorInvalidValue;
}

}  // namespace sharq
