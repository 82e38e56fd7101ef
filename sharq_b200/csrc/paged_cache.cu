// Rotary embedding of a merged qkv activation on its way into a paged key/value cache, for prompts and for single tokens.
//
// Row r of qkv holds the query, key and value heads of one token, which has position p = positions[r] of sequence s (r itself, or
// sequences[r]).  Per query and key head, with the halves (x1, x2):
//     out1 = x1 cos1 - x2 sin1,   out2 = x2 cos2 + x1 sin2         (rows p of the tables)
// The queries go to q_out [rows, heads, D], the keys to slot p % page_size of page page_table[s][p / page_size] of the key cache (and to
// k_out), the values to the same place of the value cache.  The tables and the activation are bf16, so every product is exact in float
// and a sum is rounded once to float, whichever way it is contracted; it is rounded once more, to bf16 or, divided by the head's scale, to
// e4m3 (saturating at +-448).
//
// Bound by HBM for prompts (2 bytes in and 2 out per element, the tables come from L2) and by latency for single tokens.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "decode_ops.cuh"
#include "sm100_ptx.cuh"

namespace sharq {

namespace {

__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t *>(&v);
}

__device__ __forceinline__ void unpack8(const uint4 &w, float (&f)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) f[2 * j] = lo_f(u[j]), f[2 * j + 1] = hi_f(u[j]);
}

__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}

// Eight neighbouring elements of a head into the cache.  The quotient by the scale is the float division's, by its residual from a product with
// the correctly rounded reciprocal (Markstein); 1024 and more saturate in e4m3 whatever the last bits, and a zero
// keeps its sign.  (16 divisions: 78 instead of 73 us for 16384 rows of 48 heads of 128.)
template <bool kFp8>
__device__ __forceinline__ void store8(char *at, const float (&f)[8], float scale, float reciprocal) {
  if (kFp8) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      q[j] = f[j] * reciprocal;
      const float residual = __fmaf_rn(-q[j], scale, f[j]);
      if (fabsf(q[j]) < 1024.0f && q[j] != 0.0f) q[j] = __fmaf_rn(residual, reciprocal, q[j]);
    }
    if (!(scale > 0x1p-100f && scale < 0x1p100f)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) q[j] = __fdiv_rn(f[j], scale);
    }
    *reinterpret_cast<uint2 *>(at) = make_uint2(e4m3x4(q[0], q[1], q[2], q[3]), e4m3x4(q[4], q[5], q[6], q[7]));
  } else {
    *reinterpret_cast<uint4 *>(at) = pack8(f);
  }
}

struct AppendArgs {
  const __nv_bfloat16 *qkv, *cos_t, *sin_t;
  long long row_stride;
  const int *positions, *sequences;
  __nv_bfloat16 *q_out, *k_out;
  int *error_flag;
  int rows, heads, table_rows, page_shift;  // page_shift: log2 of the page size, -1 if it is no power of two
};

// Heads per thread: one for few rows, where only the way to the result counts, and three from kManyRows rows on, whose loads are in flight
// together.  One / three, 48 heads of 128, us: 1 row 1.7 / 2.3, 64 rows 1.8 / 2.3, 256 rows 2.4 / 2.9, 512 rows 5.0 / 4.4, 2048 rows
// 16.1 / 12.0, 16384 rows in e4m3 114 / 73.  (Two: 77.)
constexpr int kManyRows = 512, kHeadsOfMany = 3;

// A thread takes 8 elements of the first half of a head and their 8 partners of the second half: threadIdx = (vector of the half head, head,
// row of the CTA), so that nothing is divided to find them; its further heads are blockDim.y apart and share the row's place and the tables.
// What it rotates is loaded first, and the row's place is found meanwhile: a thread that looked the place up before it loaded anything took
// 98 us for 16384 rows of 36 heads of 128, 53.5 to 55 now (91 to 89 % of the rate of a copy).  With the 84 registers that the compiler takes without the
// second bound (64) it is 61.7, for want of warps: what it has to spill costs less.
template <bool kFp8, int kHeads>
__global__ void __launch_bounds__(512, 2) rope_append_kernel(const __grid_constant__ AppendArgs a, const __grid_constant__ PagedCache c) {
  const int half = c.head_dim >> 1, v = threadIdx.x, row = blockIdx.x * blockDim.z + threadIdx.z, all_heads = a.heads + 2 * c.kv_heads;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (row >= a.rows) return;
  const int position = a.positions[row], seq = a.sequences != nullptr ? a.sequences[row] : row;
  const __nv_bfloat16 *x = a.qkv + row * a.row_stride + v * 8;
  const int head0 = blockIdx.y * blockDim.y * kHeads + threadIdx.y;
  uint4 w1[kHeads], w2[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int head = head0 + i * blockDim.y;
    if (head >= all_heads) break;
    w1[i] = *reinterpret_cast<const uint4 *>(x + head * c.head_dim);
    w2[i] = *reinterpret_cast<const uint4 *>(x + head * c.head_dim + half);
  }
  const bool padding = position < 0;
  const bool in_tables = !padding && position < a.table_rows && position < paged_capacity(c) && seq >= 0 && seq < c.seqs;
  uint4 wc1, wc2, ws1, ws2;
  int page = 0, in_page = 0;
  if (in_tables) {
    if (head0 < a.heads + c.kv_heads) {
      const __nv_bfloat16 *cos_at = a.cos_t + (size_t)position * c.head_dim + v * 8, *sin_at = a.sin_t + (size_t)position * c.head_dim + v * 8;
      wc1 = *reinterpret_cast<const uint4 *>(cos_at);
      wc2 = *reinterpret_cast<const uint4 *>(cos_at + half);
      ws1 = *reinterpret_cast<const uint4 *>(sin_at);
      ws2 = *reinterpret_cast<const uint4 *>(sin_at + half);
    }
    const int entry = a.page_shift >= 0 ? position >> a.page_shift : position / c.page_size;
    in_page = position - entry * c.page_size;
    page = c.page_table[seq * c.table_stride + entry];
  }
  const bool good = in_tables && page >= 0 && page < c.pages;
  if (!good && !padding && head0 == 0 && v == 0 && a.error_flag != nullptr) atomicExch(a.error_flag, kBadCacheIndex);
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    const int head = head0 + i * blockDim.y, kv = head - a.heads;  // key head, or kv_heads + value head
    if (head >= all_heads) break;
    float x1[8], x2[8];
    unpack8(w1[i], x1);
    unpack8(w2[i], x2);
    if (!good) {
      // a padding row gives zeros, a row without a place NaN; neither touches the cache
      const float fill = padding ? 0.0f : __int_as_float(0x7fffffff);
#pragma unroll
      for (int j = 0; j < 8; ++j) x1[j] = x2[j] = fill;
    } else if (kv < c.kv_heads) {
      float c1[8], c2[8], s1[8], s2[8];
      unpack8(wc1, c1);
      unpack8(wc2, c2);
      unpack8(ws1, s1);
      unpack8(ws2, s2);
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // the products are exact
        const float o1 = __fmaf_rn(x1[j], c1[j], -__fmul_rn(x2[j], s1[j]));
        x2[j] = __fmaf_rn(x2[j], c2[j], __fmul_rn(x1[j], s2[j]));
        x1[j] = o1;
      }
    }
    if (kv < c.kv_heads) {
      __nv_bfloat16 *out = nullptr;
      if (kv < 0)
        out = a.q_out + ((size_t)row * a.heads + head) * c.head_dim + v * 8;
      else if (a.k_out != nullptr)
        out = a.k_out + ((size_t)row * c.kv_heads + kv) * c.head_dim + v * 8;
      if (out != nullptr) {
        *reinterpret_cast<uint4 *>(out) = pack8(x1);
        *reinterpret_cast<uint4 *>(out + half) = pack8(x2);
      }
    }
    if (kv >= 0 && good) {
      const bool value = kv >= c.kv_heads;
      const int kv_head = value ? kv - c.kv_heads : kv, size = kFp8 ? 1 : 2;
      char *at = (value ? c.v : c.k) + page * c.page_stride + in_page * c.token_stride + kv_head * c.head_stride + v * 8 * size;
      const float scale = kFp8 ? (value ? c.v_scale : c.k_scale)[kv_head] : 1.0f;
      const float reciprocal = kFp8 ? __frcp_rn(scale) : 1.0f;
      store8<kFp8>(at, x1, scale, reciprocal);
      store8<kFp8>(at + half * size, x2, scale, reciprocal);
    }
  }
}

}  // namespace

cudaError_t run_rope_append_paged(const void *qkv, long long row_stride, int rows, int heads, const void *cos_t, const void *sin_t,
                                  int table_rows, const int *positions, const int *sequences, const PagedCache &cache, bool fp8,
                                  void *q_out, void *k_out, int *error_flag, cudaStream_t stream) {
  if (rows <= 0) return cudaSuccess;
  AppendArgs a;
  a.qkv = static_cast<const __nv_bfloat16 *>(qkv);
  a.cos_t = static_cast<const __nv_bfloat16 *>(cos_t);
  a.sin_t = static_cast<const __nv_bfloat16 *>(sin_t);
  a.row_stride = row_stride;
  a.positions = positions;
  a.sequences = sequences;
  a.q_out = static_cast<__nv_bfloat16 *>(q_out);
  a.k_out = static_cast<__nv_bfloat16 *>(k_out);
  a.error_flag = error_flag;
  a.rows = rows;
  a.heads = heads;
  a.table_rows = table_rows;
  a.page_shift = (cache.page_size & (cache.page_size - 1)) == 0 ? __builtin_ctz((unsigned)cache.page_size) : -1;
  // CTAs of up to 512 threads, the heads of a row in equal shares; short rows share one of 128
  const int vecs = cache.head_dim / 16, all_heads = heads + 2 * cache.kv_heads, per = rows >= kManyRows ? kHeadsOfMany : 1;
  const int most = 512 / vecs * per, shares = (all_heads + most - 1) / most;
  const int share = ((all_heads + shares - 1) / shares + per - 1) / per;
  int together = 128 / (share * vecs);
  if (together < 1 || shares > 1) together = 1;
  if (together > 64) together = 64;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((rows + together - 1) / together), (unsigned)shares);
  cfg.blockDim = dim3((unsigned)vecs, (unsigned)share, (unsigned)together);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const auto kernel = per == 1 ? (fp8 ? rope_append_kernel<true, 1> : rope_append_kernel<false, 1>)
                               : (fp8 ? rope_append_kernel<true, kHeadsOfMany> : rope_append_kernel<false, kHeadsOfMany>);
  return cudaLaunchKernelEx(&cfg, kernel, a, cache);
}

}  // namespace sharq
