// Products of a few bf16 rows (1 to 16) with a 4-bit weight, the activation unquantised:
//
//   y[m, n] = bf16(scale * sum_k x[m, k] * e2m1[n, k] * ue4m3[n, k / 16] + bias[n])
//
// on the payload and the dense scale factors that a quantised linear holds.  Reading the weight (9/16 byte per element) is what it costs.
// At that rate an SM gets some 42 elements per clock, so the instructions per element count: a pair of codes is one conversion to f16 (exact), its
// scale one packed product (exact: 2 x 4 significant bits, between 2^-10 and 2688), and mma.sync.m16n8k16 with the 16 rows of weight as
// the large operand does the rest, 1.3 instructions per element in all.  The k positions of an instruction may stand for any elements
// as long as both operands agree, so lane (g, t) takes 32 neighbouring elements of a row, 16 bytes, straight from where it copied them.
//
// The activation goes to f16 as well, 128 elements of a row at a time, scaled by the power of two that takes their largest to [2^14, 2^15):
// exact but for elements below 2^-39 of it.  Sums are float: the tensor core's over 128 elements, then one float accumulator.
//
// A CTA takes 128 rows of the weight (a tile of scale factors) and a stretch of K; its warps stream their parts through rings of their own
// (cp.async).  Where the row tiles do not fill the GPU, K is dealt over the CTAs of a cluster of up to 8, whose float parts meet in
// distributed shared memory and are summed in rank order: the same bits from call to call, no scratch and no second launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "decode_ops.cuh"
#include "sm100_ptx.cuh"

namespace sharq {

namespace {

constexpr int kWoWarps = 8;  // four of 32 rows each, times two over K
constexpr int kWoThreads = 32 * kWoWarps;
constexpr int kWoStages = 4;
constexpr int kWoStage = 5 * 512;  // 128 elements of 32 rows and their scale factors, 16 bytes per lane and piece
constexpr int kWoXBytes = 24576;
constexpr int kWoPitch = 132;  // floats between the columns of a float part [columns][128 rows]
constexpr int kWoXScales = 96 * 8;  // one per block of 128 elements and column: at most 96 blocks of one row at a time
constexpr int kWoSmem = kWoWarps * kWoStages * kWoStage + kWoXBytes + kWoXScales * 4;

__device__ __forceinline__ void wo_cp_async16(uint32_t smem, const void *gmem, bool valid) {
  const int bytes = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 wo_lds16(uint32_t smem) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem) : "memory");
  return v;
}
// eight e2m1 codes -> four pairs of f16
__device__ __forceinline__ void e2m1_to_f16(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t"
      ".reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t"
      "}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t scaled_pair(uint32_t w, float f) {
  const __half2 h = __floats2half2_rn(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xFFFF0000u) * f);
  return *reinterpret_cast<const uint32_t *>(&h);
}

struct WeightOnlyArgs {
  const __nv_bfloat16 *x;
  long long x_row;
  const unsigned char *qw, *sf;
  const float *scale_dev;
  const __nv_bfloat16 *bias;
  __nv_bfloat16 *y;
  float scale;
  int m, n, k, splits;
};

// kTiles: 8-row tiles of the activation (1 or 2).  blockIdx.x: stretch of K, rank in the cluster; blockIdx.y: 128 rows of the weight.
template <int kTiles>
__global__ void __launch_bounds__(kWoThreads, 2) weight_only_kernel(WeightOnlyArgs a) {
  extern __shared__ __align__(128) unsigned char smem[];
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row_warp = warp & 3, k_warp = warp >> 2;
  const uint32_t ring = ptx::smem_u32(smem) + warp * kWoStages * kWoStage + lane * 16;
  unsigned char *xs = smem + kWoWarps * kWoStages * kWoStage;
  float *x_scale = reinterpret_cast<float *>(xs + kWoXBytes);
  const uint32_t xs_addr = ptx::smem_u32(xs);

  // this CTA's blocks of 128 elements of K
  const int blocks = (a.k + 127) / 128;
  const int b0 = (int)((long long)blocks * blockIdx.x / a.splits), b1 = (int)((long long)blocks * (blockIdx.x + 1) / a.splits);

  // rows 32 i + 8 row_warp + g of the tile, i = 0..3: their scale factors for 64 elements are 16 neighbouring bytes
  const int row0 = blockIdx.y * 128 + 8 * row_warp + g;
  const long long row_bytes = a.k / 2;
  const unsigned char *w0 = a.qw + row0 * row_bytes + t * 16;
  const unsigned char *s0 = a.sf + (long long)blockIdx.y * (a.k / 64) * 512 + (t >> 1) * 512 + (8 * row_warp + g) * 16;
  int next = b0 + k_warp, put = 0;
  auto load = [&]() {
    if (next < b1) {
      const uint32_t to = ring + put * kWoStage;
      const bool in_k = next * 128 + 32 * t < a.k;  // K may end in the middle of a block
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool valid = in_k && row0 + 32 * i < a.n;
        wo_cp_async16(to + i * 512, valid ? w0 + 32 * i * row_bytes + next * 64LL : a.qw, valid);
      }
      wo_cp_async16(to + 4 * 512, in_k ? s0 + next * 1024LL : a.sf, in_k);
      next += 2;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    put = put + 1 == kWoStages ? 0 : put + 1;
  };
  for (int i = 0; i < kWoStages - 1; ++i) load();

  float acc[2][kTiles][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.0f;
  // the weight's scale goes into the blocks' factors, so that a sum is in the result's range on its way
  const float scale = a.scale_dev != nullptr ? *a.scale_dev * a.scale : a.scale;
  const int room = min(96, kWoXBytes / (256 * a.m)) & ~1;  // blocks of the activation that are held at a time
  int take = 0;
  for (int c0 = b0; c0 < b1; c0 += room) {
    const int c1 = min(b1, c0 + room);
    if (c0 != b0) __syncthreads();
    // the activation's blocks as f16, in the order in which lanes read them: [block][word of a lane's 16 bytes][row][t], 16 bytes each
    const int half_warp = threadIdx.x >> 4, sub = threadIdx.x & 15;
    for (int i = half_warp; i < (c1 - c0) * a.m; i += kWoThreads / 16) {
      const int block = i / a.m, row = i % a.m, e0 = (c0 + block) * 128 + sub * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (e0 < a.k) v = *reinterpret_cast<const uint4 *>(a.x + row * a.x_row + e0);
      uint32_t top = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
      top = max(top & 0xFFFFu, top >> 16);
      const unsigned mask = 0xFFFFu << (threadIdx.x & 16);
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(mask, top, off));
      // a block with infinities or NaN is scaled down, so that nothing finite joins them
      const int e = (int)(top >> 7), shift = e == 255 ? -120 : min(126, 141 - max(e, 1));
      const float f = __int_as_float((127 + shift) << 23);
      v = make_uint4(scaled_pair(v.x, f), scaled_pair(v.y, f), scaled_pair(v.z, f), scaled_pair(v.w, f));
      *reinterpret_cast<uint4 *>(xs + (((block * 4 + (sub & 3)) * a.m + row) * 4 + (sub >> 2)) * 16) = v;
      if (sub == 0) x_scale[block * 8 * kTiles + row] = __int_as_float((127 - shift) << 23) * scale;
    }
    __syncthreads();

    for (int block = c0 + k_warp; block < c1; block += 2) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kWoStages - 2) : "memory");
      const uint32_t from = ring + take * kWoStage;
      uint4 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = wo_lds16(from + i * 512);
      const uint4 sf = wo_lds16(from + 4 * 512);
      take = take + 1 == kWoStages ? 0 : take + 1;
      load();
      const uint32_t sw[4] = {sf.x, sf.y, sf.z, sf.w};
      uint32_t s[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t two = e4m3x2_to_f16(sw[i] >> ((t & 1) * 16));
        s[i][0] = __byte_perm(two, two, 0x1010);
        s[i][1] = __byte_perm(two, two, 0x3232);
      }
      float d[2][kTiles][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int n = 0; n < kTiles; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) d[i][n][j] = 0.0f;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint4 x[kTiles];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          x[n] = make_uint4(0, 0, 0, 0);
          if (8 * n + g < a.m) x[n] = wo_lds16(xs_addr + ((((block - c0) * 4 + q) * a.m + 8 * n + g) * 4 + t) * 16);
        }
        uint32_t h[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e2m1_to_f16(q == 0 ? w[i].x : q == 1 ? w[i].y : q == 2 ? w[i].z : w[i].w, h[i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) h[i][j] = mul_f16x2(h[i][j], s[i][q >> 1]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            mma_f16(d[i][n], h[2 * i][0], h[2 * i + 1][0], h[2 * i][1], h[2 * i + 1][1], x[n].x, x[n].y);
            mma_f16(d[i][n], h[2 * i][2], h[2 * i + 1][2], h[2 * i][3], h[2 * i + 1][3], x[n].z, x[n].w);
          }
      }
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        // columns behind the activation's last row: their products are 0, and their scales are not there
        const float f0 = 8 * n + 2 * t < a.m ? x_scale[(block - c0) * 8 * kTiles + 8 * n + 2 * t] : 0.0f;
        const float f1 = 8 * n + 2 * t + 1 < a.m ? x_scale[(block - c0) * 8 * kTiles + 8 * n + 2 * t + 1] : 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          acc[i][n][0] += d[i][n][0] * f0;
          acc[i][n][1] += d[i][n][1] * f1;
          acc[i][n][2] += d[i][n][2] * f0;
          acc[i][n][3] += d[i][n][3] * f1;
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // float parts [k_warp][column][row of the tile] over the activation's space, then the sum over the cluster's CTAs and their k_warps
  __syncthreads();
  float *part = reinterpret_cast<float *>(xs);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < kTiles; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        part[(k_warp * 8 * kTiles + 8 * n + 2 * t + (j & 1)) * kWoPitch + 32 * (2 * i + (j >> 1)) + 8 * row_warp + g] = acc[i][n][j];
  if (a.splits > 1)
    ptx::cluster_sync();
  else
    __syncthreads();
  const int rank = a.splits > 1 ? (int)ptx::cluster_ctarank() : 0;
  for (int i = rank * kWoThreads + threadIdx.x; i < 128 * a.m; i += a.splits * kWoThreads) {
    const int col = i >> 7, r = i & 127, row = blockIdx.y * 128 + r;
    float sum = 0.0f;
    for (int c = 0; c < a.splits; ++c) {
#pragma unroll
      for (int kw = 0; kw < 2; ++kw) {
        float *from = part + (kw * 8 * kTiles + col) * kWoPitch + r;
        float v;
        if (a.splits > 1)
          asm volatile(
              "{\n\t.reg .b32 remote;\n\tmapa.shared::cluster.u32 remote, %1, %2;\n\tld.shared::cluster.f32 %0, [remote];\n\t}"
              : "=f"(v)
              : "r"(ptx::smem_u32(from)), "r"(c)
              : "memory");
        else
          v = *from;
        sum += v;
      }
    }
    if (row < a.n) {
      float y = sum;
      if (a.bias != nullptr) y += __bfloat162float(a.bias[row]);
      a.y[(long long)col * a.n + row] = __float2bfloat16_rn(y);
    }
  }
  __syncwarp();
  if (a.splits > 1) ptx::cluster_sync();  // a CTA's memory is read until here
}

int wo_sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0 && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 148;
  return sms[dev];
}

}  // namespace

cudaError_t run_weight_only(const void *x, long long x_row, int m, int n, int k, const void *qw, const void *sf, const float *scale_dev,
                            float scale, const void *bias, void *y, cudaStream_t stream) {
  if (m < 1 || m > kWeightOnlyMaxRows || n < 1 || k < 64 || k % 64 != 0) return cudaErrorInvalidValue;
  const int tiles = (n + 127) / 128, blocks = (k + 127) / 128;
  if (tiles > 65535) return cudaErrorInvalidValue;
  int splits = 2 * wo_sm_count() / tiles;
  if (splits > 8) splits = 8;
  if (splits > blocks / 2) splits = blocks / 2;
  if (splits < 1) splits = 1;
  WeightOnlyArgs a;
  a.x = static_cast<const __nv_bfloat16 *>(x);
  a.x_row = x_row;
  a.qw = static_cast<const unsigned char *>(qw);
  a.sf = static_cast<const unsigned char *>(sf);
  a.scale_dev = scale_dev;
  a.scale = scale;
  a.bias = static_cast<const __nv_bfloat16 *>(bias);
  a.y = static_cast<__nv_bfloat16 *>(y);
  a.m = m;
  a.n = n;
  a.k = k;
  a.splits = splits;
  const auto kernel = m <= 8 ? weight_only_kernel<1> : weight_only_kernel<2>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kWoSmem);
  if (err != cudaSuccess) return err;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)splits;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)splits, (unsigned)tiles);
  cfg.blockDim = dim3(kWoThreads);
  cfg.dynamicSmemBytes = kWoSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = splits > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace sharq
