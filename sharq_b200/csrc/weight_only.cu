// Products of a few bf16 rows (1 to 16) with a 4-bit weight, the activation unquantised:
//
//   y[m, n] = bf16(scale * sum_k x[m, k] * e2m1[n, k] * ue4m3[n, k / 16] + bias[n])
//
// on the payload and the dense scale factors that a quantised linear holds.  Reading the weight (9/16 byte per element) is what it has to
// do: at the rate of a copy an SM gets some 42 elements per clock, so the instructions per element count.  A pair of codes is one
// conversion to f16 (exact), its scale one packed product (exact: 2 x 4 significant bits, between 2^-10 and 2688), and mma.sync.m16n8k16 with 16
// rows of weight as the large operand does the rest, from registers: the fifth generation's instructions would want the scaled weight
// in shared memory first, and have no use for so few columns.  The k positions of an instruction may stand for any elements as long
// as both operands agree, so lane (g, t) takes 32 neighbouring elements of a row, 16 bytes, straight from where they were copied.
//
// A warp keeps 256 elements of K of up to eight rows of the activation in registers, as f16 operands, and streams that slice of the weight's
// rows past them, 16 rows at a time, through a ring of its own (one tensor-map copy for each, two of them a stage; with cp.async every 16
// bytes of every lane passed the load unit, half of the time).  f16 is reached by scaling 128 elements of a row by the power of two that takes their
// largest to [2^14, 2^15): exact down to 2^-31 of it, and off by at most 2^-39 of it below that, where f16's numbers end.  Sums are float; the weight's scale is in the factors of the
// blocks of 128, so that no sum overflows that the result would not.  A CTA's 16 warps cover 4096 elements of K (or fewer, and several rows at a
// time), the CTAs of a cluster the rest; the clusters take equal shares of the rows.  The warps' sums of some rows meet in shared memory,
// those of CTAs in distributed shared memory, each added up in a fixed order: the same bits from call to call, no scratch and no second launch.
// More than eight rows are two halves of the grid, the second of which reads the weight from L2.
//
// 28672 x 4096: one row 14.1 us (4.7 TB/s, 72 % of the rate of a copy), 8 rows 17.1, 16 rows 27.9; 4096 x 4096, one row: 4.8 us.  (Tiles of 128
// rows per CTA with the activation in shared memory, 323 instead of 265 instructions per 16 rows x 256 and uneven shares: 19.8, 38 with 16
// rows and 6.6.)  The loop's instructions take 7 us to issue, below the copies' 10: what bounds it are the copies and the 4 us around
// the loop, in which they stand still, the activation's way to the registers before it and the join after.  Both eights of 16 rows in one warp, the weight converted once for 128 elements of K of each, took 34 us instead of 29 and, for
// 13 rows of 4608 x 3584, 8.8 instead of 8.0: twice as many parts to join, and clusters of two CTAs where one does.  Joining a chunk of rows while
// the next is multiplied gained nothing.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "decode_ops.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.cuh"

namespace sharq {

namespace {

constexpr int kWoWarps = 16;
constexpr int kWoThreads = 32 * kWoWarps;
constexpr int kWoStages = 2;
constexpr int kWoSums = 6144;     // bytes for a CTA's float sums of a chunk, twice
constexpr int kWoXWarp = 4096;    // of a warp's slice of the activation on its way to the registers
constexpr int kWoClusterMost = 8;
constexpr int kWoSmem = 232448;
constexpr int kWoSlice = 256;                                 // elements of K of a warp
constexpr int kWoBox = 8 * kWoSlice / 2;                      // bytes of the codes of 8 rows
constexpr int kWoCodes = 4 * kWoBox, kWoScales = 4 * 128;     // of 32 rows; 8 rows x 16 bytes of scale factors for each of 4 x 64 elements
constexpr unsigned kWoLost = 1u << 31;  // a lane's wait ran out: it waits for nothing more, and the one that copies copies nothing more (a vote took 3 %)
constexpr int kWoRing = kWoStages * (kWoCodes + kWoScales);
constexpr int kWoBars = kWoSmem - kWoWarps * kWoStages * 8 - 16;  // the barriers behind it all, and the flag of a wait that ran out
constexpr int kWoFactors = kWoBars - kWoWarps * 64;
constexpr int kWoParts = kWoFactors - 2 * kWoSums - kWoWarps * kWoRing;  // for the warps' float sums: of all of a CTA's tiles, or of two chunks of them
static_assert(kWoWarps * kWoXWarp <= kWoParts && kWoParts % 16 == 0 && kWoBars % 16 == 0, "what a CTA can have");

__device__ __forceinline__ uint4 wo_lds16(uint32_t smem) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(smem) : "memory");
  return v;
}
__device__ __forceinline__ uint16_t wo_lds2(uint32_t smem) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(smem) : "memory");
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
__device__ __forceinline__ __half2 e4m3x2_to_f16(uint16_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(w));
  return *reinterpret_cast<const __half2 *>(&r);
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, __half2 b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), b);
  return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ void mma_f16_from0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
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

__device__ __forceinline__ void copy_2d(uint32_t dst, const CUtensorMap *m, int c0, int c1, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(m),
               "r"(ptx::smem_u32(bar)), "r"(c0), "r"(c1)
               : "memory");
}
__device__ __forceinline__ void copy_3d(uint32_t dst, const CUtensorMap *m, int c0, int c1, int c2, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(m),
               "r"(ptx::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

__device__ __forceinline__ void copy_4d(uint32_t dst, const CUtensorMap *m, int c0, int c1, int c2, int c3, uint64_t *bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(m),
               "r"(ptx::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}

struct WeightOnlyArgs {
  const __nv_bfloat16 *x;
  long long x_row;
  int *error_flag;
  const float *scale_dev;
  const __nv_bfloat16 *bias;
  __nv_bfloat16 *y;
  float scale;
  int m, n, k;
  int slices;       // warps of a CTA along K
  int row_groups;   // warps of a CTA along the rows
  int passes;       // times that a cluster goes along K for all of it
  int cluster;      // CTAs
  int tiles;        // of 16 rows, of the whole weight
  int per_cluster;  // tiles
  int chunk;        // pairs of tiles whose sums are joined at a time
  int whole;        // blocks of 128 rows
  int parts_at, parts_bytes;  // of the space of kWoParts bytes, for the warps' sums; they are all of it unless the activation is read more than once
  unsigned per_tile_magic[2];  // ceil(2^32 / floats of a tile's sums) for the first and the second eight rows
  bool by_four;             // four neighbouring results are one store, and so many of the bias one load
};

// Tile j: rows 32 i + 8 c + g of a block of 128, i = 2 h and 2 h + 1, with c = j / 2 % 4 and h = j % 2: the scale factors of a pair of tiles, for
// 64 elements of K, are 16 neighbouring bytes per g.  Pairs are copied together; a share of the rows may begin or end within one.
__device__ __forceinline__ int tile_row(int j) { return (j >> 3) * 128 + (j & 1) * 64 + ((j >> 1) & 3) * 8; }

// blockIdx.x: CTA of the cluster, blockIdx.y: cluster, blockIdx.z: eight rows of the activation.  kPasses: a cluster goes along K several times
// (more than 32768 elements), which in the same kernel cost all others a tenth of their time, for the registers.
template <bool kPasses>
__global__ void __launch_bounds__(kWoThreads, 1)
    weight_only_kernel(const __grid_constant__ CUtensorMap map_tiles, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sf,
                       const __grid_constant__ WeightOnlyArgs a) {
  extern __shared__ __align__(1024) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row_first = blockIdx.z * 8, m = min(8, a.m - row_first);
  const uint32_t codes = ptx::smem_u32(smem) + warp * kWoStages * kWoCodes;  // on 1024 bytes, for the swizzle
  const uint32_t scales = ptx::smem_u32(smem) + kWoWarps * kWoStages * kWoCodes + warp * kWoStages * kWoScales;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + kWoBars) + warp * kWoStages;
  volatile int *gave_up = reinterpret_cast<volatile int *>(smem + kWoBars + kWoWarps * kWoStages * 8);
  if (threadIdx.x == 0) *gave_up = 0;
  if (lane == 0) {
    for (int i = 0; i < kWoStages; ++i) ptx::mbar_init(bars + i, 1);
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&map_tiles);
    ptx::tma_prefetch_desc(&map_sf);
  }
  unsigned char *space = smem + kWoWarps * kWoRing;
  float *parts = reinterpret_cast<float *>(space + a.parts_at), *sums = reinterpret_cast<float *>(space + kWoParts);
  int row_group = 0, slice_in = warp;
  while (slice_in >= a.slices) slice_in -= a.slices, ++row_group;
  const bool works = row_group < a.row_groups;
  const int j0 = blockIdx.y * a.per_cluster, j1 = min(j0 + a.per_cluster, a.tiles);
  const int k_first = (blockIdx.x * a.slices + slice_in) * kWoSlice, k_pass = a.cluster * a.slices * kWoSlice;

  // The pairs of this warp in order: those of its row group, pass by pass within a chunk of pairs whose sums are joined together.
  const int p0 = j0 >> 1, p1 = (j1 + 1) >> 1;
  int l_chunk = p0, l_pass = 0, l_pair = works ? p0 + row_group : p1, put = 0, k0 = k_first;
  __syncthreads();
  const bool chosen = ptx::elect_one();
  if (m <= 3 && l_pair < p1 && chosen) {
    // The first rows into L2, where they may be as old as they like: ahead of the wait for the kernels before.  More rows of the activation arrive
    // later for it: 28672 x 4096 with / without, 2 rows 14.6 / 15.2 us, 3 rows 15.1 / 15.3, 4 rows 15.7 / 15.5, 6 rows 17.5 / 17.0; 4096 x 4096
    // 5.0 / 4.9, 5.4 / 4.9, 5.4 / 5.3, 6.3 / 5.8.  (Of both stages: 15.6 instead of 14.5 with one row.)
#pragma unroll 1
    for (int i = 0; i < 4; ++i) ptx::tma_prefetch_l2_2d(&map_w, k0 / 2, tile_row(2 * l_pair) + 32 * i);
  }
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  unsigned phases = 0;  // parity of every stage's barrier, and kWoLost
  auto load = [&]() {
    if (l_pair < p1) {
      if (chosen && (phases & kWoLost) == 0) {
        // rows and elements that are not there come as zeros
        const int from = 2 * l_pair < j0 ? 1 : 0, to = 2 * l_pair + 1 < j1 ? 2 : 1, block = l_pair >> 2;
        ptx::mbar_arrive_expect_tx(bars + put, (to - from) * 2 * kWoBox + kWoScales);
        for (int h = from; h < to; ++h) {
          const uint32_t dst = codes + put * kWoCodes + h * 2 * kWoBox;
          if (block < a.whole) {
            copy_4d(dst, &map_tiles, k0 / 2, (l_pair & 3) * 8, 2 * h, block, bars + put);
          } else {
            copy_2d(dst, &map_w, k0 / 2, tile_row(2 * l_pair + h), bars + put);
            copy_2d(dst + kWoBox, &map_w, k0 / 2, tile_row(2 * l_pair + h) + 32, bars + put);
          }
        }
        copy_3d(scales + put * kWoScales, &map_sf, (l_pair & 3) * 128, k0 / 64, block, bars + put);
      }
      l_pair += a.row_groups;
      if (kPasses && l_pair >= min(l_chunk + a.chunk, p1)) {  // one row group
        if (++l_pass == a.passes) {
          l_pass = 0;
          l_chunk += a.chunk;
        }
        l_pair = l_chunk;
        k0 = k_first + l_pass * k_pass;
      }
    }
    put ^= 1;
  };
  static_assert(kWoStages == 2, "stages in turn");

  // the weight's scale goes into the factors of the activation's blocks, so that a sum is in the result's range on its way
  const float scale_of = a.scale_dev != nullptr ? *a.scale_dev : 1.0f;
  uint4 x[2][4];
  // A lane loads 16 bytes of every row of the warp's slice, and they go as f16 through shared memory to the lanes that multiply them.  Piece c of
  // row r lies at c ^ (c / 8 % 2 + 2 (r % 2)): the four pieces of eight lanes that read at once are in different banks.
  unsigned char *x_space = space + warp * kWoXWarp;
  float *factors = reinterpret_cast<float *>(smem + kWoFactors) + warp * 16;  // [block of 128 elements][column]: what its sum is multiplied by
  uint4 raw[8];
  auto load_x = [&](int from_k) {
    const bool in_k = works && from_k + lane * 8 < a.k;
    const __nv_bfloat16 *from = a.x + row_first * a.x_row + from_k + lane * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i % 4 == 0 && i >= m) break;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (i < m && in_k) raw[i] = *reinterpret_cast<const uint4 *>(from);
      from += a.x_row;
    }
  };
  auto convert_x = [&]() {
    const float scale = scale_of * a.scale;
    __syncwarp();  // the space is free
    // rows are converted four at a time, since each is a chain of exchanges, or one or two
    auto rows = [&](auto count, int half) {
      constexpr int kRows = decltype(count)::value;
      uint32_t top[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const uint4 v = raw[4 * half + r];
        top[r] = __vmaxu2(__vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu), __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
        top[r] = max(top[r] & 0xFFFFu, top[r] >> 16);
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1)  // over the 16 lanes of 128 elements
#pragma unroll
        for (int r = 0; r < kRows; ++r) top[r] = max(top[r], __shfl_xor_sync(0xffffffffu, top[r], off));
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const uint4 v = raw[4 * half + r];
        const int row = 4 * half + r;
        // a block with infinities or NaN is scaled down, so that nothing finite joins them
        const int e = (int)(top[r] >> 7), shift = e == 255 ? -120 : min(126, 141 - max(e, 1));
        const float f = __int_as_float((127 + shift) << 23);
        *reinterpret_cast<uint4 *>(x_space + row * kWoSlice * 2 + (lane ^ (((lane >> 3) & 1) | ((row & 1) << 1))) * 16) =
            make_uint4(scaled_pair(v.x, f), scaled_pair(v.y, f), scaled_pair(v.z, f), scaled_pair(v.w, f));
        if ((lane & 15) == 0) factors[(lane >> 4) * 8 + row] = __int_as_float((127 - shift) << 23) * scale;
      }
    };
    if (m == 1) {
      rows(std::integral_constant<int, 1>(), 0);
    } else if (m == 2) {
      rows(std::integral_constant<int, 2>(), 0);
    } else {
      rows(std::integral_constant<int, 4>(), 0);
      if (m > 4) rows(std::integral_constant<int, 4>(), 1);
    }
    __syncwarp();
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = b * 16 + t * 4 + q;
        x[b][q] = make_uint4(0, 0, 0, 0);
        if (g < m) x[b][q] = *reinterpret_cast<const uint4 *>(x_space + g * kWoSlice * 2 + (c ^ ((t >> 1) | ((g & 1) << 1))) * 16);
      }
    __syncwarp();
  };

  // the activation ahead of the weight: behind the first tiles of all SMs it took 5600 cycles to arrive
  if (!kPasses) load_x(k_first);
#pragma unroll 1
  for (int i = 0; i < kWoStages; ++i) load();
  if (!kPasses) {
    convert_x();
    __syncthreads();  // the warps' sums take the activation's space
  }

  // lane (g, t) takes row (g >> 1) + 4 (g & 1) of eight, so that what eight lanes read at once lies in different banks
  // (and the second 128 elements' codes lie at the same offset ^ 64)
  const int my_row = (g >> 1) | ((g & 1) << 2);
  const uint32_t my_codes = codes + my_row * 128 + ((t ^ my_row) << 4);
  const uint32_t my_scales = scales + my_row * 16 + (t >> 1) * 128 + (t & 1) * 2;
  // A tile's sums: [column odd][row of the tile / 8][column / 2][row % 8], so that what a warp stores at once lies in different banks.
  const int pairs = (m + 1) >> 1, per_tile = 32 * pairs;
  const unsigned magic = a.per_tile_magic[blockIdx.z];
  int take = 0, flip = 0;
  for (int chunk = p0; chunk < p1; chunk += a.chunk, flip ^= 1) {
    const int end = min(chunk + a.chunk, p1);
    float *part = parts + flip * (a.parts_bytes / 8);
    for (int pass = 0; pass < (kPasses ? a.passes : 1); ++pass) {
      if (kPasses) {
        load_x(k_first + pass * k_pass);
        convert_x();
      }
      if (!works) continue;
      for (int pair = chunk + row_group; pair < end; pair += a.row_groups) {
        if ((phases & kWoLost) == 0 && !ptx::mbar_wait(bars + take, (phases >> take) & 1, gave_up)) {
          for (int i = 0; i < kWoStages; ++i) ptx::mbar_drain(bars + i, (phases >> i) & 1);
          *gave_up = 1;
          if (a.error_flag != nullptr) atomicExch(a.error_flag, kWeightOnlyTimeout);
          phases |= kWoLost;
        }
        __syncwarp();
        phases ^= 1u << take;
#pragma unroll 1
        for (int half = 2 * pair < j0 ? 1 : 0; half < (2 * pair + 1 < j1 ? 2 : 1); ++half) {
          const uint32_t at = take * kWoCodes + half * 2 * kWoBox, from_sf = my_scales + take * kWoScales + half * 8;
          float acc[4];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint32_t from = (my_codes ^ (b * 64)) + at;
            const uint4 w0 = wo_lds16(from), w1 = wo_lds16(from + kWoBox);
            // the scale factors of this lane's two groups of 16 elements, of both rows
            const __half2 s0 = e4m3x2_to_f16(wo_lds2(from_sf + b * 256)), s1 = e4m3x2_to_f16(wo_lds2(from_sf + b * 256 + 4));
            float d[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t h0[4], h1[4];
              e2m1_to_f16(q == 0 ? w0.x : q == 1 ? w0.y : q == 2 ? w0.z : w0.w, h0);
              e2m1_to_f16(q == 0 ? w1.x : q == 1 ? w1.y : q == 2 ? w1.z : w1.w, h1);
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                h0[c] = mul_f16x2(h0[c], q < 2 ? __low2half2(s0) : __high2half2(s0));
                h1[c] = mul_f16x2(h1[c], q < 2 ? __low2half2(s1) : __high2half2(s1));
              }
              if (q == 0)
                mma_f16_from0(d, h0[0], h1[0], h0[1], h1[1], x[b][q].x, x[b][q].y);
              else
                mma_f16(d, h0[0], h1[0], h0[1], h1[1], x[b][q].x, x[b][q].y);
              mma_f16(d, h0[2], h1[2], h0[3], h1[3], x[b][q].z, x[b][q].w);
            }
            const float2 f = *reinterpret_cast<const float2 *>(factors + b * 8 + 2 * t);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = b == 0 ? d[c] * (c & 1 ? f.y : f.x) : fmaf(d[c], c & 1 ? f.y : f.x, acc[c]);
          }
          if (t < pairs) {
            float *to = part + ((2 * (pair - chunk) + half) * a.slices + slice_in) * per_tile + t * 8 + my_row;
            const int step = pairs * 8;
            if (kPasses && pass > 0) acc[0] += to[0], acc[2] += to[step], acc[1] += to[2 * step], acc[3] += to[3 * step];
            to[0] = acc[0], to[step] = acc[2], to[2 * step] = acc[1], to[3 * step] = acc[3];
          }
          __syncwarp();  // the next products are the whole warp's; and the stage is free
        }
        take ^= 1;
        load();
      }
    }
    __syncthreads();
    // from the first to the last of the chunk's tiles
    const int first = (max(2 * chunk, j0) - 2 * chunk) * per_tile / 4, count = (min(2 * end, j1) - 2 * chunk) * per_tile / 4;
    float4 *sum_of = reinterpret_cast<float4 *>(sums + flip * (kWoSums / 4));
    const bool lost = *gave_up != 0;  // a warp of this CTA had no weight to multiply
    // four rows of a column at a time
    auto add = [](float4 &y, const float4 &v) { y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w; };
    auto finish = [&](int i, float4 y) {
      const int tile = (int)__umulhi((unsigned)i * 4, magic), rest = i * 4 - tile * per_tile;
      const int pair = rest >> 3, v = (pair >= pairs) + (pair >= 2 * pairs) + (pair >= 3 * pairs);
      const int col = 2 * (pair - v * pairs) + (v >> 1), row = tile_row(2 * chunk + tile) + (v & 1) * 32 + (rest & 7);
      if (row >= a.n || col >= m) return;
      __nv_bfloat16 *to = a.y + (long long)(row_first + col) * a.n + row;
      if (a.by_four) {
        if (a.bias != nullptr) {
          const uint2 w = *reinterpret_cast<const uint2 *>(a.bias + row);
          add(y, make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u)));
        }
        const __nv_bfloat162 lo = __floats2bfloat162_rn(y.x, y.y), hi = __floats2bfloat162_rn(y.z, y.w);
        *reinterpret_cast<uint2 *>(to) = make_uint2(*reinterpret_cast<const uint32_t *>(&lo), *reinterpret_cast<const uint32_t *>(&hi));
      } else {
        const float of_row[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (row + j < a.n) to[j] = __float2bfloat16_rn(of_row[j] + (a.bias != nullptr ? __bfloat162float(a.bias[row + j]) : 0.0f));
      }
    };
    for (int i = first + threadIdx.x; i < count; i += kWoThreads) {
      const int tile = (int)__umulhi((unsigned)i * 4, magic);
      const float4 *from = reinterpret_cast<const float4 *>(part + tile * (a.slices - 1) * per_tile) + i;  // tile * slices * per_tile + rest
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int s0 = 0; s0 < kWoWarps; s0 += 8) {
        float4 v[8];  // all loads, then the sum
#pragma unroll
        for (int s = 0; s < 8; ++s) v[s] = s0 + s < a.slices ? from[(s0 + s) * (per_tile >> 2)] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int s = 0; s < 8; ++s) add(y, v[s]);
      }
      if (lost) y.x = y.y = y.z = y.w = __int_as_float(0x7fffffff);
      if (a.cluster == 1)
        finish(i, y);
      else
        sum_of[i] = y;
    }
    if (a.cluster > 1) {
      __syncwarp();
      ptx::cluster_sync();
      for (int i = first + blockIdx.x * kWoThreads + threadIdx.x; i < count; i += a.cluster * kWoThreads) {
        float4 v[kWoClusterMost], y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int r = 0; r < kWoClusterMost; ++r)
          v[r] = r < a.cluster ? ptx::ld_cluster_f32x4(ptx::smem_u32(sum_of + i), r) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int r = 0; r < kWoClusterMost; ++r) add(y, v[r]);
        finish(i, y);
      }
    }
  }
  __syncwarp();
  if (a.cluster > 1) ptx::cluster_sync();  // a CTA's memory is read until here
}

int wo_sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0 && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 148;
  return sms[dev];
}

// Clusters of `size` CTAs that run at once, one CTA per SM: fewer than SMs / size, since a cluster lies within a GPC.
template <typename Kernel>
cudaError_t wo_clusters(Kernel kernel, int size, int *clusters) {
  static int known[64][kWoClusterMost + 1] = {};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  if (size == 1 || dev < 0 || dev >= 64) {
    *clusters = wo_sm_count() / size;
    return cudaSuccess;
  }
  int &of = known[dev][size];
  if (of == 0) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)size);
    cfg.blockDim = dim3(kWoThreads);
    cfg.dynamicSmemBytes = kWoSmem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int n = 0;
    err = cudaOccupancyMaxActiveClusters(&n, kernel, &cfg);
    if (err != cudaSuccess) return err;
    of = n > 0 ? n : 1;
  }
  *clusters = of;
  return cudaSuccess;
}

}  // namespace

cudaError_t run_weight_only(const void *x, long long x_row, int m, int n, int k, const void *qw, const void *sf, const float *scale_dev,
                            float scale, const void *bias, void *y, int *error_flag, cudaStream_t stream) {
  if (m < 1 || m > kWeightOnlyMaxRows || n < 1 || k < 64 || k % 64 != 0) return cudaErrorInvalidValue;
  WeightOnlyArgs a;
  a.x = static_cast<const __nv_bfloat16 *>(x);
  a.x_row = x_row;
  a.error_flag = error_flag;
  a.scale_dev = scale_dev;
  a.scale = scale;
  a.bias = static_cast<const __nv_bfloat16 *>(bias);
  a.y = static_cast<__nv_bfloat16 *>(y);
  a.m = m;
  a.n = n;
  a.k = k;
  const int slices = (k - 1) / kWoSlice + 1;
  a.cluster = (slices + kWoWarps - 1) / kWoWarps;
  if (a.cluster > kWoClusterMost) a.cluster = kWoClusterMost;
  a.passes = (slices + a.cluster * kWoWarps - 1) / (a.cluster * kWoWarps);
  const int rows = m > 8 ? 8 : m, per_tile = 32 * ((rows + 1) / 2);  // floats
  while (a.passes > 1 && (slices + a.cluster * a.passes - 1) / (a.cluster * a.passes) * per_tile * 4 * 4 > ((kWoParts - kWoWarps * kWoXWarp) & ~31)) ++a.passes;
  a.slices = (slices + a.cluster * a.passes - 1) / (a.cluster * a.passes);
  a.row_groups = a.passes == 1 ? kWoWarps / a.slices : 1;
  const int left = n % 128;  // a last block of few rows has empty tiles at its end
  a.tiles = n / 128 * 8 + (left == 0 ? 0 : left > 64 ? 8 : left >= 32 ? 7 : 2 * ((left + 7) / 8) - 1);
  const auto kernel = a.passes > 1 ? weight_only_kernel<true> : weight_only_kernel<false>;
  static bool ready[2][64] = {};
  cudaError_t err = allow_smem(kernel, kWoSmem, ready[a.passes > 1]);
  if (err != cudaSuccess) return err;
  int clusters = 0;
  err = wo_clusters(kernel, a.cluster, &clusters);
  if (err != cudaSuccess) return err;
  // more than eight rows: half of the clusters for each eight, side by side, so that the second to read a row of the weight finds it in L2
  const int eights = m > 8 ? 2 : 1;
  clusters = clusters / eights > 0 ? clusters / eights : 1;
  a.per_cluster = (a.tiles + clusters - 1) / clusters;
  a.parts_at = a.passes == 1 ? 0 : kWoWarps * kWoXWarp;
  a.parts_bytes = (kWoParts - a.parts_at) & ~31;  // two halves of float4s
  // all tiles at once, or half of the space at a time; at most as many as the sums of a cluster's CTAs have room for; in pairs
  const int tile_bytes = a.slices * per_tile * 4, all = (a.per_cluster + 1) / 2, of_sums = kWoSums / (per_tile * 8);
  a.chunk = all;
  if (2 * all * tile_bytes > a.parts_bytes || (a.cluster > 1 && all > of_sums)) {
    a.chunk = a.parts_bytes / 2 / (2 * tile_bytes);
    if (a.cluster > 1 && a.chunk > of_sums) a.chunk = of_sums;
    if (a.chunk > a.row_groups) a.chunk -= a.chunk % a.row_groups;  // the pairs of a row group follow one another at equal distances
  }
  if (a.chunk < 1) return cudaErrorInvalidValue;
  if (a.row_groups > a.chunk) a.row_groups = a.chunk;
  for (int i = 0; i < eights; ++i) {
    const int floats = i == 0 ? per_tile : 32 * ((m - 8 + 1) / 2);
    a.per_tile_magic[i] = (unsigned)(((1ULL << 32) + floats - 1) / floats);
  }
  const int used = (a.tiles + a.per_cluster - 1) / a.per_cluster;
  a.whole = n / 128;
  a.by_four = n % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 7) == 0 && (reinterpret_cast<uintptr_t>(a.bias) & 7) == 0;
  CUtensorMap map_tiles, map_w, map_sf;
  // codes: 8 rows x 128 bytes at a time
  const cuuint64_t w_dims[2] = {(cuuint64_t)k / 2, (cuuint64_t)n}, w_strides[1] = {(cuuint64_t)k / 2};
  const cuuint32_t w_box[2] = {kWoSlice / 2, 8};
  // and, in whole blocks of 128 rows, a tile's 16 rows in one copy
  const cuuint64_t t_dims[4] = {(cuuint64_t)k / 2, 32, 4, (cuuint64_t)(a.whole > 0 ? a.whole : 1)};
  const cuuint64_t t_strides[3] = {(cuuint64_t)k / 2, (cuuint64_t)k / 2 * 32, (cuuint64_t)k / 2 * 128};
  const cuuint32_t t_box[4] = {kWoSlice / 2, 8, 2, 1};
  // scale factors: blocks of 128 rows, tiles of 64 elements, 8 rows x 16 bytes of 4 tiles at a time
  const cuuint64_t sf_dims[3] = {512, (cuuint64_t)k / 64, ((cuuint64_t)n + 127) / 128}, sf_strides[2] = {512, (cuuint64_t)k / 64 * 512};
  const cuuint32_t sf_box[3] = {128, kWoSlice / 64, 1};
  const CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B;
  if (!make_tensor_map(&map_tiles, 4, qw, t_dims, t_strides, t_box, swizzle) || !make_tensor_map(&map_w, 2, qw, w_dims, w_strides, w_box, swizzle) ||
      !make_tensor_map(&map_sf, 3, sf, sf_dims, sf_strides, sf_box, CU_TENSOR_MAP_SWIZZLE_NONE))
    return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)a.cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)a.cluster, (unsigned)used, (unsigned)eights);
  cfg.blockDim = dim3(kWoThreads);
  cfg.dynamicSmemBytes = kWoSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = a.cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, map_tiles, map_w, map_sf, a);
}

}  // namespace sharq
