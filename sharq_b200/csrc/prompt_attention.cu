// Attention of ragged prompts: causal, with a sliding window and a few first keys that stay visible.  32768 tokens of 32 / 8 heads of
// 128 under a window of 4096: 2.04 ms, 1010 TFLOP/s, in long runs, where the card's power is the bound (1.75 ms in a short one); 200 tokens: 11.3 us.
//
//   out[i, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[i, h] . k_j - max),   j <= p and (p - j < window or j < sinks),   p the position of query i
//
// Two products of 128 x 128 x head_dim per block of queries and tile of keys, on the tensor cores (tcgen05, bf16): S = Q K^T into tensor memory, the
// exponentials back into it as bf16 in the place of S, O += P V from there.  The exponentials take the
// special function unit as long as the products take the tensor cores (128 x 128: 1024 cycles of 16, and twice 512).
//
// A CTA works on two blocks of 128 query rows, so that one's exponentials run under the other's products, and goes from item to item by itself.  The
// query heads of a key/value head are rows of the same block, token after token (4 heads: 32 tokens of each): what a narrow window lets a
// block see is then as few tiles as can be.  The keys that a block may see are one list: the first ones, filled up to a multiple of 8, then those of the window
// from its first one on, which a tile in the middle joins by copies of 8 keys.
//
// Warps 0-3 and 4-7 hold a row per thread: maximum, exponentials and sum need no other thread.  The maximum is raised only where a score exceeds it by
// more than 2^kLazy, for the raise is a pass over O.  Probabilities carry a factor of 2^-32, so that no sum of finite values overflows, and
// enter the product as bf16, as in the library attention of prompts without a window: off by up to 2^-8 each, which leaves a result about as near as its own
// rounding to bf16.  (As two bf16 numbers, as the decode step has them, the second product would be a third more work for the tensor cores.)  The factor takes five bits
// of the exponent's argument, 2^-18 of a probability, and the exponential is the hardware's, to 2 units in the last place of a float: both are far below that.
// The second product begins when three quarters of a tile's probabilities are there.  All 128 scores of a row stay in registers, for reading tensor memory
// again took longer than the exponentials (2726 us instead of then 2085; 32 at a time with the maximum beside the exponentials 2179; a row in two threads,
// which have to meet twice, 2824).  Exponentials by a polynomial on the units that multiply, for an eighth to a half of them, 2124 to 2473: a warp's instructions
// follow one another too slowly for more of them to pay, and each takes power.
//
// Items go in turns over the CTAs, or, few ones with many tiles, in equal stretches of the list of all tiles, whose ends cut items into parts that a second kernel joins.
//
// A masked key has probability 0, which a value that is not finite (another sequence's, or memory that nothing has written) would turn to NaN.  Two
// warps look for such values in every tile where something is masked; a tile that has one is multiplied row by row, visible keys only, in plain float.
#include <cuda.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "decode_ops.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.cuh"

namespace sharq {

namespace {

constexpr int kTile = 128;  // keys of a tile, rows of a block
constexpr int kBlocks = 2;
constexpr int kSoftmaxWarps = 4 * kBlocks, kLoadWarp = kSoftmaxWarps, kMmaWarp = kLoadWarp + 1, kCheckWarp = kMmaWarp + 1, kCheckWarps = 2;
constexpr int kThreads = 32 * (kCheckWarp + kCheckWarps);
constexpr int kItemSlots = 2;
constexpr int kSoftmaxRegisters = 208, kOtherRegisters = 88;
static_assert(128 * kBlocks * kSoftmaxRegisters + 128 * kOtherRegisters <= kThreads * 168, "the shares of the registers that the block was launched with");
constexpr int kFirst = 96;  // keys whose product does not wait for the others' probabilities
constexpr float kLazy = 8.0f, kLift = -32.0f;  // in powers of two

// As ptx::mbar_wait, but the thread sleeps up to some microseconds between looks (or until the phase ends): waiting warps took 3 % of the rate, long runs of which
// are bound by the card's power.
__device__ __forceinline__ bool look(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(ok)
      : "r"(ptx::smem_u32(bar)), "r"(parity), "r"(4000)
      : "memory");
  return ok != 0;
}
// sooner: by how many cycles a wait ends ahead of the usual limit.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, volatile int *abort_flag, long long sooner) {
  if (look(bar, parity)) return true;
  const long long start = clock64();
  while (true) {
    if (look(bar, parity)) return true;
    if (*abort_flag != 0) return false;
    if (clock64() - start > ptx::kWaitLimitCycles - sooner) return false;
  }
}

template <int D>
struct Sizes {
  static constexpr int kHalves = D / 64;           // rows lie 128 bytes apart: a row of 256 bytes in two halves
  static constexpr int kHalf = kTile * 128;
  static constexpr int kBytes = kHalf * kHalves;   // of a tile, or of a block of queries
  static constexpr int kStages = D == 128 ? 5 : 9;
  static constexpr int kControl = kBlocks * kBytes + kStages * kBytes;
  static constexpr int kTotal = kControl + 1024;
  static constexpr int kOutCol = kBlocks * kTile;  // tensor memory: scores of the blocks, then their outputs
};
static_assert(Sizes<128>::kTotal <= 232448 && Sizes<64>::kTotal <= 232448, "shared memory of a CTA");

struct Args {
  const int *offsets, *k_offsets;
  __nv_bfloat16 *out;
  int rows, k_rows, seqs;
  int heads, kv_heads, group, chunks, chunk_heads, tokens;  // chunk_heads: query heads of a block; tokens: of a block
  int span;           // tokens of an item: of one block or two
  int window, sinks;  // window: 2^30 for none
  float scale_log2;   // scale * log2(e)
  bool fill;          // rows of no sequence become zeros
  bool wide;          // out begins at a multiple of 32 bytes
  bool split;         // items are cut where the CTAs' equal stretches of the list end
  float *parts;       // split: [2 * CTAs][kBlocks][kTile][head_dim] sums of probabilities times values, then [2 * CTAs][kBlocks][kTile] of their [maximum, sum]
  int4 *joins;        // split: [CTAs][2] of the item that begins in a CTA's stretch and goes on: {row0, count, first, column}, {parts (0: none), ...}
  long long sooner;   // see wait_for
  int *error_flag;
};
constexpr int kItemCost = 3;      // of an item in the list, in tiles, for its queries and its result
constexpr int kStretchLeast = 8;  // units of a CTA

// What a CTA works on: `count` tokens from row `row0` on, the first at position `first`, of heads kv and chunk.  Their keys are a list of `s_pad` first ones
// and those from position `base` on, of which there are `total` in all, in `tiles` tiles; the CTA takes those from `begin` to `end`.
struct Item {
  int state;  // 0: no more items, 1: an item, 2: one whose keys are not known (its rows come out as NaN)
  int row0, count, first, kv, chunk;
  int k_row0, base, s_pad, total, tiles;
  int begin, end, place;  // place: of the part that it leaves, -1 where it has all tiles
};

__device__ __forceinline__ void set_keys(Item &it, int keys, int window, int sinks) {
  const int last = it.first + it.count - 1, end = min(last + 1, keys);  // last < keys
  if (end <= 0) {
    it.base = it.s_pad = it.total = it.tiles = 0;
    return;
  }
  const int low = max(0, it.first - window + 1), s = min(sinks, end), pad = (s + 7) & ~7;
  it.base = low;
  it.s_pad = 0;
  if (s > 0) {
    if (low > pad)
      it.s_pad = pad;
    else
      it.base = 0;
  }
  it.total = it.s_pad + end - it.base;
  it.tiles = (it.total + kTile - 1) / kTile;
}

// Whether some query of the item does not see some key of the tile.
__device__ __forceinline__ bool is_masked(const Item &it, int tile, int window, int sinks) {
  const int v0 = tile * kTile, v1 = v0 + kTile - 1;
  if (v0 < it.s_pad) return v1 >= sinks;
  const int k0 = it.base + v0 - it.s_pad, k1 = k0 + kTile - 1, last = it.first + it.count - 1;
  return k1 > it.first || !(k0 > last - window || k1 < sinks);
}

// Which keys of the list a query sees: [low, high) and those below `sinks`.
struct Seen {
  int low, high, sinks;
};
__device__ __forceinline__ Seen seen_by(const Item &it, int position, int window, int sinks) {
  return {it.s_pad + max(position - window + 1 - it.base, 0), it.s_pad + position + 1 - it.base, max(0, min(sinks, position + 1))};
}
__device__ __forceinline__ unsigned bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1; }
__device__ __forceinline__ unsigned seen_word(const Seen &s, int v0) {  // of the keys v0 .. v0 + 31
  return (bits_below(s.high - v0) & ~bits_below(s.low - v0)) | bits_below(s.sinks - v0);
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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// pairs of floats in a register pair each
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float *a, float *b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
  return v;
}

__device__ __forceinline__ void st_global32(void *to, const uint32_t *w) {  // 32 bytes at a multiple of 32
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
               "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x4(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr)
               : "memory");
}

// bf16 operands, float sums; A and B in shared memory, both with K contiguous (B: with N contiguous, kind::f16's transposed form), or A in tensor memory
template <int N, bool kTransposeB>
__device__ __forceinline__ constexpr uint32_t make_idesc_bf16() {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((kTransposeB ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// a box of a map that encode() made, from the beginning of its 128-byte rows on
__device__ __forceinline__ void copy_4d(uint32_t dst, const CUtensorMap *m, int c1, int c2, int c3, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(m), "r"(ptx::smem_u32(bar)), "r"(0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// O of a thread's row += P V of a tile whose values are not all finite, visible keys only.  s: the row's, from the tile's first key on; first_tile: O holds nothing yet.
template <int D>
__device__ __noinline__ void multiply_visible(uint32_t tmem_p, uint32_t tmem_o, uint32_t values, Seen s, bool first_tile) {
  for (int c = 0; c < D; c += 32) {
    uint32_t o[32];
    if (first_tile) {
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0;
    } else {
      ptx::tmem_ld_32x32b_x32(tmem_o + c, o);
      ptx::tmem_ld_wait();
    }
    for (int k0 = 0; k0 < kTile; k0 += 8) {
      uint32_t p[4];
      tmem_ld_x4(tmem_p + k0 / 2, p);
      ptx::tmem_ld_wait();
      const unsigned word = seen_word(s, k0);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float pk = __uint_as_float(k % 2 == 0 ? p[k / 2] << 16 : p[k / 2] & 0xFFFF0000u);
        const uint32_t row = values + (c / 64) * Sizes<D>::kHalf + (k0 + k) * 128;
#pragma unroll
        for (int piece = 0; piece < 4; ++piece) {
          const float4 v = ptx::ld_shared_f32x4(row + (((c % 64) / 8 + piece) ^ k) * 16);  // swizzled by the row in eight
          const float w[4] = {v.x, v.y, v.z, v.w};
          if ((word >> k & 1) != 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t bits = __float_as_uint(w[i]);
              uint32_t &lo = o[piece * 8 + 2 * i], &hi = o[piece * 8 + 2 * i + 1];
              lo = __float_as_uint(fmaf(pk, __uint_as_float(bits << 16), __uint_as_float(lo)));
              hi = __float_as_uint(fmaf(pk, __uint_as_float(bits & 0xFFFF0000u), __uint_as_float(hi)));
            }
          }
        }
        __syncwarp();
      }
    }
    tmem_st_x32(tmem_o + c, o);
    tmem_st_wait();
  }
}


// Rows of the sequences seq0 + lane, all lanes: empty behind the last one, and where offsets go back, below an earlier one (`reached`: the highest
// so far), or leave the rows.
struct Bounds {
  int row0, row1;
  bool bad;
};
__device__ __forceinline__ Bounds bounds_of(const Args &a, int seq0, int lane, int *reached) {
  const int seq = seq0 + lane;
  Bounds b = {0, 0, false};
  if (seq < a.seqs) b.row0 = a.offsets[seq], b.row1 = a.offsets[seq + 1];
  int top = seq < a.seqs && b.row0 <= a.rows ? b.row0 : -1;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, top, off);
    if (lane >= off) top = max(top, up);
  }
  top = max(top, *reached);
  *reached = __shfl_sync(0xffffffffu, top, 31);
  b.bad = seq < a.seqs && !(b.row0 >= 0 && b.row0 >= top && b.row0 <= b.row1 && b.row1 <= a.rows);
  if (b.bad) b.row0 = b.row1 = 0;
  return b;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                            const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k8,
                            const __grid_constant__ CUtensorMap map_v8, const __grid_constant__ Args a) {
  using S = Sizes<D>;
  constexpr int kStages = S::kStages;
  extern __shared__ __align__(1024) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t queries = ptx::smem_u32(smem), ring = queries + kBlocks * S::kBytes;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kControl);
  uint64_t *kv_full = bars, *kv_empty = kv_full + kStages, *v_ok = kv_empty + kStages, *q_full = v_ok + kStages, *q_empty = q_full + kBlocks;
  uint64_t *s_full = q_empty + kBlocks, *p_first = s_full + kBlocks, *p_full = p_first + kBlocks, *o_full = p_full + kBlocks, *item_full = o_full + kBlocks;
  uint64_t *item_empty = item_full + kItemSlots;
  uint64_t *drained = item_empty + kItemSlots;  // for products on their way when a wait ran out
  Item *items = reinterpret_cast<Item *>(drained + 1);
  volatile int *not_finite = reinterpret_cast<volatile int *>(items + kItemSlots);  // [kStages][kCheckWarps]
  volatile int *abort_flag = not_finite + kStages * kCheckWarps;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(const_cast<int *>(abort_flag) + 1);
  unsigned *issued = tmem_slot + 1;  // copies of tiles, and of each block's queries: left here by the load warp when it has ended
  bool multiplies = false;           // the thread that issues products

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      ptx::mbar_init(kv_full + i, 1);
      ptx::mbar_init(kv_empty + i, 1);
      ptx::mbar_init(v_ok + i, kCheckWarps);
    }
    for (int i = 0; i < kBlocks; ++i) {
      ptx::mbar_init(q_full + i, 1);
      ptx::mbar_init(q_empty + i, 1);
      ptx::mbar_init(s_full + i, 1);
      ptx::mbar_init(p_first + i, 4);
      ptx::mbar_init(p_full + i, 4);
      ptx::mbar_init(o_full + i, 1);
    }
    for (int i = 0; i < kItemSlots; ++i) {
      ptx::mbar_init(item_full + i, 1);
      ptx::mbar_init(item_empty + i, kSoftmaxWarps + 1 + kCheckWarps);
    }
    ptx::mbar_init(drained, 1);
    ptx::fence_barrier_init();
    *abort_flag = 0;
    ptx::tma_prefetch_desc(&map_q);
    ptx::tma_prefetch_desc(&map_k);
    ptx::tma_prefetch_desc(&map_v);
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc<1>(tmem_slot, 512);
    ptx::tmem_relinquish<1>();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  ptx::grid_dependency_wait();

  auto give_up = [&]() {
    *abort_flag = 1;
    if (a.error_flag != nullptr) atomicExch(a.error_flag, kPromptTimeout);
  };
  // whether there is another item, whose description the load warp has left in items[n % kItemSlots]; `n`: how many there have been
  auto next_item = [&](int n) {
    const int slot = n % kItemSlots;
    if (!wait_for(item_full + slot, (n / kItemSlots) & 1, abort_flag, a.sooner)) {
      give_up();
      return false;
    }
    return items[slot].state != 0;
  };
  auto next_item_of_warp = [&](int n) {  // all lanes, which have the same answer
    const bool got = next_item(n);
    __syncwarp();
    return (bool)__all_sync(0xffffffffu, got);
  };
  auto leave_item = [&](int n) {  // the warp has read what it needs of the description
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(item_empty + n % kItemSlots);
  };

  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegisters));
    const int block = warp / 4, row = (warp % 4) * 32 + lane;
    const int token = row / a.chunk_heads, head = row % a.chunk_heads;
    const uint32_t lanes = tmem + ((uint32_t)(warp % 4) << 21);  // 32 lanes of tensor memory per warp
    const uint32_t tmem_s = lanes + block * kTile, tmem_o = lanes + S::kOutCol + block * D;
    const bool negative = a.scale_log2 < 0.0f;
    const float c = fabsf(a.scale_log2) < 1.2e-38f ? 1.2e-38f : fabsf(a.scale_log2);  // not 0: masked scores are -inf, and stay so; NaN is NaN
    if (a.fill) {  // rows of no sequence become zeros, a share of them per thread
      const long long width = (long long)a.heads * D / 8;
      auto clear = [&](int from, int to) {
        uint4 *out = reinterpret_cast<uint4 *>(a.out);
        for (long long i = from * width + (long long)blockIdx.x * (32 * kSoftmaxWarps) + threadIdx.x; i < to * width; i += (long long)gridDim.x * (32 * kSoftmaxWarps))
          out[i] = make_uint4(0, 0, 0, 0);
      };
      bool wrong = false;
      for (int i = lane; i <= a.seqs; i += 32) wrong |= a.offsets[i] < (i > 0 ? a.offsets[i - 1] : 0) || a.offsets[i] > a.rows;
      if (!__any_sync(0xffffffffu, wrong)) {
        clear(0, a.offsets[0]);
        clear(a.offsets[a.seqs], a.rows);
      } else {  // also those between the sequences that have rows, which lie in ascending order
        int reached = 0, covered = 0;
        for (int b0 = 0; b0 < a.seqs; b0 += 32) {
          const Bounds b = bounds_of(a, b0, lane, &reached);
          for (unsigned left = __ballot_sync(0xffffffffu, b.row1 > b.row0); left != 0; left &= left - 1) {
            const int in = __ffs(left) - 1, row0 = __shfl_sync(0xffffffffu, b.row0, in);
            clear(covered, row0);
            __syncwarp();
            covered = __shfl_sync(0xffffffffu, b.row1, in);
          }
        }
        clear(covered, a.rows);
      }
      __syncwarp();
    }
    unsigned tiles_done = 0, values_done = 0, items_done = 0;  // for the barriers' parities: of this block, of all, of this block
    bool ok = true;
    for (int n = 0; ok && next_item_of_warp(n); values_done += items[n % kItemSlots].end - items[n % kItemSlots].begin, leave_item(n), ++n) {
      const Item &it = items[n % kItemSlots];  // stays in shared memory, for want of registers
      if (it.count <= block * a.tokens) continue;  // nothing for this block
      const int position = it.first + min(block * a.tokens + token, it.count - 1);
      const Seen seen = seen_by(it, position, a.window, a.sinks);
      float m = -INFINITY, l = 0.0f;  // maximum in powers of two, sum
      for (int tile = it.begin; tile < it.end; ++tile) {
        if (!wait_for(s_full + block, tiles_done++ & 1, abort_flag, a.sooner)) {
          give_up();
          ok = false;
        }
        __syncwarp();
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ptx::tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) ptx::tmem_ld_32x32b_x32(tmem_s + 32 * i, s[i]);
        ptx::tmem_ld_wait();
        if (negative) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 32; ++j) s[i][j] ^= 0x80000000u;
        }
        const bool masked = is_masked(it, tile, a.window, a.sinks);
        if (masked) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned word = seen_word(seen, tile * kTile + 32 * i);
#pragma unroll
            for (int j = 0; j < 32; ++j) s[i][j] = (word >> j & 1) != 0 ? s[i][j] : 0xff800000u;
          }
        }
        float top[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          top[i] = fmaxf(__uint_as_float(s[i][0]), __uint_as_float(s[i][1]));
#pragma unroll
          for (int j = 2; j < 32; j += 2) top[i] = max3(top[i], __uint_as_float(s[i][j]), __uint_as_float(s[i][j + 1]));
        }
        const float high = max3(fmaxf(top[0], top[1]), top[2], top[3]) * c;
        const bool raise = high > m + kLazy;
        if (__any_sync(0xffffffffu, raise)) {
          const float f = raise ? exp2_approx(m - high) : 1.0f;  // from -inf: 0, and nothing to keep
          if (raise) m = high;
          l *= f;
          if (tile > it.begin) {
#pragma unroll 1
            for (int i = 0; i < D; i += 16) {
              uint32_t o[16];
              tmem_ld_x16(tmem_o + i, o);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st_x16(tmem_o + i, o);
            }
          }
        }
        // a row with no finite score so far has maximum -inf: its probabilities are 0, not exp(-inf + inf)
        const float base = (m == -INFINITY ? 0.0f : m) - kLift;
        const uint64_t c2 = pair(c, c), base2 = pair(-base, -base);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t p[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x, y;
            unpair(fma_pair(pair(__uint_as_float(s[i][2 * j]), __uint_as_float(s[i][2 * j + 1])), c2, base2), &x, &y);
            x = exp2_approx(x);
            y = exp2_approx(y);
            sum[j & 1] = add_pair(sum[j & 1], pair(x, y));
            p[j] = pack_bf16(x, y);
          }
          tmem_st_x16(tmem_s + 16 * i, p);
          if (i == kFirst / 32 - 1) {  // the product may begin with the keys so far
            tmem_st_wait();
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(p_first + block);
          }
        }
        float sums[4];
        unpair(sum[0], &sums[0], &sums[1]);
        unpair(sum[1], &sums[2], &sums[3]);
        l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        tmem_st_wait();
        if (masked) {
          const unsigned value = values_done + tile - it.begin;
          if (!wait_for(v_ok + value % kStages, (value / kStages) & 1, abort_flag, a.sooner)) {
            give_up();
            ok = false;
          }
          __syncwarp();
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if ((not_finite[value % kStages * kCheckWarps] | not_finite[value % kStages * kCheckWarps + 1]) != 0)
            multiply_visible<D>(tmem_s, tmem_o, ring + (2 * value + 1) % kStages * S::kBytes,
                                Seen{seen.low - tile * kTile, seen.high - tile * kTile, seen.sinks - tile * kTile}, tile == it.begin);
        }
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_full + block);
      }
      if (!ok) break;
      const int t = block * a.tokens + token, tiles = it.end - it.begin, state = it.state;
      const bool there = token < a.tokens && t < it.count && it.chunk * a.chunk_heads + head < a.group;
      if (tiles > 0) {
        if (!wait_for(o_full + block, items_done++ & 1, abort_flag, a.sooner)) {
          give_up();
          ok = false;
        }
        __syncwarp();
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        ptx::tc_fence_after();
      }
      if (it.place >= 0) {  // a part, to be joined with those of other CTAs
        const long long at = ((long long)it.place * kBlocks + block) * kTile + row;
        float *part = a.parts + at * D;
#pragma unroll 1
        for (int i = 0; i < D; i += 32) {
          uint32_t o[32];
          ptx::tmem_ld_32x32b_x32(tmem_o + i, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 32; j += 8) st_global32(part + i + j, &o[j]);
        }
        reinterpret_cast<float2 *>(a.parts + 2LL * gridDim.x * kBlocks * kTile * D)[at] = make_float2(m, l);
        ptx::tc_fence_before();
        continue;
      }
      __nv_bfloat16 *out = a.out + ((long long)(it.row0 + t) * a.heads + it.kv * a.group + it.chunk * a.chunk_heads + head) * D;
      const float f = 1.0f / l;
#pragma unroll 1
      for (int i = 0; i < D; i += 32) {
        uint32_t o[32];
        if (tiles > 0) {
          ptx::tmem_ld_32x32b_x32(tmem_o + i, o);
          ptx::tmem_ld_wait();
        }
#pragma unroll
        for (int j = 0; j < 32; j += 16) {
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            w[e] = pack_bf16(__uint_as_float(o[j + 2 * e]) * f, __uint_as_float(o[j + 2 * e + 1]) * f);
            if (position < 0 || tiles == 0) w[e] = 0;
            if (state == 2) w[e] = 0x7fff7fffu;
          }
          if (there && a.wide) {
            st_global32(out + i + j, w);
          } else if (there) {
            *reinterpret_cast<uint4 *>(out + i + j) = make_uint4(w[0], w[1], w[2], w[3]);
            *reinterpret_cast<uint4 *>(out + i + j + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
        __syncwarp();
      }
      ptx::tc_fence_before();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == kLoadWarp) {
      // blocks of two times `tokens` tokens, of all sequences, times heads: the list of items
      const int span = a.span, columns = a.kv_heads * a.chunks;
      bool bad = false;
      // the block `index` of rows [from, to) with keys [k0, k1)
      auto describe = [&](Item &it, int from, int to, int k0, int k1, int index) {
        const bool known = k0 >= 0 && k0 <= k1 && k1 <= a.k_rows;
        it.state = known ? 1 : 2;
        it.row0 = from + index * span;
        it.count = min(span, to - it.row0);
        it.k_row0 = k0;
        it.first = (k1 - k0) - (to - from) + index * span;
        set_keys(it, k1 - k0, a.window, a.sinks);
        if (!known) it.tiles = 0;
        it.begin = 0;
        it.end = it.tiles;
        it.place = -1;
      };
      auto keys_of = [&](int seq0, const Bounds &b) {  // of the lane's sequence
        const bool given = a.k_offsets != nullptr && seq0 + lane < a.seqs;
        return given ? make_int2(a.k_offsets[seq0 + lane], a.k_offsets[seq0 + lane + 1]) : make_int2(b.row0, b.row1);
      };
      int blocks = 0, reached = 0;
      for (int b0 = 0; b0 < a.seqs; b0 += 32) {
        const Bounds b = bounds_of(a, b0, lane, &reached);
        bad |= b.bad;
        blocks += (b.row1 - b.row0 + span - 1) / span;
      }
      blocks = __reduce_add_sync(0xffffffffu, blocks);
      // Whole items: CTAs take turns.  The last block of a sequence first: it sees most.
      long long turn = blockIdx.x;
      int b_now = 0, before_now = 0, reached_now = 0;  // of the 32 sequences that the last item was found among: later ones lie there or behind
      auto next_whole = [&](Item &it) {
        it.state = 0;
        const long long at = turn;
        turn += gridDim.x;
        if (at >= (long long)blocks * columns) return;
        const int block = (int)(at / columns), column = (int)(at - (long long)block * columns);
        it.kv = column / a.chunks;
        it.chunk = column - it.kv * a.chunks;
        int before = before_now;
        reached = reached_now;
        for (int b0 = b_now; b0 < a.seqs; b0 += 32) {
          const int ahead = reached;
          const Bounds b = bounds_of(a, b0, lane, &reached);
          int ends = (b.row1 - b.row0 + span - 1) / span;
#pragma unroll
          for (int off = 1; off < 32; off <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, ends, off);
            if (lane >= off) ends += up;
          }
          const unsigned over = __ballot_sync(0xffffffffu, before + ends > block);
          if (over != 0) {
            b_now = b0;
            before_now = before;
            reached_now = ahead;
            const int in = __ffs(over) - 1;
            const int2 k = keys_of(b0, b);
            describe(it, __shfl_sync(0xffffffffu, b.row0, in), __shfl_sync(0xffffffffu, b.row1, in), __shfl_sync(0xffffffffu, k.x, in),
                     __shfl_sync(0xffffffffu, k.y, in), before + __shfl_sync(0xffffffffu, ends, in) - 1 - block);
            return;
          }
          before += __shfl_sync(0xffffffffu, ends, 31);
        }
      };
      // Split: the list in units, kItemCost and an item's tiles each.  Finds the item that unit u belongs to -> where it begins; or, u < 0, the list's length.
      auto find = [&](Item &it, long long u) {
        long long before = 0;
        reached = 0;
        for (int b0 = 0; b0 < a.seqs; b0 += 32) {
          const Bounds b = bounds_of(a, b0, lane, &reached);
          const int2 k = keys_of(b0, b);
          for (int in = 0; in < min(32, a.seqs - b0); ++in) {
            const int from = __shfl_sync(0xffffffffu, b.row0, in), to = __shfl_sync(0xffffffffu, b.row1, in);
            const int k0 = __shfl_sync(0xffffffffu, k.x, in), k1 = __shfl_sync(0xffffffffu, k.y, in), count = (to - from + span - 1) / span;
            for (int i0 = 0; i0 < count; i0 += 32) {
              long long units = 0;
              if (i0 + lane < count) {
                describe(it, from, to, k0, k1, i0 + lane);
                units = (long long)(kItemCost + max(it.tiles, 1)) * columns;
              }
              long long ends = units;
#pragma unroll
              for (int off = 1; off < 32; off <<= 1) {
                const long long up = __shfl_up_sync(0xffffffffu, ends, off);
                if (lane >= off) ends += up;
              }
              const unsigned over = __ballot_sync(0xffffffffu, u >= 0 && before + ends > u);
              if (over != 0) {
                const int of = __ffs(over) - 1;
                const long long start = before + __shfl_sync(0xffffffffu, ends - units, of);
                describe(it, from, to, k0, k1, i0 + of);
                const int cost = kItemCost + max(it.tiles, 1), column = (int)((u - start) / cost);
                it.kv = column / a.chunks;
                it.chunk = column - it.kv * a.chunks;
                return start + (long long)column * cost;
              }
              before += __shfl_sync(0xffffffffu, ends, 31);
            }
          }
        }
        return before;
      };
      long long unit = 0, unit_end = 0, per = 0;
      if (a.split) {
        Item it;
        const long long total = find(it, -1);
        per = max((long long)kStretchLeast, (total + gridDim.x - 1) / gridDim.x);
        unit = min(total, blockIdx.x * per);
        unit_end = min(total, unit + per);
        if (lane < 2) a.joins[2 * blockIdx.x + lane] = make_int4(0, 0, 0, 0);
        __syncwarp();
      }
      auto next_part = [&](Item &it) {
        while (unit < unit_end) {
          const long long start = find(it, unit);
          const int tiles = max(it.tiles, 1), skip = (int)(unit - start), left = (int)(unit_end - unit);
          const int begin = max(0, skip - kItemCost), end = min(tiles, skip + left - kItemCost);
          unit = start + kItemCost + tiles;
          if (begin >= end) continue;
          if (begin > 0 || end < tiles) {
            it.begin = begin;
            it.end = end;
            it.place = 2 * blockIdx.x + (begin == 0 ? 1 : 0);
            if (begin == 0 && lane == 0) {
              a.joins[2 * blockIdx.x] = make_int4(it.row0, it.count, it.first, it.kv * a.chunks + it.chunk);
              a.joins[2 * blockIdx.x + 1] = make_int4(1 + (int)((tiles - end + per - 1) / per), 0, 0, 0);
            }
          }
          return;
        }
        it.state = 0;
      };
      unsigned copies = 0, loads[kBlocks] = {0, 0};
      bool ok = true;
      for (int n = 0; ok; ++n) {
        Item it;
        if (a.split)
          next_part(it);
        else
          next_whole(it);
        bad |= it.state == 2;
        const int slot = n % kItemSlots;
        if (lane == 0) {
          if (wait_for(item_empty + slot, ((n / kItemSlots) & 1) ^ 1, abort_flag, a.sooner)) {
            items[slot] = it;
            ptx::mbar_arrive(item_full + slot);
          } else {
            give_up();
            ok = false;
          }
          if (ok && it.state != 0 && it.end > it.begin) {
            auto fill = [&](int tile, bool of_keys) {
              const int stage = copies % kStages;
              if (!wait_for(kv_empty + stage, ((copies / kStages) & 1) ^ 1, abort_flag, a.sooner)) {
                give_up();
                ok = false;
                return;
              }
              const uint32_t to = ring + stage * S::kBytes;
              const int v0 = tile * kTile;
              ptx::mbar_arrive_expect_tx(kv_full + stage, S::kBytes);
              if (v0 + kTile <= it.s_pad || v0 >= it.s_pad) {
                const int key = v0 < it.s_pad ? v0 : it.base + v0 - it.s_pad;
                copy_4d(to, of_keys ? &map_k : &map_v, it.k_row0 + key, 0, it.kv, kv_full + stage);
              } else {  // the first keys end in this tile
                for (int i = 0; i < kTile; i += 8) {
                  const int key = v0 + i < it.s_pad ? v0 + i : it.base + v0 + i - it.s_pad;
                  for (int half = 0; half < S::kHalves; ++half)
                    copy_4d(to + half * S::kHalf + i * 128, of_keys ? &map_k8 : &map_v8, it.k_row0 + key, half, it.kv, kv_full + stage);
                }
              }
              ++copies;
            };
            for (int b = 0; b < kBlocks && ok; ++b) {
              if (it.count <= b * a.tokens) continue;
              if (!wait_for(q_empty + b, (loads[b] & 1) ^ 1, abort_flag, a.sooner)) {
                give_up();
                ok = false;
                break;
              }
              ++loads[b];
              ptx::mbar_arrive_expect_tx(q_full + b, a.tokens * a.chunk_heads * D * 2);
              for (int half = 0; half < S::kHalves; ++half)
                copy_4d(queries + b * S::kBytes + half * S::kHalf, &map_q, it.kv * a.group + it.chunk * a.chunk_heads, it.row0 + b * a.tokens, half,
                        q_full + b);
              if (b == 0) fill(it.begin, true);
            }
            for (int tile = it.begin; tile < it.end && ok; ++tile) {
              if (tile > it.begin) fill(tile, true);
              if (ok) fill(tile, false);
            }
          }
        }
        __syncwarp();
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (it.state == 0) break;
      }
      if (__any_sync(0xffffffffu, bad) && lane == 0 && a.error_flag != nullptr) atomicCAS(a.error_flag, 0, kBadOffsets);
      if (lane == 0) issued[0] = copies, issued[1] = loads[0], issued[2] = loads[1];
    } else if (warp == kMmaWarp) {
      multiplies = ptx::elect_one();
      if (multiplies) {
        constexpr uint32_t kScores = make_idesc_bf16<kTile, false>(), kOutputs = make_idesc_bf16<D, true>();
        unsigned copies = 0, values = 0, loads[kBlocks] = {0, 0}, probs[kBlocks] = {0, 0};
        bool ok = true;
        auto wait = [&](uint64_t *bar, unsigned parity) {
          ok = ok && wait_for(bar, parity & 1, abort_flag, a.sooner);
          if (!ok) give_up();
          return ok;
        };
        for (int n = 0; ok && next_item(n); ++n) {
          const Item it = items[n % kItemSlots];
          ptx::mbar_arrive(item_empty + n % kItemSlots);
          const int tiles = it.end - it.begin;
          if (tiles == 0) continue;
          const int active = it.count > a.tokens ? 2 : 1;
          auto scores = [&](int b, unsigned copy, bool last) {  // S of block b and the tile that is copy `copy`
            const uint32_t keys = ring + copy % kStages * S::kBytes;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
              const uint32_t at = (k / 4) * S::kHalf + (k % 4) * 32;
              mma_ss(tmem + b * kTile, ptx::make_smem_desc(queries + b * S::kBytes + at, 1024, 16, 2), ptx::make_smem_desc(keys + at, 1024, 16, 2), kScores,
                     k > 0);
            }
            ptx::tc_commit<1>(s_full + b);
            if (last) ptx::tc_commit<1>(q_empty + b);
          };
          for (int b = 0; b < active; ++b) {
            if (!wait(q_full + b, loads[b]++)) break;
            if (b == 0 && !wait(kv_full + copies % kStages, copies / kStages)) break;
            ptx::tc_fence_after();
            scores(b, copies, tiles == 1);
          }
          if (!ok) break;
          ptx::tc_commit<1>(kv_empty + copies % kStages);
          ++copies;
          for (int tile = 0; tile < tiles && ok; ++tile) {
            const unsigned value = copies, next = copies + 1;
            const bool more = tile + 1 < tiles;
            if (!wait(kv_full + value % kStages, value / kStages)) break;
            if (!wait(v_ok + values % kStages, values / kStages)) break;
            const bool by_rows = (not_finite[values % kStages * kCheckWarps] | not_finite[values % kStages * kCheckWarps + 1]) != 0;
            ++values;
            if (more && !wait(kv_full + next % kStages, next / kStages)) break;
            for (int b = 0; b < active; ++b) {
              const uint32_t from = ring + value % kStages * S::kBytes;
              for (int piece = 0; piece < 2; ++piece) {
                if (!wait((piece == 0 ? p_first : p_full) + b, probs[b])) break;
                ptx::tc_fence_after();
                if (!by_rows) {
#pragma unroll
                  for (int k = 0; k < kTile / 16; ++k)
                    if ((k < kFirst / 16) == (piece == 0))
                      mma_ts(tmem + S::kOutCol + b * D, tmem + b * kTile + k * 8, ptx::make_smem_desc(from + k * 2048, 1024, S::kHalf, 2), kOutputs,
                             tile > 0 || k > 0);
                }
              }
              if (!ok) break;
              ++probs[b];
              if (b + 1 == active) ptx::tc_commit<1>(kv_empty + value % kStages);
              if (more)
                scores(b, next, tile + 2 == tiles);
              else
                ptx::tc_commit<1>(o_full + b);
            }
            if (!ok) break;
            if (more) ptx::tc_commit<1>(kv_empty + next % kStages);
            copies += more ? 2 : 1;
          }
        }
      }
      __syncwarp();
    } else {
      const int part = warp - kCheckWarp;
      unsigned copies = 0, values = 0;
      bool ok = true;
      for (int n = 0; ok && next_item_of_warp(n); ++n) {
        const Item it = items[n % kItemSlots];
        leave_item(n);
        for (int tile = it.begin; tile < it.end; ++tile, copies += 2, ++values) {
          const unsigned copy = copies + 1;
          ok = wait_for(kv_full + copy % kStages, (copy / kStages) & 1, abort_flag, a.sooner);
          if (!ok) give_up();
          __syncwarp();
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          bool found = false;
          if (is_masked(it, tile, a.window, a.sinks)) {
            const uint32_t from = ring + copy % kStages * S::kBytes + part * (S::kBytes / kCheckWarps) + lane * 16;
            unsigned top = 0;
#pragma unroll 8
            for (int i = 0; i < S::kBytes / kCheckWarps; i += 512) {
              const float4 v = ptx::ld_shared_f32x4(from + i);
              top = __vmaxu2(top, __vmaxu2(__float_as_uint(v.x) & 0x7FFF7FFFu, __float_as_uint(v.y) & 0x7FFF7FFFu));
              top = __vmaxu2(top, __vmaxu2(__float_as_uint(v.z) & 0x7FFF7FFFu, __float_as_uint(v.w) & 0x7FFF7FFFu));
            }
            found = max(top & 0xFFFFu, top >> 16) >= 0x7F80u;
          }
          const bool any = __any_sync(0xffffffffu, found);
          if (lane == 0) {
            not_finite[values % kStages * kCheckWarps + part] = any;
            ptx::mbar_arrive(v_ok + values % kStages);
          }
          __syncwarp();
        }
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {
    // A wait ran out, in whichever warp: the others may have ended in good order and left copies and products on their way.  These land and end before
    // the memory is another CTA's.
    if (warp == kLoadWarp && lane == 0) {
      const unsigned copies = issued[0];
      for (unsigned i = copies > kStages ? copies - kStages : 0; i < copies; ++i) ptx::mbar_drain(kv_full + i % kStages, (i / kStages) & 1);
      for (int b = 0; b < kBlocks; ++b)
        if (issued[1 + b] > 0) ptx::mbar_drain(q_full + b, (issued[1 + b] - 1) & 1);
    }
    if (multiplies) {
      ptx::tc_commit<1>(drained);
      ptx::mbar_drain(drained, 0);
    }
    __syncwarp();
  }
  if (warp == kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, 512);
  }
}

// Joins the parts of the items that begin in one CTA's stretch and end in a later one's, in the order of the list: the result does not depend on timing.  A warp
// takes a row.
constexpr int kJoinWarps = 8, kJoinSlices = 8;

template <int D>
__global__ void __launch_bounds__(32 * kJoinWarps) prompt_attention_join_kernel(const __grid_constant__ Args a, int ctas) {
  ptx::grid_dependency_wait();
  const int4 item = a.joins[2 * blockIdx.x];
  const int parts = min(a.joins[2 * blockIdx.x + 1].x, ctas - (int)blockIdx.x), lane = threadIdx.x & 31;
  if (parts < 2) return;
  const int kv = item.w / a.chunks, chunk = item.w - kv * a.chunks;
  const float2 *ml = reinterpret_cast<const float2 *>(a.parts + 2LL * ctas * kBlocks * kTile * D);
  for (int row = blockIdx.y * kJoinWarps + (threadIdx.x >> 5); row < kBlocks * kTile; row += kJoinSlices * kJoinWarps) {
    const int block = row / kTile, token = row % kTile / a.chunk_heads, head = row % kTile % a.chunk_heads, t = block * a.tokens + token;
    if (token >= a.tokens || t >= item.y || chunk * a.chunk_heads + head >= a.group) continue;
    auto place = [&](int i) { return (2LL * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * kBlocks * kTile + row; };
    // the maximum first, so that the parts are read without waiting for one another (one that is not a number has such a sum, too)
    float top = -INFINITY;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, ml[place(i)].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    float sum = 0.0f, acc[D / 32];
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] = 0.0f;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const long long at = place(i);
      const float2 of = ml[at];
      const float *x = a.parts + at * D + lane * (D / 32);
      const float f = of.x == top ? 1.0f : exp2_approx(of.x - top);  // also where all are -inf: sums of nothing
      sum += of.y * f;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] += x[e] * f;
    }
    __nv_bfloat16 *out = a.out + ((long long)(item.x + t) * a.heads + kv * a.group + chunk * a.chunk_heads + head) * D + lane * (D / 32);
    const float f = 1.0f / sum;
#pragma unroll
    for (int e = 0; e < D / 32; e += 2)
      *reinterpret_cast<uint32_t *>(out + e) = item.z + t < 0 ? 0 : pack_bf16(acc[e] * f, acc[e + 1] * f);
  }
}

// Whether items are cut, from sizes of tensors alone: where what it costs (the parts' way to memory and back and the second launch, as much as some 20 tiles of 128 or 10
// of 64) is less than what CTAs wait for the one with the most tiles, as far as the average sequence tells.  Whole / cut, us, 32 / 8 heads of 128: 64 queries behind 8000
// keys 126 / 46, 512 behind 30000 455 / 243; four pieces of 500 behind 1000 149 / 160, a prompt of 2048 56 / 59; 8 heads of 64, 4095 behind 6000 137 / 121.
bool is_split(const PromptAttention &p, const Args &a, int sms) {
  const double span = a.span, items = (std::floor(p.rows / span) + p.seqs) * a.kv_heads * a.chunks, turns = items / sms;
  const double keys = (double)p.k_rows / p.seqs, ahead = std::max(0.0, keys - (double)p.rows / p.seqs), seen = (double)a.window + a.sinks;
  const double most = std::min(keys, seen + span) / kTile, average = std::min(ahead + 0.5 * (keys - ahead), seen) / kTile + 0.5;
  const double whole = turns <= 1 ? most : std::max(most, (turns + 0.5) * average), cut = turns * average + (p.head_dim == 128 ? 20 : 10);
  return p.seqs <= 128 && whole > cut;
}

size_t split_bytes(int head_dim, int ctas) {
  return 2 * (size_t)ctas * kBlocks * kTile * (head_dim + 2) * sizeof(float) + 2 * (size_t)ctas * sizeof(int4);
}

bool encode(CUtensorMap *map, const void *base, int rows, int heads, int halves, long long row_stride, long long head_stride, bool heads_first,
            int box_rows, int box_heads, int box_halves) {
  // [128 bytes][heads][rows][halves] for the queries, [128 bytes][rows][halves][heads] for keys and values; strides in elements
  const cuuint64_t row = (cuuint64_t)row_stride * 2, head = (cuuint64_t)head_stride * 2;
  if (heads_first) {
    const cuuint64_t dims[4] = {128, (cuuint64_t)heads, (cuuint64_t)rows, (cuuint64_t)halves}, strides[3] = {head, row, 128};
    const cuuint32_t box[4] = {128, (cuuint32_t)box_heads, (cuuint32_t)box_rows, 1};
    return make_tensor_map(map, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const cuuint64_t dims[4] = {128, (cuuint64_t)rows, (cuuint64_t)halves, (cuuint64_t)heads}, strides[3] = {row, 128, head};
  const cuuint32_t box[4] = {128, (cuuint32_t)box_rows, (cuuint32_t)box_halves, 1};
  return make_tensor_map(map, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

long long g_sooner = 0;  // host-side setting, see set_prompt_attention_wait_limit

Args args_of(const PromptAttention &p, int sms) {
  Args a = {};
  a.sooner = g_sooner;
  a.offsets = p.offsets;
  a.k_offsets = p.k_offsets;
  a.out = static_cast<__nv_bfloat16 *>(p.out);
  a.rows = p.rows;
  a.k_rows = p.k_rows;
  a.seqs = p.seqs;
  a.heads = p.heads;
  a.kv_heads = p.kv_heads;
  a.group = p.heads / p.kv_heads;
  a.chunks = (a.group + kTile - 1) / kTile;
  a.chunk_heads = (a.group + a.chunks - 1) / a.chunks;
  a.tokens = kTile / a.chunk_heads;
  // One block where there are SMs for each: its exponentials share theirs with no other's (200 tokens of 32 / 8 heads 9.9 us instead of 11.3).
  const long long singles = ((long long)p.rows / a.tokens + p.seqs) * a.kv_heads * a.chunks;
  a.span = singles <= sms ? a.tokens : kBlocks * a.tokens;
  a.window = p.window;
  a.sinks = p.sinks;
  a.scale_log2 = p.scale * 1.4426950408889634f;
  a.fill = p.fill;
  a.wide = reinterpret_cast<uintptr_t>(p.out) % 32 == 0;
  a.error_flag = p.error_flag;
  return a;
}

template <int D>
cudaError_t launch(const PromptAttention &p, Args a, int sms, cudaStream_t stream) {
  using S = Sizes<D>;
  CUtensorMap q, k, v, k8, v8;
  const int k_rows = std::max(p.k_rows, 1);  // a map has a row; where there is none no sequence has keys, and nothing is read
  if (!encode(&q, p.q, p.rows, p.heads, S::kHalves, p.q_row, p.q_head, true, a.tokens, a.chunk_heads, 1) ||
      !encode(&k, p.k, k_rows, p.kv_heads, S::kHalves, p.k_row, p.k_head, false, kTile, 1, S::kHalves) ||
      !encode(&v, p.v, k_rows, p.kv_heads, S::kHalves, p.v_row, p.v_head, false, kTile, 1, S::kHalves))
    return cudaErrorInvalidValue;
  // copies of 8 keys join the first ones and the window's; without first ones there are none
  if (p.sinks == 0)
    k8 = k, v8 = v;
  else if (!encode(&k8, p.k, k_rows, p.kv_heads, S::kHalves, p.k_row, p.k_head, false, 8, 1, 1) ||
           !encode(&v8, p.v, k_rows, p.kv_heads, S::kHalves, p.v_row, p.v_head, false, 8, 1, 1))
    return cudaErrorInvalidValue;
  static bool ready[64] = {};
  cudaError_t err = allow_smem(prompt_attention_kernel<D>, S::kTotal, ready);
  if (err != cudaSuccess) return err;
  const long long most = ((long long)p.rows / a.span + p.seqs) * a.kv_heads * a.chunks;
  a.split = is_split(p, a, sms);
  const int ctas = !a.split && most < sms ? (int)most : sms;
  if (a.split) {
    a.parts = static_cast<float *>(p.workspace);
    a.joins = reinterpret_cast<int4 *>(a.parts + 2LL * ctas * kBlocks * kTile * (D + 2));
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kTotal;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  err = cudaLaunchKernelEx(&cfg, prompt_attention_kernel<D>, q, k, v, k8, v8, a);
  if (err != cudaSuccess || !a.split) return err;
  cfg.gridDim = dim3((unsigned)ctas, kJoinSlices);
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, prompt_attention_join_kernel<D>, a, ctas);
}

int sm_count() {
  static int counts[64] = {};
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0) return 148;
  if (dev < 64 && counts[dev] > 0) return counts[dev];
  if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  if (dev < 64) counts[dev] = sms;
  return sms;
}

}  // namespace

void set_prompt_attention_wait_limit(long long cycles) { g_sooner = cycles > 0 ? std::max(0LL, ptx::kWaitLimitCycles - cycles) : 0; }

size_t prompt_attention_workspace_bytes(const PromptAttention &p) {
  const int sms = sm_count();
  return is_split(p, args_of(p, sms), sms) ? split_bytes(p.head_dim, sms) : 0;
}

cudaError_t run_prompt_attention(const PromptAttention &p, cudaStream_t stream) {
  const int sms = sm_count();
  return p.head_dim == 128 ? launch<128>(p, args_of(p, sms), sms, stream) : launch<64>(p, args_of(p, sms), sms, stream);
}

}  // namespace sharq
