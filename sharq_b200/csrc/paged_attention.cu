// Attention of one new token per sequence over a paged key/value cache.  131072 tokens of 8 heads of 128 in bf16: 88 us, 6.1 TB/s, 93 % of the rate
// of a copy; 128 sequences of 33 to 8192 tokens in e4m3: 117 to 129 us by where the cache lies, 95 to 86 %; one sequence of 97 tokens: 4.1 us.
//
//   out[b, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q[b, h] . k_j - max),   j < lengths[b]
//
// One pass over the cache with a running maximum and sum.  The work is bound by reading the cache: 4 flop per byte and query head of a group (the query
// heads that share a key/value head), far below what even mma.sync gives, and a legacy MMA takes its operands from registers in the
// layout in which ldmatrix delivers cache rows, without a trip through tensor memory.  Tokens (for the scores) and elements of a head (for the
// output) are the 16-row operand, the group's query heads the 8 columns, in chunks of up to 16 heads: S^T = K Q^T and O^T = V^T P^T.  The scores'
// accumulator is [token][head]; movmatrix turns the probabilities, packed to 16 bits, into the operand of the second product.
//
// A warp streams tiles of keys and values through a ring of its own in shared memory: tensor-map copies counted on the stage's barrier,
// in the 128-byte swizzle in which eight rows lie in different banks.  (The first form copied 16 bytes per lane with cp.async, and had queries as the
// 16-row operand: 655 instructions per tile of 16 tokens, 112 us for 131072 tokens of 8 heads, bound by their latency.)
//
// The tiles of all sequences and heads are one list, and every warp takes an equal stretch of it, whatever the lengths; each (sequence, head) counts
// kItemCost tiles more, for its queries and its result.  A warp writes the finished rows of a (sequence, head) that lies within its stretch, and
// leaves a float part with its maximum and sum of one that does not (two at most, at the ends).  When its warps are done, a CTA joins
// their parts in shared memory, and a second kernel, which starts early and waits, those of different CTAs, both in the order of the list: the
// result does not depend on timing.  (With warps that met at the end of every (sequence, head) 64 sequences of 10 to 300 tokens took 33 us; without the
// join of a CTA's own parts the second kernel had four times as many, 17 us for 131072 tokens of 8 heads.)
//
// The maximum is raised only when a score exceeds it by more than kLazy (then probabilities stay below 2^kLazy, and the sum and the output
// are relative to the same value): raising it costs shuffles and a pass over the output.
//
// e4m3 caches go through f16: their values are exact in it, queries are scaled to it by a power of two per head (exact down to 2^-31 of the head's
// largest, off by at most 2^-39 of that below), and probabilities carry a factor of 2^10, so that those down to 2^-24 of the maximum keep f16's full
// precision.  The probabilities enter as the sum of two numbers: for bf16 caches two bf16 numbers, 16 bits (rounded to one they made half of the result's
// error, and the reading of the cache hides the second product; both are positive, for an infinite value has an infinite product with either), for e4m3 caches
// two f16 numbers, 21 bits (with one, values that nearly cancel came out several steps off; it costs nothing for 128 sequences of 33 to 8192 tokens, 1 % for
// 8 x 2048 tokens of 8 heads, 7 % for 20 x 2000).  For bf16 caches they carry a factor of 2^-32, so that no sum of finite values overflows; 2^-94 of the
// maximum and less is 0.
//
// With a window a sequence's tiles are those with a token that is seen, so everything above goes on over a shorter list (an instance of its own: a call without a
// window runs the code it ran); hidden tokens in the tiles at the window's ends get the score -inf and values of 0.  Window 4096 of 100000 tokens of 8 heads: 12.7 us
// with 4 first tokens, whose tile makes 9 of a warp's 8, 12.0 without (4096 and 4160 tokens without a window: 11.1 and 11.8); 96 sequences of up to 12000 in e4m3, window 2048: 58 to 61 us, 0.78 to 0.74 of the rate of a copy.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "decode_ops.cuh"
#include "sm100_ptx.cuh"
#include "tensor_map.cuh"

namespace sharq {

namespace {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr float kF16Lift = 10.0f, kBf16Lift = -32.0f;  // log2 of a factor of the probabilities
constexpr int kItemCost = 2;      // in tiles (200 x 30 tokens 12.5 us, with 1, 3 or 4: 14.0, 13.8, 12.6; 128 x 64: 13.7 and 13.1, 13.3, 12.5)
constexpr int kStretchLeast = 4;  // tiles of a warp (5 sequences of up to 20011 tokens of one head 13.8 us, with 2, 6 or 8: 14.3, 14.5, 15.5)
constexpr int kAttnClusterMost = 8;
constexpr int kDirectMost = 16, kDirectFew = 10;  // tiles of a warp for which a cluster is taken at most, where its like fill two fifths of the SMs or not

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
__device__ __forceinline__ uint32_t movmatrix(uint32_t w) {  // transpose of an 8 x 8 matrix of 16-bit elements, two per lane
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));  // volatile: stays ahead of a branch that uses it
  return r;
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
// tokens of a cache [page][head][half][token][128 bytes]
__device__ __forceinline__ void copy_tokens(uint32_t dst, const CUtensorMap *m, int token, int half, int head, int page, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
      "l"(m), "r"(ptx::smem_u32(bar)), "r"(0), "r"(token), "r"(half), "r"(head), "r"(page)
      : "memory");
}

struct AttnArgs {
  const __nv_bfloat16 *q;
  long long q_row, q_head;
  const int *lengths;
  __nv_bfloat16 *out;
  float *parts;  // [2 * CTAs][D][kCols] unnormalised columns, then [2 * CTAs][kCols] of their [maximum, sum]
  int seqs, heads, group, chunks;  // chunks: pieces of 16 query heads of a group
  int box_shift;                   // log2 of the tokens of a copy: the largest power of two, at most a tile, that divides the page size
  int stretch_shift;               // direct form: log2 of the warps of a cluster
  unsigned stretches_magic, items_magic;  // list: for divide() by the stretches and by the items of a sequence
  int page_shift;                  // log2 of the page size, -1 if it is no power of two
  float scale_log2;                // scale * log2(e)
  int window, sinks;               // windowed form: tokens that are seen from the last one back, and first ones
  int *error_flag;
};

// Sizes that follow from the head and the type of the cache.  Rows lie 128 bytes apart: a row of 256 bytes in two halves, one of 64 bytes (e4m3 heads of
// 64) with zeros behind it, which the copy fills in.  A tile holds 8 KB.
template <int D, bool kFp8>
struct Tile {
  static constexpr int kSize = kFp8 ? 1 : 2;
  static constexpr int kHalves = D * kSize > 128 ? 2 : 1;
  static constexpr int kTokens = 32 / kHalves;
  static constexpr int kHalf = kTokens * 128;
  static constexpr int kBytes = kHalf * kHalves;  // of keys, or of values
  static constexpr int kStage = 2 * kBytes;
};
static_assert(Tile<128, false>::kStage == 8192 && Tile<64, true>::kStage == 8192, "a stage is a multiple of the swizzle's 1024 bytes");

// What a warp leaves of an item that does not lie within its stretch.
struct __align__(16) Part {
  int seq, item;  // item: which (head, chunk) of the sequence, below 2^17; -1: nothing
  int begins, tiles_left;
};
// A lane's wait ran out: it waits for nothing more, and copies nothing more when it is elected to.  What its warp takes part in from then on comes out
// as NaN.  (A vote on it at every tile took 1 to 3 %.)
constexpr unsigned kLost = 1u << 31;
// Forms of the kernel: the list of tiles, and the direct one with two or three CTAs per SM.
constexpr int kList = 0, kDirectTwo = 1, kDirectThree = 2;

// Shared memory of a CTA: the rings (the swizzle wants 1024 bytes), then the part at the beginning of every warp's stretch (the one at the end, and
// the only one of the direct form, goes to the warp's ring, which is free by then), two parts' maxima and sums per warp, their descriptions,
// barriers and the flag of a wait that ran out.  CTAs: per SM.
template <int D, bool kFp8, int kCols, int kForm>
struct Layout {
  static constexpr bool kDirect = kForm != kList;
  static constexpr int kCtas = kForm == kDirectThree ? 3 : 2;
  static constexpr int kStages = 2;
  static constexpr int kRing = kStages * Tile<D, kFp8>::kStage;
  static constexpr int kPart = D * kCols * 4;
  static constexpr int kParts = kAttnWarps * kRing;
  static constexpr int kMl = kParts + (kDirect ? 0 : kAttnWarps * kPart);
  static constexpr int kInfo = kMl + 2 * kAttnWarps * kCols * 8;
  static constexpr int kBars = kInfo + 2 * kAttnWarps * (int)sizeof(Part);
  static constexpr int kFlag = kBars + kAttnWarps * kStages * 8;
  static constexpr int kTotal = kFlag + 8;
  static_assert(kPart <= kRing && kCtas * (kTotal + 1024) <= 233472, "a part fits a ring, the CTAs an SM");
};

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
// Windowed form: a sequence of n tokens is seen but for [sinks, begin), begin = n - window, and the tiles that hold nothing but those, `skip` of them behind the first
// `front`, are left out of its list of tiles.
struct Gap {
  int begin, front, skip;
};
template <int kTokens, bool kWindow>
__device__ __forceinline__ Gap gap_of(const AttnArgs &a, int tokens) {
  if (!kWindow) return {0, 0, 0};
  const int begin = max(0, tokens - a.window), front = (int)(((unsigned)min(a.sinks, tokens) + kTokens - 1) / kTokens);
  return {begin, front, max(0, begin / kTokens - front)};
}
template <int kTokens, bool kWindow>
__device__ __forceinline__ int tiles_of(const AttnArgs &a, int tokens) {  // an empty sequence has one tile, without tokens
  return (tokens <= kTokens ? 1 : (tokens - 1) / kTokens + 1) - gap_of<kTokens, kWindow>(a, tokens).skip;
}

// n / d for n < 2^31 with ceil(2^32 / d) at hand (an integer division by a variable takes some hundred cycles): at most one too high
__device__ __forceinline__ int divide(int n, int d, unsigned magic) {
  const int q = d == 1 ? n : (int)__umulhi((unsigned)n, magic);
  return q * d > n ? q - 1 : q;
}

// Where a warp stands in its stretch: tiles [tile, end) of an item are its own.  An item is kItemCost + its tiles long in the list, of which `skip` lie
// in earlier stretches; `left`: how much of the stretch remains from there on.
struct Place {
  int seq, head, chunk, skip, left, tokens, tile, end;
};
template <int kTokens, bool kWindow>
__device__ __forceinline__ void enter(Place &p, const AttnArgs &a, const PagedCache &c) {
  p.tokens = length_of(a, c, p.seq).tokens;
  p.tile = max(0, p.skip - kItemCost);
  p.end = min(tiles_of<kTokens, kWindow>(a, p.tokens), p.skip + p.left - kItemCost);
}
template <int kTokens, bool kWindow>
__device__ __forceinline__ void leave(Place &p, const AttnArgs &a, const PagedCache &c) {
  p.left = max(0, p.left - (kItemCost + tiles_of<kTokens, kWindow>(a, p.tokens) - p.skip));
  if (p.left == 0) return;
  p.skip = 0;
  if (++p.chunk == a.chunks) {
    p.chunk = 0;
    ++p.head;
  }
  if (p.head == c.kv_heads) {
    p.head = 0;
    ++p.seq;
    enter<kTokens, kWindow>(p, a, c);
  } else {  // the same sequence's tokens
    p.tile = 0;
    p.end = min(tiles_of<kTokens, kWindow>(a, p.tokens), p.left - kItemCost);
  }
}

// The list of all tiles, its length and the part of it that a warp takes: less than 2^31, the launcher checks.
struct List {
  int total, per;
};
template <int kTokens, bool kWindow>
__device__ __forceinline__ List list_of(const AttnArgs &a, const PagedCache &c, int items, int stretches, int lane) {
  int per_head = 0;
#pragma unroll 4
  for (int b = lane; b < a.seqs; b += 32) per_head += kItemCost + tiles_of<kTokens, kWindow>(a, length_of(a, c, b).tokens);
  const int total = __reduce_add_sync(0xffffffffu, per_head) * items;
  return {total, max(kStretchLeast, divide(total + stretches - 1, stretches, a.stretches_magic))};
}
// the item that unit u of the list belongs to, and what of it lies before u -> the item's length
template <int kTokens, bool kWindow>
__device__ __forceinline__ int locate(Place &at, int u, const AttnArgs &a, const PagedCache &c, int items, int lane) {
  int before = 0;
  const int u_head = divide(u, items, a.items_magic);  // in units of a head: a sequence begins at items times what lies before it
  for (int b0 = 0; b0 < a.seqs; b0 += 32) {
    const int b = b0 + lane;
    const int n_units = b < a.seqs ? kItemCost + tiles_of<kTokens, kWindow>(a, length_of(a, c, b).tokens) : 0;
    int n = n_units;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, n, off);
      if (lane >= off) n += up;
    }
    const unsigned over = __ballot_sync(0xffffffffu, before + n > u_head);
    if (over != 0) {
      const int in = __ffs(over) - 1;
      const int units = __shfl_sync(0xffffffffu, n_units, in), rest = u - (before + __shfl_sync(0xffffffffu, n, in) - units) * items;
      // less than 2^16 items, so the float quotient is one off at most
      int item = (int)__fdividef((float)rest, (float)units);
      if (item * units > rest) --item;
      if (rest - item * units >= units) ++item;
      at.seq = b0 + in;
      at.skip = rest - item * units;
      at.head = a.chunks == 1 ? item : item / a.chunks;
      at.chunk = item - at.head * a.chunks;
      return units;
    }
    before += __shfl_sync(0xffffffffu, n, 31);
  }
  return 0;
}

// kCols: columns for query heads (8 or 16).  kDirect: a cluster per (sequence, head chunk), blockIdx = (rank, head chunk, sequence), whose warps take equal
// stretches of its tiles and whose CTAs join their parts through distributed shared memory; nothing is left for a second launch.
template <int D, bool kFp8, int kCols, int kForm, bool kWindow>
__global__ void __launch_bounds__(kAttnThreads, (Layout<D, kFp8, kCols, kForm>::kCtas))
    paged_attention_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           const __grid_constant__ AttnArgs a, const __grid_constant__ PagedCache c) {
  using T = Tile<D, kFp8>;
  using L = Layout<D, kFp8, kCols, kForm>;
  constexpr bool kDirect = L::kDirect;
  constexpr int kTokens = T::kTokens, kN = kCols / 8, kStages = L::kStages;
  constexpr float kLazy = kFp8 ? 4.0f : 8.0f;  // f16: 2^(10 + 4) at most
  extern __shared__ __align__(1024) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = ptx::smem_u32(smem) + warp * L::kRing;
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBars) + warp * kStages;
  volatile int *gave_up = reinterpret_cast<volatile int *>(smem + L::kFlag);
  Part *info = reinterpret_cast<Part *>(smem + L::kInfo);
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) ptx::mbar_init(bars + i, 1);
    ptx::fence_barrier_init();
    ptx::tma_prefetch_desc(&map_k);
    ptx::tma_prefetch_desc(&map_v);
  }
  if (threadIdx.x == 0) *gave_up = 0;
  if (threadIdx.x < 2 * kAttnWarps) info[threadIdx.x].item = -1;
  __syncthreads();
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();  // behind the wait: the second kernel reads the lengths ahead of its own
  const int items = c.kv_heads * a.chunks;  // (head, chunk) pairs of a sequence

  // this warp's stretch of the list of tiles
  const int stretch = blockIdx.x * kAttnWarps + warp, stretches = gridDim.x * kAttnWarps;
  Place at = {0, 0, 0, 0, 0, 0, 0, 0};
  if (kDirect) {
    at.seq = blockIdx.z;
    at.head = a.chunks == 1 ? blockIdx.y : blockIdx.y / a.chunks;
    at.chunk = blockIdx.y - at.head * a.chunks;
    at.tokens = length_of(a, c, at.seq).tokens;
    const int n_tiles = tiles_of<kTokens, kWindow>(a, at.tokens), each = (n_tiles + stretches - 1) >> a.stretch_shift;
    at.tile = stretch * each;
    at.end = min(n_tiles, at.tile + each);
    at.left = 1;  // this item and no other
  } else {
    const List list = list_of<kTokens, kWindow>(a, c, items, stretches, lane);
    const int u0 = stretch * list.per;  // stretches * per: total and a little more
    at.left = max(0, min(list.per, list.total - u0));
    if (at.left > 0) {
      locate<kTokens, kWindow>(at, u0, a, c, items, lane);
      enter<kTokens, kWindow>(at, a, c);
    }
  }

  Place next = at;  // of the tile that is loaded next
  const int box = 1 << a.box_shift, boxes = kTokens >> a.box_shift;  // pieces of `box` tokens of a page that a tile consists of
  int held_seq = -1, held_first = 0, held_page = 0;  // lane j: page of piece held_first + j of sequence held_seq
  auto settle = [&]() {  // moves on to the next item with a tile for this warp
    bool entered = false;
    while (next.tile >= next.end && next.left > 0) {
      leave<kTokens, kWindow>(next, a, c);
      entered = true;
    }
    if (entered && next.left > 0) {  // its queries on their way to the SM
      const int rows = min(16, a.group - next.chunk * 16);
      constexpr int kLines = D * 2 / 128;
      if (lane < rows * kLines)
        asm volatile("prefetch.global.L1 [%0];" ::"l"(a.q + next.seq * a.q_row + (next.head * a.group + next.chunk * 16 + lane / kLines) * a.q_head +
                                                      lane % kLines * 64));
    }
  };
  int put = 0;              // stage that is filled next
  unsigned bad_stages = 0;  // stages with a piece of no page, and kLost
  auto load = [&]() {
    if (next.left > 0) {
      const uint32_t stage = ring + put * T::kStage;
      const Gap gap = gap_of<kTokens, kWindow>(a, next.tokens);
      const int tile = kWindow && next.tile >= gap.front ? next.tile + gap.skip : next.tile;
      const int live = next.tokens - tile * kTokens;  // tokens from this tile on
      const int pieces = live <= 0 ? 0 : min(boxes, (live + box - 1) >> a.box_shift);
      const int piece0 = tile * boxes;
      if (next.seq != held_seq || piece0 < held_first || piece0 + boxes > held_first + 32) {
        held_seq = next.seq;
        held_first = piece0;
        const int token = (piece0 + lane) << a.box_shift;
        held_page = 0;
        if (token < next.tokens) held_page = c.page_table[next.seq * c.table_stride + (a.page_shift >= 0 ? token >> a.page_shift : token / c.page_size)];
      }
      bool any_bad = false;
      const bool chosen = ptx::elect_one() && (bad_stages & kLost) == 0;
      if (chosen) ptx::mbar_arrive_expect_tx(bars + put, (pieces << a.box_shift) * 256 * T::kHalves);
      for (int i = 0; i < pieces; ++i) {
        int page = __shfl_sync(0xffffffffu, held_page, piece0 + i - held_first);
        const int token = (piece0 + i) << a.box_shift;
        const int slot = a.page_shift >= 0 ? token & (c.page_size - 1) : token % c.page_size;
        if ((unsigned)page >= (unsigned)c.pages) {
          any_bad |= !(kWindow && token >= a.sinks && token + box <= gap.begin);  // a page that is not seen may be anything
          page = c.pages;  // one behind the last: zeros are filled in
        }
        if (chosen) {
          const uint32_t to = stage + (i << a.box_shift) * 128;
          copy_tokens(to, &map_k, slot, 0, next.head, page, bars + put);
          copy_tokens(to + T::kBytes, &map_v, slot, 0, next.head, page, bars + put);
          if (T::kHalves == 2 && boxes > 1) {  // a whole tile's halves are one copy
            copy_tokens(to + T::kHalf, &map_k, slot, 1, next.head, page, bars + put);
            copy_tokens(to + T::kBytes + T::kHalf, &map_v, slot, 1, next.head, page, bars + put);
          }
        }
      }
      bad_stages = (bad_stages & ~(1u << put)) | (any_bad ? 1u << put : 0);
      ++next.tile;
      put = put + 1 == kStages ? 0 : put + 1;
      settle();
    }
  };
  settle();
  for (int i = 0; i < kStages - 1; ++i) load();

  // Rows of a tile that a lane reads.  bf16: an ldmatrix takes 8 rows x 16 bytes per 8 lanes; lane & 7 is the row in the swizzle.
  // keys: matrices (tokens 0-7 | 8-15) x (16-byte piece 2k | 2k + 1), values: pieces first, as the transposed operand wants them
  const uint32_t k_lane = ((lane & 7) + ((lane >> 3) & 1) * 8) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
  const uint32_t v_lane = ((lane & 7) + (lane >> 4) * 8) * 128 + ((((lane >> 3) & 1) ^ (lane & 7)) << 4);
  // e4m3: lane (g, t) holds token row (g >> 1) + 4 (g & 1) of eight, so that the rows and pieces that a quarter of a warp reads at once lie in
  // different banks; of the values it reads piece (g >> 1) + 4 (g & 1) of the tokens of slots 2t and 2t + 1, the rows t and t + 4
  const int g_mixed = (g >> 1) | ((g & 1) << 2);
  const int my_token = kFp8 ? g_mixed : g;

  int take = 0;         // stage that is used next
  unsigned phases = 0;  // parity of every stage's barrier
  for (; at.left > 0; leave<kTokens, kWindow>(at, a, c)) {
    if (at.tile >= at.end) continue;
    const int kv = at.head, chunk = at.chunk;
    const int cols = min(16, a.group - chunk * 16);  // query heads of the chunk
    const int head0 = kv * a.group + chunk * 16;
    const bool begins = at.tile == 0;

    // queries: columns 8 n + g, zeros behind the group's heads
    uint32_t qb[kN][D / 16][2];
    float sl[kN][2];  // of columns 8 n + 2 t and the next one
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      const bool live = 8 * n + g < cols;
      const __nv_bfloat16 *q = a.q + at.seq * a.q_row + (head0 + 8 * n + g) * a.q_head;
      if (!kFp8) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          qb[n][k][0] = live ? *reinterpret_cast<const uint32_t *>(q + 2 * t + 16 * k) : 0;
          qb[n][k][1] = live ? *reinterpret_cast<const uint32_t *>(q + 2 * t + 16 * k + 8) : 0;
        }
        sl[n][0] = sl[n][1] = a.scale_log2;
      } else {
        // step k of a span of 64 elements takes the elements 16 t + 4 (k % 4) + {0, 1, 2, 3} of the span from lane t, as the keys do
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint2 w = live ? *reinterpret_cast<const uint2 *>(q + 16 * t + (k / 4) * 64 + (k % 4) * 4) : make_uint2(0, 0);
          qb[n][k][0] = w.x;
          qb[n][k][1] = w.y;
          top = __vmaxu2(top, __vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu));
        }
        top = max(top & 0xFFFFu, top >> 16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the largest value to [2^14, 2^15), or up by 2^126; a row with infinities or NaN as it is
        const int e = (int)(top >> 7), shift = e == 255 ? 0 : min(126, 141 - max(e, 1));
        const float up = __int_as_float((127 + shift) << 23), back = a.scale_log2 * c.k_scale[kv] * __int_as_float((127 - shift) << 23);
        sl[n][0] = __shfl_sync(0xffffffffu, back, 8 * t);  // lane of column 2 t
        sl[n][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const uint32_t w = qb[n][k][j];
            qb[n][k][j] = pack_f16(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xFFFF0000u) * up);
          }
      }
    }

    float o[D / 16][kN][4];  // rows of 16 elements of the head; columns as in sl
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][n][j] = 0.0f;
    // maximum (in units of log 2, the same in all lanes of a column) and this lane's share of the sum
    float m[kN][2], l[kN][2];
#pragma unroll
    for (int n = 0; n < kN; ++n) m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.0f;

    const Gap gap = gap_of<kTokens, kWindow>(a, at.tokens);
    for (int tile = at.tile; tile < at.end; ++tile) {
      const int first_token = (kWindow && tile >= gap.front ? tile + gap.skip : tile) * kTokens;
      load();
      const uint32_t keys = ring + take * T::kStage, values = keys + T::kBytes;
      const bool poison = (bad_stages >> take) & 1;
      if ((bad_stages & kLost) == 0 && !ptx::mbar_wait(bars + take, (phases >> take) & 1, gave_up)) {
        for (int i = 0; i < kStages; ++i) ptx::mbar_drain(bars + i, (phases >> i) & 1);
        *gave_up = 1;
        if (a.error_flag != nullptr) atomicExch(a.error_flag, kAttentionTimeout);
        bad_stages |= kLost;
      }
      __syncwarp();
      phases ^= 1u << take;
      const int live = at.tokens - first_token;  // tokens from this tile on

      float s[kTokens / 16][kN][4], s2[kTokens / 16][kN][4];  // [token][column], in two sums: a product waits for the one before it
#pragma unroll
      for (int b = 0; b < kTokens / 16; ++b)
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[b][n][j] = s2[b][n][j] = 0.0f;
#pragma unroll
      for (int b = 0; b < kTokens / 16; ++b) {
        if (!kFp8) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t w[4];
            ldmatrix4(w, (keys + b * 2048 + k_lane + (k / 4) * T::kHalf) ^ ((k % 4) * 32));
#pragma unroll
            for (int n = 0; n < kN; ++n) mma16816<kFp8>(k % 2 == 0 ? s[b][n] : s2[b][n], w, qb[n][k][0], qb[n][k][1]);
          }
        } else {
#pragma unroll
          for (int span = 0; span < D / 64; ++span) {
            const uint32_t row = keys + (b * 16 + my_token) * 128 + ((uint32_t)((span * 4 + t) ^ my_token) << 4);
            const uint4 lo = ld_shared16(row), hi = ld_shared16(row + 8 * 128);
            const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t w[4] = {e4m3_lo(wl[j]), e4m3_lo(wh[j]), e4m3_hi(wl[j]), e4m3_hi(wh[j])};
#pragma unroll
              for (int n = 0; n < kN; ++n) mma16816<kFp8>(j % 2 == 0 ? s[b][n] : s2[b][n], w, qb[n][span * 4 + j][0], qb[n][span * 4 + j][1]);
            }
          }
        }
      }
#pragma unroll
      for (int b = 0; b < kTokens / 16; ++b)
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[b][n][j] = (s[b][n][j] + s2[b][n][j]) * sl[n][j & 1];
      // rows of the tile that are not seen though they lie ahead of the last token
      const int hide0 = kWindow ? min(kTokens, max(0, a.sinks - first_token)) : 0, hide1 = kWindow ? min(kTokens, max(0, gap.begin - first_token)) : 0;
      if (live < kTokens || poison || (kWindow && hide0 < hide1)) {
#pragma unroll
        for (int b = 0; b < kTokens / 16; ++b)
#pragma unroll
          for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int row = b * 16 + (j >> 1) * 8 + my_token;
              if (row >= live || (kWindow && row >= hide0 && row < hide1)) s[b][n][j] = -INFINITY;
              if (poison) s[b][n][j] = __int_as_float(0x7fffffff);
            }
        // values behind the sequence: whatever the page or an earlier tile left there must not meet a probability of 0
        for (int i = max(live, 0) * 8 + lane; i < kTokens * 8; i += 32)
#pragma unroll
          for (int half = 0; half < T::kHalves; ++half)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(values + half * T::kHalf + i * 16), "r"(0) : "memory");
        for (int i = hide0 * 8 + lane; i < hide1 * 8; i += 32)
#pragma unroll
          for (int half = 0; half < T::kHalves; ++half)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(values + half * T::kHalf + i * 16), "r"(0) : "memory");
        ptx::fence_proxy_async();  // a later copy into this stage comes behind these stores
        __syncwarp();
      }
      bool raise = false;
#pragma unroll
      for (int b = 0; b < kTokens / 16; ++b)
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) raise |= s[b][n][j] > m[n][j & 1] + kLazy;
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float top = m[n][j];
#pragma unroll
            for (int b = 0; b < kTokens / 16; ++b) top = fmaxf(top, fmaxf(s[b][n][j], s[b][n][j + 2]));
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const float f = top > m[n][j] ? exp2_approx(m[n][j] - top) : 1.0f;  // from -inf: 0, and nothing to keep
            m[n][j] = top;
            l[n][j] *= f;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              o[i][n][j] *= f;
              o[i][n][j + 2] *= f;
            }
          }
      }
      // a column with no finite score so far has maximum -inf: its probabilities are 0, not exp(-inf + inf)
      float base[kN][2];
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) base[n][j] = (m[n][j] == -INFINITY ? 0.0f : m[n][j]) - (kFp8 ? kF16Lift : kBf16Lift);
#pragma unroll
      for (int b = 0; b < kTokens / 16; ++b) {
        uint32_t pb[kN][2], pb_lo[kN][2];
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            p[j] = exp2_approx(s[b][n][j] - base[n][j & 1]);
            l[n][j & 1] += p[j];
          }
          if (kFp8) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // the upper 11 bits, and what they leave
              const float x = __uint_as_float(__float_as_uint(p[2 * j]) & 0xFFFFE000u), y = __uint_as_float(__float_as_uint(p[2 * j + 1]) & 0xFFFFE000u);
              pb[n][j] = movmatrix(pack_f16(x, y));
              pb_lo[n][j] = movmatrix(pack_f16(p[2 * j] - x, p[2 * j + 1] - y));
            }
          } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              // the upper half of the bits, and what they leave, with the last bit set: never 0 beside an upper half that is not
              const uint32_t x = __float_as_uint(p[2 * j]) | 1, y = __float_as_uint(p[2 * j + 1]) | 1;
              pb[n][j] = movmatrix(__byte_perm(x, y, 0x7632));
              pb_lo[n][j] = movmatrix(pack_bf16(__uint_as_float(x) - __uint_as_float(x & 0xFFFF0000u),
                                                __uint_as_float(y) - __uint_as_float(y & 0xFFFF0000u)));
            }
          }
        }
        if (!kFp8) {
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            uint32_t w[4];
            ldmatrix4_trans(w, (values + b * 2048 + v_lane + (i / 4) * T::kHalf) ^ ((i % 4) * 32));
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              mma16816<kFp8>(o[i][n], w, pb[n][0], pb[n][1]);
              mma16816<kFp8>(o[i][n], w, pb_lo[n][0], pb_lo[n][1]);
            }
          }
        } else {
          // lane (g, t) takes D / 8 neighbouring elements of four tokens: rows g and g + 8 of tile i are its elements 2 i and 2 i + 1
          constexpr int kWords = D / 32;
          uint32_t w[4][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int in_eight = t + (j & 1) * 4;
            const uint32_t row = values + (b * 16 + (j >> 1) * 8 + in_eight) * 128;
            if (D == 128) {
              const uint4 v = ld_shared16(row + ((uint32_t)(g_mixed ^ in_eight) << 4));
              w[j][0] = v.x, w[j][1] = v.y, w[j][2] = v.z, w[j][3] = v.w;
            } else {
              const uint2 v = ld_shared8(row + ((uint32_t)((g >> 1) ^ in_eight) << 4) + (g & 1) * 8);
              w[j][0] = v.x, w[j][1] = v.y;
            }
          }
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            // elements 4 i .. 4 i + 3 of the tokens of slots 2t and 2t + 1, and of 2t + 8 and 2t + 9
            const uint32_t a0 = __byte_perm(w[0][i], w[1][i], 0x5140), a1 = __byte_perm(w[0][i], w[1][i], 0x7362);
            const uint32_t b0 = __byte_perm(w[2][i], w[3][i], 0x5140), b1 = __byte_perm(w[2][i], w[3][i], 0x7362);
            const uint32_t even[4] = {e4m3_lo(a0), e4m3_hi(a0), e4m3_lo(b0), e4m3_hi(b0)};
            const uint32_t odd[4] = {e4m3_lo(a1), e4m3_hi(a1), e4m3_lo(b1), e4m3_hi(b1)};
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              mma16816<kFp8>(o[2 * i][n], even, pb[n][0], pb[n][1]);
              mma16816<kFp8>(o[2 * i + 1][n], odd, pb[n][0], pb[n][1]);
              mma16816<kFp8>(o[2 * i][n], even, pb_lo[n][0], pb_lo[n][1]);
              mma16816<kFp8>(o[2 * i + 1][n], odd, pb_lo[n][0], pb_lo[n][1]);
            }
          }
        }
      }
      if (poison && lane == 0 && a.error_flag != nullptr) atomicCAS(a.error_flag, 0, kBadCacheIndex);
      __syncwarp();  // the stage may be filled again
      take = take + 1 == kStages ? 0 : take + 1;
    }

    // a lane that waits for nothing more reads what the others have waited for, unless all gave up: its columns are NaN
    const float lost = (bad_stages & kLost) != 0 ? __int_as_float(0x7fffffff) : 0.0f;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[n][j] += lost;
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], off);
      }
    const int n_tiles = tiles_of<kTokens, kWindow>(a, at.tokens);
    if (begins && at.end == n_tiles) {
      const int raw = a.lengths[at.seq];
      const bool bad = raw < 0 || raw > paged_capacity(c);
      if (bad && lane == 0 && a.error_flag != nullptr) atomicCAS(a.error_flag, 0, kBadCacheIndex);
      __nv_bfloat16 *out = a.out + ((long long)at.seq * a.heads + head0) * D;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        float f[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) f[j] = __fdividef(kFp8 ? c.v_scale[kv] : 1.0f, l[n][j]);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          float y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            y[j] = raw == 0 ? 0.0f : o[i][n][j] * f[j & 1];
            if (bad) y[j] = __int_as_float(0x7fffffff);
          }
          if (!kFp8) {
            // [element][column] to [column][element]
            __syncwarp();  // the stores before are of some lanes only
            const uint32_t w0 = movmatrix(pack_bf16(y[0], y[1])), w1 = movmatrix(pack_bf16(y[2], y[3]));
            if (8 * n + g < cols) {
              *reinterpret_cast<uint32_t *>(out + (8 * n + g) * D + 16 * i + 2 * t) = w0;
              *reinterpret_cast<uint32_t *>(out + (8 * n + g) * D + 16 * i + 8 + 2 * t) = w1;
            }
          } else {
            __nv_bfloat16 *to = out + (8 * n + 2 * t) * D + (D == 128 ? g_mixed : g) * (D / 8) + 2 * i;
            if (8 * n + 2 * t < cols) *reinterpret_cast<uint32_t *>(to) = pack_bf16(y[0], y[2]);
            if (8 * n + 2 * t + 1 < cols) *reinterpret_cast<uint32_t *>(to + D) = pack_bf16(y[1], y[3]);
          }
        }
      }
    } else {
      // [element][column], with the maxima and sums beside it
      const int slot = 2 * warp + (begins ? 1 : 0);
      float *part = reinterpret_cast<float *>(kDirect || begins ? smem + warp * L::kRing : smem + L::kParts + warp * L::kPart);
      float *part_ml = reinterpret_cast<float *>(smem + L::kMl) + slot * kCols * 2;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        if (g == 0) *reinterpret_cast<float4 *>(part_ml + (8 * n + 2 * t) * 2) = make_float4(m[n][0], l[n][0], m[n][1], l[n][1]);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int d0 = kFp8 ? (D == 128 ? g_mixed : g) * (D / 8) + 2 * i : 16 * i + g, d1 = kFp8 ? d0 + 1 : d0 + 8;
          *reinterpret_cast<float2 *>(part + d0 * kCols + 8 * n + 2 * t) = make_float2(o[i][n][0], o[i][n][1]);
          *reinterpret_cast<float2 *>(part + d1 * kCols + 8 * n + 2 * t) = make_float2(o[i][n][2], o[i][n][3]);
        }
      }
      if (lane == 0) info[slot] = {at.seq, at.head * a.chunks + at.chunk, begins, n_tiles - at.end};
    }
  }

  if (kDirect && tiles_of<kTokens, kWindow>(a, at.tokens) == 1) return;  // one warp of the cluster has done it all
  __syncthreads();
  constexpr int kVecs = D * kCols / 4 / kAttnThreads;  // a thread's float4s of a part; its columns are the same in all of them
  static_assert(kVecs >= 1 && kAttnThreads * 4 % kCols == 0, "every thread has a share of a part");
  const int col0 = threadIdx.x * 4 % kCols;
  float top[4], sum[4];
  float4 acc[kVecs];
  auto clear = [&]() {
#pragma unroll
    for (int j = 0; j < 4; ++j) top[j] = -INFINITY, sum[j] = 0.0f;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) acc[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  };
  auto merge = [&](int i) {  // one of the CTA's parts
    const float4 *of_ml = reinterpret_cast<const float4 *>(smem + L::kMl + (i * kCols + col0) * 8);
    const float4 p = of_ml[0], q = of_ml[1];
    const float of[4] = {p.x, p.z, q.x, q.z}, s[4] = {p.y, p.w, q.y, q.w};
    const float4 *x = reinterpret_cast<const float4 *>(kDirect || (i & 1) != 0 ? smem + (i >> 1) * L::kRing : smem + L::kParts + (i >> 1) * L::kPart);
    float f[4], f_old[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float high = fmaxf(top[j], of[j]);
      f_old[j] = top[j] == high ? 1.0f : exp2_approx(top[j] - high);  // also where both are -inf
      f[j] = of[j] == high ? 1.0f : exp2_approx(of[j] - high);
      top[j] = high;
      sum[j] = sum[j] * f_old[j] + s[j] * f[j];
    }
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      const float4 w = x[v * kAttnThreads + threadIdx.x];
      acc[v].x = acc[v].x * f_old[0] + w.x * f[0];
      acc[v].y = acc[v].y * f_old[1] + w.y * f[1];
      acc[v].z = acc[v].z * f_old[2] + w.z * f[2];
      acc[v].w = acc[v].w * f_old[3] + w.w * f[3];
    }
  };
  auto write = [&](int seq, int head, int chunk, int vec, const float4 &of) {  // finished elements
    const int cols = min(16, a.group - chunk * 16), d = vec * 4 / kCols;
    __nv_bfloat16 *out = a.out + ((long long)seq * a.heads + head * a.group + chunk * 16 + col0) * D + d;
    const float y[4] = {of.x, of.y, of.z, of.w}, scale = kFp8 ? c.v_scale[head] : 1.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col0 + j < cols) out[j * D] = __float2bfloat16_rn(y[j] * __fdividef(scale, sum[j]));
  };

  if (kDirect) {
    clear();
    for (int i = 0; i < 2 * kAttnWarps; ++i)
      if (info[i].item >= 0) merge(i);
    if (gridDim.x == 1) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v) write(at.seq, at.head, at.chunk, v * kAttnThreads + threadIdx.x, acc[v]);
      return;
    }
    __syncthreads();  // the warps' parts have been read: the CTA's takes their place
    float4 *mine = reinterpret_cast<float4 *>(smem), *mine_ml = reinterpret_cast<float4 *>(smem + L::kMl);
#pragma unroll
    for (int v = 0; v < kVecs; ++v) mine[v * kAttnThreads + threadIdx.x] = acc[v];
    if (threadIdx.x * 4 < kCols) {
      mine_ml[threadIdx.x * 2] = make_float4(top[0], sum[0], top[1], sum[1]);
      mine_ml[threadIdx.x * 2 + 1] = make_float4(top[2], sum[2], top[3], sum[3]);
    }
    __syncwarp();  // a few lanes have stored
    ptx::cluster_sync();
    // the CTAs take turns at 128 of the part's float4s, and sum in rank order
    for (int vec = blockIdx.x * kAttnThreads + threadIdx.x; vec < kVecs * kAttnThreads; vec += gridDim.x * kAttnThreads) {
      float4 p[kAttnClusterMost], q[kAttnClusterMost], x[kAttnClusterMost];
#pragma unroll
      for (int r = 0; r < kAttnClusterMost; ++r)
        if (r < (int)gridDim.x) {
          p[r] = ptx::ld_cluster_f32x4(ptx::smem_u32(mine_ml + col0 / 2), r);
          q[r] = ptx::ld_cluster_f32x4(ptx::smem_u32(mine_ml + col0 / 2 + 1), r);
          x[r] = ptx::ld_cluster_f32x4(ptx::smem_u32(mine + vec), r);
        } else {
          p[r] = q[r] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
          x[r] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
      clear();
#pragma unroll
      for (int r = 0; r < kAttnClusterMost; ++r) {
        top[0] = fmaxf(top[0], p[r].x), top[1] = fmaxf(top[1], p[r].z);
        top[2] = fmaxf(top[2], q[r].x), top[3] = fmaxf(top[3], q[r].z);
      }
      float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int r = 0; r < kAttnClusterMost; ++r) {
        const float of[4] = {p[r].x, p[r].z, q[r].x, q[r].z}, s[4] = {p[r].y, p[r].w, q[r].y, q[r].w};
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] = of[j] == top[j] ? 1.0f : exp2_approx(of[j] - top[j]);
          sum[j] += s[j] * f[j];
        }
        y.x += x[r].x * f[0];
        y.y += x[r].y * f[1];
        y.z += x[r].z * f[2];
        y.w += x[r].w * f[3];
      }
      write(at.seq, at.head, at.chunk, vec, y);
    }
    __syncwarp();
    ptx::cluster_sync();  // a CTA's memory is read until here
    return;
  }

  Part run = {0, -1, 0, 0};  // the item whose parts are being joined: neighbouring ones
  const Part of_lane = info[lane % (2 * kAttnWarps)];
  unsigned places = __ballot_sync(0xffffffffu, lane < 2 * kAttnWarps && of_lane.item >= 0);
  while (true) {
    const int i = __ffs(places) - 1;  // -1: no more
    const int from = max(i, 0);
    const Part now = {__shfl_sync(0xffffffffu, of_lane.seq, from), i < 0 ? -2 : __shfl_sync(0xffffffffu, of_lane.item, from),
                      __shfl_sync(0xffffffffu, of_lane.begins, from), __shfl_sync(0xffffffffu, of_lane.tiles_left, from)};
    places &= places - 1;
    const bool same = now.item == run.item && now.seq == run.seq;
    if (run.item >= 0 && !same) {
      if (run.begins && run.tiles_left == 0) {
        const int head = a.chunks == 1 ? run.item : run.item / a.chunks, chunk = run.item - head * a.chunks;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) write(run.seq, head, chunk, v * kAttnThreads + threadIdx.x, acc[v]);
      } else {
        // the part of an item that began in an earlier CTA goes to this CTA's first place, of one that goes on in a later one to the second
        const int place = 2 * blockIdx.x + (run.begins ? 1 : 0);
        float4 *part = reinterpret_cast<float4 *>(a.parts + place * D * kCols);
#pragma unroll
        for (int v = 0; v < kVecs; ++v) part[v * kAttnThreads + threadIdx.x] = acc[v];
        float4 *ml = reinterpret_cast<float4 *>(a.parts + 2 * gridDim.x * D * kCols + (place * kCols + col0) * 2);
        if (threadIdx.x * 4 < kCols) {
          ml[0] = make_float4(top[0], sum[0], top[1], sum[1]);
          ml[1] = make_float4(top[2], sum[2], top[3], sum[3]);
        }
      }
    }
    if (now.item < 0) break;
    if (!same) {
      clear();
      run = now;
    }
    run.tiles_left = now.tiles_left;
    merge(i);
  }
}

// Joins the parts of the items that begin in one of eight CTAs of the kernel above and go on: a quarter of the floats [element][column].  A
// warp takes an item, or, where one of them has many parts, all warps take the parts of one item after the other in turn, and their sums meet in
// shared memory.  Which items these are follows from the lengths, which are read while the kernel above runs: it lets this one start
// behind its own wait, so what precedes them both is done.
constexpr int kJoinWarps = 8;
constexpr int kJoinSlices = 4;
constexpr int kJoinBatch = 4;  // parts whose loads are in flight together; more would take registers that the kernel above still holds
constexpr int kJoinAlone = 8;  // parts that one warp joins

template <int D, int kCols, bool kFp8, bool kWindow>
__global__ void __launch_bounds__(32 * kJoinWarps) paged_attention_join_kernel(const __grid_constant__ AttnArgs a,
                                                                               const __grid_constant__ PagedCache c, int ctas) {
  constexpr int kTokens = Tile<D, kFp8>::kTokens, kVecs = D * kCols / (128 * kJoinSlices);  // float4s of a lane
  __shared__ float4 accs[kJoinWarps][kVecs][32], sums[kJoinWarps][32], tops[kJoinWarps][32];
  __shared__ int4 items_of[kJoinWarps];  // sequence, head, chunk, parts (0: nothing begins in that CTA and goes on)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, items = c.kv_heads * a.chunks;
  const int base = blockIdx.x * kJoinWarps;
  {
    const List list = list_of<kTokens, kWindow>(a, c, items, kAttnWarps * ctas, lane);
    const int span = list.per * kAttnWarps, from = (base + warp) * span, to = from + span;
    Place at = {0, 0, 0, 0, 0, 0, 0, 0};
    int parts = 0;
    if (base + warp < ctas && to < list.total) {
      const int units = locate<kTokens, kWindow>(at, to, a, c, items, lane), first = to - at.skip + kItemCost;  // unit of the item's first tile
      if (at.skip > 0 && first >= from && first < to) parts = 2 + (units - at.skip - 1) / span;
    }
    if (lane == 0) items_of[warp] = make_int4(at.seq, at.head, at.chunk, parts);
  }
  __syncthreads();
  int most = 0;
#pragma unroll
  for (int i = 0; i < kJoinWarps; ++i) most = max(most, items_of[i].w);
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (most == 0) return;
  const bool many = most > kJoinAlone;
  const int vec = blockIdx.y * kVecs * 32 + lane, col0 = lane * 4 % kCols;
  const float4 *ml = reinterpret_cast<const float4 *>(a.parts + 2LL * ctas * D * kCols);
  const float4 *data = reinterpret_cast<const float4 *>(a.parts);

#pragma unroll 1
  for (int which = many ? 0 : warp; which < (many ? kJoinWarps : warp + 1); ++which) {
    const int4 item = items_of[which];
    if (item.w == 0) continue;
    float top[4], sum[4], acc[kVecs][4];
    auto clear = [&]() {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[j] = 0.0f;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) acc[v][j] = 0.0f;
      }
    };
    clear();
#pragma unroll
    for (int j = 0; j < 4; ++j) top[j] = -INFINITY;
    const int step = many ? kJoinWarps : 1;
    for (int i0 = many ? warp : 0; i0 < item.w; i0 += step * kJoinBatch) {
      float4 p[kJoinBatch], q[kJoinBatch], x[kJoinBatch][kVecs];
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        const int i = i0 + k * step;
        if (i < item.w) {
          // part 0 lies in the second place of the item's first CTA, part i in the first place of the i-th CTA behind it
          const long long place = 2LL * (base + which + i) + (i == 0 ? 1 : 0);
          p[k] = ml[(place * kCols + col0) / 2];
          q[k] = ml[(place * kCols + col0) / 2 + 1];
#pragma unroll
          for (int v = 0; v < kVecs; ++v) x[k][v] = data[place * (D * kCols / 4) + vec + v * 32];
        } else {
          p[k] = q[k] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
#pragma unroll
          for (int v = 0; v < kVecs; ++v) x[k][v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
      }
      float high[4] = {top[0], top[1], top[2], top[3]};
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        high[0] = fmaxf(high[0], p[k].x), high[1] = fmaxf(high[1], p[k].z);
        high[2] = fmaxf(high[2], q[k].x), high[3] = fmaxf(high[3], q[k].z);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = top[j] == high[j] ? 1.0f : exp2_approx(top[j] - high[j]);  // also where both are -inf
        sum[j] *= f;
#pragma unroll
        for (int v = 0; v < kVecs; ++v) acc[v][j] *= f;
        top[j] = high[j];
      }
#pragma unroll
      for (int k = 0; k < kJoinBatch; ++k) {
        const float of[4] = {p[k].x, p[k].z, q[k].x, q[k].z}, s[4] = {p[k].y, p[k].w, q[k].y, q[k].w};
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] = of[j] == top[j] ? 1.0f : exp2_approx(of[j] - top[j]);
          sum[j] += s[j] * f[j];
        }
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          acc[v][0] += x[k][v].x * f[0];
          acc[v][1] += x[k][v].y * f[1];
          acc[v][2] += x[k][v].z * f[2];
          acc[v][3] += x[k][v].w * f[3];
        }
      }
    }
    if (many) {
      __syncthreads();  // the space is free
      tops[warp][lane] = make_float4(top[0], top[1], top[2], top[3]);
      sums[warp][lane] = make_float4(sum[0], sum[1], sum[2], sum[3]);
#pragma unroll
      for (int v = 0; v < kVecs; ++v) accs[warp][v][lane] = make_float4(acc[v][0], acc[v][1], acc[v][2], acc[v][3]);
      __syncthreads();
      if (warp != 0) continue;
#pragma unroll
      for (int w = 1; w < kJoinWarps; ++w) {
        const float4 h = tops[w][lane];
        top[0] = fmaxf(top[0], h.x), top[1] = fmaxf(top[1], h.y), top[2] = fmaxf(top[2], h.z), top[3] = fmaxf(top[3], h.w);
      }
      clear();
#pragma unroll
      for (int w = 0; w < kJoinWarps; ++w) {
        const float4 h = tops[w][lane], s = sums[w][lane];
        const float of[4] = {h.x, h.y, h.z, h.w}, l[4] = {s.x, s.y, s.z, s.w};
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] = of[j] == top[j] ? 1.0f : exp2_approx(of[j] - top[j]);
          sum[j] += l[j] * f[j];
        }
#pragma unroll
        for (int v = 0; v < kVecs; ++v) {
          const float4 x = accs[w][v][lane];
          acc[v][0] += x.x * f[0];
          acc[v][1] += x.y * f[1];
          acc[v][2] += x.z * f[2];
          acc[v][3] += x.w * f[3];
        }
      }
    }
    const int cols = min(16, a.group - item.z * 16);
    __nv_bfloat16 *out = a.out + ((long long)item.x * a.heads + item.y * a.group + item.z * 16 + col0) * D;
    const float scale = kFp8 ? c.v_scale[item.y] : 1.0f;
#pragma unroll
    for (int v = 0; v < kVecs; ++v)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col0 + j < cols) out[j * D + (vec + v * 32) * 4 / kCols] = __float2bfloat16_rn(acc[v][j] * __fdividef(scale, sum[j]));
  }
}

int attn_sm_count() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0 && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) sms[dev] = 148;
  return sms[dev];
}

// The cache as [page][head][half][token][bytes of a half], copied `box` tokens of one half or of all `halves` at a time.
bool encode(CUtensorMap *map, char *base, const PagedCache &c, int size, int box, int halves) {
  const cuuint64_t row = (cuuint64_t)c.head_dim * size, in_half = row < 128 ? row : 128;
  const cuuint64_t dims[5] = {in_half, (cuuint64_t)c.page_size, row / in_half, (cuuint64_t)c.kv_heads, (cuuint64_t)c.pages};
  // a dimension of one element is never stepped along
  const cuuint64_t strides[4] = {c.token_stride > 0 ? (cuuint64_t)c.token_stride : row, 128, c.head_stride > 0 ? (cuuint64_t)c.head_stride : row,
                                 c.page_stride > 0 ? (cuuint64_t)c.page_stride : row};
  const cuuint32_t sizes[5] = {128, (cuuint32_t)box, (cuuint32_t)halves, 1, 1};
  return make_tensor_map(map, 5, base, dims, strides, sizes, CU_TENSOR_MAP_SWIZZLE_128B);
}

unsigned magic_of(int d) { return (unsigned)(((1ULL << 32) + d - 1) / d); }  // for divide(), which does not use it for 1

// CTAs of the direct form's clusters, 0 for the list of tiles; from sizes of tensors alone, so that a captured call keeps its form.  One launch with
// a join in the cluster saves some 4 us of the list's two, but a cluster reads only what its few CTAs can, and more clusters than run at
// once begin one behind the other.  Direct / list, us, 8 heads of 128 in bf16: 1 x 97 tokens 4.1 / 9.0, 1 x 4096 10.9 / 11.7, 1 x 5000 12.4 / 12.1 (10
// tiles per warp, 64 CTAs), 1 x 6000 13.8 / 12.5, 2 x 7000 16.5 / 17.0 (128 CTAs), 8 x 4000 24.1 / 28.0, 64 x 64 9.6 / 11.4, 74 x 400 25.0 / 27.8,
// 90 x 60 13.1 / 12.5 (720 clusters of one CTA), in e4m3 14.0 / 9.6, 128 x 64 16.8 / 11.0, 128 x 256 31.6 / 30.4.
// A cluster has CTAs until its warps have a tile each, as long as SMs are free (1 x 400 tokens 4.9 us, with three tiles each 5.4; in e4m3
// 1 x 700 5.5 and 7.4); two tiles each in a single CTA are as fast, for there the CTAs have nothing to join (1 x 97: 4.1, in two CTAs 4.6); where CTAs
// share an SM four each (4 x 400 6.6, with one 6.9; 16 x 200 7.1 and 7.6).  (Eight warps to a CTA or sixteen CTAs to a cluster: 1 x 4096 10.2 or 9.9
// instead of 10.9, but 1 x 1024 6.5 instead of 5.8, and sixteen clusters of that size do not run at once; four stages instead of two: the same.)
int direct_splits(int seqs, int items, int most_tiles, int ctas) {
  const long long pairs = (long long)seqs * items;
  if (pairs > 2 * ctas || items > 65535 || seqs > 65535) return 0;
  int splits = 1;
  while (splits < kAttnClusterMost && pairs * splits * 2 <= ctas) {
    const int enough = pairs * splits * 4 > ctas ? 4 : splits == 1 ? 2 : 1;  // tiles per warp
    if (most_tiles <= splits * kAttnWarps * enough) break;
    splits *= 2;
  }
  return most_tiles <= splits * kAttnWarps * (pairs * splits * 5 >= 2 * ctas ? kDirectMost : kDirectFew) ? splits : 0;
}

// Tiles that the longest sequence of a table may have.
int tiles_at_most(const PagedCache &c, int tokens, int window, int sinks) {
  const int all = (paged_capacity(c) - 1) / tokens + 1;
  if (window == 0) return all;
  const long long seen = ((long long)sinks + tokens - 1) / tokens + ((long long)window + tokens - 2) / tokens + 1;
  return seen < all ? (int)seen : all;
}

template <int D, bool kFp8, int kCols, bool kWindow>
cudaError_t launch(AttnArgs a, const PagedCache &c, int ctas, cudaStream_t stream) {
  using T = Tile<D, kFp8>;
  constexpr int kSmem = Layout<D, kFp8, kCols, kList>::kTotal;
  int box = c.page_size & -c.page_size;
  if (box > T::kTokens) box = T::kTokens;
  a.box_shift = __builtin_ctz((unsigned)box);
  a.stretches_magic = magic_of(kAttnWarps * ctas);
  a.items_magic = magic_of(c.kv_heads * a.chunks);
  a.page_shift = (c.page_size & (c.page_size - 1)) == 0 ? __builtin_ctz((unsigned)c.page_size) : -1;
  const int halves = box == T::kTokens ? T::kHalves : 1;
  CUtensorMap map_k, map_v;
  if (!encode(&map_k, c.k, c, T::kSize, box, halves) || !encode(&map_v, c.v, c, T::kSize, box, halves)) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kAttnThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int items = c.kv_heads * a.chunks;
  const int splits = direct_splits(a.seqs, items, tiles_at_most(c, T::kTokens, a.window, a.sinks), ctas);
  if (splits > 0) {
    // Three CTAs per SM where two would leave some for a second turn, and three do not (48 x 128 tokens of 8 heads 8.0 instead of 10.7 us; with
    // fewer, or more than three can take, it is slower: 8 x 4000 26.3 instead of 24.2, 64 x 256 18.1 instead of 16.9).
    const long long all = (long long)a.seqs * items * splits;
    const bool three = kCols == 8 && all > ctas && 2 * all <= 3 * ctas;
    const auto kernel = three ? paged_attention_kernel<D, kFp8, kCols, kCols == 8 ? kDirectThree : kDirectTwo, kWindow>
                              : paged_attention_kernel<D, kFp8, kCols, kDirectTwo, kWindow>;
    // (with the smaller form's need three of two's would fit)
    cfg.dynamicSmemBytes = three ? Layout<D, kFp8, kCols, kDirectThree>::kTotal : kSmem;
    static bool ready[2][64] = {};
    const cudaError_t err = allow_smem(kernel, (int)cfg.dynamicSmemBytes, ready[three]);
    if (err != cudaSuccess) return err;
    a.stretch_shift = __builtin_ctz((unsigned)(splits * kAttnWarps));
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)splits;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    if (splits > 1) cfg.numAttrs = 2;
    cfg.gridDim = dim3((unsigned)splits, (unsigned)items, (unsigned)a.seqs);
    return cudaLaunchKernelEx(&cfg, kernel, map_k, map_v, a, c);
  }
  const auto kernel = paged_attention_kernel<D, kFp8, kCols, kList, kWindow>;
  static bool ready[64] = {};
  cudaError_t err = allow_smem(kernel, kSmem, ready);
  if (err != cudaSuccess) return err;
  cfg.gridDim = dim3((unsigned)ctas);
  err = cudaLaunchKernelEx(&cfg, kernel, map_k, map_v, a, c);
  if (err != cudaSuccess) return err;
  cfg.gridDim = dim3((unsigned)((ctas + kJoinWarps - 1) / kJoinWarps), kJoinSlices);
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<D, kCols, kFp8, kWindow>, a, c, ctas);
}

int attn_ctas() { return 2 * attn_sm_count(); }

}  // namespace

size_t paged_attention_workspace_bytes(int heads, const PagedCache &cache, bool fp8, int window, int sinks) {
  const int group = heads / cache.kv_heads, items = cache.kv_heads * ((group + 15) / 16), cols = group <= 8 ? 8 : 16;
  const int tokens = cache.head_dim * (fp8 ? 1 : 2) > 128 ? 16 : 32;  // as Tile has it
  if (direct_splits(cache.seqs, items, tiles_at_most(cache, tokens, window, sinks), attn_ctas()) > 0) return 0;
  return 2 * (size_t)attn_ctas() * cols * (cache.head_dim + 2) * sizeof(float);
}

cudaError_t run_paged_attention(const void *q, long long q_row, long long q_head, int heads, const PagedCache &cache, bool fp8,
                                const int *lengths, float scale, int window, int sinks, void *out, void *workspace, int *error_flag,
                                cudaStream_t stream) {
  const int ctas = attn_ctas(), group = heads / cache.kv_heads, cols = group <= 8 ? 8 : 16, d = cache.head_dim;
  AttnArgs a;
  a.q = static_cast<const __nv_bfloat16 *>(q);
  a.q_row = q_row;
  a.q_head = q_head;
  a.lengths = lengths;
  a.out = static_cast<__nv_bfloat16 *>(out);
  a.parts = static_cast<float *>(workspace);
  a.seqs = cache.seqs;
  a.heads = heads;
  a.group = group;
  a.chunks = (group + 15) / 16;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.window = window;
  a.sinks = sinks;
  a.error_flag = error_flag;
#define SHARQ_ATTN(D, FP8, COLS)            \
  if (d == D && fp8 == FP8 && cols == COLS) \
    return window > 0 ? launch<D, FP8, COLS, true>(a, cache, ctas, stream) : launch<D, FP8, COLS, false>(a, cache, ctas, stream);
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
