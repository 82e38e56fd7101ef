// Pages and places of a step's tokens from the sequences' lengths, in one launch.  16 sequences of one token: 4.1 us (a call takes 6.4 on the
// host); 1000 sequences, 60 prompts: 11.6 us.
//
//   need_i = ceil((length_i + count_i) / P) - ceil(length_i / P),   row r belongs to the i with offsets_i <= r < offsets_i + count_i
//
// The pages that sequence i takes from the stack of free ones, and its rows, lie at prefix sums of need and count over the sequences ahead of it.
// There is next to nothing to read or write: what counts is the chain of dependent steps.  So one cluster does it all, and every CTA of it scans all
// sequences for itself (a thread each, a block's worth at a time) instead of waiting for another's sums; pages and rows are dealt out over the cluster, and found
// by a binary search in the block's sums in shared memory.  Within the cluster, barriers separate what is read from what is overwritten: pages that
// ended sequences give back are on the stack before any is taken, and lengths change when everyone has read them.
#include <cuda_runtime.h>

#include <cstdint>

#include "decode_ops.cuh"
#include "sm100_ptx.cuh"

namespace sharq {

namespace {

constexpr int kPlanThreadsMost = 1024;
constexpr int kPlanCluster = 8, kPlanClusterMost = 16;  // what every GPU of this kind runs, and what most of its GPCs have SMs for

// Sums of what is not negative, 2^31 - 1 where they would be more: what lies beyond is never given, and such sums may be taken in any grouping.
struct Sums {
  int a, b;
};
constexpr int kMost = 0x7fffffff;
__device__ __forceinline__ int plus(int x, int y) { return (int)min((unsigned)x + (unsigned)y, (unsigned)kMost); }

// Inclusive sums over the block's threads; total: of all of them.  scratch: one per warp.
__device__ __forceinline__ Sums block_scan(Sums x, Sums *scratch, Sums *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, x.a, off), b = __shfl_up_sync(0xffffffffu, x.b, off);
    if (lane >= off) x.a = plus(x.a, a), x.b = plus(x.b, b);
  }
  __syncthreads();  // scratch may still be read from the scan before
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  // every warp sums the warps ahead of it by itself
  Sums of = lane < warps ? scratch[lane] : Sums{0, 0};
  Sums ahead = lane < warp ? of : Sums{0, 0};
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    of.a = plus(of.a, __shfl_xor_sync(0xffffffffu, of.a, off));
    of.b = plus(of.b, __shfl_xor_sync(0xffffffffu, of.b, off));
    ahead.a = plus(ahead.a, __shfl_xor_sync(0xffffffffu, ahead.a, off));
    ahead.b = plus(ahead.b, __shfl_xor_sync(0xffffffffu, ahead.b, off));
  }
  *total = of;
  return {plus(x.a, ahead.a), plus(x.b, ahead.b)};
}

// the first of `n` ascending sums that is more than x, which the last one is
__device__ __forceinline__ int first_above(const int *sums, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] > x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int tokens, int page_size) { return tokens == 0 ? 0 : (tokens - 1) / page_size + 1; }

// Rows [from, to) in groups of four that begin at multiples of four, `step` threads apart: fill(row, &position, &sequence) for each in ascending order.
template <typename Fill>
__device__ __forceinline__ void write_rows(const StepPlan &p, int from, int to, int at0, int step, bool aligned, Fill fill) {
  for (long long r0 = (from & ~3) + 4LL * at0; r0 < to; r0 += 4LL * step) {
    int position[4], sequence[4], state = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r0 + k >= from && r0 + k < to) fill((int)r0 + k, &state, &position[k], &sequence[k]);
    if (aligned && r0 >= from && r0 + 4 <= to) {
      *reinterpret_cast<int4 *>(p.positions + r0) = make_int4(position[0], position[1], position[2], position[3]);
      *reinterpret_cast<int4 *>(p.row_sequences + r0) = make_int4(sequence[0], sequence[1], sequence[2], sequence[3]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (r0 + k >= from && r0 + k < to) p.positions[r0 + k] = position[k], p.row_sequences[r0 + k] = sequence[k];
    }
  }
}

__global__ void __launch_bounds__(kPlanThreadsMost) step_plan_kernel(const __grid_constant__ StepPlan p) {
  __shared__ Sums scratch[32];
  __shared__ int need_ends[kPlanThreadsMost], row_ends[kPlanThreadsMost];
  __shared__ int held_of[kPlanThreadsMost], given_of[kPlanThreadsMost];  // given_of: length ahead of the new tokens, -1: nothing is given
  __shared__ int taken;
  const int tid = threadIdx.x, threads = blockDim.x;
  const int rank = blockIdx.x, at0 = rank * threads + tid, step = gridDim.x * threads;
  const long long room = (long long)p.max_pages * p.page_size;
  const int capacity = (int)min(room, (long long)kMost), most = p.max_tokens > 0 ? min(capacity, p.max_tokens) : capacity;
  const bool aligned = ((reinterpret_cast<uintptr_t>(p.positions) | reinterpret_cast<uintptr_t>(p.row_sequences)) & 15) == 0;
  if (tid == 0) taken = 0;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int free_given = *p.free_count;
  bool bad = free_given < 0 || free_given > p.stack_size;
  const bool no_stack = bad;
  int free_now = no_stack ? 0 : free_given;

  if (p.released != nullptr) {  // ended sequences put their pages back, the last page first
    int before = 0;
    for (int i0 = 0; i0 < p.sequences; i0 += threads) {
      const int i = i0 + tid;
      int back = 0;
      if (i < p.sequences && p.released[i] != 0) {
        const int length = p.lengths[i];
        if (length < 0 || length > capacity)
          bad = true;
        else
          back = pages_of(length, p.page_size);
      }
      Sums total;
      const Sums ends = block_scan({back, 0}, scratch, &total);
      need_ends[tid] = ends.a;
      held_of[tid] = back;
      __syncthreads();
      for (int q = at0; q < total.a; q += step) {
        const int s = first_above(need_ends, threads, q);
        const int page = q - (need_ends[s] - held_of[s]);
        const long long to = (long long)free_now + before + need_ends[s] - 1 - page;
        if (!no_stack && to < p.stack_size)
          p.stack[to] = p.table[(long long)(i0 + s) * p.table_stride + page];
        else
          bad = true;
      }
      before = plus(before, total.a);
      __syncthreads();  // the sums have been read
    }
    free_now = no_stack ? 0 : min(plus(free_now, before), p.stack_size);
    if (before > 0) {  // the pages are on the stack before any is taken
      __syncwarp();
      ptx::cluster_sync();
    }
  }

  int need_before = 0, rows_before = 0;
  bool wanting = false;  // pages, for some sequence
  for (int i0 = 0; i0 < p.sequences; i0 += threads) {
    const int i = i0 + tid;
    int length = 0, count = 0, held = 0, need = 0;
    bool fits = false, keeps = true;  // keeps: its length stays as it is
    if (i < p.sequences) {
      length = p.lengths[i];
      count = p.counts[i];
      if (p.released != nullptr && p.released[i] != 0) length = 0, keeps = false;
      fits = length >= 0 && count >= 0 && length <= most && count <= most - length;
      if (!fits && (length != -1 || count != 0)) bad = true;  // -1 may stand for a sequence that takes none, as long as none is asked for
      count = max(count, 0);
      if (fits) {
        held = pages_of(length, p.page_size);
        need = pages_of(length + count, p.page_size) - held;
      }
    }
    Sums total;
    const Sums ends = block_scan({need, count}, scratch, &total);
    const int row_end = plus(rows_before, ends.b), need_end = plus(need_before, ends.a);
    const bool given = fits && !no_stack && (need == 0 || need_end <= free_now) && row_end <= p.rows;
    if (fits && row_end > p.rows) bad = true;
    if (fits && !no_stack && need > 0 && need_end > free_now) wanting = true;
    need_ends[tid] = ends.a;
    row_ends[tid] = ends.b;
    held_of[tid] = held;
    given_of[tid] = given ? length : -1;
    // those that get pages are at the front of those that need some
    const int end_of_warp = __reduce_max_sync(0xffffffffu, given && need > 0 ? need_end : 0);
    if ((tid & 31) == 0 && end_of_warp > 0) atomicMax(&taken, end_of_warp);
    // every CTA has read these sequences' lengths, and the number of free pages
    __syncthreads();
    ptx::cluster_sync();
    if (rank == 0 && i < p.sequences) {
      p.offsets[i + 1] = min(row_end, p.rows);
      if (given)
        p.lengths[i] = length + count;
      else if (!keeps)
        p.lengths[i] = 0;
    }
    const int pages_here = min(total.a, free_now - min(need_before, free_now));
    for (int q = at0; q < pages_here; q += step) {
      const int s = first_above(need_ends, threads, q);
      if (given_of[s] < 0) continue;
      const int start = s > 0 ? need_ends[s - 1] : 0;
      p.table[(long long)(i0 + s) * p.table_stride + held_of[s] + (q - start)] = p.stack[free_now - 1 - need_before - q];
    }
    const int row0 = min(rows_before, p.rows), row1 = min(plus(rows_before, total.b), p.rows);
    write_rows(p, row0, row1, at0, step, aligned, [&](int row, int *s, int *position, int *sequence) {
      const int q = row - row0;
      if (*s < 0)
        *s = first_above(row_ends, threads, q);
      else
        while (row_ends[*s] <= q) ++*s;
      const int start = *s > 0 ? row_ends[*s - 1] : 0;
      *position = given_of[*s] < 0 ? -1 : given_of[*s] + (q - start);
      *sequence = i0 + *s;
    });
    need_before = plus(need_before, total.a);
    rows_before = plus(rows_before, total.b);
    if (i0 + threads < p.sequences) __syncthreads();  // the sums have been read
  }
  write_rows(p, min(rows_before, p.rows), p.rows, at0, step, aligned, [&](int, int *, int *position, int *sequence) {
    *position = -1;
    *sequence = 0;
  });
  if (rank == 0 && tid == 0) {
    p.offsets[0] = 0;
    if (!no_stack) *p.free_count = free_now - taken;
  }
  if ((bad || (wanting && p.strict)) && p.error_flag != nullptr) atomicCAS(p.error_flag, 0, bad ? kBadStepPlan : kPagesShort);
}

}  // namespace

// The cluster's size on this device, asked for once: 16 where such a one runs (1000 sequences with 180000 rows to write 11.6 us instead of 14.0).
static int plan_cluster(const cudaLaunchConfig_t &like) {
  static int sizes[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return kPlanCluster;
  if (sizes[dev] != 0) return sizes[dev];
  int clusters = 0;
  cudaLaunchConfig_t cfg = like;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kPlanClusterMost;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(kPlanClusterMost);
  cfg.blockDim = dim3(kPlanThreadsMost);
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const bool fits = cudaFuncSetAttribute(step_plan_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                    cudaOccupancyMaxActiveClusters(&clusters, step_plan_kernel, &cfg) == cudaSuccess && clusters > 0;
  if (!fits) (void)cudaGetLastError();  // the answer, not an error
  return sizes[dev] = fits ? kPlanClusterMost : kPlanCluster;
}

cudaError_t run_step_plan(const StepPlan &p, cudaStream_t stream) {
  // a thread per sequence as far as a block goes; a cluster where there is more to write than its first CTA does in a few turns
  const int threads = p.sequences <= 128 ? 128 : p.sequences <= 256 ? 256 : 1024;
  const bool wide = (long long)p.rows + p.sequences > 4 * threads;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  const int cluster = wide ? plan_cluster(cfg) : 1;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)cluster);
  cfg.attrs = attr;
  cfg.numAttrs = wide ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, step_plan_kernel, p);
}

}  // namespace sharq
