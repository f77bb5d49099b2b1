// The split plan: how the rows of a step are cut in chunks for the split kernels (history.hip, compact.hip) and for the
// kernels that reduce their partials.
#pragma once

#include "common.h"

namespace hla {
namespace {

constexpr int kHeads = 16;
constexpr int kTile = 16;
constexpr int kMaxSplits = 1024;

// Split plan shared by the split kernel and the kernels that reduce its partials. Every row of the call is cut in
// chunks of `chunk` 16-row tiles; the grid has S slots per row, and
//   chunk = max(ceil(max_tiles / S), ceil(2 * total_tiles / (T * S)))
// keeps every row within its S slots while about T*S/2 slots get work however ragged the rows are (short rows take
// few slots, long rows many, each holding equal work), and it is at least kMinChunk tiles (kMinChunkSmall in steps
// of fewer than kSmallStepTiles tiles over all rows), or the longest row. Slot s of a row holds tiles
// [s*chunk, (s+1)*chunk); slots past ceil(tiles / chunk) are empty.
//
// The floor: an item's time is a chain of dependent tile steps, its partial costs 16 * (R + 1) fp32 writes and as
// many epilogue reads (as many bytes as a 16-row tile of K and V); a step of many tiles streams, where 8-tile items
// keep that overhead small, and a step of few tiles is latency-bound, where 4-tile items shorten the chain more than
// their partials cost (4-tile items were faster at 256 and 504 tiles per step, 8-tile ones at 1016 and more).
constexpr int kMinChunk = 8, kMinChunkSmall = 4;
constexpr int64_t kSmallStepTiles = 768;
// (a negative length counts as none)
__device__ __forceinline__ int row_tiles(int32_t ctx, int64_t cap) {
  return (int)((min((int64_t)max(ctx, 0), cap) + kTile - 1) / kTile);
}

// Slots of a row that hold work under a plan of `chunk` tiles.
__device__ __forceinline__ int used_slots(int32_t ctx, int64_t cap, int chunk) {
  return (row_tiles(ctx, cap) + chunk - 1) / chunk;
}

// The plan's chunk. Without `fill`, the formula's chunk grows until the step has at most T*S/2 items: the tails of
// ragged rows add up to T more, and the items past T*S/2 (the split counts aim it at two workgroups per CU) would
// give some CUs a third item, on which the whole call waits. With `fill` (the multi-token kernels, launched on a
// grid of one workgroup per (token group, slot) whether the slot has work or not) it is ceil(max_tiles / S)
// instead: the longest row fills all S slots. Must be called by every thread of the block (a multiple of 64
// threads); `red` holds 2 * waves int64.
__device__ int split_chunk(const int32_t* ctx, int T, int64_t cap, int S, int64_t* red, bool fill = false) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const bool one = T <= (int)blockDim.x;  // one row per thread: its tiles stay in a register
  const int my_tiles = tid < T ? row_tiles(ctx[tid], cap) : 0;
  int mx = 0;
  int64_t sum = 0;
  for (int i = tid; i < T; i += blockDim.x) {
    const int tiles = one ? my_tiles : row_tiles(ctx[i], cap);
    mx = max(mx, tiles);
    sum += tiles;
  }
  for (int off = 32; off > 0; off >>= 1) {
    mx = max(mx, __shfl_xor(mx, off));
    sum += __shfl_xor(sum, off);
  }
  if (lane == 0) {
    red[2 * wave] = mx;
    red[2 * wave + 1] = sum;
  }
  __syncthreads();
  int64_t m = 0;
  sum = 0;
  for (int w = 0; w < waves; ++w) {
    m = max(m, red[2 * w]);
    sum += red[2 * w + 1];
  }
  const int64_t slots = (int64_t)T * S;
  int c = (int)max((int64_t)1, fill ? (m + S - 1) / S : max((m + S - 1) / S, (2 * sum + slots - 1) / slots));
  if (fill) return c;
  c = max(c, (int)min(m, (int64_t)(sum < kSmallStepTiles ? kMinChunkSmall : kMinChunk)));
  for (const int64_t target = slots / 2; c < m; ++c) {  // c and the sums are uniform over the block
    int64_t items = 0;
    for (int i = tid; i < T; i += blockDim.x) items += ((one ? my_tiles : row_tiles(ctx[i], cap)) + c - 1) / c;
    for (int off = 32; off > 0; off >>= 1) items += __shfl_xor(items, off);
    __syncthreads();  // every thread has read red
    if (lane == 0) red[wave] = items;
    __syncthreads();
    items = 0;
    for (int w = 0; w < waves; ++w) items += red[w];
    if (items <= target) break;
  }
  __syncthreads();  // red may be reused by the caller
  return c;
}

// Workgroups of the split kernel: the plan puts at most T*S/2 + T (row, chunk) items in the list; a multiple of 8
// (one share per XCD).
__host__ __device__ inline unsigned split_workgroups(int T, int S) {
  return S == 1 ? (unsigned)T : ((unsigned)T * ((S + 1) / 2 + 1) + 7u) / 8u * 8u;
}

// Work item b of the step's list of (row, slot) pairs, rows in order, each row contributing its used slots:
// row = -1 past the end of the list. The split kernel gives item b to the workgroup dispatched b-th, so consecutive
// items land on consecutive XCDs (workgroups are dealt to the XCDs round-robin) and every XCD gets the same share
// of the work, however ragged the rows are. Must be called by every thread (a multiple of 64 threads); `wsum` holds
// one int per wave, `res` two ints.
__device__ void find_item(const int32_t* ctx, int T, int64_t cap, int chunk, int b, int* wsum, int* res, int& row,
                          int& slot) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = blockDim.x;
  const int seg = (T + n - 1) / n, r0 = min(T, tid * seg), r1 = min(T, r0 + seg);
  int cnt = 0;
  for (int r = r0; r < r1; ++r) cnt += used_slots(ctx[r], cap, chunk);
  int x = cnt;  // inclusive scan over the wave
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(x, off);
    if (lane >= off) x += v;
  }
  if (lane == 63) wsum[wave] = x;
  if (tid == 0) res[0] = -1;
  __syncthreads();
  int hi = x;
  for (int w = 0; w < wave; ++w) hi += wsum[w];
  int lo = hi - cnt;
  if (b >= lo && b < hi) {  // exactly one thread owns item b
    for (int r = r0; r < r1; ++r) {
      const int u = used_slots(ctx[r], cap, chunk);
      if (b < lo + u) {
        res[0] = r;
        res[1] = b - lo;
        break;
      }
      lo += u;
    }
  }
  __syncthreads();
  row = res[0];
  slot = res[1];
}

// Plan layout (int32): [0] chunk, [1, 1 + T) used slots per row, then the work items' rows [NI] and slots [NI],
// NI = split_workgroups(T, S); rows past the end of the list are -1.
inline int64_t plan_ints(int T, int S) { return 1 + (int64_t)T + 2 * (int64_t)split_workgroups(T, S); }

}  // namespace
}  // namespace hla
