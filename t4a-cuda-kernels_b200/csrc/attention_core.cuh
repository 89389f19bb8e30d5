// What the kernels of t4a_tree_attention share: the arguments, the division of the work, and the
// joining of parts.
//
// A unit is one cache head of one sequence with a tile of its query rows (row r of a head: node
// r / group, head-in-group r % group).  Its cache rows come in tiles of kTile tokens.  All units'
// tiles lie end to end on one line, and every block takes an equal stretch of it, so a ragged
// batch, a single long sequence and a large batch load the SMs alike.  A unit that several
// blocks share leaves parts (its output over the part's own softmax sum, and the base-2 log of
// that sum); k_join weighs them by 2^(lse - max) in a fixed order.  No atomics: the same inputs
// give the same bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "cache_plan.h"

namespace t4a {
namespace cache {

constexpr int kTile = 64;

struct AttendArgs {
  View cache;
  const void* q;
  long long q_head, q_node, q_batch;  // strides in elements
  void* out;
  long long out_head, out_node, out_batch;
  float* lse;
  long long lse_head, lse_node, lse_batch;
  const int* table;
  long long table_page, table_batch;
  const int* context;
  const int* live_nodes;
  const unsigned char* mask;
  long long mask_seen, mask_node, mask_batch;
  float scale_log2;  // scale * log2(e)
  int batch, nodes, group, rows;  // rows = nodes * group
  int row_tiles, tile_rows;
  int table_pages;
  int q_bf16;      // q and out are BF16, else F16
  int pairs;       // q and out rows start on 4-byte boundaries
  float* part_out;  // [blocks][2][tile_rows][dim]
  float* part_lse;  // [blocks][2][tile_rows]
  int blocks;
};

// Tokens that sequence b's rows can see: committed ones, and all with the drafted ones.
__device__ __forceinline__ void sequence_tokens(const AttendArgs& a, int b, long long* context, int* live,
                                                long long* length) {
  const long long places = static_cast<long long>(a.table_pages) * a.cache.page_size;
  const long long c = max(0, a.context[b]);
  const int n = a.live_nodes ? min(max(0, a.live_nodes[b]), a.nodes) : a.nodes;
  *context = min(c, places);
  *live = n;
  *length = min(c + n, places);
}

__device__ __forceinline__ long long sequence_tiles(const AttendArgs& a, int b) {
  long long context, length;
  int live;
  sequence_tokens(a, b, &context, &live, &length);
  return live == 0 ? 0 : (length + kTile - 1) / kTile;  // no live row: nothing to attend
}

// Tiles of all units, and of those of the sequences before `upto`.  Called by whole warps.
__device__ __forceinline__ void count_tiles(const AttendArgs& a, int upto, long long* total, long long* before) {
  const int lane = threadIdx.x & 31;
  const long long units = static_cast<long long>(a.cache.heads) * a.row_tiles;
  long long t = 0, p = 0;
  for (int b = lane; b < a.batch; b += 32) {
    const long long n = sequence_tiles(a, b) * units;
    t += n;
    if (b < upto) p += n;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    t += __shfl_xor_sync(0xffffffffu, t, d);
    p += __shfl_xor_sync(0xffffffffu, p, d);
  }
  *total = t;
  *before = p;
}

__device__ __forceinline__ long long quota_of(const AttendArgs& a, long long total) {
  return max(1ll, (total + a.blocks - 1) / a.blocks);
}

// A block's place on the line of tiles.
struct Cursor {
  int b, head, row_tile;
  long long tile, tiles;  // within the unit
  long long left;         // of the block's stretch
};

// The start of block `block`'s stretch (left 0 where it has none).  Called by whole warps; all
// lanes get the same.
__device__ __forceinline__ Cursor find_start(const AttendArgs& a, int block) {
  const int lane = threadIdx.x & 31;
  const long long units = static_cast<long long>(a.cache.heads) * a.row_tiles;
  long long total, unused;
  count_tiles(a, 0, &total, &unused);
  const long long quota = quota_of(a, total), start = quota * block;
  Cursor c = {};
  c.left = max(0ll, min(quota, total - start));
  if (c.left == 0) return c;
  long long before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    const long long mine = b < a.batch ? sequence_tiles(a, b) * units : 0;
    long long sum = mine;  // inclusive prefix
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + sum > start);
    if (past) {
      const int at = __ffs(past) - 1;
      const long long tiles = __shfl_sync(0xffffffffu, mine, at) / units;
      const long long in = start - before - __shfl_sync(0xffffffffu, sum - mine, at);
      c.b = b0 + at;
      c.tiles = tiles;
      const long long unit = in / tiles;
      c.tile = in - unit * tiles;
      c.head = static_cast<int>(unit / a.row_tiles);
      c.row_tile = static_cast<int>(unit - static_cast<long long>(c.head) * a.row_tiles);
      return c;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  c.left = 0;
  return c;
}

// The next unit with tiles; called with left > 0, so there is one.
__device__ __forceinline__ void next_unit(const AttendArgs& a, Cursor* c) {
  c->tile = 0;
  if (++c->row_tile < a.row_tiles) return;
  c->row_tile = 0;
  if (++c->head < a.cache.heads) return;
  c->head = 0;
  do ++c->b;
  while (c->b < a.batch && (c->tiles = sequence_tiles(a, c->b)) == 0);
}

__device__ __forceinline__ bool node_sees(const AttendArgs& a, int b, int i, int j) {
  if (a.mask == nullptr) return j <= i;
  return a.mask[b * a.mask_batch + i * a.mask_node + j * a.mask_seen] != 0;
}

__device__ __forceinline__ void store_out(const AttendArgs& a, long long at, float x, float y, bool two) {
  if (a.q_bf16) {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + at;
    if (a.pairs && two) {
      *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(x, y);
    } else {
      o[0] = __float2bfloat16_rn(x);
      if (two) o[1] = __float2bfloat16_rn(y);
    }
  } else {
    __half* o = static_cast<__half*>(a.out) + at;
    if (a.pairs && two) {
      *reinterpret_cast<__half2*>(o) = __floats2half2_rn(x, y);
    } else {
      o[0] = __float2half_rn(x);
      if (two) o[1] = __float2half_rn(y);
    }
  }
}

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ long long out_row(const AttendArgs& a, int b, int head, int row) {
  const int node = row / a.group, in_group = row - node * a.group;
  return b * a.out_batch + node * a.out_node + (static_cast<long long>(head) * a.group + in_group) * a.out_head;
}

__device__ __forceinline__ void store_lse(const AttendArgs& a, int b, int head, int row, float lse2) {
  if (a.lse == nullptr) return;
  const int node = row / a.group, in_group = row - node * a.group;
  a.lse[b * a.lse_batch + node * a.lse_node + (static_cast<long long>(head) * a.group + in_group) * a.lse_head] =
      lse2 * kLn2;
}

}  // namespace cache
}  // namespace t4a
