// What the kernels of t4a_tree_attention share: the arguments, the division of the work, and the
// joining of parts.
//
// A unit is one cache head of one sequence.  Its cache rows come in tiles of kTile tokens, and all
// units' tiles lie end to end on one line, of which every group of blocks takes an equal stretch, so
// a ragged batch, a single long sequence and a large batch load the SMs alike.  A group has a block
// for each tile of a head's query rows (row r of a head: node r / group, head-in-group r % group):
// its blocks pass over the same cache rows together, and all but one find them in L2.  A unit that
// several groups share leaves parts (its output over the part's own softmax sum, and the base-2 log of
// that sum); k_join weighs them by 2^(lse - max) in a fixed order.  No atomics: the same inputs
// give the same bits.
//
// A product's sums are truncated, not rounded, so that they fall behind by up to half a unit of the last
// place with every addition: 2048 tiles in a row lost 2.0e-4 of an output in the warp-level kernel and
// 8.4e-4, four additions a tile, in the one on tensor memory.  A block therefore makes a pass of at most
// kMmaMostTiles or kTcMostTiles (6e-5 either), and adds up a unit's passes, rounded, in the place of its part.
// A pass more is a prologue and an epilogue more: 32 sequences of 64-node trees over 16384 tokens, some 570
// tiles a block in tensor memory, take 1040 us for the 1004 of one pass a unit.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "cache_plan.h"

namespace t4a {
namespace cache {

constexpr int kTile = 64;
constexpr int kMmaMostTiles = 512, kTcMostTiles = 128;  // of a pass

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
  int places;       // table pages * page_size, or the most that 32 bits allow
  int most_tiles;   // of a pass
  int passes;       // whether the tables are long enough for a block to have more than one over a unit
  int tile_pages, tile_places;  // kTile / page_size and kTile % page_size
  int q_bf16;      // q and out are BF16, else F16
  int plain_copies;  // K and V have the same strides, rows fill the padded dim, and offsets fit 32 bits
  int q_units, out_units;  // q and out rows start on 16-byte boundaries
  int pairs;       // q and out rows start on 4-byte boundaries
  float* part_out;  // [groups][row_tiles][2][tile_rows][dim]
  float* part_lse;  // [groups][row_tiles][2][tile_rows]
  int groups;       // of row_tiles blocks each
};

// Tokens that sequence b's rows can see: committed ones, and all with the drafted ones.  Places
// are below 2^31 - 2^8, so that 32-bit arithmetic holds a tile past the end.
__device__ __forceinline__ void sequence_tokens(const AttendArgs& a, int b, int* context, int* live, int* length) {
  const int c = max(0, a.context[b]), n = a.live_nodes ? min(max(0, a.live_nodes[b]), a.nodes) : a.nodes;
  *context = min(c, a.places);
  *live = n;
  *length = static_cast<int>(min(static_cast<long long>(c) + n, static_cast<long long>(a.places)));
}

__device__ __forceinline__ int sequence_tiles(const AttendArgs& a, int b) {
  int context, live, length;
  sequence_tokens(a, b, &context, &live, &length);
  return live == 0 ? 0 : (length + kTile - 1) / kTile;  // no live row: nothing to attend
}

// A block's place on the line of tiles.
struct Cursor {
  int b, head, row_tile;
  int tile, tiles;  // within the unit
  int from;         // where the block's part of the unit begins
  int left;         // of the block's stretch
};

// Tiles of all units, and of those of the sequences before `upto`.  Called by whole warps; all
// lanes get the same.  The planner keeps the number of tiles below 2^31.
struct Line {
  int total, before;
};

__device__ __forceinline__ Line read_line(const AttendArgs& a, int upto) {
  const int lane = threadIdx.x & 31, units = a.cache.heads;
  Line n = {};
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane, mine = b < a.batch ? sequence_tiles(a, b) * units : 0;
    n.total += __reduce_add_sync(0xffffffffu, mine);
    n.before += __reduce_add_sync(0xffffffffu, b < upto ? mine : 0);
  }
  return n;
}

__device__ __forceinline__ int quota_of(const AttendArgs& a, int total) {
  return max(1, (total + a.groups - 1) / a.groups);
}

// The start of a block's stretch (left 0 where it has none).
__device__ __forceinline__ Cursor find_start(const AttendArgs& a, int block) {
  const int lane = threadIdx.x & 31, units = a.cache.heads, group = block / a.row_tiles;
  Cursor c = {};
  c.row_tile = block - group * a.row_tiles;
  int total = 0, kept = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    kept = b < a.batch ? sequence_tiles(a, b) * units : 0;
    total += __reduce_add_sync(0xffffffffu, kept);
  }
  const int quota = quota_of(a, total);
  const long long far = static_cast<long long>(quota) * group;
  if (far >= total) return c;
  const int start = static_cast<int>(far);
  c.left = min(quota, total - start);
  int before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const int b = b0 + lane;
    const int mine = a.batch <= 32 ? kept : b < a.batch ? sequence_tiles(a, b) * units : 0;
    int sum = mine;  // inclusive prefix
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += o;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + sum > start);
    if (past) {
      const int at = __ffs(past) - 1;
      c.tiles = __shfl_sync(0xffffffffu, mine, at) / units;
      const int in = start - before - __shfl_sync(0xffffffffu, sum - mine, at), unit = in / c.tiles;
      c.b = b0 + at;
      c.tile = c.from = in - unit * c.tiles;
      c.head = unit;
      return c;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  c.left = 0;
  return c;
}

// Tiles of the pass that begins at the cursor.
__device__ __forceinline__ int pass_tiles(const AttendArgs& a, const Cursor& c) {
  return min(min(c.left, c.tiles - c.tile), a.most_tiles);
}

// Past a pass of n tiles: the unit's next one, or the next unit with tiles, if any are left.
__device__ __forceinline__ void next_pass(const AttendArgs& a, Cursor* c, int n) {
  c->left -= n;
  c->tile += n;
  if (c->left <= 0 || c->tile < c->tiles) return;
  c->tile = c->from = 0;
  if (++c->head < a.cache.heads) return;
  c->head = 0;
  do ++c->b;
  while (c->b < a.batch && (c->tiles = sequence_tiles(a, c->b)) == 0);
}

__device__ __forceinline__ bool node_sees(const AttendArgs& a, int b, int i, int j) {
  if (a.mask == nullptr) return j <= i;
  return a.mask[b * a.mask_batch + i * a.mask_node + j * a.mask_seen] != 0;
}

// Two neighbouring values of out, the first at an even column.
__device__ __forceinline__ void store_out(const AttendArgs& a, long long at, float x, float y) {
  if (a.q_bf16) {
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + at;
    if (a.pairs) {
      *reinterpret_cast<__nv_bfloat162*>(o) = __floats2bfloat162_rn(x, y);
    } else {
      o[0] = __float2bfloat16_rn(x);
      o[1] = __float2bfloat16_rn(y);
    }
  } else {
    __half* o = static_cast<__half*>(a.out) + at;
    if (a.pairs) {
      *reinterpret_cast<__half2*>(o) = __floats2half2_rn(x, y);
    } else {
      o[0] = __float2half_rn(x);
      o[1] = __float2half_rn(y);
    }
  }
}

// How a pass's results join those of the passes before it, whose sum's logarithm is `before`: both
// times a weight.  *lse: the pass's, then that of all.
__device__ __forceinline__ void join_passes(float before, float* lse, float* keep, float* add) {
  const float most = fmaxf(before, *lse), less = most == -INFINITY ? 0.0f : most;
  *keep = exp2f(before - less);
  *add = exp2f(*lse - less);
  const float sum = *keep + *add, over = sum == 0.0f ? 0.0f : 1.0f / sum;
  *keep *= over;
  *add *= over;
  *lse = sum == 0.0f ? -INFINITY : less + log2f(sum);
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
