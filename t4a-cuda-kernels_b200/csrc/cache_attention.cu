// t4a_tree_attention: checks, the choice of the kernel, and the joining of parts.
#include <initializer_list>

#include "attention_launch.h"

namespace t4a {
namespace cache {
namespace {

constexpr int kJoinThreads = 128, kJoinWarps = kJoinThreads / 32;

// Joins the parts of a query row of a head: nothing where one group of the attention had the whole
// unit; zeros where the sequence has nothing to see; else its parts weighed by 2^(lse - max), in a
// fixed order.  kWarps warps take a row's parts in turn: one where units have a few parts, four
// where a long sequence has dozens, which then come in a few rounds of loads.  Launched beside the
// attention, it finds its place on the line of tiles while that runs: the attention lets it start only
// behind its own wait for the kernels before, which may have written the lengths.
template <int kWarps>
__global__ void __launch_bounds__(kJoinThreads) k_join(const AttendArgs a) {
  __shared__ float sums[kWarps == 1 ? 1 : kWarps][kMaxDim], weights[kWarps], tops[kWarps];
  const int lane = threadIdx.x & 31, warp = kWarps == 1 ? 0 : threadIdx.x >> 5, dim = a.cache.dim;
  const unsigned task = blockIdx.x * (kJoinWarps / kWarps) + (kWarps == 1 ? threadIdx.x >> 5 : 0);
  const unsigned rows = static_cast<unsigned>(a.cache.heads) * a.rows;
  const int b = task / rows, in = task - b * rows, head = in / a.rows, row = in - head * a.rows;
  const bool any = b < a.batch;
  const int row_tile = row / a.tile_rows, r = row - row_tile * a.tile_rows;
  const int tiles = any ? sequence_tiles(a, b) : 0;
  const Line line = read_line(a, b);
  const int quota = quota_of(a, line.total), start = line.before + head * tiles;
  const int c0 = start / quota, c1 = tiles == 0 ? c0 : (start + tiles - 1) / quota;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (!any) return;
  const long long to = out_row(a, b, head, row);
  if (tiles == 0) {
    for (int d = 2 * (warp * 32 + lane); d < dim; d += 64 * kWarps) store_out(a, to + d, 0.0f, 0.0f);
    if (warp == 0 && lane == 0) store_lse(a, b, head, row, -INFINITY);
    return;
  }
  if (c0 == c1) return;
  auto part = [&](int c) {
    return ((static_cast<long long>(c) * a.row_tiles + row_tile) * 2 + (c == c0 ? 1 : 0)) * a.tile_rows + r;
  };
  float most = -INFINITY;
  for (int c = c0 + warp * 32 + lane; c <= c1; c += 32 * kWarps) most = fmaxf(most, a.part_lse[part(c)]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
  if constexpr (kWarps > 1) {
    if (lane == 0) tops[warp] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) most = fmaxf(most, tops[w]);
  }
  const float less = most == -INFINITY ? 0.0f : most;
  float x[8], sum = 0.0f;  // columns 2 * lane + 64 * k and the next
#pragma unroll
  for (int k = 0; k < 8; ++k) x[k] = 0.0f;
#pragma unroll 4
  for (int c = c0 + warp; c <= c1; c += kWarps) {
    const long long at = part(c);
    const float w = exp2f(a.part_lse[at] - less);
    sum += w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int d = 2 * lane + 64 * k;
      if (d >= dim) continue;
      const float2 v = *reinterpret_cast<const float2*>(a.part_out + at * dim + d);
      x[2 * k] += w * v.x;
      x[2 * k + 1] += w * v.y;
    }
  }
  if constexpr (kWarps > 1) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      *reinterpret_cast<float2*>(&sums[warp][2 * lane + 64 * k]) = make_float2(x[2 * k], x[2 * k + 1]);
    if (lane == 0) weights[warp] = sum;
    __syncthreads();
    if (warp != 0) return;
    sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      sum += weights[w];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = *reinterpret_cast<const float2*>(&sums[w][2 * lane + 64 * k]);
        x[2 * k] += v.x;
        x[2 * k + 1] += v.y;
      }
    }
  }
  const bool empty = sum == 0.0f;
  const float over = empty ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int d = 2 * lane + 64 * k;
    if (d < dim) store_out(a, to + d, x[2 * k] * over, x[2 * k + 1] * over);
  }
  if (lane == 0) store_lse(a, b, head, row, empty ? -INFINITY : less + log2f(sum));
}

constexpr int kManyTiles = 4096;

struct Choice {
  int padded, row_tiles, rows;  // row_tiles 0: the tensor-memory kernel
};

// The kernel by the query rows of a cache head.  Warp-level products over tiles of 8 rows, as few as
// hold them (2 at most for a dim over 128, whose outputs would not fit the registers), or 128 rows
// in tensor memory, where a dim over 128 does not fit beside a second block.  Measured at 16 ragged
// sequences of up to 4096 tokens, 8 cache heads, dim 128, a call warp-level against one in tensor
// memory: 16-bit cache, 8 rows 44 against 50 us, 12 rows 51 against 50, 16 rows 53 against 50; dim 96, 16
// rows 45 against 50, 24 rows 56 against 51; dim 64, 16 rows 34 against 39, 24 rows 43 against 40.  int8,
// 16 rows 49 against 70, 32 rows 69 against 72, 48 rows 114 against 77; E4M3, 32 rows 74 against 85, 48
// rows 120 against 87.
// At 131072 tokens in int8 and 32 rows: 119 against 166.  What the warp-level kernel pays for a
// unit, joining its warps' outputs, is most of a call whose blocks have a few tiles each, so 17 to 32
// rows of codes go by the tiles that all tables hold (lengths are on the device: a table much wider than
// its sequences goes to the warp-level kernel, however short they are); 8 heads, 32 rows, in E4M3 and in int8: 4 sequences of up
// to 4096 (2048 tiles) 58 against 44 and 52 against 40, 7 of up to 4099 (3640) 64 against 56 and 58
// against 50, 16 of 2048 (4096) 73 against 75 and 67 against 65, 16 of 4096 (8192) 97 against 120 and
// 91 against 104.  (Not at dim 96, which tensor memory pads to 128: 7 of up to 4099 in E4M3 take 52
// against 58; and 44 against 46 at dim 64.)
Choice choose(int kind, int dim, int rows, long long tiles) {
  Choice c;
  c.padded = dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : 256;
  c.row_tiles = rows <= 8 ? 1 : rows <= 16 || c.padded == 256 ? 2 : 4;
  c.rows = 8 * c.row_tiles;
  int most = 8 * most_row_tiles(is_quantised(kind), c.padded);
  if (is_quantised(kind) && c.padded == 128 && tiles < kManyTiles) most = 16;
  if (rows > most && c.padded <= 128) {
    c.padded = dim <= 64 ? 64 : 128;
    c.row_tiles = 0;
    c.rows = kTcTileRows;
  }
  return c;
}

int dispatch(int kind, const AttendArgs& a, const Choice& c, cudaStream_t s, int* blocks) {
  if (c.row_tiles == 0) return launch_tc(kind, a, c.padded, s, blocks);
  switch (kind) {
    case T4A_F16: return launch_mma_f16(a, c.padded, c.row_tiles, s, blocks);
    case T4A_BF16: return launch_mma_bf16(a, c.padded, c.row_tiles, s, blocks);
    case T4A_I8: return launch_mma_i8(a, c.padded, c.row_tiles, s, blocks);
    default: return launch_mma_e4m3(a, c.padded, c.row_tiles, s, blocks);
  }
}

// What does not depend on buffers: shapes, the kernel's choice and its blocks.
int plan_attention(int dtype, const t4a_kv_cache* cache, const t4a_cuda_layout* q, const t4a_cuda_layout* table,
                   bool pointers, AttendArgs* a, Choice* choice, bool* empty) {
  if (dtype != T4A_F16 && dtype != T4A_BF16) return T4A_ERR_UNSUPPORTED_DTYPE;
  T4A_TRY(check_cache(cache, false, pointers, &a->cache));
  if (!is_quantised(cache->kind) && cache->kind != dtype) return T4A_ERR_UNSUPPORTED_DTYPE;
  T4A_TRY(plan::check_layout(q));
  T4A_TRY(plan::check_layout(table));
  if (q->rank != 4 || table->rank != 2) return T4A_ERR_RANK_LENGTH;
  const long long heads = q->extents[1], nodes = q->extents[2], batch = q->extents[3];
  if (q->extents[0] != a->cache.dim || table->extents[1] != batch) return T4A_ERR_SHAPE_MISMATCH;
  *empty = heads == 0 || nodes == 0 || batch == 0;
  if (*empty) return T4A_OK;
  if (a->cache.heads == 0 || heads % a->cache.heads != 0) return T4A_ERR_SHAPE_MISMATCH;
  if (a->cache.page_size == 0) return T4A_ERR_SHAPE_MISMATCH;
  const long long group = heads / a->cache.heads;
  long long rows, all;
  if (plan::mul_overflows(nodes, group, &rows) || plan::mul_overflows(rows, batch, &all)) return T4A_ERR_OVERFLOW;
  if (rows > (1 << 24) || batch > (1 << 24) || table->extents[0] > INT_MAX) return T4A_ERR_DOMAIN_TOO_LARGE;
  a->q_bf16 = dtype == T4A_BF16;
  a->batch = static_cast<int>(batch);
  a->nodes = static_cast<int>(nodes);
  a->group = static_cast<int>(group);
  a->rows = static_cast<int>(rows);
  const long long most_places = INT_MAX - 256;
  const long long places = table->extents[0] > most_places / a->cache.page_size
                               ? most_places
                               : table->extents[0] * a->cache.page_size;
  a->places = a->cache.pages == 0 ? 0 : static_cast<int>(places);
  a->tile_pages = kTile / a->cache.page_size;
  a->tile_places = kTile % a->cache.page_size;
  // The line of tiles is counted in 32 bits.
  long long tiles = (places + kTile - 1) / kTile;
  for (long long by : {batch, static_cast<long long>(a->cache.heads)})
    if (plan::mul_overflows(tiles, by, &tiles)) return T4A_ERR_OVERFLOW;
  if (tiles > INT_MAX || batch * a->cache.heads * a->rows > INT_MAX) return T4A_ERR_DOMAIN_TOO_LARGE;
  *choice = choose(cache->kind, a->cache.dim, a->rows, tiles);
  a->tile_rows = choice->rows;
  a->most_tiles = choice->row_tiles == 0 ? kTcMostTiles : kMmaMostTiles;
  a->row_tiles = (a->rows + choice->rows - 1) / choice->rows;
  int blocks;
  T4A_TRY(dispatch(cache->kind, *a, *choice, nullptr, &blocks));
  a->groups = a->row_tiles < blocks ? blocks / a->row_tiles : 1;
  a->passes = tiles > static_cast<long long>(a->groups) * a->most_tiles;
  return T4A_OK;
}

// Parts, where there is more than one group to share a unit or more than one pass over it.
size_t part_rows(const AttendArgs& a) {
  return a.groups > 1 || a.passes ? static_cast<size_t>(a.groups) * a.row_tiles * 2 * a.tile_rows : 4;
}

size_t workspace_of(const AttendArgs& a) { return part_rows(a) * (a.cache.dim + 1) * sizeof(float); }

}  // namespace
}  // namespace cache
}  // namespace t4a

extern "C" int t4a_tree_attention_workspace_bytes(int dtype, const t4a_kv_cache* cache,
                                                  const t4a_cuda_layout* q_layout,
                                                  const t4a_cuda_layout* table_layout, size_t* bytes) {
  using namespace t4a::cache;
  if (bytes == nullptr) return T4A_ERR_NULL_ARGUMENT;
  AttendArgs a = {};
  Choice choice;
  bool empty;
  T4A_TRY(plan_attention(dtype, cache, q_layout, table_layout, false, &a, &choice, &empty));
  *bytes = empty ? 0 : workspace_of(a);
  return T4A_OK;
}

extern "C" int t4a_tree_attention(void* stream, int dtype, const t4a_kv_cache* cache, void* out,
                                  const t4a_cuda_layout* out_layout, long long out_len, float* lse,
                                  const t4a_cuda_layout* lse_layout, long long lse_len, const void* q,
                                  const t4a_cuda_layout* q_layout, long long q_len, const int* table,
                                  const t4a_cuda_layout* table_layout, long long table_len, const int* context,
                                  const int* nodes, const unsigned char* mask, const t4a_cuda_layout* mask_layout,
                                  long long mask_len, float scale, void* workspace, size_t workspace_bytes) {
  using namespace t4a;
  using namespace t4a::cache;
  AttendArgs a = {};
  Choice choice;
  bool empty;
  T4A_TRY(plan_attention(dtype, cache, q_layout, table_layout, true, &a, &choice, &empty));
  T4A_TRY(check_rows(q_layout, 4, q_len, 2));
  T4A_TRY(check_rows(out_layout, 4, out_len, 2));
  T4A_TRY(check_destination(*out_layout));
  for (int d = 0; d < 4; ++d)
    if (out_layout->extents[d] != q_layout->extents[d]) return T4A_ERR_SHAPE_MISMATCH;
  T4A_TRY(check_tensor(table_layout, 2, table_len, 4));
  if (lse != nullptr) {
    T4A_TRY(check_tensor(lse_layout, 3, lse_len, 4));
    T4A_TRY(check_destination(*lse_layout));
    for (int d = 0; d < 3; ++d)
      if (lse_layout->extents[d] != q_layout->extents[d + 1]) return T4A_ERR_SHAPE_MISMATCH;
    if (!aligned(lse, 4)) return T4A_ERR_INVALID_STRIDE;
    a.lse = lse + lse_layout->offset;
    a.lse_head = lse_layout->strides[0];
    a.lse_node = lse_layout->strides[1];
    a.lse_batch = lse_layout->strides[2];
  }
  if (mask != nullptr) {
    T4A_TRY(check_tensor(mask_layout, 3, mask_len, 1));
    if (mask_layout->extents[0] != q_layout->extents[2] || mask_layout->extents[1] != q_layout->extents[2] ||
        mask_layout->extents[2] != q_layout->extents[3])
      return T4A_ERR_SHAPE_MISMATCH;
    a.mask = mask + mask_layout->offset;
    a.mask_seen = mask_layout->strides[0];
    a.mask_node = mask_layout->strides[1];
    a.mask_batch = mask_layout->strides[2];
  }
  if (empty) return T4A_OK;
  if (q == nullptr || out == nullptr || context == nullptr || (table == nullptr && table_layout->extents[0] != 0))
    return T4A_ERR_NULL_ARGUMENT;
  if (!aligned(q, 2) || !aligned(out, 2) || !aligned(table, 4) || !aligned(context, 4) || !aligned(nodes, 4))
    return T4A_ERR_INVALID_STRIDE;
  if (workspace == nullptr || workspace_bytes < workspace_of(a)) return T4A_ERR_WORKSPACE;
  if (!aligned(workspace, 16)) return T4A_ERR_WORKSPACE;
  a.q = static_cast<const char*>(q) + q_layout->offset * 2;
  a.q_head = q_layout->strides[1];
  a.q_node = q_layout->strides[2];
  a.q_batch = q_layout->strides[3];
  a.out = static_cast<char*>(out) + out_layout->offset * 2;
  a.out_head = out_layout->strides[1];
  a.out_node = out_layout->strides[2];
  a.out_batch = out_layout->strides[3];
  a.q_units = rows_aligned(q, *q_layout, 2, 16);
  a.out_units = rows_aligned(out, *out_layout, 2, 16);
  a.pairs = rows_aligned(q, *q_layout, 2, 4) && rows_aligned(out, *out_layout, 2, 4);
  const Pages &k = a.cache.k, &v = a.cache.v;
  const long long last = (a.cache.pages - 1) * k.page + (a.cache.page_size - 1ll) * k.place + a.cache.dim * 2;
  auto small_scales = [&](const Pages& p) {
    return p.scale_page >= 0 && p.scale_place >= 0 &&
           (a.cache.pages - 1) * p.scale_page + (a.cache.page_size - 1ll) * p.scale_place <= INT_MAX;
  };
  a.plain_copies = k.page == v.page && k.place == v.place && k.page >= 0 && k.place >= 0 &&
                   a.cache.dim == choice.padded && last / 16 < 0xffffffffll && small_scales(k) && small_scales(v);
  a.table = table + table_layout->offset;
  a.table_page = table_layout->strides[0];
  a.table_batch = table_layout->strides[1];
  a.context = context;
  a.live_nodes = nodes;
  a.scale_log2 = static_cast<float>(static_cast<double>(scale) * 1.4426950408889634);
  a.part_out = static_cast<float*>(workspace);
  a.part_lse = a.part_out + part_rows(a) * a.cache.dim;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  T4A_TRY(dispatch(cache->kind, a, choice, s, nullptr));

  // At most so many parts to a unit where all are as long as each other.
  const long long rows = static_cast<long long>(a.batch) * a.cache.heads * a.rows;
  const bool few = a.groups <= 6ll * a.batch * a.cache.heads;
  return runtime::launch_early<AttendArgs>(few ? k_join<1> : k_join<kJoinWarps>,
                                           static_cast<unsigned>(few ? (rows + kJoinWarps - 1) / kJoinWarps : rows),
                                           kJoinThreads, 0, s, a);
}
