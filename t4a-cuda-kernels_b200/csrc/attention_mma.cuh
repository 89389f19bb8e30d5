// Attention over the paged cache with warp-level products (mma.sync m16n8k16): the kernel for few
// query rows a cache head, where the cache's bytes bound the call.
//
// Products are transposed: 16 tokens (or 16 columns of V) are the wide side of a product and 8
// query rows the narrow one, so that 8 rows, a decoding step's group, waste nothing:
//   S^T = K Q^T    [16 tokens x 8 rows]
//   O^T = V^T P^T  [16 columns x 8 rows], P^T from S^T by an 8x8 transpose of registers (movmatrix)
// and each code that a warp unpacks serves all kRowTiles * 8 rows.  A running maximum m and sum l
// for each row;  O = O * 2^(m_old - m) + 2^(S - m) V.  m moves only where a new maximum exceeds it
// by 2^8, so the multiplications of O are rare, and weights carry a further 2^7: they reach from
// 2^15 down, so that F16 keeps all bits of those that are 2^-21 of the largest.  O / l depends on
// neither.  Weights take V's 16-bit type, F16 over codes, since both operands of a product have one: an
// output is off by its unit roundoff of sum w|v| at most.  l adds them as they were, in F32, so that the
// log-sum-exp has no part in that.
//
// Each of a block's 4 warps takes 16 of a tile's 64 tokens, and copies just these (cp.async, 16
// bytes a lane) into its part of a ring of stages; no warp waits for another within a unit.  The
// row pitch is an odd number of 16-byte units, so that ldmatrix meets no bank twice.
//
// Quantised rows stay codes in shared memory and become F16 in registers, exactly.  K's scale
// multiplies the score.  V's scale is an addend of the exponent, S + log2(scale): the weight that
// meets the codes then is relative to the largest weight * scale of its row; l adds weight / scale.
// The weight becomes 0 from 2^-133 of the largest down, so while the scales of the seen rows lie within
// 2^90 of one another, what l loses is 2^-43 of its largest term.  Rows with a scale of 0 (or below 2^-110, which the writer does not
// make) count in the softmax alone: they have a maximum and a sum of their own, joined at the end.
// Q is F16 too.  BF16 rows become it exactly from 2^-17 up and within 2^-25 below, so a row whose
// largest magnitude is outside [1/4, 2^15) is first brought to [2^14, 2^15) by a power of two of its own,
// which its scores are multiplied by again: a row keeps 23 bits of its largest, whatever the block's
// other rows hold.  Rows without a live node are zeros.
// 32 sequences of up to 8192 tokens in I8, 4 rows a cache head, 353 MB: 70 us, 5.0 TB/s, 0.77 of a
// copy's rate; the issue slots are 0.60 taken, DRAM reads 364 MB.  8 nodes over 131072 tokens in
// I8, 32 rows, 277 MB: 120 us; there the unpacking and 64 products to 16 tokens with two blocks an
// SM bound it (issue 0.43, most stalls on fixed latencies).  One token over 1000, BF16: 8.6 us.
// ldmatrix moves pairs of codes, so a thread's codes are not where 16-bit values would be:
//   K: a thread's 4 neighbouring codes serve as k = 2c, 2c+1, 2c+8, 2c+9, and Q has the same order;
//   V (transposed): a register holds codes d, d+1 of tokens t, t+1; byte permutes make the pairs
//      (t, t+1) of d and of d+1, rows g and g + 8 of a product.
#pragma once

#include <cuda_fp8.h>

#include "attention_core.cuh"

namespace t4a {
namespace cache {

constexpr int kMmaThreads = 128;
constexpr float kSlack = 8.0f;  // log2 by which a maximum may exceed the one in use
constexpr float kLift = 7.0f;   // log2 of what all weights carry
constexpr float kLeastScale = 7.7037198e-34f;  // 2^-110: the writer's least is 2^-100 / 448

template <int Kind>
struct KindOf {
  static constexpr bool quantised = Kind == T4A_I8 || Kind == T4A_E4M3;
  static constexpr bool bf16 = Kind == T4A_BF16;
  static constexpr int bytes = quantised ? 1 : 2;
};

template <int Kind, int Dim, int kRowTiles>
struct MmaShape {
  static constexpr int bytes = KindOf<Kind>::bytes;
  static constexpr int rows = 8 * kRowTiles;
  static constexpr int pitch = Dim * bytes + 16;  // an odd number of 16-byte units
  static constexpr int chunks = Dim * bytes / 16;
  static constexpr int stage = kTile * pitch * 2 + (KindOf<Kind>::quantised ? kTile * 8 : 0) + 16;
  // Codes: two stages and four blocks an SM, 75 us for 32 sequences of up to 8192 tokens where three
  // and three took 80; 16-bit rows keep more bytes on their way in two blocks of three.
  static constexpr int stages = bytes == 1 ? 2 : 3;
  static constexpr int q_pitch = Dim * 2 + 16;
  static constexpr int q_bytes = rows * q_pitch + rows * 4;  // and a power of two for each
  static constexpr int out_pitch = Dim + 4;  // floats: the lanes of a store meet 32 banks
  static constexpr int merge = 4 * rows * (out_pitch * 4 + 16);
  static constexpr int ring = stages * stage > merge ? stages * stage : merge;
  static constexpr int shared = ring + q_bytes;
  // Blocks that an SM holds: by shared memory (each block costs 1 KB more than it asks for) and by
  // the registers that O takes.
  static constexpr int fit = 233472 / (shared + 1024);
  static constexpr int by_registers = kRowTiles == 4 || Dim * kRowTiles >= 512 ? 2 : Dim * kRowTiles >= 192 ? 3 : 4;
  static constexpr int per_sm = fit < by_registers ? fit : by_registers;
  // Q's fragments stay in registers where they are few.
  static constexpr bool hold_q = kRowTiles * Dim <= 256;
};

__device__ __forceinline__ unsigned shared_at(const void* p) {
  return static_cast<unsigned>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void copy16(unsigned to, const void* from, bool whole) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(whole ? 16 : 0) : "memory");
}

__device__ __forceinline__ void copy16(unsigned to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

__device__ __forceinline__ void copy4(unsigned to, const void* from, bool whole) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(whole ? 4 : 0) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}

__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], unsigned at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}

template <bool Bf16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Bf16)
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The first product of a sum.
template <bool Bf16>
__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Bf16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

template <bool Bf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (Bf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Two codes in the bytes that `Lo` and `Hi` name of r, as F16.  I8: 0x6400 | u is 1024 + u, so the
// code biased by 128 less 1152 is the code.
template <int Lo, int Hi>
__device__ __forceinline__ uint32_t int8_pair(uint32_t biased) {
  const uint32_t r = __byte_perm(biased, 0x64646464u, Lo | 0x40 | (Hi << 8) | 0x4000);
  const uint32_t minus = 0x64806480u;  // 1152
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&r), *reinterpret_cast<const __half2*>(&minus));
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t e4m3_pair(uint32_t codes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<unsigned short>(codes)));
  return r;
}

// Codes 0, 1 and 2, 3 of r.
template <int Kind>
__device__ __forceinline__ void neighbours(uint32_t r, uint32_t* p01, uint32_t* p23) {
  if constexpr (Kind == T4A_I8) {
    const uint32_t u = r ^ 0x80808080u;
    *p01 = int8_pair<0, 1>(u);
    *p23 = int8_pair<2, 3>(u);
  } else {
    *p01 = e4m3_pair(r);
    *p23 = e4m3_pair(r >> 16);
  }
}

// Codes 0, 2 and 1, 3 of r.
template <int Kind>
__device__ __forceinline__ void alternate(uint32_t r, uint32_t* p02, uint32_t* p13) {
  if constexpr (Kind == T4A_I8) {
    const uint32_t u = r ^ 0x80808080u;
    *p02 = int8_pair<0, 2>(u);
    *p13 = int8_pair<1, 3>(u);
  } else {
    const uint32_t u = __byte_perm(r, 0, 0x3120);
    *p02 = e4m3_pair(u);
    *p13 = e4m3_pair(u >> 16);
  }
}

// A value of a V row in shared memory, for the rare path.
template <int Kind>
__device__ __forceinline__ float row_value(const unsigned char* row, int d) {
  if constexpr (Kind == T4A_I8) return static_cast<float>(reinterpret_cast<const signed char*>(row)[d]);
  else if constexpr (Kind == T4A_E4M3) {
    __nv_fp8_e4m3 f;
    f.__x = row[d];
    return static_cast<float>(f);
  } else if constexpr (Kind == T4A_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[d]);
  else return __half2float(reinterpret_cast<const __half*>(row)[d]);
}

// Whether a register of 16-bit values or of codes holds an infinity or a NaN.
template <int Kind>
__device__ __forceinline__ bool odd_values(uint32_t r) {
  if constexpr (Kind == T4A_I8) return false;
  else if constexpr (Kind == T4A_E4M3) return __vcmpeq4(r & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
  else if constexpr (Kind == T4A_BF16) return (r & 0x7f80u) == 0x7f80u || (r & 0x7f800000u) == 0x7f800000u;
  else return (r & 0x7c00u) == 0x7c00u || (r & 0x7c000000u) == 0x7c000000u;
}

// 8x8 16-bit values across the warp, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

__device__ __forceinline__ float load_q(const AttendArgs& a, long long at) {
  return a.q_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[at])
                  : __half2float(static_cast<const __half*>(a.q)[at]);
}

// The unit's live query rows into shared memory [rows][Dim], 16 bits, in the order of K's fragments, and
// over codes what each row's scores are to be multiplied by; returns whether some row of the warp's
// has another such factor than 1.  A warp takes every fourth row.
template <int Kind, int Dim, int kRowTiles>
__device__ __forceinline__ bool stage_q(const AttendArgs& a, int b, int head, int first_row, int live,
                                        unsigned char* q_rows, float* row_factor) {
  using Shape = MmaShape<Kind, Dim, kRowTiles>;
  constexpr int kEach = Dim / 32, kMine = Shape::rows / 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float x[kMine][kEach];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int row = first_row + warp + 4 * i, node = row / a.group;
    const long long base = b * a.q_batch + node * a.q_node +
                           (static_cast<long long>(head) * a.group + (row - node * a.group)) * a.q_head;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int d = lane + 32 * k;
      x[i][k] = row < a.rows && node < live && d < a.cache.dim ? load_q(a, base + d) : 0.0f;
    }
  }
  bool shifted = false;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    float down = 1.0f;
    if (KindOf<Kind>::quantised && a.q_bf16) {
      float most = 0.0f;
#pragma unroll
      for (int k = 0; k < kEach; ++k)
        if (fabsf(x[i][k]) < INFINITY) most = fmaxf(most, fabsf(x[i][k]));
      most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most)));
      if (most != 0.0f && (most < 0.25f || most >= 32768.0f)) {
        const int e = max(static_cast<int>(__float_as_uint(most) >> 23), 16);  // biased exponent
        down = __uint_as_float(static_cast<unsigned>(min(127 + 14 + 127 - e, 253)) << 23);  // 2^(14 - (e - 127))
        shifted = true;
      }
    }
    if (KindOf<Kind>::quantised && lane == 0) row_factor[warp + 4 * i] = 1.0f / down;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int d = lane + 32 * k, in = d & 15;
      const int slot = KindOf<Kind>::quantised ? (d & ~15) + 2 * (in >> 2) + (in & 1) + ((in & 2) << 2) : d;
      unsigned char* const q_row = q_rows + (warp + 4 * i) * Shape::q_pitch;
      if constexpr (KindOf<Kind>::bf16) reinterpret_cast<__nv_bfloat16*>(q_row)[slot] = __float2bfloat16_rn(x[i][k]);
      else reinterpret_cast<__half*>(q_row)[slot] = __float2half_rn(x[i][k] * down);
    }
  }
  return shifted;
}

template <int Kind, int Dim, int kRowTiles>
__global__ void __launch_bounds__(kMmaThreads, MmaShape<Kind, Dim, kRowTiles>::per_sm) k_attend(const AttendArgs a) {
  using Shape = MmaShape<Kind, Dim, kRowTiles>;
  constexpr bool kQuantised = KindOf<Kind>::quantised, kBf16 = KindOf<Kind>::bf16;
  constexpr int kSteps = Dim / 16, kStages = Shape::stages, kRows = Shape::rows;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, c = lane & 3;
  const int dim = a.cache.dim, used = dim * Shape::bytes / 16;
  unsigned char* const q_rows = smem + Shape::ring;
  float* const row_factor = reinterpret_cast<float*>(q_rows + kRows * Shape::q_pitch);

  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Cursor at = find_start(a, blockIdx.x);

  // A stage: K's rows, V's rows, K's and V's scales, and for each warp which of its tokens are there.
  unsigned char* const my_rows = smem + 16 * warp * Shape::pitch;
  constexpr int kV = kTile * Shape::pitch, kScales = 2 * kTile * Shape::pitch;
  constexpr int kSeen = kScales + (kQuantised ? kTile * 8 : 0);

  // The pads past dim meet zeros of Q, or make columns that are not stored; they only have to be
  // finite, also after a unit's results have passed through the ring.
  auto clear_pads = [&] {
    if (dim == Dim) return;
    for (int i = threadIdx.x; i < Shape::ring / 16; i += kMmaThreads)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  };
  clear_pads();

  while (at.left > 0) {
    const int b = at.b;
    int context, live, length;
    sequence_tokens(a, b, &context, &live, &length);
    const int first_row = at.row_tile * kRows;
    const int tile0 = at.tile, n = pass_tiles(a, at);

    // This lane's token of a tile: K's row for the lower half of the warp, V's for the upper.
    const Pages& side = lane < 16 ? a.cache.k : a.cache.v;
    const unsigned char* const k_base = a.cache.k.base + at.head * a.cache.k.head;
    const unsigned char* const v_base = a.cache.v.base + at.head * a.cache.v.head;
    const float* const head_scale = kQuantised ? side.scale + at.head * side.scale_head : nullptr;
    // 32-bit strides, in 16-byte units and in scales, where plain copies serve.
    const unsigned page_units = static_cast<unsigned>(side.page >> 4), place_units = static_cast<unsigned>(side.place >> 4);
    const int scale_page = static_cast<int>(side.scale_page), scale_place = static_cast<int>(side.scale_place);
    const int* const my_table = a.table + b * a.table_batch;
    int pos = tile0 * kTile + 16 * warp + (lane & 15);  // of the next page to look up
    int in_table = pos / a.cache.page_size, place = pos - in_table * a.cache.page_size;
    const int end = min(length, (tile0 + n) * kTile);
    int page_ahead, place_ahead;  // of the next tile to copy
    auto look_up = [&] {
      page_ahead = -1;
      place_ahead = place;
      if (pos < end) page_ahead = my_table[in_table * a.table_page];
      pos += kTile;
      in_table += a.tile_pages;
      place += a.tile_places;
      if (place >= a.cache.page_size) {
        place -= a.cache.page_size;
        ++in_table;
      }
    };
    int to_stage = 0;
    auto issue = [&](bool any) {
      const int page = page_ahead, at_place = place_ahead;
      look_up();
      if (any) {
        unsigned char* const stage = smem + to_stage * Shape::stage;
        const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(a.cache.pages);
        const unsigned bits = __ballot_sync(0xffffffffu, there) & 0xffffu;
        if (lane == 0) reinterpret_cast<unsigned*>(stage + kSeen)[warp] = bits;
        const unsigned to = shared_at(my_rows + to_stage * Shape::stage);
        const unsigned scale_to = shared_at(stage + kScales + ((lane >> 4) * kTile + 16 * warp + (lane & 15)) * 4);
        if (a.plain_copies && bits == 0xffffu) {
          // All tokens are there, K and V lie alike, and 16-byte units of an offset fit 32 bits.
          const unsigned units = page * page_units + at_place * place_units;
          if constexpr (kQuantised) copy4(scale_to, head_scale + page * scale_page + at_place * scale_place, true);
#pragma unroll
          for (int u = 0; u < 16 * Shape::chunks / 32; ++u) {
            const int k = u * 32 + lane, t = k / Shape::chunks, chunk = k - t * Shape::chunks;
            const unsigned long long from =
                static_cast<unsigned long long>(__shfl_sync(0xffffffffu, units, t) + chunk) * 16;
            copy16(to + t * Shape::pitch + chunk * 16, k_base + from);
            copy16(to + kV + t * Shape::pitch + chunk * 16, v_base + from);
          }
        } else {
          const long long off = there ? page * side.page + at_place * side.place : 0;
          if constexpr (kQuantised)
            copy4(scale_to, head_scale + (there ? page * side.scale_page + at_place * side.scale_place : 0), there);
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll 4
            for (int u = 0; u < 16 * Shape::chunks / 32; ++u) {
              const int k = u * 32 + lane, t = k / Shape::chunks, chunk = k - t * Shape::chunks;
              const long long from = __shfl_sync(0xffffffffu, off, s * 16 + t);
              if (chunk < used)
                copy16(to + s * kV + t * Shape::pitch + chunk * 16, (s ? v_base : k_base) + from + chunk * 16,
                       (bits >> t) & 1);
            }
        }
      }
      to_stage = to_stage + 1 == kStages ? 0 : to_stage + 1;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    look_up();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i < n);

    const float factor = a.scale_log2;
    const bool shifted =
        __syncthreads_or(stage_q<Kind, Dim, kRowTiles>(a, b, at.head, first_row, live, q_rows, row_factor));
    // Q's fragments: [n = row g][k = 2c, 2c+1] and [k = 2c+8, 2c+9] of each step.
    uint32_t q[Shape::hold_q ? kSteps : 1][kRowTiles][2];
    const unsigned q_at = shared_at(q_rows) + (lane & 7) * Shape::q_pitch + (lane >> 3) * 16;
    if constexpr (Shape::hold_q) {
#pragma unroll
      for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
        for (int k = 0; k < kSteps; k += 2) {
          uint32_t r[4];
          ldmatrix4(r, q_at + j * 8 * Shape::q_pitch + k * 32);
          q[k][j][0] = r[0];
          q[k][j][1] = r[1];
          q[k + 1][j][0] = r[2];
          q[k + 1][j][1] = r[3];
        }
    }
    float o[kSteps][kRowTiles][4];  // [columns g / g + 8][rows 2c, 2c + 1]
#pragma unroll
    for (int k = 0; k < kSteps; ++k)
#pragma unroll
      for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[k][j][e] = 0.0f;
    // Of rows 8j + 2c + e, l a lane's own part, the others the same in all lanes of a row: at what
    // score the reference m moves, m + kSlack, and what weights are relative to, m - kLift.
    float moves[kRowTiles][2], l[kRowTiles][2], less[kRowTiles][2];
    float mz[kQuantised ? kRowTiles : 1][2], lz[kQuantised ? kRowTiles : 1][2];  // of V rows with a scale of 0
#pragma unroll
    for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        moves[j][e] = -INFINITY;
        l[j][e] = 0.0f;
        less[j][e] = 0.0f;
        if constexpr (kQuantised) {
          mz[j][e] = -INFINITY;
          lz[j][e] = 0.0f;
        }
      }

    int from_stage = 0;
    int pos0 = tile0 * kTile + 16 * warp;
    for (int i = 0; i < n; ++i, pos0 += kTile) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();
      issue(i + kStages - 1 < n);
      const unsigned char* const stage = smem + from_stage * Shape::stage;
      const unsigned rows_at = shared_at(my_rows + from_stage * Shape::stage);
      from_stage = from_stage + 1 == kStages ? 0 : from_stage + 1;
      const unsigned there = reinterpret_cast<const unsigned*>(stage + kSeen)[warp];
      if (there == 0) continue;

      float s[kRowTiles][4];  // tokens g / g + 8, rows 2c, 2c + 1
      // Matrices: tokens 0-7 and 8-15 of one 16-byte column, then of the next.
      const unsigned k_at = rows_at + (lane & 15) * Shape::pitch + (lane >> 4) * 16;
      auto times_q = [&](int k, const uint32_t(&x)[4]) {
        if constexpr (Shape::hold_q) {
#pragma unroll
          for (int j = 0; j < kRowTiles; ++j) {
            if (k == 0) mma_first<kBf16>(s[j], x, q[k][j][0], q[k][j][1]);
            else mma<kBf16>(s[j], x, q[k][j][0], q[k][j][1]);
          }
        } else {
          // Two row tiles to an ldmatrix: rows 0-7 and 8-15, each k 0-7 and 8-15.
#pragma unroll
          for (int j = 0; j < kRowTiles; j += 2) {
            uint32_t r[4];
            ldmatrix4(r, shared_at(q_rows) + (8 * j + (lane & 7) + ((lane >> 4) << 3)) * Shape::q_pitch +
                             ((lane >> 3) & 1) * 16 + k * 32);
            if (k == 0) {
              mma_first<kBf16>(s[j], x, r[0], r[1]);
              mma_first<kBf16>(s[j + 1], x, r[2], r[3]);
            } else {
              mma<kBf16>(s[j], x, r[0], r[1]);
              mma<kBf16>(s[j + 1], x, r[2], r[3]);
            }
          }
        }
      };
      if constexpr (!kQuantised) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t r[4];
          ldmatrix4(r, k_at + k * 32);
          times_q(k, r);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kSteps; k += 2) {
          uint32_t r[4], x[4];
          ldmatrix4(r, k_at + k * 16);
          neighbours<Kind>(r[0], &x[0], &x[2]);
          neighbours<Kind>(r[1], &x[1], &x[3]);
          times_q(k, x);
          neighbours<Kind>(r[2], &x[0], &x[2]);
          neighbours<Kind>(r[3], &x[1], &x[3]);
          times_q(k + 1, x);
        }
      }

      // Base-2 scores; s[j][2h + e] is token g + 8h, row 8j + 2c + e.
      float per_scale[2];
      bool nothing = false;  // a scale of 0 among the thread's tokens
      if constexpr (kQuantised) {
        const float* const scales = reinterpret_cast<const float*>(stage + kScales) + 16 * warp + g;
        float ks[2], lv[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float vs = scales[kTile + 8 * h];
          const bool zero = fabsf(vs) < kLeastScale;
          ks[h] = scales[8 * h] * factor;
          lv[h] = zero ? 0.0f : __log2f(vs);
          // A NaN, also of a scale below zero, has made the score a NaN where the row is seen, and must
          // not touch l elsewhere.
          per_scale[h] = zero ? -1.0f : lv[h] == lv[h] ? exp2_fast(-lv[h]) : 1.0f;
          nothing = nothing || zero;
        }
        if (!shifted) {
#pragma unroll
          for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = fmaf(s[j][e], ks[e >> 1], lv[e >> 1]);
        } else {
#pragma unroll
          for (int j = 0; j < kRowTiles; ++j) {
            const float2 f = *reinterpret_cast<const float2*>(row_factor + 8 * j + 2 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = fmaf(s[j][e], ks[e >> 1] * (e & 1 ? f.y : f.x), lv[e >> 1]);
          }
        }
        nothing = __any_sync(0xffffffffu, nothing);
      } else {
#pragma unroll
        for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] *= factor;
      }
      // Whether row 8j + 2c + e sees token t of the 16.
      auto sees = [&](int t, int j, int e) {
        if (!((there >> t) & 1)) return false;
        const int drafted = pos0 + t - context;
        if (drafted < 0) return true;
        const int node = (first_row + 8 * j + 2 * c + e) / a.group;
        return node < live && drafted < live && node_sees(a, b, node, drafted);
      };
      const bool partly = there != 0xffffu || pos0 + 16 > context;
      if (partly) {
#pragma unroll
        for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!sees(g + 8 * (e >> 1), j, e & 1)) s[j][e] = -INFINITY;
      }

      if (kQuantised && nothing) {
#pragma unroll
        for (int j = 0; j < (kQuantised ? kRowTiles : 0); ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float high = -INFINITY;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (per_scale[h] < 0.0f) high = fmaxf(high, s[j][2 * h + e]);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
            const float to = fmaxf(mz[j][e], high), base = to == -INFINITY ? 0.0f : to;
            lz[j][e] *= exp2_fast(mz[j][e] - base);
            mz[j][e] = to;
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (per_scale[h] < 0.0f) {
                lz[j][e] += exp2_fast(s[j][2 * h + e] - base);
                s[j][2 * h + e] = -INFINITY;
              }
          }
      }

      float top[kRowTiles][2];
      bool rises = false;
#pragma unroll
      for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float t = fmaxf(s[j][e], s[j][2 + e]);
          rises = rises || t > moves[j][e];
          top[j][e] = t;
        }
      if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
        for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top[j][e] = fmaxf(top[j][e], __shfl_xor_sync(0xffffffffu, top[j][e], d));
            const float from = moves[j][e] - kSlack, to = fmaxf(from, top[j][e]);
            const float shrink = to == -INFINITY ? 1.0f : exp2_fast(from - to);
            moves[j][e] = to + kSlack;
            less[j][e] = to == -INFINITY ? 0.0f : to - kLift;
            l[j][e] *= shrink;
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
              o[k][j][e] *= shrink;
              o[k][j][2 + e] *= shrink;
            }
          }
      }
      uint32_t p[kRowTiles][2];  // [k = tokens 2c, 2c+1 / + 8][n = row g]
#pragma unroll
      for (int j = 0; j < kRowTiles; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float w = exp2_fast(s[j][2 * h + e] - less[j][e]);
            s[j][2 * h + e] = w;
            if constexpr (kQuantised) l[j][e] = fmaf(w, per_scale[h], l[j][e]);
            else l[j][e] += w;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) p[j][h] = transpose8(pack2<kBf16>(s[j][2 * h], s[j][2 * h + 1]));
      }

      // 16-bit matrices: d 0-7 and 8-15 of tokens 0-7, then of tokens 8-15.  Codes: tokens 0-7 and
      // 8-15 of 16 codes, then of the next 16.
      const unsigned v_at =
          kQuantised ? rows_at + kV + (lane & 15) * Shape::pitch + (lane >> 4) * 16
                     : rows_at + kV + ((lane & 7) + ((lane >> 4) << 3)) * Shape::pitch + ((lane >> 3) & 1) * 16;
      if (Kind != T4A_I8 && partly) {
        // An infinity or a NaN in a row that some node does not see would reach it as 0 * inf.
        bool odd = false;
#pragma unroll
        for (int k = 0; k < Dim * Shape::bytes / 32; ++k) {
          uint32_t r[4];
          ldmatrix4(r, v_at + k * 32);
#pragma unroll
          for (int e = 0; e < 4; ++e) odd = odd || odd_values<Kind>(r[e]);
        }
        if (__any_sync(0xffffffffu, odd)) {
          for (int t = 0; t < 16; ++t) {
            const unsigned char* const row = my_rows + (stage - smem) + kV + t * Shape::pitch;
#pragma unroll
            for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float w =
                    __shfl_sync(0xffffffffu, t < 8 ? s[j][e] : s[j][2 + e], (t & 7) * 4 + c);
                if (!sees(t, j, e) || (kQuantised && w == 0.0f)) continue;
#pragma unroll
                for (int k = 0; k < kSteps; ++k) {
                  if (16 * k >= dim) break;
                  o[k][j][e] += w * row_value<Kind>(row, 16 * k + (kQuantised ? 2 * g : g));
                  o[k][j][2 + e] += w * row_value<Kind>(row, 16 * k + (kQuantised ? 2 * g + 1 : g + 8));
                }
              }
          }
          continue;
        }
      }
      if constexpr (!kQuantised) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          uint32_t r[4];
          ldmatrix4_t(r, v_at + k * 32);
#pragma unroll
          for (int j = 0; j < kRowTiles; ++j) mma<kBf16>(o[k][j], r, p[j][0], p[j][1]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kSteps; k += 2) {
          uint32_t r[4], x[4];
          ldmatrix4_t(r, v_at + k * 16);
          alternate<Kind>(r[0], &x[0], &x[1]);
          alternate<Kind>(r[1], &x[2], &x[3]);
#pragma unroll
          for (int j = 0; j < kRowTiles; ++j) mma<false>(o[k][j], x, p[j][0], p[j][1]);
          alternate<Kind>(r[2], &x[0], &x[1]);
          alternate<Kind>(r[3], &x[2], &x[3]);
#pragma unroll
          for (int j = 0; j < kRowTiles; ++j) mma<false>(o[k + 1][j], x, p[j][0], p[j][1]);
        }
      }
    }

    // The warps' results through shared memory, which the ring no longer needs.
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float* const merged = reinterpret_cast<float*>(smem);  // [4][kRows][out_pitch]
    float4* const stats = reinterpret_cast<float4*>(smem + 4 * kRows * Shape::out_pitch * 4);  // m, l, mz, lz
#pragma unroll
    for (int j = 0; j < kRowTiles; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = warp * kRows + 8 * j + 2 * c + e;
        float4 st = make_float4(moves[j][e] == -INFINITY ? -INFINITY : less[j][e], l[j][e], -INFINITY, 0.0f);
        if constexpr (kQuantised) {
          st.z = mz[j][e];
          st.w = lz[j][e];
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          st.y += __shfl_xor_sync(0xffffffffu, st.y, d);
          if constexpr (kQuantised) st.w += __shfl_xor_sync(0xffffffffu, st.w, d);
        }
        if (g == 0) stats[row] = st;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
          float* const to = merged + row * Shape::out_pitch + 16 * k;
          to[kQuantised ? 2 * g : g] = o[k][j][e];
          to[kQuantised ? 2 * g + 1 : g + 8] = o[k][j][2 + e];
        }
      }
    __syncthreads();
    // Whether the block has the unit's first tile, and all; whether passes came before this one.
    const bool begun = at.from == 0, whole = begun && tile0 + n == at.tiles, again = tile0 != at.from;
    const long long part = (static_cast<long long>(blockIdx.x) * 2 + (begun ? 1 : 0)) * kRows;
    // What the warps' outputs of row r are relative to, their common factor, and the log of the sum.
    struct RowSum {
      float less, over, lse2;
    };
    auto sum_of = [&](int r) {
      float mo = -INFINITY, ml = -INFINITY;  // references of the output and of the sum
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float4 st = stats[w * kRows + r];
        mo = fmaxf(mo, st.x);
        ml = fmaxf(ml, kQuantised ? fmaxf(st.x, st.z) : st.x);
      }
      const float less_o = mo == -INFINITY ? 0.0f : mo, less_l = ml == -INFINITY ? 0.0f : ml;
      float ll = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float4 st = stats[w * kRows + r];
        if (kQuantised && st.w != 0.0f) ll += st.w * exp2_fast(st.z - less_l);
        if (st.x == -INFINITY && st.y == 0.0f) continue;
        ll += st.y * exp2_fast(st.x - less_l);
      }
      const bool dead = (first_row + r) / a.group >= live || ll == 0.0f;
      return RowSum{less_o, dead ? 0.0f : (mo == ml ? 1.0f : exp2_fast(less_o - less_l)) / ll,
                    dead ? -INFINITY : less_l + log2f(ll)};
    };
    auto store_sum = [&](int r, float lse2) {
      if (whole) store_lse(a, b, at.head, first_row + r, lse2);
      else a.part_lse[part + r] = lse2;
    };
    // A thread takes two columns of a row.
    for (int k = threadIdx.x; k < kRows * (Dim / 2); k += kMmaThreads) {
      const int r = k / (Dim / 2), d = 2 * (k - r * (Dim / 2));
      if (first_row + r >= a.rows || d >= dim) continue;
      RowSum sum = sum_of(r);
      float x = 0.0f, y = 0.0f;
      if (sum.over != 0.0f) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float4 st = stats[w * kRows + r];
          if (st.x == -INFINITY && st.y == 0.0f) continue;
          const float weight = exp2_fast(st.x - sum.less);
          const float2 v = *reinterpret_cast<const float2*>(merged + (w * kRows + r) * Shape::out_pitch + d);
          x += v.x * weight;
          y += v.y * weight;
        }
        x *= sum.over;
        y *= sum.over;
      }
      float2* const kept = reinterpret_cast<float2*>(a.part_out + (part + r) * dim + d);
      if (again) {
        float keep, add;
        join_passes(a.part_lse[part + r], &sum.lse2, &keep, &add);
        const float2 before = *kept;
        x = before.x * keep + x * add;
        y = before.y * keep + y * add;
      }
      if (whole) store_out(a, out_row(a, b, at.head, first_row + r) + d, x, y);
      else *kept = make_float2(x, y);
      if (d == 0 && !again) store_sum(r, sum.lse2);
    }
    __syncthreads();
    if (again) {  // the sums before have been read
      if (threadIdx.x < kRows && first_row + threadIdx.x < a.rows) {
        RowSum sum = sum_of(threadIdx.x);
        float keep, add;
        join_passes(a.part_lse[part + threadIdx.x], &sum.lse2, &keep, &add);
        store_sum(threadIdx.x, sum.lse2);
      }
      __syncthreads();
    }
    next_pass(a, &at, n);
    if (at.left > 0) clear_pads();
  }
}

}  // namespace cache
}  // namespace t4a
