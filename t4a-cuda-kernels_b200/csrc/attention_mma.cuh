// Attention over the paged cache with warp-level products (mma.sync m16n8k16): the kernel for few
// query rows a cache head, where the cache's bytes bound the call.
//
// A block of 4 warps takes 16 * kRowWarps query rows; kRowWarps warps share a cache row and
// 4 / kRowWarps warps share the tokens of a tile of 64.  Cache rows come by cp.async, 16 bytes a
// lane, into a ring of stages whose row pitch is an odd number of 16-byte units, so that ldmatrix
// meets no bank twice.  With one row warp a warp loads just the tokens that it works on, and no
// block barrier is needed.
//   S = Q K^T, 16 rows x 16 tokens at a time; running maximum m and sum l for each row;
//   O = O * 2^(m_old - m) + 2^(S - m) V
// m moves only where a new maximum exceeds it by 2^8, so the 64 multiplications of O are rare, and
// weights carry a further 2^7: they reach from 2^15 down, so that F16 keeps all bits of those that
// are 2^-21 of the largest.  The quotient O / l depends on neither.
//
// Quantised rows stay codes in shared memory and become F16 in registers, exactly.  K's scale
// multiplies the score.  V's scale is an addend of the exponent, S + log2(scale): the weight that
// meets the codes then is relative to the largest weight * scale of its row, whatever the scales
// are; l adds weight / scale.  Rows with a scale of 0 (or below 2^-107, which the writer does not
// make) count in the softmax alone: they have a maximum and a sum of their own, joined at the end.
// Q is F16 too, times a power of two that brings the row's largest magnitude into [1, 2).
// ldmatrix moves pairs of codes, so a thread's codes are not where 16-bit values would be:
//   K: a thread's 4 neighbouring codes serve as k = 2c, 2c+1, 2c+8, 2c+9, and Q's fragments take
//      the same order;
//   V (transposed): a register holds codes d, d+1 of tokens t, t+1; byte permutes make the pairs
//      (t, t+1) of d and of d+1, the columns of two n-tiles.
#pragma once

#include <cuda_fp8.h>

#include "attention_core.cuh"

namespace t4a {
namespace cache {

constexpr int kMmaThreads = 128;
constexpr float kSlack = 8.0f;  // log2 by which a maximum may exceed the one in use
constexpr float kLift = 7.0f;   // log2 of what all weights carry
constexpr float kLeastScale = 6.1629758e-33f;  // 2^-107

template <int Kind>
struct KindOf {
  static constexpr bool quantised = Kind == T4A_I8 || Kind == T4A_E4M3;
  static constexpr bool bf16 = Kind == T4A_BF16;
  static constexpr int bytes = quantised ? 1 : 2;
};

template <int Kind, int Dim>
struct MmaShape {
  static constexpr int bytes = KindOf<Kind>::bytes;
  static constexpr int pitch = Dim * bytes + 16;  // an odd number of 16-byte units
  static constexpr int chunks = Dim * bytes / 16;
  static constexpr int stage = kTile * pitch * 2 + (KindOf<Kind>::quantised ? kTile * 8 : 0) + 16;
  static constexpr int stages = 3;
  static constexpr int merge = kTile * Dim * 4 + kTile * 16;
  static constexpr int shared = stages * stage > merge ? stages * stage : merge;
  // Blocks that an SM holds: by shared memory (each block costs 1 KB more than it asks for), and at
  // most 3, which leaves a thread 168 registers.
  static constexpr int fit = 233472 / (shared + 1024);
  static constexpr int per_sm = fit < 3 ? fit : 3;
};

__device__ __forceinline__ unsigned shared_at(const void* p) {
  return static_cast<unsigned>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void copy16(unsigned to, const void* from, bool whole) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(whole ? 16 : 0) : "memory");
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
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// Two neighbouring q values, zeros outside the rows.
__device__ __forceinline__ void load_q2(const AttendArgs& a, long long at, float* x, float* y) {
  if (a.q_bf16) {
    const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(a.q) + at;
    if (a.pairs) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
      *x = f.x;
      *y = f.y;
    } else {
      *x = __bfloat162float(p[0]);
      *y = __bfloat162float(p[1]);
    }
  } else {
    const __half* p = static_cast<const __half*>(a.q) + at;
    if (a.pairs) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(p));
      *x = f.x;
      *y = f.y;
    } else {
      *x = __half2float(p[0]);
      *y = __half2float(p[1]);
    }
  }
}

template <int Kind, int Dim, int kRowWarps>
__global__ void __launch_bounds__(kMmaThreads, MmaShape<Kind, Dim>::per_sm) k_attend(const AttendArgs a) {
  using Shape = MmaShape<Kind, Dim>;
  constexpr bool kQuantised = KindOf<Kind>::quantised, kBf16 = KindOf<Kind>::bf16;
  constexpr int kTokenWarps = 4 / kRowWarps, kSubs = kTile / (16 * kTokenWarps), kRows = 16 * kRowWarps;
  constexpr int kSteps = Dim / 16, kStages = Shape::stages;
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row_warp = warp % kRowWarps, token_warp = warp / kRowWarps;
  const int g = lane >> 2, c = lane & 3;  // the thread's rows g and g + 8, and its column pair, in a fragment
  const int dim = a.cache.dim, used = dim * Shape::bytes / 16;

  Cursor at = find_start(a, blockIdx.x);

  auto k_row = [&](int stage, int t) { return smem + stage * Shape::stage + t * Shape::pitch; };
  auto v_row = [&](int stage, int t) { return smem + stage * Shape::stage + (kTile + t) * Shape::pitch; };
  auto scales = [&](int stage) {  // [2][kTile]: K's, V's
    return reinterpret_cast<float*>(smem + stage * Shape::stage + 2 * kTile * Shape::pitch);
  };
  auto seen_bits = [&](int stage) {  // 16 tokens to an entry: which are there
    return reinterpret_cast<unsigned*>(smem + stage * Shape::stage + 2 * kTile * Shape::pitch +
                                       (kQuantised ? kTile * 8 : 0));
  };

  // The pads past dim enter products with zeros of Q, and columns that are not stored; they only
  // have to be finite, once.
  if (dim < Dim) {
    for (int i = threadIdx.x; i < Shape::shared / 16; i += kMmaThreads)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }

  while (at.left > 0) {
    const int b = at.b;
    long long context, length;
    int live;
    sequence_tokens(a, b, &context, &live, &length);
    const int first_row = at.row_tile * kRows + row_warp * 16;
    const long long tile0 = at.tile;
    const int n = static_cast<int>(min(at.left, at.tiles - at.tile));

    // This lane's token of a tile: K's row for the lower half of the warp, V's for the upper.
    const Pages& side = lane < 16 ? a.cache.k : a.cache.v;
    const unsigned char* const head_base = side.base + at.head * side.head;
    const float* const head_scale = kQuantised ? side.scale + at.head * side.scale_head : nullptr;
    auto find_page = [&](int i) {  // the page of the lane's token in tile i, -1 for none
      const long long pos = (tile0 + i) * kTile + 16 * warp + (lane & 15);
      if (i >= n || pos >= length) return -1;
      const int page = a.table[b * a.table_batch +
                               static_cast<long long>(static_cast<unsigned>(pos) / static_cast<unsigned>(a.cache.page_size)) *
                                   a.table_page];
      return page >= 0 && page < a.cache.pages ? page : -1;
    };
    int page_ahead = find_page(0);
    auto issue = [&](int i) {
      const int page = page_ahead;
      page_ahead = find_page(i + 1);
      if (i < n) {
        const int stage = i % kStages;
        const unsigned pos = static_cast<unsigned>((tile0 + i) * kTile) + 16 * warp + (lane & 15);
        const int place = static_cast<int>(pos % static_cast<unsigned>(a.cache.page_size));
        const bool there = page >= 0;
        long long off = 0;
        if (there) off = page * side.page + place * side.place;
        const unsigned bits = __ballot_sync(0xffffffffu, there) & 0xffffu;
        if (lane == 0) seen_bits(stage)[warp] = bits;
        if constexpr (kQuantised)
          copy4(shared_at(scales(stage) + (lane >> 4) * kTile + 16 * warp + (lane & 15)),
                head_scale + (there ? page * side.scale_page + place * side.scale_place : 0), there);
        const unsigned char* const from = head_base + off;
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int u = 0; u < (16 * Shape::chunks + 31) / 32; ++u) {
            const int k = u * 32 + lane, t = k / Shape::chunks, chunk = k - t * Shape::chunks;
            const unsigned char* row = reinterpret_cast<const unsigned char*>(
                __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(from), (s * 16 + t) & 31));
            if ((16 * Shape::chunks % 32 == 0 || k < 16 * Shape::chunks) && chunk < used)
              copy16(shared_at((s ? v_row(stage, 16 * warp + t) : k_row(stage, 16 * warp + t)) + chunk * 16),
                     row + chunk * 16, (bits >> t) & 1);
          }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto sync_tile = [&] {
      if constexpr (kRowWarps == 1) __syncwarp();
      else __syncthreads();
    };

#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) issue(i);

    // Q's fragments, and what turns a product into a base-2 score.
    uint32_t q[kSteps][4];
    float factor[2];
    {
      float most[2] = {0.0f, 0.0f};
      float x[kQuantised ? kSteps : 1][2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = first_row + g + 8 * h;
        const bool live_row = row < a.rows;
        const int node = live_row ? row / a.group : 0, in_group = live_row ? row - node * a.group : 0;
        const long long base = b * a.q_batch + node * a.q_node +
                               (static_cast<long long>(at.head) * a.group + in_group) * a.q_head;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
          float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const int d0 = kQuantised ? 16 * s + 4 * c : 16 * s + 2 * c, d1 = kQuantised ? d0 + 2 : d0 + 8;
          if (live_row && 16 * s < dim) {
            load_q2(a, base + d0, &v[0], &v[1]);
            load_q2(a, base + d1, &v[2], &v[3]);
          }
          if constexpr (kQuantised) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              most[h] = fmaxf(most[h], fabsf(v[e]));
              x[s][h][e] = v[e];
            }
          } else {
            q[s][h] = pack2<kBf16>(v[0], v[1]);
            q[s][2 + h] = pack2<kBf16>(v[2], v[3]);
          }
        }
        factor[h] = a.scale_log2;
        if constexpr (kQuantised) {
          most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 1));
          most[h] = fmaxf(most[h], __shfl_xor_sync(0xffffffffu, most[h], 2));
          int e = static_cast<int>((__float_as_uint(most[h]) >> 23) & 0xff);  // biased exponent
          e = most[h] == 0.0f || e == 0xff ? 127 : min(max(e, 1), 253);
          const float down = __uint_as_float(static_cast<unsigned>(254 - e) << 23);  // 2^(127 - e)
          factor[h] *= __uint_as_float(static_cast<unsigned>(e) << 23);
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            q[s][h] = pack2<false>(x[s][h][0] * down, x[s][h][1] * down);
            q[s][2 + h] = pack2<false>(x[s][h][2] * down, x[s][h][3] * down);
          }
        }
      }
    }

    float o[2 * kSteps][4];
#pragma unroll
    for (int j = 0; j < 2 * kSteps; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float mz[2] = {-INFINITY, -INFINITY}, lz[2] = {0.0f, 0.0f};  // of V rows with a scale of 0

    for (int i = 0; i < n; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      sync_tile();
      issue(i + kStages - 1);
      const int stage = i % kStages;
#pragma unroll 1
      for (int sub = 0; sub < kSubs; ++sub) {
        const int t0 = 16 * (token_warp + kTokenWarps * sub);
        const long long pos0 = (tile0 + i) * kTile + t0;
        const unsigned there = seen_bits(stage)[t0 >> 4];
        if (there == 0) continue;

        float s[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) s[0][e] = s[1][e] = 0.0f;
        if constexpr (!kQuantised) {
          // Matrices: tokens 0-7 and 8-15, each with d 0-7 and 8-15.
          const unsigned from = shared_at(k_row(stage, t0 + (lane & 7) + ((lane >> 4) << 3)) + ((lane >> 3) & 1) * 16);
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            uint32_t r[4];
            ldmatrix4(r, from + k * 32);
            mma<kBf16>(s[0], q[k], r[0], r[1]);
            mma<kBf16>(s[1], q[k], r[2], r[3]);
          }
        } else {
          // Matrices of 8 tokens x 16 codes: two 16-code steps of tokens 0-7, then of tokens 8-15.
          const unsigned from = shared_at(k_row(stage, t0 + (lane & 7) + ((lane >> 4) << 3)) + ((lane >> 3) & 1) * 16);
#pragma unroll
          for (int k = 0; k < kSteps; k += 2) {
            uint32_t r[4], lo, hi;
            ldmatrix4(r, from + k * 16);
            neighbours<Kind>(r[0], &lo, &hi);
            mma<false>(s[0], q[k], lo, hi);
            neighbours<Kind>(r[2], &lo, &hi);
            mma<false>(s[1], q[k], lo, hi);
            neighbours<Kind>(r[1], &lo, &hi);
            mma<false>(s[0], q[k + 1], lo, hi);
            neighbours<Kind>(r[3], &lo, &hi);
            mma<false>(s[1], q[k + 1], lo, hi);
          }
        }

        // Base-2 scores; s[j][2h + e] is row g + 8h, token 8j + 2c + e.
        float per_scale[2][2];
        bool nothing = false;  // a scale of 0 among the thread's tokens
        if constexpr (kQuantised) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int t = t0 + 8 * j + 2 * c + e;
              const float ks = scales(stage)[t], vs = scales(stage)[kTile + t];
              const bool zero = vs < kLeastScale;
              const float lv = zero ? 0.0f : __log2f(vs);
              // A NaN has made the score a NaN where the row is seen, and must not touch l elsewhere.
              per_scale[j][e] = zero ? -1.0f : vs == vs ? exp2_fast(-lv) : 1.0f;
              nothing = nothing || zero;
#pragma unroll
              for (int h = 0; h < 2; ++h) s[j][2 * h + e] = fmaf(s[j][2 * h + e] * ks, factor[h], lv);
            }
          nothing = __any_sync(0xffffffffu, nothing);
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] *= factor[e >> 1];
        }
        const bool partly = there != 0xffffu || pos0 + 16 > context;
        if (partly) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int t = 8 * j + 2 * c + (e & 1);
              const long long drafted = pos0 + t - context;
              bool sees = (there >> t) & 1;
              if (sees && drafted >= 0) {
                const int node = (first_row + g + 8 * (e >> 1)) / a.group;
                sees = node < live && node_sees(a, b, node, static_cast<int>(drafted));
              }
              if (!sees) s[j][e] = -INFINITY;
            }
        }

        if (kQuantised && nothing) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float high = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (per_scale[e >> 1][e & 1] < 0.0f) high = fmaxf(high, s[e >> 1][2 * h + (e & 1)]);
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 1));
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 2));
            const float to = fmaxf(mz[h], high), less = to == -INFINITY ? 0.0f : to;
            lz[h] *= exp2_fast(mz[h] - less);
            mz[h] = to;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (per_scale[e >> 1][e & 1] < 0.0f) {
                float& x = s[e >> 1][2 * h + (e & 1)];
                lz[h] += exp2_fast(x - less);
                x = -INFINITY;
              }
          }
        }

        uint32_t p[4];
        float top[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          top[h] = fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1]));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
          top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] + kSlack || top[1] > m[1] + kSlack)) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float to = fmaxf(m[h], top[h]);
            const float shrink = to == -INFINITY ? 1.0f : exp2_fast(m[h] - to);
            m[h] = to;
            l[h] *= shrink;
#pragma unroll
            for (int j = 0; j < 2 * kSteps; ++j) {
              o[j][2 * h] *= shrink;
              o[j][2 * h + 1] *= shrink;
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float less = m[h] == -INFINITY ? 0.0f : m[h] - kLift;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float w0 = exp2_fast(s[j][2 * h] - less), w1 = exp2_fast(s[j][2 * h + 1] - less);
            if constexpr (kQuantised) l[h] += w0 * per_scale[j][0] + w1 * per_scale[j][1];
            else l[h] += w0 + w1;
            s[j][2 * h] = w0;
            s[j][2 * h + 1] = w1;
            p[2 * j + h] = pack2<kBf16>(w0, w1);
          }
        }

        // Matrices: tokens 0-7 and 8-15 of one 16-byte column, then of the next.
        const unsigned from = shared_at(v_row(stage, t0 + (lane & 7) + (((lane >> 3) & 1) << 3)) + (lane >> 4) * 16);
        bool odd = false;
        if (partly && Kind != T4A_I8) {
          // An infinity or a NaN in a row that some node does not see would reach it as 0 * inf.
#pragma unroll
          for (int k = 0; k < Dim * Shape::bytes / 32; ++k) {
            uint32_t r[4];
            ldmatrix4(r, from + k * 32);
#pragma unroll
            for (int e = 0; e < 4; ++e) odd = odd || odd_values<Kind>(r[e]);
          }
          odd = __any_sync(0xffffffffu, odd);
        }
        if (odd) {
          for (int t = 0; t < 16; ++t) {
            const int j = t >> 3, owner = (lane & ~3) | ((t & 7) >> 1);
            const unsigned char* row = v_row(stage, t0 + t);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float w0 = __shfl_sync(0xffffffffu, j ? s[1][2 * h] : s[0][2 * h], owner);
              const float w1 = __shfl_sync(0xffffffffu, j ? s[1][2 * h + 1] : s[0][2 * h + 1], owner);
              const float w = t & 1 ? w1 : w0;
              const int node = (first_row + g + 8 * h) / a.group;
              const long long drafted = pos0 + t - context;
              const bool sees = ((there >> t) & 1) &&
                                (drafted < 0 || (node < live && node_sees(a, b, node, static_cast<int>(drafted))));
              if (!sees || (kQuantised && w == 0.0f)) continue;
#pragma unroll
              for (int k = 0; k < kSteps; ++k) {
                if (16 * k >= dim) break;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int d0 = kQuantised ? 16 * k + 4 * c + 2 * e : 16 * k + 2 * c + e;
                  const int d1 = kQuantised ? d0 + 1 : d0 + 8;
                  o[2 * k][2 * h + e] += w * row_value<Kind>(row, d0);
                  o[2 * k + 1][2 * h + e] += w * row_value<Kind>(row, d1);
                }
              }
            }
          }
          continue;
        }
        if constexpr (!kQuantised) {
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            uint32_t r[4];
            ldmatrix4_t(r, from + k * 32);
            mma<kBf16>(o[2 * k], p, r[0], r[1]);
            mma<kBf16>(o[2 * k + 1], p, r[2], r[3]);
          }
        } else {
#pragma unroll
          for (int k = 0; k < kSteps; k += 2) {
            uint32_t r[4], even0, odd0, even1, odd1;
            ldmatrix4_t(r, from + k * 16);
            alternate<Kind>(r[0], &even0, &odd0);
            alternate<Kind>(r[1], &even1, &odd1);
            mma<false>(o[2 * k], p, even0, even1);
            mma<false>(o[2 * k + 1], p, odd0, odd1);
            alternate<Kind>(r[2], &even0, &odd0);
            alternate<Kind>(r[3], &even1, &odd1);
            mma<false>(o[2 * k + 2], p, even0, even1);
            mma<false>(o[2 * k + 3], p, odd0, odd1);
          }
        }
      }
    }

    // The token warps' results through shared memory, which the ring no longer needs.
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float* const merged = reinterpret_cast<float*>(smem);  // [kTokenWarps][kRows][Dim]
    float4* const stats = reinterpret_cast<float4*>(smem + kTile * Dim * 4);  // [kTokenWarps][kRows]: m, l, mz, lz
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
        lz[h] += __shfl_xor_sync(0xffffffffu, lz[h], d);
      }
      const int row = token_warp * kRows + row_warp * 16 + g + 8 * h;
      if (c == 0) stats[row] = make_float4(m[h] - kLift, l[h], mz[h], lz[h]);
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        float* to = merged + row * Dim + 16 * k;
        if constexpr (kQuantised) {
          *reinterpret_cast<float4*>(to + 4 * c) =
              make_float4(o[2 * k][2 * h], o[2 * k + 1][2 * h], o[2 * k][2 * h + 1], o[2 * k + 1][2 * h + 1]);
        } else {
          *reinterpret_cast<float2*>(to + 2 * c) = make_float2(o[2 * k][2 * h], o[2 * k][2 * h + 1]);
          *reinterpret_cast<float2*>(to + 8 + 2 * c) = make_float2(o[2 * k + 1][2 * h], o[2 * k + 1][2 * h + 1]);
        }
      }
    }
    __syncthreads();
    const bool begun = tile0 == 0, whole = begun && n == at.tiles;
    const long long part = (static_cast<long long>(blockIdx.x) * 2 + (begun ? 1 : 0)) * kRows;
    const int tile_first = at.row_tile * kRows;
    // A thread takes two columns of a row.
    for (int k = threadIdx.x; k < kRows * (Dim / 2); k += kMmaThreads) {
      const int r = k / (Dim / 2), d = 2 * (k - r * (Dim / 2));
      if (tile_first + r >= a.rows || d >= dim) continue;
      float mo = -INFINITY, ml = -INFINITY;  // references of the output and of the sum
#pragma unroll
      for (int w = 0; w < kTokenWarps; ++w) {
        const float4 st = stats[w * kRows + r];
        mo = fmaxf(mo, st.x);
        ml = fmaxf(ml, kQuantised ? fmaxf(st.x, st.z) : st.x);
      }
      const float less_o = mo == -INFINITY ? 0.0f : mo, less_l = ml == -INFINITY ? 0.0f : ml;
      float ll = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
      for (int w = 0; w < kTokenWarps; ++w) {
        const float4 st = stats[w * kRows + r];
        if (kQuantised && st.w != 0.0f) ll += st.w * exp2_fast(st.z - less_l);
        if (st.x == -INFINITY && st.y == 0.0f) continue;
        const float weight = exp2_fast(st.x - less_o);
        const float2 v = *reinterpret_cast<const float2*>(merged + (w * kRows + r) * Dim + d);
        ll += st.y * exp2_fast(st.x - less_l);
        x += v.x * weight;
        y += v.y * weight;
      }
      const int row = tile_first + r;
      const bool dead = row / a.group >= live || ll == 0.0f;
      const float over = dead ? 0.0f : (mo == ml ? 1.0f : exp2_fast(less_o - less_l)) / ll;
      const float lse2 = dead ? -INFINITY : less_l + log2f(ll);
      x = dead ? 0.0f : x * over;
      y = dead ? 0.0f : y * over;
      if (whole) {
        store_out(a, out_row(a, b, at.head, row) + d, x, y, true);
        if (d == 0) store_lse(a, b, at.head, row, lse2);
      } else {
        *reinterpret_cast<float2*>(a.part_out + (part + r) * dim + d) = make_float2(x, y);
        if (d == 0) a.part_lse[part + r] = lse2;
      }
    }
    __syncthreads();
    at.left -= n;
    if (at.left > 0) next_unit(a, &at);
  }
}

}  // namespace cache
}  // namespace t4a
