// Rows into and out of the paged cache (t4a_cache_write, t4a_cache_read).
//
// A row is dim <= 256 values, 16 to a thread: a group of 1, 2, 4, 8 or 16 neighbouring lanes
// holds it in registers, so a quantised row is read once, its largest magnitude is a shuffle
// tree over the group, and its codes leave as one 16-byte store a thread.
//   write: a = max |x|, scale = a * (1/Q), code = nearest(x * (Q/a))
//   read:  x = code * scale
// A thread has the same part of a K row and of a V row: both loads are under way before the first
// is used, and the slot's page and place are found once (60 -> 49 us for the reads below).
// Both are bound by memory.  32768 rows of 8 heads x 128 from BF16 to E4M3, 203 MB: 39 us, 5.2 TB/s,
// 0.79 of a copy's rate (its arithmetic takes 0.72 of the issue slots; magnitudes compared as bits
// in packed pairs and integers rounded by an addition brought it from 57 us).  50001 such rows back
// to BF16, 311 MB: 48 us, 6.4 TB/s, 0.98.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "cache_plan.h"
#include "runtime.h"

namespace t4a {
namespace cache {
namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 16;               // values of a row that a thread holds
constexpr float kLeastRow = 7.8886091e-31f;  // 2^-100: Q / a stays finite above it

// What one launch does: rows x heads rows of K and of V.
struct RowsArgs {
  View cache;
  unsigned char* act[2];  // key and value rows
  long long act_head[2], act_row[2];  // strides in bytes
  const void* slots;
  long long slot_stride;
  long long tasks;  // rows * heads
  int wide_index;
  int group_shift;  // log2 of the lanes of a row
};

__device__ __forceinline__ long long load_slot(const RowsArgs& a, long long n) {
  return a.wide_index ? static_cast<const long long*>(a.slots)[n * a.slot_stride]
                      : static_cast<long long>(static_cast<const int*>(a.slots)[n * a.slot_stride]);
}

// 32-byte loads and stores (sm_100's widest).
__device__ __forceinline__ void load32(const void* p, uint32_t (&r)[8]) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p));
}

__device__ __forceinline__ void store32(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// 16 values of type T at p as F32; `Vec`: p is 32-byte aligned.
template <typename T, bool Vec>
__device__ __forceinline__ void load16(const unsigned char* p, float (&x)[kPerThread]) {
  if constexpr (Vec && sizeof(T) == 2) {
    uint32_t r[8];
    load32(p, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T* h = reinterpret_cast<const T*>(&r[i]);
      x[2 * i] = static_cast<float>(h[0]);
      x[2 * i + 1] = static_cast<float>(h[1]);
    }
  } else if constexpr (Vec) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t r[8];
      load32(p + 32 * half, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[8 * half + i] = __uint_as_float(r[i]);
    }
  } else {
    const T* t = reinterpret_cast<const T*>(p);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) x[i] = static_cast<float>(t[i]);
  }
}

template <typename T>
__device__ __forceinline__ T rounded(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

template <typename T, bool Vec>
__device__ __forceinline__ void store16(unsigned char* p, const float (&x)[kPerThread]) {
  if constexpr (Vec && sizeof(T) == 2) {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      T h[2] = {rounded<T>(x[2 * i]), rounded<T>(x[2 * i + 1])};
      r[i] = *reinterpret_cast<const uint32_t*>(h);
    }
    store32(p, r);
  } else if constexpr (Vec) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(x[8 * half + i]);
      store32(p + 32 * half, r);
    }
  } else {
    T* t = reinterpret_cast<T*>(p);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) t[i] = rounded<T>(x[i]);
  }
}

// The two 8-bit codes.
struct Int8 {
  static constexpr float kMost = 127.0f;
  // |x| <= 127.00001: adding 1.5 * 2^23 leaves the nearest integer, ties to even, in the low bits.
  static __device__ __forceinline__ uint32_t encode4(const float* x) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(__fadd_rn(x[i], 12582912.0f));
    return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
  }
  static __device__ __forceinline__ void decode4(uint32_t r, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<signed char>(r >> (8 * i)));
  }
};

struct E4m3 {
  static constexpr float kMost = 448.0f;
  static __device__ __forceinline__ uint32_t encode4(const float* x) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  static __device__ __forceinline__ void decode4(uint32_t r, float* x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(r >> (16 * i)), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};

// Where a thread's row lies: its activation rows, its slot split into page and place.  A thread has
// the same part of K's row and of V's, so that both loads are on their way before the first is
// used.  Rows run head by head, as activations usually lie.
struct Place {
  long long page, n;
  int place, head, lane;
  bool live, inside;
};

__device__ __forceinline__ Place find(const RowsArgs& a) {
  Place w;
  w.lane = threadIdx.x & ((1 << a.group_shift) - 1);
  const long long task = (static_cast<long long>(blockIdx.x) * kThreads + threadIdx.x) >> a.group_shift;
  w.live = task < a.tasks && w.lane * kPerThread < a.cache.dim;
  w.inside = false;
  if (!w.live) return w;
  if (a.tasks <= 0x7fffffffll) {  // 32-bit divisions where they serve: a 64-bit one is some 100 instructions
    const unsigned t = static_cast<unsigned>(task), q = t / static_cast<unsigned>(a.cache.heads);
    w.n = q;
    w.head = static_cast<int>(t - q * static_cast<unsigned>(a.cache.heads));
  } else {
    w.n = task / a.cache.heads;
    w.head = static_cast<int>(task - w.n * a.cache.heads);
  }
  const long long slot = load_slot(a, w.n);
  w.inside = slot >= 0 && slot < a.cache.pages * a.cache.page_size;
  if (slot <= 0x7fffffffll) {
    const unsigned s = static_cast<unsigned>(slot), q = s / static_cast<unsigned>(a.cache.page_size);
    w.page = q;
    w.place = static_cast<int>(s - q * static_cast<unsigned>(a.cache.page_size));
  } else {
    w.page = slot / a.cache.page_size;
    w.place = static_cast<int>(slot - w.page * a.cache.page_size);
  }
  return w;
}

template <typename T>
__device__ __forceinline__ unsigned char* act_at(const RowsArgs& a, const Place& w, int side) {
  return a.act[side] + w.n * a.act_row[side] + w.head * a.act_head[side] + w.lane * kPerThread * sizeof(T);
}

__device__ __forceinline__ unsigned char* row_at(const Pages& p, const Place& w) {
  return p.base + w.page * p.page + w.place * p.place + w.head * p.head;
}

__device__ __forceinline__ float* scale_at(const Pages& p, const Place& w) {
  return p.scale + w.page * p.scale_page + w.place * p.scale_place + w.head * p.scale_head;
}

// 16 values of a row as they lie.
template <typename T, bool Vec>
__device__ __forceinline__ void load_raw(const unsigned char* p, uint32_t (&r)[4 * sizeof(T)]) {
  if constexpr (Vec) {
#pragma unroll
    for (unsigned h = 0; h < sizeof(T) / 2; ++h) load32(p + 32 * h, reinterpret_cast<uint32_t(&)[8]>(r[8 * h]));
  } else if constexpr (sizeof(T) == 2) {
    const unsigned short* t = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = t[2 * i] | static_cast<uint32_t>(t[2 * i + 1]) << 16;
  } else {
    const uint32_t* t = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = t[i];
  }
}

// Value i of them.
template <typename T>
__device__ __forceinline__ float raw_value(const uint32_t* r, int i) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(r[i]);
  else if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return __uint_as_float(i & 1 ? r[i >> 1] & 0xffff0000u : r[i >> 1] << 16);
  else return __half2float(__ushort_as_half(static_cast<unsigned short>(r[i >> 1] >> (16 * (i & 1)))));
}

// The largest magnitude of a row over its group of lanes, and whether the row is finite.  Magnitudes
// are compared as bits: of non-negative floats they order like integers, with infinity and then NaN
// on top, so that neither is lost as a maximum of floats would lose a NaN; 16-bit ones in pairs.
template <typename T>
__device__ __forceinline__ float largest(const uint32_t (&r)[4 * sizeof(T)], int group, bool* fine) {
  unsigned most = 0;
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) most = __vmaxu2(most, r[i] & 0x7fff7fffu);
    most = max(most >> 16, most & 0xffffu);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) most = max(most, r[i] & 0x7fffffffu);
  }
  for (int d = 1; d < group; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
  constexpr unsigned infinity =
      sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __nv_bfloat16>::value ? 0x7f80u : 0x7c00u;
  *fine = most < infinity;
  return raw_value<T>(&most, 0);
}

template <typename T, typename Code, bool Vec>
__global__ void __launch_bounds__(kThreads) k_write_quantised(const RowsArgs a) {
  const Place w = find(a);
  uint32_t raw[2][4 * sizeof(T)];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
#pragma unroll
    for (unsigned i = 0; i < 4 * sizeof(T); ++i) raw[side][i] = 0;
    if (w.live) load_raw<T, Vec>(act_at<T>(a, w, side), raw[side]);
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    bool fine;
    const float top = largest<T>(raw[side], 1 << a.group_shift, &fine);
    if (!w.inside) continue;
    const bool kept = fine && top >= kLeastRow;
    const float inverse = __fdiv_rn(Code::kMost, kept ? top : 1.0f);
    uint32_t code[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = __fmul_rn(raw_value<T>(raw[side], 4 * i + j), inverse);
      code[i] = kept ? Code::encode4(y) : 0u;
    }
    const Pages& to = side ? a.cache.v : a.cache.k;
    *reinterpret_cast<uint4*>(row_at(to, w) + w.lane * kPerThread) = make_uint4(code[0], code[1], code[2], code[3]);
    if (w.lane == 0)
      *scale_at(to, w) = kept ? top * (1.0f / Code::kMost) : fine ? 0.0f : __uint_as_float(0x7fc00000u);
  }
}

// 16-bit rows (16-byte aligned) kept as they are, rounded from T.
template <typename T, typename C, bool Vec>
__global__ void __launch_bounds__(kThreads) k_write_plain(const RowsArgs a) {
  const Place w = find(a);
  if (!w.inside) return;
  float x[2][kPerThread];
#pragma unroll
  for (int side = 0; side < 2; ++side) load16<T, Vec>(act_at<T>(a, w, side), x[side]);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      C h[2] = {rounded<C>(x[side][2 * i]), rounded<C>(x[side][2 * i + 1])};
      r[i] = *reinterpret_cast<const uint32_t*>(h);
    }
    uint4* row = reinterpret_cast<uint4*>(row_at(side ? a.cache.v : a.cache.k, w) + w.lane * kPerThread * sizeof(C));
    row[0] = make_uint4(r[0], r[1], r[2], r[3]);
    row[1] = make_uint4(r[4], r[5], r[6], r[7]);
  }
}

template <typename T, typename Code, bool Vec>
__global__ void __launch_bounds__(kThreads) k_read_quantised(const RowsArgs a) {
  const Place w = find(a);
  if (!w.live) return;
  uint4 code[2];
  float scale[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const Pages& from = side ? a.cache.v : a.cache.k;
    code[side] = make_uint4(0, 0, 0, 0);
    scale[side] = 0.0f;
    if (!w.inside) continue;
    code[side] = *reinterpret_cast<const uint4*>(row_at(from, w) + w.lane * kPerThread);
    scale[side] = *scale_at(from, w);
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const uint32_t r[4] = {code[side].x, code[side].y, code[side].z, code[side].w};
    float x[kPerThread];
#pragma unroll
    for (int i = 0; i < 4; ++i) Code::decode4(r[i], x + 4 * i);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) x[i] *= scale[side];
    store16<T, Vec>(act_at<T>(a, w, side), x);
  }
}

template <typename T, typename C, bool Vec>
__global__ void __launch_bounds__(kThreads) k_read_plain(const RowsArgs a) {
  const Place w = find(a);
  if (!w.live) return;
  uint4 half[2][2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    half[side][0] = half[side][1] = make_uint4(0, 0, 0, 0);
    if (!w.inside) continue;
    const uint4* row =
        reinterpret_cast<const uint4*>(row_at(side ? a.cache.v : a.cache.k, w) + w.lane * kPerThread * sizeof(C));
    half[side][0] = row[0];
    half[side][1] = row[1];
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const uint4 lo = half[side][0], hi = half[side][1];
    const uint32_t r[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    float x[kPerThread];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const C* h = reinterpret_cast<const C*>(&r[i]);
      x[2 * i] = static_cast<float>(h[0]);
      x[2 * i + 1] = static_cast<float>(h[1]);
    }
    store16<T, Vec>(act_at<T>(a, w, side), x);
  }
}

template <typename T, bool Vec>
void launch_rows(const RowsArgs& a, int kind, bool write, dim3 grid, cudaStream_t s) {
  if (write) {
    switch (kind) {
      case T4A_I8: k_write_quantised<T, Int8, Vec><<<grid, kThreads, 0, s>>>(a); break;
      case T4A_E4M3: k_write_quantised<T, E4m3, Vec><<<grid, kThreads, 0, s>>>(a); break;
      case T4A_F16: k_write_plain<T, __half, Vec><<<grid, kThreads, 0, s>>>(a); break;
      default: k_write_plain<T, __nv_bfloat16, Vec><<<grid, kThreads, 0, s>>>(a); break;
    }
  } else {
    switch (kind) {
      case T4A_I8: k_read_quantised<T, Int8, Vec><<<grid, kThreads, 0, s>>>(a); break;
      case T4A_E4M3: k_read_quantised<T, E4m3, Vec><<<grid, kThreads, 0, s>>>(a); break;
      case T4A_F16: k_read_plain<T, __half, Vec><<<grid, kThreads, 0, s>>>(a); break;
      default: k_read_plain<T, __nv_bfloat16, Vec><<<grid, kThreads, 0, s>>>(a); break;
    }
  }
}

int run_rows(void* stream, int dtype, int index_dtype, const t4a_kv_cache* cache, void* const act[2],
             const t4a_cuda_layout* const layout[2], const long long len[2], const void* slots,
             const t4a_cuda_layout* slots_layout, long long slots_len, bool write) {
  RowsArgs a;
  T4A_TRY(check_cache(cache, write, true, &a.cache));
  if (!is_row_dtype(dtype)) return T4A_ERR_UNSUPPORTED_DTYPE;
  if (index_dtype != T4A_CUDA_I32 && index_dtype != T4A_CUDA_I64) return T4A_ERR_UNSUPPORTED_DTYPE;
  T4A_TRY(check_tensor(slots_layout, 1, slots_len, index_dtype == T4A_CUDA_I64 ? 8 : 4));
  const int esize = element_size(dtype);
  const long long rows = slots_layout->extents[0];
  bool vec = true;
  for (int side = 0; side < 2; ++side) {
    T4A_TRY(check_rows(layout[side], 3, len[side], esize));
    if (!write) T4A_TRY(check_destination(*layout[side]));
    if (layout[side]->extents[0] != a.cache.dim || layout[side]->extents[1] != a.cache.heads ||
        layout[side]->extents[2] != rows)
      return T4A_ERR_SHAPE_MISMATCH;
    if (rows != 0 && a.cache.heads != 0 && act[side] == nullptr) return T4A_ERR_NULL_ARGUMENT;
    if (!aligned(act[side], esize)) return T4A_ERR_INVALID_STRIDE;
    a.act[side] = static_cast<unsigned char*>(act[side]) + layout[side]->offset * esize;
    a.act_head[side] = layout[side]->strides[1] * esize;
    a.act_row[side] = layout[side]->strides[2] * esize;
    vec = vec && rows_aligned(act[side], *layout[side], esize, 32);
  }
  if (plan::mul_overflows(rows, a.cache.heads, &a.tasks)) return T4A_ERR_OVERFLOW;
  if (a.tasks == 0) return T4A_OK;
  if (slots == nullptr) return T4A_ERR_NULL_ARGUMENT;
  a.slots = static_cast<const char*>(slots) + slots_layout->offset * (index_dtype == T4A_CUDA_I64 ? 8 : 4);
  a.slot_stride = slots_layout->strides[0];
  a.wide_index = index_dtype == T4A_CUDA_I64;
  if (a.cache.page_size == 0) a.cache.page_size = 1, a.cache.pages = 0;  // no slot is inside; no division by zero
  a.group_shift = 0;
  while ((kPerThread << a.group_shift) < a.cache.dim) ++a.group_shift;
  unsigned long long blocks;
  T4A_TRY(plan::grid_of(a.tasks, kThreads >> a.group_shift, &blocks));
  const dim3 grid(static_cast<unsigned>(blocks));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case T4A_CUDA_F32:
      vec ? launch_rows<float, true>(a, cache->kind, write, grid, s)
          : launch_rows<float, false>(a, cache->kind, write, grid, s);
      break;
    case T4A_F16:
      vec ? launch_rows<__half, true>(a, cache->kind, write, grid, s)
          : launch_rows<__half, false>(a, cache->kind, write, grid, s);
      break;
    default:
      vec ? launch_rows<__nv_bfloat16, true>(a, cache->kind, write, grid, s)
          : launch_rows<__nv_bfloat16, false>(a, cache->kind, write, grid, s);
      break;
  }
  return runtime::check_launch();
}

}  // namespace
}  // namespace cache
}  // namespace t4a

extern "C" int t4a_cache_write(void* stream, int dtype, int index_dtype, const t4a_kv_cache* cache, const void* key,
                               const t4a_cuda_layout* key_layout, long long key_len, const void* value,
                               const t4a_cuda_layout* value_layout, long long value_len, const void* slots,
                               const t4a_cuda_layout* slots_layout, long long slots_len) {
  void* const act[2] = {const_cast<void*>(key), const_cast<void*>(value)};
  const t4a_cuda_layout* const layout[2] = {key_layout, value_layout};
  const long long len[2] = {key_len, value_len};
  return t4a::cache::run_rows(stream, dtype, index_dtype, cache, act, layout, len, slots, slots_layout, slots_len,
                              true);
}

extern "C" int t4a_cache_read(void* stream, int dtype, int index_dtype, const t4a_kv_cache* cache, void* key,
                              const t4a_cuda_layout* key_layout, long long key_len, void* value,
                              const t4a_cuda_layout* value_layout, long long value_len, const void* slots,
                              const t4a_cuda_layout* slots_layout, long long slots_len) {
  void* const act[2] = {key, value};
  const t4a_cuda_layout* const layout[2] = {key_layout, value_layout};
  const long long len[2] = {key_len, value_len};
  return t4a::cache::run_rows(stream, dtype, index_dtype, cache, act, layout, len, slots, slots_layout, slots_len,
                              false);
}
