// Attention over the paged cache on the tensor cores' own memory (tcgen05): the kernel for many
// query rows a cache head, where products bound the call.
//
// A block takes 128 query rows (a unit's tile of rows), one to a lane of tensor memory, and goes
// through the unit's tiles of 64 tokens:
//   S = Q K^T   [128 x 64], both from shared memory, into one of two buffers of tensor memory
//   P = 2^(S - m), by 128 threads, a row each, back into the buffer that S came from
//   O += P V    [128 x dim], P from tensor memory, V from shared memory as it lies (d fastest)
// so a row's maximum and sum need no exchange between threads, and P never leaves the SM's tensor
// memory.  Roles: four warps of softmax and results, four warps for 16-bit cache rows (eight for
// codes), and a warp that issues the products from one elected thread.  S of the tile after the next
// is issued behind P V of this one, and two blocks share an SM (256 columns of tensor memory and some
// 105 KB of shared memory each), so products run while exponentials are taken: an SM needs 512 cycles
// for a tile's products and 512 for its 8192 exponentials.
// A tile takes a block some 2700 cycles (16-bit) and its softmax bounds it, not a unit's rate: the
// barrier, the load, the maximum, the exponentials and the store follow one another, and a look at a
// barrier takes 450 cycles even when it is through.  Hence the look ahead at the next scores.  With
// the issuing thread by itself (`lane == 0`), each product and wait was serialised over the warp and
// bound the tile: 170 us for the 155 of a call below; and halves of 32 tokens at a time took 159.
// Packed F32 operations, and K and V by the same warps (228 for 168 then), were slower.
// 4 sequences of up to 16384 tokens, 512 rows a cache head, BF16, 99 GFLOP: 148 us, 670 TFLOP/s,
// 0.41 of a library product's rate; tensor pipe 0.33, DRAM reads 203 MB,
// each cache row once.
// 7 trees of 13 nodes over 4099 tokens, E4M3, 39 rows: 38 us, of which a block's five tiles are half;
// there unpacking bounds a tile (some 4500 cycles).
//
// Shared rows of Q, K and V are 128-byte lines of 64 values, their 16-byte units XORed with the
// line's number mod 8 (the 128-byte swizzle of the operand descriptors).  16-bit rows come there by
// cp.async; codes come through registers, where they become F16, exactly.  Scales, weights and rows
// with a scale of 0 are as in the kernel for few rows.
//
// Every wait is bounded (seconds): if one runs out all roles leave their loops, the results not yet
// written are NaN, and tensor memory is freed.
#pragma once

#include "attention_mma.cuh"

namespace t4a {
namespace cache {

// Rounds of a wait (a round is some 100 cycles) between looks at the other roles' failure, and looks
// before it gives up.  The inner loop is as short as it can be: a warp that polls takes issue slots
// from the warps it waits for.
constexpr unsigned kTcWaitRounds = 1u << 14, kTcWaitLooks = 1u << 10;

constexpr int kTcRows = 128;
constexpr int kTcSoftmax = 128;  // threads; the issuing warp has a warpgroup of its own
constexpr int kTcStages = 2;
constexpr int kTcSlots = 4;  // of tiles' scales and flags: they outlive a stage by two tiles
constexpr unsigned kTcColumns = 256;
constexpr float kLargeScore = 4194304.0f;  // 2^22: products below it are rounded by less than 2^-2

// What a tile's rows carry beside their values.
template <typename Flags>
struct alignas(16) TcSlot {
  float ks[kTile];  // K's scale, times the magnitude of the score's
  float lv[kTile];  // log2 of V's scale, -infinity for a scale of 0
  float rv[kTile];  // 1 / V's scale
  // A bit a token, in the words or half words that K's (of odd: V's) warps write.
  alignas(8) Flags there[8 / sizeof(Flags)];
  alignas(8) Flags zero[8 / sizeof(Flags)];
  alignas(8) Flags odd[8 / sizeof(Flags)];
};

static_assert(sizeof(TcSlot<unsigned>) % 16 == 0 && sizeof(TcSlot<unsigned short>) == sizeof(TcSlot<unsigned>),
              "slots are read 16 bytes at a time");

template <typename Flags>
__device__ __forceinline__ const unsigned* flags_of(const Flags* f) {
  return reinterpret_cast<const unsigned*>(f);
}

// Scales that change nothing, for scores that have had theirs.
struct alignas(16) TcNeutral {
  float ones[kTile], zeros[kTile];
  float keep[kTcRows];        // the weight of a row's passes before this one
  long long row_at[kTcRows];  // and where the unit's rows of q lie, -1 for none
};

struct TcBarriers {
  unsigned long long q_full, k_full[kTcStages], k_empty[kTcStages], v_full[kTcStages], v_empty[kTcStages],
      s_full[kTcSlots], p_full[2], o_done[2];
};

// Threads of the roles and their registers: equal at launch, then moved between the roles.  Codes
// take twice the warps, so that unpacking keeps up with the products.
template <bool Quantised>
struct TcRoles {
  static constexpr int loaders = Quantised ? 256 : 128;  // half of them K's rows, half V's
  static constexpr int threads = kTcSoftmax + loaders + 128;
  static constexpr int at_launch = Quantised ? 64 : 80;
  static constexpr int softmax = Quantised ? 112 : 128, loader = Quantised ? 56 : 64, issue = Quantised ? 32 : 48;
  static_assert(kTcSoftmax * softmax + loaders * loader + 128 * issue == threads * at_launch,
                "a larger sum would wait for good");
  static constexpr int side_warps = loaders / 64;         // of K, and of V
  static constexpr int warp_tokens = kTile / side_warps;  // of a tile
};

template <int Dim>
struct TcShape {
  static constexpr int blocks = Dim / 64;  // of 64 values, a line each
  static constexpr int q_bytes = kTcRows * (Dim < 128 ? 128 : Dim) * 2;  // parts take 256 bytes a row
  static constexpr int tile_bytes = kTile * Dim * 2;
  static constexpr int slots_at = q_bytes + 2 * kTcStages * tile_bytes;
  static constexpr int neutral_at = slots_at + kTcSlots * static_cast<int>(sizeof(TcSlot<unsigned>));
  static constexpr int barriers_at = neutral_at + static_cast<int>(sizeof(TcNeutral));
  static constexpr int shared = barriers_at + static_cast<int>(sizeof(TcBarriers)) + 16 + 1024;  // and alignment
  static constexpr int per_sm = 2;
};

__device__ __forceinline__ void barrier_init(unsigned long long* b, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_at(b)), "r"(count) : "memory");
}

__device__ __forceinline__ void barrier_arrive(unsigned long long* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_at(b)) : "memory");
}

// False when the phase did not complete within the limit, or another role's wait ran out.  A patient
// wait sleeps between polls: for roles that run ahead of the products.
template <bool Patient = false>
__device__ __forceinline__ bool barrier_wait(unsigned long long* b, unsigned parity, volatile int* failed) {
  const unsigned at = shared_at(b);
  for (unsigned i = 0; i < kTcWaitLooks; ++i) {
    unsigned ok;
    if constexpr (Patient) {
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, %3;\n"
          "WAIT:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra DONE;\n\tnanosleep.u32 100;\n\t"
          "sub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra WAIT;\n"
          "DONE:\n\tselp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(ok)
          : "r"(at), "r"(parity), "n"(kTcWaitRounds)
          : "memory");
    } else
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, %3;\n"
        "WAIT:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra DONE;\n\t"
        "sub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra WAIT;\n"
        "DONE:\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(at), "r"(parity), "n"(kTcWaitRounds)
        : "memory");
    if (ok) return true;
    if (*failed) return false;
  }
  *failed = 1;
  return false;
}

__device__ __forceinline__ bool barrier_test(unsigned long long* b, unsigned parity) {
  unsigned ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(shared_at(b)), "r"(parity)
      : "memory");
  return ok != 0;
}

// One lane of a whole warp, always the same: the compiler then knows that a single thread issues what
// follows, where after a test of the lane it serialises each product over the warp.
__device__ __forceinline__ bool elected() {
  unsigned one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ void tc_commit(unsigned long long* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_at(b))
               : "memory");
}

__device__ __forceinline__ void store16(unsigned at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// 32 columns of the warp's 32 lanes.
__device__ __forceinline__ void tc_load(uint32_t (&r)[32], unsigned at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}

__device__ __forceinline__ void tc_store(unsigned at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tc_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// An operand of 128-byte lines under the 128-byte swizzle; `lines` (in bytes) leads from 8 lines to
// the next 8, `across` from 64 values to the next 64 where they are the lines' own direction.
__device__ __forceinline__ unsigned long long operand(unsigned at, unsigned across, unsigned lines) {
  return static_cast<unsigned long long>((at & 0x3ffff) >> 4) | static_cast<unsigned long long>(across >> 4) << 16 |
         static_cast<unsigned long long>(lines >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

__device__ __forceinline__ void tc_mma(unsigned to, unsigned long long a, unsigned long long b, unsigned form,
                                       bool add) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(to),
      "l"(a), "l"(b), "r"(form), "r"(static_cast<unsigned>(add))
      : "memory");
}

__device__ __forceinline__ void tc_mma_from(unsigned to, unsigned a, unsigned long long b, unsigned form) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, 1, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(to),
      "r"(a), "l"(b), "r"(form)
      : "memory");
}

// F32 sums of 16-bit values, M = 128; `across`: B's lines run along N.
template <bool Bf16>
__device__ __forceinline__ unsigned tc_form(int n, bool across) {
  return 1u << 4 | (Bf16 ? 1u : 0u) << 7 | (Bf16 ? 1u : 0u) << 10 | (across ? 1u : 0u) << 16 |
         static_cast<unsigned>(n >> 3) << 17 | (kTcRows >> 4) << 24;
}

__device__ __forceinline__ void tc_load1(uint32_t* r, unsigned at) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(*r) : "r"(at));
}

__device__ __forceinline__ void tc_load16(uint32_t (&r)[16], unsigned at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}

__device__ __forceinline__ void tc_store16(unsigned at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float highest(const uint32_t (&s)[32]) {
  float x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = fmaxf(__uint_as_float(s[8 * k]), __uint_as_float(s[8 * k + 1]));
#pragma unroll
    for (int j = 2; j < 8; j += 2) x[k] = max3(x[k], __uint_as_float(s[8 * k + j]), __uint_as_float(s[8 * k + j + 1]));
  }
  return fmaxf(max3(x[0], x[1], x[2]), x[3]);
}

// Products of codes to base-2 scores.
__device__ __forceinline__ void scale_scores(uint32_t (&s)[32], const float* ks, const float* lv) {
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const float4 k = *reinterpret_cast<const float4*>(ks + j), v = *reinterpret_cast<const float4*>(lv + j);
    s[j] = __float_as_uint(fmaf(__uint_as_float(s[j]), k.x, v.x));
    s[j + 1] = __float_as_uint(fmaf(__uint_as_float(s[j + 1]), k.y, v.y));
    s[j + 2] = __float_as_uint(fmaf(__uint_as_float(s[j + 2]), k.z, v.z));
    s[j + 3] = __float_as_uint(fmaf(__uint_as_float(s[j + 3]), k.w, v.w));
  }
}

// Weights 2^(s * factor - less) as pairs of 16-bit values, and their sums (over V's scale).  (Packed
// F32 arithmetic was slower: its register pairs cost more moves than it saved.)
template <bool Quantised, bool Bf16>
__device__ __forceinline__ void weights(const uint32_t (&s)[32], uint32_t* p, float factor, float less, const float* rv,
                                        float (&l)[4]) {
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    float4 r;
    if constexpr (Quantised) r = *reinterpret_cast<const float4*>(rv + j);
    float w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = __uint_as_float(s[j + e]);
      w[e] = exp2_fast(Quantised ? x - less : fmaf(x, factor, -less));
    }
    if constexpr (Quantised) {
      l[0] = fmaf(w[0], r.x, l[0]);
      l[1] = fmaf(w[1], r.y, l[1]);
      l[2] = fmaf(w[2], r.z, l[2]);
      l[3] = fmaf(w[3], r.w, l[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) l[e] += w[e];
    }
    p[j >> 1] = pack2<Bf16>(w[0], w[1]);
    p[(j >> 1) + 1] = pack2<Bf16>(w[2], w[3]);
  }
}

// A pair of weights, times x, a power of two: rounded only where a weight leaves F16's normal range.
template <bool Bf16>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t pair, float x) {
  if constexpr (Bf16) {
    return pack2<true>(__uint_as_float(pair << 16) * x, __uint_as_float(pair & 0xffff0000u) * x);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pair));
    return pack2<false>(f.x * x, f.y * x);
  }
}

// Whether tile `tile` of a unit reaches past the context, so that some node may not see all of its
// tokens.  The loader of V and the softmax both go by this: the one takes infinities and NaNs out of
// such a tile's rows and writes the slot's `odd`, the other reads it.
__device__ __forceinline__ bool holds_drafts(int tile, int context) { return (tile + 1) * kTile > context; }

// `kPasses`: whether a block may have more than one pass over a unit, which costs the others 2%.
template <int Kind, int Dim, bool kPasses>
__global__ void __launch_bounds__(TcRoles<KindOf<Kind>::quantised>::threads, TcShape<Dim>::per_sm) k_attend_tc(const AttendArgs a) {
  using Shape = TcShape<Dim>;
  constexpr bool kQuantised = KindOf<Kind>::quantised, kBf16 = KindOf<Kind>::bf16;
  using Roles = TcRoles<kQuantised>;
  constexpr int kIssueWarp = (kTcSoftmax + Roles::loaders) / 32;
  extern __shared__ unsigned char raw[];
  unsigned char* const smem = raw + ((1024 - (shared_at(raw) & 1023)) & 1023);
  unsigned char* const q_lines = smem;
  unsigned char* const part_lines = smem;
  auto k_lines = [&](int stage) { return smem + Shape::q_bytes + stage * Shape::tile_bytes; };
  auto v_lines = [&](int stage) { return smem + Shape::q_bytes + (kTcStages + stage) * Shape::tile_bytes; };
  using Flags = std::conditional_t<kQuantised, unsigned short, unsigned>;
  TcSlot<Flags>* const slots = reinterpret_cast<TcSlot<Flags>*>(smem + Shape::slots_at);
  float* const ones = reinterpret_cast<TcNeutral*>(smem + Shape::neutral_at)->ones;
  float* const zeros = reinterpret_cast<TcNeutral*>(smem + Shape::neutral_at)->zeros;
  float* const keeps = reinterpret_cast<TcNeutral*>(smem + Shape::neutral_at)->keep;
  long long* const row_at = reinterpret_cast<TcNeutral*>(smem + Shape::neutral_at)->row_at;
  TcBarriers* const bar = reinterpret_cast<TcBarriers*>(smem + Shape::barriers_at);
  unsigned* const tmem_at = reinterpret_cast<unsigned*>(bar + 1);
  volatile int* const failed = reinterpret_cast<int*>(tmem_at + 1);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int dim = a.cache.dim;

  if (threadIdx.x < kTile) {
    ones[threadIdx.x] = 1.0f;
    zeros[threadIdx.x] = 0.0f;
  }
  if (threadIdx.x == 0) {
    barrier_init(&bar->q_full, kTcRows);
    for (int i = 0; i < kTcStages; ++i) {
      barrier_init(&bar->k_full[i], Roles::loaders / 2);
      barrier_init(&bar->v_full[i], Roles::loaders / 2);
      barrier_init(&bar->k_empty[i], 1);
      barrier_init(&bar->v_empty[i], 1);
    }
    // Two of each, in turn: a fast thread is at most one tile ahead of a slow one.
    for (int i = 0; i < 2; ++i) {
      barrier_init(&bar->p_full[i], kTcRows);
      barrier_init(&bar->o_done[i], 1);
    }
    // A tile's products and what K's warps say of its tokens: one wait for both.  A slot comes round
    // again only when its tile is through.
    for (int i = 0; i < kTcSlots; ++i) barrier_init(&bar->s_full[i], 1 + Roles::side_warps);
    *failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kIssueWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(shared_at(tmem_at)),
                 "n"(kTcColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  // The pads past dim meet zeros of Q, or make columns that are not stored; they have to be finite.
  if (dim < Dim)
    for (int i = threadIdx.x; i < Shape::slots_at / 16; i += Roles::threads)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Cursor at = find_start(a, blockIdx.x);
  tc_before();
  fence_async();
  __syncthreads();
  tc_after();
  const unsigned tmem = *tmem_at, tmem_o = tmem + 128;

  int tiles_done = 0;  // of the block, in all its units: phases and slots go by it

  if (warp >= 4 && warp < kIssueWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Roles::loader));
    // ---- cache rows: half of the warps K's, half V's, an equal part of a tile's tokens each ----
    constexpr int kTokens = Roles::warp_tokens;
    const bool is_v = warp - 4 >= Roles::side_warps;
    const int first_token = ((warp - 4) % Roles::side_warps) * kTokens;
    constexpr int kChunks = Dim * KindOf<Kind>::bytes / 16;  // of a padded row
    constexpr int kRounds = kTokens * kChunks / 32;
    constexpr unsigned kAllThere = static_cast<unsigned>((1ull << kTokens) - 1);
    const int used = dim * KindOf<Kind>::bytes / 16;
    const Pages& mine = is_v ? a.cache.v : a.cache.k;
    unsigned long long* const full = is_v ? bar->v_full : bar->k_full;
    unsigned long long* const empty = is_v ? bar->v_empty : bar->k_empty;
    auto lines = [&](int stage) { return is_v ? v_lines(stage) : k_lines(stage); };
    // The row and chunk of a lane in round u: round u's rows are kStep further on than round 0's.
    // Codes become two units each: 8 lanes then take 4 chunks of two rows, whose units the swizzle
    // keeps apart, rather than 8 of one.
    constexpr bool kPairs = kQuantised && kChunks == 8;
    constexpr int kStep = 32 / kChunks;
    const int lane_token = kPairs ? (lane >> 4) * 2 + ((lane >> 2) & 1) : lane / kChunks;
    const int chunk = kPairs ? ((lane >> 3) & 1) * 4 + (lane & 3) : lane % kChunks;
    // Swizzled place of a 16-byte unit of 8 values of row t.
    auto unit_at = [&](int t, int unit) {
      return (unit >> 3) * (kTile * 128) + t * 128 + (((unit & 7) ^ (t & 7)) << 4);
    };
    // first_token is a multiple of 8, so row u's swizzle is round 0's with (u * kStep) & 7 flipped into it
    // (lane_token < kStep, a power of 2).
    const int unit = kQuantised ? 2 * chunk : chunk;
    const unsigned lane_unit = unit_at(first_token + lane_token, unit);
    auto round_unit = [&](unsigned stage_at, int u) {
      return ((stage_at + lane_unit) ^ (((u * kStep) & 7) << 4)) + u * kStep * 128;
    };
    bool good = true;
    while (at.left > 0 && good) {
      const int b = at.b;
      int context, live, length;
      sequence_tokens(a, b, &context, &live, &length);
      const int n = kPasses ? pass_tiles(a, at) : min(at.left, at.tiles - at.tile);
      const unsigned char* const base = mine.base + at.head * mine.head;
      const int* const my_table = a.table + b * a.table_batch;
      int pos = at.tile * kTile + first_token + lane % kTokens;  // the lane's token of the next tile to look up
      int in_table = pos / a.cache.page_size, place = pos - in_table * a.cache.page_size;
      const int end = min(length, (at.tile + n) * kTile);
      int page_ahead, place_ahead;
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
      unsigned bits = 0;  // of the warp's tokens, which are there
      long long off = 0;  // of the lane's token
      float ks = 0.0f, vs = 0.0f;
      auto step = [&] {  // to the next tile
        const int page = page_ahead, at_place = place_ahead;
        look_up();
        const bool there = static_cast<unsigned>(page) < static_cast<unsigned>(a.cache.pages);
        bits = __ballot_sync(0xffffffffu, there) & kAllThere;
        off = there ? page * mine.page + at_place * mine.place : 0;
        if (kQuantised && !is_v) {
          ks = vs = 1.0f;
          if (there) {
            const Pages &k = a.cache.k, &v = a.cache.v;
            ks = k.scale[page * k.scale_page + at_place * k.scale_place + at.head * k.scale_head];
            vs = v.scale[page * v.scale_page + at_place * v.scale_place + at.head * v.scale_head];
          }
        }
      };
      uint4 code[kQuantised ? kRounds : 1];
      auto fetch = [&] {
        if constexpr (kQuantised) {
          if (a.plain_copies && bits == kAllThere) {
            const unsigned units = static_cast<unsigned>(off >> 4);
#pragma unroll
            for (int u = 0; u < kRounds; ++u) {
              const unsigned from = __shfl_sync(0xffffffffu, units, u * kStep + lane_token) + chunk;
              code[u] = *reinterpret_cast<const uint4*>(base + static_cast<unsigned long long>(from) * 16);
            }
            return;
          }
#pragma unroll
          for (int u = 0; u < kRounds; ++u) {
            const int t = u * kStep + lane_token;
            const long long from = __shfl_sync(0xffffffffu, off, t);
            code[u] = make_uint4(0, 0, 0, 0);
            if (((bits >> t) & 1) && chunk < used) code[u] = *reinterpret_cast<const uint4*>(base + from + chunk * 16);
          }
        }
      };
      // K's warps say what the tile's tokens are.
      auto describe = [&](int t) {
        TcSlot<Flags>& slot = slots[t % kTcSlots];
        if (lane == 0) slot.there[first_token / kTokens] = static_cast<Flags>(bits);
        if constexpr (kQuantised) {
          const bool zero = fabsf(vs) < kLeastScale;
          const unsigned zeros_of = __ballot_sync(0xffffffffu, zero) & kAllThere;
          if (lane == 0) slot.zero[first_token / kTokens] = static_cast<Flags>(zeros_of);
          const float lv = zero ? -INFINITY : __log2f(vs);
          if (lane < kTokens) {
            slot.ks[first_token + lane] = ks * fabsf(a.scale_log2);
            slot.lv[first_token + lane] = lv;
            // A NaN, also of a scale below zero, has made the score a NaN where the row is seen, and must
            // not touch l elsewhere.
            slot.rv[first_token + lane] = zero ? 0.0f : lv == lv ? exp2_fast(-lv) : 1.0f;
          }
        }
        __syncwarp();
        if (lane == 0) barrier_arrive(&bar->s_full[t % kTcSlots]);
      };
      look_up();
      step();
      if constexpr (kQuantised) fetch();
      for (int i = 0; i < n; ++i) {
        const int t = tiles_done + i, stage = t % kTcStages;
        const bool drafts = holds_drafts(at.tile + i, context);
        good = barrier_wait<true>(&empty[stage], ((t / kTcStages) & 1) ^ 1, failed);
        if (!good) break;
        unsigned char* const to = lines(stage);
        const unsigned to_shared = shared_at(to);
        if (!is_v) describe(t);
        unsigned odd = 0;  // tokens with an infinity or a NaN in V, where some node may not see them
        if constexpr (kQuantised) {
          // Codes to F16 lines.
#pragma unroll
          for (int u = 0; u < kRounds; ++u) {
            uint32_t x[4] = {code[u].x, code[u].y, code[u].z, code[u].w}, h[8];
            if (Kind == T4A_E4M3 && is_v && drafts) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t nan = __vcmpeq4(x[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                if (nan != 0) odd |= 1u << (u * kStep + lane_token);
                x[e] &= ~nan;
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) neighbours<Kind>(x[e], &h[2 * e], &h[2 * e + 1]);
            if (chunk < used) {
              const unsigned place_at = round_unit(to_shared, u);
              store16(place_at, h[0], h[1], h[2], h[3]);
              store16(place_at ^ 16, h[4], h[5], h[6], h[7]);
            }
          }
        } else {
          // 16-bit rows straight to their lines.
          if (a.plain_copies && bits == kAllThere) {
            const unsigned units = static_cast<unsigned>(off >> 4);
#pragma unroll
            for (int u = 0; u < kRounds; ++u) {
              const unsigned from = __shfl_sync(0xffffffffu, units, u * kStep + lane_token) + chunk;
              copy16(round_unit(to_shared, u), base + static_cast<unsigned long long>(from) * 16);
            }
          } else {
#pragma unroll 4
            for (int u = 0; u < kRounds; ++u) {
              const int in = u * kStep + lane_token;
              const long long from = __shfl_sync(0xffffffffu, off, in);
              if (chunk < used) copy16(round_unit(to_shared, u), base + from + chunk * 16, (bits >> in) & 1);
            }
          }
          if (is_v && drafts) {
            asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
            for (int u = 0; u < kRounds; ++u) {
              const int in = u * kStep + lane_token;
              if (chunk >= used) continue;
              uint32_t* const unit = reinterpret_cast<uint32_t*>(to + unit_at(first_token + in, chunk));
              for (int e = 0; e < 4; ++e) {
                uint32_t x = unit[e];
                constexpr uint32_t ones_of = kBf16 ? 0x7f80u : 0x7c00u;
                if ((x & ones_of) == ones_of) x &= 0xffff0000u, odd |= 1u << in;
                if ((x & (ones_of << 16)) == (ones_of << 16)) x &= 0xffffu, odd |= 1u << in;
                unit[e] = x;
              }
            }
          }
        }
        if (Kind != T4A_I8 && is_v && drafts) {
          odd = __reduce_or_sync(0xffffffffu, odd);
          if (lane == 0) slots[t % kTcSlots].odd[first_token / kTokens] = static_cast<Flags>(odd);
          __syncwarp();
        }
        if (kQuantised || (is_v && drafts)) {
          fence_async();
          barrier_arrive(&full[stage]);
        } else {
          // Arrives when this thread's copies have.
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(shared_at(&full[stage])) : "memory");
        }
        step();
        if (kQuantised && i + 1 < n) fetch();
      }
      tiles_done += n;
      next_pass(a, &at, n);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp >= kIssueWarp) {
    // ---- products ----
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Roles::issue));
    if (warp == kIssueWarp) {
      const unsigned form_s = tc_form<kBf16>(kTile, false), form_o = tc_form<kBf16>(Dim, true);
      const unsigned q_at = shared_at(q_lines);
      // All lanes wait together (a lane by itself takes longer), one issues.
      auto ready = [&](unsigned long long* b, unsigned parity) {
        const bool all = __all_sync(0xffffffffu, barrier_wait(b, parity, failed));
        __syncwarp();
        fence_async();  // the rows were written by ordinary stores and copies
        tc_after();
        return all;
      };
      auto scores = [&](int t) {
        const int stage = t % kTcStages;
        const unsigned k_at = shared_at(k_lines(stage));
#pragma unroll
        for (int k = 0; k < Dim / 16; ++k)
          tc_mma(tmem + (t & 1) * 64, operand(q_at + (k >> 2) * kTcRows * 128 + (k & 3) * 32, 16, 1024),
                 operand(k_at + (k >> 2) * kTile * 128 + (k & 3) * 32, 16, 1024), form_s, k > 0);
        tc_commit(&bar->k_empty[stage]);
        tc_commit(&bar->s_full[t % kTcSlots]);
      };
      auto outputs = [&](int t) {
        const int stage = t % kTcStages;
        const unsigned v_at = shared_at(v_lines(stage));
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
          tc_mma_from(tmem_o, tmem + (t & 1) * 64 + k * 8, operand(v_at + k * 2048, kTile * 128, 1024), form_o);
        tc_commit(&bar->v_empty[stage]);
        tc_commit(&bar->o_done[t & 1]);
      };
      auto k_barrier = [&](int t) { return &bar->k_full[t % kTcStages]; };
      auto stage_parity = [&](int t) { return static_cast<unsigned>((t / kTcStages) & 1); };
      bool good = true;
      unsigned unit = 0;
      while (at.left > 0 && good) {
        const int n = kPasses ? pass_tiles(a, at) : min(at.left, at.tiles - at.tile), t0 = tiles_done;
        good = ready(&bar->q_full, unit & 1) && ready(k_barrier(t0), stage_parity(t0));
        if (good && elected()) scores(t0);
        if (good && n > 1) {
          good = ready(k_barrier(t0 + 1), stage_parity(t0 + 1));
          if (good && elected()) scores(t0 + 1);
        }
        // P V of a tile, and the scores of the one after the next into the buffer that P leaves.
        for (int i = 0; i < n && good; ++i) {
          const int t = t0 + i;
          good = ready(&bar->v_full[t % kTcStages], stage_parity(t)) && ready(&bar->p_full[t & 1], (t >> 1) & 1);
          if (good && elected()) outputs(t);
          if (good && i + 2 < n) {
            good = ready(k_barrier(t + 2), stage_parity(t + 2));
            if (good && elected()) scores(t + 2);
          }
        }
        tiles_done += n;
        ++unit;
        next_pass(a, &at, n);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax: thread r has query row r of the tile ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Roles::softmax));
    const unsigned lanes = static_cast<unsigned>(warp * 32) << 16;
    const int r = threadIdx.x;
    bool good = true;
    while (at.left > 0) {
      const int b = at.b;
      int context, live, length;
      sequence_tokens(a, b, &context, &live, &length);
      const int n = kPasses ? pass_tiles(a, at) : min(at.left, at.tiles - at.tile);
      const int row = at.row_tile * kTcRows + r, node = row / a.group;
      const bool here = row < a.rows && node < live, any_here = __any_sync(0xffffffffu, here);
      // A negative scale is Q's sign, so that the largest product is the largest score.
      const unsigned flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
      // Codes: K's scales have the score's; what is left is the row's power of two.
      float factor = kQuantised ? 1.0f : fabsf(a.scale_log2);
      bool shifted = false;  // whether some row of the warp has one
      {
        // The rows into their lines: units of 8 values, so that a warp reads whole rows; then zeros
        // into the thread's lanes of O.
        constexpr int kUnits = Dim / 8;
        auto line_of = [&](int q_row, int unit) {
          return reinterpret_cast<uint4*>(q_lines + (unit >> 3) * (kTcRows * 128) + q_row * 128 +
                                          (((unit & 7) ^ (q_row & 7)) << 4));
        };
        row_at[r] = here ? b * a.q_batch + node * a.q_node +
                               (static_cast<long long>(at.head) * a.group + (row - node * a.group)) * a.q_head
                         : -1;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const int unit = r % kUnits;
#pragma unroll 1
        for (int u0 = 0; u0 < kUnits; u0 += 8) {
          uint4 x[8];
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            const long long from_at = row_at[(u0 + u) * (kTcRows / kUnits) + r / kUnits];
            x[u] = make_uint4(0, 0, 0, 0);
            if (from_at >= 0 && 8 * unit < dim) {
              const unsigned short* const from = static_cast<const unsigned short*>(a.q) + from_at + 8 * unit;
              if (a.q_units) {
                x[u] = *reinterpret_cast<const uint4*>(from);
              } else {
                uint32_t h[4];
                for (int e = 0; e < 4; ++e) h[e] = from[2 * e] | static_cast<uint32_t>(from[2 * e + 1]) << 16;
                x[u] = make_uint4(h[0], h[1], h[2], h[3]);
              }
            }
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            x[u].x ^= flip, x[u].y ^= flip, x[u].z ^= flip, x[u].w ^= flip;
            *line_of((u0 + u) * (kTcRows / kUnits) + r / kUnits, unit) = x[u];
          }
        }
        if (kQuantised && a.q_bf16) {
          // Each thread its own row, in place: BF16 to F16, exact for 2^-14 to 2^16 and off by 2^-25 below,
          // so a row whose largest magnitude is outside [1/4, 2^15) is first brought to [2^14, 2^15).
          asm volatile("bar.sync 1, 128;" ::: "memory");
          unsigned most = 0;
#pragma unroll 4
          for (int u = 0; u < kUnits; ++u) {
            const uint4 x = *line_of(r, u);
            most = __vmaxu2(most, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                                           __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
          }
          most = max(most >> 16, most & 0xffffu);
          float down = 1.0f;
          if (most != 0 && most < 0x7f80u && (most < 0x3e80u || most >= 0x4700u)) {
            const int e = max(static_cast<int>(most >> 7), 16);  // biased exponent
            down = __uint_as_float(static_cast<unsigned>(min(127 + 14 + 127 - e, 253)) << 23);
            factor = 1.0f / down;
          }
          shifted = __any_sync(0xffffffffu, down != 1.0f);
          auto f16_pair = [&](uint32_t h) {
            return pack2<false>(__uint_as_float(h << 16) * down, __uint_as_float(h & 0xffff0000u) * down);
          };
#pragma unroll 4
          for (int u = 0; u < kUnits; ++u) {
            const uint4 x = *line_of(r, u);
            *line_of(r, u) = make_uint4(f16_pair(x.x), f16_pair(x.y), f16_pair(x.z), f16_pair(x.w));
          }
        }
        uint32_t zero[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) zero[e] = 0;
#pragma unroll
        for (int d = 0; d < Dim; d += 32) tc_store(tmem_o + lanes + d, zero);
        tc_stored();
        tc_before();
        fence_async();
        barrier_arrive(&bar->q_full);
      }
      float m = -INFINITY, less = 0.0f, mz = -INFINITY, lz = 0.0f;  // less: m - kLift once m is finite
      float l4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      bool ahead = false;  // the next tile's scores are known to be there
      for (int i = 0; i < n && good; ++i) {
        const int t = tiles_done + i;
        // Warps without a live row only keep step.
        good = any_here ? __all_sync(0xffffffffu, ahead) ||
                              barrier_wait(&bar->s_full[t % kTcSlots], (t / kTcSlots) & 1, failed)
                        : barrier_wait<true>(&bar->s_full[t % kTcSlots], (t / kTcSlots) & 1, failed);
        if (!good) break;
        tc_after();
        if (any_here) {
          const TcSlot<Flags>& slot = slots[t % kTcSlots];
          const int pos0 = (at.tile + i) * kTile;
          const unsigned s_at = tmem + (t & 1) * 64 + lanes;
          const unsigned there_lo = flags_of(slot.there)[0], there_hi = flags_of(slot.there)[1];
          const bool drafts = holds_drafts(at.tile + i, context);
          const bool partly = (there_lo & there_hi) != 0xffffffffu || drafts;
          const unsigned zero_lo = kQuantised ? flags_of(slot.zero)[0] : 0u,
                         zero_hi = kQuantised ? flags_of(slot.zero)[1] : 0u;
          const bool rare = partly || (zero_lo | zero_hi) != 0 || (kQuantised && shifted);
          float now_factor = kQuantised ? 1.0f : factor;
          const float *ks = slot.ks, *lv = slot.lv;
          unsigned see_lo = there_lo, see_hi = there_hi, odd_lo = 0, odd_hi = 0;
          if (rare) {
            // Scores with what is not seen at -infinity, back to tensor memory for the common path;
            // V rows with a scale of 0 into their own sum.
            if (partly) {
              for (int j = max(0, context - pos0); j < kTile && pos0 + j < length; ++j) {
                const int drafted = pos0 + j - context;
                if (!(here && drafted < live && node_sees(a, b, node, drafted))) {
                  if (j < 32) see_lo &= ~(1u << j);
                  else see_hi &= ~(1u << (j - 32));
                }
              }
            }
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
              uint32_t s[32];
              tc_load(s, s_at + 32 * half);
              tc_loaded();
              const unsigned see = half ? see_hi : see_lo, zero = half ? zero_hi : zero_lo;
              float high = -INFINITY;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                // The factors first: a product of codes times the row's alone may pass F32's range.
                float x = __uint_as_float(s[j]) * (kQuantised ? factor * slot.ks[32 * half + j] : factor);
                if constexpr (kQuantised) {
                  if ((zero & see) >> j & 1) high = fmaxf(high, x);
                  else x += slot.lv[32 * half + j];
                }
                s[j] = __float_as_uint((see >> j) & 1 ? x : -INFINITY);
              }
              if (kQuantised && zero != 0) {
                const float to = fmaxf(mz, high), base = to == -INFINITY ? 0.0f : to;
                lz *= exp2_fast(mz - base);
                mz = to;
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if ((zero >> j) & 1) {
                    lz += exp2_fast(__uint_as_float(s[j]) - base);
                    s[j] = __float_as_uint(-INFINITY);
                  }
              }
              tc_store(s_at + 32 * half, s);
            }
            tc_stored();
            now_factor = 1.0f;
            ks = ones;
            lv = zeros;
          }
          if (Kind != T4A_I8 && drafts) {
            // Whether something was cleaned out of V, for the rows that see it: never of tokens that are
            // not there, whose place in the table leads nowhere.
            good = barrier_wait(&bar->v_full[t % kTcStages], (t / kTcStages) & 1, failed);
            const volatile unsigned* const odd = flags_of(slot.odd);
            odd_lo = good ? odd[0] & there_lo : 0;
            odd_hi = good ? odd[1] & there_hi : 0;
          }
          // Codes by halves of 32 tokens, since their loaders leave a thread few registers; P overwrites
          // scores that have been read.
          constexpr int kSides = kQuantised ? 1 : 2;  // of 32 tokens at a time
#pragma unroll 1
          for (int half = 0; half < 2; half += kSides) {
            uint32_t s[kSides][32];
#pragma unroll
            for (int q = 0; q < kSides; ++q) tc_load(s[q], s_at + 32 * (half + q));
            tc_loaded();
            if constexpr (kQuantised) scale_scores(s[0], ks + 32 * half, lv + 32 * half);
            float top = highest(s[0]);
            if constexpr (kSides == 2) top = fmaxf(top, highest(s[1]));
            if constexpr (!kQuantised) top *= now_factor;  // factors are not negative
            const bool rises = here && top > m + kSlack;
            if (__any_sync(0xffffffffu, rises)) {
              float shrink = 1.0f;
              if (rises) {
                // The reference is the maximum, whose weight is exact then; but where the tile's first
                // weights are 16 bits already it moves by whole numbers, so that they shrink exactly.
                const float steps = ceilf(top - m);
                if (kSides == 1 && half == 1 && steps <= 126.0f) {
                  shrink = __uint_as_float(static_cast<unsigned>(127 - static_cast<int>(steps)) << 23);
                  m += steps;
                } else {
                  shrink = exp2_fast(m - top);
                  m = top;
                }
                less = m - kLift;
                l4[0] *= shrink, l4[1] *= shrink, l4[2] *= shrink, l4[3] *= shrink;
              }
              if (kSides == 1 && half == 1) {
                // The first half's weights go by the old reference.
                uint32_t p[16];
                tc_load16(p, s_at);
                tc_loaded();
#pragma unroll
                for (int e = 0; e < 16; ++e) p[e] = scaled_pair<kBf16>(p[e], shrink);
                tc_store16(s_at, p);
              }
              if (i > 0) {
                good = good && barrier_wait(&bar->o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, failed);
                tc_after();
#pragma unroll 1
                for (int d = 0; d < Dim; d += 16) {
                  uint32_t o[16];
                  tc_load16(o, tmem_o + lanes + d);
                  tc_loaded();
#pragma unroll
                  for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * shrink);
                  tc_store16(tmem_o + lanes + d, o);
                }
                tc_stored();
              }
            }
            if (Kind != T4A_I8 && (kSides == 2 ? odd_lo | odd_hi : half ? odd_hi : odd_lo) != 0 && good) {
              if (i > 0) good = barrier_wait(&bar->o_done[(t - 1) & 1], ((t - 1) >> 1) & 1, failed);
              tc_after();
#pragma unroll 1
              for (int j = 32 * half; j < 32 * (half + kSides); ++j) {
                if (!(((j < 32 ? odd_lo : odd_hi) >> (j & 31)) & 1)) continue;
                uint32_t score;
                tc_load1(&score, s_at + j);
                tc_loaded();
                const bool sees = here && (((j < 32 ? see_lo : see_hi) >> (j & 31)) & 1);
                const float w = exp2_fast(__uint_as_float(score) - less);
                const int at_pos = pos0 + j;
                const int page = a.table[b * a.table_batch + (at_pos / a.cache.page_size) * a.table_page];
                const unsigned char* const v_row = a.cache.v.base + at.head * a.cache.v.head + page * a.cache.v.page +
                                                   (at_pos % a.cache.page_size) * a.cache.v.place;
#pragma unroll 1
                for (int d = 0; d < dim; d += 16) {
                  uint32_t o[16];
                  tc_load16(o, tmem_o + lanes + d);
                  tc_loaded();
#pragma unroll
                  for (int e = 0; e < 16; ++e) {
                    const float v = sees ? row_value<Kind>(v_row, d + e) : 0.0f;
                    if (!(fabsf(v) < INFINITY)) o[e] = __float_as_uint(__uint_as_float(o[e]) + w * v);
                  }
                  __syncwarp();
                  tc_store16(tmem_o + lanes + d, o);
                }
                tc_stored();
              }
            }
            // The weights' fused product keeps what the maximum's rounded one lost: up to half a unit of its
            // last place, which for large scores is a weight beyond F16.  Those are rounded first.
            if (!kQuantised && fabsf(less) >= kLargeScore) {
#pragma unroll
              for (int q = 0; q < kSides; ++q)
#pragma unroll
                for (int j = 0; j < 32; ++j) s[q][j] = __float_as_uint(__uint_as_float(s[q][j]) * now_factor);
              now_factor = 1.0f;
            }
            // A look at the next tile's scores, which are there by now as a rule: its answer takes a while.
            // (Over codes they come later than that.)
            if (!kQuantised)
              ahead = i + 1 < n && barrier_test(&bar->s_full[(t + 1) % kTcSlots], ((t + 1) / kTcSlots) & 1);
#pragma unroll
            for (int q = 0; q < kSides; ++q) {
              uint32_t p[16];
              weights<kQuantised, kBf16>(s[q], p, now_factor, less, slot.rv + 32 * (half + q), l4);
              tc_store16(s_at + 16 * (half + q), p);
            }
            tc_stored();
          }
          tc_before();
        }
        barrier_arrive(&bar->p_full[t & 1]);
      }
      const float l = (l4[0] + l4[1]) + (l4[2] + l4[3]);
      tiles_done += n;
      if (good) good = barrier_wait(&bar->o_done[(tiles_done - 1) & 1], ((tiles_done - 1) >> 1) & 1, failed);
      tc_after();
      // Whether the block has the unit's first tile, and all; whether passes came before this one.
      const bool begun = at.from == 0, whole = begun && at.tile + n == at.tiles, again = kPasses && at.tile != at.from;
      // Sums relative to the larger reference; O stays relative to its own.
      const float mo = m == -INFINITY ? 0.0f : less;
      const float ml = kQuantised ? fmaxf(m == -INFINITY ? -INFINITY : less, mz) : (m == -INFINITY ? -INFINITY : less);
      const float less_l = ml == -INFINITY ? 0.0f : ml;
      float ll = l != 0.0f ? l * exp2_fast(mo - less_l) : 0.0f;
      if (kQuantised && lz != 0.0f) ll += lz * exp2_fast(mz - less_l);
      const bool dead = !here || ll == 0.0f;
      float over = dead ? 0.0f : (mo == less_l ? 1.0f : exp2_fast(mo - less_l)) / ll;
      float lse2 = dead ? -INFINITY : less_l + log2f(ll);
      if (!good) over = lse2 = __uint_as_float(0x7fc00000u);
      const long long part = (static_cast<long long>(blockIdx.x) * 2 + (begun ? 1 : 0)) * kTcRows;
      if (again && row < a.rows) {
        float keep, add;
        join_passes(a.part_lse[part + r], &lse2, &keep, &add);
        over *= add;
        keeps[r] = keep;
      }
      if (row < a.rows) {
        if (whole) store_lse(a, b, at.head, row, lse2);
        else a.part_lse[part + r] = lse2;
      }
      // Results through Q's lines, which no product reads any more, so that a warp writes whole rows:
      // 16-bit results all at once; parts, and what joins passes before it, in F32 by halves of a row's
      // line block.
      row_at[r] = row < a.rows ? (whole ? out_row(a, b, at.head, row) : (part + r) * dim) : -1;
      if (whole && !again) {
#pragma unroll 1
        for (int d = 0; d < Dim; d += 16) {
          uint32_t o[16], h[8];
          tc_load16(o, tmem_o + lanes + d);
          tc_loaded();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = dead && good ? 0.0f : __uint_as_float(o[2 * e]) * over;
            const float y = dead && good ? 0.0f : __uint_as_float(o[2 * e + 1]) * over;
            h[e] = a.q_bf16 ? pack2<true>(x, y) : pack2<false>(x, y);
          }
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int unit = d / 8 + e;
            *reinterpret_cast<uint4*>(q_lines + r * (Dim * 2) + ((unit ^ (r & 7)) << 4)) =
                make_uint4(h[4 * e], h[4 * e + 1], h[4 * e + 2], h[4 * e + 3]);
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
        constexpr int kUnits = Dim / 8;
        const int unit = r % kUnits;
        if (8 * unit < dim) {
#pragma unroll 4
          for (int u = 0; u < kUnits; ++u) {
            const int of = u * (kTcRows / kUnits) + r / kUnits;
            const long long to = row_at[of];
            if (to < 0) continue;
            const uint4 x = *reinterpret_cast<const uint4*>(q_lines + of * (Dim * 2) + ((unit ^ (of & 7)) << 4));
            unsigned short* const out = static_cast<unsigned short*>(a.out) + to + 8 * unit;
            if (a.out_units) {
              *reinterpret_cast<uint4*>(out) = x;
            } else {
              const uint32_t h[4] = {x.x, x.y, x.z, x.w};
              for (int e = 0; e < 8; ++e) out[e] = static_cast<unsigned short>(h[e >> 1] >> (16 * (e & 1)));
            }
          }
        }
        asm volatile("bar.sync 1, 128;" ::: "memory");
      } else {
#pragma unroll 1
        for (int half = 0; half < Dim; half += 64) {
#pragma unroll 1
          for (int d = 0; d < 64; d += 16) {
            uint32_t o[16];
            tc_load16(o, tmem_o + lanes + half + d);
            tc_loaded();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x[4];
#pragma unroll
              for (int f = 0; f < 4; ++f) x[f] = dead && good ? 0.0f : __uint_as_float(o[4 * e + f]) * over;
              *reinterpret_cast<float4*>(part_lines + r * 256 + (((d / 4 + e) ^ (r & 7)) << 4)) =
                  make_float4(x[0], x[1], x[2], x[3]);
            }
          }
          asm volatile("bar.sync 1, 128;" ::: "memory");
          const int unit = r % 16;  // of 4 values
          if (again && half + 4 * unit < dim) {
            // What the passes before have left, by the same thread, and this one's.
#pragma unroll 1
            for (int of = r / 16; of < kTcRows; of += 8) {
              const long long to = row_at[of];
              if (to < 0) continue;
              float4* const kept = reinterpret_cast<float4*>(a.part_out + (part + of) * dim + half + 4 * unit);
              const float4 before = *kept;
              float4 x = *reinterpret_cast<const float4*>(part_lines + of * 256 + ((unit ^ (of & 7)) << 4));
              const float keep = keeps[of];
              x = make_float4(fmaf(before.x, keep, x.x), fmaf(before.y, keep, x.y), fmaf(before.z, keep, x.z),
                              fmaf(before.w, keep, x.w));
              if (whole) {
                store_out(a, to + half + 4 * unit, x.x, x.y);
                store_out(a, to + half + 4 * unit + 2, x.z, x.w);
              } else {
                *kept = x;
              }
            }
          } else if (half + 4 * unit < dim) {
#pragma unroll 4
            for (int u = 0; u < 16; ++u) {
              const int of = u * 8 + r / 16;
              const long long to = row_at[of];
              if (to < 0) continue;
              *reinterpret_cast<float4*>(a.part_out + to + half + 4 * unit) =
                  *reinterpret_cast<const float4*>(part_lines + of * 256 + ((unit ^ (of & 7)) << 4));
            }
          }
          asm volatile("bar.sync 1, 128;" ::: "memory");
        }
      }
      tc_before();
      next_pass(a, &at, n);
    }
  }
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTcColumns) : "memory");
  }
}

}  // namespace cache
}  // namespace t4a
