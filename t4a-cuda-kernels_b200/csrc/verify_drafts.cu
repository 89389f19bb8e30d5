// Verification of a tree of drafted tokens against the target's logits (t4a_verify_drafts).
//
// One cluster of 1, 2, 4 or 8 blocks walks one sequence's tree.  Only the rows of nodes that are
// taken are read: a tree of 32 nodes has some 4 on its path, so reading all rows at once would
// read 8 times as much.  At a node
//   r = e / Z,  e_x = exp(l_x - m),  m = max l,  Z = sum e
// Each block holds a slice of the row in shared memory as it came, each thread the same 16-byte
// vectors in every pass, so that no pass waits for another thread's values.  A warp's record
// (maximum, sum relative to it, argmax key) goes to all blocks of the cluster through distributed
// shared memory, and every warp joins all records in the same order: one cluster barrier a node.
//   Without a draft the children's tokens are left out of the row's own sum, and
//   mass = Z_rest + (children not yet turned down): sums of positive terms only, where Z - e_x
//   would cancel when a likely token is turned down.  So a node costs one exchange, whatever the
//   number of its children.
//   With a draft each child turned down costs one pass, r <- max(r - q, 0), and an exchange.  The
//   next child's r is a scalar recursion from the masses, which every block does for itself.  r
//   takes the logits' place in shared memory: beside them it takes 0.7 us off 4 chains of 5, and
//   half of the longest F32 row.
// Bound by latency: a node is a dependent load of its row, a pass over some 32 values a thread and
// a cluster barrier, some 4 us together; sequences run beside each other.  The race's row, wanted
// last, is prefetched into L2 at the start, the children's rows when their parent is read.  32
// trees of 32 nodes over a vocabulary of 128256 in BF16, 4 nodes a path: 28 us, 37 MB of rows that
// are needed (two exchanges a node, a sum and a maximum apart, took 52).  4 chains of 5 over 32003
// with a draft: 20 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "cache_plan.h"
#include "runtime.h"

namespace t4a {
namespace cache {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMostCluster = 8;
constexpr int kMostNodes = 1024;
constexpr int kMostBytes = 188416;  // of a block's slice: the logits, or with a draft r in F32

struct VerifyArgs {
  const void* logits;
  long long logits_node, logits_batch;  // strides in elements
  const float* draft;
  long long draft_node, draft_batch;
  const float* race;
  long long race_stride, race_batch;
  const int* tokens;
  const int* parents;
  const float* uniforms;
  int* count;
  int* path;
  int* said;
  float* logs;
  long long vocab;
  int nodes, slots;  // slots: vectors of a row that a block keeps
  float inverse_temperature;
};

struct Record {
  float m, s;
  unsigned long long key;
};

// Floats in their order as unsigned integers.
__device__ __forceinline__ unsigned ordered(float x) {
  const unsigned b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float from_ordered(unsigned o) {
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

// Lowest index first among equal values.
__device__ __forceinline__ unsigned long long make_key(unsigned value, long long index) {
  return (static_cast<unsigned long long>(value) << 32) | (0xffffffffu - static_cast<unsigned>(index));
}

__device__ __forceinline__ int key_index(unsigned long long key) {
  return static_cast<int>(0xffffffffu - static_cast<unsigned>(key));
}

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ unsigned cluster_blocks() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Shared {
  Record exchange[2][kMostCluster * kWarps];
  int children, child[kMostNodes], token[kMostNodes], parent[kMostNodes];
  float child_x[kMostNodes], child_q[kMostNodes], child_u[kMostNodes];  // scaled logit, draft, uniform
  float mass[kMostNodes];  // without a draft: of what the children from here on hold; else the passes' sums
  int elder[kMostNodes];   // the first child with the same token
  int mark[kMostNodes];    // of a child that is its own elder: the count of resets when it was turned down, plus 1
  int decided;             // thread 0's decision, for the block
  float total;
  int reset_at;
};

enum Mode { kGreedy, kPlain, kDraft };

template <typename T, Mode kMode>
class Walk {
 public:
  static constexpr int kVec = 16 / sizeof(T);
  static constexpr int kBatch = 4;  // vectors of a thread in flight
  static constexpr int kAhead = 4;  // children whose rows are prefetched

  __device__ Walk(const VerifyArgs& args, Shared& shared, unsigned char* kept)
      : a(args),
        sh(shared),
        held(reinterpret_cast<uint4*>(kept)),
        rank(cluster_rank()),
        blocks(cluster_blocks()),
        b(blockIdx.x / cluster_blocks()) {}

  __device__ void run() {
    const int tid = threadIdx.x;
    for (int i = tid; i < a.nodes; i += kThreads) {
      sh.token[i] = a.tokens[static_cast<long long>(b) * a.nodes + i];
      sh.parent[i] = a.parents[static_cast<long long>(b) * a.nodes + i];
    }
    first = static_cast<int>(rank) * a.slots;
    if (kMode != kGreedy && a.race_stride == 1) {
      const float* const race = a.race + static_cast<long long>(b) * a.race_batch;
      for (int i = first * kVec + tid * 32; i < min(static_cast<int>(a.vocab), (first + a.slots) * kVec); i += kThreads * 32)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(race + i));
    }
    if (blocks > 1) cluster_barrier();  // every block runs before its shared memory is written from another
    int at = 0, taken = 0;
    while (true) {
      const Record all = read_node(at);
      int next = -1;
      float total = all.s;
      if (kMode == kGreedy) {
        for (int c = 0; c < sh.children && next < 0; ++c)
          if (sh.token[sh.child[c]] == key_index(all.key)) next = c;
      } else if (sh.children != 0) {
        next = kMode == kPlain ? choose_plain(all, &total) : choose_against_draft(at, all);
      }
      if (next < 0) {
        finish(taken, all, total);
        return;
      }
      if (rank == 0 && tid == 0) {
        const long long o = static_cast<long long>(b) * a.nodes + taken;
        a.path[o] = sh.child[next];
        a.said[o] = sh.token[sh.child[next]];
        if (a.logs) a.logs[o] = log_of(sh.child_x[next], all.m, total);
      }
      at = sh.child[next];
      ++taken;
      __syncthreads();  // the child list is rewritten
    }
  }

 private:
  const VerifyArgs& a;
  Shared& sh;
  // [slots]: this block's vectors of the row.  With a draft [kVec / 4][slots]: r in F32 takes their
  // place, its elements 4 h to 4 h + 3 of vector j at h * slots + j, lanes side by side.
  uint4* const held;
  const unsigned rank, blocks;
  const int b;
  int turn = 0;  // exchanges so far
  const T* row = nullptr;
  int skew = 0;               // the row's first element within its 16-byte vector
  int first = 0, vectors = 0;  // this block's vectors of the row
  float factor = 1.0f;        // left * factor is r
  int passes = 0;             // of r <- max(r - q, 0) at this node

  // NaN counts as -infinity (fmaxf takes the other operand).
  __device__ float fix(float v) const { return fmaxf(kMode == kGreedy ? v : v * a.inverse_temperature, -INFINITY); }

  // exp(v - m), with the whole mass on infinite entries where there are some.
  static __device__ __forceinline__ float weight(float v, float m) {
    return v == m ? (m == -INFINITY ? 0.0f : 1.0f) : exp2_of(v - m);
  }
  static __device__ __forceinline__ float exp2_of(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
    return r;
  }

  static __device__ __forceinline__ float log_of(float v, float m, float total) {
    return v == -INFINITY ? -INFINITY : (v == m ? 0.0f : v - m) - logf(total);
  }

  __device__ bool in_vocab(int token) const { return token >= 0 && token < a.vocab; }

  __device__ __forceinline__ uint4 load_vector(int j) const {
    const int i = (first + j) * kVec - skew;
    if (i >= 0 && i + kVec <= a.vocab) return __ldcs(reinterpret_cast<const uint4*>(row + i));
    uint4 v;  // the row's ragged ends
    T* const r = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int e = 0; e < kVec; ++e) r[e] = i + e >= 0 && i + e < a.vocab ? row[i + e] : static_cast<T>(-INFINITY);
    return v;
  }

  // The node's children, and its row into `held`; the cluster's record of it.
  __device__ Record read_node(int at) {
    const int tid = threadIdx.x, lane = tid & 31;
    row = static_cast<const T*>(a.logits) + static_cast<long long>(b) * a.logits_batch +
          static_cast<long long>(at) * a.logits_node;
    skew = static_cast<int>((reinterpret_cast<uintptr_t>(row) / sizeof(T)) % kVec);
    const int all = static_cast<int>((a.vocab + skew + kVec - 1) / kVec);
    vectors = max(0, min(a.slots, all - first));
    passes = 0;
    uint4 raw[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (tid + u * kThreads < vectors) raw[u] = load_vector(tid + u * kThreads);
    if (at == 0) __syncthreads();  // tokens and parents
    if (tid < 32) {
      int n = 0;
      for (int i0 = at + 1; i0 < a.nodes; i0 += 32) {
        const int i = i0 + lane;
        const bool mine = i < a.nodes && sh.parent[i] == at;
        const unsigned votes = __ballot_sync(0xffffffffu, mine);
        if (mine) sh.child[n + __popc(votes & ((1u << lane) - 1))] = i;
        n += __popc(votes);
      }
      if (lane == 0) sh.children = n;
    }
    __syncthreads();
    const int children = sh.children;
    // The rows that may come next, a 128-byte line a thread, into L2: one of them is wanted a few
    // microseconds from now, when its way from memory would be the longest part of the wait.
    const int line = tid * 128;
    for (int c = 0; c < min(children, kAhead); ++c) {
      const T* const ahead = static_cast<const T*>(a.logits) + static_cast<long long>(b) * a.logits_batch +
                             static_cast<long long>(sh.child[c]) * a.logits_node;
      for (int at_byte = line; at_byte < vectors * 16; at_byte += kThreads * 128) {
        const long long i = static_cast<long long>(first) * kVec + at_byte / static_cast<int>(sizeof(T));
        if (i < a.vocab) asm volatile("prefetch.global.L2 [%0];" ::"l"(ahead + i));
      }
    }
    for (int c = tid; c < children; c += kThreads) {
      const int token = sh.token[sh.child[c]];
      sh.child_x[c] = in_vocab(token) ? fix(static_cast<float>(row[token])) : -INFINITY;
      if (kMode != kGreedy) sh.child_u[c] = a.uniforms[static_cast<long long>(b) * a.nodes + sh.child[c]];
      if (kMode == kDraft)
        sh.child_q[c] = in_vocab(token) ? a.draft[static_cast<long long>(b) * a.draft_batch +
                                                  static_cast<long long>(at) * a.draft_node + token]
                                        : 0.0f;
      if (kMode == kPlain) {
        int elder = c;
        for (int k = 0; k < c && elder == c; ++k)
          if (sh.token[sh.child[k]] == token) elder = k;
        sh.elder[c] = elder;
        sh.mark[c] = 0;
      }
    }
    Record mine;
    mine.m = -INFINITY;
    mine.key = 0;
    for (int j0 = tid; j0 < vectors; j0 += kBatch * kThreads) {
      if (j0 != tid) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (j0 + u * kThreads < vectors) raw[u] = load_vector(j0 + u * kThreads);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int j = j0 + u * kThreads;
        if (j >= vectors) continue;
        held[j] = raw[u];
        const T* const r = reinterpret_cast<const T*>(&raw[u]);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float v = fix(static_cast<float>(r[e]));
          if (kMode == kGreedy) {
            // Indices rise along a thread's walk, so the first of equals is its lowest.
            const int i = (first + j) * kVec - skew + e;
            // (-0 equals 0, so it has 0's key.)
            if (i >= 0 && i < a.vocab && (v > mine.m || mine.key == 0)) mine.key = make_key(ordered(v + 0.0f), i);
          }
          mine.m = fmaxf(mine.m, v);
        }
      }
    }
    if (kMode == kPlain) {  // the children's tokens out of the sum, by the threads that hold them
      for (int c = 0; c < children; ++c) {
        const int token = sh.token[sh.child[c]];
        if (!in_vocab(token)) continue;
        const int v = (token + skew) / kVec - first;
        if (v >= 0 && v < vectors && v % kThreads == tid)
          reinterpret_cast<T*>(&held[v])[(token + skew) % kVec] = static_cast<T>(-INFINITY);
      }
    }
    mine.s = 0.0f;
    for (int j = tid; j < vectors; j += kThreads) {
      const uint4 v = held[j];
      const T* const r = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int e = 0; e < kVec; ++e) mine.s += weight(fix(static_cast<float>(r[e])), mine.m);
    }
    return exchange(mine);
  }

  static __device__ __forceinline__ Record joined(const Record& x, const Record& y) {
    Record r;
    r.m = fmaxf(x.m, y.m);
    r.s = x.s * weight(x.m, r.m) + y.s * weight(y.m, r.m);
    r.key = max(x.key, y.key);
    return r;
  }

  // The warp's records as one, the same in all lanes: the sums are added in one order, and the value
  // is lane 0's.
  static __device__ __forceinline__ Record across(Record r) {
    const float m = from_ordered(__reduce_max_sync(0xffffffffu, ordered(r.m)));
    r.s *= weight(r.m, m);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) r.s += __shfl_xor_sync(0xffffffffu, r.s, d);
    r.s = __shfl_sync(0xffffffffu, r.s, 0);
    r.m = m;
    const unsigned high = __reduce_max_sync(0xffffffffu, static_cast<unsigned>(r.key >> 32));
    const unsigned low = __reduce_max_sync(
        0xffffffffu, static_cast<unsigned>(r.key >> 32) == high ? static_cast<unsigned>(r.key) : 0u);
    r.key = static_cast<unsigned long long>(high) << 32 | low;
    return r;
  }

  // All threads' records joined, in one order for every warp of the cluster.  Two buffers in turn: a
  // warp writes into one again only after a barrier that all warps reached after their reads of it.
  __device__ Record exchange(Record mine) {
    const int buffer = turn++ & 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    mine = across(mine);
    const int place = static_cast<int>(rank) * kWarps + warp;
    if (blocks == 1) {
      if (lane == 0) sh.exchange[buffer][place] = mine;
      __syncthreads();
    } else {
      if (lane < static_cast<int>(blocks)) {
        const unsigned local = static_cast<unsigned>(__cvta_generic_to_shared(&sh.exchange[buffer][place]));
        unsigned remote;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(lane));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1,%2};" ::"r"(remote), "f"(mine.m), "f"(mine.s) : "memory");
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote + 8), "l"(mine.key) : "memory");
      }
      __syncwarp();
      cluster_barrier();
    }
    Record all;
    all.m = -INFINITY;
    all.s = 0.0f;
    all.key = 0;
    for (int i = lane; i < static_cast<int>(blocks) * kWarps; i += 32) all = joined(all, sh.exchange[buffer][i]);
    return across(all);
  }

  // The first child taken, -1 without one; *total is the row's whole sum.
  __device__ int choose_plain(const Record& all, float* total) {
    const int n = sh.children;
    if (threadIdx.x == 0) {
      float behind = 0.0f;  // what the children from i on hold, a token once
      for (int i = n - 1; i >= 0; --i) {
        sh.mass[i] = behind;
        if (sh.elder[i] == i) behind += weight(sh.child_x[i], all.m);
      }
      const float whole = all.s + behind;
      float mass = whole;
      int from = 0, resets = 0, found = -1;
      for (int i = 0; i < n && whole > 0.0f; ++i) {
        const int e = sh.elder[i];
        const float r = sh.mark[e] == resets + 1 ? 0.0f : weight(sh.child_x[i], all.m);
        if (sh.child_u[i] * mass < r) {
          found = i;
          break;
        }
        sh.mark[e] = resets + 1;
        if (resets == 0) {
          mass = all.s + sh.mass[i];
        } else {
          mass = all.s;
          for (int k = 0; k < n; ++k)
            if (sh.elder[k] == k && sh.mark[k] != resets + 1) mass += weight(sh.child_x[k], all.m);
        }
        if (!(mass > 0.0f)) {  // nothing is left: the node's own softmax again
          mass = whole;
          from = i + 1;
          ++resets;
        }
      }
      sh.decided = found;
      sh.total = whole;
      sh.reset_at = from;
    }
    __syncthreads();
    *total = sh.total;
    return sh.decided;
  }

  __device__ int choose_against_draft(int at, const Record& all) {
    const float* q = a.draft + static_cast<long long>(b) * a.draft_batch + static_cast<long long>(at) * a.draft_node;
    int masses = 0;  // passes since the node's softmax
    for (int c = 0; c < sh.children; ++c) {
      const int token = sh.token[sh.child[c]];
      const float qx = sh.child_q[c];
      float r = weight(sh.child_x[c], all.m) / all.s;
      for (int i = 0; i < masses; ++i) r = fmaxf(r - qx, 0.0f) / sh.mass[i];
      if (in_vocab(token) && sh.child_u[c] * qx < r) return c;
      Record mine;
      mine.m = 0.0f;
      mine.s = subtract(q, all, passes > 0);
      mine.key = 0;
      const float mass = exchange(mine).s;
      if (mass > 0.0f) {
        factor = 1.0f / mass;
        ++passes;
        if (threadIdx.x == 0) sh.mass[masses] = mass;
        ++masses;
        __syncthreads();
      } else {  // nothing is left: the node's softmax again, from its logits
        masses = passes = 0;
        for (int j = threadIdx.x; j < vectors; j += kThreads) held[j] = load_vector(j);
      }
    }
    return -1;
  }

  // 16 bytes of F32 at once where they lie so.
  static __device__ __forceinline__ void load_f32(const float* p, bool whole, int i, long long n, float (&v)[kVec],
                                                  long long stride = 1) {
    if (whole && stride == 1 && (reinterpret_cast<uintptr_t>(p + i) & 15) == 0) {
#pragma unroll
      for (int h = 0; h < kVec; h += 4) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(p + i + h));
        v[h] = f.x;
        v[h + 1] = f.y;
        v[h + 2] = f.z;
        v[h + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = i + e >= 0 && i + e < n ? p[(i + e) * stride] : 0.0f;
    }
  }

  // r of this thread's vector j; `again`: after a pass, else from the logits.
  __device__ __forceinline__ void residual(int j, const Record& all, bool again, float (&r)[kVec]) const {
    if (again) {
      const float4* const left = reinterpret_cast<const float4*>(held) + j;
#pragma unroll
      for (int h = 0; h < kVec / 4; ++h) {
        const float4 x = left[h * a.slots];
        r[4 * h] = x.x * factor;
        r[4 * h + 1] = x.y * factor;
        r[4 * h + 2] = x.z * factor;
        r[4 * h + 3] = x.w * factor;
      }
    } else {
      const uint4 v = held[j];
      const T* const h = reinterpret_cast<const T*>(&v);
      const float over = kMode == kDraft ? 1.0f / all.s : 1.0f;  // the race goes by ratios
#pragma unroll
      for (int e = 0; e < kVec; ++e) r[e] = weight(fix(static_cast<float>(h[e])), all.m) * over;
    }
  }

  // r <- max(r - q, 0); the thread's sum of it.
  __device__ float subtract(const float* q, const Record& all, bool again) {
    float s = 0.0f;
    for (int j = threadIdx.x; j < vectors; j += kThreads) {
      const int i = (first + j) * kVec - skew;
      float v[kVec], r[kVec];
      load_f32(q, i >= 0 && i + kVec <= a.vocab, i, a.vocab, v);
      residual(j, all, again, r);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        r[e] = fmaxf(r[e] - v[e], 0.0f);
        s += r[e];
      }
      float4* const left = reinterpret_cast<float4*>(held) + j;
#pragma unroll
      for (int h = 0; h < kVec / 4; ++h)
        left[h * a.slots] = make_float4(r[4 * h], r[4 * h + 1], r[4 * h + 2], r[4 * h + 3]);
    }
    return s;
  }

  // The last token, its log-probability, and the places that nothing was written to.
  __device__ void finish(int taken, const Record& all, float total) {
    const int tid = threadIdx.x;
    int last;
    if (kMode == kGreedy) {
      last = key_index(all.key);
    } else {
      const float* race = a.race + static_cast<long long>(b) * a.race_batch;
      Record mine;
      mine.m = mine.s = 0.0f;
      mine.key = rank == 0 && tid == 0 ? make_key(0, 0) : 0;
#pragma unroll 2
      for (int j = tid; j < vectors; j += kThreads) {
        const int i = (first + j) * kVec - skew;
        float v[kVec], r[kVec];
        load_f32(race, i >= 0 && i + kVec <= a.vocab, i, a.vocab, v, a.race_stride);
        residual(j, all, passes > 0, r);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const float score = r[e] * v[e];
          if (score > 0.0f) mine.key = max(mine.key, make_key(__float_as_uint(score), i + e));
        }
      }
      if (kMode == kPlain && sh.children != 0 && rank == 0 && tid == 0) {
        // Children turned down before the node's softmax was taken again are back in it.
        for (int c = 0; c < sh.reset_at; ++c) {
          const int token = sh.token[sh.child[c]];
          bool back = in_vocab(token);
          for (int k = sh.reset_at; k < sh.children && back; ++k) back = sh.token[sh.child[k]] != token;
          if (!back) continue;
          const float score = weight(sh.child_x[c], all.m) * race[token * a.race_stride];
          if (score > 0.0f) mine.key = max(mine.key, make_key(__float_as_uint(score), token));
        }
      }
      last = key_index(exchange(mine).key);
    }
    if (rank != 0) return;
    const long long o = static_cast<long long>(b) * a.nodes;
    for (int i = tid; i < a.nodes; i += kThreads) {
      if (i >= taken) a.path[o + i] = -1;
      if (i > taken) a.said[o + i] = -1;
      if (i > taken && a.logs) a.logs[o + i] = 0.0f;
    }
    if (tid == 0) {
      a.count[b] = taken;
      a.said[o + taken] = last;
      if (a.logs) a.logs[o + taken] = log_of(fix(static_cast<float>(row[last])), all.m, total);
    }
  }
};

template <typename T, Mode kMode>
__global__ void __launch_bounds__(kThreads) k_verify(const VerifyArgs a) {
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ Shared sh;
  Walk<T, kMode> walk(a, sh, raw);
  walk.run();
}

template <typename T, Mode kMode>
int launch_verify(const VerifyArgs& a, int batch, int blocks, size_t bytes, cudaStream_t stream) {
  static std::atomic<unsigned long long> allowed{0};
  T4A_TRY(runtime::allow_shared(k_verify<T, kMode>, kMostBytes, &allowed));
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(batch) * blocks);
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  config.attrs = attr;
  config.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&config, k_verify<T, kMode>, a);
  if (err != cudaSuccess) {
    runtime::last_error() = static_cast<int>(err);
    cudaGetLastError();
    return T4A_ERR_CUDA;
  }
  return T4A_OK;
}

template <typename T>
int launch_mode(const VerifyArgs& a, bool greedy, int batch, int blocks, cudaStream_t stream) {
  const size_t logits = static_cast<size_t>(a.slots) * 16, r = static_cast<size_t>(a.slots) * (16 / sizeof(T)) * 4;
  if (greedy) return launch_verify<T, kGreedy>(a, batch, blocks, logits, stream);
  if (a.draft == nullptr) return launch_verify<T, kPlain>(a, batch, blocks, logits, stream);
  return launch_verify<T, kDraft>(a, batch, blocks, r, stream);
}

}  // namespace
}  // namespace cache
}  // namespace t4a

extern "C" int t4a_verify_drafts(void* stream, int dtype, const void* logits, const t4a_cuda_layout* logits_layout,
                                 long long logits_len, const int* tokens, const int* parents, const float* uniforms,
                                 const float* draft, const t4a_cuda_layout* draft_layout, long long draft_len,
                                 const float* race, const t4a_cuda_layout* race_layout, long long race_len,
                                 float temperature, int* count, int* path, int* said, float* logs) {
  using namespace t4a;
  using namespace t4a::cache;
  if (!is_row_dtype(dtype)) return T4A_ERR_UNSUPPORTED_DTYPE;
  const int esize = element_size(dtype);
  T4A_TRY(check_rows(logits_layout, 3, logits_len, esize));
  const long long vocab = logits_layout->extents[0], nodes = logits_layout->extents[1],
                  batch = logits_layout->extents[2];
  if (batch == 0) return T4A_OK;
  if (vocab == 0 || nodes == 0) return T4A_ERR_SHAPE_MISMATCH;  // every sequence says a token
  if (!(temperature >= 0.0f) || temperature > 3.0e38f || (temperature > 0.0f && temperature < 1e-30f))
    return T4A_ERR_UNSUPPORTED_OP;
  VerifyArgs a = {};
  const bool greedy = temperature == 0.0f;
  if (nodes > kMostNodes) return T4A_ERR_DOMAIN_TOO_LARGE;
  if (logits == nullptr || tokens == nullptr || parents == nullptr || count == nullptr || path == nullptr ||
      said == nullptr)
    return T4A_ERR_NULL_ARGUMENT;
  if (!aligned(logits, esize)) return T4A_ERR_INVALID_STRIDE;
  if (!greedy) {
    if (uniforms == nullptr || race == nullptr) return T4A_ERR_NULL_ARGUMENT;
    T4A_TRY(check_tensor(race_layout, 2, race_len, 4));
    if (race_layout->extents[0] != vocab || race_layout->extents[1] != batch) return T4A_ERR_SHAPE_MISMATCH;
    a.race = race + race_layout->offset;
    a.race_stride = race_layout->strides[0];
    a.race_batch = race_layout->strides[1];
    if (draft != nullptr) {
      T4A_TRY(check_rows(draft_layout, 3, draft_len, 4));
      for (int d = 0; d < 3; ++d)
        if (draft_layout->extents[d] != logits_layout->extents[d]) return T4A_ERR_SHAPE_MISMATCH;
      a.draft = draft + draft_layout->offset;
      a.draft_node = draft_layout->strides[1];
      a.draft_batch = draft_layout->strides[2];
    }
  }
  a.logits = static_cast<const char*>(logits) + logits_layout->offset * esize;
  a.logits_node = logits_layout->strides[1];
  a.logits_batch = logits_layout->strides[2];
  a.tokens = tokens;
  a.parents = parents;
  a.uniforms = uniforms;
  a.count = count;
  a.path = path;
  a.said = said;
  a.logs = logs;
  a.vocab = vocab;
  a.nodes = static_cast<int>(nodes);
  a.inverse_temperature = greedy ? 1.0f : static_cast<float>(1.0 / static_cast<double>(temperature));
  // Blocks of a cluster: a slice of at least 4096 values each, so that a block's load outweighs
  // its barriers, and as many as it takes for a slice to fit a block's shared memory.
  const int vec = 16 / esize;
  int blocks = 1;
  while (blocks < kMostCluster && vocab >= blocks * 2 * 4096ll) blocks *= 2;
  const long long vectors = (vocab + 2 * vec - 2) / vec;  // at the worst skew
  const long long slots = (vectors + blocks - 1) / blocks;
  const long long bytes = slots * (a.draft != nullptr ? vec * 4 : 16);
  if (bytes > kMostBytes) return T4A_ERR_DOMAIN_TOO_LARGE;
  if (batch * blocks > 0x7fffffffll) return T4A_ERR_LAUNCH_LIMIT;
  a.slots = static_cast<int>(slots);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case T4A_CUDA_F32: return launch_mode<float>(a, greedy, static_cast<int>(batch), blocks, s);
    case T4A_F16: return launch_mode<__half>(a, greedy, static_cast<int>(batch), blocks, s);
    default: return launch_mode<__nv_bfloat16>(a, greedy, static_cast<int>(batch), blocks, s);
  }
}
