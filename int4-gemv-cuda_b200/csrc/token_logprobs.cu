// Log probabilities of given tokens, the entropy of each row and its top alternatives, from logits:
//   lse = log sum_j e^{x_j},  logprob = x_t - lse,  entropy = lse - sum_j p_j x_j.
//
// One pass over a row, in base 2. With L = log2(e) in fp32 a thread keeps c = L m of the maximum m
// it has seen, S = sum 2^a and U = sum 2^a a with a = fma(x, L, -c), all fp32, rescaled when a tile
// of its elements raises m; then
//   logprob = ln 2 (fma(x_t, L, -c) - log2 S),  entropy = ln 2 (log2 S - U / S).
// Every element is taken by the same fma, so neither the rounding of c nor that of L (a softmax of
// x (1 + 1e-8)) shows: the first cancels, the second moves a log probability by 1e-8 of x_t's
// distance from the mean logit. -inf is taken as the type's lowest value (or -1e38), which adds 0 to
// both sums without a test. c holds to 2^16 L in size; a row whose maximum is beyond that (fp32 and
// bf16 masks of the lowest value alone, for instance), or with nothing above -inf, is summed again
// with its maximum known. A NaN or +inf makes its row NaN.
//
// Top alternatives in the same pass: the maxima of 64 groups of threads give a threshold (the n-th
// largest of them: at least n elements reach it), the first one behind a barrier in the first tile. A
// thread whose tile reaches the threshold puts the tile's maximum and place into a list in shared
// memory: one store and one atomic a warp, however many of the tile's elements do, since a warp that
// stops to sort them holds up its block. The warps take turns to renew the threshold at the tiles
// 1, 2, 4, ...; the others go on with the one they have (any of them is at most the last), so no
// barrier is needed, and the list gets about n entries between two renewals. Behind the row the
// entries that reach the last threshold (about n) are read again, a warp an entry, and their elements
// ranked by value, then by lowest index. Where the list overflows (rising logits) it is made again
// from the row with the last threshold; where that overflows too (thousands of equal logits), the n
// elements are taken one by one.
//
// Bound by HBM: each logit is read once. A thread copies its own 16-byte chunks two tiles ahead into
// its own slots of shared memory (cp.async), so the stream needs no barrier, and blocks stay for
// many rows, so the next row is on its way while one is finished. With few rows a row is split over
// a cluster of blocks that join their sums and lists through distributed shared memory.
// Measured on B200, 2048 x 128256 bf16: 90 us without alternatives, 5.8 TB/s (0.89 of a plain copy's
// 6.53; the pipe of the 2^x is three quarters busy), 107 us with one and 108 with three (119 on another
// card): what comes on top is a row's end, to which all blocks come at about the same time. One row of 32001: 3.9 us without
// alternatives, 7.5 us with five (latency). Taking the elements one by one is `top` passes over a row: 64
// rows of 128256 equal logits take 277 us with 20 alternatives, where normal ones take 13.6, and logits
// rounded to halves 18.8.
#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>

#include "decode.cuh"
#include "kernels.h"

namespace i4 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / kWarp;
constexpr int kPer = 4;    // 16-byte chunks a thread takes of a tile
constexpr int kTile = kPer * kThreads;
constexpr int kRing = 3;   // tiles of a thread's slots
constexpr int kCtas = 4;   // blocks an SM
constexpr int kGroups = 64;    // groups of threads whose maxima give the threshold
constexpr int kList = 512;     // places of the list: tiles of threads
constexpr int kPicks = 128;    // of them, those that reach the last threshold
constexpr int kKeys = 512;     // elements that are ranked
constexpr int kAtOnce = 2;     // picks a warp reads at once
constexpr int kMaxCluster = 8;
constexpr float kFar = 65536.0f;  // the largest maximum whose sums the one pass holds
constexpr float kLn2 = 0.69314718055994531f;

using Key = unsigned long long;  // order_key(value) << 32 | ~index: larger is better
__device__ __forceinline__ Key make_key(float v, int index) {
  return static_cast<Key>(order_key(v)) << 32 | static_cast<uint32_t>(~index);
}
__device__ __forceinline__ float key_value(Key k) {
  return from_order_key(static_cast<uint32_t>(k >> 32));
}
__device__ __forceinline__ int key_index(Key k) { return static_cast<int>(~static_cast<uint32_t>(k)); }
constexpr uint32_t kNegInfKey = 0x007FFFFFu;  // order_key(-inf)

struct Sums {
  float m, c, s, u;  // m only for the threshold and the test against kFar
  static __device__ __forceinline__ Sums none() { return {-INFINITY, -kFar * kLog2e, 0.0f, 0.0f}; }
  static __device__ __forceinline__ float reference(float m) {
    return fminf(fmaxf(m, -kFar), kFar) * kLog2e;
  }
  __device__ __forceinline__ void rescale(float to) {
    const float d = c - to, f = exp2_fast(d);  // d within 2^18: the sums stay finite where f is 0
    u = f * fmaf(s, d, u);
    s *= f;
    c = to;
  }
  __device__ __forceinline__ void join(Sums o) {
    const float top = fmaxf(c, o.c);
    rescale(top);
    o.rescale(top);
    s += o.s;
    u += o.u;
    m = fmaxf(m, o.m);
  }
  __device__ __forceinline__ void join_lanes() {
#pragma unroll
    for (int off = kWarp / 2; off > 0; off >>= 1) {
      Sums o;
      o.m = __shfl_xor_sync(0xffffffffu, m, off);
      o.c = __shfl_xor_sync(0xffffffffu, c, off);
      o.s = __shfl_xor_sync(0xffffffffu, s, off);
      o.u = __shfl_xor_sync(0xffffffffu, u, off);
      join(o);
    }
  }
};

// ---- A chunk in the type it is read in -----------------------------------------------------------

// The larger of two pairs of 16-bit numbers, NaN where either is one; of two fp32 numbers.
template <class T>
__device__ __forceinline__ uint32_t max_word(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t max_word<half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t max_word<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t max_word<float>(uint32_t a, uint32_t b) {
  return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
}

template <class T>
__device__ __forceinline__ uint32_t word_of(float v) {  // v in every element of a word
  if constexpr (sizeof(T) == 4) {
    return __float_as_uint(v);
  } else {
    return pack2<T>(v, v);
  }
}
template <class T>
__device__ __forceinline__ float max_of_word(uint32_t w) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(w);
  } else {
    const float2 f = unpack2<T>(w);
    return max_nan(f.x, f.y);
  }
}
template <class T>
__device__ __forceinline__ uint32_t max_words(const uint4& v) {
  return max_word<T>(max_word<T>(v.x, v.y), max_word<T>(v.z, v.w));
}

// What -inf is taken as: finite, and L times it is too.
template <class T>
constexpr float kLowest = -1e38f;
template <>
constexpr float kLowest<half> = -65504.0f;

// The chunks of memory that a row lies in, and this block's share of them.
template <class T>
struct Row {
  static constexpr int E = Chunk<T>::kElems;
  const T* row;
  int shift;   // elements of the first chunk that lie before the row
  int c0, c1;  // this block's chunks

  __device__ __forceinline__ Row(const LogprobArgs& a, int64_t index, int rank, int ranks) {
    row = static_cast<const T*>(a.logits) + index * a.row_stride;
    shift = static_cast<int>(reinterpret_cast<uintptr_t>(row) / sizeof(T) % E);
    const int64_t chunks = (static_cast<int64_t>(shift) + a.vocab + E - 1) / E;
    c0 = static_cast<int>(chunks * rank / ranks);
    c1 = static_cast<int>(chunks * (rank + 1) / ranks);
  }
  __device__ __forceinline__ const T* at(int c) const { return row + (c * E - shift); }
  __device__ __forceinline__ bool whole(int c, int vocab) const {
    return c * E >= shift && c * E - shift + E <= vocab;
  }
  // A chunk at the row's ends, or of another block: what lies outside is -inf.
  __device__ __forceinline__ uint4 partial(int c, int vocab) const {
    Chunk<T> f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = c * E - shift + i;
      f.v[i] = c < c1 && e >= 0 && e < vocab ? to_f32(row[e]) : -INFINITY;
    }
    return f.get();
  }
  __device__ __forceinline__ uint4 load(int c, int vocab) const {
    return whole(c, vocab) ? ld_stream_v4(at(c)) : partial(c, vocab);
  }
};

// What the blocks of a row send to its first block.
struct Part {
  Sums sums;
  int count;  // entries of top
  Key top[kMaxTop];
};

struct Shared {
  uint4 ring[kRing][kPer][kThreads];
  Sums warp[kWarps];
  Key best[kWarps];
  alignas(16) uint32_t group_max[kGroups];
  uint32_t threshold;  // by the block
  float least;         // renewed by its warps
  int listed, picked, keyed;
  Part parts[kMaxCluster];
  int picks[kPicks];  // first chunks from c0
  union {
    Key list[kList];  // order_key of a thread's maximum in a tile << 32 | its first chunk from c0
    Key keys[kKeys];  // behind the picking
  };
};

// The maxima of the thread's group so far.
__device__ __forceinline__ void publish(Shared& sh, float thread_max) {
  uint32_t k = order_key(thread_max);
#pragma unroll
  for (int off = kThreads / kGroups / 2; off > 0; off >>= 1) {
    k = max(k, __shfl_xor_sync(0xffffffffu, k, off));
  }
  if (threadIdx.x % (kThreads / kGroups) == 0) sh.group_max[threadIdx.x / (kThreads / kGroups)] = k;
}

// By the block, behind a barrier: the top-th largest of the groups' maxima. Four threads a group
// count what is larger; ends with a barrier.
__device__ __forceinline__ uint32_t block_threshold(Shared& sh, int top) {
  static_assert(kThreads == 4 * kGroups, "four threads a group");
  const int g = threadIdx.x / 4, q = threadIdx.x % 4;
  const uint32_t mine = sh.group_max[g];
  int rank = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = (i * 4 + q) * 4;  // the four threads read neighbours
    const uint4 o = *reinterpret_cast<const uint4*>(&sh.group_max[at]);
    rank += (o.x > mine || (o.x == mine && at < g)) + (o.y > mine || (o.y == mine && at + 1 < g)) +
            (o.z > mine || (o.z == mine && at + 2 < g)) + (o.w > mine || (o.w == mine && at + 3 < g));
  }
  rank += __shfl_xor_sync(0xffffffffu, rank, 1);
  rank += __shfl_xor_sync(0xffffffffu, rank, 2);
  if (q == 0 && rank == top - 1) sh.threshold = mine;
  __syncthreads();
  return sh.threshold;
}

// By a warp, while others go on: the same of a view of the maxima, two of them a lane. A few are
// taken off one by one; for more the 64 are sorted (a bitonic network).
constexpr int kTakeOff = 8;
__device__ __forceinline__ uint32_t warp_threshold(const Shared& sh, int top) {
  const int lane = threadIdx.x % kWarp;
  const volatile uint32_t* maxima = sh.group_max;
  uint32_t v0 = maxima[lane], v1 = maxima[lane + kWarp];
  if (top <= kTakeOff) {
    uint32_t best = 0;
    for (int i = 0; i < top; ++i) {
      const uint32_t mine = max(v0, v1);
      best = __reduce_max_sync(0xffffffffu, mine);
      if (lane == __ffs(__ballot_sync(0xffffffffu, mine == best)) - 1) {
        if (v0 == best) {
          v0 = 0;
        } else {
          v1 = 0;
        }
      }
    }
    return best;
  }
  // place of v0: lane, of v1: lane + 32; in the end falling
#pragma unroll
  for (int k = 2; k <= kGroups; k *= 2) {
#pragma unroll
    for (int j = k / 2; j > 0; j /= 2) {
      if (j == kWarp) {
        const uint32_t hi = max(v0, v1);
        v1 = min(v0, v1);
        v0 = hi;
      } else {
        const uint32_t o0 = __shfl_xor_sync(0xffffffffu, v0, j);
        const uint32_t o1 = __shfl_xor_sync(0xffffffffu, v1, j);
        const bool first = (lane & j) == 0;
        v0 = first == ((lane & k) == 0) ? max(v0, o0) : min(v0, o0);
        v1 = first == (((lane + kWarp) & k) == 0) ? max(v1, o1) : min(v1, o1);
      }
    }
  }
  const int at = top - 1;
  return __shfl_sync(0xffffffffu, at < kWarp ? v0 : v1, at % kWarp);
}

// Adds the lanes' values whose `take` holds to a list of at most `most`, one atomic a warp. The
// count goes on beyond `most`, as the sign of an overflow.
template <class V>
__device__ __forceinline__ void append(V* list, int* count, int most, bool take, V value) {
  const uint32_t who = __ballot_sync(0xffffffffu, take);
  if (who == 0) return;
  const int lane = threadIdx.x % kWarp;
  int at = 0;
  if (lane == 0) at = atomicAdd(count, __popc(who));
  at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
  if (take && at < most) list[at] = value;
}

// Puts a thread's tile into the list if its maximum reaches `least` (or is a NaN) and is not -inf:
// a rare branch, so a lane by itself.
__device__ __forceinline__ void note(Shared& sh, float top, float least, int chunk) {
  if (!(top < least) && top != -INFINITY) {
    const int at = atomicAdd(&sh.listed, 1);
    if (at < kList) sh.list[at] = static_cast<Key>(order_key(top)) << 32 | static_cast<uint32_t>(chunk);
  }
}

// ---- The rare ways, out of the stream's code -----------------------------------------------------

template <class T>
__device__ __noinline__ void remake_list(Shared& sh, const Row<T> r, int vocab, uint32_t least_key) {
  __syncthreads();  // all have read the count
  if (threadIdx.x == 0) sh.listed = 0;
  __syncthreads();
  for (int base = 0; base < r.c1 - r.c0; base += kTile) {
    const int first = base + threadIdx.x;
    float top = -INFINITY;
    for (int j = 0; j < kPer; ++j) {
      const int c = r.c0 + first + j * kThreads;
      if (c < r.c1) top = max_nan(top, max_of_word<T>(max_words<T>(r.load(c, vocab))));
    }
    note(sh, top, from_order_key(least_key), first);
  }
  __syncthreads();
}

// The largest elements of the block's share, each by a pass over it.
template <class T>
__device__ __noinline__ void take_one_by_one(Shared& sh, const Row<T> r, int vocab, int top,
                                             Part* part) {
  constexpr int E = Chunk<T>::kElems;
  const int tid = threadIdx.x;
  Key last = ~static_cast<Key>(0);
  int got = 0;
  while (got < top) {
    Key best = 0;
    for (int c = r.c0 + tid; c < r.c1; c += kThreads) {
      Chunk<T> v;
      v.set(r.load(c, vocab));
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int index = c * E - r.shift + i;
        const Key k = make_key(v.v[i], index);
        if (index >= 0 && index < vocab && k < last && k > best) best = k;
      }
    }
#pragma unroll
    for (int off = kWarp / 2; off > 0; off >>= 1) {
      const Key o = __shfl_xor_sync(0xffffffffu, best, off);
      best = o > best ? o : best;
    }
    __syncthreads();
    if (tid % kWarp == 0) sh.best[tid / kWarp] = best;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) best = sh.best[w] > best ? sh.best[w] : best;
    if (static_cast<uint32_t>(best >> 32) <= kNegInfKey) break;
    if (tid == 0) part->top[got] = best;
    last = best;
    ++got;
  }
  if (tid == 0) part->count = got;
}

// Sum of e^(x - m) and of e^(x - m) (x - m) over a whole row.
template <class T>
__device__ __noinline__ float2 sum_again(Shared& sh, const T* row, int vocab, float m) {
  float s = 0.0f, u = 0.0f;
  for (int e = threadIdx.x; e < vocab; e += kThreads) {
    const float d = max_nan(to_f32(row[e]) - m, -1000.0f), p = exp2_fast(d * kLog2e);
    s += p;
    u = fmaf(p, d, u);
  }
  s = warp_sum(s);
  u = warp_sum(u);
  __syncthreads();  // sh.warp has been read
  if (threadIdx.x % kWarp == 0) sh.warp[threadIdx.x / kWarp] = Sums{0.0f, 0.0f, s, u};
  __syncthreads();
  s = u = 0.0f;
  for (int w = 0; w < kWarps; ++w) {
    s += sh.warp[w].s;
    u += sh.warp[w].u;
  }
  return make_float2(s, u);
}

// kTop: the call asks for alternatives.
template <class T, bool kTop>
__global__ void __launch_bounds__(kThreads, kCtas) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int E = Chunk<T>::kElems;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Shared& sh = *reinterpret_cast<Shared*>(smem_raw);
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  const int tid = threadIdx.x;
  const int row_step = gridDim.x / ranks;
  wait_then_release();

  // Copies the next tile of this block's rows, one after the other, to the next slots of the ring.
  // `plain` tiles lie wholly inside of their row and before the block's last one.
  int64_t fetch_row = blockIdx.x / ranks;
  Row<T> from(a, fetch_row, rank, ranks);
  int fetch_base = from.c0, plain = 0;
  const uint4* src = nullptr;
  auto begin_plain = [&] {
    plain = from.whole(fetch_base, a.vocab) ? max(from.c1 - 1 - fetch_base, 0) / kTile : 0;
    src = reinterpret_cast<const uint4*>(from.at(fetch_base)) + tid;
  };
  begin_plain();
  constexpr uint32_t kSlot = kTile * 16;
  const uint32_t ring = smem_addr(&sh.ring[0][0][tid]), ring_end = ring + kRing * kSlot;
  uint32_t dst = ring, in = ring;
  auto fetch = [&] {
    if (plain > 0) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) cp_async_16(dst + j * kThreads * 16, src + j * kThreads);
      --plain;
      src += kTile;
      fetch_base += kTile;
    } else {
      while (fetch_row < a.rows && fetch_base >= from.c1) {
        fetch_row += row_step;
        if (fetch_row < a.rows) from = Row<T>(a, fetch_row, rank, ranks);
        fetch_base = from.c0;
      }
      if (fetch_row < a.rows) {
#pragma unroll 1
        for (int j = 0; j < kPer; ++j) {
          const int c = fetch_base + j * kThreads + tid;
          if (c < from.c1 && from.whole(c, a.vocab)) {
            cp_async_16(dst + j * kThreads * 16, from.at(c));
          } else {
            st_shared_v4(dst + j * kThreads * 16, from.partial(c, a.vocab));
          }
        }
        fetch_base += kTile;
        begin_plain();
      }
    }
    cp_async_commit();
    dst = dst + kSlot == ring_end ? ring : dst + kSlot;
  };
#pragma unroll
  for (int i = 0; i < kRing - 1; ++i) fetch();

  for (int64_t row_index = blockIdx.x / ranks; row_index < a.rows; row_index += row_step) {
    const Row<T> r(a, row_index, rank, ranks);
    if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    Sums sums = Sums::none();
    if constexpr (kTop) {
      if (tid == 0) sh.listed = sh.picked = sh.keyed = 0;
    }

    int tile = 0;
    float least = -INFINITY;
    int renew_at = 0, last_slot = 0;
    for (int base = r.c0; base < r.c1; base += kTile, ++tile) {
      cp_async_wait<kRing - 2>();
      uint4 now[kPer];
#pragma unroll
      for (int j = 0; j < kPer; ++j) now[j] = ld_shared_v4(in + j * kThreads * 16);
      last_slot = (in - ring) / kSlot;
      in = in + kSlot == ring_end ? ring : in + kSlot;
      fetch();
      uint32_t most = max_words<T>(now[0]);
#pragma unroll
      for (int j = 1; j < kPer; ++j) most = max_word<T>(most, max_words<T>(now[j]));
      const float top = max_of_word<T>(most);
      if (top > sums.m) {
        sums.m = top;
        sums.rescale(Sums::reference(top));
      }
      if constexpr (kTop) {
        if (tile == renew_at) {
          publish(sh, sums.m);
          if (tile == 0) {
            if (tid == 0) *const_cast<volatile float*>(&sh.least) = -INFINITY;  // not the last row's
            __syncthreads();
            least = from_order_key(block_threshold(sh, a.top));
          } else if (__popc(tile - 1) % kWarps == tid / kWarp) {
            // Maxima only grow, so any view of them gives a threshold that at least n elements
            // reach; where two renewals overlap the lower one may stay, which costs entries only.
            __syncwarp();
            const float renewed = from_order_key(warp_threshold(sh, a.top));
            if (tid % kWarp == 0) *const_cast<volatile float*>(&sh.least) = renewed;
            __syncwarp();
          }
          renew_at = max(2 * tile, 1);
        }
        least = fmaxf(least, *const_cast<volatile float*>(&sh.least));
        note(sh, top, least, tile * kTile + tid);
      }
      const float2 scale = make_float2(kLog2e, kLog2e), c = make_float2(-sums.c, -sums.c);
      const uint32_t low = word_of<T>(kLowest<T>);
      float2 s = make_float2(sums.s, 0.0f), u = make_float2(sums.u, 0.0f);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        Chunk<T> v;
        v.set(make_uint4(max_word<T>(now[j].x, low), max_word<T>(now[j].y, low),
                         max_word<T>(now[j].z, low), max_word<T>(now[j].w, low)));
#pragma unroll
        for (int i = 0; i < E; i += 2) {
          const float2 x = __ffma2_rn(make_float2(v.v[i], v.v[i + 1]), scale, c);
          const float2 e = make_float2(exp2_fast(x.x), exp2_fast(x.y));
          s = __fadd2_rn(s, e);
          u = __ffma2_rn(e, x, u);
        }
      }
      sums.s = s.x + s.y;
      sums.u = u.x + u.y;
    }
    if constexpr (kTop) {
      if (tile > 1) publish(sh, sums.m);
    }

    // the block's sums
    sums.join_lanes();
    if (tid % kWarp == 0) sh.warp[tid / kWarp] = sums;
    __syncthreads();
    uint32_t least_key = 0;
    if constexpr (kTop) {
      // the maxima of a row of one tile are those of its first threshold
      least_key = tile == 1 ? sh.threshold : block_threshold(sh, a.top);
      if (sh.listed > kList) remake_list<T>(sh, r, a.vocab, least_key);
      // the elements of the entries that reach the threshold, a lane an element
      const int listed = min(sh.listed, kList);
      const int lane = tid % kWarp;
      for (int e0 = tid - lane; e0 < listed; e0 += kThreads) {
        const Key entry = e0 + lane < listed ? sh.list[e0 + lane] : 0;
        append(sh.picks, &sh.picked, kPicks,
               e0 + lane < listed && static_cast<uint32_t>(entry >> 32) >= least_key,
               static_cast<int>(static_cast<uint32_t>(entry)));
      }
      __syncthreads();
      const int picked = min(sh.picked, kPicks);
      for (int e0 = tid / kWarp; e0 < picked; e0 += kAtOnce * kWarps) {
        float x[kAtOnce];
        int index[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const int e = e0 + i * kWarps;
          const int c = r.c0 + (e < picked ? sh.picks[e] : 0) + lane / E * kThreads;
          index[i] = c * E - r.shift + lane % E;
          if (e >= picked || lane >= kPer * E || c >= r.c1 || index[i] >= a.vocab) index[i] = -1;
          // the last tile is still in its slots
          x[i] = 0.0f;
          if (index[i] >= 0) {
            const int in_tile = sh.picks[e] - (tile - 1) * kTile;
            x[i] = to_f32(in_tile >= 0 ? reinterpret_cast<const T*>(
                                             &sh.ring[last_slot][lane / E][in_tile])[lane % E]
                                       : r.row[index[i]]);
          }
        }
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          const uint32_t k = order_key(x[i]);
          append(sh.keys, &sh.keyed, kKeys, index[i] >= 0 && k >= least_key && k > kNegInfKey,
                 make_key(x[i], index[i]));
        }
      }
      __syncthreads();
    }

    // this block's part, in the first block's shared memory
    if (ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    Part* part = ranks > 1 ? &cluster.map_shared_rank(&sh, 0)->parts[rank] : &sh.parts[0];
    if (tid < kWarp) {
      Sums all = tid < kWarps ? sh.warp[tid] : Sums::none();
      all.join_lanes();
      if (tid == 0) part->sums = all;
    }
    if constexpr (kTop) {
      const int count = sh.keyed;
      if (sh.listed <= kList && sh.picked <= kPicks && count <= kKeys) {
        if (tid == 0) part->count = min(count, a.top);
        for (int e = tid; e < count; e += kThreads) {
          const Key mine = sh.keys[e];
          int better = 0;
#pragma unroll 8
          for (int i = 0; i < count; ++i) better += sh.keys[i] > mine;
          if (better < a.top) part->top[better] = mine;
        }
      } else {
        take_one_by_one<T>(sh, r, a.vocab, a.top, part);
      }
    }
    if (ranks > 1) {
      cluster.sync();
      if (rank != 0) continue;  // a row of a cluster is its only one
    } else {
      __syncthreads();
    }

    // the row: every warp joins the parts' sums for itself
    Sums all = sh.parts[0].sums;
    if (ranks > 1) {
      all = tid % kWarp < ranks ? sh.parts[tid % kWarp].sums : Sums::none();
      all.join_lanes();
    }
    // the one pass holds maxima within kFar that -inf, taken as kLowest, is far below
    const bool near = fabsf(all.m) <= kFar && all.m > 0.9f * kLowest<T>;
    float entropy, log_s;
    if (near) {
      log_s = log2f(all.s);
      entropy = (log_s - all.u / all.s) * kLn2;
    } else {
      const float2 su = sum_again<T>(sh, r.row, a.vocab, all.m);
      const float s = su.x, u = su.y;
      log_s = logf(s);
      entropy = log_s - u / s;
    }
    const auto logprob = [&](float x) {
      if (!near) return x - all.m - log_s;
      // far below (-inf, a mask's lowest value) the scaled value may not hold x
      return x < -2.0f * kFar ? x - (all.c + log_s) * kLn2 : (fmaf(x, kLog2e, -all.c) - log_s) * kLn2;
    };
    if (tid == 0) {
      const int64_t t = a.tokens[row_index];
      a.logprobs[row_index] =
          t >= 0 && t < a.vocab ? logprob(to_f32(r.row[t])) : __uint_as_float(0x7FFFFFFFu);
      a.entropy[row_index] = entropy;
    }
    if constexpr (kTop) {
      float* top_logprobs = a.top_logprobs + row_index * a.top;
      int64_t* top_ids = a.top_ids + row_index * a.top;
      const int p = tid / kMaxTop, i = tid % kMaxTop;
      int total = 0;
      for (int q = 0; q < ranks; ++q) total += sh.parts[q].count;
      if (p < ranks && i < sh.parts[p].count) {
        const Key mine = sh.parts[p].top[i];
        // a part's entries are in order: its own come before it, of the others a binary search
        // counts those that are larger
        int better = i;
#pragma unroll
        for (int q = 0; q < kMaxCluster; ++q) {
          if (q >= ranks || q == p) continue;
          const Part& other = sh.parts[q];
          int larger = 0;
#pragma unroll
          for (int step = kMaxTop / 2; step > 0; step /= 2) {
            if (larger + step <= other.count && other.top[larger + step - 1] > mine) larger += step;
          }
          if (larger < other.count && other.top[larger] > mine) ++larger;
          better += larger;
        }
        if (better < a.top) {
          top_logprobs[better] = logprob(key_value(mine));
          top_ids[better] = key_index(mine);
        }
      }
      if (total < a.top && tid < kWarp) {
        // fewer than `top` logits above -inf: the lowest indices of the -inf ones follow
        for (int e0 = 0, at = total; e0 < a.vocab && at < a.top; e0 += kWarp) {
          const bool masked = e0 + tid < a.vocab && to_f32(r.row[e0 + tid]) == -INFINITY;
          const uint32_t who = __ballot_sync(0xffffffffu, masked);
          const int mine = at + __popc(who & ((1u << tid) - 1));
          if (masked && mine < a.top) {
            top_logprobs[mine] = logprob(-INFINITY);
            top_ids[mine] = e0 + tid;
          }
          at += __popc(who);
        }
      }
    }
    __syncthreads();  // the parts and the list are written again by the next row
  }
}

template <class T>
cudaError_t launch(const LogprobArgs& a, cudaStream_t stream) {
  const int64_t chunks = (static_cast<int64_t>(a.vocab) + 2 * Chunk<T>::kElems) / Chunk<T>::kElems;
  const int room = kCtas * sm_count();
  // A row is split as long as every thread keeps about a chunk (so no block is without one) and there
  // are at most two blocks an SM: what follows a row's stream costs a block as much as several tiles (64
  // rows of 128256 with 20 alternatives: 16.5 us in clusters of 4, 23.7 in clusters of 8).
  int cluster = 1;
  while (cluster < kMaxCluster && static_cast<int64_t>(a.rows) * cluster <= sm_count() &&
         chunks > static_cast<int64_t>(cluster) * kThreads) {
    cluster *= 2;
  }
  const auto kernel = a.top > 0 ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>;
  static std::once_flag once[2][64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  std::call_once(once[a.top > 0][dev & 63], [&] {
    err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Shared));
  });
  if (err != cudaSuccess) return err;
  const int blocks = cluster > 1 ? a.rows * cluster : std::min(a.rows, room);
  return launch_serialised(kernel, dim3(blocks), dim3(kThreads), sizeof(Shared), stream, cluster, a);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& a, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case kWeightF32: return launch<float>(a, stream);
    case kWeightF16: return launch<half>(a, stream);
    default: return launch<__nv_bfloat16>(a, stream);
  }
}

}  // namespace i4
