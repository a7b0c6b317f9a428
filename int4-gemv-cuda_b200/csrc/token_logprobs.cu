// Log probabilities of given tokens, the entropy of each row and its top alternatives, from logits:
//   lse = log sum_j e^{x_j},  logprob = x_t - lse,  entropy = lse - sum_j p_j x_j.
//
// One pass over a row. Each thread keeps the maximum m it has seen with S = sum e^{x - m} and
// U = sum e^{x - m} (x - m), all fp32, rescaled when a tile of its elements raises m; then
//   logprob = x_t - m - log S,  entropy = log S - U / S,
// and the differences x - m keep their small errors. -inf is taken as the type's lowest value (or
// -1e38), which adds 0 to both sums without a test an element; a thread whose maximum is not far
// above that, or beyond 1e38, takes a slower loop with the tests. A NaN or +inf makes its row NaN.
//
// Top alternatives in the same pass: the maxima of 64 groups of threads give a threshold (the n-th
// largest of them: at least n elements reach it), from the first tile and again from all so far at
// the tiles 1, 2, 4, ...; every element that reaches it goes into a list in shared memory, about n
// at each of these steps. Where the list overflows (rising logits), the pass over the row is
// repeated for the list alone, with the threshold from the maxima of the whole row; where that
// overflows too (thousands of equal logits), the n entries are taken one by one. Keys order by
// value, then by lowest index.
//
// Bound by HBM: each logit is read once. With few rows a row is split over a cluster of blocks that
// join their sums and lists through distributed shared memory.
#include <cooperative_groups.h>

#include "decode.cuh"
#include "kernels.h"

namespace i4 {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / kWarp;
constexpr int kPer = 4;        // 16-byte chunks a thread takes of a tile
constexpr int kGroups = 64;    // groups of threads whose maxima give the threshold
constexpr int kList = 2048;    // entries of the list of candidates
constexpr int kPicked = 512;   // of those that reach the last threshold
constexpr int kMaxCluster = 8;

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
  float m, s, u;  // m = -inf: nothing yet
  __device__ __forceinline__ void rescale(float to) {
    // held at -1000: sums far below count 0, not 0 times infinity
    const float d = fmaxf(m - to, -1000.0f), f = exp2_fast(d * kLog2e);
    u = f * fmaf(s, d, u);
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void join(Sums o) {
    const float top = fmaxf(m, o.m);
    if (top != -INFINITY) {
      rescale(top);
      o.rescale(top);
    }
    s += o.s;
    u += o.u;
  }
  __device__ __forceinline__ void join_lanes(int lanes) {
    for (int off = lanes / 2; off > 0; off >>= 1) {
      Sums o;
      o.m = __shfl_xor_sync(0xffffffffu, m, off);
      o.s = __shfl_xor_sync(0xffffffffu, s, off);
      o.u = __shfl_xor_sync(0xffffffffu, u, off);
      join(o);
    }
  }
};

// ---- A chunk in the type it is read in -----------------------------------------------------------

// The larger of two pairs of 16-bit numbers, NaN where either is one.
template <class T>
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b);
template <>
__device__ __forceinline__ uint32_t max2<half>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <>
__device__ __forceinline__ uint32_t max2<__nv_bfloat16>(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// What -inf is taken as: finite, and L times it is too.
template <class T>
constexpr float kLowest = -1e38f;
template <>
constexpr float kLowest<half> = -65504.0f;

template <class T>
__device__ __forceinline__ float chunk_max(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)),
                   max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    const float2 f = unpack2<T>(max2<T>(max2<T>(v.x, v.y), max2<T>(v.z, v.w)));
    return max_nan(f.x, f.y);
  }
}

template <class T>
__device__ __forceinline__ Chunk<T> raised(uint4 v) {  // at least kLowest
  Chunk<T> f;
  if constexpr (sizeof(T) == 4) {
    f.set(v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f.v[i] = max_nan(f.v[i], kLowest<T>);
  } else {
    const uint32_t low = pack2<T>(kLowest<T>, kLowest<T>);
    v.x = max2<T>(v.x, low);
    v.y = max2<T>(v.y, low);
    v.z = max2<T>(v.z, low);
    v.w = max2<T>(v.w, low);
    f.set(v);
  }
  return f;
}

// Two fp32 operations at once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

// What the blocks of a row send to its first block.
struct Part {
  Sums sums;
  int count;  // entries of top
  Key top[kMaxTop];
};

struct Shared {
  uint32_t group_max[kGroups];
  Sums warp[kWarps];
  Key best[kWarps];
  uint32_t threshold;
  int count, picked_count;
  Key picked[kPicked];
  Part parts[kMaxCluster];
  Key list[kList];
};

template <class T>
struct Row {
  static constexpr int E = Chunk<T>::kElems;
  const T* row;
  int vocab;
  int shift;  // elements of the first chunk that lie before the row

  // Chunk c of the row's memory as fp32; what lies outside of the row is -inf.
  __device__ __forceinline__ void load(int c, uint4& raw) const {
    const int e0 = c * E - shift;
    if (e0 >= 0 && e0 + E <= vocab) {
      raw = ld_stream_v4(row + e0);
    } else {
      Chunk<T> f;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        f.v[i] = e0 + i >= 0 && e0 + i < vocab ? to_f32(row[e0 + i]) : -INFINITY;
      }
      raw = f.get();
    }
  }
};

// The threshold for a list that holds the `top` largest: the top-th largest of the groups' maxima
// (0: every element, where fewer groups have elements above -inf).
__device__ __forceinline__ void find_threshold(Shared& sh, float thread_max, int top) {
  uint32_t k = order_key(thread_max);
#pragma unroll
  for (int off = kThreads / kGroups / 2; off > 0; off >>= 1) {
    k = max(k, __shfl_xor_sync(0xffffffffu, k, off));
  }
  if (threadIdx.x % (kThreads / kGroups) == 0) sh.group_max[threadIdx.x / (kThreads / kGroups)] = k;
  __syncthreads();
  if (threadIdx.x < kGroups) {
    const uint32_t mine = sh.group_max[threadIdx.x];
    int rank = 0;
#pragma unroll 16
    for (int i = 0; i < kGroups; ++i) {
      const uint32_t other = sh.group_max[i];
      rank += other > mine || (other == mine && i < static_cast<int>(threadIdx.x));
    }
    if (rank == top - 1) sh.threshold = mine;
  }
  __syncthreads();
}

template <class T>
__device__ __forceinline__ void collect(Shared& sh, const uint4& raw, float top, uint32_t least,
                                        float least_value, int first_index) {
  if (top < least_value) return;  // not taken with a NaN on either side
  Chunk<T> v;
  v.set(raw);
#pragma unroll
  for (int i = 0; i < Chunk<T>::kElems; ++i) {
    const uint32_t k = order_key(v.v[i]);
    if (k >= least && k > kNegInfKey && sh.count <= kList) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < kList) sh.list[at] = make_key(v.v[i], first_index + i);
    }
  }
}

// kTop: the call asks for alternatives.
template <class T, bool kTop>
__global__ void __launch_bounds__(kThreads, 4) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int E = Chunk<T>::kElems;
  __shared__ Shared sh;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
  const int64_t row_index = blockIdx.x / ranks;
  wait_then_release();

  const T* row = static_cast<const T*>(a.logits) + row_index * a.row_stride;
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(row) / sizeof(T) % E);
  const Row<T> r{row, a.vocab, shift};
  const int64_t chunks = (static_cast<int64_t>(shift) + a.vocab + E - 1) / E;
  const int c0 = static_cast<int>(chunks * rank / ranks);
  const int c1 = static_cast<int>(chunks * (rank + 1) / ranks);
  const int tid = threadIdx.x;
  if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  Sums sums{-INFINITY, 0.0f, 0.0f};
  uint32_t least = 0;
  float least_value = -INFINITY;
  uint4 now[kPer], next[kPer];
  const uint4 nothing = [] {
    Chunk<T> f;
#pragma unroll
    for (int i = 0; i < E; ++i) f.v[i] = -INFINITY;
    return f.get();
  }();
  auto fetch = [&](int base, uint4 (&to)[kPer]) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int c = base + j * kThreads + tid;
      to[j] = nothing;
      if (c < c1) r.load(c, to[j]);
    }
  };
  auto new_threshold = [&](float thread_max) {
    find_threshold(sh, thread_max, a.top);
    least = sh.threshold;
    least_value = from_order_key(least);
  };
  if (tid == 0) sh.count = sh.picked_count = 0;
  fetch(c0, now);
  int tile = 0;
  for (int base = c0; base < c1; base += kPer * kThreads, ++tile) {
    fetch(base + kPer * kThreads, next);
    float tops[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) tops[j] = chunk_max<T>(now[j]);
    const float top = max_nan(max_nan(tops[0], tops[1]), max_nan(tops[2], tops[3]));
    static_assert(kPer == 4, "the maximum of a tile");
    if (top > sums.m) sums.rescale(top);
    if constexpr (kTop) {
      if ((tile & (tile - 1)) == 0) new_threshold(sums.m);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        collect<T>(sh, now[j], tops[j], least, least_value, (base + j * kThreads + tid) * E - shift);
      }
    }
    if (sums.m > 0.9f * kLowest<T> && sums.m < 1e38f) {
      const float2 scale = make_float2(kLog2e, kLog2e), m = make_float2(-sums.m, -sums.m);
      float2 s = make_float2(sums.s, 0.0f), u = make_float2(sums.u, 0.0f);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const Chunk<T> v = raised<T>(now[j]);
#pragma unroll
        for (int i = 0; i < E; i += 2) {
          const float2 d = add2(make_float2(v.v[i], v.v[i + 1]), m);
          const float2 x = mul2(d, scale);
          const float2 e = make_float2(exp2_fast(x.x), exp2_fast(x.y));
          s = add2(s, e);
          u = fma2(e, d, u);
        }
      }
      sums.s = s.x + s.y;
      sums.u = u.x + u.y;
    } else {
      const float m = sums.m == -INFINITY ? 0.0f : sums.m;
#pragma unroll 1
      for (int j = 0; j < kPer; ++j) {
        Chunk<T> v;
        v.set(now[j]);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const float d = max_nan(v.v[i] - m, -1000.0f), e = exp2_fast(d * kLog2e);
          sums.s += e;
          sums.u = fmaf(e, d, sums.u);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) now[j] = next[j];
  }

  const float thread_max = sums.m;

  // the block's sums
  sums.join_lanes(kWarp);
  if (tid % kWarp == 0) sh.warp[tid / kWarp] = sums;
  __syncthreads();
  if constexpr (kTop) {
    if (sh.count > kList) {
      __syncthreads();  // all have read the count
      if (tid == 0) sh.count = 0;
      new_threshold(thread_max);
      for (int c = c0 + tid; c < c1; c += kThreads) {
        uint4 raw;
        r.load(c, raw);
        collect<T>(sh, raw, chunk_max<T>(raw), least, least_value, c * E - shift);
      }
      __syncthreads();
    } else if (sh.count > a.top && tile > 1) {
      new_threshold(thread_max);  // only what reaches the threshold of the whole row is ranked below
    }
  }

  // this block's part, in the first block's shared memory
  if (ranks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  Part* part = ranks > 1 ? &cluster.map_shared_rank(&sh, 0)->parts[rank] : &sh.parts[0];
  if (tid < kWarp) {
    Sums all = tid < kWarps ? sh.warp[tid] : Sums{-INFINITY, 0.0f, 0.0f};
    all.join_lanes(kWarp);
    if (tid == 0) part->sums = all;
  }
  if constexpr (kTop) {
    const int listed = sh.count;
    if (listed <= kList) {
      const Key* keys = sh.list;
      int count = listed;
      if (listed > 2 * kMaxTop) {
        for (int e = tid; e < listed; e += kThreads) {
          if (static_cast<uint32_t>(sh.list[e] >> 32) >= least) {
            const int at = atomicAdd(&sh.picked_count, 1);
            if (at < kPicked) sh.picked[at] = sh.list[e];
          }
        }
        __syncthreads();
        if (sh.picked_count <= kPicked) {
          keys = sh.picked;
          count = sh.picked_count;
        }
      }
      if (tid == 0) part->count = min(count, a.top);
      for (int e = tid; e < count; e += kThreads) {
        const Key mine = keys[e];
        int better = 0;
        for (int i = 0; i < count; ++i) better += keys[i] > mine;
        if (better < a.top) part->top[better] = mine;
      }
    } else {
      Key last = ~static_cast<Key>(0);
      int got = 0;
      while (got < a.top) {
        Key best = 0;
        for (int c = c0 + tid; c < c1; c += kThreads) {
          uint4 raw;
          r.load(c, raw);
          Chunk<T> v;
          v.set(raw);
#pragma unroll
          for (int i = 0; i < E; ++i) {
            const int index = c * E - shift + i;
            const Key k = make_key(v.v[i], index);
            if (index >= 0 && index < a.vocab && k < last && k > best) best = k;
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
  }
  if (ranks > 1) {
    cluster.sync();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }

  // the row: every warp joins the parts' sums for itself
  Sums all = tid % kWarp < ranks ? sh.parts[tid % kWarp].sums : Sums{-INFINITY, 0.0f, 0.0f};
  all.join_lanes(kWarp);
  const float log_s = logf(all.s);
  if (tid == 0) {
    const int64_t t = a.tokens[row_index];
    a.logprobs[row_index] =
        t >= 0 && t < a.vocab ? to_f32(row[t]) - all.m - log_s : __uint_as_float(0x7FFFFFFFu);
    a.entropy[row_index] = log_s - all.u / all.s;
  }
  if constexpr (kTop) {
    float* top_logprobs = a.top_logprobs + row_index * a.top;
    int64_t* top_ids = a.top_ids + row_index * a.top;
    int total = 0;
    for (int p = 0; p < ranks; ++p) total += sh.parts[p].count;
    const int p = tid / kMaxTop, i = tid % kMaxTop;
    if (p < ranks && i < sh.parts[p].count) {
      const Key mine = sh.parts[p].top[i];
      int better = 0;
      for (int q = 0; q < ranks; ++q) {
        for (int j = 0; j < sh.parts[q].count; ++j) better += sh.parts[q].top[j] > mine;
      }
      if (better < a.top) {
        top_logprobs[better] = key_value(mine) - all.m - log_s;
        top_ids[better] = key_index(mine);
      }
    }
    if (total < a.top && tid < kWarp) {
      // fewer than `top` logits above -inf: the lowest indices of the -inf ones follow
      for (int e0 = 0, at = total; e0 < a.vocab && at < a.top; e0 += kWarp) {
        const bool masked = e0 + tid < a.vocab && to_f32(row[e0 + tid]) == -INFINITY;
        const uint32_t who = __ballot_sync(0xffffffffu, masked);
        const int mine = at + __popc(who & ((1u << tid) - 1));
        if (masked && mine < a.top) {
          top_logprobs[mine] = -INFINITY - all.m - log_s;
          top_ids[mine] = e0 + tid;
        }
        at += __popc(who);
      }
    }
  }
}

template <class T>
cudaError_t launch(const LogprobArgs& a, cudaStream_t stream) {
  const int64_t chunks = (static_cast<int64_t>(a.vocab) + 2 * Chunk<T>::kElems) / Chunk<T>::kElems;
  int cluster = 1;
  while (cluster < kMaxCluster && static_cast<int64_t>(a.rows) * cluster * 2 <= 2 * sm_count() &&
         chunks > static_cast<int64_t>(cluster) * kThreads) {
    cluster *= 2;
  }
  const auto kernel = a.top > 0 ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>;
  return launch_serialised(kernel, dim3(static_cast<unsigned>(a.rows) * cluster), dim3(kThreads), 0,
                           stream, cluster, a);
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
