// Eviction from a paged cache by accumulated attention weight. Per sequence and KV head, of n
// positions the last `recent` stay, and of the older ones the budget - recent with the largest
// weights (of equal ones the first); keys, values and weights of what stays go to the pages of a
// new block table, in their old order.
//
// Two kernels. The choice: one block a (sequence, head), the k-th largest weight by a radix select
// over the bits of the weights as ordered integers (11 + 11 + 10 bits, a histogram in shared memory
// each), then the chosen positions in order by counting within and across warps. It reads 4 bytes
// a position, four positions at a time where pages allow. The copy is bound by HBM: a warp takes up to
// 32 positions of a head, looks their places up a lane a position, and moves them 16 bytes a lane
// through its own ring in shared memory (cp.async), sixteen reads ahead of the writes; the warps of a
// block take the heads of the same positions, whose rows are neighbours in memory; where the heads are
// fewer than the warps, several warps take a head (13 sequences of up to 20204 to 9886, 2 heads of 64:
// copy 25 us, without that 48). The new pages are not the old ones, so every block of the copy is
// independent of the others and sequences may share old pages (a common prefix).
//
// Measured on B200, 32 sequences of up to 8192 positions to 2048 (bf16, 8 heads of 128): the copy
// 78 us, 6.2 TB/s (0.95 of a plain copy's 6.53; eight reads a lane in registers instead of the ring:
// 108 us), the choice 18 us (bound by instructions), together 101 us; one sequence of 2503 to 1001
// 10.6 us (latency of two kernels).
#include <algorithm>
#include <mutex>

#include "decode.cuh"
#include "kernels.h"

namespace i4 {
namespace {

constexpr int kSelectThreads = 512;
constexpr int kSelectWarps = kSelectThreads / kWarp;
constexpr int kBins = 2048;
constexpr int kHeldKeys = 48 * 1024;  // weights kept in shared memory; longer ones are read again

__device__ __forceinline__ void bad_page(int* status) { atomicExch(status, kStatusBadPage); }

// Length of sequence b as the table can hold it.
__device__ __forceinline__ int clamped_length(int n, int most, int* status) {
  if (n < 0 || n > most) {
    bad_page(status);
    return n < 0 ? 0 : most;
  }
  return n;
}

// Sum of v over this thread and those before it, behind a barrier.
template <class V>
__device__ __forceinline__ V block_prefix(V v, V* warp_sums) {
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
#pragma unroll
  for (int off = 1; off < kWarp; off *= 2) {
    const V o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  if (lane == kWarp - 1) warp_sums[warp] = v;
  __syncthreads();
  V before = lane < warp ? warp_sums[lane] : 0;
#pragma unroll
  for (int off = kSelectWarps / 2; off > 0; off >>= 1) before += __shfl_xor_sync(0xffffffffu, before, off);
  return v + __shfl_sync(0xffffffffu, before, 0);
}

// kFour: pages of a multiple of four positions, whose weights are read four at a time.
template <bool kFour>
__global__ void __launch_bounds__(kSelectThreads, 3)
    evict_select_kernel(const PagedEvictArgs a, const Divider by_page, int held, int* status) {
  extern __shared__ __align__(16) uint32_t keys[];  // [held], held a multiple of four
  __shared__ int bins[kBins];
  __shared__ int warp_sums[kSelectWarps], found_bin, found_above;
  __shared__ unsigned long long warp_pairs[kSelectWarps];
  wait_then_release();
  const int hkv = a.cache.hkv, page = a.cache.block_size;
  const int b = blockIdx.x / hkv, head = blockIdx.x % hkv;
  const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
  const int64_t most = static_cast<int64_t>(a.max_blocks) * page;
  const int n = clamped_length(a.lens[b], most < INT32_MAX ? static_cast<int>(most) : INT32_MAX,
                               status);
  const int kept = min(n, a.budget);
  int* out = a.kept + static_cast<int64_t>(blockIdx.x) * a.budget;
  if (head == 0 && tid == 0) a.new_lens[b] = kept;
  for (int j = kept + tid; j < a.budget; j += kSelectThreads) out[j] = -1;
  if (n <= a.budget) {
    for (int j = tid; j < kept; j += kSelectThreads) out[j] = j;
    return;
  }
  const int recent = min(a.recent, a.budget);
  const int old = n - recent;       // positions to choose from
  const int want = kept - recent;   // how many of them stay (< old)
  for (int j = tid; j < recent; j += kSelectThreads) out[want + j] = old + j;
  if (want == 0) return;

  const int* table = a.table + static_cast<int64_t>(b) * a.max_blocks;
  // the weight of position j, or null
  auto weight_at = [&](int j) -> const float* {
    const int block = by_page.quotient(j), p = table[block];
    if (static_cast<unsigned>(p) >= static_cast<unsigned>(a.cache.num_blocks)) {
      bad_page(status);
      return nullptr;
    }
    return a.cache.weights + (static_cast<int64_t>(p) * hkv + head) * page + (j - block * page);
  };
  auto read_key = [&](int j) -> uint32_t {
    const float* w = weight_at(j);
    return w ? order_key(*w) : 0;
  };
  const int here = min(old, held);  // keys kept in shared memory
  if constexpr (kFour) {
    constexpr int kAtOnce = 2;
    for (int j0 = tid * 4; j0 < here; j0 += kAtOnce * kSelectThreads * 4) {
      float4 w[kAtOnce];
      bool there[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int j = j0 + i * kSelectThreads * 4;
        const float* from = j < here ? weight_at(j) : nullptr;
        there[i] = from != nullptr;
        if (there[i]) w[i] = *reinterpret_cast<const float4*>(from);
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int j = j0 + i * kSelectThreads * 4;
        if (j < here) {  // up to the next multiple of four, which held is
          *reinterpret_cast<uint4*>(&keys[j]) =
              there[i] ? make_uint4(order_key(w[i].x), order_key(w[i].y), order_key(w[i].z),
                                    order_key(w[i].w))
                       : make_uint4(0, 0, 0, 0);
        }
      }
    }
  } else {
    constexpr int kAtOnce = 8;
    for (int j0 = tid; j0 < here; j0 += kAtOnce * kSelectThreads) {
      uint32_t k[kAtOnce];  // kept apart from the stores, so that the reads do not wait for each other
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int j = j0 + i * kSelectThreads;
        k[i] = j < here ? read_key(j) : 0;
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int j = j0 + i * kSelectThreads;
        if (j < here) keys[j] = k[i];
      }
    }
  }

  // the want-th largest key, digit by digit
  constexpr int kOwn = kBins / kSelectThreads;
  const int hi = kBins - 1 - kOwn * tid;  // this thread's bins, counted from the top
#pragma unroll
  for (int i = 0; i < kOwn; ++i) bins[hi - i] = 0;
  __syncthreads();
  uint32_t prefix = 0, mask = 0;
  int left = want;  // rank still to find among the keys that match the prefix
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t digit = pass == 2 ? 0x3FF : 0x7FF;
#pragma unroll 4
    for (int j = tid; j < here; j += kSelectThreads) {
      const uint32_t k = keys[j];
      if ((k & mask) == prefix) atomicAdd(&bins[(k >> shift) & digit], 1);
    }
    for (int j = here + tid; j < old; j += kSelectThreads) {
      const uint32_t k = read_key(j);
      if ((k & mask) == prefix) atomicAdd(&bins[(k >> shift) & digit], 1);
    }
    __syncthreads();
    int own[kOwn], sum = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      own[i] = bins[hi - i];
      bins[hi - i] = 0;  // for the next pass
      sum += own[i];
    }
    int above = block_prefix(sum, warp_sums) - sum;  // keys in the bins above this thread's
    if (above < left && left <= above + sum) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        if (above < left && left <= above + own[i]) {
          found_bin = hi - i;
          found_above = above;
        }
        above += own[i];
      }
    }
    __syncthreads();
    left -= found_above;
    prefix |= static_cast<uint32_t>(found_bin) << shift;
    mask |= digit << shift;
    // found_* and warp_sums are written again behind the next pass's barrier
  }
  const uint32_t least = prefix;  // keys above it stay, and the first `left` of those equal to it

  // each warp owns a contiguous range, so ranks follow from counts of the warps before it
  auto key = [&](int j) { return j < held ? keys[j] : read_key(j); };
  const int range = ((old + kSelectWarps - 1) / kSelectWarps + kWarp - 1) / kWarp * kWarp;
  const int j0 = min(warp * range, old), j1 = min(j0 + range, old);
  int gt = 0, eq = 0;  // of this lane
#pragma unroll 4
  for (int j = j0 + lane; j < j1; j += kWarp) {
    const uint32_t k = key(j);
    gt += k > least;
    eq += k == least;
  }
  // both counts in one number: positions above `least` and equal to it before this warp's range
  const unsigned long long pair = static_cast<unsigned long long>(eq) << 32 | static_cast<uint32_t>(gt);
  const unsigned long long upto = block_prefix(pair, warp_pairs);
  const unsigned long long start = __shfl_sync(0xffffffffu, upto - pair, 0);
  int at = static_cast<int>(static_cast<uint32_t>(start)), eq_at = static_cast<int>(start >> 32);
  const uint32_t below = (1u << lane) - 1;
  for (int j = j0; j < j1; j += kWarp) {
    const bool inside = j + lane < j1;
    const uint32_t k = inside ? key(j + lane) : 0;
    const uint32_t gts = __ballot_sync(0xffffffffu, inside && k > least);
    const uint32_t eqs = __ballot_sync(0xffffffffu, inside && k == least);
    const int my_eq = eq_at + __popc(eqs & below);
    const bool stays = (gts >> lane & 1) || ((eqs >> lane & 1) && my_eq < left);
    if (stays) out[at + __popc(gts & below) + min(my_eq, left)] = j + lane;
    at += __popc(gts);
    eq_at += __popc(eqs);
  }
}

constexpr int kCopyThreads = 256;
constexpr int kCopyWarps = kCopyThreads / kWarp;
constexpr int kDepth = 16;  // 16-byte pieces a lane has in flight
constexpr int kCopySmem = kCopyWarps * kDepth * kWarp * 16;

// `span` positions a warp, at most 32; with few heads `groups` warps a head, each with its positions.
__global__ void __launch_bounds__(kCopyThreads)
    evict_copy_kernel(const PagedEvictArgs a, const Divider by_page, int span, int groups,
                      int* status) {
  extern __shared__ __align__(16) unsigned char ring_raw[];
  wait_then_release();
  const PagedCache& c = a.cache;
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  const int b = blockIdx.y;
  const int kept = a.new_lens[b];
  const int group = groups > 1 ? warp / c.hkv : 0;
  const int j0 = (blockIdx.x * groups + group) * span;
  if (group >= groups || j0 >= kept) return;
  const int* table = a.table + static_cast<int64_t>(b) * a.max_blocks;
  const int* new_table = a.new_table + static_cast<int64_t>(b) * a.new_blocks;
  const int vectors = c.dim / 8;  // 16-byte pieces of a row of keys
  const int parts = (2 * vectors + kWarp - 1) / kWarp;  // a position's key and value, a piece a lane
  const int count = min(span, kept - j0);
  const uint32_t ring = smem_addr(ring_raw) + (warp * kDepth * kWarp + lane) * 16;

  for (int h = warp - group * c.hkv; h < c.hkv; h += kCopyWarps) {
    // this lane's position: where it is and where it goes
    int from_page = -1, from_off = 0, to_page = -1, to_off = 0;
    if (lane < count) {
      const int j = j0 + lane;
      const int src = a.kept[(static_cast<int64_t>(b) * c.hkv + h) * a.budget + j];
      const int sb = by_page.quotient(src), db = by_page.quotient(j);
      from_page = table[sb];
      to_page = new_table[db];
      from_off = src - sb * c.block_size;
      to_off = j - db * c.block_size;
      if (static_cast<unsigned>(from_page) >= static_cast<unsigned>(c.num_blocks) ||
          static_cast<unsigned>(to_page) >= static_cast<unsigned>(c.num_blocks)) {
        bad_page(status);
        from_page = -1;
      } else {
        c.weights[(static_cast<int64_t>(to_page) * c.hkv + h) * c.block_size + to_off] =
            c.weights[(static_cast<int64_t>(from_page) * c.hkv + h) * c.block_size + from_off];
      }
    }
    for (int part = 0; part < parts; ++part) {
      const int piece = part * kWarp + lane;
      const bool value = piece >= vectors;
      const int64_t x = (value ? piece - vectors : piece) * 8 + h * (value ? c.v_head : c.k_head);
      uint16_t* cache = static_cast<uint16_t*>(value ? c.v : c.k) + x;  // 16-bit words of either type
      const int64_t block = value ? c.v_block : c.k_block, token = value ? c.v_token : c.k_token;
      auto read = [&](int r) {
        const int page = __shfl_sync(0xffffffffu, from_page, r % kWarp);
        const int off = __shfl_sync(0xffffffffu, from_off, r % kWarp);
        if (r < count && page >= 0 && piece < 2 * vectors) {
          cp_async_16(ring + r % kDepth * kWarp * 16, cache + page * block + off * token);
        }
        cp_async_commit();
      };
#pragma unroll 4
      for (int r = 0; r < kDepth; ++r) read(r);
#pragma unroll 4
      for (int r = 0; r < count; ++r) {
        cp_async_wait<kDepth - 1>();
        const uint4 held = ld_shared_v4(ring + r % kDepth * kWarp * 16);
        const bool there = __shfl_sync(0xffffffffu, from_page, r) >= 0;
        const int page = __shfl_sync(0xffffffffu, to_page, r);
        const int off = __shfl_sync(0xffffffffu, to_off, r);
        if (there && piece < 2 * vectors) {
          *reinterpret_cast<uint4*>(cache + page * block + off * token) = held;
        }
        read(r + kDepth);
      }
      cp_async_wait<0>();  // empty groups; the ring starts anew
    }
  }
}

}  // namespace

cudaError_t launch_paged_evict(const PagedEvictArgs& a, cudaStream_t stream) {
  int* status = device_status_word();
  if (!status) return cudaErrorInitializationError;
  const int64_t most = static_cast<int64_t>(a.max_blocks) * a.cache.block_size;
  const int held = static_cast<int>(std::min<int64_t>((most + 3) / 4 * 4, kHeldKeys));
  const bool four = a.cache.block_size % 4 == 0 && reinterpret_cast<uintptr_t>(a.cache.weights) % 16 == 0;
  const auto select = four ? evict_select_kernel<true> : evict_select_kernel<false>;
  const Divider by_page(static_cast<uint32_t>(a.cache.block_size));
  static std::once_flag once[2][64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  std::call_once(once[four][dev & 63], [&] {
    err = cudaFuncSetAttribute(select, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kHeldKeys * 4);
    if (err != cudaSuccess) return;
    err = cudaFuncSetAttribute(evict_copy_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kCopySmem);
  });
  if (err != cudaSuccess) return err;
  err = launch_serialised(select, dim3(a.batch * a.cache.hkv), dim3(kSelectThreads),
                          static_cast<size_t>(held) * 4, stream, 1, a, by_page, held, status);
  if (err != cudaSuccess) return err;
  const int64_t longest = a.budget < most ? a.budget : most;
  if (longest == 0) return cudaSuccess;
  const int groups = std::max(1, kCopyWarps / a.cache.hkv);
  // 32 positions a warp where that gives every SM three blocks, down to 8 where it does not
  auto blocks = [&](int span) { return (longest + span * groups - 1) / (span * groups); };
  int span = kWarp;
  while (span > 8 && blocks(span) * a.batch < 3 * sm_count()) span /= 2;
  return launch_serialised(evict_copy_kernel, dim3(static_cast<unsigned>(blocks(span)), a.batch),
                           dim3(kCopyThreads), kCopySmem, stream, 1, a, by_page, span, groups, status);
}

}  // namespace i4
