// Eviction from a paged cache by accumulated attention weight. Per sequence and KV head, of n
// positions the last `recent` stay, and of the older ones the budget - recent with the largest
// weights (of equal ones the first); keys, values and weights of what stays go to the pages of a
// new block table, in their old order.
//
// Two kernels. The choice: one block a (sequence, head), the k-th largest weight by a radix select
// over the bits of the weights as ordered integers (11 + 11 + 10 bits, a histogram in shared memory
// each), then the chosen positions in order by counting within and across warps. It reads 4 bytes
// a position. The copy: a warp a (position, head), 16 bytes a lane, bound by HBM. The new pages are
// not the old ones, so every block of the copy is independent of the others and sequences may
// share old pages (a common prefix).
#include <mutex>

#include "decode.cuh"
#include "kernels.h"

namespace i4 {
namespace {

constexpr int kSelectThreads = 512;
constexpr int kSelectWarps = kSelectThreads / kWarp;
constexpr int kBins = 2048;
constexpr int kReads = 8;  // weights a thread has in flight
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

// Sum of v over this thread and those before it. Ends with a barrier.
__device__ __forceinline__ int block_prefix(int v, int* warp_sums) {
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
#pragma unroll
  for (int off = 1; off < kWarp; off *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  if (lane == kWarp - 1) warp_sums[warp] = v;
  __syncthreads();
  int before = lane < warp ? warp_sums[lane] : 0;
#pragma unroll
  for (int off = kWarp / 2; off > 0; off >>= 1) before += __shfl_xor_sync(0xffffffffu, before, off);
  __syncthreads();
  return v + before;
}

__global__ void __launch_bounds__(kSelectThreads, 3)
    evict_select_kernel(const PagedEvictArgs a, const Divider by_page, int held, int* status) {
  extern __shared__ uint32_t keys[];  // [held]
  __shared__ int bins[kBins];
  __shared__ int warp_sums[kSelectWarps], found_bin, found_above;
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
  auto read_key = [&](int j) -> uint32_t {
    const int block = by_page.quotient(j), p = table[block];
    if (static_cast<unsigned>(p) >= static_cast<unsigned>(a.cache.num_blocks)) {
      bad_page(status);
      return 0;
    }
    return order_key(a.cache.weights[(static_cast<int64_t>(p) * hkv + head) * page + j - block * page]);
  };
  for (int j0 = tid; j0 < min(old, held); j0 += kReads * kSelectThreads) {
    uint32_t k[kReads];  // kept apart from the stores, so that the reads do not wait for each other
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      const int j = j0 + i * kSelectThreads;
      k[i] = j < min(old, held) ? read_key(j) : 0;
    }
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      const int j = j0 + i * kSelectThreads;
      if (j < min(old, held)) keys[j] = k[i];
    }
  }
  auto key = [&](int j) { return j < held ? keys[j] : read_key(j); };

  // the want-th largest key, digit by digit
  uint32_t prefix = 0, mask = 0;
  int left = want;  // rank still to find among the keys that match the prefix
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const int width = pass == 2 ? 10 : 11;
    for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0;
    __syncthreads();
    for (int j = tid; j < old; j += kSelectThreads) {
      const uint32_t k = key(j);
      if ((k & mask) == prefix) atomicAdd(&bins[(k >> shift) & ((1u << width) - 1)], 1);
    }
    __syncthreads();
    // thread t owns the bins t kOwn ... counted from the top; `above`: the keys in bins above them
    constexpr int kOwn = kBins / kSelectThreads;
    const int hi = kBins - 1 - kOwn * tid;
    int own = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) own += bins[hi - i];
    int above = block_prefix(own, warp_sums) - own;
    if (above < left && left <= above + own) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int here = bins[hi - i];
        if (above < left && left <= above + here) {
          found_bin = hi - i;
          found_above = above;
        }
        above += here;
      }
    }
    __syncthreads();
    left -= found_above;
    prefix |= static_cast<uint32_t>(found_bin) << shift;
    mask |= ((1u << width) - 1) << shift;
    __syncthreads();
  }
  const uint32_t least = prefix;  // keys above it stay, and the first `left` of those equal to it

  // each warp owns a contiguous range, so ranks follow from counts of the warps before it
  const int range = ((old + kSelectWarps - 1) / kSelectWarps + kWarp - 1) / kWarp * kWarp;
  const int j0 = min(warp * range, old), j1 = min(j0 + range, old);
  int gt = 0, eq = 0;
  for (int j = j0; j < j1; j += kWarp) {
    const uint32_t k = j + lane < j1 ? key(j + lane) : 0;
    gt += __popc(__ballot_sync(0xffffffffu, j + lane < j1 && k > least));
    eq += __popc(__ballot_sync(0xffffffffu, j + lane < j1 && k == least));
  }
  // positions above `least` and equal to it before this warp's range
  const int gt_upto = block_prefix(lane == 0 ? gt : 0, warp_sums);
  const int eq_upto = block_prefix(lane == 0 ? eq : 0, warp_sums);
  int at = __shfl_sync(0xffffffffu, gt_upto, 0) - gt, eq_at = __shfl_sync(0xffffffffu, eq_upto, 0) - eq;
  const uint32_t below = (1u << lane) - 1;
  for (int j = j0; j < j1; j += kWarp) {
    const uint32_t k = j + lane < j1 ? key(j + lane) : 0;
    const uint32_t gts = __ballot_sync(0xffffffffu, j + lane < j1 && k > least);
    const uint32_t eqs = __ballot_sync(0xffffffffu, j + lane < j1 && k == least);
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

// `span` positions a warp, at most 32.
__global__ void __launch_bounds__(kCopyThreads)
    evict_copy_kernel(const PagedEvictArgs a, const Divider by_page, int span, int* status) {
  extern __shared__ __align__(16) unsigned char ring_raw[];
  wait_then_release();
  const PagedCache& c = a.cache;
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  const int b = blockIdx.y;
  const int kept = a.new_lens[b];
  const int j0 = blockIdx.x * span;
  if (j0 >= kept) return;
  const int* table = a.table + static_cast<int64_t>(b) * a.max_blocks;
  const int* new_table = a.new_table + static_cast<int64_t>(b) * a.new_blocks;
  const int vectors = c.dim / 8;  // 16-byte pieces of a row of keys
  const int parts = (2 * vectors + kWarp - 1) / kWarp;  // a position's key and value, a piece a lane
  const int count = min(span, kept - j0);
  const uint32_t ring = smem_addr(ring_raw) + (warp * kDepth * kWarp + lane) * 16;

  for (int h = warp; h < c.hkv; h += kCopyWarps) {
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
  const int held = static_cast<int>(most < kHeldKeys ? most : kHeldKeys);
  const Divider by_page(static_cast<uint32_t>(a.cache.block_size));
  static std::once_flag once[64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  std::call_once(once[dev & 63], [&] {
    err = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kHeldKeys * 4);
    if (err != cudaSuccess) return;
    err = cudaFuncSetAttribute(evict_copy_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               kCopySmem);
  });
  if (err != cudaSuccess) return err;
  err = launch_serialised(evict_select_kernel, dim3(a.batch * a.cache.hkv), dim3(kSelectThreads),
                          static_cast<size_t>(held) * 4, stream, 1, a, by_page, held, status);
  if (err != cudaSuccess) return err;
  const int64_t longest = a.budget < most ? a.budget : most;
  if (longest == 0) return cudaSuccess;
  // 32 positions a warp where that gives every SM three blocks, down to 8 where it does not
  int span = kWarp;
  while (span > 8 && (longest + span - 1) / span * a.batch < 3 * sm_count()) span /= 2;
  return launch_serialised(evict_copy_kernel,
                           dim3(static_cast<unsigned>((longest + span - 1) / span), a.batch),
                           dim3(kCopyThreads), kCopySmem, stream, 1, a, by_page, span, status);
}

}  // namespace i4
