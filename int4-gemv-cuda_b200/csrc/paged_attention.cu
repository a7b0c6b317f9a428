// Attention of one new token a sequence over a paged cache of keys and values:
//   s_hj = scale q_h . k_j,  p_h = softmax_j(s_h),  o_h = sum_j p_hj v_j,
// query head h reading KV head h / (hq / hkv). Optionally the call brings the new token's key and
// value (written to the last position's slot and used from the call's tensors), and adds every
// position's attention weight, summed over the query heads of its KV head, to a buffer that
// eviction goes by.
//
// Bound by HBM and by the latency of a warp's chain of instructions: the cache is read once, 4 hq / hkv
// operations an element. Measured on B200 (fp16, 128 dims, 64 query and 8 KV heads): one sequence of
// 131072 positions 98 us, 5.5 TB/s (0.84 of a plain copy's 6.53); 64 sequences of 512 to 8192 194 us
// (0.86), 207 on another card. Of what is missing, 7 to 10 us are the scan of the lengths, the first
// loads and the second kernel; in the rest the issue slots are a third busy, the tensor pipe an eighth,
// and three warps a scheduler wait for their own results and copies. Weights cost 7 us more at 24
// sequences of up to 4096 (48 to 55 us). Small calls are bound by latency alone: 701 positions of 32
// query heads 7.6 us.
//
// Work: an item is (sequence, KV head, block of 8 or 16 query heads), cut into tiles of positions.
// All tiles in order are split evenly over the blocks of the grid whatever the lengths are, so a
// block works through the end of one item, whole items, and the beginning of another; an item that
// several blocks share is joined by a second kernel from partial sums in the workspace, in block
// order (the same result every time, and no counters that a call would have to find cleared).
// Small calls, whose time is mostly latency, give an item a cluster of blocks instead that join
// through distributed shared memory: one kernel, no scan of the lengths, and nearly all of a block's
// tiles on their way at once.
//
// A warp takes 16 positions of a tile and needs no other warp until its segment of an item ends:
// it has its own ring of K and V tiles in shared memory, filled by cp.async (a row's page is looked
// up while older tiles are in flight), its own running maximum and sum, and its own fp32
// accumulators. The warp MMAs have the positions and the dimensions as rows and 8 query heads as
// columns: S^T = K Q^T, O^T = V^T P^T, so a group of 8 heads or fewer fills half of what heads as
// rows would take (P^T gets from the first product's layout to the second's by movmatrix). P is
// given to the MMA as a sum of two 16-bit numbers, so its rounding does not show in the result (in fp16
// what lies far below the largest is another matter, see kLift).
// Positions behind the end are zero-filled in shared memory and masked, so nothing there reaches
// a sum.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <mutex>

#include "decode.cuh"
#include "kernels.h"

namespace i4 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarpTile = 16;  // positions a warp takes of a tile
constexpr int kMaxCluster = 8;
constexpr int kMaxDim = 256;
// A warp rescales its sums when a score passes their last maximum by this much (log2), not at every new
// maximum.
constexpr float kRise = 8.0f;
// The reference is taken this much below the maximum (log2), so that probabilities begin at 2^kLift. An
// fp16 number has steps of 2^-24 at the least, so what the MMA gets of a probability is off by up to
// 2^-25 there: 2^-32 of the largest one with 7, and 2^(kRise + kLift) still fits the type. bf16 has
// fp32's range and needs none.
template <class T>
constexpr float kLift = 0.0f;
template <>
constexpr float kLift<half> = 7.0f;

// What depends on the head dimension rounded up to DP and the heads of an item, 8 NT; kSmall: the
// kernel for small calls.
template <int DP, int NT, bool kSmall>
struct Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kWarps = DP == 256 ? 6 : kSmall ? 8 : 4;
  static constexpr int kThreads = kWarps * kWarp;
  static constexpr int kTile = kWarps * kWarpTile;
  static constexpr int kStages = DP == 256 ? 2 : kSmall ? (DP == 64 ? 4 : 3) : DP == 64 ? 3 : 2;
  static constexpr int kChunks = DP / 8;            // 16-byte chunks of a row
  static constexpr int kPitch = DP * 2 + 16;        // of a row in shared memory: the eight rows of
                                                    // an ldmatrix fall into different banks
  static constexpr int kHalf = kWarpTile * kPitch;  // K or V of a warp's tile
};
// Blocks an SM, and the ring stages above: what fits the shared memory, measured against its
// neighbours. At 128 dims 3 blocks x 2 stages, against 2 x 3: sequences of 512 to 8192 positions, 64
// of them, 198 against 225 us (the more blocks, the less the end of a segment shows), 131072
// positions 99 against 97 us. Small calls have one block an SM and as many tiles in flight as fit.
template <int DP, int NT>
constexpr int kCtas = DP == 64 ? 3 : DP == 128 ? (NT == 1 ? 3 : 2) : 1;
constexpr int round_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
constexpr int kSmallTiles = 8;  // of a block, at most, in the kernel for small calls

struct Plan {
  PagedAttentionArgs a;
  int group;       // query heads of a KV head
  int rows;        // query heads of an item, at most (8 or 16)
  int head_tiles;  // items of a KV head
  int items;       // items of a sequence: hkv * head_tiles
  int tile;        // positions of a tile
  int item_tiles;  // tiles of a sequence as long as the table
  int cluster;     // blocks of an item (small calls); else 0
  int blocks;      // blocks of the attention kernel
  int max_len;     // positions the table has room for
  int join_warps;   // of a head in the joining kernel
  int join_blocks;  // of that kernel, for the heads
  int score_rows;  // heads of an item rounded up to a pair
  Divider page;
  float* part_o;    // [2 blocks][rows][dim]: the segments of items that a block shares
  float2* part_ml;  // [2 blocks][rows]: their maximum (log2) and sum
  float* lse;       // [batch][hq]: log2 of the sum, for items of one block (weights only)
  float* scores;    // [tiles][tile][score_rows]: log2 scores (weights only)
  int* first_tile;  // [batch + 1]: tiles before each sequence
  int* status;
};

__device__ __forceinline__ int clamped(const Plan& p, int n) { return min(max(n, 0), p.max_len); }
// The position of the new token of a sequence of the given length; -1 where the call brings none or the
// table has no room for it (the last position there is another token's).
__device__ __forceinline__ int new_position(const Plan& p, int given) {
  return p.a.k_new && given <= p.max_len ? given - 1 : -1;
}

// The even split of `total` tiles: block c takes [start(c), start(c + 1)).
struct Split {
  int base, extra;
  __device__ __forceinline__ Split(int total, int blocks) : base(total / blocks), extra(total % blocks) {}
  __device__ __forceinline__ int start(int c) const { return c * base + min(c, extra); }
  __device__ __forceinline__ int owner(int t) const {
    const int big = extra * (base + 1);
    return t < big ? t / (base + 1) : extra + (t - big) / base;
  }
};

// ---- Warp-level pieces ---------------------------------------------------------------------------

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// The transpose of an 8 x 8 matrix of 16-bit numbers, a row of four lanes each.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <class T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1) {
  mma_16816(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4],
                                                   uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 "
      "{%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- A warp's work on a tile ---------------------------------------------------------------------

// Per warp: K and V row of each position of the tile being loaded.
using Rows = const void* [kWarpTile][2];

// By a warp, lanes 0-15 a position each: looks up the rows of 16 positions of sequence b from `pos`
// (this lane's) on, given this lane's page, writes the new token's row where its position `fresh` is among
// them, and starts the copies of K and V to `dst`. Returns the mask of positions that count.
template <class T, class S>
__device__ __forceinline__ uint32_t load_tile(const Plan& p, Rows& rows, uint32_t dst, int b, int n,
                                              int fresh_at, int item, int pos, int page) {
  const PagedAttentionArgs& a = p.a;
  const PagedCache& c = a.cache;
  const int lane = threadIdx.x % kWarp;
  const int kv = item / p.head_tiles;
  bool valid = false, append = false;
  if (lane < kWarpTile) {
    const void* k = c.k;
    const void* v = c.v;
    if (pos < n) {
      if (static_cast<unsigned>(page) < static_cast<unsigned>(c.num_blocks)) {
        const int off = pos - p.page.quotient(pos) * p.page.by;
        valid = true;
        append = pos == fresh_at;
        k = static_cast<const T*>(c.k) + page * c.k_block + off * c.k_token + kv * c.k_head;
        v = static_cast<const T*>(c.v) + page * c.v_block + off * c.v_token + kv * c.v_head;
      } else {
        atomicExch(p.status, kStatusBadPage);
      }
    }
    *reinterpret_cast<ulonglong2*>(rows[lane]) =
        make_ulonglong2(reinterpret_cast<uint64_t>(k), reinterpret_cast<uint64_t>(v));
  }
  const uint32_t mask = __ballot_sync(0xffffffffu, valid);
  const uint32_t fresh = __ballot_sync(0xffffffffu, append);
  __syncwarp();
  if (fresh) {
    // the new token's row: to its slot (once for a KV head), and read from the call's tensors
    const int64_t new_row = (static_cast<int64_t>(b) * c.hkv + kv) * c.dim;
    const int row = __ffs(fresh) - 1;
    if (item % p.head_tiles == 0) {
      uint4* k = static_cast<uint4*>(const_cast<void*>(rows[row][0]));
      uint4* v = static_cast<uint4*>(const_cast<void*>(rows[row][1]));
      for (int i = lane; i < c.dim / 8; i += kWarp) {
        k[i] = reinterpret_cast<const uint4*>(static_cast<const T*>(a.k_new) + new_row)[i];
        v[i] = reinterpret_cast<const uint4*>(static_cast<const T*>(a.v_new) + new_row)[i];
      }
    }
    __syncwarp();
    if (lane == row) {
      rows[row][0] = static_cast<const T*>(a.k_new) + new_row;
      rows[row][1] = static_cast<const T*>(a.v_new) + new_row;
    }
    __syncwarp();
  }
  // a lane copies the same chunk of every kStep-th row
  constexpr int kStep = kWarp / S::kChunks;
  const int chunk = lane % S::kChunks, row0 = lane / S::kChunks;
  dst += row0 * S::kPitch + chunk * 16;
  if (mask == 0xFFFFu && c.dim == S::kChunks * 8) {
#pragma unroll
    for (int i = 0; i < kWarpTile / kStep; ++i) {
      const ulonglong2 kv_row = *reinterpret_cast<const ulonglong2*>(rows[row0 + i * kStep]);
      const uint32_t to = dst + i * kStep * S::kPitch;
      cp_async_16(to, reinterpret_cast<const char*>(kv_row.x) + chunk * 16);
      cp_async_16(to + S::kHalf, reinterpret_cast<const char*>(kv_row.y) + chunk * 16);
    }
  } else {
#pragma unroll 4
    for (int i = 0; i < kWarpTile / kStep; ++i) {
      const int row = row0 + i * kStep;
      const ulonglong2 kv_row = *reinterpret_cast<const ulonglong2*>(rows[row]);
      const bool there = (mask >> row & 1) && chunk * 8 < c.dim;
      const int at = there ? chunk * 16 : 0;
      const uint32_t to = dst + i * kStep * S::kPitch;
      cp_async_16_or_zero(to, reinterpret_cast<const char*>(kv_row.x) + at, there);
      cp_async_16_or_zero(to + S::kHalf, reinterpret_cast<const char*>(kv_row.y) + at, there);
    }
  }
  __syncwarp();  // rows is rewritten by the next tile's
  return mask;
}

// What a row's sums are divided by, given their maximum and sum: where nothing counted they are 0, and
// so is the result.
__device__ __forceinline__ float divisor(float2 ml) { return ml.x == -INFINITY ? 1.0f : ml.y; }

// A warp's queries and sums for an item.
template <class T, int DP, int NT, class S>
struct Sums {
  uint32_t qf[DP / 16][NT][2];
  float o[DP / 16][NT][4];   // dims g, g + 8 of 16 by heads t2, t2 + 1 of 8
  float m[NT][2], l[NT][2];  // heads t2, t2 + 1: the reference of all lanes (a maximum less kLift,
                             // at most kLift + kRise below the largest score), this lane's sum
  bool any;                  // a position has counted

  __device__ __forceinline__ void load_q(const Plan& p, int b, int item) {
    const int dim = p.a.cache.dim, g = threadIdx.x % kWarp / 4, t2 = threadIdx.x % 4 * 2;
    const int kv = item / p.head_tiles, h0 = item % p.head_tiles * S::kRows;
    const T* q = static_cast<const T*>(p.a.q) +
                 (static_cast<int64_t>(b) * p.a.hq + kv * p.group + h0) * dim;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = i * 8 + g, col = k * 16 + j * 8 + t2;
          qf[k][i][j] = h0 + row < p.group && col < dim
                            ? *reinterpret_cast<const uint32_t*>(q + row * dim + col)
                            : 0u;
        }
      }
    }
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
#pragma unroll
      for (int j = 0; j < NT; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      m[j][0] = m[j][1] = -INFINITY;
      l[j][0] = l[j][1] = 0.0f;
    }
    any = false;
  }

  // Adds the 16 positions at `tile`. scores: where this warp's go (kWeights). `after_qk` is called
  // once the queries are not needed any more.
  template <bool kWeights, class F>
  __device__ __forceinline__ void add(const Plan& p, uint32_t tile, uint32_t mask, float* scores,
                                      F after_qk) {
    const int dim = p.a.cache.dim, lane = threadIdx.x % kWarp, g = lane / 4, t2 = lane % 4 * 2;
    // the lanes' rows and chunks in the ldmatrix of K (positions 0-7, 8-15 by k 0-7, then by 8-15)
    // and of V (positions 0-7 by dims 0-7, by 8-15, then positions 8-15)
    const uint32_t k_at = tile + ((lane & 7) + (lane >> 3 & 1) * 8) * S::kPitch + (lane >> 4) * 16;
    const uint32_t v_at =
        tile + ((lane & 7) + (lane >> 4) * 8) * S::kPitch + (lane >> 3 & 1) * 16 + S::kHalf;
    any |= mask != 0;
    // S^T: positions g, g + 8 by heads t2, t2 + 1
    float s[NT][4] = {};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      if (k * 16 < dim) {
        uint32_t f[4];
        ldmatrix_x4(f, k_at + k * 32);
#pragma unroll
        for (int i = 0; i < NT; ++i) mma<T>(s[i], f, qf[k][i][0], qf[k][i][1]);
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] *= p.a.scale_log2;
    }
    after_qk();
    if (mask != 0xFFFFu) {
      const bool at[2] = {(mask >> g & 1) != 0, (mask >> (g + 8) & 1) != 0};
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = at[j / 2] ? s[i][j] : -INFINITY;
      }
    }
    if constexpr (kWeights) {
      float* to = scores + g * p.score_rows;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (i * 8 + t2 < p.score_rows) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            *reinterpret_cast<float2*>(to + r * 8 * p.score_rows + i * 8 + t2) =
                make_float2(s[i][2 * r], s[i][2 * r + 1]);
          }
        }
      }
    }
    float top[NT][2];
    bool rises = false;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float v = fmaxf(s[i][j], s[i][j + 2]);
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
        top[i][j] = fmaxf(v - kLift<T>, m[i][j]);
        // the difference, which is exact where it matters: m + kRise rounds where scores are large
        rises |= v - m[i][j] > kRise + kLift<T>;
      }
    }
    if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float f = m[i][j] == -INFINITY ? 0.0f : exp2_fast(m[i][j] - top[i][j]);
          m[i][j] = top[i][j];
          l[i][j] *= f;
#pragma unroll
          for (int d = 0; d < DP / 16; ++d) {
            o[d][i][j] *= f;
            o[d][i][j + 2] *= f;
          }
        }
      }
    }
    uint32_t hi[NT][2], lo[NT][2];  // positions t2, t2 + 1 (and + 8) by head g
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float ref0 = m[i][0] == -INFINITY ? 0.0f : m[i][0];
      const float ref1 = m[i][1] == -INFINITY ? 0.0f : m[i][1];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float p0 = exp2_fast(s[i][2 * r] - ref0), p1 = exp2_fast(s[i][2 * r + 1] - ref1);
        l[i][0] += p0;
        l[i][1] += p1;
        const uint32_t h = pack2<T>(p0, p1);
        const float2 back = unpack2<T>(h);
        hi[i][r] = transposed(h);
        lo[i][r] = transposed(pack2<T>(p0 - back.x, p1 - back.y));
      }
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      if (d * 16 < dim) {
        uint32_t f[4];
        ldmatrix_x4_trans(f, v_at + d * 32);
#pragma unroll
        for (int i = 0; i < NT; ++i) mma<T>(o[d][i], f, hi[i][0], hi[i][1]);
#pragma unroll
        for (int i = 0; i < NT; ++i) mma<T>(o[d][i], f, lo[i][0], lo[i][1]);
      }
    }
  }

  // By the block: the warps' sums together, into joined and ml[0]. Ends with a barrier. A maximum of
  // -inf then says that nothing counted (an empty item, or pages that are all outside of the cache),
  // which gives zeros; where positions counted, but all scores are -inf, it is the lowest number, and
  // the result 0 / 0.
  __device__ __forceinline__ void join(float (&joined)[S::kRows][DP], float2 (&ml)[S::kWarps][S::kRows]) {
    const int warp = threadIdx.x / kWarp, g = threadIdx.x % kWarp / 4, t2 = threadIdx.x % 4 * 2;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        l[i][j] += __shfl_xor_sync(0xffffffffu, l[i][j], 4);
        l[i][j] += __shfl_xor_sync(0xffffffffu, l[i][j], 8);
        l[i][j] += __shfl_xor_sync(0xffffffffu, l[i][j], 16);
        if (any) m[i][j] = fmaxf(m[i][j], -FLT_MAX);
        if (g == 0) ml[warp][i * 8 + t2 + j] = make_float2(m[i][j], l[i][j]);
      }
    }
    __syncthreads();
    float all_m[NT][2], all_l[NT][2], f[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w) top = fmaxf(top, ml[w][i * 8 + t2 + j].x);
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w) {
          const float2 v = ml[w][i * 8 + t2 + j];
          sum += v.x == -INFINITY ? v.y : v.y * exp2_fast(v.x - top);
        }
        all_m[i][j] = top;
        all_l[i][j] = sum;
        f[i][j] = m[i][j] == -INFINITY ? 1.0f : exp2_fast(m[i][j] - top);
      }
    }
    // the warps add their sums to one place in rounds, each to another share of the dimensions, so
    // the order at every place is fixed and no warp waits for its turn
#pragma unroll 1
    for (int round = 0; round < S::kWarps; ++round) {
      const int share = (warp + round) % S::kWarps;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) {
        if (d % S::kWarps == share) {
#pragma unroll
          for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float* to = &joined[i * 8 + t2 + (j & 1)][d * 16 + g + j / 2 * 8];
              const float v = o[d][i][j] * f[i][j & 1];
              *to = round == 0 ? v : *to + v;
            }
          }
        }
      }
      __syncthreads();
    }
    if (warp == 0 && g == 0) {  // read by all warps above, before the rounds' barriers
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j) ml[0][i * 8 + t2 + j] = make_float2(all_m[i][j], all_l[i][j]);
      }
    }
    __syncthreads();
  }
};

// By a block of kThreads: adds the weights of `positions` positions of KV head kv of sequence b (whose
// new token is at `fresh`), from tile `tile0` of the sequence on, whose scores begin at tile `scores_tile`,
// for one item (block `ht` of the head's query heads) whose rows have the sums row_lse. `ready` (by all threads, if
// there are positions) sees to those while the first loads are on their way.
template <int kThreads, class F>
__device__ __forceinline__ void add_weights(const Plan& p, int b, int kv, int ht, int rows,
                                            int scores_tile, int tile0, int positions, int fresh,
                                            const float* row_lse, F ready) {
  constexpr int kAtOnce = 2, kFirst = 2;  // positions of a thread; pairs of rows loaded before `ready`
  const PagedAttentionArgs& a = p.a;
  const PagedCache& c = a.cache;
  for (int i0 = 0; i0 < positions; i0 += kAtOnce * kThreads) {
    float* to[kAtOnce];
    float2 v[kAtOnce][kFirst];
    float w[kAtOnce];
    int page[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = i0 + k * kThreads + static_cast<int>(threadIdx.x);
      page[k] = -1;
      if (i >= positions) continue;
      page[k] = a.table[static_cast<int64_t>(b) * a.max_blocks + p.page.quotient(tile0 * p.tile + i)];
      const float2* s = reinterpret_cast<const float2*>(
          p.scores + (static_cast<int64_t>(scores_tile) * p.tile + i) * p.score_rows);
#pragma unroll
      for (int r = 0; r < kFirst; ++r) {
        if (2 * r < rows) v[k][r] = s[r];
      }
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int pos = tile0 * p.tile + i0 + k * kThreads + static_cast<int>(threadIdx.x);
      to[k] = nullptr;
      w[k] = 0.0f;
      if (static_cast<unsigned>(page[k]) >= static_cast<unsigned>(c.num_blocks)) continue;
      to[k] = c.weights + (static_cast<int64_t>(page[k]) * c.hkv + kv) * c.block_size +
              (pos - p.page.quotient(pos) * static_cast<int>(p.page.by));
      // a new token's slot may hold what its page was used for before
      if (!(ht == 0 && pos == fresh)) w[k] = *to[k];
    }
    if (i0 == 0) ready();
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (!to[k]) continue;
      const int i = i0 + k * kThreads + static_cast<int>(threadIdx.x);
      const float2* s = reinterpret_cast<const float2*>(
          p.scores + (static_cast<int64_t>(scores_tile) * p.tile + i) * p.score_rows);
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < kFirst; ++r) {
        if (2 * r < rows) sum += exp2_fast(v[k][r].x - row_lse[2 * r]);
        if (2 * r + 1 < rows) sum += exp2_fast(v[k][r].y - row_lse[2 * r + 1]);
      }
#pragma unroll 2
      for (int r = kFirst; 2 * r < rows; ++r) {
        const float2 more = s[r];
        sum += exp2_fast(more.x - row_lse[2 * r]);
        if (2 * r + 1 < rows) sum += exp2_fast(more.y - row_lse[2 * r + 1]);
      }
      *to[k] = w[k] + sum;
    }
  }
}

// ---- Any call: all tiles over all blocks ---------------------------------------------------------

// A position in the order of all tiles: sequence, item of the sequence, tile of the item.
struct Walker {
  int b, item, tile, tiles, n, fresh;  // n: the length; fresh: the position of the new token, or -1

  template <int kTile>
  __device__ __forceinline__ void enter(const Plan& p) {  // to the next sequence with positions
    while (b < p.a.batch) {
      const int given = p.a.lens[b];
      n = clamped(p, given);
      fresh = new_position(p, given);
      if (n > 0) break;
      ++b;
    }
    tiles = (n + kTile - 1) / kTile;
  }
  template <int kTile>
  __device__ __forceinline__ void next(const Plan& p) {
    if (++tile < tiles) return;
    tile = 0;
    if (++item < p.items) return;
    item = 0;
    ++b;
    enter<kTile>(p);
  }
};

template <int DP, int NT>
struct Smem {
  using S = Shape<DP, NT, false>;
  alignas(128) unsigned char ring[S::kWarps][S::kStages][2][S::kHalf];
  Rows rows[S::kWarps];
  uint32_t mask[S::kWarps][S::kStages];  // positions that count
  float joined[S::kRows][DP];
  float2 ml[S::kWarps][S::kRows];
  int scan[S::kWarps];
  int start[3];  // sequence of the block's first tile, tiles before it, its length as given
};

template <class T, int DP, int NT, bool kWeights>
__global__ void __launch_bounds__(Shape<DP, NT, false>::kThreads, kCtas<DP, NT>)
    paged_attention_kernel(const __grid_constant__ Plan p) {
  using S = Shape<DP, NT, false>;
  constexpr int kTile = S::kTile, kThreads = S::kThreads, kWarps = S::kWarps;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  Smem<DP, NT>& sh = *reinterpret_cast<Smem<DP, NT>*>(smem_raw);
  // The joining kernel starts when this one has left: its blocks, waiting beside these, made the next
  // call's start late (16 x 8192 positions of 8 heads: 130 us, against 101 without).
  wait_only();
  const PagedAttentionArgs& a = p.a;
  const PagedCache& c = a.cache;
  const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;

  // Tiles before each sequence: a scan over the batch, a thread a sequence, in rounds. `find` is
  // called with each thread's sequence, the tiles before and in it, and its length as given; returns the
  // tiles in all.
  auto scan = [&](auto find) {
    int before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
      const int b = b0 + tid;
      const int given = b < a.batch ? a.lens[b] : 0;
      const int n = clamped(p, given);
      const int own = (n + kTile - 1) / kTile * p.items;
      if (given != n && blockIdx.x == 0) atomicExch(p.status, kStatusBadPage);
      int t = own;
#pragma unroll
      for (int off = 1; off < kWarp; off *= 2) {
        const int v = __shfl_up_sync(0xffffffffu, t, off);
        if (lane >= off) t += v;
      }
      if (lane == kWarp - 1) sh.scan[warp] = t;
      __syncthreads();
      int sum = 0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) t += sh.scan[w];
        sum += sh.scan[w];
      }
      if (b < a.batch) find(b, before + t - own, own, given);
      before += sum;
      __syncthreads();  // sh.scan is written again
    }
    return before;
  };
  // a batch that fits one round keeps the scan's result in registers
  int my_b = -1, my_before = 0, my_own = 0, my_given = 0;
  const int total = scan([&](int b, int before, int own, int given) {
    if (blockIdx.x == 0) {
      if (b == 0) p.first_tile[0] = 0;
      p.first_tile[b + 1] = before + own;
    }
    my_b = b;
    my_before = before;
    my_own = own;
    my_given = given;
  });
  const Split split(total, p.blocks);
  const int t0 = split.start(blockIdx.x), t1 = split.start(blockIdx.x + 1);
  if (t0 >= t1) return;
  auto is_start = [&](int b, int before, int own, int given) {
    if (before <= t0 && t0 < before + own) {
      sh.start[0] = b;
      sh.start[1] = before;
      sh.start[2] = given;
    }
  };
  if (a.batch <= kThreads) {
    if (my_b >= 0) is_start(my_b, my_before, my_own, my_given);
    __syncthreads();
  } else {
    scan(is_start);
  }
  Walker load;
  load.b = sh.start[0];
  load.n = clamped(p, sh.start[2]);
  load.fresh = new_position(p, sh.start[2]);
  load.tiles = (load.n + kTile - 1) / kTile;
  load.item = (t0 - sh.start[1]) / load.tiles;
  load.tile = (t0 - sh.start[1]) % load.tiles;
  Walker now = load;

  const uint32_t ring = smem_addr(sh.ring[warp]);
  int load_at = t0, load_stage = 0;
  // the page of this lane's position in the tile to load next, read a tile ahead
  auto position = [&] { return load.tile * kTile + warp * kWarpTile + lane; };
  auto read_page = [&] {
    const int pos = position();
    return lane < kWarpTile && load_at < t1 && pos < load.n
               ? a.table[static_cast<int64_t>(load.b) * a.max_blocks + p.page.quotient(pos)]
               : -1;
  };
  int page = read_page();
  auto load_next = [&] {
    if (load_at < t1) {
      const uint32_t mask =
          load_tile<T, S>(p, sh.rows[warp], ring + load_stage * 2 * S::kHalf, load.b, load.n,
                          load.fresh, load.item, position(), page);
      if (lane == 0) sh.mask[warp][load_stage] = mask;
      load.next<kTile>(p);
      ++load_at;
      page = read_page();
    }
    cp_async_commit();
    load_stage = load_stage + 1 == S::kStages ? 0 : load_stage + 1;
  };
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) load_next();

  Sums<T, DP, NT, S> sums;
  sums.load_q(p, now.b, now.item);
  sums.reset();
  int stage = 0, segment = t0;  // first tile of the current segment
  for (int t = t0; t < t1; ++t) {
    cp_async_wait<S::kStages - 2>();
    __syncwarp();
    const uint32_t tile = ring + stage * 2 * S::kHalf;
    const uint32_t mask = sh.mask[warp][stage];
    load_next();
    const bool item_ends = now.tile + 1 == now.tiles;
    const bool changes = item_ends && t + 1 < t1;
    Walker following = now;
    if (changes) following.template next<kTile>(p);
    // the next item's queries are on their way while this one is finished
    const auto next_q = [&] {
      if (changes) sums.load_q(p, following.b, following.item);
    };
    if (mask != 0 || kWeights) {
      sums.template add<kWeights>(
          p, tile, mask,
          kWeights ? p.scores + (static_cast<int64_t>(t) * kTile + warp * kWarpTile) * p.score_rows
                   : nullptr,
          next_q);
    } else {
      next_q();
    }
    __syncwarp();  // this stage is refilled by the next load_next
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
    if (!item_ends && t + 1 < t1) {
      ++now.tile;
      continue;
    }

    // the end of a segment
    sums.join(sh.joined, sh.ml);
    const int kv = now.item / p.head_tiles, h0 = now.item % p.head_tiles * S::kRows;
    const int rows = min(p.group - h0, S::kRows);
    const int head = kv * p.group + h0;
    const bool whole = item_ends && t - segment + 1 == now.tiles;
    if (whole) {
      T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(now.b) * a.hq + head) * c.dim;
      const int pairs = c.dim / 2;
      for (int i = tid; i < rows * pairs; i += kThreads) {
        const int row = i / pairs, d = i % pairs * 2;
        const float l_row = divisor(sh.ml[0][row]);
        *reinterpret_cast<uint32_t*>(out + row * c.dim + d) =
            pack2<T>(sh.joined[row][d] / l_row, sh.joined[row][d + 1] / l_row);
      }
      if (kWeights && tid < rows) {
        p.lse[static_cast<int64_t>(now.b) * a.hq + head + tid] =
            sh.ml[0][tid].x + log2f(sh.ml[0][tid].y);
      }
    } else {
      const int slot = 2 * blockIdx.x + (segment == t0 ? 0 : 1);
      float* to = p.part_o + static_cast<int64_t>(slot) * S::kRows * c.dim;
      for (int i = tid; i < rows * c.dim; i += kThreads) to[i] = sh.joined[i / c.dim][i % c.dim];
      if (tid < rows) p.part_ml[slot * S::kRows + tid] = sh.ml[0][tid];
    }
    __syncthreads();  // joined and ml are written again by the next segment
    if (changes) {
      now = following;
      segment = t + 1;
      sums.reset();
    }
  }
}

// ---- Small calls: a cluster of blocks an item ----------------------------------------------------
//
// Block r of an item's R takes its tiles r, r + R, ...: which tiles a block has does not depend on
// the length, so the pages of all of them are looked up while the length is on its way.
template <int DP, int NT>
struct SmallSmem {
  using S = Shape<DP, NT, true>;
  alignas(128) unsigned char ring[S::kWarps][S::kStages][2][S::kHalf];
  Rows rows[S::kWarps];
  int pages[S::kWarps][kSmallTiles][kWarpTile];
  uint32_t mask[S::kWarps][S::kStages];
  float joined[S::kRows][DP];
  float2 ml[S::kWarps][S::kRows];
  float share[S::kRows][kMaxCluster];  // of the blocks of the cluster in a row's result
  float row_lse[S::kRows];
};

template <class T, int DP, int NT, bool kWeights>
__global__ void __launch_bounds__(Shape<DP, NT, true>::kThreads)
    paged_attention_small_kernel(const __grid_constant__ Plan p) {
  using S = Shape<DP, NT, true>;
  constexpr int kTile = S::kTile, kThreads = S::kThreads;
  extern __shared__ __align__(128) unsigned char smem_raw[];
  SmallSmem<DP, NT>& sh = *reinterpret_cast<SmallSmem<DP, NT>*>(smem_raw);
  wait_then_release();
  const PagedAttentionArgs& a = p.a;
  const PagedCache& c = a.cache;
  const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
  const int ranks = p.cluster, rank = blockIdx.x % ranks, index = blockIdx.x / ranks;
  const int b = index / p.items, item = index % p.items;

  // the pages of this warp's positions, two of the block's tiles at a time
  const int own_most = (p.item_tiles - rank + ranks - 1) / ranks;  // tiles of the longest sequence
#pragma unroll
  for (int k = 0; k < kSmallTiles / 2; ++k) {
    const int i = 2 * k + lane / kWarpTile;
    const int pos = (rank + i * ranks) * kTile + warp * kWarpTile + lane % kWarpTile;
    if (i < own_most) {
      sh.pages[warp][i][lane % kWarpTile] =
          pos < p.max_len ? a.table[static_cast<int64_t>(b) * a.max_blocks + p.page.quotient(pos)] : -1;
    }
  }
  const int given = a.lens[b];
  Sums<T, DP, NT, S> sums;
  sums.load_q(p, b, item);
  sums.reset();
  const int n = clamped(p, given), fresh = new_position(p, given);
  if (given != n && tid == 0) atomicExch(p.status, kStatusBadPage);
  const int tiles = (n + kTile - 1) / kTile;
  const int own = tiles > rank ? (tiles - rank + ranks - 1) / ranks : 0;

  const uint32_t ring = smem_addr(sh.ring[warp]);
  __syncwarp();
  int loaded = 0, load_stage = 0, stage = 0;
  auto load_next = [&] {
    if (loaded < own) {
      const uint32_t mask = load_tile<T, S>(
          p, sh.rows[warp], ring + load_stage * 2 * S::kHalf, b, n, fresh, item,
          (rank + loaded * ranks) * kTile + warp * kWarpTile + lane,
          sh.pages[warp][loaded][lane % kWarpTile]);
      if (lane == 0) sh.mask[warp][load_stage] = mask;
      ++loaded;
    }
    cp_async_commit();
    load_stage = load_stage + 1 == S::kStages ? 0 : load_stage + 1;
  };
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; ++i) load_next();
#pragma unroll 1
  for (int i = 0; i < own; ++i) {
    cp_async_wait<S::kStages - 2>();
    __syncwarp();
    const uint32_t tile = ring + stage * 2 * S::kHalf;
    const uint32_t mask = sh.mask[warp][stage];
    load_next();
    if (mask != 0 || kWeights) {
      const int64_t t = static_cast<int64_t>(index) * p.item_tiles + rank + i * ranks;
      sums.template add<kWeights>(
          p, tile, mask,
          kWeights ? p.scores + (t * kTile + warp * kWarpTile) * p.score_rows : nullptr, [] {});
    }
    __syncwarp();  // this stage is refilled by the next load_next
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
  }

  const int kv = item / p.head_tiles, h0 = item % p.head_tiles * S::kRows;
  const int rows = min(p.group - h0, S::kRows);
  T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.hq + kv * p.group + h0) * c.dim;
  if (tiles == 0) {  // so for every block of the cluster
    for (int i = rank * kThreads + tid; i < rows * c.dim; i += ranks * kThreads) {
      out[i] = from_f32<T>(0.0f);
    }
    return;
  }
  // every block takes a share of the output and the weights of its own tiles; one without tiles has
  // sums of 0 and a maximum of -inf
  sums.join(sh.joined, sh.ml);
  const cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const int pairs = c.dim / 2;
  const int first = rank * kThreads + tid;
  float2 v[kMaxCluster];
  auto read = [&](int i) {
    const int row = i / pairs, d = i % pairs * 2;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      v[r] = r < ranks && i < rows * pairs
                 ? *reinterpret_cast<const float2*>(&cluster.map_shared_rank(&sh, r)->joined[row][d])
                 : make_float2(0.0f, 0.0f);
    }
  };
  read(first);
  if (tid < rows) {
    float2 ml[kMaxCluster];
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      ml[r] = r < ranks ? cluster.map_shared_rank(&sh, r)->ml[0][tid] : make_float2(-INFINITY, 0.0f);
      m = fmaxf(m, ml[r].x);
    }
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      // a part in which nothing counted is not scaled: its sums are 0
      ml[r].x = ml[r].x == -INFINITY ? 1.0f : exp2_fast(ml[r].x - m);
      l = fmaf(ml[r].y, ml[r].x, l);
    }
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) sh.share[tid][r] = ml[r].x / divisor(make_float2(m, l));
    sh.row_lse[tid] = m + log2f(l);
  }
  __syncthreads();
  for (int i = first; i < rows * pairs; i += ranks * kThreads) {
    if (i != first) read(i);
    const int row = i / pairs, d = i % pairs * 2;
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int r = 0; r < kMaxCluster; ++r) {
      if (r < ranks) {
        sum.x = fmaf(v[r].x, sh.share[row][r], sum.x);
        sum.y = fmaf(v[r].y, sh.share[row][r], sum.y);
      }
    }
    *reinterpret_cast<uint32_t*>(out + row * c.dim + d) = pack2<T>(sum.x, sum.y);
  }
  // the others read this block's part up to here; the barrier's second half is at the end
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if constexpr (kWeights) {
    for (int i = 0; i < own; ++i) {
      const int tile = rank + i * ranks;
      add_weights<kThreads>(p, b, kv, 0, rows, index * p.item_tiles + tile, tile,
                            min(kTile, n - tile * kTile), fresh, sh.row_lse, [] {});
    }
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// ---- Joining -------------------------------------------------------------------------------------
//
// A warp a (sequence, query head), or a block where items have many parts, joins what several blocks
// of the attention kernel hold of it: a lane takes four dimensions of part after part, a block's warps
// take the parts in turn and their sums are added in order. It also zeroes the output of empty
// sequences. Blocks behind those add the weights: an even share of the tiles each, a thread two
// positions at a time.
constexpr int kJoinThreads = 128;
constexpr int kJoinWarps = kJoinThreads / kWarp;
// Blocks an SM that also adds weights, in one wave: their chain of loads is the time, so all start at
// once. 24 sequences of up to 4096: 55.0 us with 6 (80 registers), 56 with 5; 57.7 with 8 and 62.5 with
// 10, which spill; 64.3 with four parts at a time and no bound (120 registers, three waves).
constexpr int kJoinCtas = 6;

// Reads of the attention kernel's workspace
struct Parts {
  const Plan& p;
  Split split;
  int begin, o0, count;  // an item's first tile, its first block and the number of its blocks
  __device__ __forceinline__ Parts(const Plan& plan, int total, int first, int tiles)
      : p(plan), split(total, plan.blocks), begin(first), o0(split.owner(first)),
        count(split.owner(first + tiles - 1) - o0 + 1) {}
  __device__ __forceinline__ int64_t slot(int i) const {
    return 2 * (o0 + i) + (split.start(o0 + i) >= begin ? 0 : 1);
  }
  // Maximum and sum of a row over all parts, by a whole warp.
  __device__ __forceinline__ float2 row(int r, int lane) const {
    float m = -INFINITY;
    for (int i = lane; i < count; i += kWarp) m = fmaxf(m, p.part_ml[slot(i) * p.rows + r].x);
#pragma unroll
    for (int off = kWarp / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    float l = 0.0f;
    for (int i = lane; i < count; i += kWarp) {
      const float2 v = p.part_ml[slot(i) * p.rows + r];
      l = fmaf(v.y, factor(v.x, m), l);
    }
    return make_float2(m, warp_sum(l));
  }
  // Of a part in which nothing counted nothing is scaled (its sums are 0).
  static __device__ __forceinline__ float factor(float m, float top) {
    return m == -INFINITY ? 1.0f : exp2_fast(m - top);
  }
};

template <class T, int kAtOnce>
__device__ __forceinline__ void join_head(const Plan& p) {
  __shared__ alignas(16) float sums[kJoinWarps][kMaxDim];
  const PagedAttentionArgs& a = p.a;
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp, dim = a.cache.dim;
  const int index = p.join_warps == 1 ? blockIdx.x * kJoinWarps + warp : blockIdx.x;
  const int sub = p.join_warps == 1 ? 0 : warp;
  if (index >= a.batch * a.hq) return;
  const int b = index / a.hq, head = index % a.hq;
  const int kv = head / p.group, h = head % p.group;
  const int item = kv * p.head_tiles + h / p.rows, row = h % p.rows;
  const int first = p.first_tile[b], tiles = (p.first_tile[b + 1] - first) / p.items;
  T* out = static_cast<T*>(a.out) + static_cast<int64_t>(index) * dim;
  if (tiles == 0) {
    if (sub == 0) {
      for (int i = lane; i < dim; i += kWarp) out[i] = from_f32<T>(0.0f);
    }
    return;
  }
  const Parts parts(p, p.first_tile[a.batch], first + item * tiles, tiles);
  if (parts.count == 1) return;
  float2 ml = make_float2(0.0f, 0.0f);
  float4 v[2] = {};
  for (int i0 = sub; i0 < parts.count; i0 += kAtOnce * p.join_warps) {
    float m[kAtOnce];
    float4 o[kAtOnce][2];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int i = i0 + k * p.join_warps;
      if (i < parts.count) {
        const int64_t at = parts.slot(i) * p.rows + row;
        m[k] = p.part_ml[at].x;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = (j * kWarp + lane) * 4;
          if (d < dim) o[k][j] = *reinterpret_cast<const float4*>(p.part_o + at * dim + d);
        }
      }
    }
    if (i0 == sub) ml = parts.row(row, lane);  // while the first parts are on their way
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      if (i0 + k * p.join_warps >= parts.count) continue;
      const float f = Parts::factor(m[k], ml.x);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if ((j * kWarp + lane) * 4 < dim) {
          v[j].x = fmaf(o[k][j].x, f, v[j].x);
          v[j].y = fmaf(o[k][j].y, f, v[j].y);
          v[j].z = fmaf(o[k][j].z, f, v[j].z);
          v[j].w = fmaf(o[k][j].w, f, v[j].w);
        }
      }
    }
  }
  if (p.join_warps > 1) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int d = (j * kWarp + lane) * 4;
      if (d < dim) *reinterpret_cast<float4*>(&sums[warp][d]) = v[j];
    }
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int d = (j * kWarp + lane) * 4;
      if (d < dim) {
#pragma unroll
        for (int w = 1; w < kJoinWarps; ++w) {
          const float4 o = *reinterpret_cast<const float4*>(&sums[w][d]);
          v[j].x += o.x;
          v[j].y += o.y;
          v[j].z += o.z;
          v[j].w += o.w;
        }
      }
    }
  }
  const float l = divisor(ml);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int d = (j * kWarp + lane) * 4;
    if (d < dim) {
      *reinterpret_cast<uint2*>(out + d) =
          make_uint2(pack2<T>(v[j].x / l, v[j].y / l), pack2<T>(v[j].z / l, v[j].w / l));
    }
  }
}

__device__ __forceinline__ void join_weights(const Plan& p, int block, int blocks) {
  __shared__ float row_lse[16];
  __shared__ int start;
  const PagedAttentionArgs& a = p.a;
  const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
  // tiles of (sequence, KV head), the items of a KV head together
  const int total = p.first_tile[a.batch];
  const Split mine(total / p.head_tiles, blocks);
  int t = mine.start(block);
  const int t1 = mine.start(block + 1);
  if (t >= t1) return;
  for (int b = tid; b < a.batch; b += kJoinThreads) {
    if (p.first_tile[b] / p.head_tiles <= t && t < p.first_tile[b + 1] / p.head_tiles) start = b;
  }
  __syncthreads();
  int b = start;
  while (t < t1) {
    while (p.first_tile[b + 1] / p.head_tiles <= t) ++b;
    const int given = a.lens[b], n = clamped(p, given), fresh = new_position(p, given);
    const int tiles = (n + p.tile - 1) / p.tile;
    const int first = p.first_tile[b] / p.head_tiles;
    const int kv = (t - first) / tiles, tile0 = (t - first) % tiles;
    const int count = min(tiles - tile0, t1 - t);
    for (int ht = 0; ht < p.head_tiles; ++ht) {
      const int begin = p.first_tile[b] + (kv * p.head_tiles + ht) * tiles;
      const int rows = min(p.group - ht * p.rows, p.rows);
      const Parts parts(p, total, begin, tiles);
      add_weights<kJoinThreads>(
          p, b, kv, ht, rows, begin + tile0, tile0, min(count * p.tile, n - tile0 * p.tile), fresh, row_lse,
          [&] {
            if (parts.count == 1) {
              if (tid < rows) {
                row_lse[tid] = p.lse[static_cast<int64_t>(b) * a.hq + kv * p.group + ht * p.rows + tid];
              }
            } else {
              for (int r = warp; r < rows; r += kJoinWarps) {
                const float2 ml = parts.row(r, lane);
                if (lane == 0) row_lse[r] = ml.x + log2f(ml.y);
              }
            }
            __syncthreads();
          });
      __syncthreads();  // row_lse is rewritten
    }
    t += count;
  }
}

template <class T, bool kWeights>
__global__ void __launch_bounds__(kJoinThreads, kWeights ? kJoinCtas : 1)
paged_join_kernel(const __grid_constant__ Plan p) {
  wait_then_release();
  if (static_cast<int>(blockIdx.x) < p.join_blocks) {
    join_head<T, kWeights ? 2 : 4>(p);
  } else if constexpr (kWeights) {
    join_weights(p, blockIdx.x - p.join_blocks, gridDim.x - p.join_blocks);
  }
}

// ---- Host ----------------------------------------------------------------------------------------

// Calls f with the Shape of a call as template arguments <DP, NT>.
template <class F>
auto with_shape(int dim, int group, F f) {
  const bool wide = group > 8;
  switch (round_dim(dim)) {
    case 64: return wide ? f.template operator()<64, 2>() : f.template operator()<64, 1>();
    case 128: return wide ? f.template operator()<128, 2>() : f.template operator()<128, 1>();
    default: return f.template operator()<256, 1>();  // 16 heads' sums do not fit the registers
  }
}

int64_t aligned_up(int64_t n) { return (n + 255) / 256 * 256; }

// Clusters of `size` blocks of the kernel for small calls that the current device runs at once. A
// cluster's blocks share a group of SMs, so that is less than SMs / size: on B200 74, 33 and 15 of 2, 4
// and 8 blocks.
template <int DP, int NT>
int clusters_at_once(int size) {
  static std::atomic<int> known[64][kMaxCluster + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return sm_count() / size;
  std::atomic<int>& count = known[dev & 63][size];
  int n = count.load(std::memory_order_relaxed);
  if (n > 0) return n;
  // the type and the weights do not matter: shared memory leaves room for one block an SM
  const auto kernel = paged_attention_small_kernel<half, DP, NT, false>;
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(Shape<DP, NT, true>::kThreads);
  cfg.dynamicSmemBytes = sizeof(SmallSmem<DP, NT>);
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = size;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(SmallSmem<DP, NT>)) !=
          cudaSuccess ||
      cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
    cudaGetLastError();  // not the next launch's
    return sm_count() / size;
  }
  count.store(n, std::memory_order_relaxed);
  return n;
}

// Fills the plan's sizes and, with a workspace, its pointers; returns the workspace's bytes, or -1
// where the sizes are out of range.
int64_t make_plan(const PagedAttentionArgs& a, Plan* p) {
  p->a = a;
  p->group = a.hq / a.cache.hkv;
  int ctas = 1, small_tile = 1;
  int (*at_once)(int) = nullptr;
  with_shape(a.cache.dim, p->group, [&]<int DP, int NT>() {
    p->rows = Shape<DP, NT, false>::kRows;
    p->tile = Shape<DP, NT, false>::kTile;
    ctas = kCtas<DP, NT>;
    small_tile = Shape<DP, NT, true>::kTile;
    at_once = clusters_at_once<DP, NT>;
  });
  p->head_tiles = (p->group + p->rows - 1) / p->rows;
  const int64_t items = static_cast<int64_t>(a.cache.hkv) * p->head_tiles;
  const int64_t len = static_cast<int64_t>(a.max_blocks) * a.cache.block_size;
  // A small call: clusters as large as SMs allow at one block each and as every block has a tile, if that
  // leaves no block more than kSmallTiles. Clusters that do not all run at once, and so take a second
  // wave, only where the smaller ones leave a block more than half of that (16 sequences, one KV head of
  // 128 dims: of up to 2000 positions 14.5 us in clusters of 8, 12.5 in clusters of 4; of up to 4000 16.6
  // and 18.8). The weights of a KV head need all its query heads in one item.
  const int64_t all_items = a.batch * items, small_tiles = (len + small_tile - 1) / small_tile;
  p->cluster = 0;
  if (all_items > 0 && all_items <= sm_count() && small_tiles > 0 &&
      (!a.cache.weights || p->head_tiles == 1)) {
    int cluster = 1;
    while (cluster < kMaxCluster && all_items * cluster * 2 <= sm_count() && cluster < small_tiles &&
           (all_items <= at_once(cluster * 2) || small_tiles > kSmallTiles / 2 * cluster)) {
      cluster *= 2;
    }
    if (small_tiles <= static_cast<int64_t>(kSmallTiles) * cluster) {
      p->cluster = cluster;
      p->tile = small_tile;
    }
  }
  const int64_t tiles = all_items * ((len + p->tile - 1) / p->tile);
  if (len > INT32_MAX - p->tile || tiles > INT32_MAX / 2 ||
      static_cast<int64_t>(a.batch) * a.hq > INT32_MAX / 4) {
    return -1;
  }
  p->items = static_cast<int>(items);
  p->max_len = static_cast<int>(len);
  p->item_tiles = static_cast<int>((len + p->tile - 1) / p->tile);
  p->score_rows = (std::min(p->group, p->rows) + 1) / 2 * 2;
  p->page = Divider(static_cast<uint32_t>(a.cache.block_size));
  const int64_t resident = static_cast<int64_t>(sm_count()) * ctas;
  p->blocks = static_cast<int>(std::max<int64_t>(1, std::min(resident, tiles)));
  // a block a head where an item has more than this many parts (1 x 131072 positions, 64 heads of 55
  // parts; with few parts a warp leaves room for four times the heads)
  constexpr int kManyParts = 6;
  p->join_warps = p->blocks > kManyParts * a.batch * items ? kJoinWarps : 1;
  p->join_blocks = (a.batch * a.hq * p->join_warps + kJoinWarps - 1) / kJoinWarps;
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += aligned_up(bytes);
    return static_cast<unsigned char*>(a.workspace) + here;
  };
  if (!p->cluster) {
    p->part_o = reinterpret_cast<float*>(take(2LL * p->blocks * p->rows * a.cache.dim * 4));
    p->part_ml = reinterpret_cast<float2*>(take(2LL * p->blocks * p->rows * 8));
    p->first_tile = reinterpret_cast<int*>(take((a.batch + 1LL) * 4));
    if (a.cache.weights) {
      p->lse = reinterpret_cast<float*>(take(static_cast<int64_t>(a.batch) * a.hq * 4));
    }
  }
  if (a.cache.weights) {
    p->scores = reinterpret_cast<float*>(take(tiles * p->tile * p->score_rows * 4));
  }
  return at;
}

template <class T, int DP, int NT, bool kWeights>
cudaError_t launch(const Plan& p, cudaStream_t stream) {
  static std::once_flag once[64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  std::call_once(once[dev & 63], [&] {
    err = cudaFuncSetAttribute(paged_attention_kernel<T, DP, NT, kWeights>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem<DP, NT>));
    if (err != cudaSuccess) return;
    err = cudaFuncSetAttribute(paged_attention_small_kernel<T, DP, NT, kWeights>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize,
                               sizeof(SmallSmem<DP, NT>));
  });
  if (err != cudaSuccess) return err;
  if (p.cluster) {
    return launch_serialised(paged_attention_small_kernel<T, DP, NT, kWeights>,
                             dim3(p.a.batch * p.items * p.cluster),
                             dim3(Shape<DP, NT, true>::kThreads), sizeof(SmallSmem<DP, NT>), stream,
                             p.cluster, p);
  }
  err = launch_serialised(paged_attention_kernel<T, DP, NT, kWeights>, dim3(p.blocks),
                          dim3(Shape<DP, NT, false>::kThreads), sizeof(Smem<DP, NT>), stream, 1, p);
  if (err != cudaSuccess) return err;
  const int blocks = kWeights ? std::max(kJoinCtas * sm_count(), p.join_blocks + sm_count())
                              : p.join_blocks;
  return launch_serialised(paged_join_kernel<T, kWeights>, dim3(blocks), dim3(kJoinThreads), 0, stream,
                           1, p);
}

}  // namespace

int64_t paged_attention_workspace_bytes(const PagedAttentionArgs& a) {
  Plan p{};
  return make_plan(a, &p);
}

cudaError_t launch_paged_attention(const PagedAttentionArgs& a, int dtype, cudaStream_t stream) {
  Plan p{};
  make_plan(a, &p);
  p.status = device_status_word();
  if (!p.status) return cudaErrorInitializationError;
  return with_shape(a.cache.dim, p.group, [&]<int DP, int NT>() {
    if (dtype == kWeightF16) {
      return a.cache.weights ? launch<half, DP, NT, true>(p, stream)
                             : launch<half, DP, NT, false>(p, stream);
    }
    return a.cache.weights ? launch<__nv_bfloat16, DP, NT, true>(p, stream)
                           : launch<__nv_bfloat16, DP, NT, false>(p, stream);
  });
}

}  // namespace i4
