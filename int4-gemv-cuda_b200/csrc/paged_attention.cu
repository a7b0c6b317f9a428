// Attention of one new token a sequence over a paged cache of keys and values:
//   s_hj = scale q_h . k_j,  p_h = softmax_j(s_h),  o_h = sum_j p_hj v_j,
// query head h reading KV head h / (hq / hkv). Optionally the call brings the new token's key and
// value (written to the last position's slot and used from the call's tensors), and adds every
// position's attention weight, summed over the query heads of its KV head, to a buffer that
// eviction goes by.
//
// Bound by HBM: the cache is read once, 4 hq / hkv operations an element.
//
// Work: an item is (sequence, KV head, block of 16 query heads), cut into tiles of 64 positions.
// All tiles in order are split evenly over the blocks of the grid whatever the lengths are, so a
// block works through the end of one item, whole items, and the beginning of another; an item that
// several blocks share is joined by a second kernel from partial sums in the workspace, in block
// order (the same result every time, and no counters that a call would have to find cleared).
//
// A warp takes 16 positions of a tile and needs no other warp until its segment of an item ends:
// it has its own ring of K and V tiles in shared memory, filled by cp.async (a row's page is looked
// up while older tiles are in flight), its own running maximum and sum, and its own fp32
// accumulators. S = Q K^T and O = P V are warp MMAs with the 16 query heads as rows (a KV head
// with fewer leaves rows unused: the tensor pipe has several times the needed rate). P is given to
// the MMA as a sum of two 16-bit numbers, so its rounding does not show in the result. Positions
// behind the end are zero-filled in shared memory and masked, so nothing there reaches a sum.
#include <algorithm>
#include <mutex>

#include "decode.cuh"
#include "kernels.h"

namespace i4 {
namespace {

constexpr int kRows = 16;       // query heads of an item
constexpr int kWarpTile = 16;   // positions a warp takes of a tile
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * kWarp;
constexpr int kTile = kWarps * kWarpTile;

// Shapes by the head dimension rounded up: ring stages (their bytes in flight an SM), blocks an SM.
constexpr int stages_of(int dp) { return dp == 256 ? 2 : 3; }
constexpr int ctas_of(int dp) { return dp == 64 ? 3 : dp == 128 ? 2 : 1; }
constexpr int round_dim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

struct Plan {
  PagedAttentionArgs a;
  int group;       // query heads of a KV head
  int head_tiles;  // blocks of 16 query heads of a KV head
  int items;       // items of a sequence: hkv * head_tiles
  int blocks;      // blocks of the attention kernel
  int max_len;     // positions the table has room for
  float* part_o;   // [2 blocks][16][dim]: the segments of items that a block shares
  float2* part_ml;  // [2 blocks][16]: their maximum (log2) and sum
  float* lse;      // [batch][hq]: log2 of the sum, for items of one block (weights only)
  float* scores;   // [tiles][min(group, 16)][64]: log2 scores (weights only)
  int* first_tile;  // [batch + 1]: tiles before each sequence
  int* status;
};

__device__ __forceinline__ int length_of(const Plan& p, int b) {
  const int n = p.a.lens[b];
  if (n < 0) return 0;
  return n > p.max_len ? p.max_len : n;
}
__device__ __forceinline__ int tiles_of(int n) { return (n + kTile - 1) / kTile; }

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

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

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

// A position in the order of all tiles: sequence, item of the sequence, tile of the item.
struct Walker {
  int b, item, tile, tiles, n;

  __device__ __forceinline__ void enter(const Plan& p) {  // to the next sequence with positions
    while (b < p.a.batch) {
      n = length_of(p, b);
      if (n > 0) break;
      ++b;
    }
    tiles = tiles_of(n);
  }
  __device__ __forceinline__ void next(const Plan& p) {
    if (++tile < tiles) return;
    tile = 0;
    if (++item < p.items) return;
    item = 0;
    ++b;
    enter(p);
  }
};

// Element size is 2 for both types: T only picks the MMA and the conversions.
template <class T, int DP>
struct Warp {
  static constexpr int kRowBytes = DP * 2;
  static constexpr int kTileBytes = kWarpTile * kRowBytes;  // K or V of a warp tile
  static constexpr int kStages = stages_of(DP);
  static constexpr int kChunks = DP / 8;
  // 16-byte chunks of a row are stored at their index XOR the row's, so that the eight rows of an
  // ldmatrix fall into different banks.
  static __device__ __forceinline__ uint32_t at(int row, int chunk) {
    return row * kRowBytes + ((chunk ^ (row & 7)) << 4);
  }
};

template <int DP>
struct Smem {
  static constexpr int kRing = kWarps * stages_of(DP) * 2 * kWarpTile * DP * 2;
  alignas(1024) unsigned char ring[kRing];
  const void* rows[kWarps][kWarpTile][2];  // K and V row of each position of the tile being loaded
  uint32_t mask[kWarps][stages_of(DP)];    // positions that count
  float joined[kRows][DP];
  float2 ml[kWarps][kRows];
  int scan[kWarps];
  int start[3];  // sequence of the block's first tile, tiles before it, tiles in all
};

template <class T, int DP, bool kWeights>
__global__ void __launch_bounds__(kThreads, ctas_of(DP)) paged_attention_kernel(const Plan p) {
  using W = Warp<T, DP>;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  Smem<DP>& sh = *reinterpret_cast<Smem<DP>*>(smem_raw);
  wait_then_release();
  const PagedAttentionArgs& a = p.a;
  const PagedCache& c = a.cache;
  const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;

  // tiles in all
  int total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kThreads) {
    int t = b0 + tid < a.batch ? tiles_of(length_of(p, b0 + tid)) * p.items : 0;
#pragma unroll
    for (int off = 1; off < kWarp; off *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, t, off);
      if (lane >= off) t += v;
    }
    if (lane == kWarp - 1) sh.scan[warp] = t;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) t += sh.scan[w];
    }
    if (blockIdx.x == 0) {
      if (b0 + tid < a.batch) p.first_tile[b0 + tid + 1] = total + t;
      if (b0 + tid == 0) p.first_tile[0] = 0;
    }
    for (int w = 0; w < kWarps; ++w) total += sh.scan[w];
    __syncthreads();
  }
  if (blockIdx.x == 0) {
    for (int b = tid; b < a.batch; b += kThreads) {
      if (a.lens[b] != length_of(p, b)) atomicExch(p.status, kStatusBadPage);
    }
  }
  const Split split(total, p.blocks);
  const int t0 = split.start(blockIdx.x), t1 = split.start(blockIdx.x + 1);
  if (t0 >= t1) return;

  // the sequence of tile t0
  for (int b0 = 0, before = 0; b0 < a.batch; b0 += kThreads) {
    const int own = b0 + tid < a.batch ? tiles_of(length_of(p, b0 + tid)) * p.items : 0;
    int t = own;
#pragma unroll
    for (int off = 1; off < kWarp; off *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, t, off);
      if (lane >= off) t += v;
    }
    if (lane == kWarp - 1) sh.scan[warp] = t;
    __syncthreads();
    int sum = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) t += sh.scan[w];
      sum += sh.scan[w];
    }
    t += before;
    if (t - own <= t0 && t0 < t) {
      sh.start[0] = b0 + tid;
      sh.start[1] = t - own;
    }
    before += sum;
    __syncthreads();
  }
  Walker load;
  load.b = sh.start[0];
  load.enter(p);
  load.item = (t0 - sh.start[1]) / load.tiles;
  load.tile = (t0 - sh.start[1]) % load.tiles;
  Walker now = load;

  // ---- loading
  const uint32_t ring = smem_addr(sh.ring) + warp * W::kStages * 2 * W::kTileBytes;
  int load_tile = t0, load_stage = 0;
  auto load_next = [&] {
    if (load_tile < t1) {
      const int kv = load.item / p.head_tiles;
      const int last = load.n - 1;
      bool valid = false, append = false;
      if (lane < kWarpTile) {
        const int pos = load.tile * kTile + warp * kWarpTile + lane;
        const void* k = c.k;
        const void* v = c.v;
        if (pos < load.n) {
          append = a.k_new != nullptr && pos == last;
          const int page = a.table[static_cast<int64_t>(load.b) * a.max_blocks + pos / c.block_size];
          if (static_cast<unsigned>(page) < static_cast<unsigned>(c.num_blocks)) {
            const int off = pos % c.block_size;
            valid = true;
            k = static_cast<const T*>(c.k) + page * c.k_block + off * c.k_token + kv * c.k_head;
            v = static_cast<const T*>(c.v) + page * c.v_block + off * c.v_token + kv * c.v_head;
          } else {
            atomicExch(p.status, kStatusBadPage);
          }
        }
        sh.rows[warp][lane][0] = k;
        sh.rows[warp][lane][1] = v;
      }
      const uint32_t mask = __ballot_sync(0xffffffffu, valid);
      const uint32_t fresh = __ballot_sync(0xffffffffu, valid && append);
      if (lane == 0) sh.mask[warp][load_stage] = mask;
      __syncwarp();
      const int64_t new_row = (static_cast<int64_t>(load.b) * c.hkv + kv) * c.dim;
      if (fresh) {
        // the new token's row: to its slot (once for a KV head), and read from the call's tensors
        const int row = __ffs(fresh) - 1;
        if (load.item % p.head_tiles == 0) {
          uint4* k = static_cast<uint4*>(const_cast<void*>(sh.rows[warp][row][0]));
          uint4* v = static_cast<uint4*>(const_cast<void*>(sh.rows[warp][row][1]));
          for (int i = lane; i < c.dim / 8; i += kWarp) {
            k[i] = reinterpret_cast<const uint4*>(static_cast<const T*>(a.k_new) + new_row)[i];
            v[i] = reinterpret_cast<const uint4*>(static_cast<const T*>(a.v_new) + new_row)[i];
          }
        }
        __syncwarp();
        if (lane == row) {
          sh.rows[warp][row][0] = static_cast<const T*>(a.k_new) + new_row;
          sh.rows[warp][row][1] = static_cast<const T*>(a.v_new) + new_row;
        }
        __syncwarp();
      }
      const uint32_t dst = ring + load_stage * 2 * W::kTileBytes;
#pragma unroll
      for (int i = 0; i < kWarpTile * W::kChunks / kWarp; ++i) {
        const int idx = i * kWarp + lane, row = idx / W::kChunks, chunk = idx % W::kChunks;
        const bool there = (mask >> row & 1) && chunk * 8 < c.dim;
        const T* k = static_cast<const T*>(sh.rows[warp][row][0]);
        const T* v = static_cast<const T*>(sh.rows[warp][row][1]);
        cp_async_16(dst + W::at(row, chunk), there ? k + chunk * 8 : k, there);
        cp_async_16(dst + W::kTileBytes + W::at(row, chunk), there ? v + chunk * 8 : v, there);
      }
      __syncwarp();  // sh.rows is rewritten by the next load
      load.next(p);
      ++load_tile;
    }
    cp_async_commit();
    load_stage = load_stage + 1 == W::kStages ? 0 : load_stage + 1;
  };
#pragma unroll
  for (int s = 0; s < W::kStages - 1; ++s) load_next();

  // ---- computing
  const int g = lane / 4, t2 = lane % 4 * 2;
  constexpr bool kHoldQ = DP <= 128;
  uint32_t qf[kHoldQ ? DP / 16 : 1][4];
  float o[DP / 8][4];
  float m[2], l[2];
  auto q_frag = [&](int k16, uint32_t (&f)[4]) {
    const int kv = now.item / p.head_tiles;
    const int h0 = now.item % p.head_tiles * kRows;
    const T* q = static_cast<const T*>(a.q) +
                 (static_cast<int64_t>(now.b) * a.hq + kv * p.group + h0) * c.dim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = g + (i & 1) * 8, col = k16 * 16 + t2 + (i >> 1) * 8;
      f[i] = h0 + row < p.group && col < c.dim
                 ? *reinterpret_cast<const uint32_t*>(q + static_cast<int64_t>(row) * c.dim + col)
                 : 0u;
    }
  };
  auto begin = [&] {
    if constexpr (kHoldQ) {
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) q_frag(k, qf[k]);
    }
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
    }
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.0f;
  };
  begin();
  int stage = 0, segment = t0;  // first tile of the current segment
  for (int t = t0; t < t1; ++t) {
    cp_async_wait<W::kStages - 2>();
    __syncwarp();
    load_next();
    const uint32_t ks = ring + stage * 2 * W::kTileBytes, vs = ks + W::kTileBytes;
    const uint32_t mask = sh.mask[warp][stage];

    // S: rows g and g + 8, positions t2, t2 + 1 of both halves of the 16
    float s[2][4] = {};
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      if (k * 16 < c.dim) {
        uint32_t b[4];
        // matrices: positions 0-7 / k 0-7, positions 0-7 / k 8-15, positions 8-15 / ...
        const int row = (lane & 7) + (lane >> 4) * 8, chunk = 2 * k + (lane >> 3 & 1);
        ldmatrix_x4(b, ks + W::at(row, chunk));
        uint32_t f[4];
        if constexpr (kHoldQ) {
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = qf[k][i];
        } else {
          q_frag(k, f);
        }
        mma<T>(s[0], f, b[0], b[1]);
        mma<T>(s[1], f, b[2], b[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int pos = i * 8 + t2 + (j & 1);
        s[i][j] = mask >> pos & 1 ? s[i][j] * a.scale_log2 : -INFINITY;
      }
    }
    if constexpr (kWeights) {
      const int rows = min(p.group, kRows);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (g + r * 8 < rows) {
            float* to = p.scores + (static_cast<int64_t>(t) * rows + g + r * 8) * kTile +
                        warp * kWarpTile + i * 8 + t2;
            *reinterpret_cast<float2*>(to) = make_float2(s[i][2 * r], s[i][2 * r + 1]);
          }
        }
      }
    }
    float top[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      top[r] = fmaxf(top[r], m[r]);
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float f = m[r] == -INFINITY ? 0.0f : exp2_fast(m[r] - top[r]);
        m[r] = top[r];
        l[r] *= f;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
          o[i][2 * r] *= f;
          o[i][2 * r + 1] *= f;
        }
      }
    }
    const float ref[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float p0 = exp2_fast(s[i][2 * r] - ref[r]), p1 = exp2_fast(s[i][2 * r + 1] - ref[r]);
        l[r] += p0 + p1;
        hi[2 * i + r] = pack2<T>(p0, p1);
        const float2 back = unpack2<T>(hi[2 * i + r]);
        lo[2 * i + r] = pack2<T>(p0 - back.x, p1 - back.y);
      }
    }
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) {
      if (d * 16 < c.dim) {
        uint32_t b[4];
        // matrices: positions 0-7 / dims 0-7, positions 8-15 / dims 0-7, then dims 8-15
        const int row = (lane & 7) + (lane >> 3 & 1) * 8, chunk = 2 * d + (lane >> 4);
        ldmatrix_x4_trans(b, vs + W::at(row, chunk));
        mma<T>(o[2 * d], hi, b[0], b[1]);
        mma<T>(o[2 * d + 1], hi, b[2], b[3]);
        mma<T>(o[2 * d], lo, b[0], b[1]);
        mma<T>(o[2 * d + 1], lo, b[2], b[3]);
      }
    }
    __syncwarp();  // this stage is refilled by the next load_next
    stage = stage + 1 == W::kStages ? 0 : stage + 1;

    // ---- the end of a segment: join the warps
    const bool item_ends = now.tile + 1 == now.tiles;
    if (!item_ends && t + 1 < t1) {
      ++now.tile;
      continue;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (lane % 4 == 0) sh.ml[warp][g + r * 8] = make_float2(m[r], l[r]);
    }
    __syncthreads();
    float all_m[2], all_l[2], f[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      all_m[r] = -INFINITY;
      all_l[r] = 0.0f;
      for (int w = 0; w < kWarps; ++w) all_m[r] = fmaxf(all_m[r], sh.ml[w][g + r * 8].x);
      for (int w = 0; w < kWarps; ++w) {
        const float2 v = sh.ml[w][g + r * 8];
        all_l[r] += v.x == -INFINITY ? v.y : v.y * exp2_fast(v.x - all_m[r]);
      }
      f[r] = m[r] == -INFINITY ? 1.0f : exp2_fast(m[r] - all_m[r]);
    }
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) {
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float2* to = reinterpret_cast<float2*>(&sh.joined[g + r * 8][i * 8 + t2]);
            float2 v = make_float2(o[i][2 * r] * f[r], o[i][2 * r + 1] * f[r]);
            if (w > 0) {
              const float2 was = *to;
              v.x += was.x;
              v.y += was.y;
            }
            *to = v;
          }
        }
      }
      __syncthreads();
    }
    const int kv = now.item / p.head_tiles, h0 = now.item % p.head_tiles * kRows;
    const int rows = min(p.group - h0, kRows);
    const int head = kv * p.group + h0;
    const bool whole = item_ends && t - segment + 1 == now.tiles;
    if (lane % 4 == 0 && warp == 0) {  // rows g and g + 8 of this warp are the block's
#pragma unroll
      for (int r = 0; r < 2; ++r) sh.ml[0][g + r * 8] = make_float2(all_m[r], all_l[r]);
    }
    __syncthreads();
    if (whole) {
      T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(now.b) * a.hq + head) * c.dim;
      for (int i = tid; i < rows * (c.dim / 2); i += kThreads) {
        const int row = i / (c.dim / 2), d = i % (c.dim / 2) * 2;
        const float inv = 1.0f / sh.ml[0][row].y;
        *reinterpret_cast<uint32_t*>(out + static_cast<int64_t>(row) * c.dim + d) =
            pack2<T>(sh.joined[row][d] * inv, sh.joined[row][d + 1] * inv);
      }
      if (kWeights && tid < rows) {
        p.lse[static_cast<int64_t>(now.b) * a.hq + head + tid] =
            sh.ml[0][tid].x + log2f(sh.ml[0][tid].y);
      }
    } else {
      const int slot = 2 * blockIdx.x + (segment == t0 ? 0 : 1);
      float* to = p.part_o + static_cast<int64_t>(slot) * kRows * c.dim;
      for (int i = tid; i < rows * c.dim; i += kThreads) to[i] = sh.joined[i / c.dim][i % c.dim];
      if (tid < rows) p.part_ml[slot * kRows + tid] = sh.ml[0][tid];
    }
    __syncthreads();  // joined and ml are written again by the next segment
    if (t + 1 < t1) {
      now.next(p);
      segment = t + 1;
      begin();
    }
  }
}

// Joins the items that several blocks share, zeroes the output of empty sequences, and (blocks
// behind those of the items) adds the weights of the tiles.
constexpr int kJoinThreads = 128;

template <class T, bool kWeights>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const Plan p) {
  extern __shared__ float factor[];  // [16][blocks of an item]
  __shared__ float row_lse[kRows];
  wait_then_release();
  const PagedAttentionArgs& a = p.a;
  const PagedCache& c = a.cache;
  const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
  const int total = p.first_tile[a.batch];
  const Split split(total, p.blocks);

  // the part of item (first tile `begin`) that block `o` holds
  auto slot_of = [&](int o, int begin) { return 2 * o + (split.start(o) >= begin ? 0 : 1); };
  // log2 of the item's sum for its rows, to row_lse, from blocks o0..o1; with kFactors also each
  // part's share of the result
  auto sums = [&](int begin, int o0, int o1, int rows, bool factors) {
    const int parts = o1 - o0 + 1;
    for (int row = warp; row < rows; row += kJoinThreads / kWarp) {
      float m = -INFINITY;
      for (int i = lane; i < parts; i += kWarp) {
        m = fmaxf(m, p.part_ml[slot_of(o0 + i, begin) * kRows + row].x);
      }
#pragma unroll
      for (int off = kWarp / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      float l = 0.0f;
      for (int i = lane; i < parts; i += kWarp) {
        const float2 v = p.part_ml[slot_of(o0 + i, begin) * kRows + row];
        const float f = v.x == -INFINITY ? 1.0f : exp2_fast(v.x - m);
        if (factors) factor[row * parts + i] = f;
        l = fmaf(v.y, f, l);
      }
      l = warp_sum(l);
      if (lane == 0) row_lse[row] = factors ? l : m + log2f(l);
    }
    __syncthreads();
  };

  const int all_items = a.batch * p.items;
  if (blockIdx.x < all_items) {
    const int b = blockIdx.x / p.items, item = blockIdx.x % p.items;
    const int kv = item / p.head_tiles, h0 = item % p.head_tiles * kRows;
    const int rows = min(p.group - h0, kRows);
    const int tiles = (p.first_tile[b + 1] - p.first_tile[b]) / p.items;
    T* out = static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.hq + kv * p.group + h0) * c.dim;
    if (tiles == 0) {
      for (int i = tid; i < rows * c.dim; i += kJoinThreads) out[i] = from_f32<T>(0.0f);
      return;
    }
    const int begin = p.first_tile[b] + item * tiles;
    const int o0 = split.owner(begin), o1 = split.owner(begin + tiles - 1);
    if (o0 == o1) return;
    sums(begin, o0, o1, rows, true);
    const int parts = o1 - o0 + 1;
    for (int i = tid; i < rows * c.dim; i += kJoinThreads) {
      const int row = i / c.dim;
      float v = 0.0f;
      for (int j = 0; j < parts; ++j) {
        v = fmaf(p.part_o[static_cast<int64_t>(slot_of(o0 + j, begin)) * kRows * c.dim + i],
                 factor[row * parts + j], v);
      }
      out[i] = from_f32<T>(v / row_lse[row]);
    }
    return;
  }

  if constexpr (kWeights) {
    // tiles of (sequence, KV head), the head tiles of a KV head together
    const int kv_total = total / p.head_tiles;
    const int blocks = gridDim.x - all_items, me = blockIdx.x - all_items;
    const Split mine(kv_total, blocks);
    int t = mine.start(me);
    const int t1 = mine.start(me + 1);
    if (t >= t1) return;
    int b = 0;  // the sequence of tile t: the last whose tiles start at or before it
    for (int step = 1 << 30; step > 0; step >>= 1) {
      if (b + step < a.batch && p.first_tile[b + step] / p.head_tiles <= t) b += step;
    }
    while (t < t1) {
      while (p.first_tile[b + 1] / p.head_tiles <= t) ++b;
      const int n = length_of(p, b), tiles = tiles_of(n);
      const int first = p.first_tile[b] / p.head_tiles;
      const int kv = (t - first) / tiles, tile0 = (t - first) % tiles;
      const int count = min(tiles - tile0, t1 - t);
      for (int ht = 0; ht < p.head_tiles; ++ht) {
        const int begin = p.first_tile[b] + (kv * p.head_tiles + ht) * tiles;
        const int o0 = split.owner(begin), o1 = split.owner(begin + tiles - 1);
        const int rows = min(p.group - ht * kRows, kRows);
        if (o0 == o1) {
          if (tid < rows) {
            row_lse[tid] = p.lse[static_cast<int64_t>(b) * a.hq + kv * p.group + ht * kRows + tid];
          }
          __syncthreads();
        } else {
          sums(begin, o0, o1, rows, false);
        }
        const int stride = min(p.group, kRows);
        for (int i = tid; i < count * kTile; i += kJoinThreads) {
          const int tile = tile0 + i / kTile, pos = tile * kTile + i % kTile;
          if (pos < n) {
            const float* s = p.scores + static_cast<int64_t>(begin + tile) * stride * kTile + i % kTile;
            float w = 0.0f;
            for (int row = 0; row < rows; ++row) w += exp2_fast(s[row * kTile] - row_lse[row]);
            const int page = a.table[static_cast<int64_t>(b) * a.max_blocks + pos / c.block_size];
            if (static_cast<unsigned>(page) < static_cast<unsigned>(c.num_blocks)) {
              float* to = c.weights + (static_cast<int64_t>(page) * c.hkv + kv) * c.block_size +
                          pos % c.block_size;
              // a new token's slot may hold what its page was used for before
              *to = ht == 0 && a.k_new && pos == n - 1 ? w : *to + w;
            }
          }
        }
        __syncthreads();  // row_lse is rewritten
      }
      t += count;
    }
  }
}

// ---- Host ----------------------------------------------------------------------------------------

int64_t aligned_up(int64_t n) { return (n + 255) / 256 * 256; }

// Fills the plan's sizes and, with a workspace, its pointers; returns the workspace's bytes.
int64_t make_plan(const PagedAttentionArgs& a, Plan* p) {
  p->a = a;
  p->group = a.hq / a.cache.hkv;
  p->head_tiles = (p->group + kRows - 1) / kRows;
  const int64_t items = static_cast<int64_t>(a.cache.hkv) * p->head_tiles;
  const int64_t len = static_cast<int64_t>(a.max_blocks) * a.cache.block_size;
  const int64_t tiles = a.batch * items * ((len + kTile - 1) / kTile);
  if (len > INT32_MAX - kTile || tiles > INT32_MAX / 2 || a.batch * items > INT32_MAX / 4) return 0;
  p->items = static_cast<int>(items);
  p->max_len = static_cast<int>(len);
  const int64_t resident = static_cast<int64_t>(sm_count()) * ctas_of(round_dim(a.cache.dim));
  p->blocks = static_cast<int>(std::max<int64_t>(1, std::min(resident, tiles)));
  int64_t at = 0;
  const auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += aligned_up(bytes);
    return static_cast<unsigned char*>(a.workspace) + here;
  };
  p->part_o = reinterpret_cast<float*>(take(2LL * p->blocks * kRows * a.cache.dim * 4));
  p->part_ml = reinterpret_cast<float2*>(take(2LL * p->blocks * kRows * 8));
  p->first_tile = reinterpret_cast<int*>(take((a.batch + 1LL) * 4));
  if (a.cache.weights) {
    p->lse = reinterpret_cast<float*>(take(static_cast<int64_t>(a.batch) * a.hq * 4));
    p->scores = reinterpret_cast<float*>(
        take(tiles * std::min(p->group, kRows) * kTile * 4));
  }
  return at;
}

template <class T, int DP, bool kWeights>
cudaError_t launch(const Plan& p, cudaStream_t stream) {
  static std::once_flag once[64];
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  if (err != cudaSuccess) return err;
  std::call_once(once[dev & 63], [&] {
    err = cudaFuncSetAttribute(paged_attention_kernel<T, DP, kWeights>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(Smem<DP>));
  });
  if (err != cudaSuccess) return err;
  err = launch_serialised(paged_attention_kernel<T, DP, kWeights>, dim3(p.blocks), dim3(kThreads),
                          sizeof(Smem<DP>), stream, 1, p);
  if (err != cudaSuccess) return err;
  const unsigned items = static_cast<unsigned>(p.a.batch) * p.items;
  return launch_serialised(paged_join_kernel<T, kWeights>,
                           dim3(items + (kWeights ? p.blocks : 0)), dim3(kJoinThreads),
                           static_cast<size_t>(p.blocks) * kRows * 4, stream, 1, p);
}

template <class T, bool kWeights>
cudaError_t launch_dim(const Plan& p, cudaStream_t stream) {
  switch (round_dim(p.a.cache.dim)) {
    case 64: return launch<T, 64, kWeights>(p, stream);
    case 128: return launch<T, 128, kWeights>(p, stream);
    default: return launch<T, 256, kWeights>(p, stream);
  }
}

template <class T>
cudaError_t launch_type(const Plan& p, cudaStream_t stream) {
  return p.a.cache.weights ? launch_dim<T, true>(p, stream) : launch_dim<T, false>(p, stream);
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
  return dtype == kWeightF16 ? launch_type<half>(p, stream) : launch_type<__nv_bfloat16>(p, stream);
}

}  // namespace i4
