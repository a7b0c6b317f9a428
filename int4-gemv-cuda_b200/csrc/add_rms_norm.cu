// Root-mean-square norm with the residual's addition: h = x + residual, y = h / rms(h) * weight,
// y in x's type or as e4m3 with one fp32 scale a row.
//
// A row is one pass: h stays in registers (fp32, not rounded before the norm) between the sum of
// its squares and the store. The 8-bit output needs max|y| = max|h w| / rms, so the same reduction
// carries max|h w| beside the sum and the row still needs no second one.
//
// Layout: rows of whole 16-byte chunks go to blocks that stay for many rows: a thread holds its
// chunks of the weight throughout and fetches the next row while this one is summed and stored.
// Other rows (odd lengths, unaligned tensors) are cut into the chunks of memory they lie in, so that
// they still move whole chunks and only their first and last one by elements.
//
// Bound by HBM: x, residual, h and y move once each.
#include <algorithm>

#include "decode.cuh"
#include "kernels.h"

namespace i4 {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr int kRowThreads = 1024;  // threads an SM gets for rows of whole chunks
constexpr float kScaleFloor = 1e-12f;  // a row of zeros still has a scale to divide by

// Four / eight e4m3 values of y, saturating (a NaN stays one).
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
}

struct NormRow {
  const NormArgs& a;
  int64_t row0;  // first element of the row in x, residual, h and y
  int shift;     // elements between the row's first chunk boundary and the row
  int chunks;    // chunks the row lies in

  template <class T>
  __device__ __forceinline__ bool whole(int c) const {
    constexpr int E = Chunk<T>::kElems;
    return a.aligned && c * E >= shift && (c + 1) * E <= shift + a.hidden;
  }
  // Elements of chunk c inside the row: calls f(i in chunk, element of the row).
  template <class T, class F>
  __device__ __forceinline__ void each(int c, F f) const {
    constexpr int E = Chunk<T>::kElems;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int e = c * E + i - shift;
      if (e >= 0 && e < a.hidden) f(i, e);
    }
  }
  template <class T>
  __device__ __forceinline__ void load(int c, Chunk<T>& h) const {
    constexpr int E = Chunk<T>::kElems;
    const T* x = static_cast<const T*>(a.x) + row0;
    const T* r = static_cast<const T*>(a.residual) + row0;
    if (whole<T>(c)) {
      h.set(*reinterpret_cast<const uint4*>(x + (c * E - shift)));
      if (a.residual) {
        Chunk<T> rc;
        rc.set(*reinterpret_cast<const uint4*>(r + (c * E - shift)));
#pragma unroll
        for (int i = 0; i < E; ++i) h.v[i] += rc.v[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) h.v[i] = 0.0f;
      each<T>(c, [&](int i, int e) {
        h.v[i] = to_f32(x[e]) + (a.residual ? to_f32(r[e]) : 0.0f);
      });
    }
  }
  template <class T>
  __device__ __forceinline__ void load_weight(int c, Chunk<T>& w) const {
    constexpr int E = Chunk<T>::kElems;
    const T* p = static_cast<const T*>(a.weight);
    if (shift == 0 && whole<T>(c)) {
      w.set(*reinterpret_cast<const uint4*>(p + c * E));
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) w.v[i] = 0.0f;
      each<T>(c, [&](int i, int e) { w.v[i] = to_f32(p[e]); });
    }
  }
  template <class T>
  __device__ __forceinline__ void store(int c, void* to, const Chunk<T>& v) const {
    constexpr int E = Chunk<T>::kElems;
    T* p = static_cast<T*>(to) + row0;
    if (whole<T>(c)) {
      *reinterpret_cast<uint4*>(p + (c * E - shift)) = v.get();
    } else {
      each<T>(c, [&](int i, int e) { p[e] = from_f32<T>(v.v[i]); });
    }
  }
  template <class T>
  __device__ __forceinline__ void store_e4m3(int c, const Chunk<T>& v) const {
    constexpr int E = Chunk<T>::kElems;
    uint8_t* p = static_cast<uint8_t*>(a.y) + row0;
    uint32_t w[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      w[i] = e4m3x4(v.v[4 * i], v.v[4 * i + 1], v.v[4 * i + 2], v.v[4 * i + 3]);
    }
    if (whole<T>(c)) {
      if constexpr (E == 8) {
        *reinterpret_cast<uint2*>(p + (c * E - shift)) = make_uint2(w[0], w[1]);
      } else {
        *reinterpret_cast<uint32_t*>(p + (c * E - shift)) = w[0];
      }
    } else {
      each<T>(c, [&](int i, int e) { p[e] = static_cast<uint8_t>(w[i / 4] >> (8 * (i % 4))); });
    }
  }
};

// The sum of `sum` and the maximum of `top` over the row's threads (`warps` warps of the block).
__device__ __forceinline__ void row_reduce(float& sum, float& top, int warps, float2* scratch) {
#pragma unroll
  for (int off = kWarp / 2; off > 0; off >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, off);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
  }
  if (warps == 1) return;
  const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
  if (lane == 0) scratch[warp] = make_float2(sum, top);
  __syncthreads();
  const float2 v = lane < warps ? scratch[lane] : make_float2(0.0f, 0.0f);
  sum = v.x;
  top = v.y;
#pragma unroll
  for (int off = kWarp / 2; off > 0; off >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, off);
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
  }
}

// kPer chunks a thread are kept in registers; kPer = 0: rows longer than a block holds, read twice.
// kRows > 1: a warp a row, kRows rows a block.
template <class T, bool Q8, int kPer, int kRows>
__global__ void __launch_bounds__(kRows > 1 ? kRows * kWarp : 1024)
    add_rms_norm_kernel(const NormArgs a) {
  __shared__ float2 scratch[kWarp];
  wait_then_release();
  constexpr int E = Chunk<T>::kElems;
  const int64_t row = kRows > 1 ? static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kWarp
                                : blockIdx.x;
  if (kRows > 1 && row >= a.rows) return;  // whole warps: a row's warp needs no other
  const int threads = kRows > 1 ? kWarp : blockDim.x;
  const int tid = kRows > 1 ? threadIdx.x % kWarp : threadIdx.x;
  const int64_t row0 = row * a.hidden;
  const int shift = a.aligned ? static_cast<int>(row0 % E) : 0;
  const NormRow r{a, row0, shift, (shift + a.hidden + E - 1) / E};

  constexpr int kHeld = kPer > 0 ? kPer : 1;
  Chunk<T> h[kHeld], w[kHeld];
  float sum = 0.0f, top = 0.0f;
  auto add = [&](const Chunk<T>& hc, const Chunk<T>& wc) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      sum = fmaf(hc.v[i], hc.v[i], sum);
      if (Q8) top = max_nan(top, fabsf(hc.v[i] * wc.v[i]));
    }
  };
  if constexpr (kPer > 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int c = tid + j * threads;
      if (c < r.chunks) {
        r.load<T>(c, h[j]);
        r.load_weight<T>(c, w[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (tid + j * threads < r.chunks) add(h[j], w[j]);
    }
  } else {
    for (int c = tid; c < r.chunks; c += threads) {
      r.load<T>(c, h[0]);
      if (Q8) r.load_weight<T>(c, w[0]);
      add(h[0], w[0]);
    }
  }
  row_reduce(sum, top, kRows > 1 ? 1 : (blockDim.x + kWarp - 1) / kWarp, scratch);

  float rstd = rsqrtf(sum / static_cast<float>(a.hidden) + a.eps);
  if constexpr (Q8) {
    float scale = rstd * top / kE4m3Max;
    if (scale < kScaleFloor) scale = kScaleFloor;  // written so that a NaN stays one
    if (tid == 0) a.scales[row] = scale;
    rstd = rstd / scale;
  }
  auto finish = [&](int c, const Chunk<T>& hc, const Chunk<T>& wc) {
    Chunk<T> y;
#pragma unroll
    for (int i = 0; i < E; ++i) y.v[i] = hc.v[i] * rstd * wc.v[i];
    if (a.h) r.store<T>(c, a.h, hc);
    if constexpr (Q8) {
      r.store_e4m3<T>(c, y);
    } else {
      r.store<T>(c, a.y, y);
    }
  };
  if constexpr (kPer > 0) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int c = tid + j * threads;
      if (c < r.chunks) finish(c, h[j], w[j]);
    }
  } else {
    for (int c = tid; c < r.chunks; c += threads) {
      r.load<T>(c, h[0]);
      r.load_weight<T>(c, w[0]);
      finish(c, h[0], w[0]);
    }
  }
}

// Rows of whole chunks. kPer chunks a thread, blocks of as many threads as a row needs; rows are
// taken in turn by the blocks of the grid.
template <class T, bool Q8, bool kResidual, int kPer>
__global__ void __launch_bounds__(1024) add_rms_norm_rows_kernel(const NormArgs a) {
  __shared__ float2 scratch[2][kWarp];
  wait_then_release();
  constexpr int E = Chunk<T>::kElems;
  const int chunks = a.hidden / E, tid = threadIdx.x;
  const int warps = blockDim.x / kWarp;
  const uint4* x = static_cast<const uint4*>(a.x);
  const uint4* residual = static_cast<const uint4*>(a.residual);
  const uint4* weight = static_cast<const uint4*>(a.weight);

  uint4 w[kPer], nx[kPer], nr[kPer];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int c = tid + j * blockDim.x;
      if (c < chunks) {
        nx[j] = ld_stream_v4(x + row * chunks + c);
        if (kResidual) nr[j] = ld_stream_v4(residual + row * chunks + c);
      }
    }
  };
  int64_t row = blockIdx.x;
  fetch(row);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int c = tid + j * blockDim.x;
    w[j] = c < chunks ? weight[c] : make_uint4(0, 0, 0, 0);
  }
  for (int turn = 0; row < a.rows; row += gridDim.x, turn ^= 1) {
    Chunk<T> h[kPer];
    float sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if (tid + j * static_cast<int>(blockDim.x) >= chunks) continue;
      h[j].set(nx[j]);
      if (kResidual) {
        Chunk<T> r;
        r.set(nr[j]);
#pragma unroll
        for (int i = 0; i < E; ++i) h[j].v[i] += r.v[i];
      }
      Chunk<T> wc;
      if (Q8) wc.set(w[j]);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        sum = fmaf(h[j].v[i], h[j].v[i], sum);
        if (Q8) top = max_nan(top, fabsf(h[j].v[i] * wc.v[i]));
      }
    }
    if (row + gridDim.x < a.rows) fetch(row + gridDim.x);
    // two scratch rows in turn: a warp writes one again only after a barrier behind its reads
    row_reduce(sum, top, warps, scratch[turn]);
    float rstd = rsqrtf(sum / static_cast<float>(a.hidden) + a.eps);
    if constexpr (Q8) {
      float scale = rstd * top / kE4m3Max;
      if (scale < kScaleFloor) scale = kScaleFloor;  // written so that a NaN stays one
      if (tid == 0) a.scales[row] = scale;
      rstd = rstd / scale;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int c = tid + j * blockDim.x;
      if (c >= chunks) continue;
      if (kResidual) static_cast<uint4*>(a.h)[row * chunks + c] = h[j].get();
      Chunk<T> y;
      y.set(w[j]);
#pragma unroll
      for (int i = 0; i < E; ++i) y.v[i] = h[j].v[i] * rstd * y.v[i];
      if constexpr (!Q8) {
        static_cast<uint4*>(a.y)[row * chunks + c] = y.get();
      } else {
        uint32_t* to = static_cast<uint32_t*>(a.y) + (row * chunks + c) * (E / 4);
        if constexpr (E == 8) {
          *reinterpret_cast<uint2*>(to) = make_uint2(e4m3x4(y.v[0], y.v[1], y.v[2], y.v[3]),
                                                     e4m3x4(y.v[4], y.v[5], y.v[6], y.v[7]));
        } else {
          *to = e4m3x4(y.v[0], y.v[1], y.v[2], y.v[3]);
        }
      }
    }
  }
}

template <class T, bool Q8>
cudaError_t launch(const NormArgs& a, cudaStream_t stream) {
  constexpr int E = Chunk<T>::kElems;
  const auto up = [](int n, int to) { return (n + to - 1) / to * to; };
  // without a residual h is x, and a caller that asks for it gets a copy from the general kernel
  if (a.aligned && a.hidden % E == 0 && a.hidden / E <= 2048 && (a.residual || !a.h)) {
    const int chunks = a.hidden / E;
    const auto rows = [&](auto with, auto without, int per) {
      const int threads = up((chunks + per - 1) / per, kWarp);
      const int ctas = std::max(1, kRowThreads / threads) * sm_count();
      return launch_serialised(a.residual ? with : without, dim3(std::min(a.rows, ctas)),
                               dim3(threads), 0, stream, 1, a);
    };
    const bool few = a.rows <= sm_count();
    if (chunks <= 256 || (few && chunks <= 1024)) {
      return rows(add_rms_norm_rows_kernel<T, Q8, true, 1>, add_rms_norm_rows_kernel<T, Q8, false, 1>, 1);
    }
    return rows(add_rms_norm_rows_kernel<T, Q8, true, 2>, add_rms_norm_rows_kernel<T, Q8, false, 2>, 2);
  }
  const int most = (E - 1 + a.hidden + E - 1) / E;  // chunks of a row at any shift
  if (most <= kWarp * 4 && a.rows > 1) {
    constexpr int kRows = 4;
    return launch_serialised(add_rms_norm_kernel<T, Q8, 4, kRows>,
                             dim3((a.rows + kRows - 1) / kRows), dim3(kRows * kWarp), 0, stream, 1,
                             a);
  }
  const auto block = [&](auto kernel, int per) {
    return launch_serialised(kernel, dim3(a.rows), dim3(up((most + per - 1) / per, kWarp)), 0,
                             stream, 1, a);
  };
  if (most <= 1024) return block(add_rms_norm_kernel<T, Q8, 1, 1>, 1);
  if (most <= 2048) return block(add_rms_norm_kernel<T, Q8, 2, 1>, 2);
  return launch_serialised(add_rms_norm_kernel<T, Q8, 0, 1>, dim3(a.rows), dim3(1024), 0, stream, 1,
                           a);
}

template <bool Q8>
cudaError_t launch_type(const NormArgs& a, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case kWeightF32: return launch<float, Q8>(a, stream);
    case kWeightF16: return launch<half, Q8>(a, stream);
    default: return launch<__nv_bfloat16, Q8>(a, stream);
  }
}

}  // namespace

cudaError_t launch_add_rms_norm(const NormArgs& a, int dtype, cudaStream_t stream) {
  return a.scales ? launch_type<true>(a, dtype, stream) : launch_type<false>(a, dtype, stream);
}

}  // namespace i4
