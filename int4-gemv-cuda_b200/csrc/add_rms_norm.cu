// Root-mean-square norm with the residual's addition: h = x + residual, y = h / rms(h) * weight,
// y in x's type or as e4m3 with one fp32 scale a row.
//
// A row is one pass: h stays in registers (fp32, not rounded before the norm) between the sum of
// its squares and the store. The 8-bit output needs max|y| = max|h w| / rms, so the same reduction
// carries max|h w| beside the sum and the row still needs no second one.
//
// Layout: a row is cut into the 16-byte chunks of memory it lies in, so that a row of odd length
// (whose start falls inside a chunk) still moves whole chunks; only the stores of its first and last
// one go by elements. Blocks stay for many rows: a thread holds its chunks of the weight throughout
// and fetches the next row while this one is summed and stored. A block's rows are a multiple of a
// chunk's elements apart, so they all start at the same place of a chunk. Unaligned tensors and rows
// of more than 2048 chunks take a plain loop that reads the row twice.
//
// Bound by HBM: x, residual, h and y move once each. Measured on B200: 6000 x 8192 fp16 with a residual
// to e4m3 55.7 us, 6.2 TB/s (0.95 of a plain copy's 6.53), to fp16 64.5 us (0.93); 6000 x 8191 89 us
// (0.67: the ends of rows, and registers); 1500 x 30000, by the plain loop, 121 us (0.46). One row of 4096
// takes 1.7 us, the time of a launch.
#include <algorithm>

#include "decode.cuh"
#include "kernels.h"

namespace i4 {
namespace {

constexpr float kE4m3Max = 448.0f;
constexpr int kRowThreads = 1024;  // threads an SM gets
// Threads of a block whose threads take kPer chunks: 544 of two leave room for a second block where
// rows of 8192 elements and a bit have 1025 chunks.
constexpr int most_threads(bool whole, int per) { return whole || per == 1 ? 1024 : per == 2 ? 544 : 704; }
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
  // Elements [lo, hi) of chunk c are inside of the row.
  template <class T>
  __device__ __forceinline__ void inside(int c, int& lo, int& hi) const {
    constexpr int E = Chunk<T>::kElems;
    lo = max(shift - c * E, 0);
    hi = min(shift + a.hidden - c * E, E);
  }
  template <class T, bool kWhole = false>
  __device__ __forceinline__ void store(int c, void* to, const Chunk<T>& v) const {
    constexpr int E = Chunk<T>::kElems;
    T* p = static_cast<T*>(to) + row0 + (c * E - shift);
    if (kWhole || whole<T>(c)) {
      *reinterpret_cast<uint4*>(p) = v.get();
    } else if (a.aligned) {  // by 32-bit words, and halves of those at the ends
      int lo, hi;
      inside<T>(c, lo, hi);
      const uint4 u = v.get();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t word = word_of4(u, j);
        if constexpr (sizeof(T) == 4) {
          if (j >= lo && j < hi) reinterpret_cast<uint32_t*>(p)[j] = word;
        } else {
          const bool first = 2 * j >= lo && 2 * j < hi, second = 2 * j + 1 >= lo && 2 * j + 1 < hi;
          if (first && second) {
            reinterpret_cast<uint32_t*>(p)[j] = word;
          } else if (first) {
            reinterpret_cast<uint16_t*>(p)[2 * j] = static_cast<uint16_t>(word);
          } else if (second) {
            reinterpret_cast<uint16_t*>(p)[2 * j + 1] = static_cast<uint16_t>(word >> 16);
          }
        }
      }
    } else {
      each<T>(c, [&](int i, int) { p[i] = from_f32<T>(v.v[i]); });
    }
  }
  template <class T, bool kWhole = false>
  __device__ __forceinline__ void store_e4m3(int c, const Chunk<T>& v) const {
    constexpr int E = Chunk<T>::kElems;
    uint8_t* p = static_cast<uint8_t*>(a.y) + row0 + (c * E - shift);
    uint32_t w[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      w[i] = e4m3x4(v.v[4 * i], v.v[4 * i + 1], v.v[4 * i + 2], v.v[4 * i + 3]);
    }
    if (kWhole || whole<T>(c)) {
      if constexpr (E == 8) {
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      } else {
        *reinterpret_cast<uint32_t*>(p) = w[0];
      }
    } else {
      int lo, hi;
      inside<T>(c, lo, hi);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (i >= lo && i < hi) p[i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i % 4)));
      }
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

// Any row: read once for the sums and once more for the result.
template <class T, bool Q8>
__global__ void __launch_bounds__(1024) add_rms_norm_kernel(const NormArgs a) {
  __shared__ float2 scratch[kWarp];
  wait_then_release();
  constexpr int E = Chunk<T>::kElems;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, threads = blockDim.x;
  const int64_t row0 = row * a.hidden;
  const int shift = a.aligned ? static_cast<int>(row0 % E) : 0;
  const NormRow r{a, row0, shift, (shift + a.hidden + E - 1) / E};
  Chunk<T> h, w;
  float sum = 0.0f, top = 0.0f;
  for (int c = tid; c < r.chunks; c += threads) {
    r.load<T>(c, h);
    if (Q8) r.load_weight<T>(c, w);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      sum = fmaf(h.v[i], h.v[i], sum);
      if (Q8) top = max_nan(top, fabsf(h.v[i] * w.v[i]));
    }
  }
  row_reduce(sum, top, threads / kWarp, scratch);
  float rstd = rsqrtf(sum / static_cast<float>(a.hidden) + a.eps);
  if constexpr (Q8) {
    float scale = rstd * top / kE4m3Max;
    if (scale < kScaleFloor) scale = kScaleFloor;  // written so that a NaN stays one
    if (tid == 0) a.scales[row] = scale;
    rstd = rstd / scale;
  }
  for (int c = tid; c < r.chunks; c += threads) {
    r.load<T>(c, h);
    r.load_weight<T>(c, w);
    Chunk<T> y;
#pragma unroll
    for (int i = 0; i < E; ++i) y.v[i] = h.v[i] * rstd * w.v[i];
    if (a.h) r.store<T>(c, a.h, h);
    if constexpr (Q8) {
      r.store_e4m3<T>(c, y);
    } else {
      r.store<T>(c, a.y, y);
    }
  }
}

// Rows of aligned tensors. kPer chunks a thread, blocks of as many threads as a row needs; rows are
// taken in turn by the blocks of the grid. kWhole: rows of whole chunks; else gridDim is a multiple
// of a chunk's elements, or no block has more than one row.
template <class T, bool Q8, bool kResidual, bool kWhole, int kPer>
__global__ void __launch_bounds__(most_threads(kWhole, kPer), kPer == 2 && !kWhole ? 2 : 1)
    add_rms_norm_rows_kernel(const NormArgs a) {
  __shared__ float2 scratch[2][kWarp];
  wait_then_release();
  constexpr int E = Chunk<T>::kElems;
  const int tid = threadIdx.x, warps = blockDim.x / kWarp;
  int64_t row = blockIdx.x;
  const int shift = kWhole ? 0 : static_cast<int>(row * a.hidden % E);
  const int chunks = (shift + a.hidden + E - 1) / E;
  const T* weight = static_cast<const T*>(a.weight);
  // elements of chunk c outside of the row
  auto outside = [&](int c, int i) {
    const int e = c * E - shift + i;
    return !kWhole && (e < 0 || e >= a.hidden);
  };
  auto whole = [&](int c) { return kWhole || (c * E >= shift && c * E - shift + E <= a.hidden); };

  uint4 w[kPer], nx[kPer], nr[kPer];
  auto fetch = [&](int64_t row) {
    const int64_t at = row * a.hidden - shift;  // of the first chunk
    const T* x = static_cast<const T*>(a.x) + at;
    const T* residual = static_cast<const T*>(a.residual) + at;
    // chunks up to the tensors' end; the last one may be cut
    const int64_t left = (static_cast<int64_t>(a.rows) * a.hidden - at) / E;
    const int inside = left < chunks ? static_cast<int>(left) : chunks;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int c = tid + j * blockDim.x;
      if (c >= chunks) continue;
      if (kWhole || c < inside) {
        // what a chunk holds of neighbouring rows (several, where they are shorter than a chunk) is
        // read, and left out of the sum; h may be x or residual, but no block writes what this one
        // takes of a chunk
        nx[j] = ld_once_v4(x + c * E);
        if (kResidual) nr[j] = ld_once_v4(residual + c * E);
      } else {  // the tensors end inside of the last chunk
        Chunk<T> fx, fr;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          fx.v[i] = outside(c, i) ? 0.0f : to_f32(x[c * E + i]);
          fr.v[i] = outside(c, i) || !kResidual ? 0.0f : to_f32(residual[c * E + i]);
        }
        nx[j] = fx.get();
        nr[j] = fr.get();
      }
    }
  };
  fetch(row);
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int c = tid + j * blockDim.x;
    Chunk<T> f;
#pragma unroll
    for (int i = 0; i < E; ++i) f.v[i] = 0.0f;
    if (kWhole) {
      if (c < chunks) f.set(*reinterpret_cast<const uint4*>(weight + c * E));
    } else if (c < chunks) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if (!outside(c, i)) f.v[i] = to_f32(weight[c * E - shift + i]);
      }
    }
    w[j] = f.get();
  }
  for (int turn = 0; row < a.rows; row += gridDim.x, turn ^= 1) {
    Chunk<T> h[kPer];
    float sum = 0.0f, top = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int c = tid + j * static_cast<int>(blockDim.x);
      if (c >= chunks) continue;
      h[j].set(nx[j]);
      if (kResidual) {
        Chunk<T> r;
        r.set(nr[j]);
#pragma unroll
        for (int i = 0; i < E; ++i) h[j].v[i] += r.v[i];
      }
      if (!whole(c)) {
#pragma unroll
        for (int i = 0; i < E; ++i) h[j].v[i] = outside(c, i) ? 0.0f : h[j].v[i];
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
    const NormRow r{a, row * a.hidden, shift, chunks};
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int c = tid + j * blockDim.x;
      if (c >= chunks) continue;
      if (kResidual) r.store<T, kWhole>(c, a.h, h[j]);
      Chunk<T> y;
      y.set(w[j]);
#pragma unroll
      for (int i = 0; i < E; ++i) y.v[i] = h[j].v[i] * rstd * y.v[i];
      if constexpr (Q8) {
        r.store_e4m3<T, kWhole>(c, y);
      } else {
        r.store<T, kWhole>(c, a.y, y);
      }
    }
  }
}

template <class T, bool Q8>
cudaError_t launch(const NormArgs& a, cudaStream_t stream) {
  constexpr int E = Chunk<T>::kElems;
  const auto up = [](int n, int to) { return (n + to - 1) / to * to; };
  const bool whole = a.hidden % E == 0;
  const int chunks = whole ? a.hidden / E : (E - 1 + a.hidden + E - 1) / E;  // at any shift
  // without a residual h is x, and a caller that asks for it gets a copy from the plain loop
  if (!a.aligned || chunks > (whole ? 2 * 1024 : 3 * most_threads(false, 3)) || (a.h && !a.residual)) {
    return launch_serialised(add_rms_norm_kernel<T, Q8>, dim3(a.rows),
                             dim3(std::min(1024, up(chunks, kWarp))), 0, stream, 1, a);
  }
  // one chunk a thread for rows of few chunks, and for few rows (latency); else two, or three
  const int per = chunks <= 256 || (a.rows <= sm_count() && chunks <= 1024) ? 1
                  : chunks <= 2 * most_threads(whole, 2)                    ? 2
                                                                            : 3;
  const int threads = up((chunks + per - 1) / per, kWarp);
  int ctas = (threads > 512 ? (threads <= most_threads(false, 2) ? 2 : 1) : kRowThreads / threads) * sm_count();
  if (!whole) ctas = ctas / E * E;
  const auto rows = [&](auto one, auto two, auto three) {
    return launch_serialised(per == 1 ? one : per == 2 ? two : three, dim3(std::min(a.rows, ctas)),
                             dim3(threads), 0, stream, 1, a);
  };
  const auto kind = [&]<bool kResidual, bool kWhole>() {
    return rows(add_rms_norm_rows_kernel<T, Q8, kResidual, kWhole, 1>,
                add_rms_norm_rows_kernel<T, Q8, kResidual, kWhole, 2>,
                add_rms_norm_rows_kernel<T, Q8, kResidual, kWhole, kWhole ? 2 : 3>);
  };
  if (a.residual) {
    return whole ? kind.template operator()<true, true>() : kind.template operator()<true, false>();
  }
  return whole ? kind.template operator()<false, true>() : kind.template operator()<false, false>();
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
