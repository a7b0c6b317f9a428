// Device helpers of the decode-step operators (add_rms_norm, paged_attention, paged_evict,
// token_logprobs): element types, 16-byte accesses, block reductions, and the order in which a
// kernel of a programmatically serialised stream waits and lets the next one start.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace i4 {

// Every decode kernel calls this first: wait for the previous kernel in the stream to complete,
// then let the next one launch. In this order a kernel that starts early (this library's GEMVs
// fetch their weights before their own wait) has everything before this kernel complete and
// visible, so weights written by a kernel that was followed by one of these are safe to prefetch.
__device__ __forceinline__ void wait_only() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void wait_then_release() {
  wait_only();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ---- Element types ------------------------------------------------------------------------------

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// Two elements in one 32-bit register, the first in the low half.
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  uint32_t u;
  memcpy(&u, &h, 4);
  return u;
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  uint32_t u;
  memcpy(&u, &h, 4);
  return u;
}

template <class T>
__device__ __forceinline__ float2 unpack2(uint32_t u);
template <>
__device__ __forceinline__ float2 unpack2<half>(uint32_t u) { return half2_bits_to_float2(u); }
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}

// The elements of one 16-byte chunk as fp32.
template <class T>
struct Chunk {
  static constexpr int kElems = 16 / sizeof(T);
  float v[kElems];

  __device__ __forceinline__ void set(const uint4& u) {
    if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(u.x);
      v[1] = __uint_as_float(u.y);
      v[2] = __uint_as_float(u.z);
      v[3] = __uint_as_float(u.w);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(word_of4(u, i));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ uint4 get() const {
    if constexpr (sizeof(T) == 4) {
      return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                        __float_as_uint(v[3]));
    } else {
      return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]),
                        pack2<T>(v[6], v[7]));
    }
  }
};

// The larger of two values; NaN if either is one.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x, to 2 units in the last place; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;

// A float as an unsigned number of the same order: NaN above everything, -0 like 0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float from_order_key(uint32_t k) {
  if (k == 0xFFFFFFFFu) return __uint_as_float(0x7FFFFFFFu);
  return __uint_as_float(k >> 31 ? k ^ 0x80000000u : ~k);
}

// Unsigned division by a number known on the host, for dividends below 2^31 (Granlund and
// Montgomery, Division by invariant integers using multiplication, 1994).
struct Divider {
  uint32_t mul, shift, by;
  Divider() = default;
  explicit Divider(uint32_t d) : by(d) {
    shift = 0;
    while ((1ull << shift) < d) ++shift;
    mul = static_cast<uint32_t>(((1ull << shift) - d) * (1ull << 32) / d + 1);
  }
  __device__ __forceinline__ uint32_t quotient(uint32_t n) const {
    return (__umulhi(mul, n) + n) >> shift;
  }
};

// 16 bytes that the kernel reads once, and may write later (so not by the read-only path), kept out
// of L1.
__device__ __forceinline__ uint4 ld_once_v4(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p)
               : "memory");
  return v;
}

// 16 bytes of shared memory by their address.
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

// ---- 16-byte asynchronous copies global -> shared, by the thread that waits for them -------------

__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// Zeros where `there` is false; src is not read then.
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---- Launch -------------------------------------------------------------------------------------

// Launches `kernel` with programmatic stream serialization (see wait_then_release), its blocks
// along x in clusters of `cluster`.
template <class... P, class... A>
cudaError_t launch_serialised(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem,
                              cudaStream_t stream, int cluster, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

}  // namespace i4
