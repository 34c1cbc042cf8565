// Elements of the model-side operators (fp32, bf16 or fp16 in memory, fp32 in registers) and the 16-bit fields of the
// counter-based generator that dropout compares.
#pragma once
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"
#include "philox.cuh"
#include "psgd_b200.h"

namespace psgd {

template <typename T> __host__ __device__ constexpr bool is_half() { return false; }
template <> __host__ __device__ constexpr bool is_half<__half>() { return true; }

PSGD_DEVI float to_f32(float v) { return v; }
PSGD_DEVI float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
PSGD_DEVI float to_f32(__half v) { return __half2float(v); }
template <typename T> PSGD_DEVI T from_f32(float v);
template <> PSGD_DEVI float from_f32<float>(float v) { return v; }
template <> PSGD_DEVI __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> PSGD_DEVI __half from_f32<__half>(float v) { return __float2half_rn(v); }

PSGD_DEVI float2 unpack2(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
PSGD_DEVI float2 unpack2(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
PSGD_DEVI uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
PSGD_DEVI uint32_t pack2(float a, float b, __half) {
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// V consecutive elements (V = 8: 16-byte aligned vectors; V = 1: any address).
template <typename T, int V>
PSGD_DEVI void load_vec(const T* __restrict__ p, float* v) {
  if constexpr (V == 1) {
    v[0] = to_f32(*p);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(w[i], T());
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}
// Eight elements from their 16-byte pieces (one, or two of fp32).
template <typename T>
PSGD_DEVI void unpack_pieces(const uint4* p, float* v) {
#pragma unroll
  for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
    const uint32_t w[4] = {p[h].x, p[h].y, p[h].z, p[h].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[4 * h + i] = __uint_as_float(w[i]);
      } else {
        const float2 f = unpack2(w[i], T());
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}
template <typename T, int V>
PSGD_DEVI void store_vec(T* p, const float* v) {
  if constexpr (V == 1) {
    *p = from_f32<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], T()), pack2(v[2], v[3], T()), pack2(v[4], v[5], T()),
                                              pack2(v[6], v[7], T()));
  }
}

// One element of a vector whose type is known at run time (PSGD_F32 / PSGD_BF16 / PSGD_F16).
PSGD_DEVI void store_any(void* p, int dtype, long long i, float v) {
  if (dtype == PSGD_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == PSGD_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

// Which elements dropout keeps: element i of a tensor (in its row-major order) belongs to block i / 8 of the generator's
// sequence `offset` under key `seed`, and is kept when 16-bit field i % 8 of that block's four words (low half first) is
// at least the threshold T = round(65536 p). Sixteen bits an element halve the generator's work against one word an
// element; the kept values are scaled by 1 / (1 - T / 65536), the inverse of the probability that is really used.
struct Keep {
  uint32_t o0, o1, k0, k1, limit;  // limit: T << 16, which a word is compared with for its high field, shifted for its low one
  bool none;                       // T = 65536: nothing is kept (words of zeros stay below every limit)
  PSGD_DEVI Keep(unsigned long long seed, unsigned long long offset, const long long* rng, uint32_t threshold) {
    if (rng) {
      seed = (unsigned long long)rng[0];
      offset = (unsigned long long)rng[1];
    }
    k0 = (uint32_t)seed;
    k1 = (uint32_t)(seed >> 32);
    o0 = (uint32_t)offset;
    o1 = (uint32_t)(offset >> 32);
    none = threshold > 65535u;
    limit = none ? 0xFFFFFFFFu : threshold << 16;
  }
  PSGD_DEVI uint4 block(unsigned long long b) const {
    if (none) return make_uint4(0u, 0u, 0u, 0u);
    return philox4x32_10(make_uint4((uint32_t)b, (uint32_t)(b >> 32), o0, o1), k0, k1);
  }
  PSGD_DEVI bool low(uint32_t word) const { return (word << 16) >= limit; }   // fields 0, 2, 4, 6
  PSGD_DEVI bool high(uint32_t word) const { return word >= limit; }          // fields 1, 3, 5, 7
  PSGD_DEVI uint32_t mask8(unsigned long long b) const {  // bit f: field f of the block is kept
    const uint4 r = block(b);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m |= (low(w[i]) ? 1u << (2 * i) : 0u) | (high(w[i]) ? 2u << (2 * i) : 0u);
    return m;
  }
};
PSGD_DEVI uint32_t word_of(const uint4& r, int i) { return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w; }

// A launch that may start while the one before it ends (its kernel waits for that one by pdl_wait before it reads anything).
template <typename... P, typename... A>
int pdl_launch(void (*kernel)(P...), dim3 grid, dim3 block, int smem, cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid, c.blockDim = block, c.dynamicSmemBytes = smem, c.stream = stream;
  cudaLaunchAttribute at = {};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &at, c.numAttrs = 1;
  if (cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...) == cudaSuccess) return PSGD_OK;
  cudaGetLastError();  // else it would be taken for a later launch's
  return PSGD_ELAUNCH;
}

// Dynamic shared memory beyond what a kernel has without asking; `done` remembers the devices where it was granted, one
// bit each. A refusal is cleared: it would be taken for a later launch's.
template <typename K>
int allow_smem(K kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev > 63) return PSGD_ELAUNCH;
  if ((done.load(std::memory_order_relaxed) >> dev) & 1) return PSGD_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return PSGD_ELAUNCH;
  }
  done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return PSGD_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace psgd
