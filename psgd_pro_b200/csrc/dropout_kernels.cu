// Dropout whose mask is a function of (seed, offset, element index) and is formed again wherever it is needed, so it is
// never stored: out = [residual +] keep ? x * scale : 0. The backward pass is the same kernel on the gradient.
//
// Bound by memory traffic with a residual (46.1M bf16 values: 49 to 51 us, 5.5 to 5.6 TB/s of 6.46 that a copy has). Without
// one (16.8M fp16 values: 16.4 us, 4.1 TB/s) by latency: a thread's loads, its ten dependent rounds and its stores follow each
// other (the issue slots are 58% busy; the multiplications alone would take some 5 us). One generator call of ten rounds
// serves 8 elements; a thread has two calls' data under way (one: 49.6 and 18.3 us), four blocks an SM (six: 49.7 and 16.5).
#include "elem.cuh"

namespace psgd {
namespace {

constexpr int DROP_THREADS = 256, DROP_UNROLL = 2, DROP_BLOCKS = 4;  // (blocks of an SM)

// Eight elements: 16 bytes, or 32 at once (two 16-byte loads would take half a sector each, twice).
template <int H>
PSGD_DEVI void load_pieces(const void* p, uint4* v) {
  if constexpr (H == 1) {
    v[0] = *reinterpret_cast<const uint4*>(p);
  } else {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0].x), "=r"(v[0].y), "=r"(v[0].z), "=r"(v[0].w), "=r"(v[1].x), "=r"(v[1].y), "=r"(v[1].z), "=r"(v[1].w)
                 : "l"(p));
  }
}
template <typename T>
PSGD_DEVI void store_pieces(T* p, const float* f) {
  if constexpr (sizeof(T) == 2) {
    store_vec<T, 8>(p, f);
  } else {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]),
                 "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
                 : "memory");
  }
}

// A generator block (8 elements) at a time, DROP_UNROLL of them DROP_THREADS apart so that their loads are under way
// together. VEC: every pointer is aligned to a block's bytes and whole blocks move as vectors; the last, partial block (and all
// without VEC) goes element by element.
template <typename T, bool VEC, bool RESIDUAL>
__global__ void __launch_bounds__(DROP_THREADS, DROP_BLOCKS)
    dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual, T* __restrict__ out, long long n,
                   uint32_t threshold, float scale, unsigned long long seed, unsigned long long offset,
                   const long long* rng) {
  constexpr int H = sizeof(T) / 2;  // 16-byte pieces to 8 elements
  const Keep keep(seed, offset, rng, threshold);
  const long long whole = VEC ? n / 8 : 0, step = (long long)gridDim.x * DROP_THREADS * DROP_UNROLL;
  for (long long b0 = (long long)blockIdx.x * DROP_THREADS * DROP_UNROLL + threadIdx.x; b0 < whole; b0 += step) {
    uint4 v[DROP_UNROLL][H], r[DROP_UNROLL][H];
#pragma unroll
    for (int u = 0; u < DROP_UNROLL; ++u) {
      const long long b = b0 + u * DROP_THREADS;
      if (b < whole) {
        load_pieces<H>(x + 8 * b, v[u]);
        if (RESIDUAL) load_pieces<H>(residual + 8 * b, r[u]);
      }
    }
#pragma unroll
    for (int u = 0; u < DROP_UNROLL; ++u) {
      const long long b = b0 + u * DROP_THREADS;
      if (b >= whole) break;
      const uint4 words = keep.block((unsigned long long)b);
      float f[8], add[8];
      unpack_pieces<T>(v[u], f);
      if (RESIDUAL) unpack_pieces<T>(r[u], add);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t w = word_of(words, i / 2);
        f[i] = (i & 1 ? keep.high(w) : keep.low(w)) ? f[i] * scale : 0.f;
        if (RESIDUAL) f[i] += add[i];
      }
      store_pieces<T>(out + 8 * b, f);
    }
  }
  const long long blocks = (n + 7) / 8;
  for (long long b = whole + (long long)blockIdx.x * DROP_THREADS + threadIdx.x; b < blocks;
       b += (long long)gridDim.x * DROP_THREADS) {
    const uint4 words = keep.block((unsigned long long)b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long at = 8 * b + i;
      if (at >= n) break;
      const uint32_t w = word_of(words, i / 2);
      float f = (i & 1 ? keep.high(w) : keep.low(w)) ? to_f32(x[at]) * scale : 0.f;
      if (RESIDUAL) f += to_f32(residual[at]);
      out[at] = from_f32<T>(f);
    }
  }
}

template <typename T, bool VEC, bool RESIDUAL>
int start(const PsgdDropout& d, cudaStream_t stream) {
  const long long want = ((d.n + 7) / 8 + DROP_THREADS - 1) / DROP_THREADS, most = (long long)DROP_BLOCKS * psgd_num_sms();
  dropout_kernel<T, VEC, RESIDUAL><<<(int)(want < most ? want : most), DROP_THREADS, 0, stream>>>(
      reinterpret_cast<const T*>(d.x), reinterpret_cast<const T*>(d.residual), reinterpret_cast<T*>(d.out), d.n, d.threshold,
      d.scale, d.seed, d.offset, d.rng);
  return cudaGetLastError() == cudaSuccess ? PSGD_OK : PSGD_ELAUNCH;
}

template <typename T>
int launch(const PsgdDropout& d, cudaStream_t stream) {
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & (8 * sizeof(T) - 1)) == 0; };
  const bool vec = aligned(d.x) && aligned(d.out) && aligned(d.residual);
  if (d.residual) return vec ? start<T, true, true>(d, stream) : start<T, false, true>(d, stream);
  return vec ? start<T, true, false>(d, stream) : start<T, false, false>(d, stream);
}

}  // namespace
}  // namespace psgd

extern "C" int psgd_dropout(const PsgdDropout* d, cudaStream_t stream) {
  using namespace psgd;
  if (!d || d->n < 0 || d->threshold > 65536u || (d->n > 0 && (!d->x || !d->out))) return PSGD_EINVAL;
  if (d->n == 0) return PSGD_OK;
  switch (d->dtype) {
    case PSGD_F32: return launch<float>(*d, stream);
    case PSGD_BF16: return launch<__nv_bfloat16>(*d, stream);
    case PSGD_F16: return launch<__half>(*d, stream);
    default: return PSGD_EINVAL;
  }
}
