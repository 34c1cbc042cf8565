// Dropout whose mask is a function of (seed, offset, element index) and is formed again wherever it is needed, so it is
// never stored: out = [residual +] keep ? x * scale : 0. The backward pass is the same kernel on the gradient.
#include "elem.cuh"

namespace psgd {
namespace {

constexpr int DROP_THREADS = 256;

// One generator block (8 elements) a thread and turn. VEC: every pointer is 16-byte aligned, so whole blocks move as
// vectors; the last, partial block (and every block without VEC) goes element by element.
template <typename T, bool VEC>
__global__ void __launch_bounds__(DROP_THREADS) dropout_kernel(const T* __restrict__ x, const T* __restrict__ residual,
                                                               T* __restrict__ out, long long n, uint32_t threshold,
                                                               float scale, unsigned long long seed,
                                                               unsigned long long offset, const long long* rng) {
  const Keep keep(seed, offset, rng, threshold);
  const long long blocks = (n + 7) / 8;
  for (long long b = (long long)blockIdx.x * DROP_THREADS + threadIdx.x; b < blocks;
       b += (long long)gridDim.x * DROP_THREADS) {
    const uint32_t m = keep.mask8((unsigned long long)b);
    const long long at = 8 * b;
    if (VEC && at + 8 <= n) {
      float v[8], r[8];
      load_vec<T, 8>(x + at, v);
      if (residual) load_vec<T, 8>(residual + at, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = (m >> i) & 1u ? v[i] * scale : 0.f;
        if (residual) v[i] += r[i];
      }
      store_vec<T, 8>(out + at, v);
    } else {
      for (int i = 0; i < 8 && at + i < n; ++i) {
        float v = (m >> i) & 1u ? to_f32(x[at + i]) * scale : 0.f;
        if (residual) v += to_f32(residual[at + i]);
        out[at + i] = from_f32<T>(v);
      }
    }
  }
}

template <typename T>
int launch(const PsgdDropout& d, cudaStream_t stream) {
  const bool vec = aligned16(d.x) && aligned16(d.out) && aligned16(d.residual);
  const long long blocks = (d.n + 7) / 8, want = (blocks + DROP_THREADS - 1) / DROP_THREADS;
  const long long most = 8LL * psgd_num_sms();
  const int grid = (int)(want < most ? want : most);
  const T* x = reinterpret_cast<const T*>(d.x);
  const T* r = reinterpret_cast<const T*>(d.residual);
  T* out = reinterpret_cast<T*>(d.out);
  if (vec)
    dropout_kernel<T, true><<<grid, DROP_THREADS, 0, stream>>>(x, r, out, d.n, d.threshold, d.scale, d.seed, d.offset, d.rng);
  else
    dropout_kernel<T, false><<<grid, DROP_THREADS, 0, stream>>>(x, r, out, d.n, d.threshold, d.scale, d.seed, d.offset, d.rng);
  return cudaGetLastError() == cudaSuccess ? PSGD_OK : PSGD_ELAUNCH;
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
