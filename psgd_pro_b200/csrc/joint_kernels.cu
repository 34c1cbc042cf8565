// The joint between two blocks of a network, one pass over its rows (d elements each):
//   u = post(y) (a norm, or y itself), k = dropout(u), out = x + scale * gate * k, normed = pre(out)
// and its backward pass. rms norm: a / sqrt(mean a^2 + eps) * weight; layer norm: (a - mean) / sqrt(var + eps) * weight
// + bias. Rows are held in registers between their first read and their last write; the variance is a second pass over
// those registers (no cancellation). statistics: (mean, 1 / deviation) of post, then of pre, per row.
//
// A row belongs to a group of `tpr` threads (whole warps), a thread to the elements (i * tpr + t) * V + [0, V) of it; a
// block holds `blockDim.y` groups, each walking rows of its own, which meet at a named barrier of the group.
#include "elem.cuh"

namespace psgd {
namespace {

constexpr int JOINT_MAX_D = PSGD_JOINT_MAX_D;
constexpr int JOINT_MAX_WARPS = 16;  // of a group
constexpr int JOINT_MAX_GROUPS = 8;  // of a block
constexpr int JOINT_THREADS = 256;   // a block's threads while a group has no more than that

// Sum of v[0..N) over the threads of a group. `red` holds two buffers taken in turn: a thread writes one again only
// after the barrier of the other's sum, which every thread reaches after its reads of the first.
template <int N>
struct GroupSum {
  float* red;
  int group, tpr, turn;
  PSGD_DEVI GroupSum(float* r) : red(r), group(threadIdx.y), tpr(blockDim.x), turn(0) {}
  PSGD_DEVI void operator()(float* v) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = warp_sum(v[k]);
    if (tpr == 32) return;
    float* at = red + ((turn * JOINT_MAX_GROUPS) + group) * (JOINT_MAX_WARPS * N);
    turn ^= 1;
    const int warps = tpr >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) at[(threadIdx.x >> 5) * N + k] = v[k];
    named_sync(1 + group, tpr);
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = 0.f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += at[w * N + k];
  }
};

// Copies a parameter vector to shared memory in fp32 (ones or zeros where it is absent).
PSGD_DEVI void stage_param(float* to, const void* from, int dtype, int d, float otherwise) {
  const int t = threadIdx.y * blockDim.x + threadIdx.x, n = blockDim.x * blockDim.y;
  for (int i = t; i < d; i += n) to[i] = from ? load_any(from, dtype, i) : otherwise;
}
template <int V>
PSGD_DEVI void load_smem(const float* p, float* v) {
  if constexpr (V == 1) v[0] = *p;
  else load_vec<float, V>(p, v);
}
template <int V>
PSGD_DEVI void load_param(const void* p, int dtype, int e, float otherwise, float* v) {
#pragma unroll
  for (int k = 0; k < V; ++k) v[k] = p ? load_any(p, dtype, e + k) : otherwise;
}

template <typename T, int V, int NV>
__global__ void __launch_bounds__(512) joint_forward_kernel(const PsgdJoint j) {
  extern __shared__ float4 smem4[];
  __shared__ float red[2 * JOINT_MAX_GROUPS * JOINT_MAX_WARPS];
  const int d = j.d, dp = (d + 7) & ~7;
  float* sw = reinterpret_cast<float*>(smem4);
  float *sb = sw + dp, *spw = sb + dp, *spb = spw + dp;
  stage_param(sw, j.weight, j.param_dtype, d, 1.f);
  stage_param(sb, j.bias, j.param_dtype, d, 0.f);
  if (j.post) {
    stage_param(spw, j.post_weight, j.param_dtype, d, 1.f);
    stage_param(spb, j.post_bias, j.param_dtype, d, 0.f);
  }
  __syncthreads();
  GroupSum<1> sum(red);
  const bool layer = j.kind == PSGD_NORM_LAYER, drop = j.threshold != 0;
  const Keep keep(j.seed, j.offset, j.rng, j.threshold);
  const int tpr = blockDim.x, t = threadIdx.x;
  const float inv_d = 1.f / (float)d;
  const long long per_gate = j.gate ? j.rows / j.gates : 1;

  // (mean, 1 / deviation) of the row in a[] (zero beyond d)
  auto statistics = [&](const float* a, float& mean, float& r) {
    mean = 0.f;
    if (layer) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV * V; ++i) s += a[i];
      sum(&s);
      mean = s * inv_d;
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((i * tpr + t) * V < d)
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float c = a[i * V + k] - mean;
          q += c * c;
        }
    sum(&q);
    r = 1.f / sqrtf(q * inv_d + j.eps);
  };

  for (long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y; row < j.rows;
       row += (long long)gridDim.x * blockDim.y) {
    const T* px = reinterpret_cast<const T*>(j.x) + row * j.ld_x;
    const T* py = reinterpret_cast<const T*>(j.y) + row * j.ld_y;
    T* po = reinterpret_cast<T*>(j.out) + row * d;
    T* pn = reinterpret_cast<T*>(j.normed) + row * d;
    const T* pg = j.gate ? reinterpret_cast<const T*>(j.gate) + (row / per_gate) * d : nullptr;
    float u[NV * V], x[NV * V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * tpr + t) * V;
#pragma unroll
      for (int k = 0; k < V; ++k) u[i * V + k] = x[i * V + k] = 0.f;
      if (e < d) {
        load_vec<T, V>(py + e, u + i * V);
        load_vec<T, V>(px + e, x + i * V);
      }
    }
    float mean_y = 0.f, r_y = 1.f, mean_o, r_o;
    if (j.post) statistics(u, mean_y, r_y);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * tpr + t) * V;
      if (e >= d) continue;
      float* ui = u + i * V;
      if (j.post) {
        float w[V], b[V];
        load_smem<V>(spw + e, w);
        load_smem<V>(spb + e, b);
#pragma unroll
        for (int k = 0; k < V; ++k) ui[k] = (ui[k] - mean_y) * r_y * w[k] + b[k];
      }
      if (drop) {
        const unsigned long long at = (unsigned long long)row * d + e;
        const uint32_t m = V == 8 ? keep.mask8(at >> 3) : (uint32_t)keep.one(at);
#pragma unroll
        for (int k = 0; k < V; ++k) ui[k] = (m >> k) & 1u ? ui[k] * j.keep_scale : 0.f;
      }
      if (pg) {
        float g[V];
        load_vec<T, V>(pg + e, g);
#pragma unroll
        for (int k = 0; k < V; ++k) ui[k] *= g[k];
      }
#pragma unroll
      for (int k = 0; k < V; ++k) x[i * V + k] += j.scale * ui[k];
      store_vec<T, V>(po + e, x + i * V);
    }
    statistics(x, mean_o, r_o);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * tpr + t) * V;
      if (e >= d) continue;
      float w[V], b[V], o[V];
      load_smem<V>(sw + e, w);
      load_smem<V>(sb + e, b);
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] = (x[i * V + k] - mean_o) * r_o * w[k] + b[k];
      store_vec<T, V>(pn + e, o);
    }
    if (t == 0) reinterpret_cast<float4*>(j.stats)[row] = make_float4(mean_y, r_y, mean_o, r_o);
  }
}

// ---- backward --------------------------------------------------------------------------------------------------------
// hat = (out - mean) r, dhat = d_normed w:  dx = d_out + r (dhat - hat mean(dhat hat) [- mean(dhat)]),
// the gradient of what was added is scale * dx; through gate, dropout and the post norm in the same way to dy.
// The parameters' gradients are sums over rows. Each group keeps its share for its own elements, in registers while a
// thread has 8 of them (V * NV = 8) and in its own slots of shared memory beyond, and writes it once, as one row of
// `part`; joint_reduce_kernel adds the rows in a fixed order. F: which of post norm, gate and layer norm are there.
constexpr int F_POST = 1, F_GATE = 2, F_LAYER = 4, F_RUNTIME = 8;

// How rows are dealt out to groups ("units"): `per_unit` consecutive rows each. With a gate, a unit holds whole gate
// groups (chunks = 0), whose gradient it then writes itself, or a chunk of one group (chunks to a group).
struct JointPlan {
  long long units, per_unit, chunks, per_gate;
  int tpr, groups, grid, vec, nv, smem;
  int slot[5];  // of dweight, dbias, dpost_weight, dpost_bias, dgate in `part`, or -1
  int slots;
};

template <typename T, int V, int NV, int F>
__global__ void __launch_bounds__(512) joint_backward_kernel(const PsgdJoint j, const JointPlan p, float* part) {
  constexpr bool REG = V * NV <= 8;
  const bool post = F & F_RUNTIME ? j.post : bool(F & F_POST);
  const bool gate = F & F_RUNTIME ? j.gate != nullptr : bool(F & F_GATE);
  const bool layer = F & F_RUNTIME ? j.kind == PSGD_NORM_LAYER : bool(F & F_LAYER);
  extern __shared__ float4 smem4[];
  __shared__ float red[2 * JOINT_MAX_GROUPS * JOINT_MAX_WARPS * 2];
  const int d = j.d, dp = (d + 7) & ~7, tpr = blockDim.x, t = threadIdx.x;
  // shared memory: the parameter vectors, or (REG false, where both do not fit) the sums as [slot][V * NV][tpr]
  float* sw = reinterpret_cast<float*>(smem4);
  float* spw = sw + dp;
  float* spb = spw + dp;
  float* slots = sw;
  if (REG) {
    stage_param(sw, j.weight, j.param_dtype, d, 1.f);
    if (post) {
      stage_param(spw, j.post_weight, j.param_dtype, d, 1.f);
      stage_param(spb, j.post_bias, j.param_dtype, d, 0.f);
    }
  }
  float acc[REG ? 5 : 1][REG ? V * NV : 1];
#pragma unroll
  for (int a = 0; a < (REG ? 5 : 1); ++a)
#pragma unroll
    for (int k = 0; k < (REG ? V * NV : 1); ++k) acc[a][k] = 0.f;
  if (!REG)
    for (int i = 0; i < p.slots * V * NV; ++i) slots[(size_t)i * tpr + t] = 0.f;
  __syncthreads();
  auto add = [&](int a, int k, float v) {
    if constexpr (REG) acc[a][k] += v;
    else slots[((size_t)p.slot[a] * (V * NV) + k) * tpr + t] += v;
  };
  auto value = [&](int a, int k) -> float {
    if constexpr (REG) return acc[a][k];
    else return slots[((size_t)p.slot[a] * (V * NV) + k) * tpr + t];
  };
  auto clear = [&](int a, int k) {
    if constexpr (REG) acc[a][k] = 0.f;
    else slots[((size_t)p.slot[a] * (V * NV) + k) * tpr + t] = 0.f;
  };

  const long long unit = (long long)blockIdx.x * blockDim.y + threadIdx.y;
  if (unit >= p.units) return;  // a whole group; nothing below waits for another group
  long long r0, r1;
  if (p.chunks) {
    const long long g = unit / p.chunks, c = unit - g * p.chunks;
    r0 = g * p.per_gate + c * p.per_unit;
    r1 = min(r0 + p.per_unit, (g + 1) * p.per_gate);
  } else {
    r0 = unit * p.per_unit;
    r1 = min(r0 + p.per_unit, j.rows);
  }
  GroupSum<2> sum(red);
  const bool drop = j.threshold != 0;
  const Keep keep(j.seed, j.offset, j.rng, j.threshold);
  const float inv_d = 1.f / (float)d;
  long long g_now = gate ? r0 / p.per_gate : 0, g_end = gate ? (g_now + 1) * p.per_gate : 0;

  for (long long row = r0; row < r1; ++row) {
    const T* pdo = j.d_out ? reinterpret_cast<const T*>(j.d_out) + row * j.ld_d_out : nullptr;
    const T* pdn = j.d_normed ? reinterpret_cast<const T*>(j.d_normed) + row * j.ld_d_normed : nullptr;
    const T* po = reinterpret_cast<const T*>(j.x) + row * j.ld_x;
    const T* py = post || gate ? reinterpret_cast<const T*>(j.y) + row * j.ld_y : nullptr;
    const T* pg = gate ? reinterpret_cast<const T*>(j.gate) + g_now * d : nullptr;
    const float4 st = reinterpret_cast<const float4*>(j.stats)[row];
    float dn[NV * V], o[NV * V], dx[NV * V], y[NV * V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * tpr + t) * V;
#pragma unroll
      for (int k = 0; k < V; ++k) dn[i * V + k] = o[i * V + k] = dx[i * V + k] = y[i * V + k] = 0.f;
      if (e < d) {
        if (pdn) load_vec<T, V>(pdn + e, dn + i * V);
        if (pdo) load_vec<T, V>(pdo + e, dx + i * V);
        load_vec<T, V>(po + e, o + i * V);
        if (post || gate) load_vec<T, V>(py + e, y + i * V);
      }
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * tpr + t) * V;
      if (e >= d) continue;
      float w[V];
      if constexpr (REG) load_smem<V>(sw + e, w);
      else load_param<V>(j.weight, j.param_dtype, e, 1.f, w);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int n = i * V + k;
        const float hat = (o[n] - st.z) * st.w;
        add(0, n, dn[n] * hat);
        if (layer) add(1, n, dn[n]);
        const float dh = dn[n] * w[k];
        o[n] = hat;
        dn[n] = dh;
        s[0] += dh * hat;
        s[1] += dh;
      }
    }
    sum(s);
    const float c1 = s[0] * inv_d, c2 = layer ? s[1] * inv_d : 0.f;
    s[0] = s[1] = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * tpr + t) * V;
      if (e >= d) continue;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int n = i * V + k;
        dx[n] += st.w * (dn[n] - o[n] * c1 - c2);
      }
      store_vec<T, V>(reinterpret_cast<T*>(j.dx) + row * d + e, dx + i * V);
      uint32_t m = 0xFFu;
      if (drop) {
        const unsigned long long at = (unsigned long long)row * d + e;
        m = V == 8 ? keep.mask8(at >> 3) : (uint32_t)keep.one(at);
      }
      float w[V], b[V], g[V];
      if (post) {
        if constexpr (REG) {
          load_smem<V>(spw + e, w);
          load_smem<V>(spb + e, b);
        } else {
          load_param<V>(j.post_weight, j.param_dtype, e, 1.f, w);
          load_param<V>(j.post_bias, j.param_dtype, e, 0.f, b);
        }
      }
      if (gate) load_vec<T, V>(pg + e, g);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int n = i * V + k;
        const bool kept = (m >> k) & 1u;
        float du = j.scale * dx[n];
        if (post) y[n] = (y[n] - st.x) * st.y;
        if (gate) {
          const float u = post ? y[n] * w[k] + b[k] : y[n];
          add(4, n, kept ? du * (u * j.keep_scale) : 0.f);
          du *= g[k];
        }
        du = kept ? du * j.keep_scale : 0.f;
        if (post) {
          add(2, n, du * y[n]);
          if (layer) add(3, n, du);
          du *= w[k];
          s[0] += du * y[n];
          s[1] += du;
        }
        dx[n] = du;
      }
      if (!post) store_vec<T, V>(reinterpret_cast<T*>(j.dy) + row * d + e, dx + i * V);
    }
    if (post) {
      sum(s);
      const float c3 = s[0] * inv_d, c4 = layer ? s[1] * inv_d : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (i * tpr + t) * V;
        if (e >= d) continue;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const int n = i * V + k;
          dx[n] = st.y * (dx[n] - y[n] * c3 - c4);
        }
        store_vec<T, V>(reinterpret_cast<T*>(j.dy) + row * d + e, dx + i * V);
      }
    }
    if (gate && row + 1 == g_end && !p.chunks) {  // the gate group ends here, and with it its gradient
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int e = (i * tpr + t) * V;
        if (e >= d) continue;
        float v[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          v[k] = value(4, i * V + k);
          clear(4, i * V + k);
        }
        store_vec<T, V>(reinterpret_cast<T*>(j.dgate) + g_now * d + e, v);
      }
      ++g_now;
      g_end += p.per_gate;
    }
  }
#pragma unroll
  for (int a = 0; a < 5; ++a) {
    if (p.slot[a] < 0 || (a == 4 && !p.chunks)) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e = (i * tpr + t) * V;
      if (e >= d) continue;
      float v[V];
#pragma unroll
      for (int k = 0; k < V; ++k) v[k] = value(a, i * V + k);
      store_vec<float, V>(part + ((size_t)p.slot[a] * p.units + unit) * dp + e, v);
    }
  }
}

// Sums of the units' rows in a fixed order: 32 columns a block, 8 threads a column, each over every eighth row.
// blockIdx.y: the four parameter vectors, then one gate group each.
__global__ void __launch_bounds__(256) joint_reduce_kernel(const PsgdJoint j, const JointPlan p, const float* part) {
  __shared__ float red[8][33];
  const int dp = (j.d + 7) & ~7, col = blockIdx.x * 32 + threadIdx.x;
  const int a = blockIdx.y < 4 ? (int)blockIdx.y : 4;
  if (p.slot[a] < 0) return;
  long long u0 = 0, u1 = p.units, at = col;
  void* out[4] = {j.dweight, j.dbias, j.dpost_weight, j.dpost_bias};
  if (a == 4) {
    const long long g = (long long)blockIdx.y - 4;
    u0 = g * p.chunks;
    u1 = u0 + p.chunks;
    at = g * j.d + col;
  }
  float s = 0.f;
  if (col < j.d)
    for (long long u = u0 + threadIdx.y; u < u1; u += 8) s += part[((size_t)p.slot[a] * p.units + u) * dp + col];
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && col < j.d) {
#pragma unroll
    for (int k = 1; k < 8; ++k) s += red[k][threadIdx.x];
    if (a < 4) store_any(out[a], j.param_dtype, at, s);
    else store_any(j.dgate, j.dtype, at, s);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
int size_of(int dtype) { return dtype == PSGD_F32 ? 4 : 2; }

bool rows_aligned(const void* p, long long ld, int dtype) {
  return aligned16(p) && (ld * size_of(dtype)) % 16 == 0;
}

int round_up(int a, int b) { return (a + b - 1) / b * b; }

bool valid(const PsgdJoint& j) {
  if (j.rows < 0 || j.d < 1 || j.d > JOINT_MAX_D || j.dtype < 0 || j.dtype > 2) return false;
  if (j.param_dtype < 0 || j.param_dtype > 2 || (j.kind != PSGD_NORM_RMS && j.kind != PSGD_NORM_LAYER)) return false;
  if (j.threshold > 65536u || (j.gate && (j.gates < 1 || j.rows % j.gates))) return false;
  return true;
}

// The block's shape: a group of up to 512 threads, as many groups as fill a block of JOINT_THREADS.
void shape(int d, bool vec, int nv_wide, int& tpr, int& groups, int& nv) {
  const int v = vec ? 8 : 1, units = (d + v - 1) / v;
  tpr = units >= 512 ? 512 : round_up(units, 32);
  nv = (units + tpr - 1) / tpr;
  if (vec) nv = nv <= 1 ? 1 : nv_wide;
  else nv = nv <= 2 ? 2 : 16;
  groups = JOINT_THREADS / tpr;
  groups = groups < 1 ? 1 : groups > JOINT_MAX_GROUPS ? JOINT_MAX_GROUPS : groups;
}

// Dynamic shared memory beyond the 48 KB that dynamic and static shared memory have without asking. A refusal is cleared:
// it would be taken for the next launch's.
template <typename K>
int allow_smem(K kernel, int smem) {
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return PSGD_ELAUNCH;
  }
  return PSGD_OK;
}
template <typename K>
int resident(K kernel, int threads, int smem, int& per_sm) {
  if (int rc = allow_smem(kernel, smem)) return rc;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem) != cudaSuccess) {
    cudaGetLastError();
    return PSGD_ELAUNCH;
  }
  if (per_sm < 1) per_sm = 1;
  return PSGD_OK;
}

template <typename T, int V, int NV>
int forward(const PsgdJoint& j, int tpr, int groups, cudaStream_t stream) {
  const int dp = round_up(j.d, 8), smem = (j.post ? 4 : 2) * dp * 4;
  auto k = joint_forward_kernel<T, V, NV>;
  int per_sm = 1;
  if (int rc = resident(k, tpr * groups, smem, per_sm)) return rc;
  const long long want = (j.rows + groups - 1) / groups, most = (long long)per_sm * psgd_num_sms();
  k<<<(int)(want < most ? want : most), dim3(tpr, groups), smem, stream>>>(j);
  return cudaGetLastError() == cudaSuccess ? PSGD_OK : PSGD_ELAUNCH;
}

template <typename T>
int forward_typed(const PsgdJoint& j, cudaStream_t stream) {
  const bool vec = j.d % 8 == 0 && rows_aligned(j.x, j.ld_x, j.dtype) && rows_aligned(j.y, j.ld_y, j.dtype) &&
                   rows_aligned(j.out, j.d, j.dtype) && rows_aligned(j.normed, j.d, j.dtype) &&
                   (!j.gate || rows_aligned(j.gate, j.d, j.dtype));
  int tpr, groups, nv;
  shape(j.d, vec, 2, tpr, groups, nv);
  if (vec) return nv == 1 ? forward<T, 8, 1>(j, tpr, groups, stream) : forward<T, 8, 2>(j, tpr, groups, stream);
  return nv == 2 ? forward<T, 1, 2>(j, tpr, groups, stream) : forward<T, 1, 16>(j, tpr, groups, stream);
}

// The plan of a backward pass; the same from a size query and from the launch.
JointPlan plan_backward(const PsgdJoint& j) {
  JointPlan p = {};
  bool vec = j.d % 8 == 0 && rows_aligned(j.x, j.ld_x, j.dtype) && rows_aligned(j.dx, j.d, j.dtype) &&
             rows_aligned(j.dy, j.d, j.dtype) && (!j.d_out || rows_aligned(j.d_out, j.ld_d_out, j.dtype)) &&
             (!j.d_normed || rows_aligned(j.d_normed, j.ld_d_normed, j.dtype)) &&
             (!(j.post || j.gate) || rows_aligned(j.y, j.ld_y, j.dtype)) &&
             (!j.gate || (rows_aligned(j.gate, j.d, j.dtype) && rows_aligned(j.dgate, j.d, j.dtype)));
  p.vec = vec;
  shape(j.d, vec, 2, p.tpr, p.groups, p.nv);
  const bool reg = (vec ? 8 : 1) * p.nv <= 8;
  const bool layer = j.kind == PSGD_NORM_LAYER;
  const bool there[5] = {true, layer, j.post != 0, j.post && layer, j.gate != nullptr};
  for (int a = 0; a < 5; ++a) p.slot[a] = there[a] ? p.slots++ : -1;
  if (!reg) p.groups = 1;
  const int dp = round_up(j.d, 8);
  p.smem = reg ? 3 * dp * 4 : p.slots * (vec ? 8 : 1) * p.nv * p.tpr * 4;
  int per_sm = 1024 / (p.tpr * p.groups);
  if (per_sm < 1) per_sm = 1;
  if (per_sm * p.smem > 200 * 1024) per_sm = 200 * 1024 / p.smem < 1 ? 1 : 200 * 1024 / p.smem;
  const long long most = (long long)psgd_num_sms() * per_sm * p.groups;
  p.per_unit = (j.rows + most - 1) / most;
  p.per_gate = 1;
  if (j.gate) {
    p.per_gate = j.rows / j.gates;
    if (p.per_gate <= p.per_unit) {
      p.per_unit = (p.per_unit + p.per_gate - 1) / p.per_gate * p.per_gate;
    } else {
      p.chunks = (p.per_gate + p.per_unit - 1) / p.per_unit;
      p.per_unit = (p.per_gate + p.chunks - 1) / p.chunks;
    }
  }
  p.units = p.chunks ? j.gates * p.chunks : (j.rows + p.per_unit - 1) / p.per_unit;
  p.grid = (int)((p.units + p.groups - 1) / p.groups);
  return p;
}

template <typename T, int V, int NV, int F>
int backward(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream) {
  auto k = joint_backward_kernel<T, V, NV, F>;
  if (int rc = allow_smem(k, p.smem)) return rc;
  k<<<p.grid, dim3(p.tpr, p.groups), p.smem, stream>>>(j, p, part);
  if (cudaGetLastError() != cudaSuccess) return PSGD_ELAUNCH;
  const dim3 grid((j.d + 31) / 32, 4 + (p.chunks ? (int)j.gates : 0));
  joint_reduce_kernel<<<grid, dim3(32, 8), 0, stream>>>(j, p, part);
  return cudaGetLastError() == cudaSuccess ? PSGD_OK : PSGD_ELAUNCH;
}

template <typename T>
int backward_typed(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream) {
  if (p.vec && p.nv == 1) {
    const int f = (j.post ? F_POST : 0) | (j.gate ? F_GATE : 0) | (j.kind == PSGD_NORM_LAYER ? F_LAYER : 0);
    switch (f) {
      case 0: return backward<T, 8, 1, 0>(j, p, part, stream);
      case 1: return backward<T, 8, 1, 1>(j, p, part, stream);
      case 2: return backward<T, 8, 1, 2>(j, p, part, stream);
      case 3: return backward<T, 8, 1, 3>(j, p, part, stream);
      case 4: return backward<T, 8, 1, 4>(j, p, part, stream);
      case 5: return backward<T, 8, 1, 5>(j, p, part, stream);
      case 6: return backward<T, 8, 1, 6>(j, p, part, stream);
      default: return backward<T, 8, 1, 7>(j, p, part, stream);
    }
  }
  if (p.vec) return backward<T, 8, 2, F_RUNTIME>(j, p, part, stream);
  return p.nv == 2 ? backward<T, 1, 2, F_RUNTIME>(j, p, part, stream) : backward<T, 1, 16, F_RUNTIME>(j, p, part, stream);
}

}  // namespace
}  // namespace psgd

extern "C" int psgd_joint_forward(const PsgdJoint* j, cudaStream_t stream) {
  using namespace psgd;
  if (!j || !valid(*j)) return PSGD_EINVAL;
  if (j->rows == 0) return PSGD_OK;
  if (!j->x || !j->y || !j->out || !j->normed || !j->stats || !aligned16(j->stats)) return PSGD_EINVAL;
  switch (j->dtype) {
    case PSGD_F32: return forward_typed<float>(*j, stream);
    case PSGD_BF16: return forward_typed<__nv_bfloat16>(*j, stream);
    default: return forward_typed<__half>(*j, stream);
  }
}

extern "C" long long psgd_joint_workspace(const PsgdJoint* j) {
  using namespace psgd;
  if (!j || !valid(*j)) return PSGD_EINVAL;
  if (j->rows == 0) return 0;
  const JointPlan p = plan_backward(*j);
  return (long long)p.slots * p.units * round_up(j->d, 8) * 4;
}

extern "C" int psgd_joint_backward(const PsgdJoint* j, void* workspace, long long bytes, cudaStream_t stream) {
  using namespace psgd;
  if (!j || !valid(*j)) return PSGD_EINVAL;
  if (j->rows == 0) return PSGD_OK;
  const JointPlan p = plan_backward(*j);
  if (!j->x || !j->stats || !aligned16(j->stats) || !j->dx || !j->dy || !j->dweight || !workspace || !aligned16(workspace))
    return PSGD_EINVAL;
  if (((j->post || j->gate) && !j->y) || (p.slot[1] >= 0 && !j->dbias) || (p.slot[2] >= 0 && !j->dpost_weight) ||
      (p.slot[3] >= 0 && !j->dpost_bias) || (p.slot[4] >= 0 && !j->dgate))
    return PSGD_EINVAL;
  if (p.chunks && j->gates > 65000) return PSGD_EINVAL;
  if (bytes < psgd_joint_workspace(j)) return PSGD_ESPACE;
  float* part = reinterpret_cast<float*>(workspace);
  switch (j->dtype) {
    case PSGD_F32: return backward_typed<float>(*j, p, part, stream);
    case PSGD_BF16: return backward_typed<__nv_bfloat16>(*j, p, part, stream);
    default: return backward_typed<__half>(*j, p, part, stream);
  }
}
