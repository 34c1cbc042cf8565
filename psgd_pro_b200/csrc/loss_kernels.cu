// Softmax cross entropy of a linear head, loss and gradients, without keeping the logits:
//   l = h w^T;  lse = log sum_v exp l_v;  loss = lse - (1 - s) l_t - s mean_v l_v + z lse^2
//   g = c [ (1 + 2 z lse) p - (1 - s) 1[v = t] - s / V ],  p = exp(l - lse);  dh = g w;  dw = g^T h
// for the rows whose target counts. The steps, each one launch:
//   plan     numbers the counted rows (the others cost nothing below, and no value of theirs is read again);
//   stage    gathers their rows of h as tensor-core operands (fp32: three bf16 limbs); zeros the other rows of dh;
//   logits   tile by tile on the tensor cores; the epilogue keeps, per row and 256 columns of the vocabulary, the
//            maximum m and sum of exp(l - m) in fp32 and, for gradients, exp(l - m) itself in 16 bits;
//   rows     joins those statistics to lse and the loss, and turns exp(l - m) into g in place;
//   grads    dh = g w and dw = g^T h as one list of tiles (w, g and h are read in the orientation they have, by
//            MN-major operand descriptors: nothing is transposed in memory).
// One pass over the vocabulary with kept exponentials costs 6 N V D operations; forming the logits again for the
// gradients, the alternative that keeps nothing, costs 8 N V D. What is kept is bounded: tokens are taken in pieces.
#include "elem.cuh"

#include <float.h>

namespace psgd {
namespace {

constexpr int LM = 128, LN = 256, LK = 64, L_STAGES = 4, L_THREADS = 192;
constexpr int L_A_BYTES = LM * LK * 2, L_B_BYTES = LN * LK * 2, L_STAGE_BYTES = L_A_BYTES + L_B_BYTES;
constexpr int L_SMEM = 1024 + L_STAGES * L_STAGE_BYTES + 256;
constexpr int L_LIMBS = 3;          // of an fp32 operand
constexpr int L_GROUP_M = 8;        // row tiles that walk the column tiles together (L2 reuse of both operands)
// Kept exponentials are fp16 of 2^15 exp(l - m), exp(l - m) in [0, 1]: 11 significant bits down to 2^-29 of the row's
// maximum in these 256 columns, so that the one rounding to 16 bits that matters is that of g.
constexpr float L_KEEP_SCALE = 32768.f;
// g is held times 2^8 when it is fp16: p below 2^-14 keeps its bits down to 2^-22 and |g| may reach 255.
constexpr float L_HALF_SCALE = 256.f;

struct LceState {  // device scalars of one call
  int counted;
  float alpha;     // factor of both gradients
  float row_unit;  // per-row upstream gradients are divided by this
};

// ---- plan ------------------------------------------------------------------------------------------------------------
// One block: thread k owns the targets [k * per, (k + 1) * per); a scan of the threads' counts numbers the counted rows in
// their order.
__global__ void __launch_bounds__(1024) lce_plan_kernel(const long long* __restrict__ target, int n, int v,
                                                        long long ignore, int reduction, int half,
                                                        const float* __restrict__ grad, int* __restrict__ rank,
                                                        int* __restrict__ row_of, int* __restrict__ row_target,
                                                        float* __restrict__ loss, LceState* state, int* err) {
  __shared__ int counts[32];
  __shared__ float tops[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5, per = (n + 1023) / 1024;
  const int a = min(n, t * per), b = min(n, a + per);
  int mine = 0;
  float top = 0.f;
  bool bad = false;
  for (int i = a; i < b; ++i) {
    const long long x = target[i];
    if (x == ignore) continue;
    if (x < 0 || x >= v) {
      bad = true;
      continue;
    }
    ++mine;
    if (reduction == PSGD_REDUCE_NONE && grad) top = fmaxf(top, fabsf(grad[i]));
  }
  int before = mine;  // inclusive scan
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += up;
  }
  top = warp_max(top);
  if (lane == 31) counts[warp] = before;
  if (lane == 0) tops[warp] = top;
  if (bad) atomicOr(err, ERR_BAD_TARGET);
  __syncthreads();
  int base = 0, total = 0;
  for (int w = 0; w < 32; ++w) {
    if (w < warp) base += counts[w];
    total += counts[w];
    top = fmaxf(top, tops[w]);
  }
  int r = base + before - mine;
  for (int i = a; i < b; ++i) {
    const long long x = target[i];
    const bool counted = x != ignore && x >= 0 && x < v;
    if (rank) rank[i] = counted ? r : -1;
    if (counted) {
      row_of[r] = i;
      row_target[r] = (int)x;
      ++r;
    } else if (reduction == PSGD_REDUCE_NONE) {
      loss[i] = 0.f;
    }
  }
  if (t == 0) {
    state->counted = total;
    // fp16 gradients: per-row upstream values are taken relative to the largest, so that g stays in range
    const float unit = half && reduction == PSGD_REDUCE_NONE && grad && top > 0.f ? top : 1.f;
    state->row_unit = unit;
    float alpha = half ? unit / L_HALF_SCALE : 1.f;
    if (reduction != PSGD_REDUCE_NONE && grad) alpha *= *grad;
    if (reduction == PSGD_REDUCE_MEAN) alpha /= (float)max(total, 1);
    state->alpha = alpha;
  }
}

// ---- stage -----------------------------------------------------------------------------------------------------------
PSGD_DEVI void limbs3(float x, float* l) {
  l[0] = __bfloat162float(__float2bfloat16_rn(x));
  const bool fine = fabsf(l[0]) <= FLT_MAX;  // an infinity or NaN is its first limb
  const float r = fine ? x - l[0] : 0.f;
  l[1] = __bfloat162float(__float2bfloat16_rn(r));
  l[2] = r - l[1];
}

// Row i of src (n rows of d) to row rank[i] (i without a rank) of the operand: itself, or its bf16 limbs `plane`
// elements apart. Rows without a rank zero their row of dh instead. The 64 threads groups beyond n zero the operand's
// rows from the count to the next multiple of 64, which a reduction over rows reads.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) lce_stage_kernel(const T* __restrict__ src, long long ld, int n, int d,
                                                        const int* __restrict__ rank, const LceState* state,
                                                        uint16_t* __restrict__ out, long long ld_out, long long plane,
                                                        T* __restrict__ dh) {
  constexpr int V = VEC ? 8 : 1;
  const int lane = threadIdx.x & 31;
  const long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= (long long)n + (rank ? 64 : 0)) return;
  long long r = i;
  if (i >= n) {
    r = state->counted + (i - n);
    if (r >= ((state->counted + 63) & ~63)) return;
  } else if (rank) {
    r = rank[i];
  }
  if (r < 0) {
    if (dh)
      for (int e = lane * V; e < d; e += 32 * V) {
        const float zero[8] = {};
        store_vec<T, V>(dh + i * d + e, zero);
      }
    return;
  }
  for (int e = lane * V; e < d; e += 32 * V) {
    if constexpr (sizeof(T) == 2) {
      T* to = reinterpret_cast<T*>(out) + r * ld_out + e;
      if constexpr (VEC) {
        *reinterpret_cast<uint4*>(to) = i < n ? *reinterpret_cast<const uint4*>(src + i * ld + e) : make_uint4(0, 0, 0, 0);
      } else {
        *to = i < n ? src[i * ld + e] : from_f32<T>(0.f);
      }
    } else {
      float x[V], l[3][V];
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] = 0.f;
      if (i < n) load_vec<T, V>(src + i * ld + e, x);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float p[3];
        limbs3(x[k], p);
        l[0][k] = p[0], l[1][k] = p[1], l[2][k] = p[2];
      }
#pragma unroll
      for (int q = 0; q < 3; ++q)
        store_vec<__nv_bfloat16, V>(reinterpret_cast<__nv_bfloat16*>(out) + q * plane + r * ld_out + e, l[q]);
    }
  }
}

// ---- the products ----------------------------------------------------------------------------------------------------
// D (M x N) = A B^T over K, in `nseg` passes over K that take the limbs segs[i] = (limb of A) | (limb of B) << 4 in turn.
// An operand is K-major (rows of M or N, K contiguous) or MN-major (rows of K, M or N contiguous: *_mn).
struct LceProblem {
  CUtensorMap ta[L_LIMBS], tb[L_LIMBS];
  int a_mn, b_mn, nseg;
  uint8_t segs[8];
  int M, N, K;    // bounds; the counted rows replace M (dyn 1) or K (dyn 2)
  int dyn, row0;  // first counted row of this piece
  int splits;     // K blocks are dealt to this many units of a tile, whose sums go to `part`
  // outputs of a gradient tile: rows through row_of (or as they are)
  const int* row_of;
  void* out;
  long long ld_out;
  float* part;       // splits > 1: [split][M][N], joined by lce_join_kernel
  const float* acc;  // earlier pieces' sums, added
  float* acc_out;    // sums so far, fp32, instead of out
};
struct LceShape {
  int M, K, tiles_m, tiles_n, kblocks, units;
};
PSGD_DEVI LceShape lce_shape(const LceProblem& p, const LceState* state) {
  LceShape s;
  const int there = max(0, state->counted - p.row0);
  s.M = p.dyn == 1 ? min(p.M, there) : p.M;
  s.K = p.dyn == 2 ? min(p.K, there) : p.K;
  s.tiles_m = (s.M + LM - 1) / LM;
  s.tiles_n = (p.N + LN - 1) / LN;
  s.kblocks = (s.K + LK - 1) / LK;
  s.units = s.tiles_m * s.tiles_n * p.splits;
  return s;
}
struct LceUnit {
  int tm, tn, k0, k1, split;
};
PSGD_DEVI LceUnit lce_unit(const LceProblem& p, const LceShape& s, int u) {
  LceUnit x;
  const int tiles = s.tiles_m * s.tiles_n;
  x.split = u / tiles;
  const int t = u - x.split * tiles;
  const int band = t / (L_GROUP_M * s.tiles_n), m0 = band * L_GROUP_M, h = min(L_GROUP_M, s.tiles_m - m0);
  const int in = t - band * L_GROUP_M * s.tiles_n;
  x.tn = in / h;
  x.tm = m0 + in - x.tn * h;
  x.k0 = (int)((long long)s.kblocks * x.split / p.splits);
  x.k1 = (int)((long long)s.kblocks * (x.split + 1) / p.splits);
  return x;
}

struct LceLogits {  // what the logits' epilogue keeps
  float2* stats;  // [row][column tile]: (maximum, sum of exp)
  float* linear;  // [row][column tile]: sum of the logits (label smoothing), or NULL
  float* target_logit;
  const int* row_target;
  void* kept;  // exp(l - m), [row][ld_kept], or NULL
  long long ld_kept;
};

struct __align__(64) LceArgs {
  LceProblem p[2];
  int nproblems;
  LceLogits logits;
  const LceState* state;
  int* err;
  unsigned long long wait_ns;
};

PSGD_DEVI uint64_t lce_desc(uint32_t saddr, bool mn) {
  // K-major: 128-byte rows, 8-row swizzle atoms 1024 bytes apart. MN-major: atoms of 64 (M or N) x 8 (K), 1024 bytes
  // apart along K; the next 64 of M or N are one 64 x 64 box (8192 bytes) on.
  uint64_t d = sdesc_k_sw128(saddr);
  if (mn) d = (d & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(8192 >> 4) << 16);
  return d;
}
template <typename T>
PSGD_DEVI uint32_t lce_idesc(bool a_mn, bool b_mn) {
  const uint32_t fmt = sizeof(T) == 2 && !is_half<T>() ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(LN >> 3) << 17) | ((uint32_t)(LM >> 4) << 24);
}

constexpr float LOG2E = 1.4426950408889634f;
PSGD_DEVI float exp_fast(float x) {  // exp of x <= 0 (or NaN); x log2 e is rounded to fp32: relative error 6e-8 |x| + 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * LOG2E));
  return y;
}

// The logits' epilogue for one row of a tile (thread = row).
template <typename KT>
PSGD_DEVI void logits_row(const LceProblem& p, const LceShape& sh, const LceLogits& g, const LceUnit& u, uint32_t tacc,
                          int row_in_tile) {
  constexpr bool WIDE = sizeof(KT) == 4;
  const long long row = (long long)u.tm * LM + row_in_tile;
  const bool live = row < sh.M;
  const int n0 = u.tn * LN, width = min(LN, p.N - n0);
  float top = -INFINITY, linear = 0.f;
  const int at = live ? g.row_target[p.row0 + row] - n0 : -1;
  for (int c = 0; c < LN; c += 32) {
    if (c >= width) break;
    float v[32];
    tmem_ld32(tacc + (uint32_t)c, v);
    if (c + 32 <= width) {
#pragma unroll
      for (int k = 0; k < 32; ++k) top = fmaxf(top, v[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 32; ++k)
        if (c + k < width) top = fmaxf(top, v[k]);
    }
    if (g.linear)
#pragma unroll
      for (int k = 0; k < 32; ++k) linear += c + k < width ? v[k] : 0.f;
    const bool here = at >= c && at < c + 32;
    if (__any_sync(0xffffffffu, here)) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < 32; ++k) x = at == c + k ? v[k] : x;
      if (here) g.target_logit[row] = x;
    }
  }
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  KT* kept = g.kept ? reinterpret_cast<KT*>(g.kept) + row * g.ld_kept + n0 : nullptr;
  for (int c = 0; c < LN; c += 32) {
    if (c >= width) break;
    float v[32];
    tmem_ld32(tacc + (uint32_t)c, v);
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      v[k] = WIDE ? expf(v[k] - ref) : exp_fast(v[k] - ref);
      if (c + k >= width) v[k] = 0.f;
      sum += v[k];
      if (!WIDE) v[k] *= L_KEEP_SCALE;
    }
    if (kept && live)
#pragma unroll
      for (int k = 0; k < 32; k += 8) store_vec<KT, 8>(kept + c + k, v + k);
  }
  if (live) {
    g.stats[row * sh.tiles_n + u.tn] = make_float2(top, sum);
    if (g.linear) g.linear[row * sh.tiles_n + u.tn] = linear;
  }
}

// The gradients' epilogue for one row of a tile.
template <typename T>
PSGD_DEVI void grad_row(const LceProblem& p, const LceShape& sh, const LceUnit& u, uint32_t tacc, int row_in_tile,
                        float alpha) {
  const long long row = (long long)u.tm * LM + row_in_tile;
  const bool live = row < sh.M, zero = u.k0 >= u.k1;
  const int n0 = u.tn * LN, width = min(LN, p.N - n0);
  const long long to = live ? (p.row_of ? p.row_of[p.row0 + row] : row) : 0;
  const bool vec = p.ld_out % 8 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
  const bool vec4 = p.N % 4 == 0;
  for (int c = 0; c < LN; c += 32) {
    if (c >= width) break;
    float v[32];
    tmem_ld32(tacc + (uint32_t)c, v);
    if (!live) continue;
    if (zero)
#pragma unroll
      for (int k = 0; k < 32; ++k) v[k] = 0.f;
    const int w = min(32, width - c);
    const long long flat = row * p.N + n0 + c;
    if (p.acc) {
#pragma unroll
      for (int k = 0; k < 32; ++k)
        if (k < w) v[k] += p.acc[flat + k];
    }
    float* wide = p.part ? p.part + (long long)u.split * p.M * p.N + flat : p.acc_out ? p.acc_out + flat : nullptr;
    if (wide) {
      if (vec4 && w == 32) {
#pragma unroll
        for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4*>(wide + k) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
      } else {
#pragma unroll
        for (int k = 0; k < 32; ++k)
          if (k < w) wide[k] = v[k];
      }
      continue;
    }
#pragma unroll
    for (int k = 0; k < 32; ++k) v[k] *= alpha;
    T* out = reinterpret_cast<T*>(p.out) + to * p.ld_out + n0 + c;
    if (vec && w == 32) {
#pragma unroll
      for (int k = 0; k < 32; k += 8) store_vec<T, 8>(out + k, v + k);
    } else {
#pragma unroll
      for (int k = 0; k < 32; ++k)
        if (k < w) out[k] = from_f32<T>(v[k]);
    }
  }
}

// OP: operand type of the tensor cores; OUT: logits (float: kept exponentials in fp32, __half: in fp16) or gradients of
// type OUT. Warp 0 copies tiles, warp 1 issues the products, warps 2..5 take the accumulators (two, in turn).
template <typename OP, typename OUT, bool LOGITS>
__global__ void __launch_bounds__(L_THREADS, 1) lce_product_kernel(const __grid_constant__ LceArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L_STAGES * L_STAGE_BYTES);
  uint64_t* empty = full + L_STAGES;
  uint64_t* tfull = empty + L_STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const LceShape s0 = lce_shape(args.p[0], args.state);
  const LceShape s1 = args.nproblems > 1 ? lce_shape(args.p[1], args.state) : LceShape{};
  const int units = s0.units + (args.nproblems > 1 ? s1.units : 0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < L_STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 4);
    }
    mbar_init(drain, 1);
    *abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    __syncwarp();
    tmem_alloc(tmem_slot, 2 * LN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, rounds = 0;
      for (int x = blockIdx.x; x < units && !*abort; x += gridDim.x) {
        const LceProblem& p = args.p[x >= s0.units];
        const LceShape& sh = x >= s0.units ? s1 : s0;
        const LceUnit u = lce_unit(p, sh, x >= s0.units ? x - s0.units : x);
        for (int seg = 0; seg < p.nseg && !*abort; ++seg) {
          const CUtensorMap* ta = &p.ta[p.segs[seg] & 15];
          const CUtensorMap* tb = &p.tb[p.segs[seg] >> 4];
          for (int k = u.k0; k < u.k1; ++k) {
            if (!mbar_wait_for(&empty[s], ph ^ 1, abort, args.wait_ns)) break;
            mbar_arrive_expect_tx(&full[s], L_STAGE_BYTES);
            ++rounds;
            uint8_t* sa = smem + s * L_STAGE_BYTES;
            uint8_t* sb = sa + L_A_BYTES;
            if (p.a_mn) {
              for (int i = 0; i < LM / 64; ++i) tma_load_2d(sa + i * 8192, ta, &full[s], u.tm * LM + i * 64, k * LK);
            } else {
              tma_load_2d(sa, ta, &full[s], k * LK, u.tm * LM);
            }
            if (p.b_mn) {
              for (int i = 0; i < LN / 64; ++i) tma_load_2d(sb + i * 8192, tb, &full[s], u.tn * LN + i * 64, k * LK);
            } else {
              tma_load_2d(sb, tb, &full[s], k * LK, u.tn * LN);
            }
            if (++s == L_STAGES) s = 0, ph ^= 1;
          }
        }
      }
      if (*abort) {  // copies in flight land before shared memory is released: the last round of each stage that had one
        for (int i = 0; i < L_STAGES; ++i) {
          const uint32_t n = rounds / L_STAGES + ((uint32_t)i < rounds % L_STAGES);
          volatile int never = 0;
          if (n) mbar_wait(&full[i], (n - 1) & 1, &never);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0, i = 0;
      bool issued = false;
      for (int x = blockIdx.x; x < units; x += gridDim.x, ++i) {
        const LceProblem& p = args.p[x >= s0.units];
        const LceShape& sh = x >= s0.units ? s1 : s0;
        const LceUnit u = lce_unit(p, sh, x >= s0.units ? x - s0.units : x);
        const uint32_t acc = i & 1, aph = (i >> 1) & 1;
        if (!mbar_wait_for(&tempty[acc], aph ^ 1, abort, args.wait_ns)) break;
        tc_fence_after();
        const uint32_t idesc = lce_idesc<OP>(p.a_mn, p.b_mn);
        const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = p.b_mn ? 2048 : 32;  // 16 of K, in bytes
        uint32_t first = 0;
        bool ok = true;
        for (int seg = 0; seg < p.nseg && ok; ++seg)
          for (int k = u.k0; k < u.k1; ++k) {
            if (!mbar_wait_for(&full[s], ph, abort, args.wait_ns)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t sa = smem_u32(smem + s * L_STAGE_BYTES), sb = sa + L_A_BYTES;
#pragma unroll
            for (int kk = 0; kk < LK / 16; ++kk) {
              umma_bf16(tmem_base + acc * LN, lce_desc(sa + kk * a_step, p.a_mn), lce_desc(sb + kk * b_step, p.b_mn), idesc,
                        first);
              first = 1;
            }
            issued = true;
            umma_commit(&empty[s]);
            if (++s == L_STAGES) s = 0, ph ^= 1;
          }
        if (!ok) break;
        umma_commit(&tfull[acc]);
      }
      if (*abort && issued) {
        umma_commit(drain);
        volatile int never = 0;
        mbar_wait(drain, 0, &never);
      }
    }
  } else {
    const int q = warp & 3;
    uint32_t i = 0;
    const float alpha = args.state->alpha;
    for (int x = blockIdx.x; x < units; x += gridDim.x, ++i) {
      const LceProblem& p = args.p[x >= s0.units];
      const LceShape& sh = x >= s0.units ? s1 : s0;
      const LceUnit u = lce_unit(p, sh, x >= s0.units ? x - s0.units : x);
      const uint32_t acc = i & 1, aph = (i >> 1) & 1;
      const bool ok = __all_sync(0xffffffffu, mbar_wait_for(&tfull[acc], aph, abort, args.wait_ns));
      if (!ok) break;
      tc_fence_after();
      const uint32_t tacc = tmem_base + ((uint32_t)(q * 32) << 16) + acc * LN;
      if constexpr (LOGITS) logits_row<OUT>(p, sh, args.logits, u, tacc, q * 32 + lane);
      else grad_row<OUT>(p, sh, u, tacc, q * 32 + lane, alpha);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem_base, 2 * LN);
  }
  if (threadIdx.x == 0 && *abort) atomicOr(args.err, ERR_TIMEOUT_FULL);
}

// ---- rows ------------------------------------------------------------------------------------------------------------
PSGD_DEVI float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v += red[w];
  return v;
}
PSGD_DEVI float block_max(float v, float* red) {
  v = warp_max(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int w = 0; w < (int)(blockDim.x >> 5); ++w) v = fmaxf(v, red[w]);
  return v;
}

struct LceRows {
  const float2* stats;
  const float* linear;
  const float* target_logit;
  const int* row_target;
  const int* row_of;
  const float* grad;  // per-row upstream gradients, or NULL
  float* loss_rows;   // [counted row] (reduction mean, sum)
  float* loss;        // [row] (reduction none)
  void* kept;         // in: exp(l - m); 16-bit g in its place
  uint16_t* limbs;    // fp32: g as three bf16 limbs `plane` apart
  long long ld_kept, plane;
  int v, tiles, row0, rows, none;
  float smoothing, z;
};

// One block a row (and 1 / gridDim.y of its columns). KT / GT: types of the kept exponentials and of g.
template <typename KT, typename GT>
__global__ void __launch_bounds__(256) lce_rows_kernel(const LceRows a, const LceState* state) {
  __shared__ float red[8];
  const int row = blockIdx.x, there = min(a.rows, max(0, state->counted - a.row0));
  KT* kept = reinterpret_cast<KT*>(a.kept) + (a.kept ? row * a.ld_kept : 0);
  const int vecs = (a.v + 7) / 8, per = (vecs + gridDim.y - 1) / gridDim.y;
  const int v0 = blockIdx.y * per, v1 = min(vecs, v0 + per);
  if (row >= there) {  // rows up to the next multiple of 64 enter the reduction over rows: zero
    if (!a.kept || row >= ((there + 63) & ~63)) return;
    const float zero[8] = {};
    for (int i = v0 + threadIdx.x; i < v1; i += 256) {
      if constexpr (sizeof(KT) == 4) {
        for (int q = 0; q < 3; ++q)
          store_vec<__nv_bfloat16, 8>(reinterpret_cast<__nv_bfloat16*>(a.limbs) + q * a.plane + row * a.ld_kept + i * 8, zero);
      } else {
        store_vec<GT, 8>(reinterpret_cast<GT*>(kept) + i * 8, zero);
      }
    }
    return;
  }
  const float2* st = a.stats + (long long)row * a.tiles;
  float top = -INFINITY;
  for (int i = threadIdx.x; i < a.tiles; i += 256) top = fmaxf(top, st[i].x);
  top = block_max(top, red);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, linear = 0.f;
  for (int i = threadIdx.x; i < a.tiles; i += 256) {
    sum += st[i].y * expf(st[i].x - ref);
    if (a.linear) linear += a.linear[(long long)row * a.tiles + i];
  }
  sum = block_sum(sum, red);
  if (a.linear) linear = block_sum(linear, red);
  const float lse = ref + logf(sum), lt = a.target_logit[row];
  const int target = a.row_target[a.row0 + row];
  if (threadIdx.x == 0 && blockIdx.y == 0) {
    float loss = a.smoothing == 0.f ? lse - lt : (1.f - a.smoothing) * (lse - lt) + a.smoothing * (lse - linear / (float)a.v);
    if (a.z != 0.f) loss += a.z * lse * lse;
    if (a.none) a.loss[a.row_of[a.row0 + row]] = loss;
    else a.loss_rows[a.row0 + row] = loss;
  }
  if (!a.kept) return;
  constexpr float unit = is_half<GT>() ? L_HALF_SCALE : 1.f;
  const float c = (a.grad ? a.grad[a.row_of[a.row0 + row]] / state->row_unit : 1.f) * unit;
  const float pull = 1.f + 2.f * a.z * lse, uniform = a.smoothing / (float)a.v;
  const float scale = sizeof(KT) == 4 ? 1.f : 1.f / L_KEEP_SCALE;
  // the target's element from its fp32 logit: p - 1 without cancellation
  const float at_target = c * (expm1f(lt - lse) + (pull - 1.f) * expf(lt - lse) + a.smoothing - uniform);
  for (int i = v0 + threadIdx.x; i < v1; i += 256) {
    const float f = expf(st[i * 8 / LN].x - lse) * scale * pull;
    float g[8];
    load_vec<KT, 8>(kept + i * 8, g);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      g[k] = c * (g[k] * f - uniform);
      if (i * 8 + k == target) g[k] = at_target;
    }
    if constexpr (sizeof(KT) == 4) {
      float l[3][8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float p[3];
        limbs3(g[k], p);
        l[0][k] = p[0], l[1][k] = p[1], l[2][k] = p[2];
      }
#pragma unroll
      for (int q = 0; q < 3; ++q)
        store_vec<__nv_bfloat16, 8>(reinterpret_cast<__nv_bfloat16*>(a.limbs) + q * a.plane + row * a.ld_kept + i * 8, l[q]);
    } else {
      store_vec<GT, 8>(reinterpret_cast<GT*>(kept) + i * 8, g);
    }
  }
}

// Sum (or mean) of the counted rows' losses in a fixed order.
__global__ void __launch_bounds__(1024) lce_loss_kernel(const float* __restrict__ rows, const LceState* state, int mean,
                                                        float* loss) {
  __shared__ float red[32];
  const int n = state->counted;
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) s += rows[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) *loss = mean ? s / (float)max(n, 1) : s;
}

// Joins the splits of dh: out[row_of[r]] = alpha * sum over splits, in their order.
template <typename T>
__global__ void __launch_bounds__(256) lce_join_kernel(const float* __restrict__ part, int splits, int M, int N, int row0,
                                                       const int* __restrict__ row_of, T* __restrict__ out,
                                                       const LceState* state) {
  const int there = min(M, max(0, state->counted - row0));
  const long long n = (long long)there * N, plane = (long long)M * N;
  const float alpha = state->alpha;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    float s = 0.f;
    for (int k = 0; k < splits; ++k) s += part[k * plane + i];
    const long long r = i / N;
    out[(long long)row_of[row0 + r] * N + (i - r * N)] = from_f32<T>(s * alpha);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------
typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  return fn;
}

// rows x cols values of 16 bits, `ld` apart, in boxes of 64 columns and box_rows rows, 128-byte swizzled.
int encode(CUtensorMap* m, const void* p, bool half, long long rows, long long cols, long long ld, int box_rows) {
  EncodeFn fn = encode_fn();
  if (!fn) return PSGD_ETMAP;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  cuuint32_t box[2] = {64u, (cuuint32_t)box_rows}, estr[2] = {1u, 1u};
  return fn(m, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims,
            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? PSGD_OK
             : PSGD_ETMAP;
}

// Where everything lies in the workspace; the same from a size query and from the call.
struct Layout {
  int limbs, tiles, piece, pieces, splits;
  bool stage_w;
  long long ld_h, ld_w, ld_kept, h_plane, w_plane, g_plane;
  size_t state, rank, row_of, row_target, loss_rows, target_logit, stats, linear, h, w, kept, g, part, acc, bytes;
};

Layout layout(const PsgdLce& a) {
  Layout l = {};
  const bool wide = a.dtype == PSGD_F32;
  auto up = [](long long x, long long m) { return (x + m - 1) / m * m; };
  l.limbs = wide ? L_LIMBS : 1;
  l.tiles = (a.v + LN - 1) / LN;
  l.ld_h = up(a.d, 8);
  l.ld_w = up(a.d, 8);
  l.ld_kept = up(a.v, 64);
  l.stage_w = wide || a.ld_w % 8 != 0 || !aligned16(a.w);
  // rows of a piece: what is kept for them stays within piece_bytes
  const long long row_bytes = (a.grads ? l.ld_kept * (wide ? 4 + 2 * L_LIMBS : 2) : 0) + (long long)l.tiles * 12;
  long long piece = a.piece_bytes / row_bytes / LM * LM;
  if (piece < LM) piece = LM;
  if (piece > up(a.n, LM)) piece = up(a.n, LM);
  l.piece = (int)piece;
  l.pieces = (int)((a.n + piece - 1) / piece);
  // dh has few tiles and a long reduction over the vocabulary: split it until its units are no longer than an SM's share
  // of the whole launch (dh and dw need the same number of products)
  const long long tiles = (piece / LM) * ((a.d + LN - 1) / LN), kblocks = (a.v + LK - 1) / LK;
  long long splits = (2 * psgd_num_sms() + tiles - 1) / tiles;
  if (splits > kblocks / 8) splits = kblocks / 8;
  if (splits > 16) splits = 16;
  l.splits = splits < 1 ? 1 : (int)splits;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return p;
  };
  l.state = take(sizeof(LceState));
  l.rank = take(4ull * a.n);
  l.row_of = take(4ull * a.n);
  l.row_target = take(4ull * a.n);
  l.loss_rows = take(4ull * a.n);
  l.target_logit = take(4ull * piece);
  l.stats = take(8ull * piece * l.tiles);
  l.linear = take(a.label_smoothing != 0.f ? 4ull * piece * l.tiles : 0);
  l.h_plane = (up(a.n, 64) + 64) * l.ld_h;
  l.h = take(2ull * l.limbs * l.h_plane);
  l.w_plane = (long long)a.v * l.ld_w;
  l.w = take(l.stage_w ? 2ull * l.limbs * l.w_plane : 0);
  l.g_plane = piece * l.ld_kept;
  if (a.grads) {
    l.kept = take((wide ? 4ull : 2ull) * l.g_plane);
    l.g = wide ? take(2ull * l.limbs * l.g_plane) : l.kept;
    l.part = take(l.splits > 1 ? 4ull * l.splits * piece * a.d : 0);
    l.acc = take(l.pieces > 1 && !wide ? 4ull * a.v * a.d : 0);
  }
  l.bytes = at;
  return l;
}

bool valid(const PsgdLce& a) {
  return a.n >= 0 && a.d >= 1 && a.v >= 1 && a.dtype >= 0 && a.dtype <= 2 && a.ld_h >= a.d && a.ld_w >= a.d &&
         a.reduction >= 0 && a.reduction <= 2 && a.piece_bytes >= 0 && a.n <= (1 << 30) && a.v <= (1 << 30);
}

template <typename K>
int launch(K kernel, const LceArgs& args, cudaStream_t stream) {
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L_SMEM) != cudaSuccess) {
    cudaGetLastError();  // else it would be taken for the next launch's
    return PSGD_ELAUNCH;
  }
  kernel<<<psgd_num_sms(), L_THREADS, L_SMEM, stream>>>(args);
  return cudaGetLastError() == cudaSuccess ? PSGD_OK : PSGD_ELAUNCH;
}

template <typename T>
int stage(const T* src, long long ld, int n, int d, const int* rank, const LceState* state, uint16_t* out, long long ld_out,
          long long plane, T* dh, cudaStream_t stream) {
  const bool vec = d % 8 == 0 && aligned16(src) && ld * sizeof(T) % 16 == 0 && aligned16(dh);
  const int grid = (int)(((long long)n + (rank ? 64 : 0) + 7) / 8);
  if (vec) lce_stage_kernel<T, true><<<grid, 256, 0, stream>>>(src, ld, n, d, rank, state, out, ld_out, plane, dh);
  else lce_stage_kernel<T, false><<<grid, 256, 0, stream>>>(src, ld, n, d, rank, state, out, ld_out, plane, dh);
  return cudaGetLastError() == cudaSuccess ? PSGD_OK : PSGD_ELAUNCH;
}

// T: type of h, w and the gradients; OP: operand type of the tensor cores; KT: type of the kept exponentials.
template <typename T, typename OP, typename KT>
int run(const PsgdLce& a, int* err, cudaStream_t stream) {
  constexpr bool half = is_half<OP>();
  const Layout l = layout(a);
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.workspace);
  LceState* state = reinterpret_cast<LceState*>(ws + l.state);
  int* rank = reinterpret_cast<int*>(ws + l.rank);
  int* row_of = reinterpret_cast<int*>(ws + l.row_of);
  int* row_target = reinterpret_cast<int*>(ws + l.row_target);
  float* loss_rows = reinterpret_cast<float*>(ws + l.loss_rows);
  uint16_t* h = reinterpret_cast<uint16_t*>(ws + l.h);
  const uint16_t* w = l.stage_w ? reinterpret_cast<uint16_t*>(ws + l.w) : reinterpret_cast<const uint16_t*>(a.w);
  const long long ld_w = l.stage_w ? l.ld_w : a.ld_w;
  const bool none = a.reduction == PSGD_REDUCE_NONE;

  lce_plan_kernel<<<1, 1024, 0, stream>>>(a.target, a.n, a.v, a.ignore_index, a.reduction, half, a.grad, rank, row_of,
                                          row_target, a.loss, state, err);
  if (cudaGetLastError() != cudaSuccess) return PSGD_ELAUNCH;
  if (int rc = stage<T>(reinterpret_cast<const T*>(a.h), a.ld_h, a.n, a.d, rank, state, h, l.ld_h, l.h_plane,
                        reinterpret_cast<T*>(a.grads ? a.dh : nullptr), stream))
    return rc;
  if (l.stage_w)
    if (int rc = stage<T>(reinterpret_cast<const T*>(a.w), a.ld_w, a.v, a.d, nullptr, state, const_cast<uint16_t*>(w), l.ld_w,
                          l.w_plane, nullptr, stream))
      return rc;

  LceArgs args = {};
  args.state = state;
  args.err = err;
  args.wait_ns = WAIT_LIMIT_NS;
  // fp32: the products of two limbs down to 2^-16 of the whole, smallest first (2^-24 is left out)
  const uint8_t six[6] = {0x20, 0x02, 0x11, 0x10, 0x01, 0x00};
  auto limbs = [&](LceProblem& p) {
    p.nseg = l.limbs == 1 ? 1 : 6;
    for (int i = 0; i < 6; ++i) p.segs[i] = l.limbs == 1 ? 0 : six[i];
    p.splits = 1;
  };
  for (int piece = 0; piece < l.pieces; ++piece) {
    const int row0 = piece * l.piece, rows = a.n - row0 < l.piece ? a.n - row0 : l.piece;
    const int rows64 = (rows + 63) / 64 * 64;
    LceProblem& p = args.p[0];
    p = LceProblem{};
    limbs(p);
    for (int i = 0; i < l.limbs; ++i) {
      if (int rc = encode(&p.ta[i], h + i * l.h_plane + (long long)row0 * l.ld_h, half, rows, a.d, l.ld_h, LM)) return rc;
      if (int rc = encode(&p.tb[i], w + i * l.w_plane, half, a.v, a.d, ld_w, LN)) return rc;
    }
    p.M = rows, p.N = a.v, p.K = a.d, p.dyn = 1, p.row0 = row0;
    args.nproblems = 1;
    LceLogits& g = args.logits;
    g.stats = reinterpret_cast<float2*>(ws + l.stats);
    g.linear = a.label_smoothing != 0.f ? reinterpret_cast<float*>(ws + l.linear) : nullptr;
    g.target_logit = reinterpret_cast<float*>(ws + l.target_logit);
    g.row_target = row_target;
    g.kept = a.grads ? ws + l.kept : nullptr;
    g.ld_kept = l.ld_kept;
    if (int rc = launch(lce_product_kernel<OP, KT, true>, args, stream)) return rc;

    LceRows r = {};
    r.stats = g.stats, r.linear = g.linear, r.target_logit = g.target_logit, r.row_target = row_target, r.row_of = row_of;
    r.grad = none ? a.grad : nullptr;
    r.loss_rows = loss_rows, r.loss = a.loss, r.kept = g.kept, r.limbs = reinterpret_cast<uint16_t*>(ws + l.g);
    r.ld_kept = l.ld_kept, r.plane = l.g_plane, r.v = a.v, r.tiles = l.tiles, r.row0 = row0, r.rows = rows, r.none = none;
    r.smoothing = a.label_smoothing, r.z = a.z_loss;
    int cols = a.grads ? (2 * psgd_num_sms() + rows64 - 1) / rows64 : 1;
    if (cols > (a.v + 2047) / 2048) cols = (a.v + 2047) / 2048;
    lce_rows_kernel<KT, OP><<<dim3(rows64, cols), 256, 0, stream>>>(r, state);
    if (cudaGetLastError() != cudaSuccess) return PSGD_ELAUNCH;
    if (!a.grads) continue;

    const uint16_t* gm = reinterpret_cast<const uint16_t*>(ws + l.g);
    LceProblem& ph = args.p[0];  // dh = g w: g K-major, w (rows of K = vocabulary) MN-major
    ph = LceProblem{};
    limbs(ph);
    for (int i = 0; i < l.limbs; ++i) {
      if (int rc = encode(&ph.ta[i], gm + i * l.g_plane, half, rows, a.v, l.ld_kept, LM)) return rc;
      if (int rc = encode(&ph.tb[i], w + i * l.w_plane, half, a.v, a.d, ld_w, 64)) return rc;
    }
    ph.b_mn = 1, ph.M = rows, ph.N = a.d, ph.K = a.v, ph.dyn = 1, ph.row0 = row0, ph.splits = l.splits;
    ph.row_of = row_of, ph.out = a.dh, ph.ld_out = a.d;
    ph.part = l.splits > 1 ? reinterpret_cast<float*>(ws + l.part) : nullptr;
    LceProblem& pw = args.p[1];  // dw = g^T h: both with rows of K = tokens
    pw = LceProblem{};
    limbs(pw);
    for (int i = 0; i < l.limbs; ++i) {
      if (int rc = encode(&pw.ta[i], gm + i * l.g_plane, half, rows64, a.v, l.ld_kept, 64)) return rc;
      if (int rc = encode(&pw.tb[i], h + i * l.h_plane + (long long)row0 * l.ld_h, half, rows64, a.d, l.ld_h, 64)) return rc;
    }
    pw.a_mn = pw.b_mn = 1, pw.M = a.v, pw.N = a.d, pw.K = rows, pw.dyn = 2, pw.row0 = row0;
    pw.out = a.dw, pw.ld_out = a.d;
    if (l.pieces > 1) {
      float* acc = sizeof(T) == 4 ? reinterpret_cast<float*>(a.dw) : reinterpret_cast<float*>(ws + l.acc);
      pw.acc = piece > 0 ? acc : nullptr;
      pw.acc_out = piece + 1 < l.pieces ? acc : nullptr;
    }
    args.nproblems = 2;
    if (int rc = launch(lce_product_kernel<OP, T, false>, args, stream)) return rc;
    if (l.splits > 1) {
      const long long n = (long long)rows * a.d, want = (n + 255) / 256, most = 8LL * psgd_num_sms();
      lce_join_kernel<T><<<(int)(want < most ? want : most), 256, 0, stream>>>(ph.part, l.splits, rows, a.d, row0, row_of,
                                                                              reinterpret_cast<T*>(a.dh), state);
      if (cudaGetLastError() != cudaSuccess) return PSGD_ELAUNCH;
    }
  }
  if (!none) {
    lce_loss_kernel<<<1, 1024, 0, stream>>>(loss_rows, state, a.reduction == PSGD_REDUCE_MEAN, a.loss);
    if (cudaGetLastError() != cudaSuccess) return PSGD_ELAUNCH;
  }
  return PSGD_OK;
}

}  // namespace
}  // namespace psgd

extern "C" long long psgd_lce_workspace(const PsgdLce* a) {
  using namespace psgd;
  if (!a || !valid(*a)) return PSGD_EINVAL;
  return (long long)layout(*a).bytes;
}

extern "C" int psgd_lce(const PsgdLce* a, int* dev_err, cudaStream_t stream) {
  using namespace psgd;
  if (!a || !valid(*a) || !dev_err || a->n < 1 || !a->h || !a->w || !a->target || !a->loss || !a->workspace ||
      !aligned16(a->workspace) || (a->grads && (!a->dh || !a->dw)))
    return PSGD_EINVAL;
  if (a->workspace_bytes < psgd_lce_workspace(a)) return PSGD_ESPACE;
  switch (a->dtype) {
    case PSGD_F32: return run<float, __nv_bfloat16, float>(*a, dev_err, stream);
    case PSGD_BF16: return run<__nv_bfloat16, __nv_bfloat16, __half>(*a, dev_err, stream);
    default: return run<__half, __half, __half>(*a, dev_err, stream);
  }
}
