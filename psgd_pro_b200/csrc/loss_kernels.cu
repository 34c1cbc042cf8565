// Softmax cross entropy of a linear head, loss and gradients, without keeping the logits:
//   l = h w^T;  lse = log sum_v exp l_v;  loss = lse - (1 - s) l_t - s mean_v l_v + z lse^2
//   g = c [ (1 + 2 z lse) p - (1 - s) 1[v = t] - s / V ],  p = exp(l - lse);  dh = g w;  dw = g^T h
// for the rows whose target counts. The steps, each one launch:
//   plan     numbers the counted rows (the others cost nothing below, and no value of theirs is read again);
//   stage    gathers their rows of h as tensor-core operands (fp32: three bf16 limbs); zeros the other rows of dh;
//   logits   tile by tile on the tensor cores; the epilogue keeps, per row and 64 or 128 columns of the vocabulary, the
//            maximum m and sum of exp(l - m) in fp32 and, for gradients, exp(l - m) itself in 16 bits;
//   rows     joins those statistics to lse and the loss, and turns exp(l - m) into g in place;
//   grads    dh = g w and dw = g^T h as one list of tiles (w, g and h are read in the orientation they have, by
//            MN-major operand descriptors: nothing is transposed in memory).
// One pass over the vocabulary with kept exponentials costs 6 N V D operations; forming the logits again for the
// gradients, the alternative that keeps nothing, costs 8 N V D. What is kept is bounded: tokens are taken in pieces.
//
// What bounds it (8192 x 2048 x 32000 bf16, 6144 rows counted, 2.42 TFLOP: 2.15 ms, 1.12 PFLOP/s under the power cap;
// alone on a cool GPU 600 + 135 + 1100 us in the three long launches): the products by what the SMs can take from L2, 64
// bytes a clock each, which a 256 x 256 tile of two SMs needs for every 512 clocks of products (13.2 TB/s and 83 to 88% of
// the tensor pipe at depth 4096, measured); at depth 1024 too, where a tile's results are a larger part of that traffic (12.3
// TB/s and 63 to 67% of the pipe in the logits, 14.3 and 75% in the gradients). `rows` moves 4 bytes a logit at 5.9 TB/s. Small calls cost their four launches, 27 us.
#include "elem.cuh"
#include "pair_rounds.h"

#include <float.h>

#include <type_traits>

namespace psgd {
namespace {

constexpr int LM = 256, LK = 64;    // rows of a tile (two CTAs of 128), depth of a copied block
constexpr int L_THREADS = 384;      // a warpgroup for copies and products, two on the accumulators
// Registers a thread: 168 at launch (384 threads); 3 * 168 = 56 + 2 * 224.
constexpr int L_REGS_LOW = 56, L_REGS_HIGH = 224;
constexpr int L_LIMBS = 3;          // of an fp32 operand
constexpr int L_GROUP_M = 4;         // row tiles that walk the column tiles together (L2 reuse of both operands)
constexpr int L_UNIT = 8;            // what a unit costs besides its K blocks (its last step), in K blocks: about 2.5 us
// Kept exponentials are fp16 of 2^15 exp(l - m), exp(l - m) in [0, 1]: 11 significant bits down to 2^-29 of the row's
// maximum in these columns (half a tile's), so that in bf16 calls the one rounding that matters is that of g.
constexpr float L_KEEP_SCALE = 32768.f;
// g is held times 2^8 when it is fp16: p below 2^-14 keeps its bits down to 2^-22 and |g| may reach 255.
constexpr float L_HALF_SCALE = 256.f;
// Upstream gradients by row have the range of fp32, which fp16 operands do not: g takes their significand alone, in [1/2, 1).
// dh multiplies a row by 2^e of its own at the end, so that rows do not affect each other; for dw, h takes 2^e, exactly but
// for what lies below 2^-29 of the largest |upstream h| of the call, which is brought just below 2^L_REACH.
constexpr int L_REACH = 15, L_NO_REACH = -1000;

struct LceState {  // device scalars of one call
  int counted;
  float alpha;  // factor of both gradients
  int reach;    // fp16 by rows: every finite |upstream h| is below 2^reach
};

// x = m 2^e with |m| in [1/2, 1) (zero, infinities and NaN: themselves, e = 0).
PSGD_DEVI float split_power(float x, int& e) {
  e = 0;
  return fabsf(x) <= FLT_MAX ? frexpf(x, &e) : x;
}

// The error word may be pinned host memory, where atomics are not to be relied on: bits are added by a plain store (when
// two kinds of error meet, one of them is reported).
PSGD_DEVI void report(int* err, int bits) {
  volatile int* w = err;
  *w = *w | bits;
  __threadfence_system();
}

// ---- plan ------------------------------------------------------------------------------------------------------------
struct LcePlan {
  const long long* target;
  long long ignore;
  const float* grad;
  int *rank, *row_of, *row_target;
  float* loss;
  LceState* state;
  int* err;
  int n, v, reduction, half;
  PSGD_DEVI bool counts(long long x, bool& bad) const {
    const bool yes = x != ignore && x >= 0 && x < v;
    bad |= x != ignore && !yes;
    return yes;
  }
  PSGD_DEVI bool none() const { return reduction == PSGD_REDUCE_NONE; }
  // A row's entries; r: its number among the counted rows (or any, if it does not count).
  PSGD_DEVI void enter(int i, long long x, bool counted, int r) const {
    if (counted) {
      row_of[r] = i;
      row_target[r] = (int)x;
    } else if (none()) {
      loss[i] = 0.f;
    }
  }
  PSGD_DEVI void finish(int total) const {
    state->counted = total;
    state->reach = L_NO_REACH;
    float alpha = half ? 1.f / L_HALF_SCALE : 1.f;
    if (!none() && grad) alpha *= *grad;
    if (reduction == PSGD_REDUCE_MEAN) alpha /= (float)max(total, 1);
    state->alpha = alpha;
  }
};

// One block numbers the counted rows in their order (8192 tokens: 9 us, two reads of the targets and a scan). 65536 at a time: every warp counts its groups of 32, the
// counts are scanned, and each row's number is its group's start plus its place in the group.
constexpr int PLAN_GROUPS = 64;  // groups of 32 targets that a warp has at a time
__global__ void __launch_bounds__(1024) lce_plan_kernel(const LcePlan a) {
  __shared__ int count[PLAN_GROUPS * 32];
  __shared__ int warp_total[32];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  bool bad = false;
  int total = 0;
  pdl_trigger();
  for (int base = 0; base < a.n; base += 1024 * PLAN_GROUPS) {
    const int groups = min(PLAN_GROUPS, (a.n - base + 1023) / 1024);
#pragma unroll 8
    for (int g = 0; g < groups; ++g) {
      const int i = base + g * 1024 + t;
      const bool counted = a.counts(i < a.n ? a.target[i] : a.ignore, bad);
      const uint32_t m = __ballot_sync(0xffffffffu, counted);
      if (lane == 0) count[g * 32 + warp] = __popc(m);
    }
    for (int g = groups * 32 + t; g < PLAN_GROUPS * 32; g += 1024) count[g] = 0;
    __syncthreads();
    // exclusive scan of the 2048 counts, two to a thread
    const int c0 = count[2 * t], c1 = count[2 * t + 1];
    int sum = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) warp_total[warp] = sum;
    __syncthreads();
    int before = total, all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += warp_total[w];
      all += warp_total[w];
    }
    before += sum - c0 - c1;
    count[2 * t] = before;
    count[2 * t + 1] = before + c0;
    total += all;
    __syncthreads();
#pragma unroll 8
    for (int g = 0; g < groups; ++g) {
      const int i = base + g * 1024 + t;
      const long long x = i < a.n ? a.target[i] : a.ignore;
      const bool counted = a.counts(x, bad);
      const uint32_t m = __ballot_sync(0xffffffffu, counted);
      const int r = count[g * 32 + warp] + __popc(m & ((1u << lane) - 1u));
      if (i >= a.n) continue;
      a.rank[i] = counted ? r : -1;
      a.enter(i, x, counted, r);
    }
    __syncthreads();
  }
  if (bad) report(a.err, ERR_BAD_TARGET);
  if (t == 0) a.finish(total);
}

// ---- stage -----------------------------------------------------------------------------------------------------------
PSGD_DEVI void limbs3(float x, float* l) {
  l[0] = __bfloat162float(__float2bfloat16_rn(x));
  const bool fine = fabsf(l[0]) <= FLT_MAX;  // an infinity or NaN is its first limb
  const float r = fine ? x - l[0] : 0.f;
  l[1] = __bfloat162float(__float2bfloat16_rn(r));
  l[2] = r - l[1];
}

// Tensor-core operands from matrices: row i of h to its number among the counted rows, row i of w to row i, itself or (WIDE)
// its bf16 limbs `plane` elements apart. Rows that do not count zero their row of dh instead. Blocks beyond the rows zero the operand's rows from
// the count to the next multiple of 64, which a reduction over rows reads.
template <typename T>
struct LceStage {
  const T* src;
  long long ld, ld_out, plane;
  uint16_t* out;
  T* dh;
  int n, blocks;  // (8 rows a block)
};
// INLINE: there was no plan launch; every block counts the rows before its own (up to PLAN_INLINE of them: the reads are
// shorter than a launch), and the last one of h finishes the plan.
constexpr int PLAN_INLINE = 2048;
template <typename T, bool WIDE, bool VEC, bool INLINE>
__global__ void __launch_bounds__(256) lce_stage_kernel(const LceStage<T> h, const LceStage<T> w, int d, const LcePlan plan) {
  constexpr int V = VEC ? 8 : 1;
  __shared__ int before[8];
  pdl_trigger();
  if (!INLINE) pdl_wait();
  const bool first = (int)blockIdx.x < h.blocks;
  const LceStage<T>& a = first ? h : w;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, i0 = (blockIdx.x - (first ? 0 : h.blocks)) * 8, i = i0 + warp;
  long long r = i;
  int counted = INLINE ? 0 : plan.state->counted;
  if (INLINE && first) {
    const bool last = (int)blockIdx.x == h.blocks - 1;  // (beyond every row: it counts them all)
    const int upto = min(i0, plan.n);
    int mine = 0;
    bool bad = false;
#pragma unroll 4
    for (int k = threadIdx.x; k < upto; k += 256) mine += plan.counts(plan.target[k], bad);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) before[warp] = mine;
    __syncthreads();
    counted = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) counted += before[k];
    if (last && threadIdx.x == 0) plan.finish(counted);
    if (last && bad) report(plan.err, ERR_BAD_TARGET);
    if (i0 < plan.n) {  // this block's rows; a warp a row, each with the targets of all eight
      const long long x = lane < 8 && i0 + lane < plan.n ? plan.target[i0 + lane] : plan.ignore;
      const uint32_t m = __ballot_sync(0xffffffffu, plan.counts(x, bad));
      r = (m >> warp) & 1u ? counted + __popc(m & ((1u << warp) - 1u)) : -1;
      if (lane == warp && i < plan.n) plan.enter(i, x, r >= 0, (int)r);
    }
  }
  if (i >= a.n) {
    if (!first || i >= a.n + 64) return;
    if (INLINE && i0 < a.n) {  // the block with the last rows: the count includes those
      const long long x = lane < 8 && i0 + lane < plan.n ? plan.target[i0 + lane] : plan.ignore;
      bool bad = false;
      counted += __popc(__ballot_sync(0xffffffffu, plan.counts(x, bad)));
    }
    r = counted + (i - a.n);
    if (r >= ((counted + 63) & ~63)) return;
  } else if (!INLINE && first) {
    r = plan.rank[i];
  }
  if (r < 0) {
    if (a.dh)
      for (int e = lane * V; e < d; e += 32 * V) {
        const float zero[8] = {};
        store_vec<T, V>(a.dh + (long long)i * d + e, zero);
      }
    return;
  }
  const bool there = i < a.n;
  const T* src = a.src + (there ? i * a.ld : 0);
  uint16_t* out = a.out + r * a.ld_out;
  for (int e = lane * V; e < d; e += 32 * V) {
    if constexpr (!WIDE) {
      T* to = reinterpret_cast<T*>(out) + e;
      if constexpr (VEC) {
        *reinterpret_cast<uint4*>(to) = there ? *reinterpret_cast<const uint4*>(src + e) : make_uint4(0, 0, 0, 0);
      } else {
        *to = there ? src[e] : from_f32<T>(0.f);
      }
    } else {
      float x[V], l[3][V];
#pragma unroll
      for (int k = 0; k < V; ++k) x[k] = 0.f;
      if (there) load_vec<T, V>(src + e, x);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float p[3];
        limbs3(x[k], p);
        l[0][k] = p[0], l[1][k] = p[1], l[2][k] = p[2];
      }
#pragma unroll
      for (int q = 0; q < 3; ++q)
        store_vec<__nv_bfloat16, V>(reinterpret_cast<__nv_bfloat16*>(out) + q * a.plane + e, l[q]);
    }
  }
}

// fp16 by rows, for every counted row, a warp each: what its row of dh is multiplied by in the end, and how far upstream times
// h reaches (a maximum: the order of its atomics does not matter).
__global__ void __launch_bounds__(256) lce_reach_kernel(const __half* __restrict__ h, long long ld, int d, const float* __restrict__ grad,
                                                        const int* __restrict__ row_of, float* __restrict__ row_scale, LceState* state) {
  pdl_trigger();
  pdl_wait();
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= state->counted) return;
  int e;
  const float m = split_power(grad[row_of[r]], e);
  if (lane == 0) row_scale[r] = ldexpf(state->alpha, e);
  if (m == 0.f || !(fabsf(m) <= FLT_MAX)) return;
  float top = 0.f;
  for (int c = lane; c < d; c += 32) {
    const float x = fabsf(__half2float(h[r * ld + c]));
    if (x <= FLT_MAX) top = fmaxf(top, x);
  }
  top = warp_max(top);
  if (lane == 0 && top > 0.f) {
    int k;
    split_power(top, k);
    atomicMax(&state->reach, e + k);
  }
}
// fp16 by rows: a piece's rows of h, done with as the logits' operand, times their upstream 2^e, as dw's.
__global__ void __launch_bounds__(256) lce_lift_kernel(__half* __restrict__ h, long long ld, int d, const float* __restrict__ grad,
                                                       const int* __restrict__ row_of, int row0, int rows, const LceState* state) {
  pdl_trigger();
  pdl_wait();
  const int r = row0 + blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (r >= min(row0 + rows, state->counted)) return;
  int e;
  const float m = split_power(grad[row_of[r]], e);
  if (!(fabsf(m) <= FLT_MAX)) return;  // (its g is infinite or NaN, and so is dw)
  const int by = e + L_REACH - state->reach;
  for (int c = lane; c < d; c += 32) {
    const float x = __half2float(h[r * ld + c]);
    // (a row that counts nothing may have any h: zero, so that it does not leave the type's range)
    if (fabsf(x) <= FLT_MAX) h[r * ld + c] = __float2half_rn(m == 0.f ? 0.f : ldexpf(x, by));
  }
}

// ---- the products ----------------------------------------------------------------------------------------------------
// D (M x N) = A B^T over K. An operand is K-major (rows of M or N, K contiguous) or MN-major (rows of K, M or N contiguous:
// *_mn). fp32 operands are three bf16 limbs: the products of limbs (i, j) with i + j <= 2 (2^-24 of the whole is left out).
struct LceProblem {
  CUtensorMap ta[L_LIMBS], tb[L_LIMBS];
  int a_mn, b_mn;
  int M, N, K;    // bounds; the counted rows replace M (dyn 1) or K (dyn 2)
  int dyn, row0;  // first counted row of this piece
  int splits;     // K blocks are dealt to this many units of a tile, whose sums go to `part`
  // outputs of a gradient tile: rows through row_of (or as they are)
  const int* row_of;
  void* out;
  long long ld_out;
  const float* row_scale;  // dh, fp16 by rows: instead of alpha, by counted row
  int lifted;              // dw, fp16 by rows: h was brought below 2^L_REACH
  float* part;       // splits > 1: [split][M][ld_part], joined by lce_join_kernel
  const float* acc;  // earlier pieces' sums [M][ld_acc], added
  float* acc_out;    // sums so far, fp32, instead of out
  long long ld_part, ld_acc;
};
// What the sums of a gradient of type T are multiplied by, but for row_scale.
template <typename T>
PSGD_DEVI float lce_alpha(const LceState* state, int lifted) {
  if constexpr (is_half<T>())
    if (lifted) return ldexpf(state->alpha, state->reach - L_REACH);
  return state->alpha;
}
struct LceShape {
  int M, K, tiles_m, tiles_n, kblocks, units, unit_kblocks;
};
template <int BN>
PSGD_DEVI LceShape lce_shape(const LceProblem& p, const LceState* state) {
  LceShape s;
  const int there = max(0, state->counted - p.row0);
  s.M = p.dyn == 1 ? min(p.M, there) : p.M;
  s.K = p.dyn == 2 ? min(p.K, there) : p.K;
  s.tiles_m = (s.M + LM - 1) / LM;
  s.tiles_n = (p.N + BN - 1) / BN;
  s.kblocks = (s.K + LK - 1) / LK;
  s.units = s.tiles_m * s.tiles_n * p.splits;
  s.unit_kblocks = s.kblocks / p.splits;
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
  const int more = s.kblocks - s.unit_kblocks * p.splits;  // splits of unit_kblocks, the first ones of one more
  x.k0 = x.split * s.unit_kblocks + min(x.split, more);
  x.k1 = x.k0 + s.unit_kblocks + (x.split < more);
  return x;
}

// The units of a cluster: its share of the first problem's, dealt in turn, then of the second's, of which the clusters
// that had one unit less of the first take as many more first as make up for it (the first problem's units are the
// longer ones: without this the longest and the shortest share would be one of them apart).
struct LceDeal {
  int c, n, h, rem, extra, base, u0, u1;
  PSGD_DEVI LceDeal(const LceShape& s0, const LceShape& s1, bool two) {
    c = blockIdx.x >> 1;
    n = gridDim.x >> 1;
    u0 = s0.units;
    u1 = two ? s1.units : 0;
    rem = u0 % n;
    h = u0 / n + (c < rem);
    extra = two && rem && s0.unit_kblocks > s1.unit_kblocks ? (s0.unit_kblocks + L_UNIT) / (s1.unit_kblocks + L_UNIT) : 0;
    base = (n - rem) * extra;
  }
  // Unit k of this cluster: (problem, index), or false.
  PSGD_DEVI bool get(int k, int& problem, int& index) const {
    problem = k >= h;
    if (!problem) {
      index = c + k * n;
      return true;
    }
    k -= h;
    const bool is_short = c >= rem;
    if (is_short && k < extra) {
      index = (c - rem) + k * (n - rem);
    } else {
      index = base + (is_short ? c - rem : c + (n - rem)) + (k - (is_short ? extra : 0)) * n;
    }
    return index < u1;
  }
};

struct LceLogits {  // what the logits' epilogue keeps
  float2* stats;  // [row][half a tile's columns]: (maximum, sum of exp)
  float* linear;  // [row][half a tile's columns]: sum of the logits (label smoothing), or NULL
  float* target_logit;
  const int* row_target;
  void* kept;  // exp(l - m), [row][ld_kept], or NULL
  long long ld_kept;
  int tiles;
};

struct __align__(64) LceArgs {
  LceProblem p[2];
  int nproblems, chunk;  // chunk: K blocks that a sum runs over before it is added in fp32
  LceLogits logits;
  const LceState* state;
  const float* loss_rows;  // summed into loss by the first block, or NULL
  float* loss;
  int mean;
  int* err;
  unsigned long long wait_ns;
};

// Shared memory of a stage: KS blocks of 64 of K, each LIMBS tiles of A (this CTA's 128 rows) and of B (its half of BN).
template <int LIMBS, int BN, bool LOGITS>
struct LceCfg {
  static constexpr int KS = LIMBS == 1 ? 2 : 1;
  static constexpr int STAGES = LIMBS == 1 || LOGITS ? 3 : 2;
  static constexpr int A = 128 * LK * 2, B = (BN / 2) * LK * 2;
  static constexpr int BLOCK = LIMBS * (A + B), STAGE = KS * BLOCK;
  static constexpr int SMEM = 1024 + STAGES * STAGE + 512 + (LOGITS ? 0 : 8 * 32 * 33 * 4);  // (grad_row's blocks)
  static constexpr int COLS = BN / 2;                  // accumulator columns of an epilogue thread
  static constexpr int ACC = (LIMBS == 1 ? 1 : 2) * BN;  // TMEM columns of an accumulator (fp32: the small products apart)
  static constexpr int TMEM = 2 * ACC < 512 ? 256 : 512;
  static_assert(2 * ACC <= 512 && SMEM <= 232448, "TMEM and shared memory of an SM");
};

PSGD_DEVI uint64_t lce_desc(uint32_t saddr, bool mn) {
  // K-major: 128-byte rows, 8-row swizzle atoms 1024 bytes apart. MN-major: atoms of 64 (M or N) x 8 (K), 1024 bytes
  // apart along K; the next 64 of M or N are one 64 x 64 box (8192 bytes) on.
  uint64_t d = sdesc_k_sw128(saddr);
  if (mn) d = (d & ~((uint64_t)0x3FFF << 16)) | ((uint64_t)(8192 >> 4) << 16);
  return d;
}
template <typename OP, int BN>
PSGD_DEVI uint32_t lce_idesc(bool a_mn, bool b_mn) {
  const uint32_t fmt = is_half<OP>() ? 0u : 1u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(LM >> 4) << 24);
}

constexpr float LOG2E = 1.4426950408889634f;
PSGD_DEVI float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 bytes at once (a whole sector of a row that other lanes do not share).
PSGD_DEVI void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
template <typename T>
PSGD_DEVI void store_row32(T* p, const float* v) {  // 32 bytes of T
  uint32_t w[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (sizeof(T) == 4) w[k] = __float_as_uint(v[k]);
    else w[k] = pack2(v[2 * k], v[2 * k + 1], T());
  }
  store32(p, w);
}

// The logits' epilogue: this thread's COLS columns of one row.
template <typename KT, int COLS>
PSGD_DEVI void logits_row(const LceProblem& p, const LceShape& sh, const LceLogits& g, long long row, int n0, float* v) {
  constexpr bool WIDE = sizeof(KT) == 4;
  const bool live = row < sh.M;
  const int width = min(COLS, p.N - n0);  // (n0 is below N: see the caller)
  const int at = live ? g.row_target[p.row0 + row] - n0 : -1;
  const bool here = at >= 0 && at < width;
  if (__any_sync(0xffffffffu, here)) {
    float x = 0.f;
#pragma unroll
    for (int k = 0; k < COLS; ++k) x = at == k ? v[k] : x;
    if (here) g.target_logit[row] = x;
  }
  float linear = 0.f;
  if (g.linear) {
    float part[4] = {};
#pragma unroll
    for (int k = 0; k < COLS; ++k) part[k & 3] += k < width ? v[k] : 0.f;
    linear = (part[0] + part[1]) + (part[2] + part[3]);
  }
  if (width < COLS)
#pragma unroll
    for (int k = 0; k < COLS; ++k)
      if (k >= width) v[k] = -INFINITY;
  // (four chains each for the maximum and the sum: with two warps to a scheduler their latency is what a tile costs here)
  float tops[4] = {v[0], v[1], v[2], v[3]}, sums[4] = {};
#pragma unroll
  for (int k = 4; k < COLS; ++k) tops[k & 3] = fmaxf(tops[k & 3], v[k]);
  const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const float ref = top == -INFINITY || top != top ? 0.f : top;
#pragma unroll
  for (int k = 0; k < COLS; ++k) {
    // 16 bits: 2^15 exp(l - m), the factor added to the exponent, whose rounding is 2^-21 at most
    v[k] = WIDE ? expf(v[k] - ref) : exp2_fast(fmaf(v[k] - ref, LOG2E, 15.f));
    sums[k & 3] += v[k];
  }
  float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  if (!WIDE) sum *= 1.f / L_KEEP_SCALE;
  if (g.kept && live) {
    KT* to = reinterpret_cast<KT*>(g.kept) + row * g.ld_kept + n0;
    constexpr int S = 32 / sizeof(KT);
#pragma unroll
    for (int k = 0; k < COLS; k += S)
      if (k < width) store_row32<KT>(to + k, v + k);  // (ld_kept is a multiple of 64: zeros up to there)
  }
  if (live) {
    const long long to = row * g.tiles + n0 / COLS;
    g.stats[to] = make_float2(top, sum);
    if (g.linear) g.linear[to] = linear;
  }
}

// The gradients' epilogue: this thread's COLS columns of one row (all lanes of a warp call it: `live` says whether the row
// is there). Rows that 32-byte stores do not fit (an odd number of columns) go through `turn`, 32 x 33 floats of the
// warp, so that a store covers neighbours of one row.
template <typename T, int COLS>
PSGD_DEVI void grad_row(const LceProblem& p, const LceShape& sh, int split, long long row, int n0, float* v, float alpha,
                        float* turn) {
  const bool live = row < sh.M;
  const int width = min(COLS, p.N - n0), lane = threadIdx.x & 31;
  if (p.acc && live) {
    const float* from = p.acc + row * p.ld_acc + n0;
#pragma unroll
    for (int k = 0; k < COLS; ++k)
      if (k < width) v[k] += from[k];
  }
  if (p.part) {  // (rows of whole sectors)
    if (!live) return;
    float* to = p.part + ((long long)split * p.M + row) * p.ld_part + n0;
#pragma unroll
    for (int k = 0; k < COLS; k += 8)
      if (k < width) store_row32<float>(to + k, v + k);
    return;
  }
  if (p.acc_out) {
    if (!live) return;
    float* to = p.acc_out + row * p.ld_acc + n0;
#pragma unroll
    for (int k = 0; k < COLS; ++k)
      if (k < width) to[k] = v[k];
    return;
  }
  constexpr int S = 32 / sizeof(T);
  if constexpr (is_half<T>())
    if (p.row_scale && live) alpha = p.row_scale[p.row0 + row];
#pragma unroll
  for (int k = 0; k < COLS; ++k) v[k] *= alpha;
  const int at = live ? (p.row_of ? p.row_of[p.row0 + row] : (int)row) : -1;
  T* base = reinterpret_cast<T*>(p.out) + n0;
  if (p.ld_out % S == 0 && (reinterpret_cast<uintptr_t>(p.out) & 31) == 0) {  // (N is ld_out: whole sectors to its end)
    T* out = base + at * p.ld_out;
#pragma unroll
    for (int k = 0; k < COLS; k += S)
      if (live && k < width) store_row32<T>(out + k, v + k);
    return;
  }
  for (int c = 0; c < COLS; c += 32) {
    if (c >= width) break;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 32; ++k) {
      // (v's index has to be known where it is compiled: one of COLS / 32 blocks is taken)
      float x = v[k];
#pragma unroll
      for (int b = 32; b < COLS; b += 32) x = c == b ? v[b + k] : x;
      turn[lane * 33 + k] = x;
    }
    __syncwarp();
    for (int r = 0; r < 32; ++r) {
      const int to = __shfl_sync(0xffffffffu, at, r);
      if (to >= 0 && c + lane < width) base[to * p.ld_out + c + lane] = from_f32<T>(turn[r * 33 + lane]);
    }
  }
}

template <int COLS>
PSGD_DEVI void add_columns(uint32_t at, float* v) {
#pragma unroll
  for (int b = 0; b < COLS; b += 32) {
    float t[32];
    tmem_ld32(at + b, t);
#pragma unroll
    for (int e = 0; e < 32; ++e) v[b + e] += t[e];
  }
}

// A cluster of two CTAs on neighbouring SMs computes 256 x BN tiles: each CTA stages its 128 rows of A and its half of
// B, the leader (rank 0) issues M = 256 products that read both CTAs' shared memory, and each CTA's TMEM receives its 128
// rows. Against one-CTA tiles of 128 x 256 this takes a third less through L2 and shared memory for a product.
//   warp 0      copies; warp 1 (leader) products; warps 4..11: TMEM lanes 32 (w % 4)..., half of the columns each.
// Handshakes (waits bounded): full[s] at the leader takes an arrival of each CTA with the bytes that it copies to stage s
// (the phase cannot end before both have told theirs, so neither waits for the other; what a pair that gives up does with
// rounds that only one of them began: pair_rounds.h), empty[s] frees it (the products' commit, in both CTAs), tfull / tempty hand the two accumulators over. An accumulator takes `chunk` blocks of K; the epilogue adds the chunks in registers and hands the accumulator
// back at once: the tensor cores' sums truncate (a bias of about 1.1e-9 a product, measured), so sums that are to be
// right to fp32 stay short there, and the last step of a tile, from registers, never holds the tensor cores up.
template <typename OP, typename OUT, int LIMBS, int BN, bool LOGITS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(L_THREADS, 1)
    lce_product_kernel(const __grid_constant__ LceArgs args) {
  using C = LceCfg<LIMBS, BN, LOGITS>;
  constexpr int S = C::STAGES, COLS = C::COLS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S * C::STAGE);
  uint64_t* empty = full + S;
  uint64_t* tfull = empty + S;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile uint32_t* issued = tmem_slot + 2;     // rounds of copies that this CTA issued
  volatile uint32_t* peer_word = tmem_slot + 3;  // the peer's, and whether it gave up, from the peer
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();  // 0: leader

  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(&full[s], 2);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 16);
    }
    mbar_init(drain, 1);
    *abort = 0;
    *issued = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane < 2 * args.nproblems * LIMBS) {  // (the maps are arguments: no launch before writes them)
    const LceProblem& p = args.p[lane / (2 * LIMBS)];
    const int m = lane % (2 * LIMBS);
    prefetch_tmap(m < LIMBS ? &p.ta[m] : &p.tb[m - LIMBS]);
  }
  pdl_trigger();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers exist before any remote arrive or copy signal
  if (warp == 1) {
    __syncwarp();
    tmem_alloc_pair(tmem_slot, C::TMEM);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_wait();  // what the launch before wrote is read from here on
  const bool two = args.nproblems > 1;
  const LceShape s0 = lce_shape<BN>(args.p[0], args.state);
  const LceShape s1 = two ? lce_shape<BN>(args.p[1], args.state) : LceShape{};
  const LceDeal deal(s0, s1, two);
  const int chunk = args.chunk / C::KS;  // rounds of the stage ring to an accumulator

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L_REGS_LOW));
    if (warp == 0 && lane == 0) {
      // ---------------- copies (both CTAs) ----------------
      int s = 0;
      uint32_t ph = 0, rounds = 0;
      int which, index;
      for (int k = 0; deal.get(k, which, index) && !*abort; ++k) {
        const LceProblem& p = args.p[which];
        const LceUnit u = lce_unit(p, which ? s1 : s0, index);
        const int row = u.tm * LM + (int)rank * 128, col = u.tn * BN + (int)rank * (BN / 2);
        for (int kb = u.k0; kb < u.k1; kb += C::KS) {
          const int subs = min(C::KS, u.k1 - kb);
          if (!mbar_wait_for(&empty[s], ph ^ 1, abort, args.wait_ns)) break;
          const uint32_t fb = mapa_shared(&full[s], 0);
          mbar_arrive_expect_tx_cluster_relaxed(fb, C::BLOCK * (uint32_t)subs);
          ++rounds;
          for (int j = 0; j < subs; ++j) {
            const int x = (kb + j) * LK;
#pragma unroll
            for (int l = 0; l < LIMBS; ++l) {
              uint8_t* sa = smem + s * C::STAGE + j * C::BLOCK + l * C::A;
              uint8_t* sb = smem + s * C::STAGE + j * C::BLOCK + LIMBS * C::A + l * C::B;
              if (p.a_mn) {
#pragma unroll
                for (int i = 0; i < 2; ++i) tma_load_2d_pair(sa + i * 8192, &p.ta[l], fb, row + i * 64, x);
              } else {
                tma_load_2d_pair(sa, &p.ta[l], fb, x, row);
              }
              if (p.b_mn) {
#pragma unroll
                for (int i = 0; i < BN / 128; ++i) tma_load_2d_pair(sb + i * 8192, &p.tb[l], fb, col + i * 64, x);
              } else {
                tma_load_2d_pair(sb, &p.tb[l], fb, x, col);
              }
            }
          }
          if (++s == S) s = 0, ph ^= 1;
        }
      }
      *issued = rounds;
    } else if (warp == 1 && lane == 0 && rank == 0) {
      // ---------------- products (leader) ----------------
      int s = 0;
      uint32_t ph = 0, i = 0;
      bool ok = true;
      int which, index;
      for (int k = 0; ok && deal.get(k, which, index); ++k) {
        const LceProblem& p = args.p[which];
        const LceUnit u = lce_unit(p, which ? s1 : s0, index);
        const uint32_t idesc = lce_idesc<OP, BN>(p.a_mn, p.b_mn);
        const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = p.b_mn ? 2048 : 32;  // 16 of K, in bytes
        const uint64_t a0 = lce_desc(smem_u32(smem), p.a_mn), b0 = lce_desc(smem_u32(smem), p.b_mn);
        int kb = u.k0;
        do {  // one accumulator
          const uint32_t acc = i & 1, aph = (i >> 1) & 1;
          ++i;
          if (!mbar_wait_for(&tempty[acc], aph ^ 1, abort, args.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t dt = tmem_base + acc * C::ACC;
          uint32_t more = 0;
          for (int r = 0; r < chunk && kb < u.k1; ++r, kb += C::KS) {
            if (!mbar_wait_for(&full[s], ph, abort, args.wait_ns)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const int subs = min(C::KS, u.k1 - kb);
#pragma unroll
            for (int j = 0; j < C::KS; ++j) {
              if (j >= subs) break;
              const uint32_t at = s * C::STAGE + j * C::BLOCK;
#pragma unroll
              for (int kk = 0; kk < LK / 16; ++kk) {
                const uint64_t ad = a0 + ((at + kk * a_step) >> 4), bd = b0 + ((at + LIMBS * C::A + kk * b_step) >> 4);
                umma_bf16_pair(dt, ad, bd, idesc, more);
                if constexpr (LIMBS == 3) {
                  constexpr uint32_t LA = C::A >> 4, LB = C::B >> 4;
                  umma_bf16_pair(dt + BN, ad, bd + 2 * LB, idesc, more);
                  umma_bf16_pair(dt + BN, ad + 2 * LA, bd, idesc, 1);
                  umma_bf16_pair(dt + BN, ad + LA, bd + LB, idesc, 1);
                  umma_bf16_pair(dt + BN, ad, bd + LB, idesc, 1);
                  umma_bf16_pair(dt + BN, ad + LA, bd, idesc, 1);
                }
                more = 1;
              }
            }
            umma_commit_pair(&empty[s], 3);
            if (++s == S) s = 0, ph ^= 1;
          }
          if (!ok) break;
          umma_commit_pair(&tfull[acc], 3);
        } while (kb < u.k1);
      }
    }
  } else {
    // ---------------- accumulators (warps 4..11 of both CTAs) ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L_REGS_HIGH));
    const int q = warp & 3, half = (warp - 4) >> 2;
    if (args.loss_rows && blockIdx.x == 0) {  // the loss itself: fixed order, by the first block's 256 threads
      const int t = threadIdx.x - 128, n = args.state->counted;
      float* red = reinterpret_cast<float*>(smem + S * C::STAGE + 256);
      float sum = 0.f;
      for (int r = t; r < n; r += 256) sum += args.loss_rows[r];
      sum = warp_sum(sum);
      if (lane == 0) red[warp - 4] = sum;
      named_sync(1, 256);
      if (t == 0) {
        for (int w = 1; w < 8; ++w) sum += red[w];
        *args.loss = args.mean ? sum / (float)max(n, 1) : sum;
      }
    }
    float* turn = reinterpret_cast<float*>(smem + S * C::STAGE + 512) + (warp - 4) * (32 * 33);
    const uint32_t lead0 = mapa_shared(&tempty[0], 0), lead1 = mapa_shared(&tempty[1], 0);
    const float alpha0 = lce_alpha<OUT>(args.state, args.p[0].lifted), alpha1 = lce_alpha<OUT>(args.state, args.p[1].lifted);
    uint32_t i = 0;
    bool ok = true;
    int which, index;
    for (int k = 0; ok && deal.get(k, which, index); ++k) {
      const LceProblem& p = args.p[which];
      const LceShape& sh = which ? s1 : s0;
      const float alpha = which ? alpha1 : alpha0;
      const LceUnit u = lce_unit(p, sh, index);
      const int rounds = (u.k1 - u.k0 + C::KS - 1) / C::KS, chunks = max(1, (rounds + chunk - 1) / chunk);
      const long long row = (long long)u.tm * LM + rank * 128 + q * 32 + lane;
      const int n0 = u.tn * BN + half * COLS;
      // The next accumulator of this unit, at this warp's lanes and columns.
      auto take = [&]() -> uint32_t {
        const uint32_t acc = i & 1, aph = (i >> 1) & 1;
        ok = __all_sync(0xffffffffu, mbar_wait_for(&tfull[acc], aph, abort, args.wait_ns));
        tc_fence_after();
        return tmem_base + ((uint32_t)(q * 32) << 16) + acc * C::ACC + half * COLS;
      };
      // (Its columns are in registers: nothing in memory is handed over, and a releasing arrive would wait for this warp's
      // stores of the tile before.)
      auto give_back = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster_relaxed(i & 1 ? lead1 : lead0);
        ++i;
      };
      if constexpr (!LOGITS && LIMBS == 1) {  // one sum over all of K: no more than 32 columns in registers
        const uint32_t at = take();
        if (!ok) break;
#pragma unroll 1
        for (int c = 0; c < COLS; c += 32) {
          float f[32];
          tmem_ld32(at + c, f);
          if (n0 + c >= p.N) break;
          if (u.k0 >= u.k1)
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] = 0.f;
          grad_row<OUT, 32>(p, sh, u.split, row, n0 + c, f, alpha, turn);
        }
        give_back();
      } else {
        float f[COLS];
        uint32_t at = take();
        if (!ok) break;
#pragma unroll
        for (int b = 0; b < COLS; b += 32) tmem_ld32(at + b, f + b);
#pragma unroll 1
        for (int c = 1; c < chunks; ++c) {
          if constexpr (LIMBS == 3) add_columns<COLS>(at + BN, f);
          give_back();
          at = take();
          if (!ok) break;
          add_columns<COLS>(at, f);
        }
        if (!ok) break;
        if constexpr (LIMBS == 3) add_columns<COLS>(at + BN, f);
        give_back();
        if (u.k0 >= u.k1)
#pragma unroll
          for (int e = 0; e < COLS; ++e) f[e] = 0.f;
        if (n0 < p.N) {
          if constexpr (LOGITS) logits_row<OUT, COLS>(p, sh, args.logits, row, n0, f);
          else grad_row<OUT, COLS>(p, sh, u.split, row, n0, f, alpha, turn);
        }
      }
    }
  }

  // Neither CTA releases shared memory or TMEM while the other may still use them. Each tells the other, before they meet,
  // how many rounds of copies it issued and whether it gave up: both are final after the block's barrier.
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0) store_cluster(mapa_shared((const void*)peer_word, rank ^ 1), *issued << 1 | (*abort != 0));
  __syncwarp();
  cluster_sync();
  if (*abort || (*peer_word & 1u)) {
    // One of them left work behind. The leader, whose barriers all copies report to, waits until those of both CTAs have
    // landed and until the products that it issued (they read both CTAs' shared memory and write both's TMEM) are done;
    // the peer waits for the leader. A CTA that gave up is behind by rounds that it never copied.
    if (rank == 0 && threadIdx.x == 0) {
      volatile int never = 0;
      for (int i = 0; i < S; ++i) {
        const StageLeft left = stage_left(*issued, *peer_word >> 1, S, i);
        if (left.arrive) mbar_arrive(&full[i]);
        if (left.wait) mbar_wait(&full[i], left.parity, &never);
      }
    }
    if (rank == 0 && warp == 1 && lane == 0) {  // (the thread that issued them)
      volatile int never = 0;
      umma_commit_pair(drain, 1);
      mbar_wait(drain, 0, &never);
    }
    __syncwarp();
    cluster_sync();
  }
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc_pair(tmem_base, C::TMEM);
  }
  if (threadIdx.x == 0 && *abort) report(args.err, ERR_TIMEOUT_FULL);
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
  int stat;  // columns to a statistic
};

// One block a row (and 1 / gridDim.y of its columns), or (WARP) one warp a row, where a row is short. KT / GT: types of
// the kept exponentials and of g.
template <typename KT, typename GT, bool WARP>
__global__ void __launch_bounds__(256) lce_rows_kernel(const LceRows a, const LceState* state) {
  __shared__ float red[8];
  pdl_trigger();
  pdl_wait();
  constexpr int STEP = WARP ? 32 : 256;
  const int t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int row = WARP ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x, there = min(a.rows, max(0, state->counted - a.row0));
  auto sum_all = [&](float v) { return WARP ? warp_sum(v) : block_sum(v, red); };
  auto max_all = [&](float v) { return WARP ? warp_max(v) : block_max(v, red); };
  KT* kept = reinterpret_cast<KT*>(a.kept) + (a.kept ? row * a.ld_kept : 0);
  const int vecs = (a.v + 7) / 8, per = (vecs + gridDim.y - 1) / gridDim.y;
  const int v0 = blockIdx.y * per, v1 = min(vecs, v0 + per);
  if (row >= there) {  // rows up to the next multiple of 64 enter the reduction over rows: zero
    if (!a.kept || row >= ((there + 63) & ~63)) return;
    const float zero[8] = {};
    for (int i = v0 + t; i < v1; i += STEP) {
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
  for (int i = t; i < a.tiles; i += STEP) top = fmaxf(top, st[i].x);
  top = max_all(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f, linear = 0.f;
  for (int i = t; i < a.tiles; i += STEP) {
    sum += st[i].y * expf(st[i].x - ref);
    if (a.linear) linear += a.linear[(long long)row * a.tiles + i];
  }
  sum = sum_all(sum);
  if (a.linear) linear = sum_all(linear);
  // lse - l_t from differences with the maximum: lse itself is rounded at the size of the logits, and a row that is all but
  // certain of its target has only the difference left (of its loss, and of 1 - p).
  const float log_sum = logf(sum), lse = ref + log_sum, lt = a.target_logit[row], short_of = log_sum - (lt - ref);
  const int target = a.row_target[a.row0 + row];
  if (t == 0 && blockIdx.y == 0) {
    float loss = a.smoothing == 0.f ? short_of : (1.f - a.smoothing) * short_of + a.smoothing * (lse - linear / (float)a.v);
    if (a.z != 0.f) loss += a.z * lse * lse;
    if (a.none) a.loss[a.row_of[a.row0 + row]] = loss;
    else a.loss_rows[a.row0 + row] = loss;
  }
  if (!a.kept) return;
  const int shift = a.stat == 64 ? 6 : 7;
  constexpr float unit = is_half<GT>() ? L_HALF_SCALE : 1.f;
  float up = a.grad ? a.grad[a.row_of[a.row0 + row]] : 1.f;
  if constexpr (is_half<GT>())
    if (a.grad) {
      int e;
      up = split_power(up, e);  // (2^e: row_scale, and dw's h)
    }
  const float c = up * unit;
  const float more = 2.f * a.z * lse, pull = 1.f + more, uniform = a.smoothing / (float)a.v;
  const float scale = sizeof(KT) == 4 ? 1.f : 1.f / L_KEEP_SCALE;
  // the target's element from its fp32 logit: p - 1 without cancellation
  const float at_target = c * (expm1f(-short_of) + more * expf(-short_of) + (a.smoothing - uniform)), inverse = 1.f / sum;
  for (int i = v0 + t; i < v1; i += STEP) {
    const float f = expf(st[(i * 8) >> shift].x - ref) * inverse * scale * pull;
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
  pdl_wait();
  const int n = state->counted;
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) s += rows[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) *loss = mean ? s / (float)max(n, 1) : s;
}

// x *= *factor, unless that is one (then nothing is read): the upstream gradient of a loss, which is nearly always one.
template <typename T>
__global__ void __launch_bounds__(256) lce_scale_kernel(T* __restrict__ x, long long n, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.f) return;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256)
    x[i] = from_f32<T>(to_f32(x[i]) * f);
}
template <typename T>
int scale(void* x, long long n, const float* factor, cudaStream_t stream) {
  const long long want = (n + 255) / 256, most = 16LL * psgd_num_sms();
  lce_scale_kernel<T><<<(int)(want < most ? want : most), 256, 0, stream>>>(reinterpret_cast<T*>(x), n, factor);
  return cudaGetLastError() == cudaSuccess ? PSGD_OK : PSGD_ELAUNCH;
}

// Joins the splits of a gradient: out[row] = alpha (or the row's factor) * sum over splits, in their order. Rows are the counted ones through
// row_of, or all M of them as they are. V: values at a time (N a multiple, or 1).
template <typename T, int V>
__global__ void __launch_bounds__(256) lce_join_kernel(const float* __restrict__ part, int splits, int M, int N,
                                                       long long ld_part, int row0, const int* __restrict__ row_of,
                                                       const float* __restrict__ row_scale, int lifted, T* __restrict__ out,
                                                       const LceState* state) {
  pdl_wait();
  const int there = row_of ? min(M, max(0, state->counted - row0)) : M, per_row = N / V;
  const long long n = (long long)there * per_row, plane = M * ld_part;
  const float alpha = lce_alpha<T>(state, lifted);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int r = (int)(i / per_row), c = (int)(i - (long long)r * per_row) * V;
    float s[V] = {};
#pragma unroll 4
    for (int k = 0; k < splits; ++k) {
      float x[V];
      load_vec<float, V>(part + k * plane + r * ld_part + c, x);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += x[e];
    }
    const float by = is_half<T>() && row_scale ? row_scale[row0 + r] : alpha;
#pragma unroll
    for (int e = 0; e < V; ++e) s[e] *= by;
    store_vec<T, V>(out + (long long)(row_of ? row_of[row0 + r] : r) * N + c, s);
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
  int limbs, tiles, piece, pieces, splits, splits_w, bn, bn_grads, stat;
  bool stage_w;
  long long ld_h, ld_w, ld_kept, ld_part, h_plane, w_plane, g_plane;
  size_t state, rank, row_of, row_target, loss_rows, row_scale, target_logit, stats, linear, h, w, kept, g, part, part_w, acc, bytes;
};

// Whether the operands are three bf16 limbs: fp32 ones, and 16-bit ones of up to 2^20 products, where limbs cost the call
// 6 us on the GPU (7 x 32 x 85: 22.6 us against 16.4), less than its host code takes (28 us), and leave the gradients no rounding
// but their own. Beyond, g is rounded to 16 bits (1e-3 of the gradients in the 2-norm, less where dw's sum over n or dh's over v
// has many terms of one size, more where one term leads: 1.7e-3 at most, as much as their own rounding): limbs would cost 10
// us and more from 2^24 products on, and six times the products in the end.
bool wide_operands(const PsgdLce& a) {
  return a.dtype == PSGD_F32 || (double)a.n * a.v * a.d <= (double)(1 << 20);
}

Layout layout(const PsgdLce& a) {
  Layout l = {};
  const bool wide = wide_operands(a);
  auto up = [](long long x, long long m) { return (x + m - 1) / m * m; };
  l.limbs = wide ? L_LIMBS : 1;
  // Narrow tiles (128 columns) where wide ones would not go twice around the clusters; fp32 always (three limbs a stage).
  const int clusters = psgd_num_sms() / 2;
  const long long wide_tiles = (((long long)a.n + LM - 1) / LM) * ((a.v + 255) / 256);
  l.bn = wide || wide_tiles < 2 * clusters ? 128 : 256;
  const long long wide_grads = (((long long)a.n + LM - 1) / LM + (a.v + LM - 1) / LM) * ((a.d + 255) / 256);
  // (and for widths that fill their last wide tile to less than half: 4 / 3 of the products of narrow ones, or twice)
  l.bn_grads = wide || wide_grads < 2 * clusters || (a.d <= 384 && (a.d + 127) / 128 % 2) ? 128 : 256;
  l.ld_part = up(a.d, 8);
  l.stat = l.bn / 2;
  l.tiles = (a.v + l.stat - 1) / l.stat;
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
  // dh reduces over the vocabulary, dw over the tokens, and either may have few tiles. They need the same number of
  // products: splits until a unit is at most a quarter of a cluster's share of both keep the shares even.
  const long long tiles_n = (a.d + l.bn_grads - 1) / l.bn_grads;
  const long long tiles_h = ((piece + LM - 1) / LM) * tiles_n, tiles_w = (((long long)a.v + LM - 1) / LM) * tiles_n;
  const long long kb_h = (a.v + LK - 1) / LK, kb_w = (piece + LK - 1) / LK;
  const long long quarter = (tiles_h * (kb_h + L_UNIT) + tiles_w * (kb_w + L_UNIT)) / (4 * clusters) + 1;
  auto split = [&](long long tiles, long long kb) -> int {
    long long n = (kb + quarter - 1) / quarter;
    if (n > (kb + 7) / 8) n = (kb + 7) / 8;
    if (n > 16) n = 16;
    return tiles >= 4 * clusters ? 1 : (int)n;  // (many units are even enough, and partial sums are not free)
  };
  l.splits = split(tiles_h, kb_h);
  l.splits_w = l.pieces > 1 ? 1 : split(tiles_w, kb_w);
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
  l.row_scale = take(!wide && a.dtype == PSGD_F16 && a.grads && a.reduction == PSGD_REDUCE_NONE ? 4ull * a.n : 0);
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
    l.part = take(l.splits > 1 ? 4ull * l.splits * piece * l.ld_part : 0);
    l.part_w = take(l.splits_w > 1 ? 4ull * l.splits_w * a.v * l.ld_part : 0);
    l.acc = take(l.pieces > 1 && a.dtype != PSGD_F32 ? 4ull * a.v * l.ld_part : 0);
  }
  l.bytes = at;
  return l;
}

bool valid(const PsgdLce& a) {
  return a.n >= 0 && a.d >= 1 && a.v >= 1 && a.dtype >= 0 && a.dtype <= 2 && a.ld_h >= a.d && a.ld_w >= a.d &&
         a.reduction >= 0 && a.reduction <= 2 && a.piece_bytes >= 0 && a.n <= PSGD_LCE_MAX && a.d <= PSGD_LCE_MAX && a.v <= PSGD_LCE_MAX;
}

template <typename OP, typename OUT, int LIMBS, int BN, bool LOGITS>
int product(const LceArgs& args, cudaStream_t stream) {
  using C = LceCfg<LIMBS, BN, LOGITS>;
  auto k = lce_product_kernel<OP, OUT, LIMBS, BN, LOGITS>;
  static std::atomic<unsigned long long> done{0};
  if (int rc = allow_smem(k, C::SMEM, done)) return rc;
  long long units = 0;  // (at most; the counted rows decide)
  for (int i = 0; i < args.nproblems; ++i) {
    const LceProblem& p = args.p[i];
    units += (long long)((p.M + LM - 1) / LM) * ((p.N + BN - 1) / BN) * p.splits;
  }
  const long long clusters = psgd_num_sms() / 2;
  return pdl_launch(k, dim3(2 * (int)(units < clusters ? units : clusters)), dim3(L_THREADS), C::SMEM, stream, args);
}
template <typename OP, typename OUT, int LIMBS, bool LOGITS>
int product_bn(int bn, const LceArgs& args, cudaStream_t stream) {
  if constexpr (LIMBS == 1)
    if (bn == 256) return product<OP, OUT, 1, 256, LOGITS>(args, stream);
  return product<OP, OUT, LIMBS, 128, LOGITS>(args, stream);
}

// T: type of h, w and the gradients. OP: operand type of the tensor cores; KT: type of the kept exponentials.
template <typename T, bool WIDE>
int run(const PsgdLce& a, int* err, cudaStream_t stream) {
  using OP = std::conditional_t<WIDE, __nv_bfloat16, T>;
  using KT = std::conditional_t<WIDE, float, __half>;
  constexpr bool half = is_half<OP>();
  constexpr int LIMBS = WIDE ? L_LIMBS : 1;
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
  const bool none = a.reduction == PSGD_REDUCE_NONE, mean = a.reduction == PSGD_REDUCE_MEAN;

  const LcePlan plan = {a.target, a.ignore_index, a.grad, rank, row_of, row_target, a.loss, state, err, a.n, a.v, a.reduction, half};
  const LceStage<T> sh = {reinterpret_cast<const T*>(a.h), a.ld_h, l.ld_h, l.h_plane, h,
                          reinterpret_cast<T*>(a.grads ? a.dh : nullptr), a.n, (int)((a.n + 7LL) / 8 + 8)};
  const LceStage<T> sw = {reinterpret_cast<const T*>(a.w), a.ld_w, l.ld_w, l.w_plane, const_cast<uint16_t*>(w),
                          nullptr, a.v, l.stage_w ? (a.v + 7) / 8 : 0};
  const bool vec = a.d % 8 == 0 && aligned16(a.h) && a.ld_h * sizeof(T) % 16 == 0 && aligned16(sh.dh) &&
                   (!l.stage_w || (aligned16(a.w) && a.ld_w * sizeof(T) % 16 == 0));
  const dim3 stage_grid(sh.blocks + sw.blocks);
  if (a.n <= PLAN_INLINE) {
    auto k = vec ? lce_stage_kernel<T, WIDE, true, true> : lce_stage_kernel<T, WIDE, false, true>;
    k<<<stage_grid, 256, 0, stream>>>(sh, sw, a.d, plan);
    if (cudaGetLastError() != cudaSuccess) return PSGD_ELAUNCH;
  } else {
    lce_plan_kernel<<<1, 1024, 0, stream>>>(plan);
    if (cudaGetLastError() != cudaSuccess) return PSGD_ELAUNCH;
    if (int rc = pdl_launch(vec ? lce_stage_kernel<T, WIDE, true, false> : lce_stage_kernel<T, WIDE, false, false>, stage_grid, dim3(256),
                            0, stream, sh, sw, a.d, plan))
      return rc;
  }

  // fp16 by rows: what to multiply dh's rows and dw with
  const bool by_rows = half && a.grads && none && a.grad;
  float* row_scale = reinterpret_cast<float*>(ws + l.row_scale);
  if constexpr (half)
    if (by_rows)
      if (int rc = pdl_launch(lce_reach_kernel, dim3((a.n + 7) / 8), dim3(256), 0, stream, (const __half*)h, l.ld_h, a.d, a.grad,
                              (const int*)row_of, row_scale, state))
        return rc;

  LceArgs args = {};
  args.state = state;
  args.err = err;
  args.wait_ns = wait_limit();
  for (int piece = 0; piece < l.pieces; ++piece) {
    const int row0 = piece * l.piece, rows = a.n - row0 < l.piece ? a.n - row0 : l.piece;
    const int rows64 = (rows + 63) / 64 * 64;
    LceProblem& p = args.p[0];
    p = LceProblem{};
    p.splits = 1;
    for (int i = 0; i < l.limbs; ++i) {
      if (int rc = encode(&p.ta[i], h + i * l.h_plane + (long long)row0 * l.ld_h, half, rows, a.d, l.ld_h, 128)) return rc;
      if (int rc = encode(&p.tb[i], w + i * l.w_plane, half, a.v, a.d, ld_w, l.bn / 2)) return rc;
    }
    p.M = rows, p.N = a.v, p.K = a.d, p.dyn = 1, p.row0 = row0;
    args.nproblems = 1;
    // The loss is fp32 whatever the operands are: sums of at most 1024 products (512 for fp32 operands) stay in the tensor
    // cores, which keeps their truncation at 1e-6 of a logit.
    args.chunk = LIMBS == 1 ? 16 : 8;
    args.loss_rows = nullptr;
    LceLogits& g = args.logits;
    g.stats = reinterpret_cast<float2*>(ws + l.stats);
    g.linear = a.label_smoothing != 0.f ? reinterpret_cast<float*>(ws + l.linear) : nullptr;
    g.target_logit = reinterpret_cast<float*>(ws + l.target_logit);
    g.row_target = row_target;
    g.kept = a.grads ? ws + l.kept : nullptr;
    g.ld_kept = l.ld_kept;
    g.tiles = l.tiles;
    if (int rc = product_bn<OP, KT, LIMBS, true>(l.bn, args, stream)) return rc;

    LceRows r = {};
    r.stats = g.stats, r.linear = g.linear, r.target_logit = g.target_logit, r.row_target = row_target, r.row_of = row_of;
    r.grad = none ? a.grad : nullptr;
    r.loss_rows = loss_rows, r.loss = a.loss, r.kept = g.kept, r.limbs = reinterpret_cast<uint16_t*>(ws + l.g);
    r.ld_kept = l.ld_kept, r.plane = l.g_plane, r.v = a.v, r.tiles = l.tiles, r.row0 = row0, r.rows = rows, r.none = none;
    r.smoothing = a.label_smoothing, r.z = a.z_loss, r.stat = l.stat;
    int cols = a.grads ? (2 * psgd_num_sms() + rows64 - 1) / rows64 : 1;
    if (cols > (a.v + 2047) / 2048) cols = (a.v + 2047) / 2048;
    const bool by_warp = a.v <= 2048 && rows64 >= 2 * psgd_num_sms();  // (one warp's trip over a row is then no longer)
    if (int rc = by_warp ? pdl_launch(lce_rows_kernel<KT, OP, true>, dim3(rows64 / 8), dim3(256), 0, stream, r, (const LceState*)state)
                         : pdl_launch(lce_rows_kernel<KT, OP, false>, dim3(rows64, cols), dim3(256), 0, stream, r, (const LceState*)state))
      return rc;
    if (!a.grads) continue;
    if constexpr (half)
      if (by_rows && a.dw)
        if (int rc = pdl_launch(lce_lift_kernel, dim3((rows + 7) / 8), dim3(256), 0, stream, (__half*)h, l.ld_h, a.d, a.grad,
                                (const int*)row_of, row0, rows, (const LceState*)state))
          return rc;

    const uint16_t* gm = reinterpret_cast<const uint16_t*>(ws + l.g);
    args.nproblems = 0;
    if (a.dh) {  // dh = g w: g K-major, w (rows of K = vocabulary) MN-major
      LceProblem& ph = args.p[args.nproblems++] = LceProblem{};
      for (int i = 0; i < l.limbs; ++i) {
        if (int rc = encode(&ph.ta[i], gm + i * l.g_plane, half, rows, a.v, l.ld_kept, 128)) return rc;
        if (int rc = encode(&ph.tb[i], w + i * l.w_plane, half, a.v, a.d, ld_w, 64)) return rc;
      }
      ph.b_mn = 1, ph.M = rows, ph.N = a.d, ph.K = a.v, ph.dyn = 1, ph.row0 = row0, ph.splits = l.splits;
      ph.row_scale = by_rows ? row_scale : nullptr;
      ph.row_of = row_of, ph.out = a.dh, ph.ld_out = a.d, ph.ld_part = l.ld_part;
      ph.part = l.splits > 1 ? reinterpret_cast<float*>(ws + l.part) : nullptr;
    }
    if (a.dw) {  // dw = g^T h: both with rows of K = tokens
      LceProblem& pw = args.p[args.nproblems++] = LceProblem{};
      for (int i = 0; i < l.limbs; ++i) {
        if (int rc = encode(&pw.ta[i], gm + i * l.g_plane, half, rows64, a.v, l.ld_kept, 64)) return rc;
        if (int rc = encode(&pw.tb[i], h + i * l.h_plane + (long long)row0 * l.ld_h, half, rows64, a.d, l.ld_h, 64)) return rc;
      }
      pw.a_mn = pw.b_mn = 1, pw.M = a.v, pw.N = a.d, pw.K = rows, pw.dyn = 2, pw.row0 = row0, pw.splits = l.splits_w;
      pw.lifted = by_rows;
      pw.out = a.dw, pw.ld_out = a.d, pw.ld_part = l.ld_part;
      pw.part = l.splits_w > 1 ? reinterpret_cast<float*>(ws + l.part_w) : nullptr;
      if (l.pieces > 1) {
        float* acc = sizeof(T) == 4 ? reinterpret_cast<float*>(a.dw) : reinterpret_cast<float*>(ws + l.acc);
        pw.acc = piece > 0 ? acc : nullptr;
        pw.acc_out = piece + 1 < l.pieces ? acc : nullptr;
        pw.ld_acc = sizeof(T) == 4 ? a.d : l.ld_part;
      }
    }
    args.chunk = LIMBS == 1 ? 1 << 20 : 8;  // (a 16-bit gradient's own rounding is a hundred times the truncation)
    if (!none && piece + 1 == l.pieces) args.loss_rows = loss_rows, args.loss = a.loss, args.mean = mean;
    if (int rc = product_bn<OP, T, LIMBS, false>(l.bn_grads, args, stream)) return rc;
    auto join = [&](const LceProblem& p, void* out) {
      const bool eight = a.d % 8 == 0 && aligned16(out);
      const long long n = (long long)p.M * a.d / (eight ? 8 : 1), want = (n + 255) / 256, most = 8LL * psgd_num_sms();
      return pdl_launch(eight ? lce_join_kernel<T, 8> : lce_join_kernel<T, 1>, dim3((int)(want < most ? want : most)),
                        dim3(256), 0, stream, (const float*)p.part, p.splits, p.M, a.d, p.ld_part, row0, p.row_of,
                        p.row_scale, p.lifted, reinterpret_cast<T*>(out), (const LceState*)state);
    };
    for (int i = 0; i < args.nproblems; ++i)
      if (args.p[i].part)
        if (int rc = join(args.p[i], args.p[i].out)) return rc;
  }
  if (!none && !a.grads)
    return pdl_launch(lce_loss_kernel, dim3(1), dim3(1024), 0, stream, (const float*)loss_rows, (const LceState*)state, (int)mean,
                  a.loss);
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
      !aligned16(a->workspace) || (a->grads && !a->dh && !a->dw))
    return PSGD_EINVAL;
  if (a->workspace_bytes < psgd_lce_workspace(a)) return PSGD_ESPACE;
  const bool wide = wide_operands(*a);
  switch (a->dtype) {
    case PSGD_F32: return run<float, true>(*a, dev_err, stream);
    case PSGD_BF16: return wide ? run<__nv_bfloat16, true>(*a, dev_err, stream) : run<__nv_bfloat16, false>(*a, dev_err, stream);
    default: return wide ? run<__half, true>(*a, dev_err, stream) : run<__half, false>(*a, dev_err, stream);
  }
}

extern "C" int psgd_lce_scale(void* x, int dtype, long long n, const float* factor, cudaStream_t stream) {
  using namespace psgd;
  if (n < 0 || !factor || (n > 0 && !x)) return PSGD_EINVAL;
  if (n == 0) return PSGD_OK;
  switch (dtype) {
    case PSGD_F32: return scale<float>(x, n, factor, stream);
    case PSGD_BF16: return scale<__nv_bfloat16>(x, n, factor, stream);
    case PSGD_F16: return scale<__half>(x, n, factor, stream);
    default: return PSGD_EINVAL;
  }
}
