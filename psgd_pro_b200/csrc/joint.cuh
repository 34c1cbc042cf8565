// The joint between two blocks of a network, one pass over its rows (d elements each):
//   u = post(y) (a norm, or y itself), k = dropout(u), out = x + scale * gate * k, normed = pre(out)
// and its backward pass. rms norm: a / sqrt(mean a^2 + eps) * weight; layer norm: (a - mean) / sqrt(var + eps) * weight
// + bias. statistics: (mean, 1 / deviation) of post, then of pre, per row.
//
// Both passes would be bound by memory traffic (a row in and out once), and the forward pass nearly is (8192 x 2048 bf16,
// rms norms and a gate: 28 us, 4.8 TB/s of 6.46 that a copy has; 23.6 us under the profiler). About 100 instructions per thread for 8 elements are
// what the SMs can issue in the time that the copies take, so arithmetic goes two elements to an instruction
// (f32x2), everything a call does not have is compiled out, what is constant along a column is kept out of the rows'
// loop, and a thread has 16 elements, which halves the share of the sums over a row against 8 (46 us, and 28 million
// warp instructions against 12). The rows to come are copied to shared memory asynchronously, each thread its own
// 16-byte pieces (which therefore need no barrier).
//
// A row belongs to a group of `tpr` threads (whole warps) and a thread to 8 * NV elements of it (Place). A block holds
// blockDim.y groups, each with rows of its own, whose threads meet at a named barrier of the group.
#pragma once
#include "elem.cuh"

namespace psgd {

constexpr int JOINT_MAX_D = PSGD_JOINT_MAX_D;
// Dynamic shared memory that needs no asking (48 KB with the kernels' static one), and what is asked for otherwise.
constexpr int JOINT_SMEM_FREE = 40 * 1024, JOINT_SMEM_MOST = 224 * 1024;
constexpr int JOINT_MAX_GROUPS = 8;  // of a block, where a group has more than a warp
// Kernels by the elements that a thread has of a row and the threads of a block: 8 (rows of up to 256 elements, a warp
// each), 16 (up to 2048 elements: 128 threads; up to 4096: 256; beyond: 512, whose registers do not hold all the sums).
enum JointWidth { W8 = 0, W16 = 1, W16_256 = 2, W16_512 = 3 };
PSGD_HD constexpr int width_nv(int w) { return w == W8 ? 1 : 2; }
PSGD_HD constexpr int width_threads(int w) { return w == W16_512 ? 512 : w == W16_256 ? 256 : 128; }

// How rows are dealt out to blocks: consecutive ones, `per_block` each. With a gate a block holds whole gate groups
// (chunks = 0: a group of threads takes a gate group at a time and writes its gradient itself) or a chunk of one gate
// group (`chunks` to a gate group, whose gradient a block writes itself if there is one). A group of threads takes every blockDim.y-th row (gate group) of its block.
struct JointPlan {
  int blocks, per_block, chunks, per_gate;
  int tpr, groups, vec, nv, wide, stages, ring, smem;  // ring: bytes of shared memory before the backward pass's columns
  int slot[5];  // of dweight, dbias, dpost_weight, dpost_bias, dgate in `part` [slot][block][d up to 8], or -1
  int slots;
};

int joint_forward_f32(const PsgdJoint& j, const JointPlan& p, cudaStream_t stream);
int joint_forward_bf16(const PsgdJoint& j, const JointPlan& p, cudaStream_t stream);
int joint_forward_f16(const PsgdJoint& j, const JointPlan& p, cudaStream_t stream);
int joint_backward_f32(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream);
int joint_backward_bf16(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream);
int joint_backward_f16(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream);

// ---- two fp32 values in one register pair -----------------------------------------------------------------------------
struct F2 {
  unsigned long long v;
};
PSGD_DEVI F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
PSGD_DEVI F2 f2(float a) { return f2(a, a); }
PSGD_DEVI float2 un2(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
PSGD_DEVI F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
PSGD_DEVI F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
PSGD_DEVI F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
PSGD_DEVI float sum2(F2 a) {
  const float2 f = un2(a);
  return f.x + f.y;
}

PSGD_DEVI F2 where_nonzero(F2 m, F2 v) {  // v where m is not zero, zero elsewhere
  const float2 a = un2(m), b = un2(v);
  return f2(a.x != 0.f ? b.x : 0.f, a.y != 0.f ? b.y : 0.f);
}

// Eight 16-bit elements as four pairs.
template <typename T>
PSGD_DEVI void unpack8(uint4 a, F2* v) {
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2(w[i], T());
    v[i] = f2(f.x, f.y);
  }
}

// Bytes [by, by + 16) of the 32 bytes x, y (by < 16).
PSGD_DEVI uint4 from_byte(const uint4& x, const uint4& y, uint32_t by) {
  uint32_t z[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  if (by & 4u)
#pragma unroll
    for (int k = 0; k < 7; ++k) z[k] = z[k + 1];
  if (by & 8u)
#pragma unroll
    for (int k = 0; k < 5; ++k) z[k] = z[k + 2];
  const uint32_t bits = (by & 3u) * 8;
  return make_uint4(__funnelshift_r(z[0], z[1], bits), __funnelshift_r(z[1], z[2], bits), __funnelshift_r(z[2], z[3], bits),
                    __funnelshift_r(z[3], z[4], bits));
}
PSGD_DEVI uint4 shuffle_up(const uint4& v) {
  return make_uint4(__shfl_up_sync(0xffffffffu, v.x, 1), __shfl_up_sync(0xffffffffu, v.y, 1),
                    __shfl_up_sync(0xffffffffu, v.z, 1), __shfl_up_sync(0xffffffffu, v.w, 1));
}
// The elements of a row that are this thread's: vectors of eight, each H pieces of 16 bytes (T of 16 bits: one of 8
// elements; fp32: two of 4), a piece at e(i, h), neighbouring threads' pieces side by side. VEC: every row starts on a
// 16-byte boundary and d is a multiple of 8, so pieces are whole and aligned. Otherwise a piece straddles two aligned
// ones, of which this thread moves one and a neighbour the other (see Ring16::read and store_row), and the last
// piece may be cut off by the row's end.
template <typename T, bool VEC>
struct Place {
  static constexpr int H = (int)sizeof(T) / 2, E = 8 / H;  // pieces to a vector, elements to a piece
  int d, tpr, t;
  PSGD_DEVI Place(int d_) : d(d_), tpr(blockDim.x), t(threadIdx.x) {}
  PSGD_DEVI int e(int i, int h) const { return ((i * H + h) * tpr + t) * E; }
  PSGD_DEVI bool piece(int i, int h) const { return e(i, h) < d; }
  PSGD_DEVI bool whole(int i, int h) const { return VEC ? piece(i, h) : e(i, h) + E <= d; }
  PSGD_DEVI bool any(int i) const { return piece(i, 0); }
  PSGD_DEVI bool has(int i, int k) const { return e(i, k / E) + (VEC ? 0 : k % E) < d; }
  PSGD_DEVI F2 only(F2 v, int i, int k) const {  // elements 2 k, 2 k + 1 of vector i, zero where there are none
    if constexpr (VEC) {
      return has(i, 2 * k) ? v : f2(0.f);
    } else {
      const float2 f = un2(v);
      return f2(has(i, 2 * k) ? f.x : 0.f, has(i, 2 * k + 1) ? f.y : 0.f);
    }
  }
  // Vector i of a row of T or of fp32 (a parameter, a sum, a gate); zero beyond d. Aligned where VEC.
  template <typename S>
  PSGD_DEVI void load(const S* row, int i, F2* v) const {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      F2* to = v + h * (E / 2);
      if (!piece(i, h)) {
#pragma unroll
        for (int k = 0; k < E / 2; ++k) to[k] = f2(0.f);
      } else if constexpr (!VEC) {
        float f[E];
#pragma unroll
        for (int k = 0; k < E; ++k) f[k] = e(i, h) + k < d ? to_f32(row[e(i, h) + k]) : 0.f;
#pragma unroll
        for (int k = 0; k < E / 2; ++k) to[k] = f2(f[2 * k], f[2 * k + 1]);
      } else if constexpr (sizeof(S) == 4) {
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
          const float4 a = reinterpret_cast<const float4*>(row + e(i, h))[q];
          to[2 * q] = f2(a.x, a.y), to[2 * q + 1] = f2(a.z, a.w);
        }
      } else {
        unpack8<S>(*reinterpret_cast<const uint4*>(row + e(i, h)), to);
      }
    }
  }
  // Vector i into a row of fp32 sums, aligned and as long as d rounded up to 8.
  PSGD_DEVI void store_sums(float* row, int i, const F2* v) const {
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (piece(i, h))
#pragma unroll
        for (int q = 0; q < E / 4; ++q) {
          const float2 a = un2(v[h * (E / 2) + 2 * q]), b = un2(v[h * (E / 2) + 2 * q + 1]);
          reinterpret_cast<float4*>(row + e(i, h))[q] = make_float4(a.x, a.y, b.x, b.y);
        }
  }
  PSGD_DEVI uint4 pack(int h, const F2* v) const {
    float f[E];
#pragma unroll
    for (int k = 0; k < E / 2; ++k) {
      const float2 a = un2(v[h * (E / 2) + k]);
      f[2 * k] = a.x, f[2 * k + 1] = a.y;
    }
    if constexpr (H == 2) return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    else return make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()), pack2(f[4], f[5], T()), pack2(f[6], f[7], T()));
  }
  PSGD_DEVI static T element(const uint4& w, int k) {  // k is known where it is compiled
    const uint32_t x = k * (int)sizeof(T) / 4 == 0 ? w.x : k * (int)sizeof(T) / 4 == 1 ? w.y : k * (int)sizeof(T) / 4 == 2 ? w.z : w.w;
    if constexpr (H == 2) {
      return __uint_as_float(x);
    } else {
      const uint16_t half = (uint16_t)(k & 1 ? x >> 16 : x & 0xFFFFu);
      return *reinterpret_cast<const T*>(&half);
    }
  }
  // Vector i into a row of T; every thread of the warp calls it. Without VEC, where the row lies `off` bytes past a
  // boundary, a thread stores the aligned 16 bytes that end in its piece: the last `off` bytes of the piece before and
  // the first ones of its own. What a warp has no neighbour for, and the row's end, go element by element.
  PSGD_DEVI void store(T* row, int i, const F2* v) const {
    if constexpr (VEC) {
#pragma unroll
      for (int h = 0; h < H; ++h)
        if (piece(i, h)) *reinterpret_cast<uint4*>(row + e(i, h)) = pack(h, v);
    } else {
      const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;
      const int lane = t & 31, back = (int)(off / sizeof(T));  // elements that the thread's own store leaves to the next
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const uint4 mine = pack(h, v);
        const int at = e(i, h);
        uint4 out = mine;
        if (off) out = from_byte(shuffle_up(mine), mine, 16u - off);
        const bool full = at - back + E <= d && (lane > 0 || off == 0);
        if (full) *reinterpret_cast<uint4*>(row + at - back) = out;
        // The first thread's own elements, the last one's left-over ones, and the row's end (where the last thread's store is cut
        // off, nothing is left over).
        const bool rest = full && lane == 31 && off;
        if (!full || rest) {
          const int first = full ? at : at - back, least = full ? E - back : lane > 0 ? 0 : back;
          if (full) out = mine;
#pragma unroll
          for (int k = 0; k < E; ++k)
            if (k >= least && first + k < d) row[first + k] = element(out, k);
        }
      }
    }
  }
  // A parameter vector of fp32 or of T, `otherwise` where it is missing; zero beyond d in any case (the sums over a row rely
  // on it).
  PSGD_DEVI void param(const void* p, int dtype, float otherwise, int i, F2* v) const {
    if (!p) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = only(f2(otherwise), i, k);
    } else if (dtype == PSGD_F32) {
      load(reinterpret_cast<const float*>(p), i, v);
    } else {
      load(reinterpret_cast<const T*>(p), i, v);
    }
  }
  // v with what dropout does not keep set to zero.
  PSGD_DEVI void drop(const Keep& keep, long long row, int i, F2* v) const {
    const unsigned long long at0 = (unsigned long long)row * d;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const unsigned long long first = at0 + e(i, h);
      if constexpr (VEC) {  // (d is a multiple of 8: a piece lies in one block of the generator)
        const uint4 words = keep.block(first >> 3);
        const bool upper = H == 2 && (first & 4);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          const uint32_t w = upper ? word_of(words, k + 2) : word_of(words, k);
          const float2 f = un2(v[h * (E / 2) + k]);
          v[h * (E / 2) + k] = f2(keep.low(w) ? f.x : 0.f, keep.high(w) ? f.y : 0.f);
        }
      } else {
        const uint32_t o = (uint32_t)first & 7u;
        uint32_t m = keep.mask8(first >> 3) >> o;
        if (o + E > 8) m |= keep.mask8((first >> 3) + 1) << (8 - o);
#pragma unroll
        for (int k = 0; k < E / 2; ++k) {
          const float2 f = un2(v[h * (E / 2) + k]);
          v[h * (E / 2) + k] = f2((m >> (2 * k)) & 1u ? f.x : 0.f, (m >> (2 * k + 1)) & 1u ? f.y : 0.f);
        }
      }
    }
  }
};

// Sum of v[0..N) over the threads of a group of at most WARPS warps. `red` holds two buffers taken in turn: a thread writes
// one again only after the barrier of the other's sum, which every thread reaches after its reads of the first. The
// places of warps that are not there stay zero.
template <int N, int WARPS>
struct GroupSum {
  static_assert(WARPS % 4 == 0, "sums are read four at a time");
  static constexpr int FLOATS = 2 * JOINT_MAX_GROUPS * WARPS * N;
  float* at;
  int tpr, turn;
  PSGD_DEVI GroupSum(float* red) : at(red + threadIdx.y * (WARPS * N)), tpr(blockDim.x), turn(0) {
    if (tpr == 32) return;
    for (int i = threadIdx.y * blockDim.x + threadIdx.x; i < FLOATS; i += blockDim.x * blockDim.y) red[i] = 0.f;
    __syncthreads();
  }
  PSGD_DEVI void operator()(float* v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
    if (tpr == 32) return;
    float* to = at + turn;
    turn ^= JOINT_MAX_GROUPS * WARPS * N;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < N; ++k) to[k * WARPS + (threadIdx.x >> 5)] = v[k];
    named_sync(1 + threadIdx.y, tpr);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < WARPS; w += 4) {
        const float4 b = *reinterpret_cast<const float4*>(to + k * WARPS + w);
        v[k] += (b.x + b.y) + (b.z + b.w);
      }
    }
  }
};

// ---- the rows to come -------------------------------------------------------------------------------------------------
// A ring of `stages` rows' pieces, ARR arrays each, in shared memory: this thread's 16-byte pieces, a block's threads
// side by side (no bank conflicts). fetch() starts a row's copies (null arrays are skipped), wait() waits for the oldest
// row, read() unpacks a piece of it. Without VEC the copies are of the aligned 16 bytes in which the thread's piece
// begins (never beyond the row's end), the last thread of a warp copies the next ones too, and read() takes the rest of
// the piece from the next thread's; what lies beyond d reads as zero. Every thread of a warp calls all of them.
template <typename T, bool VEC, int NV, int ARR>
struct Ring16 {
  using At = Place<T, VEC>;
  static constexpr int H = At::H;  // 16-byte pieces to 8 elements
  uint32_t base, apart, extra, extra_apart, stage, extra_stage, put, get;  // bytes
  int stages, put_turn, get_turn;
  PSGD_DEVI Ring16(void* smem, int s) : put(0), get(0), stages(s), put_turn(0), get_turn(0) {
    const uint32_t threads = blockDim.x * blockDim.y, thread = threadIdx.y * blockDim.x + threadIdx.x;
    apart = threads * 16;
    stage = apart * (ARR * NV * H);
    base = smem_u32(smem) + thread * 16;
    extra_apart = threads / 32 * 16;
    extra_stage = extra_apart * (ARR * NV * H);
    extra = smem_u32(smem) + stage * s + thread / 32 * 16;
  }
  PSGD_DEVI static void copy(uint32_t to, const void* p, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(p), "r"(n) : "memory");
  }
  PSGD_DEVI void fetch(const At& at, const T* const* rows, bool there) {
    if (!VEC) __syncwarp();  // (the row that was there has been read by the thread before, too)
    if (there)
#pragma unroll
      for (int a = 0; a < ARR; ++a)
        if (rows[a])
#pragma unroll
          for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int h = 0; h < H; ++h) {
              const int n = (a * NV + i) * H + h;
              if constexpr (VEC) {
                if (at.piece(i, h))
                  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + put + apart * n), "l"(rows[a] + at.e(i, h))
                               : "memory");
              } else {
                const char* p = reinterpret_cast<const char*>(rows[a] + at.e(i, h));
                const char* end = reinterpret_cast<const char*>(rows[a] + at.d);
                const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;
                p -= off;
                if (p < end) copy(base + put + apart * n, p, (int)min((long long)(end - p), 16LL));
                p += 16;
                if ((threadIdx.x & 31) == 31 && off && p < end)
                  copy(extra + put_turn * extra_stage + extra_apart * n, p, (int)min((long long)(end - p), 16LL));
              }
            }
    asm volatile("cp.async.commit_group;" ::: "memory");
    put += stage;
    if (++put_turn == stages) put = 0, put_turn = 0;
  }
  PSGD_DEVI void wait() {  // one group was committed for each of the stages - 1 rows after the oldest
    if (stages == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else if (stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (!VEC) __syncwarp();  // (the next thread's pieces are read, too)
  }
  PSGD_DEVI static uint4 word4(uint32_t at) {
    uint4 x;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(at) : "memory");
    return x;
  }
  // Vector i of array a, whose row is `row` (its address alone is used).
  PSGD_DEVI void read(const At& at, const T* row, int a, int i, F2* v) const {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int n = (a * NV + i) * H + h;
      uint4 x = make_uint4(0u, 0u, 0u, 0u);
      if constexpr (VEC) {
        if (at.piece(i, h)) x = word4(base + get + apart * n);
      } else {
        const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u;
        x = word4(base + get + apart * n);
        if (off)
          x = from_byte(x, word4((threadIdx.x & 31) == 31 ? extra + get_turn * extra_stage + extra_apart * n : base + get + apart * n + 16), off);
      }
      if constexpr (H == 2) {
        v[2 * h] = f2(__uint_as_float(x.x), __uint_as_float(x.y));
        v[2 * h + 1] = f2(__uint_as_float(x.z), __uint_as_float(x.w));
      } else {
        unpack8<T>(x, v);
      }
      if (!VEC && !at.whole(i, h))
#pragma unroll
        for (int k = 0; k < At::E / 2; ++k) v[h * (At::E / 2) + k] = at.only(v[h * (At::E / 2) + k], i, h * (At::E / 2) + k);
    }
  }
  PSGD_DEVI void next() {
    get += stage;
    if (++get_turn == stages) get = 0, get_turn = 0;
  }
};

// ---- forward ----------------------------------------------------------------------------------------------------------
constexpr int F_POST = 1, F_GATE = 2, F_LAYER = 4, F_DROP = 8, F_DIRECT = 16, F_RUNTIME = 32;

PSGD_HD constexpr int joint_forward_blocks(int w, int f) { return w == W8 ? 7 : w == W16 ? ((f & F_LAYER) || (f & F_RUNTIME) ? 3 : 4) : 1; }

// What is constant along a column is formed once: f = scale gate post_weight (and with it the post norm's bias), with the
// gate where it has one row; other gates multiply row by row.
template <typename T, bool VEC, int W, int F>
__global__ void __launch_bounds__(width_threads(W), joint_forward_blocks(W, F)) joint_forward_kernel(const PsgdJoint j, const JointPlan p) {
  constexpr int NV = width_nv(W), P = NV * 4;
  const bool post = F & F_RUNTIME ? j.post != 0 : bool(F & F_POST);
  const bool layer = F & F_RUNTIME ? j.kind == PSGD_NORM_LAYER : bool(F & F_LAYER);
  const bool drop = F & F_RUNTIME ? j.threshold != 0 : bool(F & F_DROP);
  extern __shared__ uint4 smem[];
  using Sum = GroupSum<1, width_threads(W) / 32>;
  __shared__ __align__(16) float red[Sum::FLOATS];
  const int d = j.d;
  const Place<T, VEC> at(d);
  Sum sum(red);
  const Keep keep(drop ? j.seed : 0, drop ? j.offset : 0, drop ? j.rng : nullptr, j.threshold);
  const float inv_d = 1.f / (float)d;
  const int step = gridDim.x * blockDim.y, rows_all = (int)j.rows, ld_x = (int)j.ld_x, ld_y = (int)j.ld_y;
  const bool one_gate = j.gate && p.per_gate == rows_all, row_gate = j.gate && !one_gate;
  Ring16<T, VEC, NV, 2> ring(smem, p.stages);

  auto sources = [&](int row, const T** rows) {
    rows[0] = reinterpret_cast<const T*>(j.x) + (long long)row * ld_x;
    rows[1] = reinterpret_cast<const T*>(j.y) + (long long)row * ld_y;
  };
  int row = blockIdx.x * blockDim.y + threadIdx.y, ahead = row;
  for (int s = 0; s + 1 < p.stages; ++s, ahead += step) {
    const T* rows[2];
    sources(ahead, rows);
    ring.fetch(at, rows, ahead < rows_all);
  }
  F2 w[P], b[P], f[P], fb[P];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const F2 c = f2(j.scale * (drop ? j.keep_scale : 1.f));
    at.param(j.weight, j.param_dtype, 1.f, i, w + i * 4);
    if (layer) at.param(j.bias, j.param_dtype, 0.f, i, b + i * 4);
    at.param(post ? j.post_weight : nullptr, j.param_dtype, 1.f, i, f + i * 4);
    if (post && layer) at.param(j.post_bias, j.param_dtype, 0.f, i, fb + i * 4);
    F2 g[4] = {c, c, c, c};
    if (one_gate) {
      at.load(reinterpret_cast<const T*>(j.gate), i, g);
#pragma unroll
      for (int k = 0; k < 4; ++k) g[k] = mul2(g[k], c);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[i * 4 + k] = mul2(f[i * 4 + k], g[k]);
      if (post && layer) fb[i * 4 + k] = mul2(fb[i * 4 + k], g[k]);
    }
  }
  // (mean, 1 / deviation) of a row (zero beyond d); the variance is a second pass over the registers: no cancellation
  auto statistics = [&](const F2* a, float& mean, float& r) {
    mean = 0.f;
    F2 q = f2(0.f);
    if (layer) {
#pragma unroll
      for (int i = 0; i < P; ++i) q = add2(q, a[i]);
      float s = sum2(q);
      sum(&s);
      mean = s * inv_d;
      q = f2(0.f);
      const F2 m = f2(-mean);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (at.any(i))
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const F2 c = at.only(add2(a[i * 4 + k], m), i, k);
            q = fma2(c, c, q);
          }
    } else {
#pragma unroll
      for (int i = 0; i < P; ++i) q = fma2(a[i], a[i], q);
    }
    float s = sum2(q);
    sum(&s);
    r = rsqrtf(s * inv_d + j.eps);
  };

  for (; row < rows_all; row += step) {
    F2 u[P], x[P];
    const T* rows[2];
    sources(ahead, rows);
    ring.fetch(at, rows, ahead < rows_all);
    ahead += step;
    ring.wait();
    sources(row, rows);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      ring.read(at, rows[0], 0, i, x + i * 4);
      ring.read(at, rows[1], 1, i, u + i * 4);
    }
    ring.next();
    T* po = reinterpret_cast<T*>(j.out) + (long long)row * d;
    T* pn = reinterpret_cast<T*>(j.normed) + (long long)row * d;
    float mean_y = 0.f, r_y = 1.f, mean_o, r_o;
    if (post) statistics(u, mean_y, r_y);
    const F2 ry = f2(r_y), my = f2(-mean_y * r_y);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      F2* ui = u + i * 4;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (post) ui[k] = layer ? fma2(ui[k], ry, my) : mul2(ui[k], ry);
        ui[k] = post && layer ? fma2(ui[k], f[i * 4 + k], fb[i * 4 + k]) : mul2(ui[k], f[i * 4 + k]);
      }
      if (row_gate) {
        const int g = p.per_gate == 1 ? row : (int)((unsigned)row / (unsigned)p.per_gate);
        F2 v[4];
        at.load(reinterpret_cast<const T*>(j.gate) + (long long)g * d, i, v);
#pragma unroll
        for (int k = 0; k < 4; ++k) ui[k] = mul2(ui[k], v[k]);
      }
      if (drop) at.drop(keep, row, i, ui);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[i * 4 + k] = add2(x[i * 4 + k], ui[k]);
      at.store(po, i, x + i * 4);
    }
    statistics(x, mean_o, r_o);
    const F2 ro = f2(r_o), mo = f2(-mean_o * r_o);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      F2 o[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        o[k] = layer ? fma2(x[i * 4 + k], ro, mo) : mul2(x[i * 4 + k], ro);
        o[k] = layer ? fma2(o[k], w[i * 4 + k], b[i * 4 + k]) : mul2(o[k], w[i * 4 + k]);
      }
      at.store(pn, i, o);
    }
    if (threadIdx.x == 0) reinterpret_cast<float4*>(j.stats)[row] = make_float4(mean_y, r_y, mean_o, r_o);
  }
}

// ---- backward ---------------------------------------------------------------------------------------------------------
// hat = (out - mean) r, dhat = d_normed w:  dx = d_out + r (dhat - hat mean(dhat hat) [- mean(dhat)]).
// Let m be dx where dropout kept the element (0 elsewhere), c its scale times the residual scale, yh the post norm's
// (y - mean) r (or y). Then, with f = c gate post_weight constant along a column (of a gate group):
//   dy = f m, through the post norm as above;  A = sum m yh and B = sum m over rows give
//   dpost_weight = c gate A, dpost_bias = c gate B, dgate = c (post_weight A + post_bias B): one multiply-add a row for
//   three gradients. dweight = sum d_normed hat, dbias = sum d_normed.
// Bound by the latency of its instructions, and of the two sums over a row that follow each other, with 16 warps on an SM to
// hide it (8192 x 2048 bf16, rms norms and a gate: 49 us with the last step, of which 41 us here at 54% of the issue slots, 4.9
// TB/s; 16384 x 1024, layer norm and dropout: 43 us, the generator being a third of it): five sixths of the instructions are unpacking, the two sums over a row and the multiply-adds that the
// formulas ask for.
// The sums over rows are kept in registers and written once a block, as rows of `part`, which
// joint_reduce_kernel adds in a fixed order.
struct JointRows {  // a group's rows: every groups-th one, or (direct) every groups-th gate group's
  int row, g, end, per_gate, groups;
  bool direct;
  PSGD_DEVI bool there() const { return direct ? g < end : row < end; }
  PSGD_DEVI bool last_of_gate() const { return row + 1 == (g + 1) * per_gate; }
  PSGD_DEVI void next() {
    if (!direct) {
      row += groups;
    } else if (last_of_gate()) {
      g += groups;
      row = g * per_gate;
    } else {
      ++row;
    }
  }
};

// Threads of a block, and blocks that an SM holds, by the registers that a thread needs. Fewer and larger blocks leave fewer
// sums over rows to the last step, smaller ones even out the SMs (8192 x 2048, rms: 128 threads 52.7 us, 256 49.2, 512 48.4;
// 16384 x 1024, layer norm with dropout: 44.6, 43.2, 47.2).
PSGD_HD constexpr bool joint_heavy(int f) { return (f & F_RUNTIME) || (f & F_DIRECT) || ((f & F_POST) && (f & F_LAYER)); }
PSGD_HD constexpr int joint_backward_threads(int w, int f) {
  return w == W8 ? 256 : w == W16 ? ((f & F_LAYER) && (f & F_GATE) && !joint_heavy(f) ? 384 : 256) : width_threads(w);
}
PSGD_HD constexpr int joint_backward_blocks(int w, int f) {
  return w == W8 ? (joint_heavy(f) ? 2 : 3) : w == W16 && !joint_heavy(f) && !((f & F_LAYER) && (f & F_GATE)) ? 2 : 1;
}

// A thread's own copies of column vectors in shared memory: what each row needs once costs a load there, not registers.
template <int P>
struct Columns {
  uint32_t base, apart;
  PSGD_DEVI Columns(uint32_t at, int index) {
    apart = blockDim.x * blockDim.y * 16;
    base = at + index * (P / 2) * apart + (threadIdx.y * blockDim.x + threadIdx.x) * 16;
  }
  PSGD_DEVI void put(int i, const F2* v) const {  // the four pairs of vector i
#pragma unroll
    for (int k = 0; k < 2; ++k)
      asm volatile("st.shared.v2.b64 [%0], {%1, %2};" ::"r"(base + (i * 2 + k) * apart), "l"(v[2 * k].v), "l"(v[2 * k + 1].v)
                   : "memory");
  }
  PSGD_DEVI void get(int i, F2* v) const {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];"
                   : "=l"(v[2 * k].v), "=l"(v[2 * k + 1].v)
                   : "r"(base + (i * 2 + k) * apart)
                   : "memory");
  }
};

template <typename T, bool VEC, int W, int F>
__global__ void __launch_bounds__(joint_backward_threads(W, F), joint_backward_blocks(W, F))
    joint_backward_kernel(const PsgdJoint j, const JointPlan p, float* part) {
  constexpr int NV = width_nv(W), P = NV * 4;
  constexpr bool RT = F & F_RUNTIME;
  const bool post = RT ? j.post != 0 : bool(F & F_POST);
  const bool gate = RT ? j.gate != nullptr : bool(F & F_GATE);
  const bool layer = RT ? j.kind == PSGD_NORM_LAYER : bool(F & F_LAYER);
  const bool drop = RT ? j.threshold != 0 : bool(F & F_DROP);
  const bool direct = RT ? gate && p.chunks == 0 : bool(F & F_DIRECT);
  const bool use_y = post || gate;
  extern __shared__ uint4 smem[];
  constexpr int NS = RT || (F & F_LAYER) ? 2 : 1;
  using Sum = GroupSum<NS, width_threads(W) / 32>;
  __shared__ __align__(16) float red[Sum::FLOATS];
  const int d = j.d, dp = (d + 7) & ~7;
  const Place<T, VEC> at(d);
  pdl_trigger();
  Sum sum(red);
  const Keep keep(drop ? j.seed : 0, drop ? j.offset : 0, drop ? j.rng : nullptr, j.threshold);
  const float inv_d = 1.f / (float)d, c = j.scale * (drop ? j.keep_scale : 1.f);
  constexpr int ARRAYS = RT || (F & (F_POST | F_GATE)) ? 4 : 3;  // d_normed, d_out, out and, where it is needed, y
  Ring16<T, VEC, NV, ARRAYS> ring(smem, p.stages);

  JointRows it;
  it.groups = blockDim.y, it.direct = direct, it.per_gate = p.per_gate;
  int gate_row = 0;  // of a block that holds (part of) one gate group
  if (direct) {
    const int held = p.per_block / p.per_gate, g0 = blockIdx.x * held;
    it.g = g0 + threadIdx.y;
    it.end = min(g0 + held, (int)j.gates);
    it.row = it.g * p.per_gate;
  } else if (p.chunks) {
    gate_row = blockIdx.x / p.chunks;
    const int r0 = gate_row * p.per_gate + (blockIdx.x - gate_row * p.chunks) * p.per_block;
    it.row = r0 + threadIdx.y;
    it.end = min(r0 + p.per_block, (gate_row + 1) * p.per_gate);
    it.g = 0;
  } else {
    it.row = blockIdx.x * p.per_block + threadIdx.y;
    it.end = (int)min((blockIdx.x + 1LL) * p.per_block, j.rows);
    it.g = 0;
  }

  // f, per column, of a gate group
  auto column_factor = [&](int g, int i, F2* f) {
    if (post) at.param(j.post_weight, j.param_dtype, 1.f, i, f);
    else
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = f2(1.f);
    if (gate) {
      F2 v[4];
      at.load(reinterpret_cast<const T*>(j.gate) + (long long)g * d, i, v);
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = mul2(f[k], v[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = mul2(f[k], f2(c));
  };
  const int ld_dn = (int)j.ld_d_normed, ld_do = (int)j.ld_d_out, ld_x = (int)j.ld_x, ld_y = (int)j.ld_y;
  auto sources = [&](long long row, const T** rows) {
    rows[0] = j.d_normed ? reinterpret_cast<const T*>(j.d_normed) + row * ld_dn : nullptr;
    rows[1] = j.d_out ? reinterpret_cast<const T*>(j.d_out) + row * ld_do : nullptr;
    rows[2] = reinterpret_cast<const T*>(j.x) + row * ld_x;
    rows[3] = use_y ? reinterpret_cast<const T*>(j.y) + row * ld_y : nullptr;
  };

  F2 dw[P], db[P], A[P], B[P], dpw[P], dpb[P];
  const bool scaled = post || gate;  // f is not one number
  const Columns<P> ws(smem_u32(smem) + p.ring, 0), fs(smem_u32(smem) + p.ring, 1);
#pragma unroll
  for (int k = 0; k < P; ++k) dw[k] = db[k] = A[k] = B[k] = dpw[k] = dpb[k] = f2(0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    F2 v[4];
    at.param(j.weight, j.param_dtype, 1.f, i, v);
    ws.put(i, v);
    if (scaled && !direct) {
      column_factor(gate_row, i, v);
      fs.put(i, v);
    }
  }

  JointRows ahead = it;
  for (int s = 0; s + 1 < p.stages; ++s) {
    const T* rows[4];
    const bool there = ahead.there();
    sources(ahead.row, rows);
    ring.fetch(at, rows, there);
    if (there) ahead.next();
  }
  bool fresh = true;  // the gate group's factor is to be formed
  for (; it.there(); it.next()) {
    const int row = it.row;
    const float4 st = reinterpret_cast<const float4*>(j.stats)[row];
    F2 dn[P], hat[P], dx[P], y[P];
    const T* rows[4];
    const bool there = ahead.there();
    sources(ahead.row, rows);
    ring.fetch(at, rows, there);
    if (there) ahead.next();
    ring.wait();
    sources(row, rows);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (j.d_normed) ring.read(at, rows[0], 0, i, dn + i * 4);
      else
#pragma unroll
        for (int k = 0; k < 4; ++k) dn[i * 4 + k] = f2(0.f);
      ring.read(at, rows[2], 2, i, hat + i * 4);
    }
    F2 s0 = f2(0.f), s1 = f2(0.f);
    {
      const F2 r = f2(st.w), m = f2(-st.z * st.w);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        F2 w[4];
        ws.get(i, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = i * 4 + e;
          hat[k] = layer ? fma2(hat[k], r, m) : mul2(hat[k], r);
          dw[k] = fma2(dn[k], hat[k], dw[k]);
          if (layer) db[k] = add2(db[k], dn[k]);
          dn[k] = mul2(dn[k], w[e]);
          s0 = fma2(dn[k], hat[k], s0);
          if (layer) s1 = add2(s1, dn[k]);
        }
      }
    }
    float s[2] = {sum2(s0), sum2(s1)};
    sum(s);
    // (read after the sum: what waits in shared memory needs no registers)
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (j.d_out) ring.read(at, rows[1], 1, i, dx + i * 4);
      else
#pragma unroll
        for (int k = 0; k < 4; ++k) dx[i * 4 + k] = f2(0.f);
      if (use_y) ring.read(at, rows[3], 3, i, y + i * 4);
    }
    ring.next();
    if (direct && fresh) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        F2 v[4];
        column_factor(it.g, i, v);
        fs.put(i, v);
      }
    }
    const F2 r = f2(st.w), c1 = f2(-s[0] * inv_d), c2 = f2(layer ? -s[1] * inv_d : 0.f);
    const F2 ry = f2(st.y), my = f2(-st.x * st.y);
    s0 = s1 = f2(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = i * 4 + k;
        F2 t = fma2(hat[n], c1, dn[n]);
        if (layer) t = add2(t, c2);
        dx[n] = fma2(r, t, dx[n]);
      }
      at.store(reinterpret_cast<T*>(j.dx) + (long long)row * d, i, dx + i * 4);
      F2 f[4];
      if (scaled) fs.get(i, f);
      else
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = f2(c);
      if (drop && at.any(i)) at.drop(keep, row, i, dx + i * 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = i * 4 + k;
        const F2 m = at.only(dx[n], i, k);  // (beyond d a layer norm's dx is not zero)
        if (use_y) {
          if (post) y[n] = layer ? fma2(y[n], ry, my) : mul2(y[n], ry);
          else if (drop) y[n] = where_nonzero(m, y[n]);  // (an infinity that was dropped stays out of the gate's gradient)
          A[n] = fma2(m, y[n], A[n]);
        }
        if (post && layer) B[n] = add2(B[n], m);
        dx[n] = mul2(m, f[k]);
        if (post) {
          s0 = fma2(dx[n], y[n], s0);
          if (layer) s1 = add2(s1, dx[n]);
        }
      }
      if (!post) at.store(reinterpret_cast<T*>(j.dy) + (long long)row * d, i, dx + i * 4);
    }
    if (post) {
      s[0] = sum2(s0), s[1] = sum2(s1);
      sum(s);
      const F2 c3 = f2(-s[0] * inv_d), c4 = f2(layer ? -s[1] * inv_d : 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int n = i * 4 + k;
          F2 t = fma2(y[n], c3, dx[n]);
          if (layer) t = add2(t, c4);
          dx[n] = mul2(ry, t);
        }
        at.store(reinterpret_cast<T*>(j.dy) + (long long)row * d, i, dx + i * 4);
      }
    }
    if (direct) {
      fresh = it.last_of_gate();
      if (fresh) {  // the gate group ends here, and with it its gradient
        const T* pg = reinterpret_cast<const T*>(j.gate) + (long long)it.g * d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          F2 g[4], pw[4], pb[4], v[4];
          at.load(pg, i, g);
          if (post) {
            at.param(j.post_weight, j.param_dtype, 1.f, i, pw);
            if (layer) at.param(j.post_bias, j.param_dtype, 0.f, i, pb);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int n = i * 4 + k;
            const F2 a = mul2(A[n], f2(c)), b = mul2(B[n], f2(c));
            v[k] = post ? mul2(a, pw[k]) : a;
            if (post && layer) v[k] = fma2(b, pb[k], v[k]);
            if (post) dpw[n] = fma2(a, g[k], dpw[n]);
            if (post && layer) dpb[n] = fma2(b, g[k], dpb[n]);
            A[n] = B[n] = f2(0.f);
          }
          at.store(reinterpret_cast<T*>(j.dgate) + (long long)it.g * d, i, v);
        }
      }
    }
  }

  // What this group has of the block's rows of `part`: dweight, dbias, then from A and B.
  if (!direct) {
    const T* pg = gate ? reinterpret_cast<const T*>(j.gate) + (long long)gate_row * d : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      F2 g[4], pw[4], pb[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) g[k] = f2(1.f);
      if (gate) at.load(pg, i, g);
      if (gate && post) {
        at.param(j.post_weight, j.param_dtype, 1.f, i, pw);
        if (layer) at.param(j.post_bias, j.param_dtype, 0.f, i, pb);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = i * 4 + k;
        const F2 a = mul2(A[n], f2(c)), b = mul2(B[n], f2(c));
        dpw[n] = gate ? mul2(a, g[k]) : a;
        if (layer) dpb[n] = gate ? mul2(b, g[k]) : b;
        A[n] = post && gate ? mul2(a, pw[k]) : a;
        if (post && gate && layer) A[n] = fma2(b, pb[k], A[n]);
      }
    }
  }
  // The groups' shares are added in their order through shared memory, in two buffers in turn, so that one barrier a vector
  // is enough (a buffer is written again only after the barrier of the vector between, which follows every read of it).
  // The ring is done with.
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float* share = reinterpret_cast<float*>(smem);
  int turn = 0;
  auto write = [&](int a, const F2* v) {
    if (p.slot[a] < 0) return;
    float* mine = share + turn * blockDim.y * dp;
    turn ^= 1;
#pragma unroll
    for (int i = 0; i < NV; ++i) at.store_sums(mine + threadIdx.y * dp, i, v + i * 4);
    __syncthreads();
    float* to = part + ((size_t)p.slot[a] * p.blocks + blockIdx.x) * dp;
    T* whole = a == 4 && p.chunks == 1 ? reinterpret_cast<T*>(j.dgate) + (long long)gate_row * d : nullptr;
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < d; c += blockDim.x * blockDim.y) {
      float t = mine[c];
      for (int g = 1; g < (int)blockDim.y; ++g) t += mine[g * dp + c];
      if (whole) whole[c] = from_f32<T>(t);
      else to[c] = t;
    }
  };
  write(0, dw);
  if (layer) write(1, db);
  if (post) write(2, dpw);
  if (post && layer) write(3, dpb);
  if (gate && !direct) write(4, A);
}

// Rows of over 4096 elements: 512 threads have 128 registers each, which the sums over rows half fill. The row stays in
// shared memory and each step of it goes through the thread's elements eight at a time,
// forming again what the step before had; everything else is as above. (2000 x 8192 bf16, layer norms and a gate: 114 us, 27% of
// a copy's rate, with 32 bytes of a thread spilled; with all of a row in registers 165 us. With gate groups of few rows, whose
// sums take more registers, 712 bytes are spilled, with unaligned rows 816: 3000 x 4099, a gate a row: 404 us, 8%.)
template <typename T, bool VEC, bool DIRECT>
__global__ void __launch_bounds__(512, 1) joint_backward_wide_kernel(const PsgdJoint j, const JointPlan p, float* part) {
  constexpr int W = W16_512, NV = width_nv(W), P = NV * 4;
  const bool post = j.post != 0, gate = j.gate != nullptr, layer = j.kind == PSGD_NORM_LAYER, drop = j.threshold != 0;
  constexpr bool direct = DIRECT;
  const bool use_y = post || gate;
  extern __shared__ uint4 smem[];
  using Sum = GroupSum<2, width_threads(W) / 32>;
  __shared__ __align__(16) float red[Sum::FLOATS];
  const int d = j.d, dp = (d + 7) & ~7;
  const Place<T, VEC> at(d);
  pdl_trigger();
  Sum sum(red);
  const Keep keep(drop ? j.seed : 0, drop ? j.offset : 0, drop ? j.rng : nullptr, j.threshold);
  const float inv_d = 1.f / (float)d, c = j.scale * (drop ? j.keep_scale : 1.f);
  Ring16<T, VEC, NV, 4> ring(smem, p.stages);

  JointRows it;
  it.groups = blockDim.y, it.direct = direct, it.per_gate = p.per_gate;
  int gate_row = 0;  // of a block that holds (part of) one gate group
  if (direct) {
    const int held = p.per_block / p.per_gate, g0 = blockIdx.x * held;
    it.g = g0 + threadIdx.y;
    it.end = min(g0 + held, (int)j.gates);
    it.row = it.g * p.per_gate;
  } else if (p.chunks) {
    gate_row = blockIdx.x / p.chunks;
    const int r0 = gate_row * p.per_gate + (blockIdx.x - gate_row * p.chunks) * p.per_block;
    it.row = r0 + threadIdx.y;
    it.end = min(r0 + p.per_block, (gate_row + 1) * p.per_gate);
    it.g = 0;
  } else {
    it.row = blockIdx.x * p.per_block + threadIdx.y;
    it.end = (int)min((blockIdx.x + 1LL) * p.per_block, j.rows);
    it.g = 0;
  }

  // f, per column, of a gate group
  auto column_factor = [&](int g, int i, F2* f) {
    if (post) at.param(j.post_weight, j.param_dtype, 1.f, i, f);
    else
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = f2(1.f);
    if (gate) {
      F2 v[4];
      at.load(reinterpret_cast<const T*>(j.gate) + (long long)g * d, i, v);
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = mul2(f[k], v[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = mul2(f[k], f2(c));
  };
  const int ld_dn = (int)j.ld_d_normed, ld_do = (int)j.ld_d_out, ld_x = (int)j.ld_x, ld_y = (int)j.ld_y;
  auto sources = [&](long long row, const T** rows) {
    rows[0] = j.d_normed ? reinterpret_cast<const T*>(j.d_normed) + row * ld_dn : nullptr;
    rows[1] = j.d_out ? reinterpret_cast<const T*>(j.d_out) + row * ld_do : nullptr;
    rows[2] = reinterpret_cast<const T*>(j.x) + row * ld_x;
    rows[3] = use_y ? reinterpret_cast<const T*>(j.y) + row * ld_y : nullptr;
  };

  F2 dw[P], db[P], A[P], B[P], dpw[P], dpb[P];
  const bool scaled = post || gate;  // f is not one number
  const Columns<P> ws(smem_u32(smem) + p.ring, 0), fs(smem_u32(smem) + p.ring, 1);
#pragma unroll
  for (int k = 0; k < P; ++k) dw[k] = db[k] = A[k] = B[k] = dpw[k] = dpb[k] = f2(0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    F2 v[4];
    at.param(j.weight, j.param_dtype, 1.f, i, v);
    ws.put(i, v);
    if (scaled && !direct) {
      column_factor(gate_row, i, v);
      fs.put(i, v);
    }
  }

  JointRows ahead = it;
  for (int s = 0; s + 1 < p.stages; ++s) {
    const T* rows[4];
    const bool there = ahead.there();
    sources(ahead.row, rows);
    ring.fetch(at, rows, there);
    if (there) ahead.next();
  }
  bool fresh = true;  // the gate group's factor is to be formed
  for (; it.there(); it.next()) {
    const int row = it.row;
    const float4 st = reinterpret_cast<const float4*>(j.stats)[row];
    const T* rows[4];
    const bool there = ahead.there();
    sources(ahead.row, rows);
    ring.fetch(at, rows, there);
    if (there) ahead.next();
    ring.wait();
    sources(row, rows);
    auto get = [&](int a, int i, F2* v) {
      if (rows[a]) ring.read(at, rows[a], a, i, v);
      else
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = f2(0.f);
    };
    const F2 r = f2(st.w), m0 = f2(layer ? -st.z * st.w : 0.f), ry = f2(st.y), my = f2(layer ? -st.x * st.y : 0.f);
    auto hats = [&](int i, F2* dh, F2* hat) {  // d_normed and hat of vector i
      get(0, i, dh);
      get(2, i, hat);
#pragma unroll
      for (int k = 0; k < 4; ++k) hat[k] = fma2(hat[k], r, m0);
    };
    F2 s0 = f2(0.f), s1 = f2(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      F2 dh[4], hat[4], w[4];
      hats(i, dh, hat);
      ws.get(i, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        dw[i * 4 + k] = fma2(dh[k], hat[k], dw[i * 4 + k]);
        db[i * 4 + k] = add2(db[i * 4 + k], dh[k]);
        dh[k] = mul2(dh[k], w[k]);
        s0 = fma2(dh[k], hat[k], s0);
        s1 = add2(s1, dh[k]);
      }
    }
    float s[2] = {sum2(s0), sum2(s1)};
    sum(s);
    const F2 c1 = f2(-s[0] * inv_d), c2 = f2(layer ? -s[1] * inv_d : 0.f);
    if (direct && fresh) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        F2 v[4];
        column_factor(it.g, i, v);
        fs.put(i, v);
      }
    }
    // dx of vector i, and with it what reaches dy before the post norm, and yh (or y)
    auto back = [&](int i, F2* dx, F2* m, F2* y) {
      F2 dh[4], hat[4], w[4];
      hats(i, dh, hat);
      ws.get(i, w);
      get(1, i, dx);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        dx[k] = fma2(r, add2(fma2(hat[k], c1, mul2(dh[k], w[k])), c2), dx[k]);
        m[k] = dx[k];
      }
      if (drop && at.any(i)) at.drop(keep, row, i, m);
#pragma unroll
      for (int k = 0; k < 4; ++k) m[k] = at.only(m[k], i, k);
      if (use_y) get(3, i, y);
      if (post)
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = fma2(y[k], ry, my);
    };
    auto factor = [&](int i, F2* f) {
      if (scaled) fs.get(i, f);
      else
#pragma unroll
        for (int k = 0; k < 4; ++k) f[k] = f2(c);
    };
    s0 = s1 = f2(0.f);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      F2 dx[4], m[4], y[4], f[4];
      back(i, dx, m, y);
      factor(i, f);
      at.store(reinterpret_cast<T*>(j.dx) + (long long)row * d, i, dx);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (use_y && !post && drop) y[k] = where_nonzero(m[k], y[k]);
        if (use_y) A[i * 4 + k] = fma2(m[k], y[k], A[i * 4 + k]);
        B[i * 4 + k] = add2(B[i * 4 + k], m[k]);
        m[k] = mul2(m[k], f[k]);
        if (post) {
          s0 = fma2(m[k], y[k], s0);
          s1 = add2(s1, m[k]);
        }
      }
      if (!post) at.store(reinterpret_cast<T*>(j.dy) + (long long)row * d, i, m);
    }
    if (post) {
      s[0] = sum2(s0), s[1] = sum2(s1);
      sum(s);
      const F2 c3 = f2(-s[0] * inv_d), c4 = f2(layer ? -s[1] * inv_d : 0.f);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        F2 dx[4], m[4], y[4], f[4];
        back(i, dx, m, y);
        factor(i, f);
#pragma unroll
        for (int k = 0; k < 4; ++k) m[k] = mul2(ry, add2(fma2(y[k], c3, mul2(m[k], f[k])), c4));
        at.store(reinterpret_cast<T*>(j.dy) + (long long)row * d, i, m);
      }
    }
    ring.next();
    if (direct) {
      fresh = it.last_of_gate();
      if (fresh) {  // the gate group ends here, and with it its gradient
        const T* pg = reinterpret_cast<const T*>(j.gate) + (long long)it.g * d;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          F2 g[4], pw[4], pb[4], v[4];
          at.load(pg, i, g);
          if (post) {
            at.param(j.post_weight, j.param_dtype, 1.f, i, pw);
            if (layer) at.param(j.post_bias, j.param_dtype, 0.f, i, pb);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int n = i * 4 + k;
            const F2 a = mul2(A[n], f2(c)), b = mul2(B[n], f2(c));
            v[k] = post ? mul2(a, pw[k]) : a;
            if (post && layer) v[k] = fma2(b, pb[k], v[k]);
            if (post) dpw[n] = fma2(a, g[k], dpw[n]);
            if (post && layer) dpb[n] = fma2(b, g[k], dpb[n]);
            A[n] = B[n] = f2(0.f);
          }
          at.store(reinterpret_cast<T*>(j.dgate) + (long long)it.g * d, i, v);
        }
      }
    }
  }

  // What this group has of the block's rows of `part`: dweight, dbias, then from A and B.
  if (!direct) {
    const T* pg = gate ? reinterpret_cast<const T*>(j.gate) + (long long)gate_row * d : nullptr;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      F2 g[4], pw[4], pb[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) g[k] = f2(1.f);
      if (gate) at.load(pg, i, g);
      if (gate && post) {
        at.param(j.post_weight, j.param_dtype, 1.f, i, pw);
        if (layer) at.param(j.post_bias, j.param_dtype, 0.f, i, pb);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = i * 4 + k;
        const F2 a = mul2(A[n], f2(c)), b = mul2(B[n], f2(c));
        dpw[n] = gate ? mul2(a, g[k]) : a;
        if (layer) dpb[n] = gate ? mul2(b, g[k]) : b;
        A[n] = post && gate ? mul2(a, pw[k]) : a;
        if (post && gate && layer) A[n] = fma2(b, pb[k], A[n]);
      }
    }
  }
  // The groups' shares are added in their order through shared memory, in two buffers in turn, so that one barrier a vector
  // is enough (a buffer is written again only after the barrier of the vector between, which follows every read of it).
  // The ring is done with.
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  float* share = reinterpret_cast<float*>(smem);
  int turn = 0;
  auto write = [&](int a, const F2* v) {
    if (p.slot[a] < 0) return;
    float* mine = share + turn * blockDim.y * dp;
    turn ^= 1;
#pragma unroll
    for (int i = 0; i < NV; ++i) at.store_sums(mine + threadIdx.y * dp, i, v + i * 4);
    __syncthreads();
    float* to = part + ((size_t)p.slot[a] * p.blocks + blockIdx.x) * dp;
    T* whole = a == 4 && p.chunks == 1 ? reinterpret_cast<T*>(j.dgate) + (long long)gate_row * d : nullptr;
    for (int c = threadIdx.y * blockDim.x + threadIdx.x; c < d; c += blockDim.x * blockDim.y) {
      float t = mine[c];
      for (int g = 1; g < (int)blockDim.y; ++g) t += mine[g * dp + c];
      if (whole) whole[c] = from_f32<T>(t);
      else to[c] = t;
    }
  };
  write(0, dw);
  if (layer) write(1, db);
  if (post) write(2, dpw);
  if (post && layer) write(3, dpb);
  if (gate && !direct) write(4, A);
}

// ---- launches of one element type -------------------------------------------------------------------------------------
template <typename T, bool VEC, int W, int F>
int joint_forward_launch(const PsgdJoint& j, const JointPlan& p, cudaStream_t stream) {
  auto k = joint_forward_kernel<T, VEC, W, F>;
  static std::atomic<unsigned long long> done{0};
  if (p.smem > JOINT_SMEM_FREE)
    if (int rc = allow_smem(k, JOINT_SMEM_MOST, done)) return rc;
  k<<<p.blocks, dim3(p.tpr, p.groups), p.smem, stream>>>(j, p);
  return cudaGetLastError() == cudaSuccess ? PSGD_OK : PSGD_ELAUNCH;
}
template <typename K>
int joint_backward_start(K k, std::atomic<unsigned long long>& done, const PsgdJoint& j, const JointPlan& p, float* part,
                         cudaStream_t stream) {
  if (p.smem > JOINT_SMEM_FREE)
    if (int rc = allow_smem(k, JOINT_SMEM_MOST, done)) return rc;
  k<<<p.blocks, dim3(p.tpr, p.groups), p.smem, stream>>>(j, p, part);
  return cudaGetLastError() == cudaSuccess ? PSGD_OK : PSGD_ELAUNCH;
}

template <typename T, bool VEC, int W, int F>
int joint_backward_launch(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  return joint_backward_start(joint_backward_kernel<T, VEC, W, F>, done, j, p, part, stream);
}

template <typename T, bool VEC, bool DIRECT>
int joint_backward_wide(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  return joint_backward_start(joint_backward_wide_kernel<T, VEC, DIRECT>, done, j, p, part, stream);
}

inline int joint_flags(const PsgdJoint& j, const JointPlan& p) {
  return (j.post ? F_POST : 0) | (j.gate ? F_GATE : 0) | (j.kind == PSGD_NORM_LAYER ? F_LAYER : 0) |
         (j.threshold ? F_DROP : 0) | (j.gate && !p.chunks ? F_DIRECT : 0);
}

// The kernel compiled for the flags f (F and up that can occur; the forward kernels take the gate at run time).
template <typename T, bool VEC, int W, int F = 0>
int joint_forward_pick(int f, const PsgdJoint& j, const JointPlan& p, cudaStream_t stream) {
  if constexpr (F >= F_DIRECT) {
    return PSGD_EINVAL;
  } else {
    if constexpr (!(F & F_GATE))
      if (f == F) return joint_forward_launch<T, VEC, W, F>(j, p, stream);
    return joint_forward_pick<T, VEC, W, F + 1>(f, j, p, stream);
  }
}
template <typename T, bool VEC, int W, int F = 0>
int joint_backward_pick(int f, const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream) {
  if constexpr (F >= F_RUNTIME) {
    return PSGD_EINVAL;
  } else {
    if constexpr (!(F & F_DIRECT) || (F & F_GATE))
      if (f == F) return joint_backward_launch<T, VEC, W, F>(j, p, part, stream);
    return joint_backward_pick<T, VEC, W, F + 1>(f, j, p, part, stream);
  }
}

template <typename T>
int joint_forward_of(const PsgdJoint& j, const JointPlan& p, cudaStream_t stream) {
  const int f = joint_flags(j, p) & ~(F_GATE | F_DIRECT);
  switch (p.wide) {
    case W8: return p.vec ? joint_forward_pick<T, true, W8>(f, j, p, stream) : joint_forward_pick<T, false, W8>(f, j, p, stream);
    case W16: return p.vec ? joint_forward_pick<T, true, W16>(f, j, p, stream) : joint_forward_pick<T, false, W16>(f, j, p, stream);
    case W16_256:
      return p.vec ? joint_forward_pick<T, true, W16_256>(f, j, p, stream)
                   : joint_forward_launch<T, false, W16_256, F_RUNTIME>(j, p, stream);
    default:
      return p.vec ? joint_forward_launch<T, true, W16_512, F_RUNTIME>(j, p, stream)
                   : joint_forward_launch<T, false, W16_512, F_RUNTIME>(j, p, stream);
  }
}

template <typename T>
int joint_backward_of(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream) {
  const int f = joint_flags(j, p);
  switch (p.wide) {
    case W8:
      return p.vec ? joint_backward_pick<T, true, W8>(f, j, p, part, stream)
                   : joint_backward_pick<T, false, W8>(f, j, p, part, stream);
    case W16:
      return p.vec ? joint_backward_pick<T, true, W16>(f, j, p, part, stream)
                   : joint_backward_pick<T, false, W16>(f, j, p, part, stream);
    case W16_256:
      return p.vec ? joint_backward_pick<T, true, W16_256>(f, j, p, part, stream)
                   : joint_backward_launch<T, false, W16_256, F_RUNTIME>(j, p, part, stream);
    default:
      if (f & F_DIRECT)
        return p.vec ? joint_backward_wide<T, true, true>(j, p, part, stream) : joint_backward_wide<T, false, true>(j, p, part, stream);
      return p.vec ? joint_backward_wide<T, true, false>(j, p, part, stream) : joint_backward_wide<T, false, false>(j, p, part, stream);
  }
}

}  // namespace psgd
