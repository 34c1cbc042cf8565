// Entry points of the joint between two blocks (joint.cuh): shapes, work split and the last step of the sums over rows.
#include "joint.cuh"

namespace psgd {
namespace {

// Sums of the blocks' rows in a fixed order: 32 columns a block, 32 threads a column, each over every 32nd row, eight at a
// time (a row's latency is what this launch costs: 293 rows of 3 vectors of 2048, about 5 us, half of it hidden behind the
// launch before). blockIdx.y: the parameter vectors that are there, then the gate groups.
__global__ void __launch_bounds__(1024) joint_reduce_kernel(const PsgdJoint j, const JointPlan p, const float* part) {
  __shared__ float red[32][33];
  const int dp = (j.d + 7) & ~7, col = blockIdx.x * 32 + threadIdx.x, vectors = p.slots - (p.slot[4] >= 0);
  int a = 4;
  if ((int)blockIdx.y < vectors)
    for (int k = 0; k < 4; ++k)
      if (p.slot[k] == (int)blockIdx.y) a = k;
  int b0 = 0, b1 = p.blocks;
  long long to = 0;
  void* out[4] = {j.dweight, j.dbias, j.dpost_weight, j.dpost_bias};
  if (a == 4) {
    const int g = (int)blockIdx.y - vectors;
    b0 = g * p.chunks;
    b1 = b0 + p.chunks;
    to = (long long)g * j.d;
  }
  float s[8] = {};
  pdl_wait();
  if (col < j.d) {
    const float* from = part + (size_t)p.slot[a] * p.blocks * dp + col;
    int b = b0 + threadIdx.y;
    for (; b + 7 * 32 < b1; b += 8 * 32)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] += from[(size_t)(b + 32 * k) * dp];
#pragma unroll
    for (int k = 0; k < 7; ++k)
      if (b + 32 * k < b1) s[k] += from[(size_t)(b + 32 * k) * dp];
  }
  red[threadIdx.y][threadIdx.x] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  const float v = warp_sum(red[threadIdx.x][threadIdx.y]);  // a warp a column
  const int c = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && c < j.d) {
    if (a < 4) store_any(out[a], j.param_dtype, c, v);
    else store_any(j.dgate, j.dtype, to + c, v);
  }
}

constexpr int JOINT_DIRECT_ROWS = 32;

int size_of(int dtype) { return dtype == PSGD_F32 ? 4 : 2; }

bool rows_aligned(const void* p, long long ld, int dtype) {
  return aligned16(p) && (ld * size_of(dtype)) % 16 == 0;
}

int round_up(int a, int b) { return (a + b - 1) / b * b; }

bool params_aligned(const PsgdJoint& j) {
  return aligned16(j.weight) && aligned16(j.bias) && aligned16(j.post_weight) && aligned16(j.post_bias);
}

bool valid(const PsgdJoint& j) {
  if (j.rows < 0 || j.rows > (1 << 30) || j.d < 1 || j.d > JOINT_MAX_D || j.dtype < 0 || j.dtype > 2) return false;
  if ((j.param_dtype != PSGD_F32 && j.param_dtype != j.dtype) || (j.kind != PSGD_NORM_RMS && j.kind != PSGD_NORM_LAYER)) return false;
  const long long most = 1LL << 31;
  if (j.ld_x >= most || j.ld_y >= most || j.ld_d_out >= most || j.ld_d_normed >= most) return false;
  // (rows do not overlap; a matrix that is not there has no stride)
  if (j.rows > 1 && ((j.x && j.ld_x < j.d) || (j.y && j.ld_y < j.d) || (j.d_out && j.ld_d_out < j.d) || (j.d_normed && j.ld_d_normed < j.d)))
    return false;
  if (j.threshold > 65536u || (j.gate && (j.gates < 1 || j.rows % j.gates))) return false;
  return true;
}

// The kernel for rows of d elements, and as many groups as make up a block of `threads` (of the kernel's width for 0).
void shape(int d, JointPlan& p, int threads) {
  p.wide = d <= 256 ? W8 : d <= 2048 ? W16 : d <= 4096 ? W16_256 : W16_512;
  p.nv = width_nv(p.wide);
  p.tpr = round_up((d + 8 * p.nv - 1) / (8 * p.nv), 32);
  p.groups = (threads ? threads : width_threads(p.wide)) / p.tpr;
  if (p.groups < 1) p.groups = 1;
  if (p.tpr > 32 && p.groups > JOINT_MAX_GROUPS) p.groups = JOINT_MAX_GROUPS;
}

// Blocks that an SM holds at once: as many as the kernel was compiled for, and as the shared memory allows.
int per_sm(const JointPlan& p, int compiled) {
  const int threads = p.tpr * p.groups, by_regs = compiled * width_threads(p.wide) / threads;
  const int by_smem = 220 * 1024 / (p.smem + 2 * 1024);
  const int n = by_regs < by_smem ? by_regs : by_smem;
  return n < 1 ? 1 : n;
}

// Shared memory of the rings.
int ring_bytes(const JointPlan& p, int arrays, int dtype) {
  const int threads = p.tpr * p.groups;
  return p.stages * arrays * p.nv * size_of(dtype) / 2 * (threads + (p.vec ? 0 : threads / 32)) * 16;
}

JointPlan plan_forward(const PsgdJoint& j) {
  JointPlan p = {};
  p.vec = j.d % 8 == 0 && params_aligned(j) && rows_aligned(j.x, j.ld_x, j.dtype) && rows_aligned(j.y, j.ld_y, j.dtype) &&
          rows_aligned(j.out, j.d, j.dtype) && rows_aligned(j.normed, j.d, j.dtype) &&
          (!j.gate || rows_aligned(j.gate, j.d, j.dtype));
  shape(j.d, p, 0);
  p.stages = j.dtype == PSGD_F32 ? 2 : 3;
  p.smem = ring_bytes(p, 2, j.dtype);
  p.per_gate = j.gate ? (int)(j.rows / j.gates) : 1;
  const int want = ((int)j.rows + p.groups - 1) / p.groups, most = per_sm(p, joint_forward_blocks(p.wide, joint_flags(j, p))) * psgd_num_sms();
  p.blocks = want < most ? want : most;
  return p;
}

// The plan of a backward pass; the same from a size query and from the launch.
JointPlan plan_backward(const PsgdJoint& j) {
  JointPlan p = {};
  p.vec = j.d % 8 == 0 && params_aligned(j) && rows_aligned(j.x, j.ld_x, j.dtype) && rows_aligned(j.dx, j.d, j.dtype) &&
          rows_aligned(j.dy, j.d, j.dtype) && (!j.d_out || rows_aligned(j.d_out, j.ld_d_out, j.dtype)) &&
          (!j.d_normed || rows_aligned(j.d_normed, j.ld_d_normed, j.dtype)) &&
          (!(j.post || j.gate) || rows_aligned(j.y, j.ld_y, j.dtype)) &&
          (!j.gate || (rows_aligned(j.gate, j.d, j.dtype) && rows_aligned(j.dgate, j.d, j.dtype)));
  // Gate groups of few rows are a thread group's each (direct); longer ones are dealt out in chunks.
  p.per_gate = j.gate ? (int)(j.rows / j.gates) : 1;
  p.chunks = j.gate && p.per_gate > JOINT_DIRECT_ROWS;  // (how many: below)
  shape(j.d, p, 0);
  const bool compiled = p.wide == W8 || p.wide == W16 || (p.wide == W16_256 && p.vec);
  const int f = joint_flags(j, p) | (compiled ? 0 : F_RUNTIME);
  shape(j.d, p, joint_backward_threads(p.wide, f));
  const int rows = (int)j.rows, per_sm = joint_backward_blocks(p.wide, f), most = per_sm * psgd_num_sms();
  const int fair = (rows + most - 1) / most;
  if (p.chunks) p.chunks = (p.per_gate + fair - 1) / fair;
  const bool layer = j.kind == PSGD_NORM_LAYER;
  const bool there[5] = {true, layer, j.post != 0, j.post && layer, j.gate != nullptr};
  for (int a = 0; a < 5; ++a) p.slot[a] = there[a] ? p.slots++ : -1;
  // Rows ahead: two for 16-bit types, one for fp32, as far as shared memory goes.
  const int threads = p.tpr * p.groups, columns = threads * p.nv * 64;
  const int arrays = (f & F_RUNTIME) || j.post || j.gate ? 4 : 3;  // (as the kernel compiled for f has)
  const int room = 220 * 1024 / per_sm - columns;
  p.stages = j.dtype == PSGD_F32 ? 2 : 3;
  while (p.stages > 1 && ring_bytes(p, arrays, j.dtype) > room) --p.stages;
  p.ring = ring_bytes(p, arrays, j.dtype);
  p.smem = p.ring + columns;
  const int share = 2 * p.groups * round_up(j.d, 8) * 4;
  if (p.smem < share) p.smem = share;
  if (p.chunks) {
    p.per_block = (p.per_gate + p.chunks - 1) / p.chunks;
  } else if (j.gate) {
    int held = fair / p.per_gate;  // gate groups of a block: a multiple of its thread groups where there are enough
    held = held < 1 ? 1 : held > p.groups ? (held + p.groups - 1) / p.groups * p.groups : held;
    p.per_block = held * p.per_gate;
  } else {
    p.per_block = fair < p.groups ? p.groups : fair;
  }
  p.blocks = p.chunks ? (int)j.gates * p.chunks : (rows + p.per_block - 1) / p.per_block;
  return p;
}

}  // namespace
}  // namespace psgd

extern "C" int psgd_joint_forward(const PsgdJoint* j, cudaStream_t stream) {
  using namespace psgd;
  if (!j || !valid(*j)) return PSGD_EINVAL;
  if (j->rows == 0) return PSGD_OK;
  if (!j->x || !j->y || !j->out || !j->normed || !j->stats || !aligned16(j->stats)) return PSGD_EINVAL;
  const JointPlan p = plan_forward(*j);
  switch (j->dtype) {
    case PSGD_F32: return joint_forward_f32(*j, p, stream);
    case PSGD_BF16: return joint_forward_bf16(*j, p, stream);
    default: return joint_forward_f16(*j, p, stream);
  }
}

extern "C" long long psgd_joint_workspace(const PsgdJoint* j) {
  using namespace psgd;
  if (!j || !valid(*j)) return PSGD_EINVAL;
  if (j->rows == 0) return 0;
  const JointPlan p = plan_backward(*j);
  return (long long)p.slots * p.blocks * round_up(j->d, 8) * 4;
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
  if (bytes < (long long)p.slots * p.blocks * round_up(j->d, 8) * 4) return PSGD_ESPACE;
  float* part = reinterpret_cast<float*>(workspace);
  int rc;
  switch (j->dtype) {
    case PSGD_F32: rc = joint_backward_f32(*j, p, part, stream); break;
    case PSGD_BF16: rc = joint_backward_bf16(*j, p, part, stream); break;
    default: rc = joint_backward_f16(*j, p, part, stream);
  }
  if (rc) return rc;
  // (a gate group of several chunks has over 32 rows to a chunk on 148 SMs: their number stays within the grid's limit)
  const dim3 grid((j->d + 31) / 32, p.slots - (p.slot[4] >= 0) + (p.chunks > 1 ? (int)j->gates : 0));
  return pdl_launch(joint_reduce_kernel, grid, dim3(32, 32), 0, stream, *j, p, (const float*)part);
}
