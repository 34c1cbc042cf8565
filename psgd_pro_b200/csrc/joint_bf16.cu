// The joint's kernels (joint.cuh) for bf16 rows.
#include "joint.cuh"

namespace psgd {

int joint_forward_bf16(const PsgdJoint& j, const JointPlan& p, cudaStream_t stream) {
  return joint_forward_of<__nv_bfloat16>(j, p, stream);
}
int joint_backward_bf16(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream) {
  return joint_backward_of<__nv_bfloat16>(j, p, part, stream);
}

}  // namespace psgd
