// The joint's kernels (joint.cuh) for fp32 rows.
#include "joint.cuh"

namespace psgd {

int joint_forward_f32(const PsgdJoint& j, const JointPlan& p, cudaStream_t stream) {
  return joint_forward_of<float>(j, p, stream);
}
int joint_backward_f32(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream) {
  return joint_backward_of<float>(j, p, part, stream);
}

}  // namespace psgd
