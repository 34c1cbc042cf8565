// The joint's kernels (joint.cuh) for fp16 rows.
#include "joint.cuh"

namespace psgd {

int joint_forward_f16(const PsgdJoint& j, const JointPlan& p, cudaStream_t stream) {
  return joint_forward_of<__half>(j, p, stream);
}
int joint_backward_f16(const PsgdJoint& j, const JointPlan& p, float* part, cudaStream_t stream) {
  return joint_backward_of<__half>(j, p, part, stream);
}

}  // namespace psgd
