// Instances of the tensor-core paged attention for 16-bit pages.
#include "asg_paged_tensor.cuh"

namespace asg {
namespace paged {

Choice choose_tensor16(const AttentionArgs& a, int cache_type) {
  if (cache_type == ASG_TYPE_BF16) return choose_tensor<BF16>(a);
  if (cache_type == ASG_TYPE_F16) return choose_tensor<F16>(a);
  return Choice{};
}

}  // namespace paged
}  // namespace asg
