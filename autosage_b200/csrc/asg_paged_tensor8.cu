// Instances of the tensor-core paged attention for 8-bit pages.
#include "asg_paged_tensor.cuh"

namespace asg {
namespace paged {

Choice choose_tensor8(const AttentionArgs& a, int cache_type) {
  if (a.type == ASG_TYPE_F32) return cache_type == ASG_TYPE_E4M3 ? choose_tensor<E4M3, true>(a) : choose_tensor<INT8, true>(a);
  return cache_type == ASG_TYPE_E4M3 ? choose_tensor<E4M3>(a) : choose_tensor<INT8>(a);
}

}  // namespace paged
}  // namespace asg
