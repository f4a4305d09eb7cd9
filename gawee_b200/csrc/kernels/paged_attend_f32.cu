// Attention over a paged key/value cache of f32 pages.
#include "paged_attend.cuh"

namespace gawee {
namespace kern {

cudaError_t launch_kv_attend_f32(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s) {
  return paged::attend_lanes<float>(p, shape, s);
}

}  // namespace kern
}  // namespace gawee
