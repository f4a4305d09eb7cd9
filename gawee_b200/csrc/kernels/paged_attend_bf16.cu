// Attention over a paged key/value cache of bf16 pages.
#include "paged_attend.cuh"

namespace gawee {
namespace kern {

cudaError_t launch_kv_attend_bf16(const KvAttendParams& p, KvAttendShape* shape, cudaStream_t s) {
  return paged::attend_16bit<__nv_bfloat16>(p, shape, s);
}

}  // namespace kern
}  // namespace gawee
