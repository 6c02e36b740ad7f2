// Attention over a cache of Q8_0 keys and Q8_0 values (kv_attend.h, kv_many.h).
#include "kv_launch.h"

namespace komp {

hipError_t launch_attend_q8_q8(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream) {
  return launch_attend_format<KV_Q8_0, KV_Q8_0>(a, plan, batch, stream);
}

}  // namespace komp
