// The attention kernels of one pair of cache formats, chosen by head size, query type and plan.
#pragma once

#include "kv_attend.h"
#include "kv_many.h"

namespace komp {

// Run the kernel of `plan`: few columns or many.
template <int NB, int KF, int VF, int MODE>
hipError_t launch_attend_mode(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.splits) * static_cast<unsigned>(a.groups), static_cast<unsigned>(a.c.heads),
                  static_cast<unsigned>(batch));
  auto run = [&](auto kern, int threads) {
    const Timing tm = timing_slot(KIND_PROBE);
    if (tm.on) {
      hipExtLaunchKernelGGL(kern, grid, dim3(threads), 0, stream, tm.start, tm.stop, 0, a);
    } else {
      hipLaunchKernelGGL(kern, grid, dim3(threads), 0, stream, a);
    }
    return hipGetLastError();
  };
  if (plan.many) {
    const dim3 heads_first(grid.y, grid.z, grid.x);
    if constexpr (MODE == KV_BF16) {
      if (a.lse == nullptr) return launch_attend_many<NB, KF, VF, MODE, KV_ALL_SCALED>(a, heads_first, stream);
      return launch_attend_many<NB, KF, VF, MODE, KV_VALUES_SCALED>(a, heads_first, stream);
    } else {
      return launch_attend_many<NB, KF, VF, MODE, KV_EXACT>(a, heads_first, stream);
    }
  }
  return run(kv_attend_few_kernel<NB, KF, VF, MODE>, kAttendWaves * 64);
}
template <int NB, int KF, int VF>
hipError_t launch_attend_blocks(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream) {
  if (a.type == KV_F32) return launch_attend_mode<NB, KF, VF, KV_F32>(a, plan, batch, stream);
  if (a.type == KV_F16) return launch_attend_mode<NB, KF, VF, KV_F16>(a, plan, batch, stream);
  return launch_attend_mode<NB, KF, VF, KV_BF16>(a, plan, batch, stream);
}

template <int KF, int VF>
hipError_t launch_attend_format(const AttendArgs& a, const AttendPlan& plan, int batch, hipStream_t stream) {
  switch (a.c.dim) {
    case 64: return launch_attend_blocks<2, KF, VF>(a, plan, batch, stream);
    case 96: return launch_attend_blocks<3, KF, VF>(a, plan, batch, stream);
    case 128: return launch_attend_blocks<4, KF, VF>(a, plan, batch, stream);
    default: return launch_attend_blocks<8, KF, VF>(a, plan, batch, stream);
  }
}

}  // namespace komp
