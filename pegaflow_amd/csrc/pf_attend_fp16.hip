// pf_attend_fp16.hip — the attention kernels for fp16 rows.
#include "pf_attend_kernels.h"

namespace pf {

hipError_t launch_attend_fp16(const AttendParams& p, hipStream_t stream) {
  return launch_type<FP16>(p, stream);
}

}  // namespace pf
