// pf_attend_bf16.hip — the attention kernels for bf16 rows.
#include "pf_attend_kernels.h"

namespace pf {

hipError_t launch_attend_bf16(const AttendParams& p, hipStream_t stream) {
  return launch_type<BF16>(p, stream);
}

}  // namespace pf
