// pf_shared_fp16.hip — the kernels of attention behind shared tokens for fp16 rows.
#include "pf_attend_shared.h"

namespace pf {

hipError_t launch_shared_fp16(const AttendParams& p, hipStream_t stream) {
  return launch_shared_type<FP16>(p, stream);
}

}  // namespace pf
