// pf_shared_bf16.hip — the kernels of attention behind shared tokens for bf16 rows.
#include "pf_attend_shared.h"

namespace pf {

hipError_t launch_shared_bf16(const AttendParams& p, hipStream_t stream) {
  return launch_shared_type<BF16>(p, stream);
}

}  // namespace pf
