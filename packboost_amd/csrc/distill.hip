// The loss of distillation from a teacher's best rows, and its gradient; see soft_grads.h.
#include "soft_grads.h"

namespace pb {

hipError_t launch_distill(const SetLayout& s, const ReportArgs& a, int32_t type, hipStream_t stream) {
    return launch_mode<true>(s, a, type, stream);
}

}  // namespace pb
