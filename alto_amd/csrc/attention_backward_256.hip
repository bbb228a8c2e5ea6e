// Kernels of the attention backward for heads of 256.
#define ALTO_ATTENTION_BACKWARD_KERNELS
#include "attention_backward.h"

namespace alto {
template int launch_attn_bwd<4>(const AttnBwdArgs&, const AttnBwdSeqs&, const AttnBwdPlan&, int64_t, hipStream_t);
}  // namespace alto
