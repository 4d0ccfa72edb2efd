// Attention's kernels for bfloat16 operands.
#include "attention_kernels.h"

namespace gefen {
namespace attn {
template int launch_width<bf16_t>(Pass, const Params&, hipStream_t);
}  // namespace attn
}  // namespace gefen
