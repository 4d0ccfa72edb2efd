// Attention's kernels for float32 operands.
#include "attention_kernels.h"

namespace gefen {
namespace attn {
template int launch_width<float>(Pass, const Params&, hipStream_t);
}  // namespace attn
}  // namespace gefen
