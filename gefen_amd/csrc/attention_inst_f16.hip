// Attention's kernels for float16 operands.
#include "attention_kernels.h"

namespace gefen {
namespace attn {
template int launch_width<f16_t>(Pass, const Params&, hipStream_t);
template int launch_range<f16_t>(const Params&, hipStream_t);
}  // namespace attn
}  // namespace gefen
