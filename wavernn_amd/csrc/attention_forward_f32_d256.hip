#include "attention_forward.h"

namespace wrnn {
namespace attn {
template int forward<float, 256>(const Params&, hipStream_t);
}  // namespace attn
}  // namespace wrnn
