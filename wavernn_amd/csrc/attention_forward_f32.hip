#include "attention_forward.h"

namespace wrnn {
namespace attn {
template int forward<float, 64>(const Params&, hipStream_t);
template int forward<float, 128>(const Params&, hipStream_t);
}  // namespace attn
}  // namespace wrnn
