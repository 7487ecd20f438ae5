#include "attention_backward.h"

namespace wrnn {
namespace attn {
template int backward<float, 256>(const Params&, float*, hipStream_t);
}  // namespace attn
}  // namespace wrnn
