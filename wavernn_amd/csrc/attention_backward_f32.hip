#include "attention_backward.h"

namespace wrnn {
namespace attn {
template int backward<float, 64>(const Params&, float*, hipStream_t);
template int backward<float, 128>(const Params&, float*, hipStream_t);
}  // namespace attn
}  // namespace wrnn
