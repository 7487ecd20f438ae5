#include "attention_backward.h"

template int wrnn::attn::backward<__bf16>(const Params&, float*, hipStream_t);
