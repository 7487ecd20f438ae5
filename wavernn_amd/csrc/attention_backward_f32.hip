#include "attention_backward.h"

template int wrnn::attn::backward<float>(const Params&, float*, hipStream_t);
