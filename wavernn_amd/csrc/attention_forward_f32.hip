#include "attention_forward.h"

template int wrnn::attn::forward<float>(const Params&, hipStream_t);
