#include "attention_forward.h"

template int wrnn::attn::forward<__bf16>(const Params&, hipStream_t);
