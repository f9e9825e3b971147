// The categorical kernels on bfloat16 logits.
#define PFPN_CATEGORICAL_TYPE bf16_t
#include "categorical_impl.h"
