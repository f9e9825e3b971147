// The categorical kernels on float16 logits.
#define PFPN_CATEGORICAL_TYPE f16_t
#include "categorical_impl.h"
