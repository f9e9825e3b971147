// The categorical kernels on float32 logits.
#define PFPN_CATEGORICAL_TYPE float
#include "categorical_impl.h"
