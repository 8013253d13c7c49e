// Loss of a linear layer, float16 operands.
#include "az_head.cuh"

AZ_HEAD_UNIT(f16, DT_F16)
