// Loss of a linear layer, bfloat16 operands.
#include "az_head.cuh"

AZ_HEAD_UNIT(bf16, DT_BF16)
