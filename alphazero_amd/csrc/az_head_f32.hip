// Loss of a linear layer, float32 operands.
#include "az_head.cuh"

AZ_HEAD_UNIT(f32, DT_F32)
