// C entry points of the loss of a linear layer (kernels and plans: az_head.cuh).
#include "az_head.cuh"

using namespace az;

extern "C" int64_t az_linear_ce_workspace(const az_linear_ce_args* args, int32_t backward) {
    if (const int rc = check_args(args)) return rc;
    return (backward ? backward_layout(*args) : forward_layout(*args)).bytes;
}

extern "C" int az_linear_ce_forward(const az_linear_ce_args* args, float* kept, float* loss, float* ce, float* ent, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
    if (const int rc = check_args(args)) return rc;
    if (!kept || !loss || !workspace) return fail(AZ_ERR_ARG, "null argument");
    if (workspace_bytes < forward_layout(*args).bytes || ((uintptr_t)workspace & 255)) return fail(AZ_ERR_ARG, "workspace too small or not at a multiple of 256");
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (args->dtype == AZ_DT_F32) return ce_forward_f32(*args, kept, loss, ce, ent, ws, st);
    if (args->dtype == AZ_DT_BF16) return ce_forward_bf16(*args, kept, loss, ce, ent, ws, st);
    return ce_forward_f16(*args, kept, loss, ce, ent, ws, st);
}

extern "C" int az_linear_ce_backward(const az_linear_ce_args* args, const float* kept, const float* grad, void* grad_x, void* grad_weight,
                                     void* grad_bias, void* workspace, int64_t workspace_bytes, void* stream) {
    if (const int rc = check_args(args)) return rc;
    if (!kept || !grad || !workspace) return fail(AZ_ERR_ARG, "null argument");
    if (!grad_x && !grad_weight && !grad_bias) return AZ_OK;
    if (((uintptr_t)grad_x | (uintptr_t)grad_weight) & 15) return fail(AZ_ERR_ARG, "gradients start at a multiple of 16 bytes");
    if (workspace_bytes < backward_layout(*args).bytes || ((uintptr_t)workspace & 255)) return fail(AZ_ERR_ARG, "workspace too small or not at a multiple of 256");
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    if (args->dtype == AZ_DT_F32) return ce_backward_f32(*args, kept, grad, grad_x, grad_weight, grad_bias, ws, st);
    if (args->dtype == AZ_DT_BF16) return ce_backward_bf16(*args, kept, grad, grad_x, grad_weight, grad_bias, ws, st);
    return ce_backward_f16(*args, kept, grad, grad_x, grad_weight, grad_bias, ws, st);
}
