// Gradients of the residual norm for bf16 tensors.
#define WIDEK_RNORM_BWD_BODY
#include "residual_norm_bwd.cuh"

template int widek::rnorm::BwdLaunch::run<__nv_bfloat16>();
