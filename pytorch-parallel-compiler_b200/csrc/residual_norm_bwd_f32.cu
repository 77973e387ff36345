// Gradients of the residual norm for f32 tensors.
#define WIDEK_RNORM_BWD_BODY
#include "residual_norm_bwd.cuh"

template int widek::rnorm::BwdLaunch::run<float>();
