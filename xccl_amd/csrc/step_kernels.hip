// step_kernels.hip -- launches of the optimizer step's kernels (step_kernel.hpp).
#include "step_kernel.hpp"

#include <stdio.h>

using namespace xccl_rocm;

namespace {

xccl_status_t launched(const char *what)
{
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        fprintf(stderr, "xccl mc_rocm: launch of %s failed: %s\n", what, hipGetErrorString(e));
        return XCCL_ERR_NO_MESSAGE;
    }
    return XCCL_OK;
}

typedef void (*AdamwKernel)(AdamwKernelArgs);

template <typename P, bool Eight>
AdamwKernel adamw_by_grad(xccl_dt_t grad)
{
    switch ((int)grad) {
    case XCCL_DT_FLOAT32: return adamw_kernel<P, float, Eight>;
    case XCCL_DT_FLOAT16: return adamw_kernel<P, _Float16, Eight>;
    default:              return adamw_kernel<P, __bf16, Eight>;
    }
}

template <bool Eight>
AdamwKernel adamw_by_types(xccl_dt_t param, xccl_dt_t grad)
{
    switch ((int)param) {
    case XCCL_DT_FLOAT32: return adamw_by_grad<float, Eight>(grad);
    case XCCL_DT_FLOAT16: return adamw_by_grad<_Float16, Eight>(grad);
    default:              return adamw_by_grad<__bf16, Eight>(grad);
    }
}

} // namespace

extern "C" {

xccl_status_t step_launch_grad_norm(const xccl_rocm_step_plan_t *plan, double *stats, void *hip_stream)
{
    NormArgs a;
    a.entries     = plan->entries;
    a.chunks      = plan->chunk_table;
    a.partials    = plan->partials;
    a.arrivals    = plan->arrivals;
    a.stats       = stats;
    a.peer_stride = plan->layout.peer_stride;
    a.n_chunks    = (uint32_t)plan->chunks;
    a.n_peers     = plan->layout.n_peers;
    a.writes_fold = plan->writes_fold;
    a.grid        = a.n_chunks < 1 ? 1 : a.n_chunks < STEP_NORM_GRID ? a.n_chunks : STEP_NORM_GRID;
    const dim3        grid(a.grid), block(kStepThreads);
    const hipStream_t s = (hipStream_t)hip_stream;
    switch ((int)plan->layout.grad_dtype) {
    case XCCL_DT_FLOAT32:
        hipLaunchKernelGGL(grad_norm_kernel<float>, grid, block, 0, s, a);
        break;
    case XCCL_DT_FLOAT16:
        hipLaunchKernelGGL(grad_norm_kernel<_Float16>, grid, block, 0, s, a);
        break;
    default:
        hipLaunchKernelGGL(grad_norm_kernel<__bf16>, grid, block, 0, s, a);
        break;
    }
    return launched("grad_norm");
}

xccl_status_t step_launch_adamw(const xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args, void *hip_stream)
{
    const xccl_rocm_step_layout_t &l = plan->layout;
    AdamwKernelArgs a;
    a.entries     = plan->entries;
    a.chunks      = plan->chunk_table;
    a.stats       = args->stats;
    a.clock       = args->clock;
    a.peer_stride = l.peer_stride;
    a.n_peers     = args->use_folded ? 0 : l.n_peers;
    a.use_folded  = args->use_folded != 0;
    a.copy        = l.copy_dtype == XCCL_DT_UNSUPPORTED ? 0 : l.copy_dtype == XCCL_DT_FLOAT16 ? 1 : 2;
    a.b1          = (float)args->beta1;
    a.omb1        = (float)(1 - args->beta1);
    a.b2          = (float)args->beta2;
    a.omb2        = (float)(1 - args->beta2);
    a.eps         = (float)args->eps;
    a.beta1       = args->beta1;
    a.beta2       = args->beta2;
    a.lr          = args->lr;
    a.grad_scale  = args->grad_scale;
    a.max_norm    = args->max_norm;
    a.step        = args->step;

    const hipStream_t s = (hipStream_t)hip_stream;
    if (plan->chunks != 0) {
        const AdamwKernel k = l.state_bits == 8 ? adamw_by_types<true>(l.param_dtype, l.grad_dtype)
                                                : adamw_by_types<false>(l.param_dtype, l.grad_dtype);
        hipLaunchKernelGGL(k, dim3((unsigned)plan->chunks), dim3(kStepThreads), 0, s, a);
        const xccl_status_t st = launched("adamw");
        if (st != XCCL_OK) {
            return st;
        }
    }
    if (args->clock != nullptr) {
        hipLaunchKernelGGL(clock_kernel, dim3(1), dim3(1), 0, s, args->clock, args->stats);
        return launched("the step clock");
    }
    return XCCL_OK;
}

} // extern "C"
