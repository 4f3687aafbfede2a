// step_kernels.hip -- launches of the optimizer step's kernels (step_kernel.hpp).
#include "step_kernel.hpp"

#include <math.h>
#include <stdio.h>
#include <string.h>

using namespace xccl_rocm;

namespace {

xccl_status_t launch(const char *what, const void *fn, unsigned grid, unsigned block, void *args, unsigned lds, void *hip_stream)
{
    void            *argv[1] = {args};
    const hipError_t e       = hipLaunchKernel(fn, dim3(grid), dim3(block), argv, lds, (hipStream_t)hip_stream);
    if (e != hipSuccess) {
        fprintf(stderr, "xccl mc_rocm: launch of %s failed: %s\n", what, hipGetErrorString(e));
        return XCCL_ERR_NO_MESSAGE;
    }
    return XCCL_OK;
}

// Chunks of one launch of the step, 2^33 elements: a grid may not have 2^32 threads.
constexpr size_t kStepLaunchChunks = (size_t)1 << 23;
static_assert(kStepLaunchChunks * kStepTiles * 64 < (size_t)1 << 32, "threads of a launch");

typedef void (*AdamwKernel)(AdamwKernelArgs);

template <typename P, typename G>
AdamwKernel adamw_by_form(bool eight, bool peers)
{
    return eight ? (peers ? adamw_kernel<P, G, true, true> : adamw_kernel<P, G, true, false>)
                 : (peers ? adamw_kernel<P, G, false, true> : adamw_kernel<P, G, false, false>);
}

template <typename P>
AdamwKernel adamw_by_grad(xccl_dt_t grad, bool eight, bool peers)
{
    switch ((int)grad) {
    case XCCL_DT_FLOAT32: return adamw_by_form<P, float>(eight, peers);
    case XCCL_DT_FLOAT16: return adamw_by_form<P, _Float16>(eight, peers);
    default:              return adamw_by_form<P, __bf16>(eight, peers);
    }
}

AdamwKernel adamw_by_types(xccl_dt_t param, xccl_dt_t grad, bool eight, bool peers)
{
    switch ((int)param) {
    case XCCL_DT_FLOAT32: return adamw_by_grad<float>(grad, eight, peers);
    case XCCL_DT_FLOAT16: return adamw_by_grad<_Float16>(grad, eight, peers);
    default:              return adamw_by_grad<__bf16>(grad, eight, peers);
    }
}

// LDS that a workgroup (one wave) of the step asks for and never touches, to
// bound how many share a compute unit: as many as keep 54 KiB of loads in
// flight, one gradient vector counted (56 KiB with 8-bit states, which take
// longer from load to store).  More of them only disturb each other's order of
// access to memory; a step that mostly stays in the memory-side cache does not
// mind.  Measured, us at 0 / 6 / 7 / 8 / 10 / 12 / 16 KiB asked for (32 / 26 /
// 22 / 20 / 16 / 13 / 10 waves):
//   32-bit states, all 32 bits, 256 Mi elements   1217 1229 1190 1163 1149 1111 1152
//   32-bit states, bf16 gradient and copy, 64 Mi   307  304  299  295  293  293  300
//   32-bit states, 3 peers, bf16 copy, 32 Mi       241  238  233  231  229  216  229
//   8-bit states, 32-bit gradient, 256 Mi          718  671  646  674  707  834 1019
//   8-bit states, bf16 gradient and copy, 64 Mi    174  175  175  181  188  217  266
//   8-bit states, bf16, 1 peer, 24 Mi (200 MB)      52   56   61   67   73   89  111
//   32-bit states, fp16, 8 Mi (100 MB)              32   31   31   32   32   33   35
unsigned adamw_lds(const xccl_rocm_step_plan_t *plan, uint32_t n_peers)
{
    const xccl_rocm_step_layout_t &l       = plan->layout;
    const unsigned                 grad    = l.grad_dtype == XCCL_DT_FLOAT32 ? 4 : 2;
    const unsigned                 param   = l.param_dtype == XCCL_DT_FLOAT32 ? 4 : 2;
    const unsigned                 states  = l.state_bits == 8 ? 2 : 8;
    const unsigned                 loads   = (grad + param + states) * kStepTile;
    const unsigned                 waves   = (l.state_bits == 8 ? 56 : 54) * 1024 / loads;
    const size_t                   touched = plan->chunks * STEP_CHUNK * ((1 + n_peers) * grad + param + states);
    if (waves >= 32 || touched <= (size_t)192 << 20) {
        return 0;
    }
    return 160 * 1024 / waves & ~511u;
}

} // namespace

extern "C" {

xccl_status_t step_launch_grad_norm(const xccl_rocm_step_plan_t *plan, double *stats, void *hip_stream)
{
    const bool fold = plan->layout.n_peers != 0;
    NormArgs   a;
    a.entries     = plan->entries;
    a.chunks      = plan->chunk_table;
    a.pieces      = plan->pieces;
    a.partials    = plan->partials;
    a.arrivals    = plan->arrivals;
    a.stats       = stats;
    a.peer_stride = plan->layout.peer_stride;
    a.n_chunks    = (uint32_t)plan->chunks;
    a.n_peers     = plan->layout.n_peers;
    a.writes_fold = plan->writes_fold;
    a.grid        = step_norm_grid(plan->chunks, fold, plan->layout.grad_dtype == XCCL_DT_FLOAT32 ? 4 : 2);
    const void *fn;
    switch ((int)plan->layout.grad_dtype) {
    case XCCL_DT_FLOAT32: fn = fold ? (const void *)fold_norm_kernel<float> : (const void *)grad_norm_kernel<float>; break;
    case XCCL_DT_FLOAT16: fn = fold ? (const void *)fold_norm_kernel<_Float16> : (const void *)grad_norm_kernel<_Float16>; break;
    default:              fn = fold ? (const void *)fold_norm_kernel<__bf16> : (const void *)grad_norm_kernel<__bf16>; break;
    }
    return launch("grad_norm", fn, a.grid, kNormWaves * 64, &a, 0, hip_stream);
}

xccl_status_t step_launch_adamw(const xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args, void *hip_stream)
{
    const xccl_rocm_step_layout_t &l = plan->layout;
    AdamwKernelArgs                a;
    a.entries     = plan->entries;
    a.from        = nullptr;
    a.stats       = args->stats;
    a.zero[0]     = 0;
    a.zero[1]     = 0;
    a.grad_scale  = args->grad_scale;
    a.max_norm    = args->max_norm;
    a.clip        = args->max_norm > 0 && args->clock == nullptr;
    a.s.g         = (float)args->grad_scale;
    a.peer_stride = l.peer_stride;
    a.n_peers     = args->use_folded ? 0 : l.n_peers;
    a.use_folded  = args->use_folded != 0;
    a.copy        = l.copy_dtype == XCCL_DT_UNSUPPORTED ? 0 : l.copy_dtype == XCCL_DT_FLOAT16 ? 1 : 2;
    a.b1          = (float)args->beta1;
    a.omb1        = (float)(1 - args->beta1);
    a.b2          = (float)args->beta2;
    a.omb2        = (float)(1 - args->beta2);
    a.eps         = (float)args->eps;
    if (args->clock != nullptr) {
        ClockArgs c;
        c.clock      = args->clock;
        c.stats      = args->stats != nullptr ? args->stats : plan->zeros;
        c.to         = plan->scalars;
        c.beta1      = args->beta1;
        c.beta2      = args->beta2;
        c.grad_scale = args->grad_scale;
        c.max_norm   = args->max_norm;
        const xccl_status_t st = launch("the step's clock", (const void *)step_clock_kernel, 1, 1, &c, 0, hip_stream);
        if (st != XCCL_OK) {
            return st;
        }
        a.from = plan->scalars;
        memset(&a.s, 0, sizeof(a.s));
    } else {
        step_rate(a.s, args->beta1, args->beta2, args->lr, args->step);
    }
    const AdamwKernel k   = adamw_by_types(l.param_dtype, l.grad_dtype, l.state_bits == 8, a.n_peers != 0);
    const unsigned    lds = adamw_lds(plan, a.n_peers);
    xccl_status_t     st  = XCCL_OK;
    for (size_t done = 0; done < plan->chunks && st == XCCL_OK; done += kStepLaunchChunks) {
        const size_t left = plan->chunks - done;
        a.chunks          = plan->chunk_table + done;
        st = launch("adamw", (const void *)k, (unsigned)(left < kStepLaunchChunks ? left : kStepLaunchChunks) * kStepTiles, 64,
                    &a, lds, hip_stream);
    }
    return st;
}

} // extern "C"
