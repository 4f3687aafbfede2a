/*
 * step_plan.h -- what the host side of the optimizer step (mc_step.c, C) and
 * its kernels (step_kernels.hip) share, and what mc_step.c takes from
 * mc_rocm.c.  Internal to the component.
 */
#ifndef XCCL_ROCM_STEP_PLAN_H_
#define XCCL_ROCM_STEP_PLAN_H_

#include "xccl_rocm_step.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One non-empty tensor, as the kernels read it. */
typedef struct step_entry {
    const char *grad;
    const char *peers;
    char       *folded;
    char       *param;
    char       *copy;
    char       *avg;
    char       *sq;
    float      *avg_scale;
    float      *sq_scale;
    uint64_t    size;
    double      decay;
} step_entry_t;

/* STEP_CHUNK consecutive elements of a tensor (fewer at its end): a workgroup's unit of work. */
#define STEP_CHUNK 4096u
typedef struct step_chunk {
    uint32_t entry;
    uint32_t index;
} step_chunk_t;

/* grad_norm runs at most this many workgroups; each leaves one partial result. */
#define STEP_NORM_GRID 2048u
typedef struct step_partial {
    double sum;
    double bad;
} step_partial_t;

struct xccl_rocm_step_plan {
    xccl_rocm_step_layout_t layout;
    int                     device;
    int                     writes_fold;
    size_t                  chunks;
    char                   *memory;   /* device: the one allocation behind the four pointers below */
    step_entry_t           *entries;
    step_chunk_t           *chunk_table;
    step_partial_t         *partials; /* STEP_NORM_GRID of them */
    uint32_t               *arrivals; /* workgroups of grad_norm that are through; zero between launches */
};

#define STEP_INTERNAL __attribute__((visibility("hidden")))

/* Enqueue on hip_stream (step_kernels.hip). */
STEP_INTERNAL xccl_status_t step_launch_grad_norm(const xccl_rocm_step_plan_t *plan, double *stats, void *hip_stream);
STEP_INTERNAL xccl_status_t step_launch_adamw(const xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args,
                                              void *hip_stream);

/* Runs `launch(arg, stream)` where reduce_multi_nb would have put a reduction
 * (mc_rocm.c): on the caller's stream, or on the calling thread's behind
 * whatever that thread has enqueued. */
STEP_INTERNAL xccl_status_t mc_rocm_enqueue(xccl_status_t (*launch)(void *arg, void *hip_stream), void *arg,
                                            xccl_stream_t *stream, xccl_mc_event_t **event, int want_sync);

#ifdef __cplusplus
}
#endif
#endif /* XCCL_ROCM_STEP_PLAN_H_ */
