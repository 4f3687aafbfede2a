/*
 * xccl_rocm_step.h -- what a data-parallel trainer does with a gradient that
 * a scatter-reduce or an allreduce has just delivered: its global norm, and
 * an AdamW step over many tensors at once, with optimizer states in 32 or in
 * 8 bits.  The reference has no counterpart; the entries stand beside
 * reduce / reduce_multi and take the same operands where they meet: a
 * gradient may still be `1 + n_peers` vectors, the local one and the peers'
 * `peer_stride` bytes apart, exactly as the last scatter-reduce round leaves
 * them (reference src/team_lib/ucx/allreduce/allreduce_sra.c:281-284), and is
 * then folded in registers instead of by a pass of its own.
 *
 * With a = the folded gradient of an element, everything in 32 bits:
 *
 *   fold    a = grad + peer{0};  a = peer{j} + a,  j = 1 .. n_peers-1
 *   stats   stats[0] = sum of a^2 over all elements of all tensors,
 *           stats[1] = how many of them are infinite or NaN      (64 bits);
 *           where grad_norm writes the fold, a is what it has written
 *   clip    k = min(1, max_norm / (sqrt(stats[0]) * grad_scale + 1e-6))
 *   step    g = a * (grad_scale * k)
 *           m = beta1 m + (1 - beta1) g
 *           v = beta2 v + ((1 - beta2) g) g
 *           p = p (1 - lr weight_decay)
 *               - lr / (1 - beta1^t) * m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
 *
 * A whole step is skipped, nothing written and nothing counted, when the
 * `stats` it is given say that an element was not finite (or are no sum of
 * squares: negative, infinite, NaN): the usual answer to a loss scale that was
 * too large.  Without `stats` such an element goes through the formulas and
 * poisons its own parameter and states only (its block's states, with states
 * in 8 bits).
 *
 * The two doubles of `stats` can be summed over ranks with the component's
 * own FLOAT64 SUM before the step reads them.
 *
 * States in 8 bits.  A block is XCCL_ROCM_STEP_BLOCK consecutive elements of
 * one tensor (the last may be shorter) and has one 32-bit scale per state, a
 * power of two: the smallest that keeps the block's largest magnitude at or
 * below 448 of it, and no smaller than 2^-126.  exp_avg holds m / scale and
 * exp_avg_sq holds sqrt(v) / scale, each rounded to the nearest e4m3 number (4
 * exponent bits, 3 mantissa bits, no infinities; ties to even).  sqrt(v) > 0 is
 * never rounded to 0: its code is at least the smallest, 2^-9, because a zero
 * there would divide a non-zero m by eps alone.  The parameter is updated from
 * m and v as they were before this rounding.  States that are all zero bytes,
 * scales included, are a valid start.
 */
#ifndef XCCL_ROCM_STEP_H_
#define XCCL_ROCM_STEP_H_

#include "xccl_rocm_mem_component.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The 16-bit type with the exponent of FLOAT32.  XCCL's enumeration has no
 * such member (reference src/api/xccl.h:391-407); the entries of this header
 * take this value, every other entry refuses it. */
#define XCCL_ROCM_DT_BFLOAT16 ((xccl_dt_t)15)

#define XCCL_ROCM_STEP_BLOCK     256u
#define XCCL_ROCM_STEP_MAX_PEERS 255u

/* What all tensors of a plan have in common. */
typedef struct xccl_rocm_step_layout {
    xccl_dt_t grad_dtype;  /* FLOAT32, FLOAT16 or BFLOAT16 */
    xccl_dt_t param_dtype; /* the same three; XCCL_DT_UNSUPPORTED if state_bits is 0 */
    xccl_dt_t copy_dtype;  /* FLOAT16 or BFLOAT16, beside FLOAT32 parameters; XCCL_DT_UNSUPPORTED: no copy */
    uint32_t  state_bits;  /* 32 or 8; 0: a plan of gradients only, for grad_norm */
    uint32_t  n_peers;     /* gradient vectors besides the local one, at most XCCL_ROCM_STEP_MAX_PEERS */
    size_t    peer_stride; /* bytes between them, a multiple of the gradient's element size */
} xccl_rocm_step_layout_t;

/*
 * One tensor.  Pointers are device (or managed) memory of the current device,
 * aligned to their element type and to nothing more.  `folded` is where
 * grad_norm writes the folded gradient (rounded once to grad_dtype); given for
 * all tensors or for none, only with peers, and may be exactly `grad` or
 * exactly `peers`; a step after that reads `folded` (use_folded), since the
 * vectors it would fold are no longer what they were.  Apart from that nothing
 * that is written may overlap anything else of the plan.  A tensor of size 0 is
 * passed over.
 */
typedef struct xccl_rocm_step_tensor {
    void  *grad;
    void  *peers;             /* vector 0 of the peers; NULL if n_peers is 0 */
    void  *folded;            /* NULL: the fold is not written */
    void  *param;
    void  *copy;              /* receives the new parameter, rounded to copy_dtype */
    void  *exp_avg;           /* m: float, or codes */
    void  *exp_avg_sq;        /* v: float, or codes of sqrt(v) */
    float *exp_avg_scale;     /* 8 bits only: one per block */
    float *exp_avg_sq_scale;
    size_t size;              /* elements */
    double weight_decay;
} xccl_rocm_step_tensor_t;

/* Step number and learning rate in memory that the device reads: for steps that
 * are captured into a graph, and for steps that may be skipped. */
typedef struct xccl_rocm_step_clock {
    double   lr;
    uint64_t steps; /* steps done so far; a step that is not skipped adds 1 */
} xccl_rocm_step_clock_t;

/* 0 <= beta1, beta2 < 1.  eps and grad_scale are positive normal 32-bit numbers
 * (from 1.2e-38): eps = 0, which would divide 0 by 0 where m and v are, and a
 * gradient that is switched off or negated by its scale are refused.  lr and
 * max_norm are finite and not negative.  What a clock holds is not looked at. */
typedef struct xccl_rocm_adamw_args {
    double   lr, beta1, beta2, eps;
    double   grad_scale;  /* of every folded gradient, e.g. 1 / (ranks * loss scale) */
    double   max_norm;    /* > 0: clip to this norm of the scaled gradient (needs stats); 0: do not clip */
    uint64_t step;        /* number of this step, from 1 */
    const double           *stats; /* what grad_norm wrote, or NULL */
    xccl_rocm_step_clock_t *clock; /* replaces lr and step, or NULL */
    int      use_folded;  /* 1: the gradient is what grad_norm wrote to `folded`, not grad and peers */
} xccl_rocm_adamw_args_t;

/* A plan holds the table of a list of tensors on the device that was current
 * when it was made, and the scratch memory of grad_norm. */
typedef struct xccl_rocm_step_plan xccl_rocm_step_plan_t;

/*
 * The object a component exports beside its vtable, found by the loader as
 * xccl_<memory type name>_mem_component_step.
 *
 * plan_create checks the list (XCCL_ERR_INVALID_PARAM for what the comments
 * above do not allow, XCCL_ERR_UNSUPPORTED for a type without a kernel; says
 * on stderr which tensor), allocates, and synchronises: not inside a capture.
 * The list itself is not kept.  plan_destroy waits for the device, may be called
 * while some stream is being captured, and leaves the plan as it was if it
 * returns an error; graphs that hold calls on the plan must not run any more, and
 * it comes before the component is finalized, which frees no plans.  On the
 * device a plan takes 96 bytes per tensor and 8 (24 without peers) per 1024
 * elements.
 *
 * Steps are fastest when a tensor's arrays begin on 128-byte lines; with states
 * in 32 bits it is enough that they all begin at the same place of one, as
 * slices of flat buffers do.
 *
 * grad_norm and adamw are complete on return.  The _nb forms only enqueue, on
 * `stream` or, if that is NULL, on the component's stream of the calling
 * thread, in order with that thread's reductions; `event` as for
 * reduce_multi_nb.  With event == NULL they may be captured into a graph;
 * grad_norm is one kernel, adamw one, or two with a clock.  Results of equal
 * inputs are equal bit for bit on one device.
 *
 * `stats` (two doubles) and `clock` are memory of the plan's device, managed
 * memory, or pinned host memory; anything else is XCCL_ERR_INVALID_PARAM.
 *
 * Calls on one plan have to be ordered by the caller: they share its scratch
 * memory, and adamw writes its tensors.  That goes for graphs that hold such
 * calls as well; two plans over the same tensors are independent as far as
 * grad_norm without `folded` goes.  The plan's device must be the current one
 * (XCCL_ERR_INVALID_PARAM), `stream` must belong to it.
 */
#define XCCL_ROCM_STEP_VERSION 1u
typedef struct xccl_rocm_step_component {
    uint32_t version;
    xccl_status_t (*plan_create)(const xccl_rocm_step_layout_t *layout, const xccl_rocm_step_tensor_t *tensors,
                                 size_t count, xccl_rocm_step_plan_t **plan);
    xccl_status_t (*plan_destroy)(xccl_rocm_step_plan_t *plan);
    xccl_status_t (*grad_norm)(xccl_rocm_step_plan_t *plan, double *stats);
    xccl_status_t (*grad_norm_nb)(xccl_rocm_step_plan_t *plan, double *stats, xccl_stream_t *stream,
                                  xccl_mc_event_t **event);
    xccl_status_t (*adamw)(xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args);
    xccl_status_t (*adamw_nb)(xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args, xccl_stream_t *stream,
                              xccl_mc_event_t **event);
} xccl_rocm_step_component_t;

/* Defined by xccl_rocm_mem_component.so. */
extern const xccl_rocm_step_component_t *const xccl_rocm_mem_component_step;

/* ------------------------------------------------------------------------
 * Dispatcher (libxccl_mc.so).  No component for the memory type (host memory
 * included): XCCL_ERR_UNSUPPORTED; a component without the object above:
 * XCCL_ERR_NOT_IMPLEMENTED.  An empty event pool falls back to the blocking
 * entry if stream == NULL (*event is NULL then), as for the reductions.
 * ---------------------------------------------------------------------- */
xccl_status_t xccl_mem_component_step_plan_create(const xccl_rocm_step_layout_t *layout,
                                                  const xccl_rocm_step_tensor_t *tensors, size_t count,
                                                  ucs_memory_type_t mem_type, xccl_rocm_step_plan_t **plan);
xccl_status_t xccl_mem_component_step_plan_destroy(xccl_rocm_step_plan_t *plan, ucs_memory_type_t mem_type);
xccl_status_t xccl_mem_component_grad_norm(xccl_rocm_step_plan_t *plan, double *stats, ucs_memory_type_t mem_type);
xccl_status_t xccl_mem_component_grad_norm_nb(xccl_rocm_step_plan_t *plan, double *stats, ucs_memory_type_t mem_type,
                                              xccl_stream_t *stream, xccl_mc_event_t **event);
xccl_status_t xccl_mem_component_adamw(xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args,
                                       ucs_memory_type_t mem_type);
xccl_status_t xccl_mem_component_adamw_nb(xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args,
                                          ucs_memory_type_t mem_type, xccl_stream_t *stream,
                                          xccl_mc_event_t **event);

#ifdef __cplusplus
}
#endif
#endif /* XCCL_ROCM_STEP_H_ */
