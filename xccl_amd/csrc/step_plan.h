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

/* One non-empty tensor, as the kernels read it.  `shift`: elements by which its
 * chunks are moved towards its start, so that they begin on cache lines of as
 * much of what the kernels touch as possible. */
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
    uint32_t    shift;
} step_entry_t;

/* Chunk i of a tensor: those of its elements that lie in [i * STEP_CHUNK - shift, (i + 1) * STEP_CHUNK - shift). */
#define STEP_CHUNK 1024u
typedef struct step_chunk {
    uint32_t entry;
    uint32_t index;
} step_chunk_t;
/* Where the local gradient vector's part of a chunk lies, and its elements: for grad_norm without peers, which does so
 * little with each chunk that looking up chunk, entry and address one after the other would take longer than that. */
typedef struct step_piece {
    const char *grad;
    uint64_t    left;
} step_piece_t;
#define STEP_MAX_CHUNKS 0x1fffffffu /* so that the kernels' counts of chunks and their parts stay within 32 bits */

/* grad_norm runs at most this many workgroups, without and with peers; each leaves one partial result. */
#define STEP_NORM_GRID 512u
#define STEP_FOLD_GRID 1024u
#define STEP_NORM_WAVES 4u    /* of a workgroup */
#define STEP_NORM_BYTES 4096u /* that a wave requests at once without peers: one chunk of 32-bit elements, two of 16-bit ones */
#define STEP_FOLD_TILES 2u    /* of 256 elements, that a wave folds at once */

/* Workgroups of grad_norm: a wave for each piece of work that it takes at once, up to a grid that is resident at once and
 * then goes round.  A workgroup that found no work would still leave a partial result and count itself in. */
static inline uint32_t step_norm_grid(size_t chunks, int fold, size_t elem)
{
    const size_t at_once = STEP_NORM_BYTES / (STEP_CHUNK * elem); /* chunks of a wave */
    const size_t waves   = fold ? chunks * (STEP_CHUNK / 256 / STEP_FOLD_TILES) : (chunks + at_once - 1) / at_once;
    const size_t want    = (waves + STEP_NORM_WAVES - 1) / STEP_NORM_WAVES;
    const size_t most    = fold ? STEP_FOLD_GRID : STEP_NORM_GRID;

    return (uint32_t)(want < 1 ? 1 : want < most ? want : most);
}

typedef struct step_partial {
    double   sum;
    uint64_t bad;
} step_partial_t;

/* Arrivals are counted in two levels, one counter per 128-byte line: STEP_ARRIVAL_SHARDS of them behind the last one. */
#define STEP_ARRIVAL_SHARDS 64u
#define STEP_ARRIVAL_STRIDE 32u
#define STEP_ARRIVAL_BYTES ((1 + STEP_ARRIVAL_SHARDS) * STEP_ARRIVAL_STRIDE * 4)

/* What depends on step number, rate and norm. */
typedef struct step_scalars {
    double lr;
    float  size;   /* lr / (1 - beta1^t) */
    float  inv_c2; /* 1 / sqrt(1 - beta2^t) */
    float  g;      /* factor of the folded gradient */
} step_scalars_t;

struct xccl_rocm_step_plan {
    xccl_rocm_step_layout_t layout;
    int                     device;
    int                     writes_fold;
    size_t                  chunks;
    char                   *memory;   /* device: the one allocation behind the pointers below */
    step_entry_t           *entries;
    step_chunk_t           *chunk_table;
    step_piece_t           *pieces;   /* one per chunk; without peers only */
    step_partial_t         *partials; /* STEP_FOLD_GRID of them */
    uint32_t               *arrivals; /* workgroups of grad_norm that are through (STEP_ARRIVAL_BYTES); zero between launches */
    double                 *zeros;    /* two of them: stats of a step that has none */
    step_scalars_t         *scalars;  /* of the step that runs, where there is a clock */
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
