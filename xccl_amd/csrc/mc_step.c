/*
 * mc_step.c -- host side of the optimizer step (include/xccl_rocm_step.h):
 * checks the caller's list of tensors, lays the plan's tables out on the
 * device once, and enqueues the kernels of step_kernels.hip the way
 * mc_rocm.c enqueues a reduction.
 */
#include "step_plan.h"

#include <float.h>
#include <hip/hip_runtime_api.h>
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

/* Byte counts below stay far from wrapping. */
#define STEP_MAX_SIZE ((size_t)1 << 44)

static size_t step_dt_size(xccl_dt_t dt)
{
    switch ((int)dt) {
    case XCCL_DT_FLOAT32:
        return 4;
    case XCCL_DT_FLOAT16:
    case (int)XCCL_ROCM_DT_BFLOAT16:
        return 2;
    default:
        return 0;
    }
}

static xccl_status_t step_check_layout(const xccl_rocm_step_layout_t *l)
{
    const size_t grad = step_dt_size(l->grad_dtype);

    if (l->state_bits != 0 && l->state_bits != 8 && l->state_bits != 32) {
        return XCCL_ERR_INVALID_PARAM;
    }
    if (grad == 0) {
        return XCCL_ERR_UNSUPPORTED;
    }
    if (l->n_peers > XCCL_ROCM_STEP_MAX_PEERS || (l->n_peers > 0 && l->peer_stride % grad != 0)) {
        return XCCL_ERR_INVALID_PARAM;
    }
    if (l->state_bits == 0) {
        return l->param_dtype == XCCL_DT_UNSUPPORTED && l->copy_dtype == XCCL_DT_UNSUPPORTED ? XCCL_OK
                                                                                             : XCCL_ERR_INVALID_PARAM;
    }
    if (step_dt_size(l->param_dtype) == 0) {
        return XCCL_ERR_UNSUPPORTED;
    }
    if (l->copy_dtype != XCCL_DT_UNSUPPORTED &&
        (l->param_dtype != XCCL_DT_FLOAT32 || step_dt_size(l->copy_dtype) != 2)) {
        return XCCL_ERR_UNSUPPORTED;
    }
    return XCCL_OK;
}

/* A stretch of memory that a call on the plan reads or writes. */
typedef struct step_range {
    uintptr_t   lo, hi;
    size_t      tensor;
    const char *what;
    int         written;
} step_range_t;

typedef struct step_ranges {
    step_range_t *at;
    size_t        used;
} step_ranges_t;

static int step_range_order(const void *a, const void *b)
{
    const step_range_t *x = (const step_range_t *)a, *y = (const step_range_t *)b;

    return x->lo != y->lo ? (x->lo < y->lo ? -1 : 1) : (x->hi != y->hi ? (x->hi < y->hi ? -1 : 1) : 0);
}

/* `ptr` of `bytes` bytes has to be there (`want`) or absent, aligned, and must not run past the address space. */
static int step_add(step_ranges_t *r, size_t tensor, const char *what, const void *ptr, int want, size_t bytes,
                    size_t align, int written)
{
    const uintptr_t lo = (uintptr_t)ptr;

    if ((ptr != NULL) != (want != 0)) {
        fprintf(stderr, "xccl mc_rocm: step plan: tensor %zu %s `%s`\n", tensor, want ? "lacks" : "must not have", what);
        return 0;
    }
    if (ptr == NULL) {
        return 1;
    }
    if (lo % align != 0 || lo + bytes < lo) {
        fprintf(stderr, "xccl mc_rocm: step plan: tensor %zu: `%s` at %p is not aligned to its %zu-byte elements\n",
                tensor, what, ptr, align);
        return 0;
    }
    r->at[r->used++] = (step_range_t){.lo = lo, .hi = lo + bytes, .tensor = tensor, .what = what, .written = written};
    return 1;
}

/* The ranges of one tensor, or 0 if something about it is wrong. */
static int step_check_tensor(const xccl_rocm_step_layout_t *l, const xccl_rocm_step_tensor_t *t, size_t i, int folds,
                             step_ranges_t *r)
{
    const size_t gs = step_dt_size(l->grad_dtype), ps = step_dt_size(l->param_dtype), n = t->size;
    const size_t cs = l->copy_dtype == XCCL_DT_UNSUPPORTED ? 2 : step_dt_size(l->copy_dtype);
    const int    steps = l->state_bits != 0, eight = l->state_bits == 8;
    const size_t ss = eight ? 1 : 4, scales = (n + XCCL_ROCM_STEP_BLOCK - 1) / XCCL_ROCM_STEP_BLOCK * 4;
    const int    on_grad = t->folded != NULL && t->folded == t->grad;
    const int    on_peer = t->folded != NULL && t->folded == t->peers && !on_grad;
    uint32_t     j;

    if (n > STEP_MAX_SIZE || !(t->weight_decay >= 0) || isinf(t->weight_decay)) {
        fprintf(stderr, "xccl mc_rocm: step plan: tensor %zu: size %zu, weight decay %g\n", i, n, t->weight_decay);
        return 0;
    }
    if (!step_add(r, i, "grad", t->grad, 1, n * gs, gs, on_grad)) {
        return 0;
    }
    if (l->n_peers == 0 && t->peers != NULL) {
        fprintf(stderr, "xccl mc_rocm: step plan: tensor %zu must not have `peers`\n", i);
        return 0;
    }
    for (j = 0; j < l->n_peers; j++) {
        const uintptr_t off = (uintptr_t)j * l->peer_stride;

        if (l->peer_stride > SIZE_MAX / XCCL_ROCM_STEP_MAX_PEERS / 2 || (uintptr_t)t->peers + off < off ||
            !step_add(r, i, "peers", t->peers == NULL ? NULL : (char *)t->peers + off, 1, n * gs, gs,
                      on_peer && j == 0)) {
            return 0;
        }
    }
    /* on top of `grad` or of the first peer it is that range, counted as written */
    if (folds ? !(on_grad || on_peer) : t->folded != NULL) {
        if (!step_add(r, i, "folded", t->folded, folds, n * gs, gs, 1)) {
            return 0;
        }
    }
    return step_add(r, i, "param", t->param, steps, n * ps, ps ? ps : 1, 1) &&
           step_add(r, i, "copy", t->copy, l->copy_dtype != XCCL_DT_UNSUPPORTED, n * cs, cs, 1) &&
           step_add(r, i, "exp_avg", t->exp_avg, steps, n * ss, ss, 1) &&
           step_add(r, i, "exp_avg_sq", t->exp_avg_sq, steps, n * ss, ss, 1) &&
           step_add(r, i, "exp_avg_scale", t->exp_avg_scale, eight, scales, 4, 1) &&
           step_add(r, i, "exp_avg_sq_scale", t->exp_avg_sq_scale, eight, scales, 4, 1);
}

/* Nothing written may overlap anything else. */
static int step_check_overlap(step_ranges_t *r)
{
    const step_range_t *reach = NULL, *wrote = NULL; /* the ranges so far that reach furthest, of all and of the written */
    size_t              i;

    qsort(r->at, r->used, sizeof(*r->at), step_range_order);
    for (i = 0; i < r->used; i++) {
        const step_range_t *x = &r->at[i], *y = x->written ? reach : wrote;

        if (y != NULL && y->hi > x->lo) {
            fprintf(stderr, "xccl mc_rocm: step plan: `%s` of tensor %zu overlaps `%s` of tensor %zu\n", x->what,
                    x->tensor, y->what, y->tensor);
            return 0;
        }
        if (reach == NULL || x->hi > reach->hi) {
            reach = x;
        }
        if (x->written && (wrote == NULL || x->hi > wrote->hi)) {
            wrote = x;
        }
    }
    return 1;
}

/* Whether kernels on `device` may touch the byte at p: memory of that device, managed, or (`pinned`) of the host and at
 * the same address for the device. */
static int step_reaches(int device, uintptr_t p, int pinned)
{
    hipPointerAttribute_t a;

    if (hipPointerGetAttributes(&a, (void *)p) != hipSuccess) {
        (void)hipGetLastError();
        return 0;
    }
    return a.type == hipMemoryTypeManaged || a.isManaged || (a.type == hipMemoryTypeDevice && a.device == device) ||
           (pinned && a.type == hipMemoryTypeHost && (uintptr_t)a.devicePointer == p);
}

/* First and last byte of every range are memory that the current device may touch. */
static int step_check_memory(const step_ranges_t *r, int device)
{
    size_t i;

    for (i = 0; i < r->used; i++) {
        if (!step_reaches(device, r->at[i].lo, 0) || !step_reaches(device, r->at[i].hi - 1, 0)) {
            fprintf(stderr, "xccl mc_rocm: step plan: `%s` of tensor %zu is not memory of device %d\n", r->at[i].what,
                    r->at[i].tensor, device);
            return 0;
        }
    }
    return 1;
}

/* `stats` or `clock` of a call, 16 bytes that its kernels read or write. */
static int step_check_words(const char *what, const void *ptr, int device)
{
    const uintptr_t p = (uintptr_t)ptr, last = p + 15;

    if (last < p || !step_reaches(device, p, 1) || !step_reaches(device, last, 1)) {
        fprintf(stderr, "xccl mc_rocm: step: `%s` at %p is not memory of device %d\n", what, ptr, device);
        return 0;
    }
    return 1;
}

static size_t step_up(size_t n)
{
    return (n + 255) & ~(size_t)255;
}

/* A wave's stores that begin and end inside 128-byte lines leave two lines
 * half written, and its loads touch one line more.  Chunks are moved by up to
 * 63 elements so that as many of the arrays as possible, by bytes touched, have
 * them on lines: all of them where the tensors are slices of flat buffers at
 * the same place.  Blocks of 8-bit states begin with the tensor and cannot move.
 * Measured, step in 32 bits on 32 Mi elements, all arrays 4 bytes off their
 * lines: 137 us on lines, 174-218 us as they lie. */
static uint32_t step_shift(const xccl_rocm_step_layout_t *l, const xccl_rocm_step_tensor_t *t)
{
    const struct {
        const void *ptr;
        size_t      elem;
        unsigned    times;
    } arrays[] = {
        {t->grad, step_dt_size(l->grad_dtype), 1},   {t->peers, step_dt_size(l->grad_dtype), l->n_peers},
        {t->folded, step_dt_size(l->grad_dtype), 2}, {t->param, step_dt_size(l->param_dtype), 3},
        {t->copy, 2, 2},                             {t->exp_avg, 4, 3},
        {t->exp_avg_sq, 4, 3},
    };
    uint32_t shift, best = 0;
    size_t   score, most = 0, k;

    if (l->state_bits == 8) {
        return 0;
    }
    for (shift = 0; shift < 64; shift++) {
        for (score = 0, k = 0; k < sizeof(arrays) / sizeof(arrays[0]); k++) {
            /* chunk 1 begins at element STEP_CHUNK - shift */
            if (arrays[k].ptr != NULL && ((uintptr_t)arrays[k].ptr + (STEP_CHUNK - shift) * arrays[k].elem) % 128 == 0) {
                score += arrays[k].times * arrays[k].elem;
            }
        }
        if (score > most) {
            most = score;
            best = shift;
        }
    }
    return best;
}

/* Lays the tables out in host memory, and on the device in one allocation. */
static xccl_status_t step_build(xccl_rocm_step_plan_t *plan, const xccl_rocm_step_tensor_t *tensors, size_t count)
{
    size_t        i, entries = 0, chunks = 0, bytes, at_chunks, at_pieces, at_partials, at_arrivals, at_scalars;
    uint32_t      k;
    char         *image;
    step_entry_t *e;
    step_chunk_t *c;
    step_piece_t *g;
    void         *stream = NULL;
    xccl_status_t st;

    for (i = 0; i < count; i++) {
        if (tensors[i].size != 0) {
            entries++;
            chunks += (tensors[i].size + step_shift(&plan->layout, &tensors[i]) + STEP_CHUNK - 1) / STEP_CHUNK;
        }
    }
    if (chunks > STEP_MAX_CHUNKS) {
        fprintf(stderr, "xccl mc_rocm: step plan: %zu pieces of %u elements, at most %u are possible\n", chunks,
                STEP_CHUNK, STEP_MAX_CHUNKS);
        return XCCL_ERR_INVALID_PARAM;
    }
    at_chunks   = step_up(entries * sizeof(*e));
    at_pieces   = at_chunks + step_up(chunks * sizeof(*c));
    at_partials = at_pieces + (plan->layout.n_peers == 0 ? step_up(chunks * sizeof(*g)) : 0);
    at_arrivals = at_partials + STEP_FOLD_GRID * sizeof(step_partial_t);
    at_scalars  = at_arrivals + step_up(STEP_ARRIVAL_BYTES);
    bytes       = at_scalars + 256;
    image       = (char *)calloc(1, bytes);
    if (image == NULL) {
        return XCCL_ERR_NO_MEMORY;
    }
    e = (step_entry_t *)image;
    c = (step_chunk_t *)(image + at_chunks);
    g = (step_piece_t *)(image + at_pieces);
    for (i = 0, entries = 0; i < count; i++) {
        const xccl_rocm_step_tensor_t *t = &tensors[i];

        if (t->size == 0) {
            continue;
        }
        e[entries] = (step_entry_t){
            .grad = (const char *)t->grad, .peers = (const char *)t->peers, .folded = (char *)t->folded,
            .param = (char *)t->param, .copy = (char *)t->copy, .avg = (char *)t->exp_avg,
            .sq = (char *)t->exp_avg_sq, .avg_scale = t->exp_avg_scale, .sq_scale = t->exp_avg_sq_scale,
            .size = t->size, .decay = t->weight_decay, .shift = step_shift(&plan->layout, t),
        };
        for (k = 0; k < (t->size + e[entries].shift + STEP_CHUNK - 1) / STEP_CHUNK; k++) {
            const size_t end  = (size_t)(k + 1) * STEP_CHUNK - e[entries].shift;
            const size_t from = k == 0 ? 0 : end - STEP_CHUNK;

            *c++ = (step_chunk_t){.entry = (uint32_t)entries, .index = k};
            if (plan->layout.n_peers == 0) {
                *g++ = (step_piece_t){.grad = e[entries].grad + from * step_dt_size(plan->layout.grad_dtype),
                                      .left = (end < t->size ? end : t->size) - from};
            }
        }
        entries++;
    }
    st = xccl_rocm_mem_component.get_stream(&stream);
    if (st == XCCL_OK && hipMalloc((void **)&plan->memory, bytes) != hipSuccess) {
        (void)hipGetLastError();
        plan->memory = NULL;
        st           = XCCL_ERR_NO_MEMORY;
    }
    if (st == XCCL_OK &&
        (hipMemcpyAsync(plan->memory, image, bytes, hipMemcpyHostToDevice, (hipStream_t)stream) != hipSuccess ||
         hipStreamSynchronize((hipStream_t)stream) != hipSuccess)) {
        (void)hipGetLastError();
        (void)hipFree(plan->memory);
        st = XCCL_ERR_NO_MESSAGE;
    }
    free(image);
    plan->chunks      = chunks;
    plan->entries     = (step_entry_t *)plan->memory;
    plan->chunk_table = (step_chunk_t *)(plan->memory + at_chunks);
    plan->pieces      = (step_piece_t *)(plan->memory + at_pieces);
    plan->partials    = (step_partial_t *)(plan->memory + at_partials);
    plan->arrivals    = (uint32_t *)(plan->memory + at_arrivals);
    plan->zeros       = (double *)(plan->memory + at_scalars + 128);
    plan->scalars     = (step_scalars_t *)(plan->memory + at_scalars);
    return st;
}

static xccl_status_t mc_step_plan_create(const xccl_rocm_step_layout_t *layout, const xccl_rocm_step_tensor_t *tensors,
                                         size_t count, xccl_rocm_step_plan_t **out)
{
    xccl_rocm_step_plan_t *plan;
    step_ranges_t          ranges = {NULL, 0};
    xccl_status_t          st;
    size_t                 i, per_tensor;
    int                    folds = 0;

    if (layout == NULL || out == NULL || (tensors == NULL && count > 0)) {
        return XCCL_ERR_INVALID_PARAM;
    }
    *out = NULL;
    st   = step_check_layout(layout);
    if (st != XCCL_OK) {
        return st;
    }
    per_tensor = 9 + layout->n_peers;
    if (count > ((size_t)1 << 31) / per_tensor) {
        return XCCL_ERR_INVALID_PARAM;
    }
    for (i = 0; i < count; i++) {
        folds |= tensors[i].size != 0 && tensors[i].folded != NULL;
    }
    if (folds && layout->n_peers == 0) {
        fprintf(stderr, "xccl mc_rocm: step plan: `folded` without peers\n");
        return XCCL_ERR_INVALID_PARAM;
    }
    ranges.at = (step_range_t *)malloc((count * per_tensor + 1) * sizeof(*ranges.at));
    plan      = (xccl_rocm_step_plan_t *)calloc(1, sizeof(*plan));
    if (ranges.at == NULL || plan == NULL) {
        st = XCCL_ERR_NO_MEMORY;
    }
    for (i = 0; i < count && st == XCCL_OK; i++) {
        if (tensors[i].size != 0 && !step_check_tensor(layout, &tensors[i], i, folds, &ranges)) {
            st = XCCL_ERR_INVALID_PARAM;
        }
    }
    if (st == XCCL_OK && !step_check_overlap(&ranges)) {
        st = XCCL_ERR_INVALID_PARAM;
    }
    if (st == XCCL_OK) {
        plan->layout      = *layout;
        plan->writes_fold = folds;
        if (hipGetDevice(&plan->device) != hipSuccess) {
            (void)hipGetLastError();
            st = XCCL_ERR_NO_MESSAGE;
        } else if (!step_check_memory(&ranges, plan->device)) {
            st = XCCL_ERR_INVALID_PARAM;
        } else {
            st = step_build(plan, tensors, count);
        }
    }
    free(ranges.at);
    if (st != XCCL_OK) {
        free(plan);
        return st;
    }
    *out = plan;
    return XCCL_OK;
}

static xccl_status_t mc_step_plan_destroy(xccl_rocm_step_plan_t *plan)
{
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    hipError_t           e, swapped;

    if (plan == NULL) {
        return XCCL_ERR_INVALID_PARAM;
    }
    /* In the thread's usual mode hipFree is an error while any stream of the process is being captured, and invalidates
     * that capture, which need not have anything to do with the plan. */
    swapped = hipThreadExchangeStreamCaptureMode(&mode);
    e       = hipFree(plan->memory); /* waits for the device */
    if (swapped == hipSuccess) {
        (void)hipThreadExchangeStreamCaptureMode(&mode);
    }
    if (e != hipSuccess && e != hipErrorDeinitialized) {
        (void)hipGetLastError();
        return XCCL_ERR_NO_MESSAGE; /* the plan is as it was */
    }
    free(plan);
    return XCCL_OK;
}

static xccl_status_t step_check_device(const xccl_rocm_step_plan_t *plan)
{
    int device = -1;

    if (hipGetDevice(&device) != hipSuccess) {
        (void)hipGetLastError();
        return XCCL_ERR_NO_MESSAGE;
    }
    if (device != plan->device) {
        fprintf(stderr, "xccl mc_rocm: step plan of device %d used while device %d is current\n", plan->device, device);
        return XCCL_ERR_INVALID_PARAM;
    }
    return XCCL_OK;
}

typedef struct step_call {
    const xccl_rocm_step_plan_t  *plan;
    const xccl_rocm_adamw_args_t *args;
    double                       *stats;
} step_call_t;

static xccl_status_t step_enqueue_norm(void *arg, void *hip_stream)
{
    const step_call_t *c = (const step_call_t *)arg;

    return step_launch_grad_norm(c->plan, c->stats, hip_stream);
}

static xccl_status_t step_enqueue_adamw(void *arg, void *hip_stream)
{
    const step_call_t *c = (const step_call_t *)arg;

    return step_launch_adamw(c->plan, c->args, hip_stream);
}

static xccl_status_t step_grad_norm(xccl_rocm_step_plan_t *plan, double *stats, xccl_stream_t *stream,
                                    xccl_mc_event_t **event, int want_sync)
{
    step_call_t   call = {.plan = plan, .stats = stats};
    xccl_status_t st;

    if (plan == NULL || stats == NULL || (uintptr_t)stats % sizeof(double) != 0) {
        return XCCL_ERR_INVALID_PARAM;
    }
    st = step_check_device(plan);
    if (st == XCCL_OK && !step_check_words("stats", stats, plan->device)) {
        st = XCCL_ERR_INVALID_PARAM;
    }
    return st != XCCL_OK ? st : mc_rocm_enqueue(step_enqueue_norm, &call, stream, event, want_sync);
}

/* Not finite, or outside [low, high). */
static int step_outside(double x, double low, double high)
{
    return !(x >= low && x < high);
}

static xccl_status_t step_adamw(xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *a, xccl_stream_t *stream,
                                xccl_mc_event_t **event, int want_sync)
{
    step_call_t   call = {.plan = plan, .args = a};
    xccl_status_t st;

    if (plan == NULL || a == NULL || plan->layout.state_bits == 0) {
        return XCCL_ERR_INVALID_PARAM;
    }
    /* eps is added in 32 bits and keeps the quotient finite where m and v are 0: it has to be a normal number there */
    if (step_outside(a->beta1, 0, 1) || step_outside(a->beta2, 0, 1) || step_outside(a->eps, FLT_MIN, FLT_MAX) ||
        step_outside(a->grad_scale, FLT_MIN, FLT_MAX) || step_outside(a->max_norm, 0, INFINITY) ||
        (a->clock == NULL && (step_outside(a->lr, 0, FLT_MAX) || a->step == 0)) ||
        (a->max_norm > 0 && a->stats == NULL) || (uintptr_t)a->stats % sizeof(double) != 0 ||
        (uintptr_t)a->clock % sizeof(double) != 0 || (a->use_folded && !plan->writes_fold)) {
        return XCCL_ERR_INVALID_PARAM;
    }
    st = step_check_device(plan);
    if (st == XCCL_OK && ((a->stats != NULL && !step_check_words("stats", a->stats, plan->device)) ||
                          (a->clock != NULL && !step_check_words("clock", a->clock, plan->device)))) {
        st = XCCL_ERR_INVALID_PARAM;
    }
    return st != XCCL_OK ? st : mc_rocm_enqueue(step_enqueue_adamw, &call, stream, event, want_sync);
}

static xccl_status_t mc_step_grad_norm(xccl_rocm_step_plan_t *plan, double *stats)
{
    return step_grad_norm(plan, stats, NULL, NULL, 1);
}

static xccl_status_t mc_step_grad_norm_nb(xccl_rocm_step_plan_t *plan, double *stats, xccl_stream_t *stream,
                                          xccl_mc_event_t **event)
{
    return step_grad_norm(plan, stats, stream, event, 0);
}

static xccl_status_t mc_step_adamw(xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args)
{
    return step_adamw(plan, args, NULL, NULL, 1);
}

static xccl_status_t mc_step_adamw_nb(xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args,
                                      xccl_stream_t *stream, xccl_mc_event_t **event)
{
    return step_adamw(plan, args, stream, event, 0);
}

static const xccl_rocm_step_component_t mc_step_component = {
    .version      = XCCL_ROCM_STEP_VERSION,
    .plan_create  = mc_step_plan_create,
    .plan_destroy = mc_step_plan_destroy,
    .grad_norm    = mc_step_grad_norm,
    .grad_norm_nb = mc_step_grad_norm_nb,
    .adamw        = mc_step_adamw,
    .adamw_nb     = mc_step_adamw_nb,
};

__attribute__((visibility("default"))) const xccl_rocm_step_component_t *const xccl_rocm_mem_component_step =
    &mc_step_component;
