/*
 * step_harness.c -- host-only stand-in for the device behind
 * xccl_amd/csrc/mc_step.c, so that what the optimizer step's entries refuse,
 * and what they do when the runtime fails, can be tested without a GPU.
 * Built by tests/test_step_calls.py together with mc_step.c.
 *
 * "Device memory" of device 0 is [HARNESS_BASE, HARNESS_BASE + 1 GiB), pinned
 * host memory the GiB behind it, memory of device 1 the one behind that.  None
 * of it is ever dereferenced.
 */
#include "step_plan.h"

#include <hip/hip_runtime_api.h>
#include <stdlib.h>
#include <string.h>

#define HARNESS_BASE ((uintptr_t)0x7f0000000000)
#define HARNESS_GIB  ((uintptr_t)1 << 30)

static long       launches, allocations;
static hipError_t free_result;
static int        capture_mode, mode_at_free;

long harness_launches(void) { return launches; }
long harness_allocations(void) { return allocations; }
void harness_fail_free(int error) { free_result = (hipError_t)error; }
int  harness_mode_at_free(void) { return mode_at_free; }
int  harness_mode(void) { return capture_mode; }
unsigned harness_norm_grid(size_t chunks, int fold, size_t elem) { return step_norm_grid(chunks, fold, elem); }
unsigned harness_norm_most(int fold) { return fold ? STEP_FOLD_GRID : STEP_NORM_GRID; }

hipError_t hipGetDevice(int *device)
{
    *device = 0;
    return hipSuccess;
}

hipError_t hipGetLastError(void) { return hipSuccess; }

hipError_t hipPointerGetAttributes(hipPointerAttribute_t *a, const void *ptr)
{
    const uintptr_t p = (uintptr_t)ptr;

    memset(a, 0, sizeof(*a));
    a->type   = hipMemoryTypeUnregistered;
    a->device = -2;
    if (p >= HARNESS_BASE && p < HARNESS_BASE + 3 * HARNESS_GIB) {
        const unsigned part = (unsigned)((p - HARNESS_BASE) / HARNESS_GIB);

        a->type          = part == 1 ? hipMemoryTypeHost : hipMemoryTypeDevice;
        a->device        = part == 2;
        a->devicePointer = (void *)p;
    }
    return hipSuccess;
}

hipError_t hipMalloc(void **ptr, size_t size)
{
    *ptr = malloc(size);
    allocations++;
    return *ptr != NULL ? hipSuccess : hipErrorOutOfMemory;
}

hipError_t hipFree(void *ptr)
{
    mode_at_free = capture_mode;
    if (free_result != hipSuccess) {
        return free_result;
    }
    free(ptr);
    allocations--;
    return hipSuccess;
}

hipError_t hipMemcpyAsync(void *dst, const void *src, size_t size, hipMemcpyKind kind, hipStream_t stream)
{
    (void)kind;
    (void)stream;
    memcpy(dst, src, size);
    return hipSuccess;
}

hipError_t hipStreamSynchronize(hipStream_t stream)
{
    (void)stream;
    return hipSuccess;
}

hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode *mode)
{
    const int old = capture_mode;

    capture_mode = (int)*mode;
    *mode        = (hipStreamCaptureMode)old;
    return hipSuccess;
}

xccl_status_t step_launch_grad_norm(const xccl_rocm_step_plan_t *plan, double *stats, void *hip_stream)
{
    (void)plan;
    (void)stats;
    (void)hip_stream;
    launches++;
    return XCCL_OK;
}

xccl_status_t step_launch_adamw(const xccl_rocm_step_plan_t *plan, const xccl_rocm_adamw_args_t *args, void *hip_stream)
{
    (void)plan;
    (void)args;
    (void)hip_stream;
    launches++;
    return XCCL_OK;
}

xccl_status_t mc_rocm_enqueue(xccl_status_t (*launch)(void *arg, void *hip_stream), void *arg, xccl_stream_t *stream,
                              xccl_mc_event_t **event, int want_sync)
{
    (void)stream;
    (void)event;
    (void)want_sync;
    return launch(arg, NULL);
}

static xccl_status_t harness_get_stream(void **stream)
{
    *stream = NULL;
    return XCCL_OK;
}

xccl_rocm_mem_component_t xccl_rocm_mem_component = {.get_stream = harness_get_stream};
