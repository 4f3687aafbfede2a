"""Calls of the optimizer step on the GPU that differ in their pointers, plans and surroundings rather than in their sizes."""
import numpy as np
import pytest

from step_util import F32, NONE, Problem, adamw, grad_norm, ok
from xccl_amd import hip, mc
from xccl_amd.types import MemType, Status

pytestmark = pytest.mark.gpu
INVALID = Status.ERR_INVALID_PARAM


@pytest.fixture(autouse=True)
def _component(rocm):
    return rocm


def test_stats_and_clock_of_plain_host_memory():
    """Refused by every entry, inside a capture as well, which goes on."""
    p = Problem([5000], F32, F32, NONE, 32)
    stream = mc.Stream(hip.stream_create())
    host = np.full(4, -1.0)
    end = hip.DeviceBuffer(8)                                 # 16 bytes from here on run past the allocation
    try:
        grad_norm(p)
        want = p.read_stats().tobytes()
        p.set_stats(-1.0, -1.0)
        hip.stream_begin_capture(stream.hip_stream)
        for where in (host.ctypes.data, 0x1000, end.ptr):
            assert mc.xccl_mem_component_grad_norm(p.plan.handle, where, MemType.ROCM) == INVALID
            assert mc.xccl_mem_component_grad_norm_nb(p.plan.handle, where, MemType.ROCM) == (INVALID, None)
            assert mc.xccl_mem_component_grad_norm_nb(p.plan.handle, where, MemType.ROCM, stream, False)[0] == INVALID
            for name in ("stats", "clock"):
                args = p.args()
                setattr(args, name, where)
                assert mc.xccl_mem_component_adamw(p.plan.handle, args, MemType.ROCM) == INVALID
                assert mc.xccl_mem_component_adamw_nb(p.plan.handle, args, MemType.ROCM, stream, False)[0] == INVALID
        ok(mc.xccl_mem_component_grad_norm_nb(p.plan.handle, p.stats, MemType.ROCM, stream, False))
        graph = hip.stream_end_capture(stream.hip_stream)
        run = hip.graph_instantiate(graph)
        hip.graph_launch(run, stream.hip_stream)
        hip.stream_synchronize(stream.hip_stream)
        assert p.read_stats().tobytes() == want and (host == -1.0).all()
        hip.graph_destroy(graph, run)
        p.arena.download()
        assert all(p.arena.unchanged(x) for t in p.tensors for x in (t.param, t.avg, t.sq))
    finally:
        hip.stream_synchronize(stream.hip_stream)
        hip.stream_destroy(stream.hip_stream)
        end.close()
        p.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_stats_and_clock_in_pinned_host_memory(bits):
    """The host reads the norm and writes the rate where the kernels do; a skipped step does not count there either."""
    p = Problem([5000, 300], F32, F32, NONE, bits)
    at = hip.host_malloc(64)
    words = np.ctypeslib.as_array((np.ctypeslib.ctypes.c_double * 8).from_address(at))
    counts = words.view(np.uint64)
    try:
        grad_norm(p)
        want = p.read_stats()
        words[:] = 0
        ok(mc.xccl_mem_component_grad_norm(p.plan.handle, at + 8, MemType.ROCM))
        assert words[1:3].tobytes() == want.tobytes()
        words[4], counts[5] = 2e-3, 9
        args = p.args(step=0, lr=np.nan, max_norm=0.01)
        args.stats, args.clock = at + 8, at + 32
        adamw(p, args)
        p.check_step(args, 10, lr=2e-3, stats=want)
        assert counts[5] == 10
        words[2] = 3.0                                        # that many elements were not finite
        before = p.arena.now.copy()
        adamw(p, args)
        p.arena.download()
        assert counts[5] == 10 and np.array_equal(p.arena.now, before)
    finally:
        hip.host_free(at)
        p.close()


def test_a_plan_is_destroyed_while_a_stream_is_captured():
    """By its owner or by garbage collection, whenever that comes: the capture goes on, in every mode."""
    p = Problem([5000], F32, bits=0)
    stream = mc.Stream(hip.stream_create())
    try:
        grad_norm(p)
        want = p.read_stats().tobytes()
        for mode in (0, 1, 2):                               # global, thread-local, relaxed
            first, second = mc.StepPlan(p.layout, p.table), mc.StepPlan(p.layout, p.table)
            p.set_stats(-1.0, -1.0)
            hip.stream_begin_capture(stream.hip_stream, mode)
            ok(mc.xccl_mem_component_grad_norm_nb(p.plan.handle, p.stats, MemType.ROCM, stream, False))
            first.close()
            assert first.handle is None
            del second
            graph = hip.stream_end_capture(stream.hip_stream)
            run = hip.graph_instantiate(graph)
            for _ in range(3):
                hip.graph_launch(run, stream.hip_stream)
                hip.stream_synchronize(stream.hip_stream)
                assert p.read_stats().tobytes() == want, mode
                p.set_stats(-1.0, -1.0)
            hip.graph_destroy(graph, run)
    finally:
        hip.stream_synchronize(stream.hip_stream)
        hip.stream_destroy(stream.hip_stream)
        p.close()


def test_the_runtimes_own_streams():
    """The legacy default stream and the per-thread one belong to the current device."""
    p = Problem([5000], F32, F32, NONE, 32)
    try:
        grad_norm(p)
        want = p.read_stats().tobytes()
        for handle in (0, 1, 2):                              # default, legacy, per thread
            p.set_stats(-1.0, -1.0)
            ok(mc.xccl_mem_component_grad_norm_nb(p.plan.handle, p.stats, MemType.ROCM, mc.Stream(handle), False))
            hip.device_synchronize()
            assert p.read_stats().tobytes() == want, handle
    finally:
        p.close()


def test_destroying_a_plan_waits_for_its_calls():
    """A plan that is closed behind a call which still runs: the call is complete when close() returns."""
    n = 1 << 26
    buf = hip.DeviceBuffer(16 * n)
    hip.memset(buf.ptr, 0, 16 * n)
    e = mc.StepTensor(grad=buf.ptr, param=buf.ptr + 4 * n, exp_avg=buf.ptr + 8 * n, exp_avg_sq=buf.ptr + 12 * n, size=n)
    args = mc.AdamwArgs(lr=1.0, beta1=0.5, beta2=0.5, eps=1.0, grad_scale=1.0, step=1)
    stream = mc.Stream(hip.stream_create())
    try:
        for k, one in enumerate((None, stream)):
            ones = np.full(16, float(k + 1), np.float32)
            buf.upload(ones, 4 * (n - 16))
            plan = mc.StepPlan(mc.StepLayout(F32, F32, NONE, 32, 0, 0), [e])
            for _ in range(8):
                ok(mc.xccl_mem_component_adamw_nb(plan.handle, args, MemType.ROCM, one, False))
            plan.close()
            m = buf.download(np.float32, 16, 12 * n - 64)
            if k == 0:
                assert (m == 1 - 2.0 ** -8).all()            # m = 0.5 m + 0.5, eight times
            else:
                assert (m == 2 - 2.0 ** -8 * (2 - (1 - 2.0 ** -8))).all()
    finally:
        hip.stream_synchronize(stream.hip_stream)
        hip.stream_destroy(stream.hip_stream)
        buf.close()
