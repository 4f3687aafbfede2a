"""What the optimizer step's entries do with a plan in hand, without a GPU: mc_step.c over a stand-in for the device
(tests/step_harness.c), so that a call which should have been refused launches nothing."""
import ctypes
import os
import subprocess

import pytest

from xccl_amd import mc
from xccl_amd.types import Dt, Status

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "xccl_amd", "csrc")
F32, NONE = int(Dt.FLOAT32), int(Dt.UNSUPPORTED)
INVALID = Status.ERR_INVALID_PARAM
MB, GB = 1 << 20, 1 << 30
DEVICE, PINNED, OTHER_DEVICE = (0x7F0000000000 + k * GB for k in range(3))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("step") / "libstep_harness.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-g", "-Wall", "-Wextra", "-Werror", "-D__HIP_PLATFORM_AMD__", "-I",
                    "/opt/rocm/include", "-I", os.path.join(ROOT, "include"), "-I", CSRC, "-o", out,
                    os.path.join(ROOT, "tests", "step_harness.c"), os.path.join(CSRC, "mc_step.c"), "-lm",
                    "-Wl,-Bsymbolic"], check=True)      # its own device, whatever else the process loaded
    lib = ctypes.CDLL(out)
    lib.harness_launches.restype = lib.harness_allocations.restype = ctypes.c_long
    return lib


@pytest.fixture(scope="module")
def step(lib):
    return ctypes.POINTER(mc.RocmStepComponent).in_dll(lib, "xccl_rocm_mem_component_step").contents


@pytest.fixture()
def plan(step):
    lay = mc.StepLayout(F32, F32, NONE, 32, 0, 0)
    table = (mc.StepTensor * 1)(mc.StepTensor(grad=DEVICE, param=DEVICE + MB, exp_avg=DEVICE + 2 * MB,
                                              exp_avg_sq=DEVICE + 3 * MB, size=1000))
    out = ctypes.c_void_p()
    assert step.plan_create(ctypes.byref(lay), table, 1, ctypes.byref(out)) == Status.OK
    yield out.value
    assert step.plan_destroy(out) == Status.OK


def entries(step, plan, stats, clock):
    """Every entry that takes these pointers: (name, call)."""
    args = mc.AdamwArgs(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, grad_scale=1.0, step=1, stats=stats, clock=clock)
    out = [("adamw", lambda: step.adamw(plan, ctypes.byref(args))),
           ("adamw_nb", lambda: step.adamw_nb(plan, ctypes.byref(args), None, None))]
    if clock is None:
        out += [("grad_norm", lambda: step.grad_norm(plan, stats)),
                ("grad_norm_nb", lambda: step.grad_norm_nb(plan, stats, None, None))]
    return out


HOST = ctypes.create_string_buffer(64)


@pytest.mark.parametrize("which", ["stats", "clock"])
@pytest.mark.parametrize("where", [(ctypes.addressof(HOST) + 15) // 16 * 16, 0x1000, 2 ** 64 - 8, OTHER_DEVICE, OTHER_DEVICE + MB,
                                   DEVICE - 8, OTHER_DEVICE + GB - 8], ids=hex)
def test_stats_and_clock_that_the_device_cannot_reach(lib, step, plan, which, where):
    """Plain host memory, no memory at all, memory of another device, and 16 bytes that begin before or end behind it."""
    before = lib.harness_launches()
    for name, call in entries(step, plan, where if which == "stats" else DEVICE + 8 * MB, where if which == "clock" else None):
        assert call() == INVALID, name
    assert lib.harness_launches() == before


@pytest.mark.parametrize("where", [DEVICE, DEVICE + GB - 16, PINNED, PINNED + GB - 16], ids=hex)
def test_stats_and_clock_that_it_can_reach(lib, step, plan, where):
    """Device memory to its last byte, and pinned host memory."""
    before, calls = lib.harness_launches(), entries(step, plan, where, None) + entries(step, plan, where, where)
    for name, call in calls:
        assert call() == Status.OK, name
    assert lib.harness_launches() == before + len(calls) == before + 6


def test_a_plan_that_cannot_be_freed_stays(lib, step):
    """An error of the runtime leaves the plan as it was: usable, and destroyed by the next try."""
    lay = mc.StepLayout(F32, NONE, NONE, 0, 0, 0)
    table = (mc.StepTensor * 1)(mc.StepTensor(grad=DEVICE, size=1000))
    out = ctypes.c_void_p()
    before = lib.harness_allocations()
    assert step.plan_create(ctypes.byref(lay), table, 1, ctypes.byref(out)) == Status.OK
    try:
        lib.harness_fail_free(900)                       # hipErrorStreamCaptureUnsupported
        assert step.plan_destroy(out) == Status.ERR_NO_MESSAGE
        assert lib.harness_allocations() == before + 1
        # looked at without being called, which a plan that is gone would not survive
        assert mc.StepLayout.from_address(out.value).grad_dtype == F32
    finally:
        lib.harness_fail_free(0)
    assert step.grad_norm(out, DEVICE + MB) == Status.OK
    assert step.plan_destroy(out) == Status.OK
    assert lib.harness_allocations() == before


def test_freeing_leaves_captures_alone(lib, step):
    """The runtime's free would invalidate any capture that is going on: it runs in the relaxed mode, which is put back."""
    lay = mc.StepLayout(F32, NONE, NONE, 0, 0, 0)
    table = (mc.StepTensor * 1)(mc.StepTensor(grad=DEVICE, size=1000))
    out = ctypes.c_void_p()
    assert step.plan_create(ctypes.byref(lay), table, 1, ctypes.byref(out)) == Status.OK
    before = lib.harness_mode()
    assert step.plan_destroy(out) == Status.OK
    assert lib.harness_mode_at_free() == 2 and lib.harness_mode() == before == 0


def test_close_says_so(monkeypatch):
    """StepPlan.close() on a plan that could not be destroyed: an exception, and the handle is kept for another try."""
    results = [Status.ERR_NO_MESSAGE, Status.OK]
    seen = []

    def destroy(handle, mem_type):
        seen.append(handle)
        return results[len(seen) - 1]
    monkeypatch.setattr(mc, "xccl_mem_component_step_plan_create", lambda *a: (Status.OK, 0x1230))
    monkeypatch.setattr(mc, "xccl_mem_component_step_plan_destroy", destroy)
    plan = mc.StepPlan(mc.StepLayout(), [])
    with pytest.raises(RuntimeError, match="step_plan_destroy"):
        plan.close()
    assert plan.handle == 0x1230
    plan.close()
    plan.close()                                         # nothing left to do
    assert plan.handle is None and seen == [0x1230, 0x1230]


@pytest.mark.parametrize("elem", [4, 2])
@pytest.mark.parametrize("fold", [0, 1])
def test_no_workgroup_of_the_norm_without_work(lib, fold, elem):
    """As many workgroups of four waves as the chunks of 1024 elements keep busy, up to the most there are.  A wave takes 4 KiB at
    once without peers, half a chunk with them."""
    most = lib.harness_norm_most(fold)
    per_wave = 512 if fold else 4096 // elem                 # elements
    for chunks in [0, 1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 2047, 2048, 2049, 4095, 4096, 4097, 8193, 0x1fffffff]:
        grid = lib.harness_norm_grid(ctypes.c_size_t(chunks), fold, ctypes.c_size_t(elem))
        waves = -(-chunks * 1024 // per_wave)
        assert grid == max(1, min(most, -(-waves // 4))), (chunks, grid)
        assert grid == 1 or (grid - 1) * 4 < waves            # the last workgroup has a wave with work
