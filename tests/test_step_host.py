"""The optimizer step's boundary without a GPU: symbols, structure sizes, and every list of tensors and every argument that
is refused before a device is touched (the addresses below are never dereferenced)."""
import ctypes
import math
import os
import re
import subprocess

import pytest

from xccl_amd import mc
from xccl_amd.types import BFLOAT16, Dt, MemType, Status

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32, F16, NONE = int(Dt.FLOAT32), int(Dt.FLOAT16), int(Dt.UNSUPPORTED)
INVALID, UNSUPPORTED = Status.ERR_INVALID_PARAM, Status.ERR_UNSUPPORTED


@pytest.fixture(scope="module", autouse=True)
def _loaded():
    assert mc.xccl_mem_component_init() == Status.OK


def _header():
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "xccl_rocm_step.h")).read(), flags=re.S)


def test_symbols_and_object():
    lib = mc.dispatch_lib()
    names = set(re.findall(r"\b(xccl_mem_component_[a-z_]+)\s*\(", _header()))
    assert names == {"xccl_mem_component_step_plan_create", "xccl_mem_component_step_plan_destroy",
                     "xccl_mem_component_grad_norm", "xccl_mem_component_grad_norm_nb", "xccl_mem_component_adamw",
                     "xccl_mem_component_adamw_nb"}
    for n in names:
        assert hasattr(lib, n), n
    step = mc.step_component()
    assert step.version == 1
    for name, _ in mc.RocmStepComponent._fields_[1:]:
        assert ctypes.cast(getattr(step, name), ctypes.c_void_p).value, name


def test_structures_match_the_header(tmp_path):
    """Sizes and offsets of the Python mirror against a compiler's."""
    pairs = {"xccl_rocm_step_layout_t": mc.StepLayout, "xccl_rocm_step_tensor_t": mc.StepTensor,
             "xccl_rocm_step_clock_t": mc.StepClock, "xccl_rocm_adamw_args_t": mc.AdamwArgs}
    lines = []
    for c, py in pairs.items():
        lines.append('printf("%%zu\\n", sizeof(%s));' % c)
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (c, f) for f, *_ in py._fields_]
    lines.append('printf("%d %u %u\\n", (int)XCCL_ROCM_DT_BFLOAT16, XCCL_ROCM_STEP_BLOCK, XCCL_ROCM_STEP_MAX_PEERS);')
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "xccl_rocm_step.h"\nint main(void) { %s return 0; }\n' % "\n".join(lines))
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], check=True)
    out = subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()
    want = []
    for py in pairs.values():
        want += [ctypes.sizeof(py)] + [getattr(py, f).offset for f, *_ in py._fields_]
    assert [int(x) for x in out] == want + [BFLOAT16, mc.STEP_BLOCK, mc.STEP_MAX_PEERS]


def test_bfloat16_is_not_a_type_of_the_reductions():
    for op in range(17):
        assert mc.component_lib().xccl_rocm_reduce_supported(BFLOAT16, op) == UNSUPPORTED


BASE = 0x7F0000000000
MB = 1 << 20


def tensor(**kw):
    """A valid list entry for 32-bit parameters, gradients and states, at addresses of no memory."""
    t = dict(grad=BASE, param=BASE + MB, exp_avg=BASE + 2 * MB, exp_avg_sq=BASE + 3 * MB, size=1000, weight_decay=0.0)
    t.update(kw)
    return mc.StepTensor(**t)


def layout(**kw):
    l = dict(grad_dtype=F32, param_dtype=F32, copy_dtype=NONE, state_bits=32, n_peers=0, peer_stride=0)
    l.update(kw)
    return mc.StepLayout(**l)


def create(lay, *tensors):
    st, plan = mc.xccl_mem_component_step_plan_create(lay, tensors, MemType.ROCM)
    assert plan is None
    return st


PEERS = dict(n_peers=2, peer_stride=8 * MB)
EIGHT = dict(exp_avg_scale=BASE + 4 * MB, exp_avg_sq_scale=BASE + 5 * MB)


@pytest.mark.parametrize("lay, why", [
    (dict(grad_dtype=int(Dt.FLOAT64)), UNSUPPORTED), (dict(grad_dtype=int(Dt.INT32)), UNSUPPORTED),
    (dict(grad_dtype=99), UNSUPPORTED), (dict(grad_dtype=-1), UNSUPPORTED), (dict(param_dtype=int(Dt.FLOAT64)), UNSUPPORTED),
    (dict(param_dtype=NONE), UNSUPPORTED), (dict(copy_dtype=F32), UNSUPPORTED), (dict(copy_dtype=int(Dt.INT8)), UNSUPPORTED),
    (dict(param_dtype=F16, copy_dtype=F16), UNSUPPORTED), (dict(state_bits=16), INVALID), (dict(state_bits=4), INVALID),
    (dict(state_bits=0), INVALID), (dict(state_bits=0, param_dtype=NONE, copy_dtype=F16), INVALID),
    (dict(n_peers=256, peer_stride=4096), INVALID), (dict(n_peers=1, peer_stride=4095), INVALID),
    (dict(n_peers=0xffffffff, peer_stride=0), INVALID),
], ids=str)
def test_layouts_refused(lay, why):
    assert create(layout(**lay), tensor()) == why
    assert create(layout(**lay)) == why           # also for an empty list


@pytest.mark.parametrize("lay, change", [
    ({}, dict(grad=None)), ({}, dict(param=None)), ({}, dict(exp_avg=None)), ({}, dict(exp_avg_sq=None)),
    ({}, dict(grad=BASE + 2)), ({}, dict(param=BASE + MB + 1)), ({}, dict(exp_avg=BASE + 2 * MB + 3)),
    ({}, dict(copy=BASE + 6 * MB)), (dict(copy_dtype=F16), {}), (dict(copy_dtype=F16), dict(copy=BASE + 6 * MB + 1)),
    ({}, dict(peers=BASE + 6 * MB)), ({}, dict(folded=BASE + 6 * MB)), (PEERS, {}),
    (PEERS, dict(peers=BASE + 6 * MB + 1)), (PEERS, dict(peers=BASE + 6 * MB, folded=BASE + 5 * MB + 2)),
    ({}, EIGHT), (dict(state_bits=8), {}), (dict(state_bits=8), dict(EIGHT, exp_avg_scale=None)),
    (dict(state_bits=8), dict(EIGHT, exp_avg_sq_scale=BASE + 5 * MB + 2)),
    (dict(state_bits=0, param_dtype=NONE), {}), (dict(grad_dtype=F16), dict(grad=BASE + 1)),
    ({}, dict(weight_decay=-0.1)), ({}, dict(weight_decay=math.nan)), ({}, dict(weight_decay=math.inf)),
    ({}, dict(size=(1 << 44) + 1)), ({}, dict(size=2 ** 64 - 1)), ({}, dict(grad=2 ** 64 - 8)),
    (dict(n_peers=255, peer_stride=2 ** 62), dict(peers=BASE + 6 * MB)),
    # what is written must not overlap anything else
    ({}, dict(param=BASE)), ({}, dict(param=BASE + 3996)), ({}, dict(exp_avg=BASE + MB)), ({}, dict(exp_avg=BASE + 3 * MB + 3996)),
    ({}, dict(exp_avg_sq=BASE + 2 * MB + 4)), (dict(copy_dtype=F16), dict(copy=BASE + MB + 3998)),
    (dict(copy_dtype=F16), dict(copy=BASE + 500)), (PEERS, dict(peers=BASE + MB)), (PEERS, dict(peers=BASE - 6 * MB)),
    (PEERS, dict(peers=BASE + 16 * MB, folded=BASE + 4)), (PEERS, dict(peers=BASE + 16 * MB, folded=BASE + 24 * MB)),
    (dict(state_bits=8), dict(EIGHT, exp_avg_scale=BASE + 2 * MB + 996)), (dict(state_bits=8), dict(EIGHT, exp_avg_sq_scale=BASE + 4 * MB + 12)),
], ids=str)
def test_tensors_refused(lay, change):
    assert create(layout(**lay), tensor(**change)) == INVALID
    # the same entry of size 0 is passed over, whatever it says; the plan itself then needs a device
    if not ({"weight_decay", "size"} & set(change)):
        st, plan = mc.xccl_mem_component_step_plan_create(layout(**lay), [tensor(**dict(change, size=0))], MemType.ROCM)
        assert st != INVALID
        if plan:
            mc.xccl_mem_component_step_plan_destroy(plan, MemType.ROCM)


def test_lists_refused():
    l = layout()
    assert create(l, tensor(), tensor()) == INVALID                          # the same tensor twice
    assert create(l, tensor(), tensor(param=BASE + 9 * MB)) == INVALID       # the same states twice
    far = dict(param=BASE + 11 * MB, exp_avg=BASE + 12 * MB, exp_avg_sq=BASE + 13 * MB)
    assert create(l, tensor(), tensor(grad=BASE + MB + 400, **far)) == INVALID  # a gradient inside another's parameter
    p = layout(**PEERS)
    folded = tensor(peers=BASE + 16 * MB, folded=BASE + 6 * MB)
    plain = tensor(grad=BASE + 10 * MB, peers=BASE + 17 * MB, **far)
    assert create(p, folded, plain) == INVALID and create(p, plain, folded) == INVALID   # `folded` for all or for none
    shared = tensor(peers=BASE + 16 * MB, folded=BASE), tensor(peers=BASE + 17 * MB, folded=BASE, **far)
    assert create(p, *shared) == INVALID                                      # one gradient, written for two tensors
    assert mc.dispatch_lib().xccl_mem_component_step_plan_create(None, None, 0, int(MemType.ROCM), None) == INVALID
    plan = ctypes.c_void_p()
    lib = mc.dispatch_lib()
    assert lib.xccl_mem_component_step_plan_create(ctypes.byref(l), None, 1, int(MemType.ROCM), ctypes.byref(plan)) == INVALID
    table = (mc.StepTensor * 1)(tensor())
    assert lib.xccl_mem_component_step_plan_create(ctypes.byref(l), table, 2 ** 40, int(MemType.ROCM), ctypes.byref(plan)) == INVALID
    assert lib.xccl_mem_component_step_plan_create(ctypes.byref(l), table, 1, int(MemType.ROCM), None) == INVALID


def test_what_may_touch_or_be_shared_passes_the_checks():
    """These get as far as the device: XCCL_ERR_NO_MESSAGE without one, XCCL_ERR_INVALID_PARAM with one (no such memory)."""
    from xccl_amd import hip
    want = INVALID if hip.device_count() > 0 else Status.ERR_NO_MESSAGE
    far = dict(param=BASE + 11 * MB, exp_avg=BASE + 12 * MB, exp_avg_sq=BASE + 13 * MB)
    assert create(layout(), tensor()) == want
    assert create(layout(), tensor(param=BASE + 4000, exp_avg=BASE + 8000, exp_avg_sq=BASE + 12000)) == want  # end to end
    assert create(layout(), tensor(), tensor(**far)) == want                                # one gradient, read twice
    # interleaved peers, as segments of flat vectors lie; the fold over the local vector and over the first peer's
    two = [tensor(peers=BASE + 32 * MB), tensor(grad=BASE + 10 * MB, peers=BASE + 32 * MB + 4000, **far)]
    for where in (None, "grad", "peers"):
        for t in two:
            t.folded = getattr(t, where) if where else None
        assert create(layout(**PEERS), *two) == want, where
    assert create(layout(n_peers=2, peer_stride=0), tensor(peers=BASE + 6 * MB)) == want    # one peer's vector twice
    assert create(layout(state_bits=0, param_dtype=NONE), tensor(param=None, exp_avg=None, exp_avg_sq=None)) == want


class FakePlan(ctypes.Structure):
    """Start of xccl_rocm_step_plan: enough for the argument checks, which come before anything else."""
    _fields_ = [("layout", mc.StepLayout), ("device", ctypes.c_int), ("writes_fold", ctypes.c_int), ("rest", ctypes.c_char * 256)]


GOOD = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, grad_scale=1.0, max_norm=0.0, step=1)


@pytest.mark.parametrize("change", [
    dict(lr=-1.0), dict(lr=math.nan), dict(lr=math.inf), dict(beta1=1.0), dict(beta1=-0.1), dict(beta1=math.nan), dict(beta2=1.0),
    dict(beta2=math.nan), dict(eps=0.0), dict(eps=1e-39), dict(eps=math.nan), dict(eps=math.inf), dict(grad_scale=0.0), dict(grad_scale=1e-39),
    dict(grad_scale=-1.0), dict(grad_scale=math.nan), dict(grad_scale=math.inf), dict(max_norm=-1.0), dict(max_norm=math.nan),
    dict(max_norm=math.inf), dict(max_norm=1.0), dict(step=0), dict(stats=BASE + 4), dict(clock=BASE + 4), dict(use_folded=1),
], ids=str)
def test_adamw_arguments_refused(change):
    plan = FakePlan(layout=layout(), device=0, writes_fold=0)
    args = mc.AdamwArgs(**dict(GOOD, **change))
    assert mc.xccl_mem_component_adamw(ctypes.addressof(plan), args, MemType.ROCM) == INVALID
    assert mc.xccl_mem_component_adamw_nb(ctypes.addressof(plan), args, MemType.ROCM) == (INVALID, None)


def test_calls_refused():
    plan = FakePlan(layout=layout(state_bits=0, param_dtype=NONE), device=0)
    here, args = ctypes.addressof(plan), mc.AdamwArgs(**GOOD)
    assert mc.xccl_mem_component_adamw(here, args, MemType.ROCM) == INVALID       # a plan of gradients only
    assert mc.xccl_mem_component_adamw(None, args, MemType.ROCM) == INVALID
    assert mc.dispatch_lib().xccl_mem_component_adamw(here, None, int(MemType.ROCM)) == INVALID
    assert mc.xccl_mem_component_grad_norm(here, None, MemType.ROCM) == INVALID
    assert mc.xccl_mem_component_grad_norm(here, BASE + 4, MemType.ROCM) == INVALID
    assert mc.xccl_mem_component_grad_norm(None, BASE, MemType.ROCM) == INVALID
    assert mc.xccl_mem_component_step_plan_destroy(None, MemType.ROCM) == INVALID


@pytest.mark.parametrize("mt", [MemType.HOST, MemType.LAST, 99, -1], ids=str)
def test_no_component(mt):
    args = mc.AdamwArgs(**GOOD)
    assert mc.xccl_mem_component_step_plan_create(layout(), [], mt) == (UNSUPPORTED, None)
    assert mc.xccl_mem_component_step_plan_destroy(BASE, mt) == UNSUPPORTED
    assert mc.xccl_mem_component_grad_norm(BASE, BASE, mt) == UNSUPPORTED
    assert mc.xccl_mem_component_grad_norm_nb(BASE, BASE, mt) == (UNSUPPORTED, None)
    assert mc.xccl_mem_component_adamw(BASE, args, mt) == UNSUPPORTED
    assert mc.xccl_mem_component_adamw_nb(BASE, args, mt) == (UNSUPPORTED, None)


def test_component_without_the_step(tmp_path):
    """A component that has no such object (here the host-memory stand-in): XCCL_ERR_NOT_IMPLEMENTED, in a process of its own
    because a loaded component stays."""
    lib = str(tmp_path / "xccl_cuda_mem_component.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-DFAKE_MEMTYPE=1", "-DFAKE_SYMBOL=xccl_cuda_mem_component", "-I", os.path.join(ROOT, "include"), "-o", lib,
                    os.path.join(ROOT, "tests", "fake_component.c")], check=True)
    code = ("from xccl_amd import mc\nfrom xccl_amd.types import MemType, Status\n"
            "assert mc.xccl_mem_component_init(%r) == Status.OK\n"
            "assert mc.dispatch_lib().xccl_mem_component_get(int(MemType.CUDA))\n"
            "assert mc.xccl_mem_component_step_plan_create(mc.StepLayout(), [], MemType.CUDA) == (Status.ERR_NOT_IMPLEMENTED, None)\n"
            "assert mc.xccl_mem_component_adamw(1, mc.AdamwArgs(), MemType.CUDA) == Status.ERR_NOT_IMPLEMENTED\n"
            "assert mc.xccl_mem_component_grad_norm_nb(1, 8, MemType.CUDA) == (Status.ERR_NOT_IMPLEMENTED, None)\n" % str(tmp_path))
    subprocess.run(["python3", "-c", code], check=True, cwd=ROOT)
