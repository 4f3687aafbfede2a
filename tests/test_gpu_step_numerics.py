"""The optimizer step on the GPU where its arithmetic is easily lost: folds that are not written, roots of numbers near the
smallest ones, scales at their borders.  Tolerances as in step_util.py, where not said otherwise."""
import numpy as np
import pytest

from step_util import BF16, F16, F32, NAMES, NONE, SIZE, U, Problem, adamw, encode, grad_norm, ok
from xccl_amd import hip, mc
from xccl_amd.types import MemType

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _component(rocm):
    return rocm


def set_gradient(problem, i, vector, at, value):
    """Element `at` of vector `vector` (0: the local one) of tensor i, on the device and in the problem."""
    t, e, size = problem.tensors[i], problem.table[i], SIZE[problem.grad]
    where = e.grad if vector == 0 else e.peers + (vector - 1) * problem.stride
    hip.memcpy_htod(where + at * size, encode(np.array([value]), problem.grad))
    t.g[vector][at] = value


def check_norm_in_32_bits(problem):
    """stats of a fold that is written nowhere: its only roundings are those of the additions in 32 bits."""
    total, bad = problem.read_stats()
    low = high = 0.0
    for t in problem.tensors:
        a, ea = problem.fold_of(t)
        low += float(np.sum(np.maximum(np.abs(a) - ea, 0) ** 2))
        high += float(np.sum((np.abs(a) + ea) ** 2))
    slack = (sum(t.n for t in problem.tensors) + 2) * 2.0 ** -53   # every partial sum is rounded once
    assert low * (1 - slack) <= total <= high * (1 + slack), (total, low, high)
    assert bad == 0


@pytest.mark.parametrize("grad", [F16, BF16, F32], ids=NAMES.get)
@pytest.mark.parametrize("peers", [1, 3, 8])
def test_norm_of_a_fold_that_is_not_written(grad, peers):
    """Without `folded` the norm is that of the sum in 32 bits, not of that sum rounded to the gradient's type."""
    p = Problem([1, 255, 256, 257, 3000, 4099], grad, F32, NONE, 32, peers=peers, shift=True)
    try:
        grad_norm(p)
        check_norm_in_32_bits(p)
    finally:
        p.close()


def test_a_fold_beyond_its_type_that_is_not_written():
    """fp16 vectors whose sum has no fp16 value: finite in 32 bits, not counted, and the step that folds them itself is done,
    clipped by the norm of what it steps."""
    p = Problem([700, 300], F16, F32, NONE, 32, peers=1, magnitude=1.0)
    try:
        for i, at, value in ((0, 5, 40000.0), (0, 699, -60000.0), (1, 256, 65504.0)):
            set_gradient(p, i, 0, at, value)
            set_gradient(p, i, 1, at, value)
        grad_norm(p)
        check_norm_in_32_bits(p)
        stats = p.read_stats()
        args = p.args(max_norm=1.0, use_stats=True)
        adamw(p, args)
        p.check_step(args, 5, stats=stats)
    finally:
        p.close()
