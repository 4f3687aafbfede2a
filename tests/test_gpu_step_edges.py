"""The optimizer step on the GPU at the borders of its pieces: 4 elements to a lane, 256 to a tile and to a block of 8-bit states,
1024 to a chunk; and the norm where a round of its workgroups ends (2048 chunks without peers in 32 bits, 4096 in 16, 2048 of a
fold).  Tolerances as in step_util.py."""
import numpy as np
import pytest

from step_util import BF16, F16, F32, HALF, NAMES, NONE, SMALL, Problem, adamw, assert_near, decode, grad_norm

pytestmark = pytest.mark.gpu

SIZES = [1, 5, 253, 254, 255, 256, 257, 259, 511, 513, 767, 769, 1020, 1021, 1023, 1024, 1025, 1027, 1279, 1281, 2047, 2048, 2049, 3073]
TYPES = [F32, BF16, F16]


@pytest.fixture(autouse=True)
def _component(rocm):
    return rocm


def check_stats(p, values, errors):
    total, bad = p.read_stats()
    low = sum(float(np.sum(np.maximum(np.abs(a) - e, 0) ** 2)) for a, e in zip(values, errors))
    high = sum(float(np.sum((np.abs(a) + e) ** 2)) for a, e in zip(values, errors))
    slack = (sum(len(a) for a in values) + 2) * 2.0 ** -53      # every partial sum is rounded once
    assert low * (1 - slack) <= total <= high * (1 + slack), (total, low, high)
    assert bad == 0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("grad", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("peers", [0, 3])
def test_step(grad, param, bits, peers):
    for shift in (False, True):
        p = Problem(SIZES, grad, param, F16 if param == F32 and shift else NONE, bits, peers=peers, shift=shift, seed=21 + shift)
        try:
            args = p.args()
            adamw(p, args)
            p.check_step(args, 5)
            assert all(p.arena.unchanged(t.grad) for t in p.tensors)
        finally:
            p.close()


@pytest.mark.parametrize("grad", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("peers, fold", [(0, None), (1, None), (3, "own"), (3, "grad")])
def test_norm(grad, peers, fold):
    for shift in (False, True):
        p = Problem(SIZES, grad, F32, NONE, 32, peers=peers, fold=fold, shift=shift, seed=31 + shift)
        try:
            grad_norm(p)
            p.arena.download()
            values, errors = zip(*(p.fold_of(t) for t in p.tensors))
            if fold:
                for i, t in enumerate(p.tensors):
                    written = decode(p.arena.get(t.folded if fold == "own" else t.grad), grad)
                    a, e = values[i], errors[i]
                    assert_near(written, a, e + HALF[grad] * (np.abs(a) + e) + SMALL[grad], "fold of tensor %d" % i)
                values = [decode(p.arena.get(t.folded if fold == "own" else t.grad), grad) for t in p.tensors]
                errors = [0.0] * len(values)
            check_stats(p, values, errors)
        finally:
            p.close()


@pytest.mark.parametrize("peers", [0, 1])
@pytest.mark.parametrize("grad", [F32, BF16], ids=NAMES.get)
@pytest.mark.parametrize("chunks", [2, 2047, 2048, 2049, 4096, 4097, 6145])
def test_norm_at_the_end_of_a_round(grad, peers, chunks):
    """An element more and less than so many chunks, in one tensor, and each chunk a tensor of its own."""
    for sizes in ([chunks * 1024 - 1], [chunks * 1024 + 1], [1024] * chunks):
        p = Problem(sizes, grad, bits=0, peers=peers)
        try:
            grad_norm(p)
            values, errors = zip(*(p.fold_of(t) for t in p.tensors))
            check_stats(p, values, errors)
            first = p.read_stats().tobytes()
            grad_norm(p)
            assert p.read_stats().tobytes() == first
        finally:
            p.close()
