"""The optimizer step on the GPU where its arithmetic is easily lost: folds that are not written, roots of numbers near the
smallest ones, scales at their borders.  Tolerances as in step_util.py, where not said otherwise."""
import numpy as np
import pytest

from step_util import BF16, BLOCK, E4M3, F16, F32, NAMES, NONE, SIZE, SLACK, U, Problem, adamw, decode, encode, grad_norm
from xccl_amd import hip

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


# ---- exact states in 8 bits: with beta1 = beta2 = 0 and factors of 1, m is the gradient and v its square rounded once ----

def scale_of(x):
    """The smallest power of two that keeps |x| at or below 448 of it, and no smaller than 2^-126."""
    frac, e = np.frexp(np.abs(x).astype(np.float64) / 448)
    return np.where(x == 0, 2.0 ** -126, np.maximum(np.ldexp(1.0, np.where(frac == 0.5, e - 1, e)), 2.0 ** -126))


def nearest_e4m3(y):
    """Nearest values of e4m3, ties to even, of magnitudes up to 448."""
    _, e = np.frexp(np.maximum(np.abs(y), 2.0 ** -6))
    step = np.ldexp(1.0, e - 4)
    return np.rint(y / step) * step


def check_exact_states(g):
    """One element that is not zero in every block; scales and codes bit for bit."""
    n = (len(g) - 1) * BLOCK + 77                     # the last block is short
    at = np.arange(len(g)) * BLOCK + np.arange(len(g)) * 37 % 77
    p = Problem([n], F32, F32, NONE, 8, start="zero")
    try:
        full = np.zeros(n, np.float32)
        full[at] = g
        hip.memcpy_htod(p.table[0].grad, full)
        adamw(p, p.args(lr=0.0, beta1=0.0, beta2=0.0, grad_scale=1.0))
        p.arena.download()
        t = p.tensors[0]
        root = np.sqrt(full * full)                   # in 32 bits, each operation rounded to nearest
        for what, codes, scale, x in (("m", t.avg, t.avg_scale, full), ("root of v", t.sq, t.sq_scale, root)):
            want = scale_of(x[at])
            got = p.arena.get(scale).view(np.float32).astype(np.float64)
            bad = np.flatnonzero(got != want)
            assert not len(bad), "%s: %d of %d scales; first for %r: got %r want %r" % (
                what, len(bad), len(at), x[at][bad[0]], got[bad[0]], want[bad[0]])
            value = nearest_e4m3(x[at] / want)
            if what != "m":
                value = np.where(x[at] > 0, np.maximum(value, 2.0 ** -9), value)
            got = E4M3[p.arena.get(codes)[at]]
            bad = np.flatnonzero(got != value)
            assert not len(bad), "%s: %d of %d codes; first for %r: got %r want %r" % (
                what, len(bad), len(at), x[at][bad[0]], got[bad[0]], value[bad[0]])
            rest = np.ones(n, bool)
            rest[at] = False
            assert not (p.arena.get(codes)[rest] & 127).any(), what
    finally:
        p.close()


def test_roots_at_the_border_of_a_scale():
    """Roots one unit of the last place below, at and above 1.75 2^j, where the scale of the block doubles, for every j that a
    root may have: from those of subnormal v to the largest."""
    j = np.repeat(np.arange(-74, 63), 6)
    k = np.tile([-2, -1, 0, 1, 2, 3], 137)
    g = np.ldexp(1.75 + k * 2.0 ** -23, j)
    check_exact_states(np.concatenate([g, [0.0]]).astype(np.float32))


@pytest.mark.parametrize("low, high", [(-149, -126), (-126, -100), (-80, -60), (-60, -40), (-10, 10), (40, 63)])
def test_states_of_any_magnitude(low, high):
    """Gradients of every exponent, subnormal ones and those whose square vanishes or is subnormal among them."""
    rng = np.random.RandomState(low + 200)
    g = np.ldexp(1 + rng.rand(3000), rng.randint(low, high, 3000)) * rng.choice([-1, 1], 3000)
    check_exact_states(g.astype(np.float32))


def test_roots_of_decayed_states():
    """v = beta2 4^j exactly, from codes of 1, scales of 2^j and no gradient: mantissas of v whose root lies at the border of a
    scale, for every j down to those where v is subnormal."""
    border = np.float32((1.75 + 2.0 ** -23) ** 2 / 4).view(np.int32)
    mantissas = np.concatenate([np.arange(border - 8, border + 8, dtype=np.int32).view(np.float32),
                                np.float32([0.25, 0.3, 0.5, 0.6, 1 - 2.0 ** -24])])
    j = np.arange(-74, 64)
    n = BLOCK * len(j)
    p = Problem([n], F32, F32, NONE, 8, start="zero")
    try:
        t, e = p.tensors[0], p.table[0]
        codes = np.zeros(n, np.uint8)
        codes[::BLOCK] = 0x38
        hip.memcpy_htod(e.grad, np.zeros(n, np.float32))
        for beta2 in mantissas:
            hip.memcpy_htod(e.exp_avg_sq, codes)
            hip.memcpy_htod(e.exp_avg_sq_scale, np.ldexp(1.0, j).astype(np.float32))
            adamw(p, p.args(lr=0.0, beta2=float(beta2)))
            v = np.ldexp(1.0, 2 * j).astype(np.float32) * beta2
            root = np.sqrt(v)
            want = scale_of(root)
            p.arena.download()
            got = p.arena.get(t.sq_scale).view(np.float32).astype(np.float64)
            bad = np.flatnonzero(got != want)
            assert not len(bad), "beta2 %r: %d scales; first for v = %r: got %r want %r" % (
                beta2, len(bad), v[bad[0]], got[bad[0]], want[bad[0]])
            value = np.where(v > 0, np.maximum(nearest_e4m3(root / want), 2.0 ** -9), 0.0)
            assert np.array_equal(E4M3[p.arena.get(t.sq)[::BLOCK]], value), beta2
    finally:
        p.close()


# ---- steps on subnormal v ----

@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", [F32, BF16], ids=NAMES.get)
def test_step_on_the_smallest_v(grad, bits):
    """v of every exponent from the smallest 32-bit number up, and an eps that does not hide them.  Where v is subnormal its
    rounding is no longer relative, so the update is held against the interval that v's bound leaves."""
    n, rng = 4096 + 77, np.random.RandomState(3)
    p = Problem([n], grad, F32, NONE, bits, start="zero")
    try:
        t = p.tensors[0]
        exponents = rng.randint(-149, -90, n)
        if bits == 8:
            exponents = np.repeat(rng.randint(-149, -90, n // BLOCK + 1), BLOCK)[:n]
        root = np.sqrt(np.ldexp(1 + rng.rand(n), exponents))
        t.g = [decode(encode(root * rng.uniform(2, 4, n) * rng.choice([-1, 1], n), grad), grad)]
        hip.memcpy_htod(p.table[0].grad, encode(t.g[0], grad))
        if bits == 32:
            t.m = (root * rng.randn(n)).astype(np.float32).astype(np.float64)
            t.v = (root * root).astype(np.float32).astype(np.float64)
            hip.memcpy_htod(p.table[0].exp_avg, t.m.astype(np.float32))
            hip.memcpy_htod(p.table[0].exp_avg_sq, t.v.astype(np.float32))
        eps = float(np.finfo(np.float32).tiny)
        args = p.args(eps=eps, grad_scale=1.0)
        adamw(p, args)
        p.arena.download()
        b1, b2, tiny = args.beta1, args.beta2, 2.0 ** -150
        g = t.g[0]
        m = b1 * t.m + (1 - b1) * g
        em = U * (3 * np.abs(b1 * t.m) + 3 * np.abs((1 - b1) * g)) * SLACK + 3 * tiny
        v = b2 * t.v + (1 - b2) * g * g
        # as in check_step, and each of the roundings off by up to half a step of a subnormal number
        ev = U * (4 * b2 * t.v + 4 * (1 - b2) * g * g) * SLACK + (3 + np.abs(g)) * tiny
        size, c2 = args.lr / (1 - b1 ** 5), np.sqrt(1 - b2 ** 5)
        low = np.sqrt(np.maximum(v - ev, 0)) * (1 - 2 * U) / c2 * (1 - 3 * U) + eps * (1 - 2 * U)
        high = np.sqrt(v + ev) * (1 + 2 * U) / c2 * (1 + 3 * U) + eps * (1 + 2 * U)
        a, b = size * (np.abs(m) - em), size * (np.abs(m) + em)
        most, least = b / low * (1 + 6 * U), np.where(a > 0, a / high, a / low) * (1 - 6 * U)
        kept = t.p * (1 - args.lr * t.decay)
        got = decode(p.arena.get(t.param), F32)
        ep = 3 * U * (np.abs(t.p) + most) * SLACK
        sign = np.where(m < 0, -1.0, 1.0)
        update = (kept - got) * sign
        bad = ~((update >= least - ep) & (update <= most + ep))
        i = int(np.argmax(bad))
        assert not bad.any(), "%d of %d; first at %d: v %r m %r update %r, allowed %r to %r" % (
            bad.sum(), n, i, v[i], m[i], update[i], least[i] - ep[i], most[i] + ep[i])
        assert (most[v > 2.0 ** -126] / np.abs(least[v > 2.0 ** -126]) < 1 + 1e-5).mean() > 0.9   # the intervals say something
        assert (v < 2.0 ** -126).mean() > 0.2
    finally:
        p.close()
