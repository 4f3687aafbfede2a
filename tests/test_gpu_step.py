"""The optimizer step on the GPU against its plain form in 64 bits (step_util.py, where the tolerances come from)."""
import ctypes
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

from step_util import (BF16, BLOCK, E4M3, F16, F32, HALF, NAMES, NONE, SIZE, SLACK, SMALL, U, Problem, adamw, assert_near,
                       decode, encode, grad_norm, ok)
from xccl_amd import hip, mc
from xccl_amd.types import Dt, MemType, Op, Status

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# around the lane (4), the tile and block (256), the chunk (4096), and what is left over
EDGES = [0, 1, 2, 3, 4, 5, 63, 64, 255, 256, 257, 0, 511, 1023, 4095, 4096, 4097, 8193, 12345]
TYPES = [F32, BF16, F16]


@pytest.fixture(autouse=True)
def _component(rocm):
    return rocm


def run_step(problem, step=5, **kw):
    args = problem.args(step=step, **kw)
    adamw(problem, args)
    return args


def check_norm(problem):
    """stats and the folded gradient against 64 bits; returns the values that were summed."""
    problem.arena.download()
    got = problem.read_stats()
    values = []
    total = low = high = 0.0
    for i, t in enumerate(problem.tensors):
        a, ea = problem.fold_of(t)
        if problem.peers:
            ea = ea + HALF[problem.grad] * (np.abs(a) + ea) + SMALL[problem.grad]
            if problem.fold:
                at = {"own": t.folded, "grad": t.grad, "peers": None}[problem.fold]
                if at is None:
                    raw = problem.arena.get(problem.slab)[t.pos * SIZE[problem.grad]:][:t.n * SIZE[problem.grad]]
                else:
                    raw = problem.arena.get(at)
                written = decode(raw, problem.grad)
                assert_near(written, a, ea, "tensor %d: folded gradient" % i)
                a, ea = written, 0.0
        values.append(a)
        total += float(np.sum(a * a))
        low += float(np.sum(np.maximum(np.abs(a) - ea, 0) ** 2))
        high += float(np.sum((np.abs(a) + ea) ** 2))
    n = sum(t.n for t in problem.tensors)
    slack = (n + 2) * 2.0 ** -53   # every partial sum is rounded once
    assert low * (1 - slack) <= got[0] <= high * (1 + slack), (got[0], total, low, high)
    assert got[1] == 0
    return values


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("param", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("grad", TYPES, ids=NAMES.get)
def test_step_types(bits, param, grad):
    """Every type of gradient and parameter, sizes around every boundary, pieces off alignment by an element or two."""
    for shift, copy in ((False, NONE), (True, BF16 if param == F32 else NONE), (True, F16 if param == F32 else NONE)):
        p = Problem(EDGES, grad, param, copy, bits, shift=shift, seed=11 + shift)
        try:
            args = run_step(p)
            p.check_step(args, 5)
            assert all(p.arena.unchanged(t.grad) for t in p.tensors)
        finally:
            p.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_first_steps_from_zero_states(bits):
    """Steps 1 and 2 from states of zero bytes; the second is checked from what the first left."""
    p = Problem([1, 300, 4097], F32, F32, NONE, bits, start="zero")
    try:
        args = run_step(p, step=1)
        p.check_step(args, 1)
        for t in p.tensors:
            t.p = decode(p.arena.get(t.param), F32)
            if bits == 32:
                t.m, t.v = decode(p.arena.get(t.avg), F32), decode(p.arena.get(t.sq), F32)
            else:
                scale = lambda piece: np.repeat(p.arena.get(piece).view(np.float32).astype(np.float64), BLOCK)[:t.n]  # noqa: E731
                t.m = E4M3[p.arena.get(t.avg)] * scale(t.avg_scale)
                t.v = (E4M3[p.arena.get(t.sq)] * scale(t.sq_scale)) ** 2
        args = run_step(p, step=2)
        p.check_step(args, 2)
    finally:
        p.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """Hundreds of tensors in one call, most of them small."""
    rng = np.random.RandomState(3)
    sizes = [int(x) for x in np.exp(rng.uniform(0, np.log(9000), 700))]
    p = Problem(sizes, BF16, F32, BF16, bits, shift=True)
    try:
        p.check_step(run_step(p, step=100), 100)
    finally:
        p.close()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("step, kw", [(1, {}), (3, dict(beta1=0.0, beta2=0.0)), (10 ** 6, dict(beta2=0.999, eps=1e-6)),
                                      (2 ** 40, dict(beta1=0.99, lr=0.0)), (7, dict(grad_scale=1e-4, lr=10.0))], ids=str)
def test_hyperparameters(bits, step, kw):
    p = Problem([1000, 4096], F32, F32, NONE, bits)
    try:
        p.check_step(run_step(p, step=step, **kw), step)
    finally:
        p.close()


@pytest.mark.parametrize("magnitude", [1e-30, 1e-18, 1e-8, 1e8, 1e15])
@pytest.mark.parametrize("bits", [32, 8])
def test_magnitudes(bits, magnitude):
    """Gradients far from 1: scales of the 8-bit blocks follow, and nothing overflows on the way."""
    p = Problem([257, 5000], F32, F32, NONE, bits, magnitude=magnitude)
    try:
        p.check_step(run_step(p), 5)
    finally:
        p.close()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("peers", [1, 2, 7, 16])
def test_step_folds_the_peers(bits, grad, peers):
    """The gradient as 2 to 17 vectors, the peers' an odd number of elements apart."""
    p = Problem([1, 255, 256, 3000, 4099], grad, F32, NONE, bits, peers=peers, shift=True, peer_pad=1)
    try:
        p.check_step(run_step(p, grad_scale=1.0 / (1 + peers)), 5)
    finally:
        p.close()


def test_most_peers():
    p = Problem([1, 300], BF16, F32, NONE, 32, peers=mc.STEP_MAX_PEERS, fold="own")
    try:
        grad_norm(p)
        values = check_norm(p)
        p.check_step(run_step(p, grad_scale=1.0 / 256, use_folded=True), 5, folds=values)
    finally:
        p.close()


@pytest.mark.parametrize("stride", [0, (1 << 32) + 68])
def test_peer_strides(stride):
    """The same vector as every peer's, and vectors more than 2^32 bytes apart."""
    n, peers = 5000, 2
    rng = np.random.RandomState(4)
    rows = [rng.randn(n).astype(np.float32) for _ in range(1 + peers)]
    buf = hip.DeviceBuffer((peers - 1) * stride + n * 4 + 256)
    p = Problem([n], F32, F32, NONE, 32, peers=peers)
    try:
        t = p.tensors[0]
        t.g = [r.astype(np.float64) for r in (rows if stride else [rows[0], rows[2], rows[2]])]
        hip.memcpy_htod(p.table[0].grad, rows[0])
        for j in range(peers):
            buf.upload(rows[1 + j], j * stride + 4)
        p.table[0].peers, p.layout.peer_stride = buf.ptr + 4, stride
        p.plan.close()
        p.plan = mc.StepPlan(p.layout, p.table)
        grad_norm(p)
        a, ea = p.fold_of(t)
        slack = (n + 2) * 2.0 ** -53 + 2 * U
        got = p.read_stats()
        assert np.sum(np.maximum(np.abs(a) - ea, 0) ** 2) * (1 - slack) <= got[0] <= np.sum((np.abs(a) + ea) ** 2) * (1 + slack)
        p.check_step(run_step(p), 5)
    finally:
        p.close()
        buf.close()


def test_a_fold_that_overflows_its_type():
    """fp16 vectors whose sum has no fp16 value: infinite as written, counted, and the step that reads it is skipped."""
    p = Problem([700], F16, F32, NONE, 32, peers=1, fold="own", magnitude=1.0, plant=[(0, 5, 40000.0), (0, 699, -60000.0)])
    try:
        for at, value in ((5, 40000.0), (699, -60000.0)):
            hip.memcpy_htod(p.table[0].grad + 2 * at, encode(np.array([value]), F16))
        grad_norm(p)
        assert p.read_stats()[1] == 2 and np.isinf(p.read_stats()[0])
        run_step(p, use_stats=True, use_folded=True)
        p.arena.download()
        folded = decode(p.arena.get(p.tensors[0].folded), F16)
        assert folded[5] == np.inf and folded[699] == -np.inf and np.isfinite(folded[6:699]).all()
        assert p.arena.unchanged(p.tensors[0].param)
    finally:
        p.close()


@pytest.mark.parametrize("copy", [F16, BF16], ids=NAMES.get)
def test_large_parameters(copy):
    """Parameters beyond the copy's type: the copy is infinite there, as rounding says, and the parameter is what it is."""
    p = Problem([3000], F32, F32, copy, 32, params=1e5)
    try:
        p.check_step(run_step(p), 5)
        assert copy == BF16 or np.isinf(decode(p.arena.get(p.tensors[0].copy), copy)).any()
    finally:
        p.close()


@pytest.mark.parametrize("fold", [None, "own", "grad", "peers"])
@pytest.mark.parametrize("grad", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("peers", [1, 3, 8])
def test_norm_folds_and_the_step_reads_it(fold, grad, peers):
    """grad_norm over the peers, written beside or over its operands; the clipped step then reads what was written."""
    p = Problem(EDGES, grad, F32, NONE, 32, peers=peers, fold=fold, shift=True)
    try:
        grad_norm(p)
        values = check_norm(p)
        stats = p.read_stats()
        if fold:
            args = run_step(p, max_norm=0.01, use_stats=True, use_folded=True)
            p.check_step(args, 5, stats=stats, folds=values)
        else:
            args = run_step(p, max_norm=0.01, use_stats=True)
            p.check_step(args, 5, stats=stats)
    finally:
        p.close()


@pytest.mark.parametrize("grad", TYPES, ids=NAMES.get)
def test_norm_of_many_tensors(grad):
    """One vector per tensor, a plan of gradients only; equal bits on every call."""
    rng = np.random.RandomState(5)
    sizes = EDGES + [int(x) for x in np.exp(rng.uniform(0, np.log(60000), 300))]
    p = Problem(sizes, grad, bits=0, shift=True)
    try:
        grad_norm(p)
        check_norm(p)
        first = p.read_stats().tobytes()
        for _ in range(3):
            grad_norm(p)
            assert p.read_stats().tobytes() == first
        assert mc.xccl_mem_component_adamw(p.plan.handle, p.args(), MemType.ROCM) == Status.ERR_INVALID_PARAM
    finally:
        p.close()


@pytest.mark.parametrize("magnitude", [1e-38, 1e-25, 1e25, 1e37])
def test_norm_needs_64_bits(magnitude):
    """Squares that a 32-bit number cannot hold."""
    p = Problem([100000], F32, bits=0, magnitude=magnitude)
    try:
        grad_norm(p)
        check_norm(p)
    finally:
        p.close()


@pytest.mark.parametrize("n", [1, 5000, 1 << 20])
def test_norm_of_more_chunks_than_workgroups(n):
    """From one workgroup to workgroups that take several chunks (2048 of 4096 elements at once), in one tensor and in many."""
    for sizes in ([n * 9], [n] * 9):
        p = Problem(sizes, BF16, bits=0)
        try:
            grad_norm(p)
            check_norm(p)
        finally:
            p.close()


@pytest.mark.parametrize("grad", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("peers", [0, 1])
def test_norm_counts_everywhere(grad, peers):
    """Elements that are not finite in the first and last place of tensors, in every part of a wave's rounds: exact count, and
    the next call on mended gradients is as if nothing had been."""
    sizes = [3, 4097, 9000001, 1025]
    plant = [(0, 2, np.nan), (1, 0, np.inf), (1, 4096, -np.inf), (3, 1024, np.nan)]
    plant += [(2, at, (np.inf, -np.inf, np.nan)[at % 3]) for at in (0, 1, 1023, 1024, 4194303, 4194304, 8388608, 9000000)]
    p = Problem(sizes, grad, bits=0, peers=peers, fold="own" if peers else None, plant=plant, shift=True)
    try:
        grad_norm(p)
        total, bad = p.read_stats()
        assert bad == len(plant) and not np.isfinite(total)
        for k, at, _ in plant:
            t = p.tensors[k]
            t.g[-1][at] = 0.0
            where = p.table[k].peers if peers else p.table[k].grad
            hip.memcpy_htod(where + at * SIZE[grad], encode(np.zeros(1), grad))
        p.arena.image = p.arena.dev.download(np.uint8, p.arena.size)
        grad_norm(p)
        check_norm(p)
    finally:
        p.close()


def test_empty_lists():
    for sizes in ([], [0, 0, 0]):
        p = Problem(sizes)
        try:
            grad_norm(p)
            assert p.read_stats().tolist() == [0.0, 0.0]
            p.set_clock(1e-3, 41)
            run_step(p, use_stats=True, max_norm=1.0, use_clock=True)
            assert p.read_clock() == 42
            p.arena.download()
        finally:
            p.close()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("peers", [0, 2])
def test_skipped_step(bits, value, peers):
    """One element that is not finite: counted, and the step writes nothing and does not count."""
    p = Problem([10, 4096, 700], F16, F32, BF16, bits, peers=peers, fold="own" if peers else None,
                plant=[(1, 4095, value), (2, 0, value), (2, 699, value)])
    try:
        p.set_clock(1e-3, 6)
        grad_norm(p)
        total, bad = p.read_stats()
        assert bad == 3 and not np.isfinite(total)
        run_step(p, max_norm=1.0, use_stats=True, use_clock=True, use_folded=bool(peers))
        run_step(p, use_stats=True, use_clock=True, use_folded=bool(peers))       # without clipping too
        assert p.read_clock() == 6
        p.arena.download()
        for t in p.tensors:
            assert all(p.arena.unchanged(x) for x in (t.param, t.copy, t.avg, t.sq, t.avg_scale, t.sq_scale) if x is not None)
        # sums over ranks that went wrong
        for wrong in ((1.0, np.nan), (1.0, -1.0), (np.nan, 0.0), (np.inf, 0.0), (-1.0, 0.0)):
            p.set_stats(*wrong)
            run_step(p, max_norm=1.0, use_stats=True, use_clock=True, use_folded=bool(peers))
            run_step(p, max_norm=1.0, use_stats=True, use_folded=bool(peers))
        assert p.read_clock() == 6
        p.arena.download()
        assert all(p.arena.unchanged(t.param) for t in p.tensors)
    finally:
        p.close()


@pytest.mark.parametrize("value", [np.inf, np.nan])
def test_what_is_not_finite_stays_where_it_is(value):
    """Without `stats` an element that is not finite spoils itself, in 8 bits its block's states, and nothing else."""
    for bits in (32, 8):
        p = Problem([2000, 300], F32, F32, NONE, bits, plant=[(0, 700, value)])
        clean = Problem([2000, 300], F32, F32, NONE, bits, plant=[(0, 700, 0.001)])
        try:
            run_step(p)
            run_step(clean)
            p.arena.download()
            clean.arena.download()
            for t, c in zip(p.tensors, clean.tensors):
                same = np.ones(t.n, bool)
                if t is p.tensors[0]:
                    same[700] = False
                    assert not np.isfinite(decode(p.arena.get(t.param), F32)[700])
                assert np.array_equal(decode(p.arena.get(t.param), F32)[same], decode(clean.arena.get(c.param), F32)[same])
                if bits == 32:
                    for a, b in ((t.avg, c.avg), (t.sq, c.sq)):
                        assert np.array_equal(decode(p.arena.get(a), F32)[same], decode(clean.arena.get(b), F32)[same])
                else:
                    block = np.ones(t.n, bool)
                    if t is p.tensors[0]:
                        block[512:768] = False
                        assert np.isnan(E4M3[p.arena.get(t.avg)[700]]) and np.isnan(E4M3[p.arena.get(t.sq)[700]])
                    for a, b in ((t.avg, c.avg), (t.sq, c.sq)):
                        assert np.array_equal(p.arena.get(a)[block], clean.arena.get(b)[block])
        finally:
            p.close()
            clean.close()


@pytest.mark.parametrize("norm_ratio", [0.25, 1.0, 4.0])
def test_clipping(norm_ratio):
    """Below, at and above the norm; the coefficient multiplies the scaled gradient."""
    p = Problem([5000, 77], BF16, F32, NONE, 32)
    try:
        grad_norm(p)
        stats = p.read_stats()
        args = run_step(p, grad_scale=0.125, max_norm=norm_ratio * float(np.sqrt(stats[0])) * 0.125, use_stats=True)
        p.check_step(args, 5, stats=stats)
    finally:
        p.close()


def test_zero_gradients_and_padding():
    """All gradients zero: norm 0, no division by it, states decay, parameters decay only; all-zero states give no update."""
    p = Problem([300, 4096], F32, F32, NONE, 8, magnitude=0.0, start="zero")
    try:
        grad_norm(p)
        assert p.read_stats().tolist() == [0.0, 0.0]
        args = run_step(p, max_norm=1.0, use_stats=True)
        p.check_step(args, 5, stats=[0.0, 0.0])
        for t in p.tensors:
            assert not p.arena.get(t.avg).any() and not p.arena.get(t.sq).any()
    finally:
        p.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_clock_replaces_step_and_rate(bits):
    p = Problem([3000], F32, F32, NONE, bits)
    try:
        p.set_clock(2e-3, 9)
        args = run_step(p, step=0, lr=np.nan, use_clock=True)
        p.check_step(args, 10, lr=2e-3)
        assert p.read_clock() == 10
    finally:
        p.close()


def test_captured_and_replayed():
    """norm and clipped step in one graph, replayed with eager work and synchronisation between the replays; every replay has
    the bits of the same eager sequence."""
    kw = dict(grad=BF16, param=F32, copy=BF16, bits=8, peers=2, fold="own")
    sizes = [100, 5000, 257]
    eager, graphed = Problem(sizes, **kw), Problem(sizes, **kw)
    stream = mc.Stream(hip.stream_create())
    other = Problem([20000], F32, bits=0)
    try:
        for p in (eager, graphed):
            p.set_clock(1e-3, 0)
        args = {id(p): p.args(max_norm=1e-3, use_stats=True, use_clock=True, use_folded=True) for p in (eager, graphed)}
        hip.stream_begin_capture(stream.hip_stream)
        ok(mc.xccl_mem_component_grad_norm_nb(graphed.plan.handle, graphed.stats, MemType.ROCM, stream, False))
        ok(mc.xccl_mem_component_adamw_nb(graphed.plan.handle, args[id(graphed)], MemType.ROCM, stream, False))
        graph = hip.stream_end_capture(stream.hip_stream)
        run = hip.graph_instantiate(graph)
        assert graphed.read_clock() == 0
        pieces = lambda p: [x for t in p.tensors for x in (t.folded, t.param, t.copy, t.avg, t.sq, t.avg_scale, t.sq_scale)]  # noqa: E731
        for replay in range(4):
            hip.graph_launch(run, stream.hip_stream)
            grad_norm(other)                                                     # eager work beside it
            hip.stream_synchronize(stream.hip_stream)
            grad_norm(eager)
            adamw(eager, args[id(eager)])
            eager.arena.download()
            graphed.arena.download()
            assert graphed.read_stats().tobytes() == eager.read_stats().tobytes()
            assert graphed.read_clock() == eager.read_clock() == replay + 1
            for a, b in zip(pieces(eager), pieces(graphed)):
                assert np.array_equal(eager.arena.get(a), graphed.arena.get(b)), replay
        hip.graph_destroy(graph, run)
    finally:
        hip.stream_synchronize(stream.hip_stream)
        for p in (eager, graphed, other):
            p.close()
        hip.stream_destroy(stream.hip_stream)


def test_two_plans_over_the_same_gradients_at_once():
    """Two graphs and two streams, each with a plan of its own: the scratch memory of one is not the other's."""
    p = Problem([300000, 12345], F32, bits=0)
    twin = mc.StepPlan(p.layout, p.table)
    streams = [mc.Stream(hip.stream_create()) for _ in range(2)]
    out = hip.DeviceBuffer(32)
    try:
        grad_norm(p)
        want = p.read_stats().tobytes()
        graphs = []
        for k, (s, plan) in enumerate(zip(streams, (p.plan, twin))):
            hip.stream_begin_capture(s.hip_stream)
            for _ in range(20):
                ok(mc.xccl_mem_component_grad_norm_nb(plan.handle, out.ptr + 16 * k, MemType.ROCM, s, False))
            g = hip.stream_end_capture(s.hip_stream)
            graphs.append((g, hip.graph_instantiate(g)))
        for _ in range(5):
            hip.memset(out.ptr, 0xFF, 32)
            for (_, run), s in zip(graphs, streams):
                hip.graph_launch(run, s.hip_stream)
            for s in streams:
                hip.stream_synchronize(s.hip_stream)
            assert out.download(np.uint8, 32).tobytes() == want + want
        for g, run in graphs:
            hip.graph_destroy(g, run)
    finally:
        for s in streams:
            hip.stream_synchronize(s.hip_stream)
            hip.stream_destroy(s.hip_stream)
        twin.close()
        out.close()
        p.close()


def test_events_and_the_threads_own_stream():
    """stream None: behind the thread's reductions, whatever queue those took; the event tells when it is complete."""
    n = 4096 * 3 + 5
    p = Problem([n], F32, F32, NONE, 32)
    other = np.random.RandomState(2).randn(n).astype(np.float32)
    src = hip.DeviceBuffer(other.nbytes)
    src.upload(other)
    t = p.tensors[0]
    try:
        for size in (n, 64):      # a reduction too large for, and one small enough for, the component's own completion words
            p.arena.dev.upload(p.arena.image)
            st, ev = mc.xccl_mem_component_reduce_multi_nb(p.table[0].grad, src.ptr, p.table[0].grad, 1, size, 0, Dt.FLOAT32, Op.SUM,
                                                           MemType.ROCM)
            ok(st)
            st, ev2 = mc.xccl_mem_component_grad_norm_nb(p.plan.handle, p.stats, MemType.ROCM)
            ok(st)
            args = p.args(max_norm=0.5, use_stats=True)
            st, ev3 = mc.xccl_mem_component_adamw_nb(p.plan.handle, args, MemType.ROCM)
            ok(st)
            assert ev2 and ev3
            ok(mc.xccl_mc_event_wait(ev3))
            assert mc.xccl_mc_event_query(ev3) == Status.OK and mc.xccl_mc_event_query(ev2) == Status.OK
            for e in (ev, ev2, ev3):
                if e:
                    ok(mc.xccl_mc_event_free(e))
            g = t.g[0].copy()
            g[:size] = (t.g[0][:size].astype(np.float32) + other[:size]).astype(np.float64)
            stats = p.read_stats()
            assert abs(stats[0] - np.sum(g * g)) <= (n + 2) * 2.0 ** -53 * np.sum(g * g)
            p.check_step(args, 5, stats=stats, folds=[g])
            # and a reduction behind the step sees what it wrote
            ok(mc.xccl_mem_component_adamw_nb(p.plan.handle, args, MemType.ROCM, None, False))
            ok(mc.xccl_mem_component_reduce_multi(p.table[0].param, src.ptr, src.ptr, 1, 64, 0, Dt.FLOAT32, Op.SUM, MemType.ROCM))
            p.arena.download()
            want = decode(p.arena.get(t.param), F32)[:64].astype(np.float32) + other[:64]
            assert np.array_equal(src.download(np.float32, 64), want)
            src.upload(other)
    finally:
        src.close()
        p.close()


@pytest.mark.parametrize("grad", [F32, BF16], ids=NAMES.get)
def test_hand_over_to_the_components_own_queue(grad):
    """A step that has been waited for, then a reduction of what it wrote on the component's own dispatch queue, which is
    ordered against no stream; and the reduction's result as the next step's gradient."""
    n = 20000
    p = Problem([n], grad, F32, NONE, 32)
    out = hip.DeviceBuffer(n * 4)
    lib = mc.component_lib()
    try:
        args = p.args()
        for round_ in range(60):
            adamw(p, args)
            before = lib.xccl_rocm_direct_launch_count()
            ok(mc.xccl_mem_component_reduce(p.table[0].param, p.table[0].exp_avg, out.ptr, n, Dt.FLOAT32, Op.SUM, MemType.ROCM))
            assert lib.xccl_rocm_direct_launch_count() > before
            p.arena.download()
            t = p.tensors[0]
            want = p.arena.get(t.param).view(np.float32) + p.arena.get(t.avg).view(np.float32)
            assert np.array_equal(out.download(np.float32, n), want), round_
            if grad == F32:
                ok(mc.xccl_mem_component_reduce(p.table[0].grad, out.ptr, p.table[0].grad, n, Dt.FLOAT32, Op.MAX, MemType.ROCM))
                grad_norm(p)
                g = np.where(t.g[0].astype(np.float32) > want, t.g[0].astype(np.float32), want).astype(np.float64)
                assert abs(p.read_stats()[0] - np.sum(g * g)) <= (n + 2) * 2.0 ** -53 * np.sum(g * g), round_
                t.g[0] = g
    finally:
        out.close()
        p.close()


def test_event_pool_exhausted():
    """No event left: with a stream the error and nothing enqueued, without one the blocking entry."""
    p = Problem([1000], F32, bits=0)
    stream = mc.Stream(hip.stream_create())
    held = []
    try:
        while True:
            st, ev = mc.xccl_mem_component_grad_norm_nb(p.plan.handle, p.stats, MemType.ROCM, stream)
            if st != Status.OK:
                break
            held.append(ev)
            assert len(held) <= 64
        assert st == Status.ERR_NO_RESOURCE and len(held) == 64 and ev is None
        hip.stream_synchronize(stream.hip_stream)
        p.set_stats(-1.0, -1.0)
        assert mc.xccl_mem_component_grad_norm_nb(p.plan.handle, p.stats, MemType.ROCM, stream)[0] == Status.ERR_NO_RESOURCE
        hip.stream_synchronize(stream.hip_stream)
        assert p.read_stats().tolist() == [-1.0, -1.0]
        assert mc.xccl_mem_component_grad_norm_nb(p.plan.handle, p.stats, MemType.ROCM) == (Status.OK, None)
        check_norm(p)
    finally:
        hip.stream_synchronize(stream.hip_stream)
        for ev in held:
            mc.xccl_mc_event_free(ev)
        hip.stream_destroy(stream.hip_stream)
        p.close()


def test_plan_outlives_close():
    """close() (the dispatcher's free_cache) releases the component's streams and events; a plan is the caller's and works on."""
    code = (
        "import sys\n"
        "sys.path[:0] = [%r, %r]\n"
        "from step_util import *\n"
        "hip.set_device(0)\n"
        "assert mc.xccl_mem_component_init() == Status.OK\n"
        "p = Problem([5000, 3], F32, F32, NONE, 8)\n"
        "grad_norm(p)\n"
        "first = p.read_stats().tobytes()\n"
        "mc.xccl_mem_component_free_cache()\n"
        "grad_norm(p)\n"
        "assert p.read_stats().tobytes() == first\n"
        "args = p.args(max_norm=1.0, use_stats=True)\n"
        "ok(mc.xccl_mem_component_adamw_nb(p.plan.handle, args, MemType.ROCM, None, False))\n"
        "mc.xccl_mem_component_free_cache()\n"     # waits for the step
        "p.check_step(args, 5, stats=p.read_stats())\n"
        "p.close()\n"
        "print('done')\n") % (ROOT, os.path.join(ROOT, "tests"))
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout.strip().endswith("done"), out.stdout + out.stderr


def test_several_threads():
    """Blocking calls from four threads, a plan each."""
    problems = [Problem([5000 + 17 * k, 300], F32, F32, NONE, 8 if k % 2 else 32, seed=k) for k in range(4)]
    errors = []

    def work(p):
        try:
            hip.set_device(0)
            for _ in range(10):
                grad_norm(p)
            adamw(p, p.args(max_norm=1.0, use_stats=True))
        except BaseException as e:  # noqa: B902
            errors.append(e)
    try:
        threads = [threading.Thread(target=work, args=(p,)) for p in problems]
        [t.start() for t in threads]
        [t.join() for t in threads]
        assert not errors, errors
        for p in problems:
            stats = p.read_stats()
            p.check_step(p.args(max_norm=1.0), 5, stats=stats)
            check_norm(p)
    finally:
        for p in problems:
            p.close()


def test_memory_that_is_not_the_devices():
    """Plain and pinned host memory, and a tensor that runs past its allocation, are refused before anything is launched."""
    n = 1 << 20
    buf = hip.DeviceBuffer(4 * n * 4)
    host = np.zeros(n, np.float32)
    pinned = hip.host_malloc(4096)
    lay = mc.StepLayout(F32, F32, NONE, 32, 0, 0)

    def create(**kw):
        e = dict(grad=buf.ptr, param=buf.ptr + 4 * n, exp_avg=buf.ptr + 8 * n, exp_avg_sq=buf.ptr + 12 * n, size=1000, weight_decay=0.0)
        e.update(kw)
        return mc.xccl_mem_component_step_plan_create(lay, [mc.StepTensor(**e)], MemType.ROCM)
    try:
        st, plan = create()
        ok(st)
        ok(mc.xccl_mem_component_step_plan_destroy(plan, MemType.ROCM))
        assert create(grad=host.ctypes.data) == (Status.ERR_INVALID_PARAM, None)
        assert create(exp_avg=pinned) == (Status.ERR_INVALID_PARAM, None)
        assert create(param=0x1000) == (Status.ERR_INVALID_PARAM, None)
        assert create(exp_avg_sq=buf.ptr + 12 * n, size=1 << 40) == (Status.ERR_INVALID_PARAM, None)
    finally:
        hip.host_free(pinned)
        buf.close()


def test_managed_memory():
    n = 3000
    rng = np.random.RandomState(1)
    g = rng.randn(n).astype(np.float32)
    p = hip.malloc_managed(n * 4 + 16)
    plan = None
    try:
        ctypes.memmove(p, g.ctypes.data, n * 4)
        plan = mc.StepPlan(mc.StepLayout(F32, NONE, NONE, 0, 0, 0), [mc.StepTensor(grad=p, size=n)])
        at = p + n * 4 + (-(p + n * 4)) % 8
        ok(mc.xccl_mem_component_grad_norm(plan.handle, at, MemType.ROCM))
        got = np.frombuffer((ctypes.c_char * 16).from_address(at), np.float64)
        want = float(np.sum(g.astype(np.float64) ** 2))
        assert abs(got[0] - want) <= (n + 2) * 2.0 ** -53 * want and got[1] == 0
    finally:
        if plan:
            plan.close()
        hip.free(p)


def test_offsets_beyond_32_bits():
    """A tensor of more than 2^32 elements (norm), and states whose byte offsets pass 2^32 (step in 32 and in 8 bits)."""
    n = (1 << 32) + 4096 * 3 + 77
    buf = hip.DeviceBuffer(n * 2)
    stats = hip.DeviceBuffer(16)
    hip.memset(buf.ptr, 0x3C, n * 2)                     # 0x3c3c in bf16 = 0.011474609375
    value = float(decode(np.array([0x3C3C], np.uint16), BF16)[0])
    plan = mc.StepPlan(mc.StepLayout(BF16, NONE, NONE, 0, 0, 0), [mc.StepTensor(grad=buf.ptr, size=n)])
    try:
        ok(mc.xccl_mem_component_grad_norm(plan.handle, stats.ptr, MemType.ROCM))
        got = stats.download(np.float64, 2)
        assert abs(got[0] - n * value * value) <= 1e-6 * n * value * value and got[1] == 0
        last = np.array([0x7F80], np.uint16)             # infinity in the very last element
        buf.upload(last, (n - 1) * 2)
        ok(mc.xccl_mem_component_grad_norm(plan.handle, stats.ptr, MemType.ROCM))
        assert stats.download(np.float64, 2)[1] == 1
    finally:
        plan.close()
        buf.close()
    # bytes of 0x3c are 0.0114871... in 32 bits and 1.5 as an e4m3 code; parameters, states and gradients all hold them
    n = (1 << 30) + 4096 + 7
    buf = hip.DeviceBuffer(n * 16)
    raw = np.frombuffer(b"\x3c" * 4, np.float32).astype(np.float64)[0]
    try:
        for bits in (32, 8):
            hip.memset(buf.ptr, 0x3C, n * 16)
            e = mc.StepTensor(grad=buf.ptr, param=buf.ptr + 4 * n, exp_avg=buf.ptr + 8 * n, exp_avg_sq=buf.ptr + 12 * n, size=n,
                              weight_decay=0.5)
            if bits == 8:
                e.exp_avg_sq = buf.ptr + 9 * n
                e.exp_avg_scale, e.exp_avg_sq_scale = (buf.ptr + 10 * n + 255) // 256 * 256, (buf.ptr + 12 * n + 255) // 256 * 256
            plan = mc.StepPlan(mc.StepLayout(F32, F32, NONE, bits, 0, 0), [e])
            args = mc.AdamwArgs(lr=0.01, beta1=0.9, beta2=0.95, eps=1e-8, grad_scale=1.0, step=3)
            ok(mc.xccl_mem_component_adamw(plan.handle, args, MemType.ROCM))
            plan.close()
            m, v = (raw, raw) if bits == 32 else (1.5 * raw, (1.5 * raw) ** 2)
            m, v = 0.9 * m + 0.1 * raw, 0.95 * v + 0.05 * raw * raw
            p = raw * (1 - 0.005) - 0.01 / (1 - 0.9 ** 3) * m / (np.sqrt(v / (1 - 0.95 ** 3)) + 1e-8)
            for at in (0, (1 << 30) - 8, n - 5000, n - 16):
                got = buf.download(np.float32, 16, 4 * n + 4 * at).astype(np.float64)
                assert_near(got, np.full(16, p), 32 * U * (abs(p) + raw), "parameter at %d, %d bits" % (at, bits))
            assert buf.download(np.uint8, 64, 4 * n - 64).tobytes() == b"\x3c" * 64            # gradients are only read
    finally:
        buf.close()
        stats.close()


def test_more_elements_than_one_launch_takes():
    """A step over more than 2^33 elements goes out in several launches; the places on both sides of the seam, and the last."""
    n = (1 << 33) + 4096 + 77
    grad, param, codes = hip.DeviceBuffer(n * 2), hip.DeviceBuffer(n * 2), hip.DeviceBuffer(n * 2 + 256)
    scales = hip.DeviceBuffer(2 * (n // BLOCK + 1) * 4)
    try:
        for b, byte in ((grad, 0x3C), (param, 0x3D), (codes, 0x30), (scales, 0x3B)):
            hip.memset(b.ptr, byte, b.nbytes)
        scale = np.frombuffer(b"\x3b" * 4, np.float32).astype(np.float64)[0]
        g, p0 = (float(decode(np.array([x], np.uint16), BF16)[0]) for x in (0x3C3C, 0x3D3D))
        plan = mc.StepPlan(mc.StepLayout(BF16, BF16, NONE, 8, 0, 0), [mc.StepTensor(
            grad=grad.ptr, param=param.ptr, exp_avg=codes.ptr, exp_avg_sq=codes.ptr + n, exp_avg_scale=scales.ptr,
            exp_avg_sq_scale=scales.ptr + (n // BLOCK + 1) * 4, size=n, weight_decay=0.5)])
        ok(mc.xccl_mem_component_adamw(plan.handle, mc.AdamwArgs(lr=0.01, beta1=0.9, beta2=0.95, eps=1e-8, grad_scale=1.0, step=3),
                                       MemType.ROCM))
        plan.close()
        m = 0.9 * E4M3[0x30] * scale + 0.1 * g
        v = 0.95 * (E4M3[0x30] * scale) ** 2 + 0.05 * g * g
        p = p0 * (1 - 0.005) - 0.01 / (1 - 0.9 ** 3) * m / (np.sqrt(v / (1 - 0.95 ** 3)) + 1e-8)
        for at in (0, (1 << 32) - 8, (1 << 33) - 1032, (1 << 33) - 8, (1 << 33) + 1016, n - 16):
            got = decode(param.download(np.uint16, 16, 2 * at), BF16)
            assert_near(got, np.full(16, p), HALF[BF16] * abs(p) + 32 * U * (abs(p) + p0), "parameter at %d" % at)
        for at in (0, 1 << 33, n - 16):
            s = scales.download(np.float32, 1, at // BLOCK * 4).astype(np.float64)[0]
            assert_near(E4M3[codes.download(np.uint8, 16, at)] * s, np.full(16, m), 2.0 ** -4 * m * SLACK, "exp_avg at %d" % at)
    finally:
        for b in (grad, param, codes, scales):
            b.close()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("ranks", [2, 4])
def test_a_sharded_training_step(bits, ranks):
    """The operators together, as a sharded optimizer uses them between scatter-reduce and allgather: every rank folds the other
    ranks' vectors of its segment and takes their norm, the sums go through the k-nomial allreduce of the replayed team library,
    and the step runs on the segment.  The ranks' parameters together are those of one step on the whole vector."""
    count = 20011
    rng = np.random.RandomState(ranks)
    grads = [rng.randn(count).astype(np.float32) * 0.01 for _ in range(ranks)]
    shards, stats_in = [], []
    try:
        at = 0
        for r in range(ranks):
            off, length = mc.sra_segment(count, r, ranks, ranks)
            p = Problem([length], F32, F32, BF16, bits, peers=ranks - 1, fold="own", seed=50 + r)
            t = p.tensors[0]
            # own segment, then the peers' in the order in which they arrive
            t.g = [grads[(r + k) % ranks][off:off + length].astype(np.float64) for k in range(ranks)]
            hip.memcpy_htod(p.table[0].grad, t.g[0].astype(np.float32))
            hip.memcpy_htod(p.table[0].peers, np.concatenate([x.astype(np.float32) for x in t.g[1:]]))
            at += length
            shards.append((off, p))
        assert at == count
        for _, p in shards:
            ok(mc.xccl_mem_component_grad_norm_nb(p.plan.handle, p.stats, MemType.ROCM, None, False))
        ok(mc.xccl_mem_component_grad_norm(shards[0][1].plan.handle, shards[0][1].stats, MemType.ROCM))   # all behind it are done
        folds = []
        for _, p in shards:
            folds.append(check_norm(p))
            stats_in.append(p.read_stats())
        ptrs = [p.stats for _, p in shards]
        st, _ = mc.replay_run("allreduce_knomial", ptrs, ptrs, 2, Dt.FLOAT64, Op.SUM, radix=4)
        ok(st)
        # every rank adds the others' sums to its own in an order of its own: ranks - 1 roundings of the total each
        want = sum(s[0] for s in stats_in)
        whole = sum(g.astype(np.float64) for g in grads)
        most = np.sum(sum(np.abs(g.astype(np.float64)) for g in grads) ** 2)
        for (_, p), fold in zip(shards, folds):
            total = p.read_stats()
            assert abs(total[0] - want) <= 2 * ranks * 2.0 ** -53 * want and total[1] == 0
            assert abs(total[0] - np.sum(whole ** 2)) <= 4 * ranks * U * most
            args = p.args(max_norm=0.1, grad_scale=1.0 / ranks, use_stats=True, use_folded=True)
            adamw(p, args)
            p.check_step(args, 5, stats=total, folds=fold)
    finally:
        for _, p in shards:
            p.close()
