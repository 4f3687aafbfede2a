"""Plain 64-bit form of the optimizer step (include/xccl_rocm_step.h) and the arithmetic of its tolerances.

U is half a step of a 32-bit number.  A bound is the sum of the roundings on the way, each at most U (2U for a hardware
square root or reciprocal) of the value it rounds; products of two of them are covered by the factor SLACK."""
import numpy as np

from xccl_amd import hip, mc
from xccl_amd.types import BFLOAT16, Dt, MemType, Status

U = 2.0 ** -24
SLACK = 1.001
TINY = 2.0 ** -63      # square root of the smallest normal 32-bit number: what a flushed square root loses
BLOCK = mc.STEP_BLOCK
F32, F16, BF16, NONE = int(Dt.FLOAT32), int(Dt.FLOAT16), BFLOAT16, int(Dt.UNSUPPORTED)
SIZE = {F32: 4, F16: 2, BF16: 2}
HALF = {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}              # half a step, relative
SMALL = {F32: 2.0 ** -150, F16: 2.0 ** -25, BF16: 2.0 ** -134}  # half a step of a subnormal
NAMES = {F32: "f32", F16: "f16", BF16: "bf16", NONE: "none"}


def encode(x, dt):
    """Bytes of x rounded to nearest even."""
    with np.errstate(over="ignore", invalid="ignore"):
        if dt == F32:
            return np.asarray(x, np.float32)
        if dt == F16:
            return np.asarray(x, np.float16)
        bits = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
        up = (bits + 0x7FFF + ((bits >> 16) & 1)) >> 16
        return np.where(np.isnan(np.asarray(x, np.float32)), (bits >> 16) | 0x40, up).astype(np.uint16)


def decode(raw, dt):
    raw = np.frombuffer(raw.tobytes(), dtype={F32: np.float32, F16: np.float16, BF16: np.uint16}[dt])
    if dt == BF16:
        return (raw.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return raw.astype(np.float64)


def _e4m3():
    """The 256 values an e4m3 code stands for."""
    v = np.zeros(256)
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        x = np.nan if (c & 127) == 127 else (f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
        v[c] = -x if c & 128 else x
    return v


E4M3 = _e4m3()


def blocks(n):
    return -(-n // BLOCK)


def spread(scale, n):
    """Scales of the blocks, one per element."""
    return np.repeat(scale, BLOCK)[:n]


def block_max(x):
    padded = np.zeros(blocks(len(x)) * BLOCK)
    padded[:len(x)] = np.abs(x)
    return padded.reshape(-1, BLOCK).max(1)


def quantize(x):
    """Valid codes and scales for x (not necessarily the nearest codes): a start for 8-bit states."""
    scale = np.maximum(np.exp2(np.ceil(np.log2(np.maximum(block_max(x), 2.0 ** -110) / 448))), 2.0 ** -126)
    order = np.argsort(E4M3[:127])
    table = E4M3[:127][order]
    y = np.abs(x) / spread(scale, len(x))
    code = order[np.clip(np.searchsorted(table, y), 0, 126)].astype(np.uint8)
    return code | np.where(x < 0, 128, 0).astype(np.uint8), scale.astype(np.float32)


class Arena:
    """Device memory with a host image; every piece lies at a chosen offset behind a guard, and `check` says whether any
    byte outside the pieces has changed."""

    GUARD = 192

    def __init__(self):
        self.pieces, self.size, self.dev = [], 0, None

    def add(self, data, shift=0):
        """`shift` bytes past a 64-byte boundary; returns the piece's number."""
        raw = np.ascontiguousarray(data).view(np.uint8).reshape(-1)
        start = (self.size + self.GUARD + 63) // 64 * 64 + shift
        self.pieces.append((start, raw))
        self.size = start + raw.size
        return len(self.pieces) - 1

    def upload(self):
        self.size += self.GUARD
        self.image = np.random.RandomState(7).randint(0, 256, self.size, dtype=np.uint8)
        self.inside = np.zeros(self.size, dtype=bool)
        for start, raw in self.pieces:
            self.image[start:start + raw.size] = raw
            self.inside[start:start + raw.size] = True
        self.dev = hip.DeviceBuffer(self.size)
        self.dev.upload(self.image)

    def ptr(self, piece):
        return None if piece is None else self.dev.ptr + self.pieces[piece][0]

    def download(self):
        self.now = self.dev.download(np.uint8, self.size)
        assert np.array_equal(self.now[~self.inside], self.image[~self.inside]), "bytes outside the tensors changed"

    def get(self, piece):
        start, raw = self.pieces[piece]
        return self.now[start:start + raw.size]

    def unchanged(self, piece):
        start, raw = self.pieces[piece]
        return np.array_equal(self.get(piece), self.image[start:start + raw.size])

    def close(self):
        if self.dev:
            self.dev.close()


class Tensor:
    pass


class Problem:
    """A list of tensors on the device, its plan, and what the formulas give in 64 bits."""

    def __init__(self, sizes, grad=F32, param=F32, copy=NONE, bits=32, peers=0, fold=None, shift=0, seed=1, magnitude=1e-3,
                 start=None, plant=(), peer_pad=0, params=0.05):
        """`fold`: None, "own", "grad" or "peers": where the folded gradient is written.  `shift`: elements every piece is
        moved off alignment, differently for each.  `plant`: (tensor, element, value) put into the last gradient vector.
        `start`: "zero" for states that are all zero.  `params`: magnitude of the parameters."""
        rng = np.random.RandomState(seed)
        self.grad, self.param, self.copy, self.bits, self.peers, self.fold = grad, param, copy, bits, peers, fold
        self.arena, self.tensors = Arena(), []
        total = sum(sizes) + peer_pad
        pos, slab = 0, np.zeros((peers, max(total, 1)))
        for i, n in enumerate(sizes):
            t = Tensor()
            t.n, t.decay = n, (0.1 if i % 3 else 0.0)
            mag = magnitude * 10.0 ** rng.uniform(-1, 1)
            rows = [rng.randn(n) * mag for _ in range(1 + peers)]
            for k, at, value in plant:
                if k == i:
                    rows[-1][at] = value
            t.g = [decode(encode(r, grad), grad) for r in rows]
            off = lambda dt_size, k=0: ((i * 5 + k * 3 + 1) % 4) * dt_size if shift else 0  # noqa: E731
            t.grad = self.arena.add(encode(t.g[0], grad), off(SIZE[grad]))
            for j in range(peers):
                slab[j, pos:pos + n] = t.g[1 + j]
            t.pos, pos = pos, pos + n
            t.folded = self.arena.add(encode(np.zeros(n), grad), off(SIZE[grad], 1)) if fold == "own" else None
            if bits:
                t.p = decode(encode(rng.randn(n) * params, param), param)
                t.param = self.arena.add(encode(t.p, param), off(SIZE[param], 2))
                t.copy = None if copy == NONE else self.arena.add(encode(np.zeros(n), copy), off(2, 3))
                m, v = rng.randn(n) * mag * 0.3, mag * mag * (0.2 + rng.rand(n)) * 10.0 ** rng.uniform(-6, 0, n)
                if start == "zero":
                    m, v = m * 0, v * 0
                if bits == 32:
                    t.m, t.v = m.astype(np.float32).astype(np.float64), v.astype(np.float32).astype(np.float64)
                    t.avg = self.arena.add(t.m.astype(np.float32), off(4, 1))
                    t.sq = self.arena.add(t.v.astype(np.float32), off(4, 2))
                    t.avg_scale = t.sq_scale = None
                else:
                    (mc_, ms), (rc, rs) = quantize(m), quantize(np.sqrt(v))
                    if start == "zero":
                        ms, rs = ms * 0, rs * 0
                    t.m = E4M3[mc_] * spread(ms.astype(np.float64), n)
                    t.v = (E4M3[rc] * spread(rs.astype(np.float64), n)) ** 2
                    t.avg, t.sq = self.arena.add(mc_, off(1)), self.arena.add(rc, off(1, 1))
                    t.avg_scale, t.sq_scale = self.arena.add(ms), self.arena.add(rs)
            self.tensors.append(t)
        self.slab = self.arena.add(encode(slab, grad), SIZE[grad] if shift else 0) if peers else None
        self.stride = slab.shape[1] * SIZE[grad]
        self.stats_piece = self.arena.add(np.full(2, np.nan))
        self.clock_piece = self.arena.add(np.zeros(2, np.uint64))
        self.arena.upload()
        a = self.arena
        self.stats, self.clock = a.ptr(self.stats_piece), a.ptr(self.clock_piece)
        self.layout = mc.StepLayout(grad, param if bits else NONE, copy if bits else NONE, bits, peers, self.stride if peers else 0)
        self.table = []
        for t in self.tensors:
            e = mc.StepTensor(grad=a.ptr(t.grad), size=t.n, weight_decay=t.decay)
            if peers:
                e.peers = a.ptr(self.slab) + t.pos * SIZE[grad]
            e.folded = {None: None, "own": a.ptr(t.folded), "grad": e.grad, "peers": e.peers}[fold]
            if bits:
                e.param, e.copy, e.exp_avg, e.exp_avg_sq = a.ptr(t.param), a.ptr(t.copy), a.ptr(t.avg), a.ptr(t.sq)
                e.exp_avg_scale, e.exp_avg_sq_scale = a.ptr(t.avg_scale), a.ptr(t.sq_scale)
            self.table.append(e)
        self.plan = mc.StepPlan(self.layout, self.table)

    def close(self):
        self.plan.close()
        self.arena.close()

    # ---- what the formulas give ----

    def fold_of(self, t):
        """The folded gradient, and the bound of its rounding in 32 bits."""
        a, mag = t.g[0].copy(), np.abs(t.g[0])
        for p in t.g[1:]:
            a, mag = a + p, mag + np.abs(p)
        return a, self.peers * U * mag * SLACK

    def args(self, step=5, lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, grad_scale=0.5, max_norm=0.0, use_stats=False,
             use_clock=False, use_folded=False):
        return mc.AdamwArgs(lr=lr, beta1=beta1, beta2=beta2, eps=eps, grad_scale=grad_scale, max_norm=max_norm, step=step,
                            stats=self.stats if use_stats else None, clock=self.clock if use_clock else None,
                            use_folded=int(use_folded))

    def set_stats(self, total, bad):
        hip.memcpy_htod(self.stats, np.array([total, bad], np.float64))

    def set_clock(self, lr, steps):
        hip.memcpy_htod(self.clock, np.array([np.float64(lr).view(np.uint64), steps], np.uint64))

    def read_stats(self):
        out = np.empty(2)
        hip.memcpy_dtoh(out, self.stats)
        return out

    def read_clock(self):
        out = np.empty(2, np.uint64)
        hip.memcpy_dtoh(out, self.clock)
        return int(out[1])

    def check_step(self, args, step, lr=None, stats=None, folds=None, m_only=False):
        """Compares what lies on the device with one step from the starting values.  `stats`: the sums the step has read;
        `folds`: the gradients it has read, where those are not the fold itself."""
        self.arena.download()
        f32 = lambda x: float(np.float32(x))  # noqa: E731
        b1, b2, lr = args.beta1, args.beta2, args.lr if lr is None else lr
        k = args.grad_scale
        if args.max_norm > 0:
            k *= min(1.0, args.max_norm / (np.sqrt(stats[0]) * args.grad_scale + 1e-6))
        size, c2 = lr / (1 - b1 ** step), np.sqrt(1 - b2 ** step)
        for i, t in enumerate(self.tensors):
            what = "tensor %d of %d elements" % (i, t.n)
            a, ea = self.fold_of(t) if folds is None else (folds[i], 0.0)
            g = a * k
            eg = np.abs(k) * ea + 2 * U * np.abs(g)                    # the factor, the product
            m = b1 * t.m + (1 - b1) * g
            em = ((1 - b1) * eg + U * (3 * np.abs(b1 * t.m) + 3 * np.abs((1 - b1) * g))) * SLACK   # constants, products, the sum
            v = b2 * t.v + (1 - b2) * g * g
            ev = ((1 - b2) * 2 * np.abs(g) * eg + U * (4 * b2 * t.v + 4 * (1 - b2) * g * g)) * SLACK  # and, in 8 bits, the square
            r = np.sqrt(v)
            er = np.sqrt(v + ev) - np.sqrt(np.maximum(v - ev, 0)) + 2 * U * r + TINY
            d = r / c2 + args.eps
            upd = size * m / d
            eupd = (size * em + np.abs(upd) * er / c2) / d + 12 * U * np.abs(upd)   # size, c2, eps, product, sum, quotient, product
            p = t.p * (1 - lr * t.decay) - upd
            ep = (eupd + 3 * U * (np.abs(t.p) + np.abs(upd))) * SLACK               # the factor, the product, the difference
            got = decode(self.arena.get(t.param), self.param)
            assert_near(got, p, ep + HALF[self.param] * (np.abs(p) + ep) + SMALL[self.param], what + ": parameter")
            if t.copy is not None:
                c = decode(self.arena.get(t.copy), self.copy)
                want = decode(encode(got, self.copy), self.copy)
                assert np.array_equal(c, want), what + ": the copy is not the parameter rounded once"
            if self.bits == 32:
                # where results are subnormal a rounding is off by up to SMALL instead of U of the value: the decayed state, the
                # gradient's term and their sum are each rounded once, so 3 of them
                assert_near(decode(self.arena.get(t.avg), F32), m, em + 3 * SMALL[F32], what + ": exp_avg")
                assert_near(decode(self.arena.get(t.sq), F32), v, ev + 3 * SMALL[F32], what + ": exp_avg_sq")
            elif t.n:
                self.check_codes(t.avg, t.avg_scale, m, em, False, what + ": exp_avg")
                self.check_codes(t.sq, t.sq_scale, r, er, True, what + ": exp_avg_sq")

    def check_codes(self, codes, scale, x, ex, positive, what):
        n = len(x)
        scale = self.arena.get(scale).view(np.float32).astype(np.float64)
        frac, _ = np.frexp(scale)
        assert np.all(frac == 0.5), what + ": a scale is not a power of two"
        low, high = block_max(np.maximum(np.abs(x) - ex, 0)), block_max(np.abs(x) + ex)
        assert np.all((high <= 448 * scale * (1 + U)) | (low <= 448 * scale)), what + ": a scale is too small"
        assert np.all((scale == 2.0 ** -126) | (high > 224 * scale)), what + ": a scale is too large"
        s = spread(scale, n)
        y = E4M3[self.arena.get(codes)] * s
        # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the smallest normal code
        bound = np.maximum(2.0 ** -4 * (np.abs(x) + ex), 2.0 ** -10 * s) + ex
        if positive:
            assert np.all((y > 0) | (x - ex <= 0)), what + ": a value above zero became zero"
            bound = np.maximum(bound, np.where(x < 2.0 ** -9 * s, 2.0 ** -9 * s, 0))
        assert_near(y, x, bound, what)


def assert_near(got, want, bound, what):
    off = np.abs(got - want)
    bad = ~(off <= bound)
    if np.any(bad):
        i = int(np.flatnonzero(bad)[0])
        b = np.broadcast_to(bound, off.shape)
        raise AssertionError("%s: %d of %d values are off; first at %d: got %r want %r, off %.3g, bound %.3g" % (
            what, int(bad.sum()), off.size, i, got[i], want[i], off[i], b[i]))


def ok(st):
    assert (st[0] if isinstance(st, tuple) else st) == Status.OK, st


def adamw(problem, args):
    ok(mc.xccl_mem_component_adamw(problem.plan.handle, args, MemType.ROCM))


def grad_norm(problem):
    ok(mc.xccl_mem_component_grad_norm(problem.plan.handle, problem.stats, MemType.ROCM))
