"""The operators over a model's columns (normalisation, routing, distillation, the 8-bit product) against plain ones in 64
bits, through the C ABI.

Tolerances are derived: every fp32 operation is off by at most 2^-24 of its result, a sum of n terms by at most its depth
in additions times 2^-24 of the sum of magnitudes, a final rounding by half a step of the output's type
(columns_ref.HALF_STEP). The depths below count the additions one value passes through in the kernels, rounded up.
"""
import ctypes as C
import threading

import numpy as np
import pytest

import columns_ref as ref
from bidmat_amd import hip_abi
from bidmat_amd.device import DeviceArray
from columns_ref import EPS24, HALF_STEP, TINY, TYPES, decode, encode, np_type

pytestmark = pytest.mark.gpu
F = np.float32


class Columns:
    """A dense operand on the device: rows of `a` are its columns, `pad` unused elements between them, `shift` elements in
    front, all filled with a pattern that must survive."""

    def __init__(self, a, pad=0, shift=0):
        self.m, self.n = a.shape
        self.ld, self.shift = self.n + pad, shift
        self.host = np.full(shift + self.m * self.ld, 77, dtype=a.dtype)
        self.view(self.host)[:, :self.n] = a
        self.dev = DeviceArray.from_numpy(self.host)
        self.ptr = self.dev.ptr + shift * a.dtype.itemsize

    def view(self, flat):
        return flat[self.shift:self.shift + self.m * self.ld].reshape(self.m, self.ld)

    def get(self):
        """The operand's values; what lies between and in front of them has to be as it was."""
        now = self.dev.numpy()
        assert np.array_equal(now[:self.shift], self.host[:self.shift])
        assert np.array_equal(self.view(now)[:, self.n:], self.view(self.host)[:, self.n:])
        return self.view(now)[:, :self.n].copy()


def empty(m, n, dtype, pad=0, shift=0):
    return Columns(np.full((m, n), 55, dtype=dtype), pad, shift)


def ok(code):
    hip_abi.check(code)


def dev(a):
    return DeviceArray.from_numpy(a)


def ptr(d):
    return None if d is None else d.ptr


def within(got, want, bound, what):
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want) - bound
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    bad = ~(same | (off <= 0))
    assert not bad.any(), "%s: %d of %d values outside, first at %s: %r, want %r +- %r" % (
        what, bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0], np.broadcast_to(bound, bad.shape)[bad][0])


# ---------------------------------------------------------------- normalisation
# depth: 8 * 4 additions in a thread, 6 in a wave, 16 over waves; half of it survives the root; 12 for the other steps
NORM_DEPTH = 40


def norm_case(hip, rng, n, m, t, res, want_h, want_y, group, pad=0, shift=0, x=None, eps=1e-5, stream=None):
    x = rng.standard_normal((m, n)) * 2 if x is None else x
    X = encode(x, t)
    R = encode(rng.standard_normal((m, n)), t) if res else None
    w = (1 + 0.1 * rng.standard_normal(n)).astype(F)
    dX, dR, dw = Columns(X, pad, shift), Columns(R, pad, shift) if res else None, dev(w)
    H = empty(m, n, np_type(t), pad, shift) if want_h else None
    Y = empty(m, n, np_type(t), pad + 1, shift) if want_y else None
    Q = empty(m, n, np.uint8, pad, shift) if group is not None else None
    ng = 1 if not group else -(-n // group)
    S = empty(m, ng, np.float32) if group is not None else None
    ld = n + pad
    ok(hip.bidmat_rmsnorm(n, m, t, dX.ptr, ld, ptr(dR), ld, dw.ptr, eps, ptr(H), ld, ptr(Y), ld + 1, ptr(Q), ld, ptr(S), group or 0, stream))
    ok(hip.bidmat_synchronize())
    h, y, s = ref.rmsnorm(decode(X, t), None if R is None else decode(R, t), w.astype(np.float64), float(F(eps)), group)
    if want_h:
        within(decode(H.get(), t), h, (HALF_STEP[t] + EPS24) * np.abs(h) * 1.01 + TINY[t], "h")
    rel = NORM_DEPTH * EPS24
    if want_y:
        within(decode(Y.get(), t), y, (HALF_STEP[t] * 1.01 + rel) * np.abs(y) + TINY[t], "y")
    if group is not None:
        got_s = S.get().astype(np.float64)
        within(got_s, s, (rel + 2 * EPS24) * s, "scales")
        each = np.repeat(got_s, group or n, 1)[:, :n]
        got = ref.E4M3[Q.get()] * each
        within(got, y, np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * each) * 1.001 + 2 * rel * np.abs(y), "codes")
    return dX, H, Y, Q, S


@pytest.mark.parametrize("n", [1, 5, 8, 63, 64, 129, 256, 511, 512, 1000, 1001, 2048, 2049, 4096, 8200, 16384, 32768])
@pytest.mark.parametrize("t", TYPES)
def test_rmsnorm_heights(hip, n, t):
    rng = np.random.default_rng(n * 3 + t)
    for m in (1, 3, 9):
        norm_case(hip, rng, n, m, t, True, True, True, 0)
        norm_case(hip, rng, n, m, t, False, False, True, 32)
    norm_case(hip, rng, n, 5, t, True, False, False, 64)
    norm_case(hip, rng, n, 5, t, True, True, False, 128, pad=3, shift=1)


@pytest.mark.parametrize("t", TYPES)
def test_rmsnorm_many_columns(hip, t):
    rng = np.random.default_rng(t)
    norm_case(hip, rng, 72, 5000, t, True, True, True, 32)
    norm_case(hip, rng, 1024, 2500, t, True, True, False, 128)
    norm_case(hip, rng, 6000, 700, t, True, False, True, 64, pad=5)


def test_rmsnorm_small_and_large_values(hip):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((6, 300))
    x[0] = 0
    x[1] *= 1e-18
    x[2] *= 1e15
    x[3] *= 1e-3
    x[4, 7:] = 0
    for group in (None, 0, 32):
        norm_case(hip, rng, 300, 6, 0, False, True, True, group, x=x, eps=1e-6)


@pytest.mark.parametrize("n", [40, 300, 3000, 9000])
@pytest.mark.parametrize("t", [0, 2])
def test_rmsnorm_squares_beyond_single_precision(hip, n, t):
    rng = np.random.default_rng(n)
    x = rng.standard_normal((5, n))
    x[1] *= 1e21
    x[2, 0] = 3e37
    x[4] *= 1e35
    norm_case(hip, rng, n, 5, t, False, True, True, 32, x=x)
    norm_grad_case(hip, rng, n, 5, t, True, H=x)


def test_rmsnorm_nan_and_infinity_stay_in_their_columns(hip):
    rng = np.random.default_rng(6)
    n = 200
    x = rng.standard_normal((5, n))
    x[1, 7], x[3, 199] = np.nan, np.inf
    for t in TYPES:
        X = encode(x, t)
        d, w = Columns(X), dev(np.ones(n, F))
        Y, Q, S = empty(5, n, np_type(t)), empty(5, n, np.uint8), empty(5, 7, np.float32)
        ok(hip.bidmat_rmsnorm(n, 5, t, d.ptr, n, None, n, w.ptr, 1e-5, None, n, Y.ptr, n, Q.ptr, n, S.ptr, 32, None))
        y, q = decode(Y.get(), t), ref.E4M3[Q.get()]
        assert np.isnan(y[1]).all() and np.isnan(q[1]).all()
        assert np.isnan(y[3, 199]) and np.isnan(q[3, 199])
        for c in (0, 2, 4):
            assert np.isfinite(y[c]).all() and np.isfinite(q[c]).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [96, 1001, 8192])
def test_rmsnorm_in_place(hip, t, n):
    rng = np.random.default_rng(n + t)
    m = 7
    X, R, w = encode(rng.standard_normal((m, n)), t), encode(rng.standard_normal((m, n)), t), dev(np.ones(n, F))
    x, r, H, Y = Columns(X), Columns(R), empty(m, n, np_type(t)), empty(m, n, np_type(t))
    ok(hip.bidmat_rmsnorm(n, m, t, x.ptr, n, r.ptr, n, w.ptr, 1e-5, H.ptr, n, Y.ptr, n, None, n, None, 0, None))
    h, y = H.get(), Y.get()
    ok(hip.bidmat_rmsnorm(n, m, t, x.ptr, n, r.ptr, n, w.ptr, 1e-5, r.ptr, n, x.ptr, n, None, n, None, 0, None))
    assert np.array_equal(r.get(), h) and np.array_equal(x.get(), y)


def norm_grad_case(hip, rng, n, m, t, with_dh, pad=0, shift=0, beta=0, in_place=False, H=None):
    H, dY = encode(rng.standard_normal((m, n)) * 2 if H is None else H, t), encode(rng.standard_normal((m, n)), t)
    dH = encode(rng.standard_normal((m, n)), t) if with_dh else None
    w = (1 + 0.1 * rng.standard_normal(n)).astype(F)
    dw0 = rng.standard_normal(n).astype(F)
    h, dy, dh = Columns(H, pad, shift), Columns(dY, pad, shift), Columns(dH, pad, shift) if with_dh else None
    dx = dy if in_place else empty(m, n, np_type(t), pad, shift)
    dww, d_w, ld = dev(dw0), dev(w), n + pad
    ok(hip.bidmat_rmsnorm_grad(n, m, t, h.ptr, ld, d_w.ptr, 1e-5, dy.ptr, ld, ptr(dh), ld, dx.ptr, ld, dww.ptr, beta, None))
    want, wantw, size, sizew = ref.rmsnorm_grad(decode(H, t), w.astype(np.float64), float(F(1e-5)), decode(dY, t),
                                                None if dH is None else decode(dH, t))
    within(decode(dx.get(), t), want, HALF_STEP[t] * 1.01 * np.abs(want) + TINY[t] + 2 * NORM_DEPTH * EPS24 * size, "dx")
    # columns in a row of one workgroup, 256 / 8 of them over a workgroup, 64 of its 512 shares in a row, 6 halvings
    depth = m / 512 + 32 + 8 + 6 + NORM_DEPTH
    within(dww.numpy().astype(np.float64), wantw + beta * dw0, depth * EPS24 * (sizew + beta * np.abs(dw0)), "dw")
    return dx, dww


@pytest.mark.parametrize("n", [1, 7, 64, 100, 512, 513, 1001, 2048, 4096, 8200, 16384, 32768])
@pytest.mark.parametrize("t", TYPES)
def test_rmsnorm_grad_heights(hip, n, t):
    rng = np.random.default_rng(n * 5 + t)
    norm_grad_case(hip, rng, n, 1, t, False)
    norm_grad_case(hip, rng, n, 37, t, True, beta=1)
    norm_grad_case(hip, rng, n, 6, t, True, pad=3, shift=1)
    norm_grad_case(hip, rng, n, 11, t, False, in_place=True)


@pytest.mark.parametrize("t", TYPES)
def test_rmsnorm_grad_many_columns_same_bits_every_time(hip, t):
    for n, m in ((72, 20000), (1024, 3000), (3000, 1500)):
        a = norm_grad_case(hip, np.random.default_rng(9), n, m, t, True)
        b = norm_grad_case(hip, np.random.default_rng(9), n, m, t, True)
        assert np.array_equal(a[1].numpy(), b[1].numpy()) and np.array_equal(a[0].get(), b[0].get())


def test_rmsnorm_grad_against_differences(hip):
    """The gradient of sum(g * y) along a direction against a central difference of the operator in 64 bits."""
    rng = np.random.default_rng(11)
    n, m, eps = 300, 5, 1e-5
    h, g, w = rng.standard_normal((m, n)).astype(F), rng.standard_normal((m, n)).astype(F), (1 + 0.1 * rng.standard_normal(n)).astype(F)
    dx, dw = empty(m, n, np.float32), dev(np.zeros(n, F))
    a, b, c = Columns(h), Columns(g), dev(w)
    ok(hip.bidmat_rmsnorm_grad(n, m, 0, a.ptr, n, c.ptr, eps, b.ptr, n, None, n, dx.ptr, n, dw.ptr, 0, None))
    dh, dv = rng.standard_normal((m, n)), rng.standard_normal(n)

    def f(s):
        return (ref.rmsnorm(h + s * dh, None, w + s * dv, eps)[1] * g).sum()
    d = 1e-5
    want = (f(d) - f(-d)) / (2 * d)
    got = (dx.get().astype(np.float64) * dh).sum() + (dw.numpy().astype(np.float64) * dv).sum()
    # a central difference is off by d^2 / 6 of the third derivative (of the size of the sum of |terms|)
    size = np.abs(g).sum() * np.abs(dh).max()
    assert abs(got - want) < size * (d * d + 2 * NORM_DEPTH * EPS24 + 2.0 ** -52 / d)


# ---------------------------------------------------------------- routing
def route_case(hip, rng, E, m, t, kind, bias, groups, tg, k, renorm, pad=0, shift=0, Z=None, counts=True, extra=True):
    z = rng.standard_normal((m, E)) * 1.5 if Z is None else Z
    Zt = encode(z, t)
    b = (0.05 * rng.standard_normal(E)).astype(F) if bias is True else bias
    scale = 2.5 if renorm else 1.0
    d, db = Columns(Zt, pad, shift), dev(b) if b is not None else None
    G, ir = empty(m, k, np.float32), empty(m, k, np.int32)
    ic, jc, cnt = dev(np.full(m * k, -1, np.int32)), dev(np.full(m + 1, -1, np.int32)), dev(np.full(E, -1, np.int32))
    ok(hip.bidmat_route(E, m, t, d.ptr, E + pad, ptr(db), kind, groups, tg, k, int(renorm), scale, G.ptr, ir.ptr, ic.ptr if extra else None,
                        jc.ptr if extra else None, cnt.ptr if counts else None, None))
    ok(hip.bidmat_synchronize())
    zd = decode(Zt, t)
    want_ir, want_w, want_counts = ref.route(zd, b, kind, groups, tg, k, renorm, scale)
    assert np.array_equal(ir.get(), want_ir)
    # exp's argument is off by |z - max| * 2^-24; sums pass through at most 32 additions in a lane and 6 over lanes
    fin = np.where(np.isfinite(zd), np.abs(zd), 0).max()
    within(G.get().astype(np.float64), want_w, (2 * fin + 60) * EPS24 * np.abs(want_w) + 2.0 ** -126, "weights")
    if extra:
        assert np.array_equal(ic.numpy(), np.repeat(np.arange(m), k))
        assert np.array_equal(jc.numpy(), np.arange(m + 1) * k)
    if counts:
        assert np.array_equal(cnt.numpy(), want_counts)
    return d, G, ir


@pytest.mark.parametrize("E,groups,tg,k", [(1, 1, 1, 1), (2, 1, 1, 1), (8, 1, 1, 2), (8, 4, 2, 3), (16, 16, 5, 5), (60, 1, 1, 4), (60, 5, 3, 7),
                                           (64, 8, 4, 8), (64, 64, 9, 9), (100, 4, 1, 25), (128, 1, 1, 6), (160, 8, 3, 6), (256, 8, 4, 8),
                                           (256, 1, 1, 64), (257, 1, 1, 9), (384, 3, 2, 16), (512, 8, 8, 10), (1000, 5, 2, 33),
                                           (1020, 51, 7, 8), (1024, 1, 1, 8), (1024, 32, 8, 16)])
@pytest.mark.parametrize("kind", [0, 1])
def test_route_shapes(hip, E, groups, tg, k, kind):
    rng = np.random.default_rng(E * 7 + groups + kind)
    for t in TYPES:
        for bias in (True, None):
            route_case(hip, rng, E, 1, t, kind, bias, groups, tg, k, True)
            route_case(hip, rng, E, 7, t, kind, bias, groups, tg, k, False, pad=3, shift=1)
    route_case(hip, rng, E, 301, 2, kind, True, groups, tg, k, True, counts=False, extra=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("E,groups,tg,k", [(64, 1, 1, 4), (256, 8, 4, 8), (60, 1, 1, 4)])
def test_route_many_columns(hip, E, groups, tg, k, t):
    rng = np.random.default_rng(E + t)
    m = 6000
    route_case(hip, rng, E, m, t, 1, True, groups, tg, k, True)
    route_case(hip, rng, E, m, t, 0, None, groups, tg, k, False)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("bias", [None, "zero", "steps"])
def test_route_ties_go_to_the_lowest_index(hip, kind, bias):
    """Scores of few different values, equal scores, and keys that are equal or next to each other in fp32 only."""
    rng = np.random.default_rng(3 + kind)
    E, m = 96, 400
    b = None if bias is None else np.zeros(E, F) if bias == "zero" else (rng.integers(0, 3, E) * 0.125).astype(F)
    few = rng.integers(-2, 3, (m, E)).astype(np.float64)
    same = np.full((4, E), 0.75)
    # neighbours in fp32 around 1: their sigmoids differ by less than an fp32 step
    close = (1 + rng.integers(0, 4, (m, E)) * 2.0 ** -23).astype(F)
    # far out, where sigmoid and the small softmax values leave no difference in fp32
    far = (rng.integers(0, 5, (m, E)) * 2.0 + 20).astype(F)
    for groups, tg, k in ((1, 1, 5), (8, 3, 7), (4, 2, 1), (1, 1, 60)):
        for z in (few, same, close, far):
            for t in (0, 2):
                route_case(hip, rng, E, len(z), t, kind, b, groups, tg, k, False, Z=z)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_closed_experts_padding_and_nan(hip, kind, renorm):
    rng = np.random.default_rng(8)
    E, m = 64, 40
    z = rng.standard_normal((m, E))
    z[3:6] = -np.inf
    z[7, :62] = -np.inf
    z[8, 2:] = -np.inf
    z[9, ::2] = -np.inf
    z[10, 5] = np.nan
    z[11, 6] = np.inf
    z[12, :] = 200.0
    z[13, :] = -200.0
    z[14, 0] = 1e4
    for groups, tg, k in ((1, 1, 6), (8, 2, 6), (4, 4, 33)):
        for bias in (None, True):
            for t in TYPES:
                if t == 0 or kind == 1 or renorm or True:
                    route_case(hip, rng, E, m, t, kind, bias, groups, tg, k, renorm, Z=z)


@pytest.mark.parametrize("kind", [0, 1])
def test_route_biases_that_are_not_finite(hip, kind):
    rng = np.random.default_rng(33)
    E = 64
    b = (0.05 * rng.standard_normal(E)).astype(F)
    b[[3, 40]], b[17], b[[5, 63]] = -np.inf, np.inf, np.nan
    for groups, tg, k in ((1, 1, 6), (8, 3, 6), (2, 2, 20)):
        for m in (5, 200):
            route_case(hip, rng, E, m, 0, kind, b, groups, tg, k, False)
    b[:] = -np.inf
    route_case(hip, rng, E, 70, 0, kind, b, 1, 1, 6, True)


@pytest.mark.parametrize("E,groups,tg,k", [(16, 4, 2, 5), (48, 16, 3, 7), (256, 16, 16, 16), (250, 10, 4, 16), (240, 3, 1, 16), (17, 1, 1, 16),
                                           (256, 2, 1, 2), (96, 12, 5, 1)])
def test_route_sixteen_lanes(hip, E, groups, tg, k):
    """More shapes of the kernel that takes four columns per wave: few and many groups, every column length, rows of few scores."""
    rng = np.random.default_rng(E + k)
    for t in TYPES:
        for kind in (0, 1):
            for bias in (None, True):
                m = int(rng.integers(65, 300))
                z = rng.standard_normal((m, E)) * 1.5
                z[rng.random((m, E)) < 0.3] = -np.inf
                z[::7] = np.round(z[::7])
                route_case(hip, rng, E, m, t, kind, bias, groups, tg, k, bool(rng.integers(2)), Z=z, pad=int(rng.integers(3)))


# Column counts on both sides of where one workgroup ends and where it takes several columns per wave; tied keys send columns
# to the decision in 64 bits.
@pytest.mark.parametrize("m", [2, 8, 9, 16, 17, 32, 33, 48, 49, 63])
@pytest.mark.parametrize("E,groups,tg,k", [(16, 4, 2, 5), (60, 1, 1, 4), (256, 8, 4, 8), (256, 1, 1, 16), (100, 1, 1, 30), (384, 8, 4, 8),
                                           (1000, 5, 2, 33)])
def test_route_few_columns(hip, E, groups, tg, k, m):
    rng = np.random.default_rng(E + m)
    for t in TYPES:
        route_case(hip, rng, E, m, t, 1, True, groups, tg, k, True)
        route_case(hip, rng, E, m, t, 0, None, groups, tg, k, False, pad=2, shift=1)
        steps = np.round(rng.standard_normal((m, E)) * 2) / 2
        steps[m // 2, :] = -np.inf
        route_case(hip, rng, E, m, t, 1, np.zeros(E, np.float32), groups, tg, k, True, Z=steps)


# Up to 32 experts in a lane: ties (decided in 64 bits), closed columns, biases, every kind of weights.
@pytest.mark.parametrize("E,groups,tg,k", [(272, 1, 1, 5), (300, 4, 3, 16), (384, 8, 4, 8), (512, 16, 5, 16), (512, 1, 1, 1), (511, 7, 2, 9)])
def test_route_up_to_512_experts(hip, E, groups, tg, k):
    rng = np.random.default_rng(E + k)
    m = 260
    for t in TYPES:
        for kind in (0, 1):
            route_case(hip, rng, E, m, t, kind, True, groups, tg, k, True)
            route_case(hip, rng, E, m, t, kind, None, groups, tg, k, False, pad=1, shift=1)
            steps = np.round(rng.standard_normal((m, E)) * 2) / 2
            steps[rng.random((m, E)) < 0.3] = -np.inf
            steps[5] = -np.inf
            steps[6, 3:] = -np.inf
            route_case(hip, rng, E, m, t, kind, None, groups, tg, k, True, Z=steps)
            route_case(hip, rng, E, m, t, kind, np.zeros(E, np.float32), groups, tg, k, True, Z=steps)


# Groups without a bias compare p = softmax or sigmoid in 64 bits, where it saturates (ties go to the lower expert) and where
# scores differ by less than it can show.
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("E,groups,tg,k", [(64, 4, 2, 6), (256, 4, 3, 10), (172, 4, 4, 12), (480, 8, 5, 16)])
def test_route_scores_whose_values_meet(hip, E, groups, tg, k, kind):
    rng = np.random.default_rng(E + kind)
    m = 210
    z = rng.standard_normal((m, E))
    z[::7] = rng.choice([15, 19.5, 20.5, 25, 36, 37, 40, 50, 60, 100], (len(z[::7]), E))
    z[1::7] = -rng.choice([0, 600, 690, 710, 730, 744, 746, 760, 900, 2000], (len(z[1::7]), E))
    z[2::7] = rng.integers(-20, 20, (len(z[2::7]), E)) * 1e-20
    z[3::7] = 1 + rng.integers(-20, 20, (len(z[3::7]), E)) * 2.0 ** -23
    z[4::7] = np.round(z[4::7] * 4) / 4
    z[5::7] = -8 + rng.integers(-20, 20, (len(z[5::7]), E)) * 2.0 ** -6
    for t in TYPES:
        for renorm in (False, True):
            route_case(hip, rng, E, m, t, kind, None, groups, tg, k, renorm, Z=z)


def route_grad_case(hip, rng, E, m, t, kind, k, renorm, pad=0, shift=0, in_place=False, Z=None):
    z = rng.standard_normal((m, E)) * 1.5 if Z is None else Z
    d, G, ir = route_case(hip, rng, E, m, t, kind, True, 1, 1, k, renorm, pad, shift, Z=z)
    scale = 2.5 if renorm else 1.0
    dG = rng.standard_normal((m, k)).astype(F)
    ddG = dev(dG)
    dZ = d if in_place else empty(m, E, np_type(t), pad, shift)
    ok(hip.bidmat_route_grad(E, m, t, d.ptr, E + pad, kind, k, int(renorm), scale, G.ptr, ir.ptr, ddG.ptr, dZ.ptr, E + pad, None))
    zd = decode(encode(z, t), t)
    want, size = ref.route_grad(zd, kind, renorm, scale, G.get(), ir.get(), dG)
    fin = np.where(np.isfinite(zd), np.abs(zd), 0).max()
    within(decode(dZ.get(), t), want, HALF_STEP[t] * 1.01 * np.abs(want) + TINY[t] + (8 * fin + 160) * EPS24 * size, "dz")


@pytest.mark.parametrize("E,k", [(1, 1), (8, 2), (60, 4), (64, 64), (65, 9), (256, 8), (1000, 33), (1024, 8)])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_grad(hip, E, k, kind, renorm):
    rng = np.random.default_rng(E + k + kind)
    for t in TYPES:
        route_grad_case(hip, rng, E, 1, t, kind, k, renorm)
        route_grad_case(hip, rng, E, 9, t, kind, k, renorm, pad=3, shift=1)
        route_grad_case(hip, rng, E, 130, t, kind, k, renorm, in_place=True)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_grad_of_closed_experts_and_padding_is_zero(hip, kind, renorm):
    rng = np.random.default_rng(21)
    z = rng.standard_normal((12, 64))
    z[2] = -np.inf
    z[5, 3:] = -np.inf
    z[7, ::3] = -np.inf
    for t in TYPES:
        route_grad_case(hip, rng, 64, 12, t, kind, 6, renorm, Z=z)


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_grad_against_differences(hip, kind, renorm):
    rng = np.random.default_rng(31)
    E, m, k = 32, 6, 5
    z = (rng.standard_normal((m, E)) * 1.5).astype(F)
    d, G, ir = route_case(hip, rng, E, m, 0, kind, None, 1, 1, k, renorm, Z=z)
    dG = rng.standard_normal((m, k)).astype(F)
    a, dZ = dev(dG), empty(m, E, np.float32)
    scale = 2.5 if renorm else 1.0
    ok(hip.bidmat_route_grad(E, m, 0, d.ptr, E, kind, k, int(renorm), scale, G.ptr, ir.ptr, a.ptr, dZ.ptr, E, None))
    to = rng.standard_normal((m, E))
    step = 1e-6                                              # no choice of experts changes over so short a way
    hi, lo = (ref.route(z + s * to, None, kind, 1, 1, k, renorm, scale) for s in (step, -step))
    assert np.array_equal(hi[0], ir.get()) and np.array_equal(lo[0], ir.get())
    want = ((hi[1] - lo[1]) * dG).sum() / (2 * step)
    got = (dZ.get().astype(np.float64) * to).sum()
    size = (np.abs(dG).max() * scale * np.abs(to).max()) * m * k
    assert abs(got - want) < size * (200 * EPS24 + 2.0 ** -52 / step + step * step)


# ---------------------------------------------------------------- distillation
def teacher(rng, V, lengths, sort=True, repeats=False):
    jc = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    ir = np.concatenate([np.zeros(0, np.int64)] + [np.sort(r) if sort else r for r in (
        rng.integers(0, V, n) if repeats else rng.choice(V, n, replace=False) for n in lengths)]).astype(np.int32)
    return (3 + 2 * rng.standard_normal(ir.size)).astype(F), ir, jc


def distill_case(hip, rng, V, m, t, lengths, tau=1.0, weight=None, pad=0, shift=0, in_place=False, sort=True, repeats=False, Z=None,
                 T=None, ir=None, stream=None):
    Zt = encode(rng.standard_normal((m, V)) * 2 if Z is None else Z, t)
    T0, ir0, jc = teacher(rng, V, lengths, sort, repeats)
    T, ir = T0 if T is None else T, ir0 if ir is None else ir
    nnz, ld = int(jc[-1]), V + pad
    z, dT, dir_, djc = Columns(Zt, pad, shift), dev(T), dev(ir), dev(jc)
    dwt = None if weight is None else dev(weight.astype(F))
    loss, lse, loss2, lse2 = (dev(np.full(m, 9, F)) for _ in range(4))
    dZ2 = empty(m, V, np_type(t), pad, shift)
    base = (V, m, t, z.ptr, ld, nnz, dT.ptr, dir_.ptr, djc.ptr, tau, ptr(dwt))
    ok(hip.bidmat_distill(*base, loss2.ptr, lse2.ptr, None, 0, stream))                        # without the gradient
    ok(hip.bidmat_distill_grad(*base, lse2.ptr, dZ2.ptr, ld, stream))                          # the gradient alone
    dZ = z if in_place else empty(m, V, np_type(t), pad, shift)
    ok(hip.bidmat_distill(*base, loss.ptr, lse.ptr, dZ.ptr, ld, stream))                       # both
    ok(hip.bidmat_synchronize())
    wf = None if weight is None else weight.astype(F).astype(np.float64)
    zd = decode(Zt, t)
    want, wlse, wd, eloss, ez = ref.distill(zd, T, ir, jc, float(F(tau)), wf)
    top = np.where(np.isfinite(zd), np.abs(zd), 0).max(1) / tau
    for a, b in ((loss, lse), (loss2, lse2)):
        within(b.numpy().astype(np.float64), wlse, EPS24 * (8 * (top + np.abs(wlse)) + 160), "lse")
        within(a.numpy().astype(np.float64), want, eloss + 160 * EPS24 * np.abs(want), "loss")
    for d in (dZ, dZ2):
        within(decode(d.get(), t), wd, HALF_STEP[t] * 1.01 * np.abs(wd) + TINY[t] + ez, "dz")
    return loss, lse, dZ


@pytest.mark.parametrize("V", [1, 2, 7, 64, 1000, 2047, 2048, 4099, 20001, 65536, 131072, 131080])
@pytest.mark.parametrize("t", TYPES)
def test_distill_heights(hip, V, t):
    rng = np.random.default_rng(V + t)
    k = min(V, 20)
    distill_case(hip, rng, V, 1, t, [k])
    distill_case(hip, rng, V, 5, t, [k, 0, 1, min(V, 70), k // 2], tau=2.0, weight=rng.random(5), sort=False)
    distill_case(hip, rng, V, 3, t, [k, 1, k], tau=0.5, pad=3, shift=1, in_place=True)


@pytest.mark.parametrize("t", TYPES)
def test_distill_many_columns(hip, t):
    rng = np.random.default_rng(40 + t)
    m = 700
    distill_case(hip, rng, 3001, m, t, rng.integers(0, 40, m), tau=1.5, weight=rng.random(m))
    distill_case(hip, rng, 1024, m, t, rng.integers(0, 300, m), in_place=True, sort=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("V", [50, 5000, 70000])
def test_distill_repeated_rows_add(hip, t, V):
    rng = np.random.default_rng(V)
    distill_case(hip, rng, V, 6, t, [9, 64, 65, 300, 0, 2], repeats=True, sort=True)
    distill_case(hip, rng, V, 6, t, [9, 64, 65, 300, 0, 2], repeats=True, sort=False, in_place=True)


# Many columns too tall for a workgroup's registers: the first part waits in LDS; the tallest are cut into chunks.
@pytest.mark.parametrize("V,t", [(65544, 0), (98304, 0), (98305, 0), (131073, 2), (163840, 1), (163841, 2), (204800, 1), (204801, 2)])
def test_distill_tall_columns(hip, V, t):
    rng = np.random.default_rng(V)
    m = 160
    lengths = rng.integers(0, 30, m)
    distill_case(hip, rng, V, m, t, lengths, tau=1.5, weight=rng.random(m), sort=False, repeats=True, in_place=V % 2 == 0)


def test_distill_long_teacher_columns(hip):
    rng = np.random.default_rng(50)
    distill_case(hip, rng, 9000, 3, 0, [9000, 5000, 3], sort=True)
    distill_case(hip, rng, 9000, 3, 2, [6000, 0, 4500], sort=False, repeats=True, in_place=True)


# Rows in no order, all different or with a single one stored twice, far apart: few entries, and so many that the rows are told
# apart in ranges.
@pytest.mark.parametrize("V,lengths", [(1000, [64, 63, 65, 200]), (40000, [399, 401, 900, 20000]), (140000, [70, 700, 800, 40000])])
@pytest.mark.parametrize("twice", [False, True])
def test_distill_rows_in_no_order(hip, V, lengths, twice):
    rng = np.random.default_rng(V + twice)
    T, ir, jc = teacher(rng, V, lengths, sort=False)
    if twice:
        for a, b in zip(jc[:-1], jc[1:]):
            ir[b - 1] = ir[a]
    T = np.minimum(T, 6)
    for t in (0, 2):
        distill_case(hip, np.random.default_rng(V), V, len(lengths), t, lengths, T=T, ir=ir)
        distill_case(hip, np.random.default_rng(V), V, len(lengths), t, lengths, T=T, ir=ir, in_place=True)


@pytest.mark.parametrize("V", [300, 40000])
def test_distill_masks_and_rows_outside(hip, V):
    """Student logits of -inf, teacher logits of -inf (some, and all of a column), rows outside the matrix, weight 0."""
    rng = np.random.default_rng(60)
    m, k = 8, 12
    z = rng.standard_normal((m, V))
    T, ir, jc = teacher(rng, V, [k] * m)
    z[1, ::2] = -np.inf
    z[1, ir[k:2 * k]] = rng.standard_normal(k)
    z[2, ir[2 * k + 3]] = -np.inf                        # the teacher wants what the student excludes: loss +inf
    T[3 * k:4 * k:2] = -np.inf
    T[4 * k:5 * k] = -np.inf                             # an empty teacher
    ir[5 * k:5 * k + 3] = [V, -1, 2 ** 31 - 1]
    z[6] = np.nan                                        # weight 0: nothing is read into the result
    weight = np.array([1, .5, 1, 1, 1, 2, 0, 1.])
    for t in TYPES:
        for in_place in (False, True):
            loss, _, dZ = distill_case_raw(hip, z, T, ir, jc, t, weight, in_place)
            zd = decode(encode(z, t), t)
            want, _, wd, eloss, ez = ref.distill(zd, T, ir, jc, 1.0, weight)
            assert want[2] == np.inf and want[4] == 0 and want[6] == 0
            within(loss, want, np.where(np.isfinite(eloss), eloss, 0), "loss")
            within(dZ, wd, HALF_STEP[t] * 1.01 * np.abs(wd) + TINY[t] + np.nan_to_num(ez, posinf=0), "dz")


def distill_case_raw(hip, z, T, ir, jc, t, weight, in_place, tau=1.0):
    m, V = z.shape
    a = Columns(encode(z, t))
    dT, di, dj, w = dev(T), dev(ir), dev(jc), dev(weight.astype(F))
    loss, lse = dev(np.zeros(m, F)), dev(np.zeros(m, F))
    dZ = a if in_place else empty(m, V, np_type(t))
    ok(hip.bidmat_distill(V, m, t, a.ptr, V, ir.size, dT.ptr, di.ptr, dj.ptr, tau, w.ptr, loss.ptr, lse.ptr, dZ.ptr, V, None))
    return loss.numpy().astype(np.float64), lse.numpy(), decode(dZ.get(), t)


@pytest.mark.parametrize("V", [100, 9000, 140000])
@pytest.mark.parametrize("t", TYPES)
def test_distill_every_choice_of_outputs(hip, V, t):
    """loss, lse and dZ alone and together, and the gradient alone in place of the logits."""
    rng = np.random.default_rng(V + t)
    m = 6
    T, ir, jc = teacher(rng, V, [5, 0, 80, 1, 64, 65], sort=False)
    z = encode(rng.standard_normal((m, V)), t)
    a, dT, di, dj = Columns(z), dev(T), dev(ir), dev(jc)
    base = (V, m, t, a.ptr, V, ir.size, dT.ptr, di.ptr, dj.ptr, 1.5, None)
    zd = decode(z, t)
    want, wlse, wd, eloss, ez = ref.distill(zd, T, ir, jc, 1.5, None)
    elose = EPS24 * (8 * (np.abs(zd).max(1) + np.abs(wlse)) + 160)
    for with_loss, with_lse, with_dz in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1), (1, 1, 0)):
        loss, lse, dZ = dev(np.full(m, 7, F)), dev(np.full(m, 7, F)), empty(m, V, np_type(t))
        untouched = dZ.get()
        ok(hip.bidmat_distill(*base, loss.ptr if with_loss else None, lse.ptr if with_lse else None, dZ.ptr if with_dz else None, V, None))
        if with_loss:
            within(loss.numpy().astype(np.float64), want, eloss + 160 * EPS24 * np.abs(want), "loss")
        if with_lse:
            within(lse.numpy().astype(np.float64), wlse, elose, "lse")
        if with_dz:
            within(decode(dZ.get(), t), wd, HALF_STEP[t] * 1.01 * np.abs(wd) + TINY[t] + ez, "dz")
        assert with_loss or (loss.numpy() == 7).all()
        assert with_lse or (lse.numpy() == 7).all()
        assert with_dz or np.array_equal(dZ.get(), untouched)
    lse = dev(wlse.astype(F))
    dZ = empty(m, V, np_type(t))
    ok(hip.bidmat_distill_grad(*base, lse.ptr, dZ.ptr, V, None))
    ok(hip.bidmat_distill_grad(*base, lse.ptr, a.ptr, V, None))
    assert np.array_equal(a.get(), dZ.get())


def test_distill_without_entries_at_all(hip):
    for V in (10, 5000):
        a, dZ = Columns(np.full((3, V), np.nan, F)), empty(3, V, np.float32)
        jc, loss = dev(np.zeros(4, np.int32)), dev(np.ones(3, F))
        ok(hip.bidmat_distill(V, 3, 0, a.ptr, V, 0, None, None, jc.ptr, 1.0, None, loss.ptr, None, dZ.ptr, V, None))
        assert not loss.numpy().any() and not dZ.get().any()


def test_distill_large_offsets_cancel(hip):
    """Logits around 1000: the loss is a difference of large numbers that the kernels take before they sum."""
    rng = np.random.default_rng(70)
    distill_case(hip, rng, 3000, 4, 0, [10] * 4, Z=1000 + rng.standard_normal((4, 3000)))


@pytest.mark.parametrize("V", [70, 5000, 140000])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
def test_distill_masks_of_the_lowest_value(hip, V, t, tau):
    """Masked logits hold the type's most negative number: some rows, a column but one row, the teacher's too. A column of
    nothing else has the uniform softmax: its loss and gradient are finite, q is 1 / V."""
    rng = np.random.default_rng(V)
    low = {0: -3.4028234663852886e38, 1: -65504.0, 2: -3.3895313892515355e38}[t]
    m, k = 5, 9
    z = rng.standard_normal((m, V))
    T, ir, jc = teacher(rng, V, [k] * m)
    z[1, rng.choice(V, V // 2, replace=False)] = low
    z[1, ir[k:2 * k]] = 1.0
    z[2] = low
    z[2, ir[2 * k]] = 0.5
    T[2 * k + 1:3 * k] = np.float32(-3.4e38)
    T[3 * k:4 * k - 1] = np.float32(-3.4e38)
    z[4] = low
    T[4 * k:5 * k] = np.float32(-3.4e38)
    for in_place in (False, True):
        loss, lse, dZ = distill_case_raw(hip, z, T, ir, jc, t, np.ones(m), in_place, tau)
        want, _, wd, eloss, ez = ref.distill(decode(encode(z, t), t)[:4], T, ir, jc[:5], tau, np.ones(4))
        within(loss[:4], want, eloss + 160 * EPS24 * np.abs(want), "loss")
        within(dZ[:4], wd, HALF_STEP[t] * 1.01 * np.abs(wd) + TINY[t] + ez, "dz")
        # the uniform column: q = 1 / V, p = 1 / k
        share = np.zeros(V)
        share[ir[4 * k:]] = 1 / k
        u = tau * (1 / V - share)
        within(dZ[4], u, HALF_STEP[t] * 1.01 * np.abs(u) + TINY[t] + 200 * EPS24 * tau * (1 / V + share), "uniform dz")
        assert abs(loss[4] - tau * tau * np.log(V / k)) <= 200 * EPS24 * tau * tau * (np.log(V) + np.log(k) + 1)


def test_distill_against_differences(hip):
    rng = np.random.default_rng(71)
    V, m, tau = 500, 4, 2.0
    z = rng.standard_normal((m, V)).astype(F)
    T, ir, jc = teacher(rng, V, [10, 0, 7, 30])
    weight = rng.random(m).astype(F)
    _, _, dZ = distill_case_raw(hip, z, T, ir, jc, 0, weight, False, tau)
    to = rng.standard_normal((m, V))
    d = 1e-5
    f = [ref.distill(z + s * to, T, ir, jc, tau, weight)[0].sum() for s in (d, -d)]
    want, got = (f[0] - f[1]) / (2 * d), (dZ * to).sum()
    size = np.abs(to).max() * weight.sum() * tau * 2
    assert abs(got - want) < size * (200 * EPS24 + d * d + 2.0 ** -50 * 100 / d)


# ---------------------------------------------------------------- the 8-bit product
def q8_case(hip, rng, k, rows, lengths, group, beta=0, pad=0, shift=0, stream=None):
    m = len(lengths)
    jc = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    ir = rng.integers(0, rows, int(jc[-1])).astype(np.int32)
    S = rng.standard_normal(ir.size).astype(F)
    codes = rng.integers(0, 256, (rows, k)).astype(np.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x30
    ng = 1 if group == 0 else -(-k // group)
    scales = (0.01 + rng.random((rows, ng))).astype(F)
    C0 = rng.standard_normal((m, k)).astype(F)
    q, s, v, i, j, c = Columns(codes, pad, shift), dev(scales), dev(S), dev(ir), dev(jc), Columns(C0)
    ok(hip.bidmat_dsmult_q8_csc(k, m, ir.size, q.ptr, k + pad, s.ptr, group, v.ptr, i.ptr, j.ptr, c.ptr, beta, stream))
    ok(hip.bidmat_synchronize())
    want, size = ref.q8_product(codes, scales, group, S, ir, jc)
    # terms in a row of one wave, its groups, segments; two roundings per term
    depth = min(max(lengths, default=0), 1024) + 8 + max(lengths, default=0) / 1024 + 3
    within(c.get().astype(np.float64), want + beta * C0, depth * EPS24 * (size + beta * np.abs(C0)), "C")
    return c


@pytest.mark.parametrize("k", [1, 7, 16, 17, 33, 64, 100, 128, 256, 257, 512, 1000, 1024, 1040, 2500])
@pytest.mark.parametrize("group", [0, 32, 64, 128])
def test_dsmult_q8_heights(hip, k, group):
    rng = np.random.default_rng(k + group)
    q8_case(hip, rng, k, 50, [0, 1, 5, 64, 65, 0, 200, 2], group)
    q8_case(hip, rng, k, 50, [3, 0, 130], group, beta=1, pad=5, shift=3)
    q8_case(hip, rng, k, 9, [1], group)


# More rows than a wave takes at once, and enough nonzeros for the rest to be a launch of its own.
@pytest.mark.parametrize("k,group", [(1025, 0), (1040, 32), (1280, 128), (1281, 64), (2049, 0), (2304, 32)])
@pytest.mark.parametrize("beta", [0, 1])
def test_dsmult_q8_rows_past_a_wave(hip, k, group, beta):
    rng = np.random.default_rng(k)
    lengths = rng.integers(0, 90, 1500)
    lengths[[3, 700]] = 700
    assert lengths.sum() >= 65536
    q8_case(hip, rng, k, 40, lengths, group, beta=beta, pad=3, shift=1)


def test_dsmult_q8_more_columns_than_a_launch_takes(hip):
    rng = np.random.default_rng(73)
    m, rows, long = (1 << 24) + 777, 50, 3000
    lengths = np.zeros(m, np.int64)
    lengths[rng.integers(0, m, 100000)] = rng.integers(1, 4, 100000)
    lengths[[0, (1 << 24) - 1, 1 << 24, m - 1]] = long             # cut into segments on both sides of the border
    jc = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    ir = rng.integers(0, rows, int(jc[-1])).astype(np.int32)
    S = rng.standard_normal(ir.size).astype(F)
    codes = rng.integers(0, 0x7F, (rows, 1)).astype(np.uint8)
    scales = (0.01 + rng.random((rows, 1))).astype(F)
    q, s, v, i, j = dev(codes.reshape(-1)), dev(scales.reshape(-1)), dev(S), dev(ir), dev(jc)
    C = dev(np.full(m, 7, F))
    ok(hip.bidmat_dsmult_q8_csc(1, m, ir.size, q.ptr, 1, s.ptr, 0, v.ptr, i.ptr, j.ptr, C.ptr, 0, None))
    ok(hip.bidmat_synchronize())
    A, _ = ref.q8_product(codes, scales, 0, np.ones(rows, F), np.arange(rows, dtype=np.int32), np.arange(rows + 1, dtype=np.int32))
    terms = S.astype(np.float64) * A[ir, 0]
    cols = np.repeat(np.arange(m), lengths)
    want, size = np.bincount(cols, terms, m), np.bincount(cols, np.abs(terms), m)
    within(C.numpy().astype(np.float64), want, (long + 14) * EPS24 * size, "C")


@pytest.mark.parametrize("k", [48, 256, 1024])
def test_dsmult_q8_long_columns_and_many(hip, k):
    rng = np.random.default_rng(k)
    q8_case(hip, rng, k, 300, [1024, 1025, 5000, 0, 3, 2048], 32)
    q8_case(hip, rng, k, 300, rng.integers(0, 12, 3000), 0, beta=1)
    q8_case(hip, rng, k, 300, rng.integers(0, 90, 600), 128)


def test_dsmult_q8_short_segments(hip):
    old = hip.bidmat_get_option(b"seglen")
    ok(hip.bidmat_set_option(b"seglen", 64))
    try:
        rng = np.random.default_rng(1)
        a = q8_case(hip, rng, 200, 100, [500, 0, 63, 64, 65, 129, 1000], 64)
        rng = np.random.default_rng(1)
        b = q8_case(hip, rng, 200, 100, [500, 0, 63, 64, 65, 129, 1000], 64)
        assert np.array_equal(a.get(), b.get())
    finally:
        ok(hip.bidmat_set_option(b"seglen", old))


def test_dsmult_q8_of_a_range_of_columns(hip):
    """Columns [3, 8) of a matrix through Sjc + 3 and the whole matrix's arrays, columns among them that are cut."""
    rng = np.random.default_rng(4)
    lengths = [700, 3, 0, 900, 257, 2, 0, 1500, 40, 300]
    k, rows = 80, 60
    jc = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    ir, S = rng.integers(0, rows, int(jc[-1])).astype(np.int32), rng.standard_normal(int(jc[-1])).astype(F)
    codes, scales = rng.integers(0, 0x7F, (rows, k)).astype(np.uint8), (0.01 + rng.random((rows, 1))).astype(F)
    q, s, v, i, j, c = Columns(codes), dev(scales), dev(S), dev(ir), dev(jc), empty(5, k, np.float32)
    ok(hip.bidmat_dsmult_q8_csc(k, 5, int(jc[8] - jc[3]), q.ptr, k, s.ptr, 0, v.ptr, i.ptr, j.ptr + 12, c.ptr, 0, None))
    want, size = ref.q8_product(codes, scales, 0, S, ir, jc[3:9])
    within(c.get().astype(np.float64), want, 300 * EPS24 * size, "C")


def test_dsmult_q8_every_code(hip):
    """All 256 codes through a product with one nonzero of value 1 and scale 1: the decoded values themselves."""
    codes = np.arange(256, dtype=np.uint8)[None]
    q, s, one, z, j, c = Columns(codes), dev(np.ones((1, 1), F)), dev(np.ones(1, F)), dev(np.zeros(1, np.int32)), dev(np.array([0, 1], np.int32)), empty(1, 256, np.float32)
    ok(hip.bidmat_dsmult_q8_csc(256, 1, 1, q.ptr, 256, s.ptr, 0, one.ptr, z.ptr, j.ptr, c.ptr, 0, None))
    got = c.get()[0]
    assert np.array_equal(got, ref.E4M3.astype(F), equal_nan=True)


def test_rmsnorm_codes_round_to_nearest_even(hip):
    """A column whose largest value is 448 times its scale: the codes of given quotients, ties among them."""
    mags = ref.E4M3[:127]
    ties = (mags[:-1] + mags[1:]) / 2
    vals = np.concatenate([mags, ties, np.nextafter(ties.astype(F), F(0)), np.nextafter(ties.astype(F), F(1e9))])
    n = vals.size
    # mean(h^2) of this column is not 1: w undoes the normalisation up to rounding, so compare with what the scale says
    x, w = vals.astype(F)[None], np.full(n, 1.0, F)
    a, dw, Y, Q, S = Columns(x), dev(w), empty(1, n, np.float32), empty(1, n, np.uint8), empty(1, 1, np.float32)
    ok(hip.bidmat_rmsnorm(n, 1, 0, a.ptr, n, None, n, dw.ptr, 0.0, None, n, Y.ptr, n, Q.ptr, n, S.ptr, 0, None))
    y, s, q = Y.get()[0].astype(np.float64), float(S.get()[0, 0]), ref.E4M3[Q.get()[0]]
    want = y / s
    gap = np.abs(q[:, None] - want[:, None])
    nearest = np.abs(mags[None, :] - want[:, None]).min(1)
    assert (gap[:, 0] <= nearest + 4 * EPS24 * want).all()


# ---------------------------------------------------------------- more columns than one launch takes
def test_millions_of_columns(hip):
    rng = np.random.default_rng(95)
    n, m = 3, 4300000
    x = encode(rng.standard_normal((m, n)), 2)
    X, Y, w = dev(x), DeviceArray(n * m, np.uint16), dev(np.ones(n, F))
    ok(hip.bidmat_rmsnorm(n, m, 2, X.ptr, n, None, n, w.ptr, 1e-5, None, n, Y.ptr, n, None, n, None, 0, None))
    _, y, _ = ref.rmsnorm(decode(x, 2), None, np.ones(n), float(F(1e-5)))
    within(decode(Y.numpy().reshape(m, n), 2), y, (HALF_STEP[2] * 1.01 + NORM_DEPTH * EPS24) * np.abs(y) + TINY[2], "y")
    # one teacher entry per column: loss = lse - x at it, dz = q - 1 there
    ir, jc = rng.integers(0, n, m).astype(np.int32), np.arange(m + 1, dtype=np.int32)
    T, di, dj, loss = dev(np.ones(m, F)), dev(ir), dev(jc), DeviceArray(m, F)
    ok(hip.bidmat_distill(n, m, 2, X.ptr, n, m, T.ptr, di.ptr, dj.ptr, 1.0, None, loss.ptr, None, Y.ptr, n, None))
    xd = decode(x, 2)
    q = np.exp(xd) / np.exp(xd).sum(1, keepdims=True)
    within(loss.numpy().astype(np.float64), -np.log(q[np.arange(m), ir]), 200 * EPS24 * (1 + np.abs(xd).max(1)), "loss")
    q[np.arange(m), ir] -= 1
    within(decode(Y.numpy().reshape(m, n), 2), q, HALF_STEP[2] * 1.01 * np.abs(q) + 400 * EPS24, "dz")
    G, ir1, dG = DeviceArray(m, F), DeviceArray(m, np.int32), dev(rng.standard_normal(m).astype(F))
    ok(hip.bidmat_route(n, m, 2, X.ptr, n, None, 0, 1, 1, 1, 0, 1.0, G.ptr, ir1.ptr, None, None, None, None))
    assert np.array_equal(ir1.numpy(), xd.argmax(1))
    ok(hip.bidmat_route_grad(n, m, 2, X.ptr, n, 0, 1, 0, 1.0, G.ptr, ir1.ptr, dG.ptr, Y.ptr, n, None))
    p = np.exp(xd) / np.exp(xd).sum(1, keepdims=True)
    d = dG.numpy().astype(np.float64)[:, None]
    top = xd.argmax(1)[:, None]
    want = p * (np.where(np.arange(n) == top, d, 0) - np.take_along_axis(p, top, 1) * d)
    within(decode(Y.numpy().reshape(m, n), 2), want, HALF_STEP[2] * 1.01 * np.abs(want) + 400 * EPS24 * np.abs(d), "route dz")


# ---------------------------------------------------------------- streams, graphs, threads
def test_a_stream_of_its_own_and_captured_graphs(hip):
    """Every operator recorded once, replayed several times with new data and eager work between the replays: each replay gives
    the bits of the eager call."""
    rng = np.random.default_rng(80)
    n, m, E, k, V = 520, 70, 64, 6, 9000
    s = C.c_void_p()
    ok(hip.bidmat_stream_create(C.byref(s)))
    x, r, h, y, q = (Columns(np.zeros((m, n), t)) for t in (F, F, F, F, np.uint8))
    w, sc, dw = dev(np.ones(n, F)), empty(m, 5, np.float32), dev(np.zeros(n, F))
    z, G, ir, jc, cnt = Columns(np.zeros((m, E), F)), empty(m, k, np.float32), empty(m, k, np.int32), dev(np.zeros(m + 1, np.int32)), dev(np.zeros(E, np.int32))
    dG, dz, dx = Columns(np.zeros((m, k), F)), empty(m, E, np.float32), empty(m, n, np.float32)
    T, tir, tjc = teacher(rng, V, [8] * m)
    dT, dtir, dtjc = dev(T), dev(tir), dev(tjc)
    L, dL, loss, lse, dL2 = Columns(np.zeros((m, V), F)), empty(m, V, np.float32), dev(np.zeros(m, F)), dev(np.zeros(m, F)), empty(m, V, np.float32)
    S, sir, sjc = np.ones(2000, F), rng.integers(0, m, 2000).astype(np.int32), np.array([0, 1500, 1500, 2000], np.int32)
    dS, dsir, dsjc, c = dev(S), dev(sir), dev(sjc), empty(3, n, np.float32)

    def calls():
        ok(hip.bidmat_rmsnorm(n, m, 0, x.ptr, n, r.ptr, n, w.ptr, 1e-5, h.ptr, n, y.ptr, n, q.ptr, n, sc.ptr, 128, s))
        ok(hip.bidmat_rmsnorm_grad(n, m, 0, h.ptr, n, w.ptr, 1e-5, y.ptr, n, r.ptr, n, dx.ptr, n, dw.ptr, 0, s))
        ok(hip.bidmat_route(E, m, 0, z.ptr, E, None, 0, 4, 2, k, 1, 1.0, G.ptr, ir.ptr, None, jc.ptr, cnt.ptr, s))
        ok(hip.bidmat_route_grad(E, m, 0, z.ptr, E, 0, k, 1, 1.0, G.ptr, ir.ptr, dG.ptr, dz.ptr, E, s))
        ok(hip.bidmat_distill(V, m, 0, L.ptr, V, T.size, dT.ptr, dtir.ptr, dtjc.ptr, 2.0, None, loss.ptr, lse.ptr, dL.ptr, V, s))
        ok(hip.bidmat_distill_grad(V, m, 0, L.ptr, V, T.size, dT.ptr, dtir.ptr, dtjc.ptr, 2.0, None, lse.ptr, dL2.ptr, V, s))
        ok(hip.bidmat_dsmult_q8_csc(n, 3, 2000, q.ptr, n, sc.ptr, 128, dS.ptr, dsir.ptr, dsjc.ptr, c.ptr, 0, s))

    outs = (h, y, q, sc, dx, G, ir, dz, dL, dL2, c)
    vecs = (dw, jc, cnt, loss, lse)

    def fill(seed):
        g = np.random.default_rng(seed)
        for a in (x, r, z, dG, L):
            a.dev.upload(g.standard_normal(a.dev.n).astype(F))

    def take():
        ok(hip.bidmat_stream_synchronize(s))
        return [a.get() for a in outs] + [v.numpy() for v in vecs]

    def spoil():
        for a in outs:
            a.dev.upload(np.full(a.dev.n, 3, a.dev.dtype))
        for v in vecs:
            v.upload(np.full(v.n, 3, v.dtype))

    fill(0)
    calls()
    ok(hip.bidmat_stream_synchronize(s))
    graph = C.c_void_p()
    ok(hip.bidmat_graph_begin_capture(s))
    calls()
    ok(hip.bidmat_graph_end_capture(s, C.byref(graph)))
    for seed in range(4):
        fill(seed)
        ok(hip.bidmat_synchronize())
        calls()
        want = take()
        spoil()
        ok(hip.bidmat_synchronize())
        ok(hip.bidmat_graph_launch(graph, s))
        for i, (a, b) in enumerate(zip(take(), want)):
            assert np.array_equal(a, b, equal_nan=True), "replay %d, output %d" % (seed, i)
    ok(hip.bidmat_graph_destroy(graph))
    ok(hip.bidmat_stream_destroy(s))


def test_two_threads_on_streams_of_their_own(hip):
    failed = []

    def work(seed):
        try:
            s = C.c_void_p()
            ok(hip.bidmat_stream_create(C.byref(s)))
            rng = np.random.default_rng(seed)
            for _ in range(3):
                distill_case(hip, rng, 9000 + seed, 12, 0, [30] * 12, stream=s)
                q8_case(hip, rng, 128, 60, [3000, 4, 2000], 32, stream=s)
                norm_case(hip, rng, 900 + seed, 40, 0, True, True, True, 32, stream=s)
            ok(hip.bidmat_stream_destroy(s))
        except BaseException as e:      # noqa: B036 - reported by the main thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]


# ---------------------------------------------------------------- offsets past 32 bits
def _last(dev_ptr, first, count, dtype):
    out = np.empty(count, dtype)
    ok(hip_abi.load().bidmat_memcpy_d2h(out.ctypes.data, dev_ptr + first * out.itemsize, out.nbytes))
    return out


def _tail(dev_ptr, first, a):
    ok(hip_abi.load().bidmat_memcpy_h2d(dev_ptr + first * a.itemsize, np.ascontiguousarray(a).ctypes.data, a.nbytes))


def test_rmsnorm_offsets_past_32_bits(hip):
    rng = np.random.default_rng(90)
    n, m = 32768, 65600                                  # 2.15e9 elements
    X, Y, Q, S, dw = DeviceArray.zeros(n * m, np.uint16), DeviceArray(n * m, np.uint16), DeviceArray(n * m, np.uint8), DeviceArray(m, F), DeviceArray(n, F)
    last = encode(rng.standard_normal((2, n)), 2)
    _tail(X.ptr, n * (m - 2), last)
    w = dev(np.ones(n, F))
    ok(hip.bidmat_rmsnorm(n, m, 2, X.ptr, n, None, n, w.ptr, 1e-5, None, n, Y.ptr, n, Q.ptr, n, S.ptr, 0, None))
    h, y, s = ref.rmsnorm(decode(last, 2), None, np.ones(n), float(F(1e-5)), 0)
    got = decode(_last(Y.ptr, n * (m - 2), 2 * n, np.uint16).reshape(2, n), 2)
    within(got, y, (HALF_STEP[2] * 1.01 + NORM_DEPTH * EPS24) * np.abs(y) + TINY[2], "y")
    q = ref.E4M3[_last(Q.ptr, n * (m - 2), 2 * n, np.uint8).reshape(2, n)] * _last(S.ptr, m - 2, 2, F)[:, None]
    within(q, y, np.maximum(2.0 ** -4 * np.abs(y), 2.0 ** -10 * s) * 1.01, "codes")
    ok(hip.bidmat_rmsnorm_grad(n, m, 2, X.ptr, n, w.ptr, 1e-5, Y.ptr, n, None, n, Y.ptr, n, dw.ptr, 0, None))
    want, wantw, size, sizew = ref.rmsnorm_grad(decode(last, 2), np.ones(n), float(F(1e-5)), got, None)
    within(decode(_last(Y.ptr, n * (m - 2), 2 * n, np.uint16).reshape(2, n), 2), want,
           HALF_STEP[2] * 1.01 * np.abs(want) + TINY[2] + 2 * NORM_DEPTH * EPS24 * size, "dx")
    within(dw.numpy().astype(np.float64), wantw, 400 * EPS24 * sizew, "dw")         # the other columns are zeros


def test_route_and_distill_offsets_past_32_bits(hip):
    rng = np.random.default_rng(91)
    V, m, k = 131072, 16500, 8                           # 2.16e9 elements
    Z, loss = DeviceArray.zeros(V * m, np.uint16), DeviceArray(m, F)
    last = encode(rng.standard_normal((2, V)) * 2, 2)
    _tail(Z.ptr, V * (m - 2), last)
    T, ir, jc = teacher(rng, V, [k, k])
    full_jc = np.concatenate([np.zeros(m - 2, np.int32), jc]).astype(np.int32)
    dT, di, dj = dev(T), dev(ir), dev(full_jc)
    ok(hip.bidmat_distill(V, m, 2, Z.ptr, V, 2 * k, dT.ptr, di.ptr, dj.ptr, 1.0, None, loss.ptr, None, Z.ptr, V, None))
    want, _, wd, eloss, ez = ref.distill(decode(last, 2), T, ir, jc, 1.0, None)
    within(_last(loss.ptr, m - 2, 2, F).astype(np.float64), want, eloss + 160 * EPS24 * np.abs(want), "loss")
    within(decode(_last(Z.ptr, V * (m - 2), 2 * V, np.uint16).reshape(2, V), 2), wd, HALF_STEP[2] * 1.01 * np.abs(wd) + TINY[2] + ez, "dz")
    # the same memory as the scores of 1024 experts
    E, m = 1024, V * m // 1024
    ok(hip.bidmat_memset(Z.ptr, 0, V * 16500 * 2))
    z = encode(rng.standard_normal((3, E)), 2)
    _tail(Z.ptr, E * (m - 3), z)
    G, ir_, cnt = DeviceArray(m * k, F), DeviceArray(m * k, np.int32), DeviceArray(E, np.int32)
    ok(hip.bidmat_route(E, m, 2, Z.ptr, E, None, 0, 1, 1, k, 0, 1.0, G.ptr, ir_.ptr, None, None, cnt.ptr, None))
    wi, ww, _ = ref.route(decode(z, 2), None, 0, 1, 1, k, False, 1.0)
    assert np.array_equal(_last(ir_.ptr, k * (m - 3), 3 * k, np.int32).reshape(3, k), wi)
    within(_last(G.ptr, k * (m - 3), 3 * k, F).astype(np.float64).reshape(3, k), ww, 80 * EPS24 * ww, "weights")
    assert int(cnt.numpy().astype(np.int64).sum()) == m * k and np.array_equal(_last(ir_.ptr, 0, k, np.int32), np.arange(k))
    dG = DeviceArray.zeros(m * k, F)
    d = rng.standard_normal((3, k)).astype(F)
    _tail(dG.ptr, k * (m - 3), d)
    ok(hip.bidmat_route_grad(E, m, 2, Z.ptr, E, 0, k, 0, 1.0, G.ptr, ir_.ptr, dG.ptr, Z.ptr, E, None))
    wd, size = ref.route_grad(decode(z, 2), 0, False, 1.0, ww, wi, d)
    within(decode(_last(Z.ptr, E * (m - 3), 3 * E, np.uint16).reshape(3, E), 2), wd, HALF_STEP[2] * 1.01 * np.abs(wd) + TINY[2] + 200 * EPS24 * size, "dz")


def test_dsmult_q8_offsets_past_32_bits(hip):
    rng = np.random.default_rng(92)
    k, rows = 1024, 2100500                              # 2.15e9 codes
    Q, S = DeviceArray.zeros(k * rows, np.uint8), DeviceArray.zeros(8 * rows, F)
    codes = rng.integers(0, 0x7F, (2, k)).astype(np.uint8)
    sc = (0.01 + rng.random((2, 8))).astype(F)
    _tail(Q.ptr, k * (rows - 2), codes)
    _tail(S.ptr, 8 * (rows - 2), sc)
    v, ir, jc = np.array([2, -1, 3], F), np.array([rows - 1, 0, rows - 2], np.int32), np.array([0, 2, 3], np.int32)
    a, b, c, out = dev(v), dev(ir), dev(jc), empty(2, k, np.float32)
    ok(hip.bidmat_dsmult_q8_csc(k, 2, 3, Q.ptr, k, S.ptr, 128, a.ptr, b.ptr, c.ptr, out.ptr, 0, None))
    A = ref.E4M3[codes] * np.repeat(sc.astype(np.float64), 128, 1)
    want = np.stack([2 * A[1], 3 * A[0]])
    within(out.get().astype(np.float64), want, 4 * EPS24 * np.abs(want), "C")
