"""The operators over a model's columns at the edges of what they accept: sums that leave fp32 on either side, log-sums that
hold few digits, empty matrices, operands that lie between one another, and calls from two threads.

Tolerances are those of test_gpu_columns.py: 2^-24 per fp32 operation, half a step of the output's type for its rounding.
"""
import ctypes as C
import threading

import numpy as np
import pytest

import columns_ref as ref
from bidmat_amd.device import DeviceArray
from bidmat_amd.mats import GMat, GSMat, Mat
from columns_ref import EPS24, HALF_STEP, TINY, TYPES, decode, encode, np_type
from test_gpu_columns import NORM_DEPTH, Columns, dev, empty, norm_case, ok, teacher, within

pytestmark = pytest.mark.gpu
F = np.float32
MOST = {0: 3.4028234663852886e38, 1: 65504.0, 2: 3.3895313892515355e38}      # largest finite value of a type


# ---------------------------------------------------------------- normalisation: sums outside fp32
HEIGHTS = [1, 2, 40, 300, 1001, 4096, 9000, 32768]


@pytest.mark.parametrize("n", HEIGHTS)
@pytest.mark.parametrize("t", [0, 2])
def test_rmsnorm_of_the_largest_values(hip, n, t):
    """Squares whose sum leaves fp32 by up to the largest finite values in every row, and eps that counts beside them."""
    rng = np.random.default_rng(n + t)
    x = rng.standard_normal((6, n))
    x[0] = 1e37
    x[1] = MOST[t] * np.where(np.arange(n) % 2, -1, 1)
    x[2, :2] = MOST[t]
    x[3] = 1e35
    x[4] *= 1e19
    for eps in (0.0, 1e-5, 1e36, 3.4e38):
        for group in (0, 32):
            norm_case(hip, rng, n, 6, t, False, True, True, group, x=x, eps=eps)


def grad_edge(hip, H, dY, w, eps, t, over=None):
    """over: what dX lies on ('h' or 'dy')."""
    m, n = H.shape
    w = w.astype(F)
    H, dY = encode(H, t), encode(dY, t)
    h, dy, dw, dww = Columns(H), Columns(dY), dev(w), dev(np.zeros(n, F))
    dx = h if over == "h" else dy if over == "dy" else empty(m, n, np_type(t))
    ok(hip.bidmat_rmsnorm_grad(n, m, t, h.ptr, n, dw.ptr, eps, dy.ptr, n, None, n, dx.ptr, n, dww.ptr, 0, None))
    want, wantw, size, sizew = ref.rmsnorm_grad(decode(H, t), w.astype(np.float64), float(F(eps)), decode(dY, t), None)
    with np.errstate(over="ignore"):
        fits = np.abs(want) * (1 + 2.0 ** -7) < MOST[t]          # the rest may be rounded to an infinity
    got = decode(dx.get(), t)
    within(np.where(fits, got, 0), np.where(fits, want, 0), HALF_STEP[t] * 1.01 * np.abs(want) + TINY[t] + 2 * NORM_DEPTH * EPS24 * size, "dx")
    within(dww.numpy().astype(np.float64), wantw, (NORM_DEPTH + 48) * EPS24 * sizew + 2.0 ** -149, "dw")


def grad_edges(hip, h, g, w, t, scales):
    """Columns one by one (so that none hides behind another in dw) and together, the result by itself and in place."""
    for eps in scales:
        for c in range(len(h)):
            grad_edge(hip, h[c:c + 1], g[c:c + 1], w, eps, t)
        for over in (None, "h", "dy"):
            grad_edge(hip, h, g, w, eps, t, over)


@pytest.mark.parametrize("n", HEIGHTS + [20000])
@pytest.mark.parametrize("t", [0, 2])
def test_rmsnorm_grad_of_the_largest_values(hip, n, t):
    """Sums of squares and of products that leave fp32, h aligned with the gradient or not."""
    rng = np.random.default_rng(n * 2 + t)
    w = 1 + 0.1 * rng.standard_normal(n)
    sign = np.sign(rng.standard_normal((7, n)))
    h, g = sign * (0.5 + rng.random((7, n))), rng.standard_normal((7, n))
    h[0], g[0] = 1e35, 1
    h[1], g[1] = MOST[t] * sign[1], sign[1]
    h[2, n // 2], g[2, n // 2] = 2e38, 2
    h[3] = 1e37
    h[4], g[4] = 1e3, 1e36
    h[5] *= 1e19
    grad_edges(hip, h, g, w, t, (0.0, 1e-5, 1e36))


@pytest.mark.parametrize("n", HEIGHTS)
@pytest.mark.parametrize("t", [0, 2])
def test_rmsnorm_of_the_smallest_values(hip, n, t):
    """Squares that fp32 holds with few digits or as 0, without an eps that would hide it and with one of their size."""
    rng = np.random.default_rng(n + t)
    x = np.sign(rng.standard_normal((8, n))) * (0.5 + rng.random((8, n)))
    x *= np.array([1, 1e-18, 1e-19, 3e-22, 1e-23, 1e-30, 1e-37, 1e-40])[:, None]
    x[3, 0] = 1e-19
    for eps in (0.0, 1e-45, 1e-43, 1e-38):
        for group in (0, 32):
            norm_case(hip, rng, n, 8, t, False, True, True, group, x=x, eps=eps)


@pytest.mark.parametrize("n", HEIGHTS + [20000])
@pytest.mark.parametrize("t", [0, 2])
def test_rmsnorm_grad_of_the_smallest_values(hip, n, t):
    """Squares and products that fp32 holds with few digits or as 0."""
    rng = np.random.default_rng(n * 2 + t)
    w = 1 + 0.1 * rng.standard_normal(n)
    sign = np.sign(rng.standard_normal((6, n)))
    h, g = sign * (0.5 + rng.random((6, n))), rng.standard_normal((6, n))
    h[0] *= 1e-23
    h[1] *= 3e-22
    h[2], g[2] = 1e-18 * h[2], 1e-27 * sign[2]
    h[3], g[3] = 1e-41 if t == 0 else 1e-39, 1e-4          # below the normal numbers
    h[4] *= 1e-19
    grad_edges(hip, h, g, w, t, (0.0, 1e-45, 1e-38, 1e-5))


@pytest.mark.parametrize("t", [0, 2])
@pytest.mark.parametrize("n,m", [(3, 8500000), (70, 40000), (1001, 5000), (3000, 2500), (9000, 700)])
def test_rmsnorm_grad_of_columns_out_of_range_among_many(hip, t, n, m):
    """Columns of many magnitudes, some of which leave fp32 and some of the gradients' products, in every workgroup (and in more
    columns than one launch takes)."""
    rng = np.random.default_rng(n)
    w = 1 + 0.1 * rng.standard_normal(n)
    h = rng.standard_normal((m, n)).astype(F)
    g = rng.standard_normal((m, n)).astype(F)
    odd = rng.random(m) < 0.1
    h[odd] *= (10.0 ** rng.choice([-30, -25, -21, -12, 19, 25, 35], odd.sum())).astype(F)[:, None]
    g[rng.random(m) < 0.02] *= F(1e-25)
    for over in (None, "h", "dy"):
        grad_edge(hip, h, g, w, 0.0, t, over)


# ---------------------------------------------------------------- distillation: the gradient from a kept log-sum
@pytest.mark.parametrize("V", [70, 1000, 5000, 140000])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
def test_distill_grad_of_large_logits(hip, V, t, tau):
    """Common offsets and masks of the type's lowest value: q = exp(x - lse) for the lse that is given, never above 1. A column
    of masks alone has an lse without the digits of log V: its q are 0 or 1, not infinite."""
    rng = np.random.default_rng(V)
    m, k = 6, 9
    z = rng.standard_normal((m, V))
    T, ir, jc = teacher(rng, V, [k] * m)
    z[0] += 1000
    z[1] = -MOST[t]
    z[2] = -MOST[t]
    z[2, ir[2 * k]] = 0.5
    z[3, rng.choice(V, V // 2, replace=False)] = -MOST[t]
    z[4] = 30000 + 8 * z[4]
    a = Columns(encode(z, t))
    dT, di, dj, loss, lse = dev(T), dev(ir), dev(jc), dev(np.zeros(m, F)), dev(np.zeros(m, F))
    dZ = empty(m, V, np_type(t))
    base = (V, m, t, a.ptr, V, ir.size, dT.ptr, di.ptr, dj.ptr, tau, None)
    ok(hip.bidmat_distill(*base, loss.ptr, lse.ptr, None, V, None))
    ok(hip.bidmat_distill_grad(*base, lse.ptr, dZ.ptr, V, None))
    ok(hip.bidmat_distill_grad(*base, lse.ptr, a.ptr, V, None))
    zd, l = decode(encode(z, t), t), lse.numpy().astype(np.float64)
    # products of 24-bit numbers are exact in 64 bits, and so is the difference up to its own rounding
    x = np.minimum((zd - l[:, None] * tau) / tau, 0)
    q = np.exp(x)
    p, share, ptot = np.zeros((m, V)), np.zeros((m, V)), np.zeros((m, 1))
    for c in range(m):
        s = T[jc[c]:jc[c + 1]].astype(np.float64) / tau
        e = np.exp(s - s.max())
        p[c, ir[jc[c]:jc[c + 1]]] = e / e.sum()
        ptot[c] = np.abs(s).max() + abs(s.max() + np.log(e.sum()))
    want = tau * (q - p)
    with np.errstate(invalid="ignore"):
        eq = np.where(q > 0, q * (8 * np.abs(x) + 20), 0)
    # the exponential is 0 below 2^-126, and is taken of q or of weight * tau * q: off by less than max(tau, 1) * 2^-126 in dz
    bound = HALF_STEP[t] * 1.01 * np.abs(want) + TINY[t] + max(tau, 1) * 2.0 ** -126 + tau * (EPS24 * (eq + p * (8 * ptot + 160 + k)))
    for d in (dZ, a):
        within(decode(d.get(), t), want, bound, "dz")


@pytest.mark.parametrize("m", [1, 5, 70000])
def test_distill_without_rows(hip, m):
    """A matrix of no rows: every column's loss is 0 and its log-sum that of nothing, -inf."""
    jc = dev(np.zeros(m + 1, np.int32))
    loss, lse = dev(np.full(m + 1, 7, F)), dev(np.full(m + 1, 7, F))
    ok(hip.bidmat_distill(0, m, 0, None, 0, 0, None, None, jc.ptr, 1.0, None, loss.ptr, lse.ptr, None, 0, None))
    assert (loss.numpy()[:m] == 0).all() and (lse.numpy()[:m] == -np.inf).all() and loss.numpy()[m] == 7 and lse.numpy()[m] == 7
    lse.upload(np.full(m + 1, 7, F))
    ok(hip.bidmat_distill(0, m, 0, None, 0, 0, None, None, jc.ptr, 1.0, None, loss.ptr, None, None, 0, None))
    assert (lse.numpy() == 7).all()
    ok(hip.bidmat_distill_grad(0, m, 0, None, 0, 0, None, None, jc.ptr, 1.0, None, lse.ptr, loss.ptr, 0, None))
    assert (lse.numpy() == 7).all() and (loss.numpy()[:m] == 0).all()
    # through the matrix interface, into a vector that held something else
    base = int(Mat.get("ioneBased"))
    nothing = GSMat.from_csc(0, m, np.zeros(0, F), np.zeros(0, np.int32), np.full(m + 1, base, np.int32))
    out = GMat.from_numpy(np.full((1, m), 5, F))
    assert (GMat.zeros(0, m).distill(nothing, out=out).numpy() == 0).all()


# ---------------------------------------------------------------- the matrix interface
def gate_of(data, ir, jc, rows):
    base = int(Mat.get("ioneBased"))
    return GSMat.from_csc(rows, len(jc) - 1, np.asarray(data, F), np.asarray(ir, np.int32) + base, np.asarray(jc, np.int32) + base)


def test_route_grad_wants_a_gate(hip):
    """routeGrad takes what route returned, or a matrix that has such a pattern, and values of that very pattern."""
    rng = np.random.default_rng(4)
    E, m, k = 12, 6, 2
    z = GMat.from_numpy(rng.standard_normal((E, m)).astype(F))
    gate = z.route(k)
    data, ir, jc = gate.to_csc()
    base = int(Mat.get("ioneBased"))
    ir, jc = ir.reshape(-1) - base, jc - base
    values = GMat.from_numpy(rng.standard_normal((1, m * k)).astype(F))
    dgate = gate.with_values(values)
    want = z.routeGrad(gate, dgate).numpy()
    # the same pattern from the host, shared or not
    same = gate_of(data, ir, jc, E)
    for a, b in ((same, same.with_values(values)), (same, dgate), (gate, same.with_values(values))):
        assert np.array_equal(z.routeGrad(a, b).numpy(), want)
    other = ir.copy()
    other[:2] = [r for r in range(E) if r not in ir[:2]][:2]
    twice = ir.copy()
    twice[1] = twice[0]
    uneven = jc.copy()
    uneven[1] += 1                                       # columns of 3 and 1
    for a, b in ((gate, gate_of(data, other, jc, E)), (gate_of(data, twice, jc, E),) * 2, (gate_of(data, ir, uneven, E),) * 2,
                 (gate, gate_of(data, ir, uneven, E))):
        with pytest.raises(RuntimeError):
            z.routeGrad(a, b)
    # a matrix whose indices are written again is looked at again
    reused = gate.with_values(values)
    gate2 = GMat.from_numpy(rng.standard_normal((E, m)).astype(F)).route(k, out=gate)
    with pytest.raises(RuntimeError):
        z.routeGrad(gate2, reused)



def test_a_refused_route_leaves_its_output_alone(hip):
    rng = np.random.default_rng(5)
    E, m = 12, 6
    z = GMat.from_numpy(rng.standard_normal((E, m)).astype(F))
    gate = z.route(4)
    before = [a.copy() for a in gate.to_csc()]
    for bad in (dict(topk=2, ngroups=5), dict(topk=3, scale=0.0), dict(topk=2, ngroups=3, topgroups=4), dict(topk=13)):
        with pytest.raises(RuntimeError):
            z.route(**bad, out=gate)
        assert all(np.array_equal(a, b) for a, b in zip(gate.to_csc(), before))


# ---------------------------------------------------------------- the 8-bit product
def put(d, first, a):
    ok(d.lib.bidmat_memcpy_h2d(d.ptr + first * d.dtype.itemsize, np.ascontiguousarray(a, d.dtype).ctypes.data, a.size * d.dtype.itemsize))


def test_dsmult_q8_with_almost_2_to_the_31_nonzeros(hip):
    """As many nonzeros as an int counts, zeros but for the first and the last ones."""
    rng = np.random.default_rng(8)
    k, rows, m, nnz, some = 4, 50, 65536, 2 ** 31 - 1, 1000
    jc = np.minimum(np.arange(m + 1, dtype=np.int64) * (nnz // m + 1), nnz).astype(np.int32)
    assert jc[-1] == nnz and (np.diff(jc) > 0).all()
    codes, scales = rng.integers(0, 0x7F, (rows, k)).astype(np.uint8), (0.01 + rng.random((rows, 1))).astype(F)
    ir, v = DeviceArray.zeros(nnz, np.int32), DeviceArray.zeros(nnz, F)
    want, size = np.zeros((m, k)), np.zeros((m, k))
    for first, col in ((0, 0), (nnz - some, m - 1)):
        r, x = rng.integers(0, rows, some).astype(np.int32), rng.standard_normal(some).astype(F)
        put(ir, first, r)
        put(v, first, x)
        a, b = ref.q8_product(codes, scales, 0, x, r, np.array([0, some], np.int32))
        want[col], size[col] = a[0], b[0]
    q, s, j, c = Columns(codes), dev(scales), dev(jc), empty(m, k, F)
    ok(hip.bidmat_dsmult_q8_csc(k, m, nnz, q.ptr, k, s.ptr, 0, v.ptr, ir.ptr, j.ptr, c.ptr, 0, None))
    within(c.get().astype(np.float64), want, 1100 * EPS24 * size, "C")


def test_dsmult_q8_scratch_is_bounded(hip):
    """Partial sums take 256 MiB and the growth of a scratch buffer at most, however many nonzeros there are."""
    rng = np.random.default_rng(6)
    k, rows, m, each = 2048, 300, 50000, 320
    lengths = np.full(m, each)
    lengths[[7, m - 1]] = 5000
    jc = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    nnz = int(jc[-1])                                    # at 128 nonzeros a partial sum these were 1.0 GB
    ir, S = rng.integers(0, rows, nnz).astype(np.int32), rng.standard_normal(nnz).astype(F)
    codes, scales = rng.integers(0, 0x7F, (rows, k)).astype(np.uint8), (0.01 + rng.random((rows, 1))).astype(F)
    q, s, v, i, j, c = Columns(codes), dev(scales), dev(S), dev(ir), dev(jc), DeviceArray(m * k, F)
    st, free, total = C.c_void_p(), C.c_longlong(), C.c_longlong()
    ok(hip.bidmat_stream_create(C.byref(st)))
    ok(hip.bidmat_mem_info(C.byref(free), C.byref(total)))
    before = free.value
    ok(hip.bidmat_dsmult_q8_csc(k, m, nnz, q.ptr, k, s.ptr, 0, v.ptr, i.ptr, j.ptr, c.ptr, 0, st))
    ok(hip.bidmat_stream_synchronize(st))
    ok(hip.bidmat_mem_info(C.byref(free), C.byref(total)))
    assert before - free.value <= 1.2 * 2 ** 28 + 2 ** 25
    ok(hip.bidmat_stream_destroy(st))
    got = c.numpy().reshape(m, k)
    for col in (0, 7, 8, 12345, m - 2, m - 1):
        a, b = jc[col], jc[col + 1]
        want, size = ref.q8_product(codes, scales, 0, S[a:b], ir[a:b], np.array([0, b - a], np.int32))
        within(got[col].astype(np.float64), want[0], 1100 * EPS24 * size[0], "C")


# ---------------------------------------------------------------- routing
@pytest.mark.parametrize("E,k", [(64, 6), (1000, 20)])
@pytest.mark.parametrize("m", [3, 100])
@pytest.mark.parametrize("scale", [1e30, 2.5, -1e-30])
def test_route_renormalised_with_a_large_scale(hip, E, k, m, scale):
    """Sigmoids whose sum is small: scale over that sum leaves fp32 where the weights do not."""
    rng = np.random.default_rng(E)
    z = encode(-28 + 0.5 * rng.standard_normal((m, E)), 0)
    a, G, ir = Columns(z), empty(m, k, F), empty(m, k, np.int32)
    ok(hip.bidmat_route(E, m, 0, a.ptr, E, None, 1, 1, 1, k, 1, scale, G.ptr, ir.ptr, None, None, None, None))
    wi, ww, _ = ref.route(decode(z, 0), None, 1, 1, 1, k, True, float(F(scale)))
    assert np.array_equal(ir.get(), wi)
    within(G.get().astype(np.float64), ww, (2 * 30 + 60) * EPS24 * np.abs(ww), "weights")


# ---------------------------------------------------------------- operands that lie between one another
def test_row_slices_of_one_matrix(hip):
    """Operands that are different rows of one matrix (one leading dimension, no element in common) are no overlap."""
    rng = np.random.default_rng(3)
    n, m, gap = 100, 40, 7
    ld = 2 * n + gap
    both = np.full((m, ld), 5, F)
    both[:, :n] = rng.standard_normal((m, n))
    a, w = dev(both), dev(np.ones(n, F))
    ok(hip.bidmat_rmsnorm(n, m, 0, a.ptr, ld, None, n, w.ptr, 1e-5, None, n, a.ptr + 4 * n, ld, None, n, None, 0, None))
    got = a.numpy().reshape(m, ld)
    _, y, _ = ref.rmsnorm(both[:, :n].astype(np.float64), None, np.ones(n), float(F(1e-5)))
    assert np.array_equal(got[:, :n], both[:, :n]) and (got[:, 2 * n:] == 5).all()
    within(got[:, n:2 * n], y, (NORM_DEPTH + 1) * EPS24 * np.abs(y), "y")
    # a row in common, other leading dimensions, a vector in between
    for args in ((a.ptr + 4 * (n - 1), ld), (a.ptr + 4 * (ld - n + 1), ld), (a.ptr + 4 * n, ld - 1)):
        assert hip.bidmat_rmsnorm(n, m, 0, a.ptr, ld, None, n, w.ptr, 1e-5, None, n, *args, None, n, None, 0, None) == 1
    assert hip.bidmat_rmsnorm(n, m, 0, a.ptr, ld, None, n, a.ptr + 4 * n, 1e-5, None, n, a.ptr + 4 * n, ld, None, n, None, 0, None) == 1


# ---------------------------------------------------------------- what the other tests leave open
def test_rmsnorm_codes_at_exact_ties(hip):
    """h = +-1 makes rs 1, and a largest weight of 448 makes the scale 1: the codes are those of the weights themselves. Quotients
    half way between two codes go to the even one."""
    mags = ref.E4M3[:127]
    ties = (mags[:-1] + mags[1:]) / 2
    vals = np.concatenate([mags, ties, np.nextafter(ties.astype(F), F(0)), np.nextafter(ties.astype(F), F(1e9))]).astype(F)
    want = np.concatenate([np.arange(127), [i + (i & 1) for i in range(126)], np.arange(126), np.arange(1, 127)])
    for group in (0, 32, 128):
        # a 448 at the head of every 32 rows
        w = np.concatenate([np.full((-(-vals.size // 31), 1), 448, F), np.pad(vals, (0, -vals.size % 31)).reshape(-1, 31)], 1).reshape(-1)
        code = np.concatenate([np.full((-(-vals.size // 31), 1), 126), np.pad(want, (0, -vals.size % 31)).reshape(-1, 31)], 1).reshape(-1)
        n = w.size
        x = np.where(np.arange(n) % 3, -1, 1).astype(F)[None]
        a, dw, Q, S = Columns(x), dev(w), empty(1, n, np.uint8), empty(1, -(-n // (group or n)), F)
        ok(hip.bidmat_rmsnorm(n, 1, 0, a.ptr, n, None, n, dw.ptr, 0.0, None, n, None, n, Q.ptr, n, S.ptr, group, None))
        assert (S.get() == 1).all()
        got = Q.get()[0]
        assert np.array_equal(got & 0x7F, code) and np.array_equal(got >> 7, x[0] < 0)


@pytest.mark.parametrize("n", [40, 200, 3000, 9000])
@pytest.mark.parametrize("t", TYPES)
def test_rmsnorm_of_an_infinity_is_zero_elsewhere(hip, n, t):
    rng = np.random.default_rng(n)
    x = rng.standard_normal((3, n))
    x[1, n // 3], x[2, n - 1] = np.inf, -np.inf
    a, w = Columns(encode(x, t)), dev(np.ones(n, F))
    Y, Q, S = empty(3, n, np_type(t)), empty(3, n, np.uint8), empty(3, -(-n // 32), F)
    ok(hip.bidmat_rmsnorm(n, 3, t, a.ptr, n, None, n, w.ptr, 1e-5, None, n, Y.ptr, n, Q.ptr, n, S.ptr, 32, None))
    for out in (decode(Y.get(), t), ref.E4M3[Q.get()]):
        assert np.isfinite(out[0]).all()
        for c in (1, 2):
            assert np.array_equal(np.isnan(out[c]), np.isinf(x[c])) and (out[c][~np.isinf(x[c])] == 0).all()


def test_a_teacher_of_a_range_of_columns(hip):
    """Tjc + 3 with the whole teacher's arrays and number of values."""
    rng = np.random.default_rng(12)
    for V in (300, 20000, 140000):
        T, ir, jc = teacher(rng, V, [5, 0, 70, 9, 0, 130, 3])
        z = rng.standard_normal((3, V)).astype(F)
        a, dT, di, dj, loss, lse = Columns(z), dev(T), dev(ir), dev(jc), dev(np.zeros(3, F)), dev(np.zeros(3, F))
        dZ, dZ2 = empty(3, V, F), empty(3, V, F)
        base = (V, 3, 0, a.ptr, V, ir.size, dT.ptr, di.ptr, dj.ptr + 12, 1.0, None)
        ok(hip.bidmat_distill(*base, loss.ptr, lse.ptr, dZ.ptr, V, None))
        ok(hip.bidmat_distill_grad(*base, lse.ptr, dZ2.ptr, V, None))
        want, _, wd, eloss, ez = ref.distill(z.astype(np.float64), T, ir, jc[3:7], 1.0, None)
        within(loss.numpy().astype(np.float64), want, eloss + 160 * EPS24 * np.abs(want), "loss")
        for d in (dZ, dZ2):
            within(d.get().astype(np.float64), wd, HALF_STEP[0] * 1.01 * np.abs(wd) + ez, "dz")


def test_routing_and_weight_gradients_from_two_threads(hip):
    """Both keep scratch per stream: threads on streams of their own get the bits of a call by itself."""
    E, k, n, m = 60, 4, 300, 5000
    g = np.random.default_rng(14)
    data = [[g.standard_normal((m, s)).astype(F) for s in (E, n, n)] for _ in range(2)]
    failed = []

    def calls(which, stream, times):
        z, h, dy = (Columns(a) for a in data[which])
        w = dev(np.ones(n, F))
        outs = []
        for _ in range(times):
            G, ir, cnt, dx, dw = empty(m, k, F), empty(m, k, np.int32), dev(np.full(E, -1, np.int32)), empty(m, n, F), dev(np.full(n, 3, F))
            ok(hip.bidmat_route(E, m, 0, z.ptr, E, None, 0, 1, 1, k, 0, 1.0, G.ptr, ir.ptr, None, None, cnt.ptr, stream))
            ok(hip.bidmat_rmsnorm_grad(n, m, 0, h.ptr, n, w.ptr, 1e-5, dy.ptr, n, None, n, dx.ptr, n, dw.ptr, 0, stream))
            ok(hip.bidmat_stream_synchronize(stream))
            outs.append([G.get(), ir.get(), cnt.numpy(), dx.get(), dw.numpy()])
        return outs

    alone = [calls(i, None, 1)[0] for i in range(2)]

    def work(which):
        try:
            s = C.c_void_p()
            ok(hip.bidmat_stream_create(C.byref(s)))
            for out in calls(which, s, 5):
                for a, b in zip(out, alone[which]):
                    assert np.array_equal(a, b)
            ok(hip.bidmat_stream_destroy(s))
        except BaseException as e:      # noqa: B036 - reported by the main thread
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed[0]


@pytest.mark.parametrize("n,m", [(40, 9), (40, 5000), (600, 3000), (1001, 3), (5000, 700), (20000, 300)])
@pytest.mark.parametrize("over", [None, "dh", "h", "dy"])
def test_rmsnorm_grad_of_columns_out_of_range_with_every_operand(hip, n, m, over):
    """dH given, dw added to or absent, dX by itself or on any of the inputs, with unused rows between columns."""
    rng = np.random.default_rng(n + m)
    odd = rng.random(m) < 0.3
    odd[:2] = True, False
    H, dY, dH = (rng.standard_normal((m, n)).astype(F) for _ in range(3))
    H[odd] *= (10.0 ** rng.choice([-30, -24, 25, 36], odd.sum())).astype(F)[:, None]
    w, dw0 = (1 + 0.1 * rng.standard_normal(n)).astype(F), rng.standard_normal(n).astype(F)
    dh64 = dH.astype(np.float64)
    want, wantw, size, sizew = ref.rmsnorm_grad(H.astype(np.float64), w.astype(np.float64), 0.0, dY.astype(np.float64), dh64)
    for beta, with_dw in ((0, True), (1, True), (0, False)):
        h, dy, dh, d_w, dw = Columns(H, 3, 1), Columns(dY, 3, 1), Columns(dH, 3, 1), dev(w), dev(dw0)
        dx = {"h": h, "dy": dy, "dh": dh, None: None}[over] or empty(m, n, F, 3, 1)
        ok(hip.bidmat_rmsnorm_grad(n, m, 0, h.ptr, n + 3, d_w.ptr, 0.0, dy.ptr, n + 3, dh.ptr, n + 3, dx.ptr, n + 3, dw.ptr if with_dw else None,
                                   beta, None))
        fits = np.abs(want) < MOST[0]
        within(np.where(fits, dx.get(), 0).astype(np.float64), np.where(fits, want, 0),
               HALF_STEP[0] * 1.01 * np.abs(want) + TINY[0] + 2 * NORM_DEPTH * EPS24 * size, "dx")
        if with_dw:
            within(dw.numpy().astype(np.float64), wantw + beta * dw0, (NORM_DEPTH + 48 + m / 512) * EPS24 * (sizew + np.abs(dw0)), "dw")
        else:
            assert np.array_equal(dw.numpy(), dw0)


@pytest.mark.parametrize("E,groups,k,m", [(64, 1, 12, 5), (64, 1, 12, 300), (256, 4, 16, 300), (1000, 1, 40, 100)])
@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("renorm", [False, True])
def test_route_weights_far_below_the_largest(hip, E, groups, k, m, kind, renorm):
    """Whole scores, whose differences are exact: the weights are right to a few units however small they are. expf is off by one
    unit (2 * 2^-24), the sum over a column (terms e^-x, each off by (x + 2) * 2^-24: 3 * 2^-24 of the sum; at most 10 additions that
    count) by 13, the reciprocal, the product and the scale by one each."""
    rng = np.random.default_rng(E + k)
    z = -rng.choice(np.arange(1, 80), (m, E)).astype(np.float64)
    z[:, 3] = 0
    z[:, 5] = -70                                        # few open experts: the far ones are taken too
    z[:, 6 + k:] = -np.inf
    a, G, ir = Columns(encode(z, 0)), empty(m, k, F), empty(m, k, np.int32)
    ok(hip.bidmat_route(E, m, 0, a.ptr, E, None, kind, groups, groups, k, int(renorm), 1.0, G.ptr, ir.ptr, None, None, None, None))
    wi, ww, _ = ref.route(z, None, kind, groups, groups, k, renorm, 1.0)
    assert np.array_equal(ir.get(), wi)
    within(G.get().astype(np.float64), ww, 18 * EPS24 * np.abs(ww), "weights")
