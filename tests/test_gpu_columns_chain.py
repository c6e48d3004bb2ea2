"""The operators over a model's columns together with the products they stand beside, as a small model with experts uses them,
forward and backward, against the same chain in 64 bits:

    H = A*S            documents as sparse columns over a vocabulary, embedded         (bidmat_dsmult_csc)
    Y = rmsnorm(H + R)                                                                 (bidmat_rmsnorm)
    Z = W^T Y          scores: DDS over the full pattern is a dense product            (bidmat_dds_csc)
    G = route(Z)       experts x documents, sparse                                     (bidmat_route)
    M = P*G            every document's mixture of the experts' vectors                (bidmat_dsmult_csc)
    L = O^T M          logits over the vocabulary                                      (bidmat_dds_csc)
    loss = distill(L, T)                                                               (bidmat_distill)

and back: dM = O dL, dP = dM *^ G, dG = DDS(P, dM, G), dZ, dY = W dZ, dH, dA = dH *^ S. Every stage is fp32 with sums
of at most a few hundred terms; the tolerance is the 1e-4 of the sparse products, on the 2-norm of each result.
"""
import ctypes as C

import numpy as np
import pytest

import columns_ref as ref
from bidmat_amd import hip_abi
from bidmat_amd.device import DeviceArray
from bidmat_amd.mats import DDS, GMat, GSMat, Mat
from util import dense_full, make_plan, random_csc

pytestmark = pytest.mark.gpu
F = np.float32
TOL = 1e-4


def ok(code):
    hip_abi.check(code)


def near(got, want, what, tol=TOL):
    got = np.asarray(got, np.float64).reshape(want.shape)
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want), what


class Model:
    def __init__(self, seed, k=96, V=300, m=130, E=32, topk=4, kind=1, renorm=True):
        g = np.random.default_rng(seed)
        self.k, self.V, self.m, self.E, self.topk, self.kind, self.renorm, self.eps, self.tau = k, V, m, E, topk, kind, renorm, 1e-5, 2.0
        self.scale = 1.5
        self.S, self.Sir, self.Sjc = random_csc(g, V, m, lengths=g.integers(1, 40, m))
        self.T, self.Tir, self.Tjc = random_csc(g, V, m, lengths=g.integers(0, 12, m))
        self.T = (4 * self.T).astype(F)
        # matrices as (columns, rows) arrays, the library's memory
        self.A, self.O = g.standard_normal((V, k)).astype(F), (g.standard_normal((V, k)) / 4).astype(F)
        self.W, self.P = (g.standard_normal((E, k)) / 6).astype(F), g.standard_normal((E, k)).astype(F)
        self.R, self.w = g.standard_normal((m, k)).astype(F), (1 + 0.1 * g.standard_normal(k)).astype(F)
        self.bias = (0.05 * g.standard_normal(E)).astype(F)
        self.weight = (g.random(m) / m).astype(F)

    def forward(self, A=None, fixed=None):
        """In 64 bits; `fixed`: the experts to take (so that small changes of A do not change them)."""
        A = self.A.astype(np.float64) if A is None else A
        S = dense_full(self.V, self.m, self.S, self.Sir, self.Sjc)
        o = {"H": S.T @ A}
        o["h"], o["Y"], _ = ref.rmsnorm(o["H"], self.R.astype(np.float64), self.w.astype(np.float64), float(F(self.eps)))
        o["Z"] = o["Y"] @ self.W.astype(np.float64).T
        o["ir"], o["g"], _ = ref.route(o["Z"], self.bias, self.kind, 4, 2, self.topk, self.renorm, self.scale)
        if fixed is not None:
            p = 1 / (1 + np.exp(-o["Z"])) if self.kind == 1 else np.exp(o["Z"]) / np.exp(o["Z"]).sum(1, keepdims=True)
            g = np.take_along_axis(p, fixed, 1)
            o["ir"], o["g"] = fixed, self.scale * (g / g.sum(1, keepdims=True) if self.renorm else g)
        G = np.zeros((self.m, self.E))
        np.put_along_axis(G, o["ir"], o["g"], 1)
        o["G"], o["M"] = G, G @ self.P.astype(np.float64)
        o["L"] = o["M"] @ self.O.astype(np.float64).T
        o["loss"], _, o["dL"], _, _ = ref.distill(o["L"], self.T, self.Tir, self.Tjc, self.tau, self.weight.astype(np.float64))
        return o

    def backward(self, o):
        S = dense_full(self.V, self.m, self.S, self.Sir, self.Sjc)
        b = {"dM": o["dL"] @ self.O.astype(np.float64)}
        b["dO"] = o["dL"].T @ o["M"]
        b["dP"] = o["G"].T @ b["dM"]
        b["dg"] = np.take_along_axis(b["dM"] @ self.P.astype(np.float64).T, o["ir"], 1)
        b["dZ"], _ = ref.route_grad(o["Z"], self.kind, self.renorm, self.scale, o["g"], o["ir"], b["dg"])
        b["dY"] = b["dZ"] @ self.W.astype(np.float64)
        b["dW"] = b["dZ"].T @ o["Y"]
        b["dH"], b["dw"], _, _ = ref.rmsnorm_grad(o["h"], self.w.astype(np.float64), float(F(self.eps)), b["dY"], None)
        b["dA"] = S @ b["dH"]
        return b


def full_pattern(rows, cols):
    return np.tile(np.arange(rows, dtype=np.int32), cols), (np.arange(cols + 1) * rows).astype(np.int32)


@pytest.mark.parametrize("kind,renorm", [(0, False), (0, True), (1, False), (1, True)])
def test_forward_and_backward(hip, kind, renorm):
    x = Model(5 + kind, kind=kind, renorm=renorm)
    k, V, m, E, tk = x.k, x.V, x.m, x.E, x.topk
    up = lambda a: DeviceArray.from_numpy(a)                  # noqa: E731
    new = lambda *s: DeviceArray.zeros(int(np.prod(s)))       # noqa: E731
    newi = lambda n: DeviceArray.zeros(n, np.int32)           # noqa: E731
    A, O, W, P, R, w, bias, weight = (up(a) for a in (x.A, x.O, x.W, x.P, x.R, x.w, x.bias, x.weight))
    S, Sir, Sjc, T, Tir, Tjc = (up(a) for a in (x.S, x.Sir, x.Sjc, x.T, x.Tir, x.Tjc))
    Eir, Ejc = (up(a) for a in full_pattern(E, m))
    Vir, Vjc = (up(a) for a in full_pattern(V, m))
    H, h, Y, Z, M, L = new(m, k), new(m, k), new(m, k), new(m, E), new(m, k), new(m, V)
    g, ir, jc, counts = new(m, tk), newi(m * tk), newi(m + 1), newi(E)
    loss, dL, dM, dO, dP, dg, dZ, dY, dW, dH, dw, dA = (new(m), new(m, V), new(m, k), new(V, k), new(E, k), new(m, tk), new(m, E), new(m, k),
                                                       new(E, k), new(m, k), new(k), new(V, k))
    ok(hip.bidmat_dsmult_csc(k, m, x.S.size, A.ptr, S.ptr, Sir.ptr, Sjc.ptr, H.ptr, 0, None))
    ok(hip.bidmat_rmsnorm(k, m, 0, H.ptr, k, R.ptr, k, w.ptr, x.eps, h.ptr, k, Y.ptr, k, None, k, None, 0, None))
    ok(hip.bidmat_dds_csc(k, m, E * m, W.ptr, Y.ptr, Eir.ptr, Ejc.ptr, Z.ptr, 0, None))
    ok(hip.bidmat_route(E, m, 0, Z.ptr, E, bias.ptr, kind, 4, 2, tk, int(renorm), x.scale, g.ptr, ir.ptr, None, jc.ptr, counts.ptr, None))
    ok(hip.bidmat_dsmult_csc(k, m, m * tk, P.ptr, g.ptr, ir.ptr, jc.ptr, M.ptr, 0, None))
    ok(hip.bidmat_dds_csc(k, m, V * m, O.ptr, M.ptr, Vir.ptr, Vjc.ptr, L.ptr, 0, None))
    ok(hip.bidmat_distill(V, m, 0, L.ptr, V, x.T.size, T.ptr, Tir.ptr, Tjc.ptr, x.tau, weight.ptr, loss.ptr, None, dL.ptr, V, None))
    # and back
    gate, words, full_e, full_v = (make_plan(hip, *a, k) for a in (
        (E, m, m * tk, ir, jc), (V, m, x.S.size, Sir, Sjc), (E, m, E * m, Eir, Ejc), (V, m, V * m, Vir, Vjc)))
    ok(hip.bidmat_dsmult_csc(k, m, V * m, O.ptr, dL.ptr, Vir.ptr, Vjc.ptr, dM.ptr, 0, None))
    ok(hip.bidmat_dsmultT_plan(full_v, k, M.ptr, dL.ptr, dO.ptr, 0, None))
    ok(hip.bidmat_dsmultT_plan(gate, k, dM.ptr, g.ptr, dP.ptr, 0, None))
    ok(hip.bidmat_dds_csc(k, m, m * tk, P.ptr, dM.ptr, ir.ptr, jc.ptr, dg.ptr, 0, None))
    ok(hip.bidmat_route_grad(E, m, 0, Z.ptr, E, kind, tk, int(renorm), x.scale, g.ptr, ir.ptr, dg.ptr, dZ.ptr, E, None))
    ok(hip.bidmat_dsmult_csc(k, m, E * m, W.ptr, dZ.ptr, Eir.ptr, Ejc.ptr, dY.ptr, 0, None))
    ok(hip.bidmat_dsmultT_plan(full_e, k, Y.ptr, dZ.ptr, dW.ptr, 0, None))
    ok(hip.bidmat_rmsnorm_grad(k, m, 0, h.ptr, k, w.ptr, x.eps, dY.ptr, k, None, k, dH.ptr, k, dw.ptr, 0, None))
    ok(hip.bidmat_dsmultT_plan(words, k, dH.ptr, S.ptr, dA.ptr, 0, None))
    ok(hip.bidmat_synchronize())
    o = x.forward()
    assert np.array_equal(ir.numpy().reshape(m, tk), o["ir"])
    assert np.array_equal(counts.numpy(), np.bincount(o["ir"].ravel(), minlength=E))
    for name, d in (("Y", Y), ("Z", Z), ("g", g), ("M", M), ("L", L), ("loss", loss), ("dL", dL)):
        near(d.numpy(), o[name], name)
    b = x.backward(o)
    for name, d in (("dM", dM), ("dO", dO), ("dP", dP), ("dg", dg), ("dZ", dZ), ("dY", dY), ("dW", dW), ("dH", dH), ("dw", dw), ("dA", dA)):
        near(d.numpy(), b[name], name)
    # the whole gradient against differences of the loss, the experts held
    to = np.random.default_rng(1).standard_normal(x.A.shape)
    step = 1e-5
    up_, down = (x.forward(x.A + s * to, o["ir"])["loss"].sum() for s in (step, -step))
    want, got = (up_ - down) / (2 * step), (dA.numpy().astype(np.float64).reshape(x.A.shape) * to).sum()
    assert abs(got - want) <= TOL * np.linalg.norm(b["dA"]) * np.linalg.norm(to)
    for p in (gate, words, full_e, full_v):
        ok(hip.bidmat_plan_destroy(p))


def test_documents_gathered_by_expert_in_eight_bits(hip):
    """Serving: the normalised columns in 8 bits, summed per expert over the transposed gate."""
    x = Model(9, k=256, m=400, E=16)
    o = x.forward()
    k, m, E, tk = x.k, x.m, x.E, x.topk
    H, R, w = (DeviceArray.from_numpy(a) for a in (o["H"].astype(F), x.R, x.w))
    Q, sc = DeviceArray.zeros(m * k, np.uint8), DeviceArray.zeros(m * 2)
    ok(hip.bidmat_rmsnorm(k, m, 0, H.ptr, k, R.ptr, k, w.ptr, x.eps, None, k, None, k, Q.ptr, k, sc.ptr, 128, None))
    Z, bias = DeviceArray.from_numpy(o["Z"].astype(F)), DeviceArray.from_numpy(x.bias)
    g, ir, jc = DeviceArray.zeros(m * tk), DeviceArray.zeros(m * tk, np.int32), DeviceArray.zeros(m + 1, np.int32)
    ok(hip.bidmat_route(E, m, 0, Z.ptr, E, bias.ptr, 1, 4, 2, tk, 1, 1.0, g.ptr, ir.ptr, None, jc.ptr, None, None))
    td, tir, tjc = DeviceArray.zeros(m * tk), DeviceArray.zeros(m * tk, np.int32), DeviceArray.zeros(E + 1, np.int32)
    ok(hip.bidmat_csc_transpose(E, m, m * tk, g.ptr, ir.ptr, jc.ptr, td.ptr, tir.ptr, tjc.ptr))
    out = DeviceArray.zeros(E * k)
    ok(hip.bidmat_dsmult_q8_csc(k, E, m * tk, Q.ptr, k, sc.ptr, 128, td.ptr, tir.ptr, tjc.ptr, out.ptr, 0, None))
    ok(hip.bidmat_synchronize())
    G = np.zeros((m, E))
    np.put_along_axis(G, ir.numpy().reshape(m, tk).astype(np.int64), g.numpy().reshape(m, tk).astype(np.float64), 1)
    codes = ref.E4M3[Q.numpy().reshape(m, k)] * np.repeat(sc.numpy().reshape(m, 2).astype(np.float64), 128, 1)
    near(out.numpy(), G.T @ codes, "sum of the codes")
    # against the columns themselves: each code is off by at most 2^-4 of its value or 2^-10 of its scale
    off = np.maximum(2.0 ** -4 * np.abs(o["Y"]), 2.0 ** -10 * np.repeat(sc.numpy().reshape(m, 2), 128, 1)) * 1.01
    assert (np.abs(out.numpy().reshape(E, k) - G.T @ o["Y"]) <= G.T @ off + TOL * np.abs(G.T @ o["Y"]) + 1e-4).all()


def test_the_matrix_interface(hip):
    """The same operators on GMat / GSMat: results of the right types and patterns, and the chain through them."""
    x = Model(11, kind=0, renorm=True)
    o = x.forward()
    b = x.backward(o)
    y, h = GMat.from_numpy(o["H"].T).rmsnorm(GMat.from_numpy(x.w), x.eps, residual=GMat.from_numpy(x.R.T))
    near(y.numpy().T, o["Y"], "y")
    near(h.numpy().T, o["h"], "h")
    z = GMat.from_numpy(o["Z"].T)
    gate = z.route(x.topk, bias=GMat.from_numpy(x.bias), ngroups=4, topgroups=2, scale=x.scale)
    data, ir, jc = gate.to_csc()
    assert np.array_equal(ir.reshape(x.m, x.topk) - 1, o["ir"]) and np.array_equal(jc, 1 + x.topk * np.arange(x.m + 1))
    near(data, o["g"].ravel(), "gate")
    p = GMat.from_numpy(x.P.T)
    M = p * gate
    near(M.numpy().T, o["M"], "M")
    base = int(Mat.get("ioneBased"))
    T = GSMat.from_csc(x.V, x.m, x.T, x.Tir + base, x.Tjc + base)
    logits, grad = GMat.from_numpy(o["L"].T), GMat.zeros(x.V, x.m)
    loss = logits.distill(T, x.tau, weight=GMat.from_numpy(x.weight), grad=grad)
    assert loss.shape == (1, x.m)
    near(loss.numpy().ravel(), o["loss"], "loss")
    near(grad.numpy().T, o["dL"], "dL")
    dgate = DDS(p, GMat.from_numpy(b["dM"].T), gate)
    assert dgate.same_pattern(gate)
    near(GMat.from_numpy(b["dM"].T).xT(gate).numpy().T, b["dP"], "dP")
    dz = z.routeGrad(gate, dgate, scale=x.scale)
    near(dz.numpy().T, b["dZ"], "dZ")
    dw = GMat.zeros(x.k, 1)
    for _ in range(2):
        dh = h.rmsnormGrad(GMat.from_numpy(x.w), GMat.from_numpy(b["dY"].T), x.eps, dw=dw)
    near(dh.numpy().T, b["dH"], "dH")
    near(dw.numpy().ravel(), 2 * b["dw"], "dw")
    # another gate into the same matrix: its pattern is its own again
    again = z.route(x.topk, out=gate)
    assert again.same(gate) and not dgate.same_pattern(gate)
    for bad in (lambda: z.route(0), lambda: z.route(x.topk, ngroups=5), lambda: z.rmsnorm(GMat.zeros(3, 1)),
                lambda: logits.distill(gate), lambda: logits.distill(T, -1.0), lambda: z.routeGrad(T, dgate)):
        with pytest.raises(RuntimeError):
            bad()


def test_cached_outputs_belong_to_all_operands_and_settings(hip):
    """With the operator cache on, calls that differ in any operand or setting have outputs of their own."""
    rng = np.random.default_rng(9)
    n, m, k = 24, 10, 4
    x, w1, w2, dy, dh = (GMat.from_numpy(rng.standard_normal(s).astype(np.float32)) for s in ((n, m), (n, 1), (n, 1), (n, m), (n, m)))
    teacher = GMat.from_numpy(rng.standard_normal((n, m)).astype(np.float32)).route(3)
    weight = GMat.from_numpy(rng.random((1, m)).astype(np.float32))

    def calls():
        g1, g2 = x.route(k), x.route(k, sigmoid=True)
        return [x.rmsnorm(w1)[0], x.rmsnorm(w2)[0], x.rmsnorm(w1, eps=0.5)[0], x.rmsnorm(w1, residual=dy)[0],
                x.rmsnormGrad(w1, dy), x.rmsnormGrad(w2, dy), x.rmsnormGrad(w1, dy, eps=0.5), x.rmsnormGrad(w1, dy, dh=dh),
                x.route(k).contents(), x.route(k, scale=1.0 + 2.0 ** -20).contents(), x.route(k, renorm=False).contents(),
                x.routeGrad(g1, g1), x.routeGrad(g2, g1, sigmoid=True), x.routeGrad(g1, g1, renorm=False), x.routeGrad(g1, g1, scale=2.0),
                x.distill(teacher), x.distill(teacher, 2.0), x.distill(teacher, weight=weight)]

    plain = [a.numpy().copy() for a in calls()]
    Mat.set("useGPUcache", 1)
    try:
        kept = calls()
        for i, (a, b) in enumerate(zip(kept, plain)):
            assert np.array_equal(a.numpy(), b), i
    finally:
        Mat.set("useGPUcache", 0)
        Mat.clear_caches()
