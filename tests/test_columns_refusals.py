"""Arguments that the operators over a model's columns refuse, before any work on a device: every call here returns 1
(hipErrorInvalidValue) without a GPU. Addresses are made up and never read."""
import pytest

from bidmat_amd import hip_abi

P, FAR, FARTHER = 0x10000000, 0x20000000, 0x30000000      # apart by more than any operand below covers
F32, F16, BF16 = hip_abi.F32, hip_abi.F16, hip_abi.BF16


def norm(**k):
    a = dict(nrows=64, ncols=4, type=BF16, X=P, ldx=64, R=None, ldr=64, w=FAR, eps=1e-5, H=None, ldh=64, Y=FARTHER, ldy=64, Q=None,
             ldq=64, scales=None, group=0, stream=None)
    a.update(k)
    return hip_abi.load().bidmat_rmsnorm(*a.values())


def norm_grad(**k):
    a = dict(nrows=64, ncols=4, type=BF16, H=P, ldh=64, w=FAR, eps=1e-5, dY=FARTHER, lddy=64, dH=None, lddh=64, dX=0x40000000, lddx=64,
             dw=None, beta=0, stream=None)
    a.update(k)
    return hip_abi.load().bidmat_rmsnorm_grad(*a.values())


def route(**k):
    a = dict(E=64, ncols=4, type=F32, Z=P, ldz=64, bias=None, kind=1, ngroups=8, topgroups=4, topk=8, renorm=1, scale=1.0, data=FAR,
             ir=FARTHER, ic=None, jc=None, counts=None, stream=None)
    a.update(k)
    return hip_abi.load().bidmat_route(*a.values())


def route_grad(**k):
    a = dict(E=64, ncols=4, type=F32, Z=P, ldz=64, kind=1, topk=8, renorm=1, scale=1.0, data=FAR, ir=FAR, dG=FAR, dZ=FARTHER, lddz=64,
             stream=None)
    a.update(k)
    return hip_abi.load().bidmat_route_grad(*a.values())


def distill(**k):
    a = dict(V=100, ncols=4, type=F16, Z=P, ldz=100, nnz=8, T=FAR, ir=FAR, jc=FAR, tau=1.0, weight=None, loss=FAR, lse=None, dZ=FARTHER,
             lddz=100, stream=None)
    a.update(k)
    return hip_abi.load().bidmat_distill(*a.values())


def distill_grad(**k):
    a = dict(V=100, ncols=4, type=F16, Z=P, ldz=100, nnz=8, T=FAR, ir=FAR, jc=FAR, tau=1.0, weight=None, lse=FAR, dZ=FARTHER, lddz=100,
             stream=None)
    a.update(k)
    return hip_abi.load().bidmat_distill_grad(*a.values())


def q8(**k):
    a = dict(k=64, ncols=4, nnz=8, Q=P, ldq=64, scales=FAR, group=32, S=FAR, ir=FAR, jc=FAR, C=FARTHER, beta=0, stream=None)
    a.update(k)
    return hip_abi.load().bidmat_dsmult_q8_csc(*a.values())


NAN, INF = float("nan"), float("inf")
COMMON = [dict(ncols=-1), dict(type=3), dict(type=-1)]


@pytest.mark.parametrize("bad", COMMON + [
    dict(nrows=-1), dict(nrows=32769, ldx=32769, ldy=32769), dict(X=None), dict(w=None), dict(Y=None), dict(eps=-1.0), dict(eps=NAN),
    dict(eps=INF), dict(ldx=63), dict(ldy=63), dict(R=FAR, ldr=63), dict(H=FAR + 64 * 64, ldh=63), dict(Q=FAR), dict(scales=FAR),
    dict(group=16), dict(group=-32), dict(X=P + 1), dict(Y=FARTHER + 1), dict(Y=P + 2), dict(Y=P, ldy=65), dict(H=FARTHER),
    dict(H=FARTHER + 128), dict(Q=P, scales=FAR), dict(Q=FARTHER, scales=FAR), dict(R=FARTHER - 2)])
def test_rmsnorm(bad):
    assert norm(**bad) == 1


@pytest.mark.parametrize("bad", COMMON + [
    dict(nrows=-1), dict(nrows=32769), dict(H=None), dict(w=None), dict(dY=None), dict(dX=None), dict(eps=-1.0), dict(eps=NAN),
    dict(beta=2), dict(ldh=63), dict(lddy=63), dict(lddx=63), dict(dH=P, lddh=63), dict(dX=P + 2), dict(dX=P, lddx=65), dict(dX=P + 1)])
def test_rmsnorm_grad(bad):
    assert norm_grad(**bad) == 1


@pytest.mark.parametrize("bad", COMMON + [
    dict(E=0), dict(E=1025, ldz=1025, ngroups=1, topgroups=1), dict(Z=None), dict(data=None), dict(ir=None), dict(kind=2), dict(renorm=2),
    dict(ngroups=0), dict(ngroups=7), dict(topgroups=0), dict(topgroups=9), dict(topk=0), dict(topk=33), dict(topk=65, topgroups=8),
    dict(E=128, ldz=128, ngroups=128), dict(scale=0.0), dict(scale=NAN), dict(scale=INF), dict(ldz=63), dict(Z=P + 2),
    dict(ncols=2 ** 28)])
def test_route(bad):
    assert route(**bad) == 1


@pytest.mark.parametrize("bad", COMMON + [
    dict(E=0), dict(E=1025, ldz=1025, lddz=1025), dict(Z=None), dict(data=None), dict(ir=None), dict(dG=None), dict(dZ=None), dict(kind=-1),
    dict(renorm=-1), dict(topk=0), dict(topk=65), dict(scale=0.0), dict(scale=NAN), dict(ldz=63), dict(lddz=63), dict(dZ=P + 4),
    dict(dZ=P, lddz=65), dict(ncols=2 ** 28)])
def test_route_grad(bad):
    assert route_grad(**bad) == 1


@pytest.mark.parametrize("bad", COMMON + [
    dict(V=-1), dict(V=2 ** 30 + 1, ldz=2 ** 30 + 1), dict(Z=None), dict(T=None), dict(ir=None), dict(jc=None), dict(nnz=-1), dict(tau=0.0),
    dict(tau=-1.0), dict(tau=NAN), dict(tau=INF), dict(tau=1e-45), dict(tau=1e-31), dict(tau=1e31), dict(tau=9e-19), dict(tau=1.1e18), dict(ldz=99), dict(lddz=99), dict(dZ=P + 2), dict(dZ=P, lddz=101),
    dict(Z=P + 1)])
def test_distill(bad):
    assert distill(**bad) == 1
    assert distill_grad(**bad) == 1


def test_distill_needs_an_output():
    assert distill(loss=None, lse=None, dZ=None) == 1
    assert distill_grad(lse=None) == 1
    assert distill_grad(dZ=None) == 1


@pytest.mark.parametrize("bad", [
    dict(k=-1), dict(ncols=-1), dict(nnz=-1), dict(Q=None), dict(scales=None), dict(S=None), dict(ir=None), dict(jc=None), dict(C=None),
    dict(ldq=63), dict(group=16), dict(group=256), dict(beta=2)])
def test_dsmult_q8(bad):
    assert q8(**bad) == 1


def test_overlapping_operands_are_refused():
    n = 64 * 4                                           # elements of the dense operands above
    assert norm(H=P + 2 * n - 2) == 1 and norm(H=FAR + 4) == 1 and norm(Y=FAR + 128) == 1
    assert norm(Q=0x50000000, scales=0x50000000 + 3) == 1 and norm(Q=0x50000000, scales=P + 4) == 1
    assert norm_grad(dw=FAR) == 1 and norm_grad(dw=0x40000000 + 8) == 1 and norm_grad(dw=FARTHER + 4) == 1
    assert route(ir=FAR) == 1 and route(ic=FAR + 4) == 1 and route(jc=FARTHER + 8) == 1 and route(counts=P) == 1 and route(bias=FAR + 4) == 1
    assert route_grad(dZ=FAR) == 1
    assert distill(loss=FARTHER + 4) == 1 and distill(lse=FAR) == 1 and distill(loss=P) == 1 and distill(weight=FAR + 4, loss=FAR + 16) == 1
    assert distill_grad(dZ=FAR) == 1
    assert q8(C=FAR) == 1 and q8(C=P) == 1 and q8(C=FARTHER + 2) == 1 and q8(scales=FAR + 2) == 1


def test_nothing_to_do_is_no_error():
    assert norm(nrows=0) == 0 and norm(ncols=0) == 0
    assert norm_grad(nrows=0) == 0 and norm_grad(ncols=0) == 0
    assert route(ncols=0) == 0 and route_grad(ncols=0) == 0
    assert distill(ncols=0, nnz=0) == 0 and distill(V=0, nnz=0) == 0
    assert q8(k=0) == 0 and q8(ncols=0) == 0
