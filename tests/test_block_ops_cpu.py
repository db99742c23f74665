"""The operators around the expert GEMMs without a GPU: argument checks of the C
ABI and of the torch functions, operator schemas, and the 64-bit restatements
that the GPU tests compare with, against small cases done by hand."""
import ctypes

import pytest
import torch

import block_ref as R
from ferret_b200 import _lib, build, ops

P = ctypes.c_void_p(0x1000)          # never dereferenced: validation fails first
ODD = ctypes.c_void_p(0x1001)


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


def test_norm_validation(L):
    f = L.ferret_add_rms_norm
    ok = dict(x=P, ldx=256, r=P, ldr=256, w=P, wdt=0, dt=0, T=4, K=256, eps=1e-6, y=P, ro=P, q=P,
              s=P, flags=0, st=None)

    def rc(**kw):
        return f(*dict(ok, **kw).values())

    for kw in (dict(dt=3), dict(dt=-1), dict(wdt=1), dict(T=-1), dict(K=0), dict(K=32776, ldx=40000),
               dict(K=200), dict(ldx=255), dict(ldr=255), dict(eps=-1.0), dict(eps=float("nan"))):
        assert rc(**kw) == -1, kw
    for kw in (dict(x=None), dict(w=None), dict(y=None, q=None), dict(s=None), dict(r=None)):
        assert rc(**kw) == -3, kw
    for kw in (dict(x=ODD), dict(r=ODD), dict(w=ODD), dict(y=ODD), dict(ro=ODD), dict(q=ODD),
               dict(s=ODD)):
        assert rc(**kw) == -2, kw
    assert rc(T=0, x=None, y=None) == 0


def test_route_validation(L):
    ok = dict(z=P, ld=64, dt=2, b=P, m=P, T=4, E=64, topk=4, g=8, kg=4, gt=2, sc=1.0, fl=0, w=P,
              ids=P, st=None)

    def rc(**kw):
        return L.ferret_moe_route(*dict(ok, **kw).values())

    for kw in (dict(dt=7), dict(T=-1), dict(E=0), dict(E=1025, ld=1025), dict(topk=0), dict(topk=33),
               dict(topk=65), dict(ld=63), dict(g=3), dict(g=0), dict(g=64), dict(kg=0), dict(kg=9),
               dict(gt=0), dict(gt=3), dict(topk=9, kg=1), dict(T=2 ** 30, topk=4), dict(E=60, ld=60)):
        assert rc(**kw) == -1, kw
    for kw in (dict(z=None), dict(w=None), dict(ids=None)):
        assert rc(**kw) == -3, kw
    for kw in (dict(z=ODD), dict(b=ODD), dict(w=ODD), dict(ids=ODD)):
        assert rc(**kw) == -2, kw
    assert rc(T=0, z=None) == 0
    back = dict(g=P, z=P, ld=64, dt=2, ids=P, T=4, E=64, topk=4, sc=1.0, fl=0, out=P, st=None)

    def rb(**kw):
        return L.ferret_moe_route_backward(*dict(back, **kw).values())

    for kw in (dict(dt=3), dict(T=-1), dict(E=0), dict(E=2000, ld=2000), dict(topk=0), dict(topk=33),
               dict(ld=1)):
        assert rb(**kw) == -1, kw
    assert rb(g=None) == -3 and rb(out=None) == -3 and rb(out=ODD) == -2 and rb(T=0) == 0


def test_balance_validation(L):
    size = L.ferret_moe_balance_loss_workspace_size
    assert size(0, 8) == 0 and size(4, 0) == 0 and size(4, 1025) == 0
    assert 0 < size(1, 8) <= size(100_000, 8) == size(10_000_000, 8)
    ok = dict(z=P, ld=64, dt=2, ids=P, m=P, T=4, E=64, topk=4, c=0.1, fl=0, loss=P, cnt=P, ps=P, n=P,
              ws=P, bytes=1 << 24, st=None)

    def rc(**kw):
        return L.ferret_moe_balance_loss(*dict(ok, **kw).values())

    for kw in (dict(dt=3), dict(T=-1), dict(E=0), dict(E=1025, ld=1025), dict(topk=0), dict(ld=63)):
        assert rc(**kw) == -1, kw
    for kw in (dict(z=None), dict(ids=None), dict(loss=None), dict(cnt=None), dict(ps=None),
               dict(n=None)):
        assert rc(**kw) == -3, kw
    assert rc(loss=ODD) == -2 and rc(ws=ODD) == -2
    assert rc(ws=None) == -7 and rc(bytes=size(4, 64) - 1) == -7
    back = dict(g=P, z=P, ld=64, dt=2, cnt=P, n=P, m=P, T=4, E=64, topk=4, c=0.1, fl=0, out=P, st=None)

    def rb(**kw):
        return L.ferret_moe_balance_loss_backward(*dict(back, **kw).values())

    for kw in (dict(dt=3), dict(T=-1), dict(E=0), dict(topk=0), dict(ld=63)):
        assert rb(**kw) == -1, kw
    assert rb(g=None) == -3 and rb(cnt=None) == -3 and rb(out=ODD) == -2 and rb(T=0) == 0


def test_int4_linear_validation(L):
    ok = dict(x=P, ldx=256, w=P, s=P, z=P, b=P, dt=0, T=4, K=256, N=64, g=64, y=P, st=None)

    def rc(**kw):
        return L.ferret_int4_linear(*dict(ok, **kw).values())

    for kw in (dict(dt=2), dict(T=-1), dict(K=0), dict(N=0), dict(N=60), dict(g=0), dict(g=16),
               dict(g=96), dict(ldx=248), dict(ldx=260), dict(K=1 << 21, ldx=1 << 21),
               dict(T=1 << 22), dict(N=1 << 24)):
        assert rc(**kw) == -1, kw
    for kw in (dict(x=None), dict(w=None), dict(s=None), dict(y=None)):
        assert rc(**kw) == -3, kw
    A8 = ctypes.c_void_p(0x1008)
    for kw in (dict(x=A8), dict(w=A8), dict(s=A8), dict(z=ODD), dict(b=ODD), dict(y=ODD)):
        assert rc(**kw) == -2, kw
    assert rc(T=0, x=None) == 0


CALLS = {
    "add_rms_norm": lambda: ops.add_rms_norm(torch.zeros(2, 128), torch.ones(128)),
    "moe_route": lambda: ops.moe_route(torch.zeros(2, 8), 2),
    "moe_route_backward": lambda: ops.moe_route_backward(
        torch.zeros(2, 2), torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32)),
    "moe_balance_loss": lambda: ops.moe_balance_loss(
        torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32), 0.1),
    "moe_balance_loss_backward": lambda: ops.moe_balance_loss_backward(
        torch.ones(()), torch.zeros(2, 8), torch.zeros(8, dtype=torch.int32),
        torch.ones(1, dtype=torch.int32), 2, 0.1),
    "int4_linear": lambda: ops.int4_linear(
        torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(8, 16, dtype=torch.int32),
        torch.zeros(2, 16, dtype=torch.bfloat16)),
    "fp8_gather_rows": lambda: ops.fp8_gather_rows(
        torch.zeros(2, 128, dtype=torch.float8_e4m3fn), torch.zeros(2, 1),
        torch.zeros(2, dtype=torch.int32)),
    "fp8_moe_block": lambda: ops.fp8_moe_block(
        torch.zeros(2, 256, dtype=torch.bfloat16), None, torch.ones(256, dtype=torch.bfloat16),
        torch.zeros(4, 256, dtype=torch.bfloat16), *[torch.zeros(4, 256, 256)] * 4, 2),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_host_tensors_are_refused(name):
    with pytest.raises((ValueError, TypeError)):
        CALLS[name]()


def test_schemas():
    import ferret_b200.torch_ops  # noqa: F401
    F = torch.ops.ferret_moe
    assert "Tensor? bias=None" in str(F.moe_route.default._schema)
    assert "Tensor? token_mask=None" in str(F.moe_balance_loss.default._schema)
    for name in ("add_rms_norm", "add_rms_norm_fp8", "int4_linear"):
        assert hasattr(F, name)


# --------------------------------------------- the restatements, done by hand

def test_reference_route_by_hand():
    z = torch.tensor([[0.0, 1.0, 1.0, -float("inf")], [2.0, 0.0, 1.0, 3.0]])
    w, ids = R.route(z, 3)
    assert ids.tolist() == [[1, 2, 0], [3, 0, 2]]
    e = torch.exp(z.double())
    assert torch.allclose(w[0], torch.stack([e[0, 1], e[0, 2], e[0, 0]]) / e[0].sum())
    _, ids = R.route(z, 2, n_group=2, topk_group=1)           # sums of p: groups (0,1) and (2,3)
    assert ids.tolist() == [[1, 0], [3, 2]]
    _, ids = R.route(z, 2, bias=torch.tensor([5.0, 0.0, 0.0, 0.0]), token_mask=torch.tensor([1, 0]))
    assert ids.tolist() == [[0, 1], [-1, -1]]


def test_reference_balance_by_hand():
    z = torch.zeros(2, 4)
    ids = torch.tensor([[0, 1], [0, 4]], dtype=torch.int32)
    loss, counts, sums, n, dz = R.balance(z, ids, 1.0)
    assert counts.tolist() == [2, 1, 0, 0] and n == 2 and sums.tolist() == [0.5] * 4
    assert abs(loss - 4 / (2 * 4) * 1.5) < 1e-12
    assert torch.allclose(dz[0], 0.5 * 0.25 * (torch.tensor([2.0, 1, 0, 0]).double() - 0.75))


def test_reference_int4_by_hand():
    w = torch.tensor([[0x76543210, -1], [0, 0], [0, 0], [0, 0]], dtype=torch.int32)
    x = torch.zeros(1, 32)
    x[0, 3], x[0, 8] = 2.0, 1.0
    scale = torch.tensor([[0.5, 0.25]])
    y, _ = R.int4(x, w, scale)
    assert y.tolist() == [[(3 - 8) * 1.0 - 8 * 0.5, (15 - 8) * 0.5 - 8 * 0.25]]


def test_reference_norm_by_hand():
    y, s = R.norm(torch.tensor([[1.0, 2.0]]), torch.tensor([1.0, 3.0]), torch.tensor([[2.0, 2.0]]), 0.0)
    assert s.tolist() == [[3.0, 4.0]]
    assert torch.allclose(y, torch.tensor([[3.0, 12.0]]).double() / 12.5 ** 0.5)
