"""What autograd is told by the operators around the expert GEMMs: second
derivatives, operators without a backward pass, tensors written in place."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda_device):
    from ferret_b200 import ops as _ops
    return _ops


@pytest.fixture(scope="module")
def F(ops):
    import ferret_b200.torch_ops  # noqa: F401
    return torch.ops.ferret_moe


# ---------------------------------------------------------- second derivatives

def route(F, z):
    return F.moe_route(z, 3, "sigmoid")[0]


def balance(F, z):
    ids = torch.zeros(z.shape[0], 2, dtype=torch.int32, device="cuda")
    return F.moe_balance_loss(z, ids, 0.5)[0]


@pytest.mark.parametrize("op", [route, balance])
@pytest.mark.parametrize("outer", [lambda v: v.sum(), lambda v: (v * v).sum()])
def test_second_derivatives_raise(F, op, outer):
    """Whether or not another term keeps the graph, and whether or not the incoming
    gradient has one."""
    z = torch.randn(6, 8, device="cuda", requires_grad=True)
    first, = torch.autograd.grad(outer(op(F, z)), z)
    for other in (lambda z: 0.0, lambda z: (z ** 3).sum()):
        grad, = torch.autograd.grad(outer(op(F, z)) + other(z), z, create_graph=True)
        more = 3 * z.detach() ** 2 if torch.is_tensor(other(z)) else 0.0
        assert torch.equal(grad.detach(), first + more)
        with pytest.raises(RuntimeError, match="once"):
            torch.autograd.grad(grad.square().sum(), z)
        with pytest.raises(RuntimeError, match="once"):
            grad.square().sum().backward()
