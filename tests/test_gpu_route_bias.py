"""moe_route with selection biases near the largest finite value."""
import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda_device):
    from ferret_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("first,second", [(2e38, 3e38), (3e38, 2e38), (3.4e38, 1.6e38), (1.7e38, 3.4e38),
                                          (-3e38, -2e38), (2.5e38, 2.5e38)])
def test_groups_whose_sums_pass_the_largest_fp32(ops, scoring, first, second):
    """Two keys of a group add up to more than fp32 holds; the larger sum still wins."""
    E = 64
    g = torch.Generator(device="cuda").manual_seed(1)
    z = torch.randn(20, E, generator=g, device="cuda")
    bias = torch.empty(E, device="cuda")
    bias[:E // 2], bias[E // 2:] = first, second
    for n_group, keep in ((2, 1), (8, 3)):
        kw = dict(scoring=scoring, bias=bias, n_group=n_group, topk_group=keep, renormalize=True)
        _, ids = ops.moe_route(z, 5, **kw)
        assert torch.equal(ids.cpu().long(), R.route(z, 5, **kw)[1])
