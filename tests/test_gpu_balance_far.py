"""Sigmoid scores of the balance loss far from zero, against the definition formed
from logarithms of the sigmoids in 64 bits (which do not underflow).

Tolerances.  A probability is e^(z - shift) / (1 + e^z) over a sum, shift the row's
largest negative logit.  z - shift and its product with log2(e) are rounded once
each and log2(e) itself is off by 2^-26 of itself, which moves the exponent by at most
2.25 |z - shift| 2^-24; the rest (ex2, additions of the sum, quotients) is below
64 * 2^-24, and what is below 2^-126 counts as 0.  Sums over the tokens add 256 *
2^-24 of themselves.  The gradient p (1 - s) (c - sum c p) factor has the errors of p, those
of 1 - s (e^-|z|, 1.25 |z| 2^-24, and 64 * 2^-24 with the rest) and of the row's sum."""
import math

import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops(cuda_device):
    from ferret_b200 import ops as _ops
    return _ops


def check(ops, logits, ids, coef=0.5, scale=1e3):
    loss, counts, sums, n = ops.moe_balance_loss(logits, ids, coef, scoring="sigmoid")
    dz = ops.moe_balance_loss_backward(torch.tensor(scale, device="cuda"), logits, counts, n,
                                       ids.shape[1], coef, scoring="sigmoid")
    z = R.clean(logits)
    T, E = z.shape
    log = torch.nn.functional.logsigmoid(z)
    live = log > -math.inf
    m = log.max(1, keepdim=True).values
    v = torch.where(live, log - torch.where(m == -math.inf, 0.0, m), -math.inf)
    e = torch.exp(v)
    p = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    c = counts.double().cpu()
    factor = scale * coef * E / (ids.shape[1] * T * T)
    rest = torch.sigmoid(-z)
    want = factor * p * rest * (c - (p * c).sum(1, keepdim=True))
    # |z - shift| where the exponential is not 0
    far = torch.where(live, v.abs(), 0.0).clamp(max=90.0)
    rel = (64 + 2.25 * far) * R.U
    floor = 2.0 ** -124
    assert int(n) == T
    assert ((sums.double().cpu() - p.sum(0)).abs()
            <= (p * rel).sum(0) + p.sum(0) * 256 * R.U + T * floor).all()
    exact = coef * E / (ids.shape[1] * T * T) * float((c * p.sum(0)).sum())
    slack = coef * E / (ids.shape[1] * T * T) * float((c * (p * (rel + 256 * R.U)).sum(0)).sum())
    assert abs(float(loss) - exact) <= slack + exact * 2 * R.U + 1e-37
    spread = float((c - c.mean()).abs().max()) + 1
    slope = (64 + 1.25 * z.abs().clamp(max=90.0)) * R.U
    row = (p * rel).sum(1, keepdim=True)
    t = logits.dtype
    bound = want.abs() * R.half_step(t) + R.smallest(t) + factor * spread * (
        4 * p * rest * (rel + slope + row) + floor)
    bound = torch.where(live, bound, 0.0)
    assert dz.dtype == t
    assert ((dz.double().cpu() - want).abs() <= bound).all()
    return sums, dz


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E", [8, 33, 60, 128, 160, 256, 500, 1024])
def test_rows_of_far_negative_logits(ops, dtype, E):
    g = torch.Generator(device="cuda").manual_seed(E)
    at = [-86.0, -87.0, -88.0, -90.0, -104.0, -120.0, -200.0, -745.0, -1000.0, -30000.0]
    z = torch.tensor(at, device="cuda").repeat_interleave(4)[:, None].expand(-1, E).clone()
    z[1::4] += torch.randn(len(at), E, generator=g, device="cuda")
    z[2::4] += 20 * torch.randn(len(at), E, generator=g, device="cuda").clamp(-2, 2)
    z[3::4, ::3] = -math.inf
    ids = torch.randint(0, E, (z.shape[0], 2), generator=g, device="cuda").to(torch.int32)
    sums, dz = check(ops, z.to(dtype), ids)
    assert abs(float(sums.double().sum()) - z.shape[0]) <= z.shape[0] * 1e-4     # every row counts


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E", [8, 48, 100, 200])
def test_rows_across_the_smallest_normal_sigmoid(ops, dtype, E):
    """Logits on both sides of -87.3, where e^z leaves the normal range, and rows that
    hold ordinary and far logits together."""
    g = torch.Generator(device="cuda").manual_seed(3 * E)
    z = -87.3 + 3 * torch.randn(24, E, generator=g, device="cuda")
    z[8:12, 1:] = -90.0
    z[8:12, 0] = torch.tensor([-86.0, -60.0, 0.0, 5.0], device="cuda")
    z[12:18] = 40 * torch.randn(6, E, generator=g, device="cuda")
    z[18, ::2] = math.nan
    z[19, 1:] = -math.inf
    z[20, 3] = math.inf
    ids = torch.randint(-1, E + 1, (24, 3), generator=g, device="cuda").to(torch.int32)
    check(ops, z.to(dtype), ids)


def test_far_rows_among_ordinary_ones(ops):
    """The ordinary rows of a batch are not moved by its far rows."""
    T, E = 3000, 160
    g = torch.Generator(device="cuda").manual_seed(7)
    z = 1.5 * torch.randn(T, E, generator=g, device="cuda")
    ids = z.argsort(dim=1, descending=True)[:, :6].to(torch.int32).contiguous()
    far = z.clone()
    far[::7] -= 150.0
    _, dz = check(ops, z, ids)
    _, dz_far = check(ops, far, ids)
    keep = torch.arange(T, device="cuda") % 7 != 0
    assert torch.equal(dz[keep], dz_far[keep])
    assert (dz_far[::7] != 0).any(1).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_of_the_lowest_finite_value_is_closed(ops, dtype):
    """A mask of the type's lowest value that leaves nothing: p = 0, as with -inf.  Beside
    other logits such a value has p = 0 by the definition."""
    z = torch.zeros(4, 16, device="cuda", dtype=dtype)
    low = torch.finfo(dtype).min
    z[1], z[2, 2:] = low, low
    z[3], z[3, 5] = low, -500.0
    ids = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    loss, counts, sums, n = ops.moe_balance_loss(z, ids, 1.0, scoring="sigmoid")
    want = torch.full((16,), 1 / 16)
    want[:2] += 0.5
    want[5] += 1.0
    assert torch.allclose(sums.cpu(), want, rtol=1e-5, atol=0)
    one = torch.full((), 1e3, device="cuda")
    dz = ops.moe_balance_loss_backward(one, z, counts, n, 1, 1.0, scoring="sigmoid")
    assert (dz[1] == 0).all() and (dz[2, 2:] == 0).all() and (dz[2, :2] != 0).all()
