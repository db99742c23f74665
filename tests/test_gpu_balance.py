"""moe_balance_loss and its gradient against the definition in 64 bits.

Tolerances.  A probability is within 64 * 2^-24 (expf and its rounded argument,
37 additions of the sum, the quotient); its sum over T tokens adds the roundings
of a lane's own tokens and of the joins, at most 256 for the sizes here.  The
gradient is p (c - sum c p) factor: its bound counts p times the largest
|c - mean|."""
import math

import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu
P_REL = 64 * R.U
SUM_REL = (64 + 256) * R.U
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops(cuda_device):
    from ferret_b200 import ops as _ops
    return _ops


def make(T, E, topk, dtype=torch.float32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = 1.5 * torch.randn(T, E, generator=g, device="cuda") \
        + 0.7 * torch.randn(E, generator=g, device="cuda")
    ids = z.argsort(dim=1, descending=True)[:, :topk].to(torch.int32).contiguous()
    return z.to(dtype), ids


def check(ops, logits, ids, coef=0.02, scoring="softmax", mask=None, scale=3.0):
    grad = torch.tensor(scale, device="cuda")
    loss, counts, sums, n = ops.moe_balance_loss(logits, ids, coef, scoring=scoring, token_mask=mask)
    dz = ops.moe_balance_loss_backward(grad, logits, counts, n, ids.shape[1], coef, scoring=scoring,
                                       token_mask=mask)
    rl, rc, rs, rn, rd = R.balance(logits, ids, coef, scoring, mask, scale)
    E = logits.shape[1]
    assert loss.shape == () and loss.dtype == torch.float32 and counts.dtype == torch.int32
    assert torch.equal(counts.cpu().long(), rc) and int(n) == rn
    assert ((sums.double().cpu() - rs).abs() <= rs * SUM_REL + 1e-37).all()
    assert abs(float(loss) - rl) <= abs(rl) * (SUM_REL + 2 * R.U)
    assert dz.dtype == logits.dtype and dz.shape == logits.shape
    if rn:
        factor = abs(scale * coef) * E / (ids.shape[1] * rn * rn)
        spread = (rc.double() - rc.double().mean()).abs().max() + 1
        p = R.scores(R.clean(logits), scoring)
        if scoring == "sigmoid":
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
        t = logits.dtype
        bound = rd.abs() * R.half_step(t) + 4 * p * spread * factor * P_REL + R.smallest(t) + 1e-37
        assert ((dz.double().cpu() - rd).abs() <= bound).all()
    return loss, counts, sums, n, dz


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,topk", [(1, 1, 1), (2, 3, 2), (257, 8, 2), (100, 33, 4), (37, 60, 6),
                                      (700, 128, 1), (333, 160, 6), (1025, 256, 8), (50, 500, 10),
                                      (9, 1024, 40)])
def test_loss_and_gradient(ops, dtype, scoring, T, E, topk):
    logits, ids = make(T, E, topk, dtype, T + E)
    check(ops, logits, ids, scoring=scoring, scale=1e4 if dtype == torch.float16 else 3.0)
    mask = torch.rand(T, device="cuda") > 0.4
    check(ops, logits, ids, scoring=scoring, mask=mask, scale=1e4 if dtype == torch.float16 else 3.0)


def test_an_even_batch_costs_the_coefficient(ops):
    E, topk = 16, 2
    ids = torch.arange(64, device="cuda", dtype=torch.int32).remainder(E).view(32, topk).contiguous()
    loss, counts, _, _ = ops.moe_balance_loss(torch.zeros(32, E, device="cuda"), ids, 0.5)
    assert (counts == 4).all() and abs(float(loss) - 0.5) <= 0.5 * SUM_REL


def test_what_masks_and_closed_logits_hide(ops):
    logits, ids = make(64, 40, 4, torch.float32, 2)
    ids[5] = -1
    ids[6, 1:] = 40
    ids[7, 0] = 2 ** 31 - 1
    logits[8, 3:] = -math.inf
    logits[9] = -math.inf
    logits[10, ::3] = math.nan
    logits[11, 4] = math.inf
    logits[12] = torch.finfo(torch.float32).min
    mask = torch.ones(64, dtype=torch.bool, device="cuda")
    mask[20:40] = False
    for scoring in ("softmax", "sigmoid"):
        want = check(ops, logits, ids, scoring=scoring, mask=mask)
        dirty, dirty_ids = logits.clone(), ids.clone()
        dirty[20:30], dirty[30:40], dirty_ids[20:40] = math.nan, math.inf, 7
        got = check(ops, dirty, dirty_ids, scoring=scoring, mask=mask)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        assert (got[4][20:40] == 0).all()
        loss, counts, sums, n, dz = check(ops, logits, ids, scoring=scoring,
                                          mask=torch.zeros_like(mask))
        assert float(loss) == 0 and int(n) == 0 and (counts == 0).all() and (sums == 0).all()
        assert (dz == 0).all()


def test_no_tokens(ops):
    z = torch.empty(0, 12, device="cuda")
    ids = torch.empty(0, 3, device="cuda", dtype=torch.int32)
    loss, counts, sums, n = ops.moe_balance_loss(z, ids, 0.1)
    assert float(loss) == 0 and int(n) == 0 and (counts == 0).all() and (sums == 0).all()
    one = torch.ones((), device="cuda")
    assert ops.moe_balance_loss_backward(one, z, counts, n, 3, 0.1).shape == (0, 12)


def test_strided_logits(ops):
    big, ids = make(90, 131, 4, torch.bfloat16, 8)
    ids = ids.remainder(96).contiguous()
    for view in (big[:, :96], big[:, 1:97], big[:, 32:128]):
        check(ops, view, ids)


def test_repeats_bit_for_bit_and_replays(ops):
    logits, ids = make(20_000, 256, 8, torch.float32, 5)
    one = torch.ones((), device="cuda")

    def step():
        loss, counts, sums, n = ops.moe_balance_loss(logits, ids, 0.01)
        return loss, counts, sums, n, ops.moe_balance_loss_backward(one, logits, counts, n, 8, 0.01)

    want = step()
    for a, b in zip(step(), want):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    torch.cuda.synchronize()
    for g, _ in graphs:                                     # two graphs side by side
        with torch.cuda.stream(torch.cuda.Stream()):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_long_batch(ops):
    """Sums over 200,000 tokens: 64-bit reference from the probabilities in fp64."""
    T, E = 200_003, 32
    logits, ids = make(T, E, 2, torch.float32, 6)
    loss, counts, sums, n = ops.moe_balance_loss(logits, ids, 0.01)
    rs = torch.softmax(logits.double(), 1).sum(0)
    assert ((sums.double() - rs).abs() <= rs * SUM_REL).all()
    assert torch.equal(counts.long(), torch.bincount(ids.flatten().long(), minlength=E))


def test_gradient_against_differences(ops):
    """The loss along a direction, counts fixed: central difference in fp64 of the
    probabilities' sums that the kernel returns; off by h^2 / 6 of a third
    derivative and by the sums' roundings over h."""
    T, E, topk, h = 40, 12, 3, 2.0 ** -6
    logits, ids = make(T, E, topk, torch.float32, 3)
    for scoring in ("softmax", "sigmoid"):
        _, counts, _, n = ops.moe_balance_loss(logits, ids, 1.0, scoring=scoring)
        one = torch.ones((), device="cuda")
        dz = ops.moe_balance_loss_backward(one, logits, counts, n, topk, 1.0, scoring=scoring)
        along = torch.randn(T, E, device="cuda").clamp(-1, 1)

        def at(z):
            sums = ops.moe_balance_loss(z, ids, 1.0, scoring=scoring)[2].double()
            return E / (topk * T * T) * (counts.double() * sums).sum()

        up, down = logits + h * along, logits - h * along
        want = (at(up) - at(down)) / 2
        got = (dz.double() * (up.double() - down.double()) / 2).sum()
        size = E / (topk * T * T) * float(counts.double().max()) * T
        assert abs(float(got - want)) <= size * (4 * h ** 3 + 2 * SUM_REL)


def test_more_than_2_to_the_31_logits(ops):
    T, E = 2_097_160, 1024
    logits = torch.zeros(T, E, dtype=torch.bfloat16, device="cuda")
    logits[-3:] = torch.randn(3, E, device="cuda")
    ids = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    ids[-1] = 1023
    loss, counts, sums, n = ops.moe_balance_loss(logits, ids, 1.0)
    assert int(counts[0]) == T - 1 and int(counts[1023]) == 1 and int(n) == T
    assert abs(float(sums.double().sum()) / T - 1) <= 1e-4
    one = torch.full((), 1e6, device="cuda")
    dz = ops.moe_balance_loss_backward(one, logits, counts, n, 1, 1.0)
    tail = ops.moe_balance_loss_backward(one, logits[-3:].clone(), counts, n, 1, 1.0)
    assert torch.equal(dz[-3:], tail) and bool((tail != 0).any())


def test_refusals(ops):
    from ferret_b200._lib import FerretError
    z, ids = make(8, 32, 2)
    mask = torch.ones(8, dtype=torch.bool, device="cuda")
    one = torch.ones((), device="cuda")
    _, counts, _, n = ops.moe_balance_loss(z, ids, 0.1)
    for f in (lambda: ops.moe_balance_loss(z, ids.long(), 0.1),
              lambda: ops.moe_balance_loss(z, ids[:4], 0.1),
              lambda: ops.moe_balance_loss(z, ids[0], 0.1),
              lambda: ops.moe_balance_loss(z, ids, 0.1, scoring="x"),
              lambda: ops.moe_balance_loss(z, ids, 0.1, token_mask=mask.int()),
              lambda: ops.moe_balance_loss(z.double(), ids, 0.1),
              lambda: ops.moe_balance_loss(z.t(), ids, 0.1),
              lambda: ops.moe_balance_loss_backward(one.double(), z, counts, n, 2, 0.1),
              lambda: ops.moe_balance_loss_backward(one.view(1), z, counts, n, 2, 0.1),
              lambda: ops.moe_balance_loss_backward(one, z, counts[:-1], n, 2, 0.1),
              lambda: ops.moe_balance_loss_backward(one, z, counts, n.long(), 2, 0.1),
              lambda: ops.moe_balance_loss_backward(one.cpu(), z, counts, n, 2, 0.1)):
        with pytest.raises((ValueError, TypeError)):
            f()
    with pytest.raises(FerretError):
        ops.moe_balance_loss(torch.zeros(2, 1025, device="cuda"), ids[:2], 0.1)
    with pytest.raises(FerretError):
        ops.moe_balance_loss_backward(one, z, counts, n, 0, 0.1)
