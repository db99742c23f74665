"""moe_route and its gradient against the definition in 64 bits.

Ids have to be equal: the order is that of the exact keys.  Weights: a score is
within 2 ulp of expf, whose argument z - max is rounded once (|z - max| 2^-24,
at most 20 here), plus the sum (32 + 5 additions) and a quotient, for both
numerator and sum: below 128 * 2^-24 relative; gradients are products of a few
such factors and a difference g - mean(g), so their bound counts the size of
the terms, not of the difference."""
import math

import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu
REL = 128 * R.U
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops(cuda_device):
    from ferret_b200 import ops as _ops
    return _ops


def make(T, E, dtype=torch.float32, seed=0, spread=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")
    return (spread * f(T, E) + 0.7 * f(E)).to(dtype), 0.05 * f(E)


def check(ops, logits, topk, **kw):
    w, ids = ops.moe_route(logits, topk, **kw)
    rw, rid = R.route(logits, topk, **kw)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32
    assert torch.equal(ids.cpu().long(), rid), (ids.cpu() != rid).nonzero()[:4]
    assert ((w.double().cpu() - rw).abs() <= rw * REL + 1e-37).all()
    return w, ids


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring,renorm", [("softmax", False), ("softmax", True),
                                            ("sigmoid", False), ("sigmoid", True)])
@pytest.mark.parametrize("T,E,topk", [(1, 1, 1), (3, 5, 5), (37, 60, 4), (130, 256, 8), (9, 384, 8),
                                      (5, 1024, 32), (17, 33, 9), (65, 8, 2), (4, 1000, 6)])
def test_choice_and_weights(ops, dtype, scoring, renorm, T, E, topk):
    logits, bias = make(T, E, dtype, T + E)
    check(ops, logits, topk, scoring=scoring, renormalize=renorm, scale=2.5)
    check(ops, logits, topk, scoring=scoring, renormalize=renorm, bias=bias)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E,n_group,keep,topk", [(256, 8, 4, 8), (160, 8, 3, 6), (72, 8, 2, 5),
                                                 (64, 32, 5, 3), (64, 2, 1, 8), (1024, 16, 2, 32),
                                                 (12, 4, 4, 6), (32, 32, 7, 7), (250, 2, 1, 3)])
def test_groups(ops, scoring, E, n_group, keep, topk):
    for dtype in (torch.float32, torch.bfloat16):
        logits, bias = make(61, E, dtype, E + n_group)
        for top in (1, 2):
            for b in (None, bias):
                check(ops, logits, topk, scoring=scoring, bias=b, n_group=n_group, topk_group=keep,
                      group_top=top, renormalize=True)


def test_many_tokens_share_a_warp(ops):
    """Long batches run several tokens through a warp and weigh them together."""
    logits, bias = make(30_011, 64, torch.float32, 5)
    kw = dict(scoring="sigmoid", bias=bias, n_group=4, topk_group=2, renormalize=True)
    mask = torch.rand(30_011, device="cuda") > 0.3
    w, ids = ops.moe_route(logits, 6, token_mask=mask, **kw)
    for lo in (0, 14_000, 29_980):
        part = slice(lo, lo + 31)
        rw, rid = R.route(logits[part], 6, token_mask=mask[part], **kw)
        assert torch.equal(ids[part].cpu().long(), rid)
        assert ((w[part].double().cpu() - rw).abs() <= rw * REL).all()
    for lo in range(0, 30_011, 700):                       # rows do not depend on their batch
        part = slice(lo, min(lo + 700, 30_011))
        w1, id1 = ops.moe_route(logits[part], 6, token_mask=mask[part], **kw)
        assert torch.equal(w1, w[part]) and torch.equal(id1, ids[part])


@pytest.mark.parametrize("kw", [{}, {"scoring": "sigmoid"}, {"scoring": "sigmoid", "bias": True},
                                {"bias": True}, {"n_group": 4, "topk_group": 2},
                                {"n_group": 4, "topk_group": 2, "scoring": "sigmoid", "bias": True}])
def test_equal_and_nearly_equal_keys(ops, kw):
    """Ties go to the lower id; keys that differ in their last bits keep their order."""
    E = 128
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randint(0, 4, (200, E), generator=g, device="cuda").float()
    z[50:100] = 1.0                                            # all equal
    z[100:150] += 3e-7 * torch.randint(0, 3, (50, E), generator=g, device="cuda")
    z[150:] = 2.0 + torch.rand(50, E, generator=g, device="cuda") * 1e-6
    kw = dict(kw)
    if kw.pop("bias", False):
        kw["bias"] = torch.where(torch.arange(E, device="cuda") % 3 == 0, 0.25, 0.25 + 6e-8)
    for topk in (1, 8, 32):
        check(ops, z, topk, **kw)
        check(ops, z.bfloat16(), topk, **kw)


def test_closed_experts_and_empty_rows(ops):
    z, bias = make(12, 64, torch.float32, 9)
    low = torch.finfo(torch.float32).min
    z[0] = -math.inf                                           # nothing open
    z[1] = math.nan
    z[2, 3:] = -math.inf                                       # three open, topk 6
    z[3] = low                                                 # masked with the lowest value
    z[4, 10:] = low
    z[5, ::2] = math.nan
    z[6, 7] = math.inf
    z[7, [4, 9]] = math.inf
    z[8] = -200.0                                              # sigmoids underflow
    z[9] = 90.0
    z[10] = -0.0
    z[10, 5] = 0.0
    mask = torch.ones(12, dtype=torch.bool, device="cuda")
    mask[11] = False
    closing = bias.clone()
    closing[0], closing[1] = -math.inf, math.nan
    for scoring in ("softmax", "sigmoid"):
        for renorm in (False, True):
            for b in (None, bias, closing):
                w, ids = check(ops, z, 6, scoring=scoring, renormalize=renorm, bias=b,
                               token_mask=mask)
                assert (ids[[0, 1, 11]] == -1).all() and (w[[0, 1, 11]] == 0).all()
                assert torch.isfinite(w).all()
                check(ops, z, 6, scoring=scoring, renormalize=renorm, bias=b, n_group=4,
                      topk_group=2, token_mask=mask)
    _, ids = ops.moe_route(z, 6, token_mask=torch.zeros_like(mask))
    assert (ids == -1).all()


def test_strided_logits_and_no_tokens(ops):
    big, _ = make(50, 131, torch.float32, 2)
    for view in (big[:, :128], big[:, 1:129], big[::2, 3:]):
        check(ops, view, 5)
    w, ids = ops.moe_route(big[:0], 5)
    assert w.shape == (0, 5) and ids.shape == (0, 5)
    flat = big.bfloat16().flatten()
    check(ops, flat[1:1 + 40 * 64].view(40, 64), 4, scoring="sigmoid")


def test_ids_feed_the_permutation(ops):
    z, _ = make(300, 16, torch.bfloat16, 4)
    mask = torch.arange(300, device="cuda") < 271
    w, ids = ops.moe_route(z, 3, token_mask=mask)
    _, offs, _ = ops.moe_permute(ids, 16)
    assert int(offs[-1]) == 271 * 3
    counts = torch.bincount(ids[:271].flatten().long(), minlength=16)
    assert torch.equal(offs[1:] - offs[:-1], counts.int())


# ------------------------------------------------------------------ gradients

def check_grad(ops, logits, ids, grad, scoring, renorm, scale=2.5):
    got = ops.moe_route_backward(grad, logits, ids, scoring=scoring, renormalize=renorm, scale=scale)
    want = R.route_grad(grad, logits, ids, scoring, renorm, scale)
    assert got.dtype == logits.dtype and got.shape == logits.shape
    size = scale * torch.where(ids >= 0, grad, 0).abs().sum(1, keepdim=True).double().cpu()
    p = R.scores(R.clean(logits), scoring)
    if renorm:                                             # the chosen weights, in their places
        at = torch.where((ids >= 0) & (ids < logits.shape[1]), ids, -1).cpu().long()
        own = R.weights(R.clean(logits), at, scoring, True, 1.0)
        p = torch.zeros_like(p).scatter_add_(1, at.clamp(min=0), own)
    t = logits.dtype
    bound = want.abs() * R.half_step(t) + 2 * p * size * REL + R.smallest(t) + 1e-37
    assert ((got.double().cpu() - want).abs() <= bound).all()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
@pytest.mark.parametrize("T,E,topk", [(1, 1, 1), (5, 3, 2), (41, 60, 4), (130, 256, 8), (3, 1024, 32),
                                      (7, 500, 5), (12, 384, 1)])
def test_gradient(ops, dtype, scoring, renorm, T, E, topk):
    logits, _ = make(T, E, dtype, 3 * T + E)
    _, ids = ops.moe_route(logits, topk, scoring=scoring)
    grad = torch.randn(T, topk, device="cuda")
    got = check_grad(ops, logits, ids, grad, scoring, renorm)
    if renorm or scoring == "sigmoid":                     # zero where nothing was chosen
        open_ = torch.ones(T, E, dtype=torch.bool, device="cuda").scatter_(1, ids.long(), False)
        assert (got[open_] == 0).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_gradient_of_odd_ids(ops, scoring, renorm):
    """Repeated ids add up, ids outside the experts and closed experts count for nothing."""
    logits, _ = make(6, 40, torch.float32, 1)
    logits[4] = -math.inf
    logits[5, 7] = -math.inf
    ids = torch.tensor([[3, 3, 3, 5, -1], [0, 39, 0, 39, 40], [-1] * 5, [1, 2, 3, 4, 2 ** 30],
                        [1, 2, 3, 4, 5], [7, 8, 7, 9, 10]], dtype=torch.int32, device="cuda")
    grad = torch.randn(6, 5, device="cuda")
    got = ops.moe_route_backward(grad, logits, ids, scoring=scoring, renormalize=renorm, scale=2.0)
    want = R.route_grad(grad, logits, ids, scoring, renorm, 2.0)
    assert ((got.double().cpu() - want).abs() <= 12 * grad.abs().max().item() * REL).all()
    assert (got[2] == 0).all() and (got[4] == 0).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_gradient_against_differences(ops, scoring, renorm):
    """sum(g w) along a direction: the central difference with h = 2^-6 is off by
    h^2 / 6 of a third derivative (below 4 sum|g| here: scores and their first
    three derivatives are below 1) and by the weights' roundings over h."""
    T, E, topk, h = 20, 24, 4, 2.0 ** -6
    logits, _ = make(T, E, torch.float32, 12)
    _, ids = ops.moe_route(logits, topk, scoring=scoring)
    grad, along = torch.randn(T, topk, device="cuda"), torch.randn(T, E, device="cuda").clamp(-1, 1)
    dz = ops.moe_route_backward(grad, logits, ids, scoring=scoring, renormalize=renorm, scale=1.5)

    def at(z):
        """The weights of the chosen ids, whatever their order at z."""
        w, i = ops.moe_route(z, E, scoring=scoring)
        full = torch.zeros_like(z).scatter_(1, i.long(), w).gather(1, ids.long()).double()
        if renorm:
            full = full / full.sum(1, keepdim=True)
        return 1.5 * full

    up, down = logits + h * along, logits - h * along
    step = (up.double() - down.double()) / 2
    want = (grad.double() * (at(up) - at(down))).sum(1) / 2
    got = (dz.double() * step).sum(1)
    size = 1.5 * grad.abs().double().sum(1)
    assert ((got - want).abs() <= size * (4 * h ** 3 + 2 * REL)).all()


def test_more_than_2_to_the_31_logits(ops):
    T, E = 2_097_160, 1024
    logits = torch.zeros(T, E, dtype=torch.bfloat16, device="cuda")
    logits[-8:] = torch.randn(8, E, device="cuda")
    tail = logits[-8:].clone()
    w, ids = ops.moe_route(logits, 4)
    w1, id1 = ops.moe_route(tail, 4)
    assert torch.equal(w[-8:], w1) and torch.equal(ids[-8:], id1)
    assert torch.equal(ids[0].cpu(), torch.arange(4, dtype=torch.int32))
    grad = torch.randn(T, 4, device="cuda")
    got = ops.moe_route_backward(grad, logits, ids)
    want = ops.moe_route_backward(grad[-8:].contiguous(), tail, id1)
    assert torch.equal(got[-8:], want)


def test_capture_two_streams_and_repeat(ops):
    logits, bias = make(4000, 256, torch.float32, 21)
    kw = dict(scoring="sigmoid", bias=bias, n_group=8, topk_group=4, renormalize=True)
    grad = torch.randn(4000, 8, device="cuda")
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            w, ids = ops.moe_route(logits, 8, **kw)
            dz = ops.moe_route_backward(grad, logits, ids, scoring="sigmoid", renormalize=True)
        graphs.append((g, (w, ids, dz)))
    logits.copy_(make(4000, 256, torch.float32, 22)[0])
    w, ids = ops.moe_route(logits, 8, **kw)
    want = (w, ids, ops.moe_route_backward(grad, logits, ids, scoring="sigmoid", renormalize=True))
    torch.cuda.synchronize()
    for g, _ in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        for a, b in zip(out, want):
            assert torch.equal(a, b)


def test_refusals(ops):
    from ferret_b200._lib import FerretError
    z, bias = make(8, 64)
    mask = torch.ones(8, dtype=torch.bool, device="cuda")
    for f in (lambda: ops.moe_route(z.int(), 4), lambda: ops.moe_route(z.t(), 4),
              lambda: ops.moe_route(z[0], 4), lambda: ops.moe_route(z, 4, scoring="relu"),
              lambda: ops.moe_route(z, 4, bias=bias[:-1]),
              lambda: ops.moe_route(z, 4, bias=bias.half()),
              lambda: ops.moe_route(z, 4, bias=bias.cpu()),
              lambda: ops.moe_route(z, 4, token_mask=mask[:-1]),
              lambda: ops.moe_route(z, 4, token_mask=mask.int()),
              lambda: ops.moe_route(z[:1].expand(8, 64), 4)):
        with pytest.raises((ValueError, TypeError)):
            f()
    for kw in (dict(topk=65), dict(topk=0), dict(topk=33), dict(topk=4, n_group=3),
               dict(topk=4, n_group=128), dict(topk=4, n_group=8, topk_group=9),
               dict(topk=4, n_group=8, topk_group=0), dict(topk=9, n_group=8, topk_group=1),
               dict(topk=4, n_group=8, topk_group=2, group_top=3)):
        with pytest.raises((FerretError, RuntimeError)):
            ops.moe_route(z, **kw)
    with pytest.raises(FerretError):
        ops.moe_route(torch.zeros(2, 1025, device="cuda"), 4)
    _, ids = ops.moe_route(z, 4)
    g = torch.zeros(8, 4, device="cuda")
    for f in (lambda: ops.moe_route_backward(g[:, :3], z, ids),
              lambda: ops.moe_route_backward(g.half(), z, ids),
              lambda: ops.moe_route_backward(g, z, ids.long()),
              lambda: ops.moe_route_backward(g, z[:4], ids),
              lambda: ops.moe_route_backward(g, z, ids[0])):
        with pytest.raises((ValueError, TypeError)):
            f()
