"""The operators together, as they are used: norm -> router -> experts on the norm's
FP8 rows -> combine, the balance loss of the same routing, and their operator
forms with gradients."""
import numpy as np
import pytest
import torch

import block_ref as R
from oracle import oracle as O

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda_device):
    from ferret_b200 import ops as _ops
    return _ops


def weights(E, H, I, seed=0):
    from ferret_b200 import data
    g = torch.Generator().manual_seed(seed)
    w13, s13 = data.per_block_cast_to_fp8(torch.randn(E, 2 * I, H, generator=g) * 0.02)
    w2, s2 = data.per_block_cast_to_fp8(torch.randn(E, H, I, generator=g) * 0.02)
    gate = (torch.randn(E, H, generator=g) * 0.05).to(torch.bfloat16)
    norm = (1 + 0.1 * torch.randn(H, generator=g)).to(torch.bfloat16)
    return [t.cuda() for t in (norm, gate, w13, s13, w2, s2)]


@pytest.mark.parametrize("T", [1, 37, 300])
def test_block_equals_its_parts(ops, T):
    E, H, I, topk = 16, 512, 256, 4
    norm, gate, w13, s13, w2, s2 = weights(E, H, I)
    x, r = (torch.randn(T, H, device="cuda").to(torch.bfloat16) for _ in range(2))
    mask = torch.arange(T, device="cuda") != 3
    kw = dict(scoring="sigmoid", renormalize=True, n_group=4, topk_group=2, scale=2.5,
              token_mask=mask)
    out, res, ids, logits = ops.fp8_moe_block(x, r, norm, gate, w13, s13, w2, s2, topk, **kw)
    y, res1, q, s = ops.add_rms_norm(x, norm, r, quant=True)
    assert torch.equal(res, res1)
    # router logits: fp32 sums of H products, against 64 bits
    exact = y.double() @ gate.double().t()
    size = y.double().abs() @ gate.double().abs().t()
    assert ((logits.double() - exact).abs() <= size * H * R.U).all()
    w, id1 = ops.moe_route(logits, topk, **kw)
    assert torch.equal(ids, id1)
    # The experts from the FP8 rows, step by step: each GEMM against the oracle on the
    # GPU's own input rows (a bf16 step of the first one's output can move its
    # e4m3 value by a whole step of 2^-3, so the bar holds per GEMM, not across
    # the quantization), and the block equal to the steps.
    rows, offs, mi = O.moe_permute(ids.cpu().numpy(), E)
    n = int(offs[-1])
    d_rows, d_offs, _ = ops.moe_permute(ids, E)
    assert np.array_equal(d_rows.cpu().numpy(), rows)
    a, a_s = ops.fp8_gather_rows(q, s, d_rows, topk)
    y1 = torch.zeros(T * topk, I, device="cuda", dtype=torch.bfloat16)
    ops.m_grouped_fp8_gemm_nt_contiguous((a, a_s), (w13, s13), y1, None, expert_offsets=d_offs,
                                         silu=True)
    q2, sc2 = ops.per_token_cast_to_fp8(y1)
    y2 = torch.zeros(T * topk, H, device="cuda", dtype=torch.bfloat16)
    ops.m_grouped_fp8_gemm_scatter((q2, sc2), (w2, s2), y2, d_offs, d_rows)
    assert torch.equal(ops.moe_combine(y2, w, ids, E), out)

    def close(got, a, a_s, w, w_s, silu):
        u8 = lambda t: t.cpu().view(torch.uint8).numpy()
        ref = O.fp8_grouped_gemm(u8(a)[:n], a_s.cpu().numpy()[:n], u8(w), w_s.cpu().numpy(), mi[:n],
                                 silu=silu)
        err = O.rel_err(got[:n].float().cpu().numpy(), ref)
        assert err["nan"] == 0 and err["max_rel"] < 1e-2, err

    if n:
        close(y1, a, a_s, w13, s13, True)
        close(y2[d_rows[:n].long()], q2, sc2, w2, s2, False)
    if T > 3:
        assert (out[3] == 0).all()
    assert ops.last_device_status() == 0


def test_block_without_residual_and_without_tokens(ops):
    E, H, I, topk = 8, 256, 128, 2
    p = weights(E, H, I, 1)
    x = torch.randn(5, H, device="cuda").to(torch.bfloat16)
    out, res, ids, logits = ops.fp8_moe_block(x, None, *p, topk)
    assert res is x and out.shape == (5, H) and torch.isfinite(out).all()
    out, _, ids, logits = ops.fp8_moe_block(x[:0], None, *p, topk)
    assert out.shape == (0, H) and ids.shape == (0, topk) and logits.shape == (0, E)


def test_block_replays_from_a_graph_with_the_balance_loss(ops):
    E, H, I, topk = 16, 512, 256, 4
    p = weights(E, H, I, 2)
    x, r = (torch.randn(200, H, device="cuda").to(torch.bfloat16) for _ in range(2))

    def step():
        out, res, ids, logits = ops.fp8_moe_block(x, r, *p, topk, renormalize=True)
        loss, counts, sums, n = ops.moe_balance_loss(logits, ids, 0.01)
        grad = ops.moe_balance_loss_backward(torch.ones((), device="cuda"), logits, counts, n, topk,
                                             0.01)
        return out, res, ids, logits, loss, counts, grad

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    x.copy_(torch.randn_like(x))
    g.replay()
    want = step()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # the counts are what the expert placement takes
    from ferret_b200 import ep
    assert sorted(ep.balanced_placement(got[5].cpu().long(), 4).tolist()) == list(range(E))


def test_fp8_gather_rows(ops):
    x = torch.randn(7, 256, device="cuda").to(torch.bfloat16)
    q, s = ops.per_token_cast_to_fp8(x)
    rows = torch.tensor([13, 0, -1, 6, 6], dtype=torch.int32, device="cuda")
    a, b = ops.fp8_gather_rows(q, s, rows, 2)
    src = [6, 0, None, 3, 3]
    for i, j in enumerate(src):
        if j is None:
            assert (a[i].float() == 0).all() and (b[i] == 0).all()
        else:
            assert torch.equal(a[i].view(torch.uint8), q[j].view(torch.uint8))
            assert torch.equal(b[i], s[j])


# ------------------------------------------------------------- operator forms

def test_operator_forms_match(ops):
    import ferret_b200.torch_ops  # noqa: F401
    F = torch.ops.ferret_moe
    x, r = (torch.randn(6, 256, device="cuda").to(torch.bfloat16) for _ in range(2))
    w = torch.rand(256, device="cuda").to(torch.bfloat16)
    for a, b in zip(F.add_rms_norm(x, r, w), ops.add_rms_norm(x, w, r)):
        assert torch.equal(a, b)
    for a, b in zip(F.add_rms_norm_fp8(x, r, w, 1e-5, True),
                    ops.add_rms_norm(x, w, r, 1e-5, quant=True, use_ue8m0=True)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    z, bias = torch.randn(50, 32, device="cuda"), torch.randn(32, device="cuda")
    got = F.moe_route(z, 4, "sigmoid", bias, 4, 2, 2, True, 2.0, None)
    want = ops.moe_route(z, 4, scoring="sigmoid", bias=bias, n_group=4, topk_group=2, group_top=2,
                         renormalize=True, scale=2.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    got = F.moe_balance_loss(z, want[1], 0.1)
    assert all(torch.equal(a, b) for a, b in zip(got, ops.moe_balance_loss(z, want[1], 0.1)))
    raw = torch.randint(-2 ** 31, 2 ** 31, (32, 64), device="cuda").to(torch.int32)
    sc = torch.rand(8, 64, device="cuda").to(torch.bfloat16)
    assert torch.equal(F.int4_linear(x, raw, sc), ops.int4_linear(x, raw, sc))


def test_a_training_step_of_the_router(ops):
    """A leaf's gradient through the gate, the weights and the balance loss, from
    autograd, against the explicit backward functions and 64 bits."""
    import ferret_b200.torch_ops  # noqa: F401
    F = torch.ops.ferret_moe
    T, H, E, topk = 64, 128, 24, 4
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(T, H, generator=g, device="cuda")
    gate = torch.randn(E, H, generator=g, device="cuda").mul_(0.1).requires_grad_(True)
    dw = torch.randn(T, topk, generator=g, device="cuda")
    mask = torch.rand(T, generator=g, device="cuda") > 0.2
    logits = x @ gate.t()
    w, ids = F.moe_route(logits, topk, "sigmoid", None, 1, 1, 2, True, 2.0, mask)
    loss, counts, sums, n = F.moe_balance_loss(logits, ids, 0.5, "sigmoid", mask)
    assert w.requires_grad and loss.requires_grad
    assert not (ids.requires_grad or counts.requires_grad or sums.requires_grad)
    ((w * dw).sum() + 3 * loss).backward()
    z = logits.detach()
    dz = ops.moe_route_backward(dw, z, ids, scoring="sigmoid", renormalize=True, scale=2.0) \
        + ops.moe_balance_loss_backward(torch.tensor(3.0, device="cuda"), z, counts, n, topk, 0.5,
                                        scoring="sigmoid", token_mask=mask)
    assert torch.allclose(gate.grad, dz.t() @ x, rtol=1e-5, atol=1e-5)
    exact = R.route_grad(dw, z, ids, "sigmoid", True, 2.0) \
        + R.balance(z, ids, 0.5, "sigmoid", mask, 3.0)[4]
    assert torch.allclose(dz.double().cpu(), exact, rtol=1e-4, atol=1e-5)
    # gradients of only one of the two, and of broadcast incoming gradients
    for one in (lambda w, loss: w.sum(), lambda w, loss: loss):
        z2 = z.clone().requires_grad_(True)
        w2, id2 = F.moe_route(z2, topk)
        l2 = F.moe_balance_loss(z2, id2, 0.5)[0]
        one(w2, l2).backward()
        assert torch.isfinite(z2.grad).all() and bool((z2.grad != 0).any())


def test_autograd_refuses_capture(ops):
    """Differentiable calls are refused inside a capture; the explicit functions and
    calls that record nothing are not."""
    import ferret_b200.torch_ops  # noqa: F401
    F = torch.ops.ferret_moe
    z = torch.randn(16, 8, device="cuda", requires_grad=True)
    F.moe_route(z, 2)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="moe_route_backward"):
        with torch.cuda.graph(g):
            F.moe_route(z, 2)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g), torch.no_grad():
        w, ids = F.moe_route(z, 2)
    g.replay()
    assert torch.equal(ids, ops.moe_route(z.detach(), 2)[1])


def test_block_refusals(ops):
    E, H, I, topk = 8, 256, 128, 2
    norm, gate, w13, s13, w2, s2 = weights(E, H, I, 3)
    x = torch.randn(5, H, device="cuda").to(torch.bfloat16)
    ok = (x, None, norm, gate, w13, s13, w2, s2)

    def call(i, t, **kw):
        args = list(ok)
        args[i] = t
        return lambda: ops.fp8_moe_block(*args, topk, **kw)

    for f in (call(0, x.float()), call(0, x[:, ::2]), call(1, x[:4]), call(2, norm[:-1]),
              call(3, gate[:-1]), call(3, gate.cpu()), call(4, w13[:, :, :128].contiguous()),
              call(5, s13[:, :1].contiguous()), call(6, w2[:, :128].contiguous()),
              call(7, s2[:4]), call(0, x, scoring="other"), call(0, x, bias=norm)):
        with pytest.raises((ValueError, TypeError)):
            f()
    assert ops.last_device_status() == 0
