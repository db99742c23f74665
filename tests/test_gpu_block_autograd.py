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


@pytest.mark.parametrize("op", [route, balance])
def test_a_captured_backward_pass_is_refused(F, op):
    """Of a forward pass recorded before the capture on the same stream; the process and
    the leaf go on."""
    z = torch.randn(6, 8, device="cuda", requires_grad=True)
    want, = torch.autograd.grad(op(F, z).sum(), z)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = op(F, z)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="_backward instead"):
        with torch.cuda.graph(graph, stream=side):
            torch.autograd.grad(out.sum(), z)
    torch.cuda.synchronize()
    again, = torch.autograd.grad(op(F, z).sum(), z)
    assert torch.equal(again, want)


# ------------------------------------------------ operators without a backward

def norm_inputs():
    x, r = (torch.randn(5, 256, device="cuda").to(torch.bfloat16) for _ in range(2))
    return [x, r, (1 + 0.1 * torch.randn(256, device="cuda")).to(torch.bfloat16)]


def int4_inputs():
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randint(-2 ** 31, 2 ** 31, (32, 64), generator=g, device="cuda").to(torch.int32)
    return [torch.randn(5, 256, device="cuda").to(torch.bfloat16),
            torch.rand(8, 64, device="cuda").to(torch.bfloat16),
            torch.randn(64, device="cuda").to(torch.bfloat16)], w


def bare(ops, F):
    def int4(f, t, w):
        return f(t[0], w, t[1], None, t[2])
    return {
        "norm": (norm_inputs, lambda t: ops.add_rms_norm(t[0], t[2], t[1])[:2]),
        "norm fp8": (norm_inputs, lambda t: ops.add_rms_norm(t[0], t[2], t[1], quant=True)),
        "norm only fp8": (norm_inputs, lambda t: ops.add_rms_norm(t[0], t[2], t[1], quant=True,
                                                                  normed=False)),
        "norm out": (norm_inputs, lambda t: ops.add_rms_norm(
            t[0], t[2], t[1], residual_out=torch.empty(7, 256, device="cuda",
                                                       dtype=torch.bfloat16)[1:6])),
        "op norm": (norm_inputs, lambda t: F.add_rms_norm(t[0], t[1], t[2])),
        "op norm fp8": (norm_inputs, lambda t: F.add_rms_norm_fp8(t[0], t[1], t[2])),
        "int4": (int4_inputs, lambda t, w: ops.int4_linear(t[0], w, t[1], bias=t[2])),
        "int4 out": (int4_inputs, lambda t, w: ops.int4_linear(
            t[0], w, t[1], bias=t[2], out=torch.empty(5, 64, device="cuda", dtype=torch.bfloat16))),
        "op int4": (int4_inputs, lambda t, w: F.int4_linear(t[0], w, t[1], None, t[2])),
    }


FORMS = ["norm", "norm fp8", "norm only fp8", "norm out", "op norm", "op norm fp8", "int4",
         "int4 out", "op int4"]


def flat(out):
    return [t for t in (out if isinstance(out, (list, tuple)) else [out]) if t is not None]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_gradient_that_would_be_lost_raises(ops, F, form, which):
    make, call = bare(ops, F)[form]
    made = make()
    inputs, more = made if isinstance(made, tuple) else (made, None)
    run = (lambda t: call(t)) if more is None else (lambda t: call(t, more))
    want = flat(run(inputs))
    assert not any(t.requires_grad for t in want)
    inputs[which] = inputs[which].requires_grad_(True)
    got = flat(run(inputs))                                # the forward pass runs as ever
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.equal(a.detach().view(torch.uint8), b.view(torch.uint8))
    for out in got:
        with pytest.raises(RuntimeError, match="no backward"):     # another path does not hide it
            (out.float().sum() + inputs[which].float().sum()).backward()
        inputs[which].grad = None
    with torch.no_grad():
        assert not any(t.requires_grad for t in flat(run(inputs)))


def test_a_written_output_keeps_its_identity(ops):
    x, r, w = norm_inputs()
    w.requires_grad_(True)
    out = ops.add_rms_norm(x, w, r, residual_out=r)
    assert out[1] is r and r.requires_grad
    big = torch.zeros(9, 256, device="cuda", dtype=torch.bfloat16)
    x, r, _ = norm_inputs()
    out = ops.add_rms_norm(x, w, r, residual_out=big[2:7])
    assert out[1].data_ptr() == big[2:7].data_ptr()
    with pytest.raises(RuntimeError, match="no backward"):
        big.float().sum().backward()


def test_the_whole_layer(ops):
    from test_gpu_moe_block import weights
    E, H, I, topk = 8, 256, 128, 2
    norm, gate, w13, s13, w2, s2 = weights(E, H, I, 4)
    x, r = (torch.randn(6, H, device="cuda").to(torch.bfloat16) for _ in range(2))
    rest = (w13, s13, w2, s2, topk)
    want = ops.fp8_moe_block(x, r, norm, gate, *rest)
    for which in range(4):
        args = [t.clone() for t in (x, r, norm, gate)]
        args[which].requires_grad_(True)
        got = ops.fp8_moe_block(*args, *rest)
        for a, b in zip(got, want):
            assert torch.equal(a.detach(), b)
        for out in (got[0], got[1], got[3]):
            with pytest.raises(RuntimeError, match="no backward"):
                (out.float().sum() + args[which].float().sum()).backward()
    for which in (1, 3):                                   # the scales of the experts' weights
        moved = list(rest)
        moved[which] = moved[which].clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="no backward"):
            ops.fp8_moe_block(x, r, norm, gate, *moved)[0].float().sum().backward()
    x.requires_grad_(True)
    out, res, _, logits = ops.fp8_moe_block(x, None, norm, gate, *rest)
    assert res is x
    with pytest.raises(RuntimeError, match="no backward"):
        out.float().sum().backward()


# ----------------------------------------------------- tensors written in place

def written_calls(ops):
    x, r, w = norm_inputs()
    (a, scale, bias), q = int4_inputs()
    return {
        "residual_out": (5, 256, lambda out: ops.add_rms_norm(x, w, r, residual_out=out)),
        "residual": (5, 256, lambda out: ops.add_rms_norm(x, w, out, residual_out=out)),
        "x": (5, 256, lambda out: ops.add_rms_norm(out, w, r, residual_out=out)),
        "out": (5, 64, lambda out: ops.int4_linear(a, q, scale, bias=bias, out=out)),
    }


WRITTEN = ["residual_out", "residual", "x", "out"]


@pytest.mark.parametrize("what", WRITTEN)
def test_autograd_sees_that_a_tensor_was_written(ops, what):
    rows, cols, call = written_calls(ops)[what]
    leaf = torch.randn(rows, cols, device="cuda").to(torch.bfloat16).requires_grad_(True)
    for inside in (torch.no_grad(), torch.enable_grad()):
        h = leaf * 1
        later = (h * h).sum()                              # saves h
        before = h._version
        with inside:
            call(h)
        assert h._version > before
        with pytest.raises(RuntimeError, match="inplace"):
            later.backward()
    plain = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    before = plain._version
    call(plain)
    assert plain._version > before


@pytest.mark.parametrize("what", WRITTEN)
def test_leaves_are_not_written_while_autograd_records(ops, what):
    rows, cols, call = written_calls(ops)[what]
    leaf = torch.randn(rows, cols, device="cuda").to(torch.bfloat16).requires_grad_(True)
    big = torch.randn(rows + 2, cols, device="cuda").to(torch.bfloat16).requires_grad_(True)
    for t, whole in ((leaf, leaf), (big[1:-1], big)):
        before = whole.detach().clone()
        with pytest.raises(RuntimeError, match="leaf"):
            call(t)
        assert torch.equal(whole.detach(), before)
    with torch.no_grad():
        call(leaf)                                         # as an optimizer's step would
        call(big[1:-1])
    with torch.inference_mode():
        inner = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
        call(inner)
    call(inner)


def test_written_tensors_that_overlap_inputs_are_refused(ops):
    """Only refusals here, and neighbours without a shared byte."""
    K = 128
    buf = torch.randn(64 * K, device="cuda").to(torch.bfloat16)
    w = torch.ones(K, device="cuda", dtype=torch.bfloat16)
    r = torch.randn(4, K, device="cuda").to(torch.bfloat16)
    rows = lambda at, n=4, step=K: buf.as_strided((n, K), (step, 1), at)
    x = rows(0)
    for out in (rows(8), rows(K), rows(3 * K), rows(4 * K - 1)):
        for first, second in ((x, r), (r, x)):
            with pytest.raises(ValueError, match="overlap"):
                ops.add_rms_norm(first, w, second, residual_out=out)
    with pytest.raises(ValueError, match="overlap"):       # the same start, other rows
        ops.add_rms_norm(rows(0, step=2 * K), w, r, residual_out=x)
    with pytest.raises(ValueError, match="overlap"):
        ops.add_rms_norm(r, buf[K:2 * K], r.clone(), residual_out=x)
    with pytest.raises(ValueError, match="overlap"):       # between two rows, one byte too far
        ops.add_rms_norm(rows(0, step=5 * K), w, r, residual_out=rows(K + 1))
    for first, out in ((rows(0, step=5 * K), rows(K)), (x, x), (x, rows(4 * K))):
        want = ops.add_rms_norm(first.clone(), w, r)
        got = ops.add_rms_norm(first, w, r, residual_out=out)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    q = torch.zeros(K // 8, K, dtype=torch.int32, device="cuda")
    scale = torch.ones(4, K, device="cuda", dtype=torch.bfloat16)
    x = rows(0)
    half = lambda t: t.view(torch.bfloat16).flatten()[:4 * K].view(4, K)
    for kw, out in ((dict(x=x, w=q, w_scale=scale), x), (dict(x=x, w=q, w_scale=scale), rows(8)),
                    (dict(x=r, w=q, w_scale=scale), half(q)),
                    (dict(x=r, w=q, w_scale=scale), scale),
                    (dict(x=r, w=q, w_scale=scale, bias=buf[:K]), x)):
        with pytest.raises(ValueError, match="overlap"):
            ops.int4_linear(**kw, out=out)
    assert ops.int4_linear(x, q, scale, out=rows(4 * K)).shape == (4, K)
