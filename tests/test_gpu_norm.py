"""add_rms_norm against the definition in 64 bits.

Tolerances.  s = x + residual is rounded once in fp32 (2^-24), the sum of the
squares of up to 32768 terms runs through at most 32 terms of a thread, 5
levels of a warp and 5 of the warps (42 roundings and those of the squares,
halved by the square root), the root, the quotient, two products: below
32 * 2^-24 relative.  An output adds half a step of its type.  An e4m3 value is
off by 2^-4 of itself or, among its subnormals, by 2^-10 of its scale."""
import numpy as np
import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu
FP32 = 32 * R.U


@pytest.fixture(scope="module")
def ops(cuda_device):
    from ferret_b200 import ops as _ops
    return _ops


def make(T, K, dtype, seed=0, residual=True, weight=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x = (f(T, K) * torch.exp(f(K))).to(dtype)
    r = (3 * f(T, K)).to(dtype) if residual else None
    return x, (1 + 0.2 * f(K)).to(weight or dtype), r


def check(out, x, w, r, eps=1e-6, quant=False):
    y, ro, q, s = out
    ry, rs = R.norm(x, w, r, eps)
    t = x.dtype
    if y is not None:
        assert y.dtype == t and y.shape == x.shape and y.is_contiguous()
        bound = ry.abs() * (R.half_step(t) + FP32) + R.smallest(t)
        assert ((y.double().cpu() - ry).abs() <= bound).all()
    if r is None:
        assert ro is None
    else:
        assert ((ro.double().cpu() - rs).abs()
                <= rs.abs() * (R.half_step(t) + R.U) + R.smallest(t)).all()
    if not quant:
        assert q is None and s is None
        return
    T, K = x.shape
    b = ry.reshape(T, K // 128, 128)
    amax = b.abs().amax(2).clamp(min=float(np.float32(1e-4)))
    assert ((s.double().cpu() - amax / 448).abs() <= amax / 448 * (FP32 + 2 * R.U)).all()
    got = q.double().cpu().reshape(b.shape) * s.double().cpu()[:, :, None]
    bound = torch.maximum(b.abs() * 2.0 ** -4, amax[:, :, None] / 448 * 2.0 ** -10)
    assert ((got - b).abs() <= bound * (1 + 1e-5) + b.abs() * FP32).all()


DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K", [(1, 1), (3, 7), (5, 128), (2, 1000), (7, 1001), (33, 4096),
                                 (1, 7168), (1300, 100), (2500, 1024), (1301, 1032), (1, 32768),
                                 (1200, 2048), (1190, 7168), (301, 8193)])
def test_norm_sizes(ops, dtype, T, K):
    x, w, r = make(T, K, dtype, T + K)
    check(ops.add_rms_norm(x, w, r), x, w, r)
    check(ops.add_rms_norm(x, w), x, w, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K", [(1, 128), (5, 640), (64, 7168), (1300, 256), (2000, 1024),
                                 (1200, 7168), (1290, 1152)])
def test_norm_fp8(ops, dtype, T, K):
    x, w, r = make(T, K, dtype, T * 3 + K)
    check(ops.add_rms_norm(x, w, r, quant=True), x, w, r, quant=True)
    out = ops.add_rms_norm(x, w, quant=True, normed=False)
    assert out[0] is None
    check(out, x, w, None, quant=True)


@pytest.mark.parametrize("ue8m0", [False, True])
@pytest.mark.parametrize("T", [3, 1300])
def test_fp8_is_the_quantizer_of_the_unrounded_norm(ops, ue8m0, T):
    """With fp32 in and out y is the value that was quantized, so the bytes and
    scales follow from it bit for bit."""
    from ferret_b200 import data
    x, w, r = make(T, 768, torch.float32, 4)
    x[0], r[0] = 0, 0                                  # a block below the clamp
    y, _, q, s = ops.add_rms_norm(x, w, r, quant=True, use_ue8m0=ue8m0)
    b = y.cpu().reshape(T, 6, 128)
    amax = b.abs().amax(2).clamp(min=1e-4)
    scale = data.ceil_pow2(amax / 448.0) if ue8m0 else amax / 448.0
    f = torch.reciprocal(scale) if ue8m0 else torch.reciprocal(amax) * 448.0
    want = (b * f[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(s.cpu(), scale)
    assert torch.equal(q.cpu().view(torch.uint8).reshape(T, 6, 128), want.view(torch.uint8))


def test_fp32_weight_eps_and_zero_rows(ops):
    x, w, r = make(9, 512, torch.bfloat16, 1, weight=torch.float32)
    check(ops.add_rms_norm(x, w, r, 0.1), x, w, r, eps=0.1)
    z = torch.zeros_like(x)
    y, ro, q, s = ops.add_rms_norm(z, w, z.clone(), quant=True)
    assert (y == 0).all() and (ro == 0).all() and (q.float() == 0).all()


@pytest.mark.parametrize("T", [4, 1250])
def test_strided_and_unaligned_rows(ops, T):
    K = 1024
    big = torch.randn(T, 3 * K + 8, device="cuda").to(torch.bfloat16)
    w = torch.rand(K, device="cuda").to(torch.bfloat16)
    for x, r in ((big[:, :K], big[:, K:2 * K]),              # aligned, strided
                 (big[:, 1:K + 1], big[:, 8:K + 8]),         # odd start
                 (big[:, :K].contiguous(), big[:, 3:K + 3])):
        check(ops.add_rms_norm(x, w, r, quant=True), x, w, r, quant=True)
    flat = torch.randn(T * K + 3, device="cuda").to(torch.bfloat16)
    x = flat[3:].view(T, K)                                  # contiguous at an odd address
    check(ops.add_rms_norm(x, w, None, quant=True), x, w, None, quant=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,K", [(1, 32768), (3, 32761), (1, 5), (1300, 33), (1300, 1021), (40, 4099)])
@pytest.mark.parametrize("start", [0, 1, 3, 7])
def test_rows_that_share_their_distance_from_a_boundary(ops, dtype, T, K, start):
    """Odd row lengths and odd base addresses: every row starts somewhere else, the
    same in x, residual and (when given) residual_out."""
    def at(seed):
        flat = make(1, T * K + 8, dtype, seed)[0].flatten()
        return flat[start:start + T * K].view(T, K)

    x, r, w = at(1), at(2), make(1, K, dtype, 3)[1]
    check(ops.add_rms_norm(x, w, r), x, w, r)
    out = at(4)
    before = out.clone()
    check(ops.add_rms_norm(x, w, r, residual_out=out), x, w, r)
    check(ops.add_rms_norm(x, w), x, w, None)
    assert not torch.equal(before, out)


@pytest.mark.parametrize("T,K", [(3, 640), (1400, 2048), (1400, 513)])
def test_residual_in_place(ops, T, K):
    x, w, r = make(T, K, torch.bfloat16, 8)
    y0, r0, _, _ = ops.add_rms_norm(x, w, r)
    r1 = r.clone()
    y1, out, _, _ = ops.add_rms_norm(x, w, r1, residual_out=r1)
    assert out is r1 and torch.equal(r1, r0) and torch.equal(y1, y0)
    x1 = x.clone()
    y2, _, _, _ = ops.add_rms_norm(x1, w, r, residual_out=x1)
    assert torch.equal(x1, r0) and torch.equal(y2, y0)


def test_rows_around_are_left_alone(ops):
    x, w, r = make(5, 384, torch.bfloat16, 3)
    big = torch.full((9, 384), 7.0, device="cuda", dtype=torch.bfloat16)
    ops.add_rms_norm(x, w, r, residual_out=big[2:7])
    assert (big[:2] == 7).all() and (big[7:] == 7).all()


def test_no_rows(ops):
    x = torch.empty(0, 256, device="cuda", dtype=torch.bfloat16)
    y, ro, q, s = ops.add_rms_norm(x, torch.ones(256, device="cuda", dtype=torch.bfloat16), x,
                                   quant=True)
    assert y.shape == (0, 256) and ro.shape == (0, 256) and q.shape == (0, 256) and s.shape == (0, 2)


def test_nan_and_inf_stay_in_their_row(ops):
    x, w, r = make(1200, 2048, torch.bfloat16, 6)
    want = ops.add_rms_norm(x, w, r, quant=True)
    x[1, 5], x[3, 6] = float("nan"), float("inf")
    got = ops.add_rms_norm(x, w, r, quant=True)
    assert torch.isnan(got[0][1]).all() and torch.isnan(got[0][3, 6])
    keep = torch.ones(1200, dtype=torch.bool, device="cuda")
    keep[1] = keep[3] = False
    for a, b in zip(got, want):
        assert torch.equal(a[keep].view(torch.uint8), b[keep].view(torch.uint8))


def test_more_than_2_to_the_31_elements(ops):
    T, K = 300_001, 7168
    x = torch.randn(1, K, device="cuda").to(torch.bfloat16).expand(T, K).contiguous()
    x[-1] = torch.randn(K, device="cuda")
    w = torch.rand(K, device="cuda").to(torch.bfloat16)
    y, _, q, s = ops.add_rms_norm(x, w, quant=True)
    tail = x[-2:].clone()
    check((y[-2:], None, q[-2:], s[-2:]), tail, w, None, quant=True)


def test_captured_on_a_side_stream_and_replayed(ops):
    T, K = 1300, 2048
    x, w, r = make(T, K, torch.bfloat16, 2)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.add_rms_norm(x, w, r, quant=True)
        graphs.append((g, out))
    x.copy_(make(T, K, torch.bfloat16, 77)[0])
    want = ops.add_rms_norm(x, w, r, quant=True)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for (g, _), s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
            g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        for a, b in zip(out, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_refusals(ops):
    x, w, r = make(4, 256, torch.bfloat16)
    bad = [
        lambda: ops.add_rms_norm(x, w[:-1], r),
        lambda: ops.add_rms_norm(x, w, r[:, :-1]),
        lambda: ops.add_rms_norm(x, w, r.float()),
        lambda: ops.add_rms_norm(x, w.half(), r),
        lambda: ops.add_rms_norm(x, w.cpu(), r),
        lambda: ops.add_rms_norm(x.t(), w, None),
        lambda: ops.add_rms_norm(x[:1].expand(4, 256), w, None),
        lambda: ops.add_rms_norm(x[:, :100].contiguous(), w[:100], None, quant=True),
        lambda: ops.add_rms_norm(x, w, None, normed=False),
        lambda: ops.add_rms_norm(x, w, None, residual_out=r),
        lambda: ops.add_rms_norm(x, w, r, residual_out=r[:, ::2]),
        lambda: ops.add_rms_norm(x.int(), w, None),
        lambda: ops.add_rms_norm(x[0], w, None),
    ]
    for f in bad:
        with pytest.raises((ValueError, TypeError)):
            f()
    from ferret_b200._lib import FerretError
    big = torch.zeros(1, 32776, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(FerretError):
        ops.add_rms_norm(big, big[0], None)
    with pytest.raises(FerretError):
        ops.add_rms_norm(x, w, r, -1.0)
    assert ops.last_device_status() == 0
