"""int4_linear against the definition in 64 bits.

Tolerance.  Products of an activation and an integer are exact; 32 of them are
added by the tensor core (each addition within 2^-23 of the sum of magnitudes),
the K / 32 block sums are scaled and added in fp32: below (K / 32 + 40) 2^-23 of
sum |x w|, the magnitudes of nibble - zero included, plus half a step of the
output's type."""
import pytest
import torch

import block_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(cuda_device):
    from ferret_b200 import ops as _ops
    return _ops


def make(T, K, N, group, dtype, zeros=False, bias=False, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + K + N)
    ints = lambda *s: torch.randint(-2 ** 31, 2 ** 31, s, generator=g, device="cuda").to(torch.int32)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    scale = (0.01 * torch.randn(K // group, N, generator=g, device="cuda")).to(dtype)
    return dict(x=x, w=ints(K // 8, N), w_scale=scale,
                w_zero=ints(K // group, N // 8) if zeros else None,
                bias=torch.randn(N, generator=g, device="cuda").to(dtype) if bias else None)


def check(y, a):
    ref, size = R.int4(a["x"], a["w"], a["w_scale"], a["w_zero"], a["bias"])
    K = a["x"].shape[1]
    t = a["x"].dtype
    assert y.dtype == t and y.shape == ref.shape
    bound = ref.abs() * (R.half_step(t) + 2 * R.U) + size * (K / 32 + 40) * 2 ** -23 + R.smallest(t)
    assert ((y.double().cpu() - ref).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("zeros,bias", [(False, False), (True, True)])
@pytest.mark.parametrize("T,K,N,group", [
    (1, 32, 8, 32), (1, 7168, 4096, 32), (3, 64, 16, 64), (8, 512, 128, 128), (9, 96, 136, 96),
    (16, 1024, 264, 32), (17, 2048, 1000, 128), (32, 4096, 520, 64), (33, 256, 72, 256),
    (70, 544, 40, 32), (5, 960, 200, 160), (2, 16384, 64, 128), (1, 2080, 2056, 2080),
    (4, 1536, 24, 96), (12, 4096, 7176, 128)])
def test_sizes(ops, dtype, zeros, bias, T, K, N, group):
    a = make(T, K, N, group, dtype, zeros, bias)
    check(ops.int4_linear(**a), a)


def test_every_nibble_and_column(ops):
    """One-hot activations read the dequantized matrix back, exactly."""
    K, N = 64, 48
    a = make(K, K, N, 32, torch.float16, zeros=True)
    a["x"] = torch.eye(K, device="cuda", dtype=torch.float16)
    a["w_scale"] = torch.full((2, N), 0.5, device="cuda", dtype=torch.float16)
    ref, _ = R.int4(a["x"], a["w"], a["w_scale"], a["w_zero"])
    assert torch.equal(ops.int4_linear(**a).double().cpu(), ref)


def test_matches_the_expert_kernel(ops):
    """One expert, one slot: the same weights through moe_wna16_w13, whose weights
    are rounded to bf16 after scaling (2^-9 each)."""
    from ferret_b200 import data
    raw, scale = data.int4_weights(1, 512, 1024, device="cuda")
    x = data.activations(4, 1024).cuda()
    y = ops.int4_linear(x, raw[0], scale[0])
    ids = torch.zeros(4, 1, dtype=torch.int32, device="cuda")
    z = ops.moe_wna16_w13(x, ops.Int4W13Weights(raw, scale), ids, silu=False)
    _, size = R.int4(x, raw[0], scale[0])
    assert ((y.double() - z.double()).cpu().abs() <= size * 2 ** -8 + 1e-6).all()


def test_strided_rows_out_and_neighbours(ops):
    a = make(6, 512, 264, 64, torch.bfloat16, bias=True)
    big = torch.randn(6, 520 + 512, device="cuda").to(torch.bfloat16)
    a["x"] = big[:, 8:520]
    out = torch.full((10, 264), 3.0, device="cuda", dtype=torch.bfloat16)
    y = ops.int4_linear(**a, out=out[2:8])
    assert y.data_ptr() == out[2:8].data_ptr()
    check(y, a)
    assert (out[:2] == 3).all() and (out[8:] == 3).all()


def test_special_activations(ops):
    a = make(9, 256, 64, 32, torch.bfloat16)
    want = ops.int4_linear(**a)
    a["x"][4, 7], a["x"][6] = float("nan"), 0
    got = ops.int4_linear(**a)
    assert torch.isnan(got[4]).all() and (got[6] == 0).all()
    keep = [0, 1, 2, 3, 5, 7, 8]
    assert torch.equal(got[keep], want[keep])


def test_no_tokens(ops):
    a = make(1, 64, 16, 32, torch.bfloat16)
    a["x"] = a["x"][:0]
    assert ops.int4_linear(**a).shape == (0, 16)


def test_repeats_captures_and_streams(ops):
    a = make(16, 7168, 2048, 32, torch.bfloat16)
    want = ops.int4_linear(**a)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = ops.int4_linear(**a)
        graphs.append((g, y))
    torch.cuda.synchronize()
    for g, _ in graphs:
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                g.replay()
    torch.cuda.synchronize()
    for _, y in graphs:
        assert torch.equal(y, want)
    assert ops.last_device_status() == 0


def test_more_than_2_to_the_31_words(ops):
    K, N = 16384, (1 << 20) + 8
    w = torch.zeros(K // 8, N, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    w[:, -8:] = torch.randint(-2 ** 31, 2 ** 31, (K // 8, 8), generator=g, device="cuda").to(torch.int32)
    scale = torch.full((K // 128, N), 0.01, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(1, K, generator=g, device="cuda").to(torch.bfloat16)
    y = ops.int4_linear(x, w, scale)
    a = dict(x=x, w=w[:, -8:], w_scale=scale[:, -8:], w_zero=None, bias=None)
    check(y[:, -8:], a)


def test_refusals(ops):
    from ferret_b200._lib import FerretError
    a = make(4, 256, 64, 64, torch.bfloat16, zeros=True, bias=True)

    def call(**kw):
        return lambda: ops.int4_linear(**dict(a, **kw))

    x, w = a["x"], a["w"]
    for f in (call(x=x.float()), call(x=x.half()), call(x=x[:, :248].contiguous()), call(x=x.t()),
              call(x=x[:1].expand(4, 256)), call(w=w.long()), call(w=w[:, ::2]),
              call(w_scale=a["w_scale"][:3]), call(w_scale=a["w_scale"][:, :-1]),
              call(w_scale=a["w_scale"].half()), call(w_zero=a["w_zero"][:, :-1]),
              call(bias=a["bias"].float()), call(bias=a["bias"][:-1]), call(w=w.cpu()),
              call(out=torch.empty(4, 63, device="cuda", dtype=torch.bfloat16)),
              call(out=torch.empty(64, 4, device="cuda", dtype=torch.bfloat16).t())):
        with pytest.raises((ValueError, TypeError)):
            f()
    narrow = dict(w=w[:, :60].contiguous(), w_scale=a["w_scale"][:, :60].contiguous(), w_zero=None,
                  bias=None)
    wide = torch.randn(4, 268, device="cuda").to(torch.bfloat16)
    for f in (call(**narrow), call(x=wide[:, 1:257]), call(x=wide[:, 4:260]),
              call(w_scale=torch.ones(16, 64, device="cuda", dtype=torch.bfloat16), w_zero=None)):
        with pytest.raises(FerretError):
            f()
