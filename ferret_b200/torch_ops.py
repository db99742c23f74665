"""Torch operator registrations: ``torch.ops.ferret_moe.*``.

The reference's kernels are reached from torch code either through ctypes
shims or as TORCH_LIBRARY operators (examples/tcgen05-gemm/matmul.cpp:73-95);
this module gives the library the operator form, with the tensor signatures
of the baselines it replaces:

* ``ferret_moe::fp8_grouped_gemm_nt_contiguous(Tensor a, Tensor a_scale,
  Tensor w, Tensor w_scale, Tensor(a!) out, Tensor m_indices, bool silu=False,
  bool disable_ue8m0_cast=True) -> ()`` -- DeepGEMM's
  m_grouped_fp8_gemm_nt_contiguous (baselines/fp8-group-gemm/baseline_dsv3_decode.py:55-57;
  ``disable_ue8m0_cast=False`` declares power-of-two scales);
* ``ferret_moe::per_token_cast_to_fp8(Tensor x, bool use_ue8m0=False) ->
  (Tensor, Tensor)`` (baseline_dsv3_decode.py:42);
* ``ferret_moe::moe_align_block_size(Tensor topk_ids, int block_size,
  int num_experts) -> (Tensor, Tensor, Tensor)``
  (baselines/kimi-moe-w13-int4/baseline_marlin.py:123-126);
* ``ferret_moe::int4_moe_w13(Tensor hidden, Tensor w_raw, Tensor w_scale,
  Tensor topk_ids, bool silu=True) -> Tensor`` -- the raw compressed-tensors
  INT4 weights ([E, K/8, N] int32, [E, K/32, N] bf16), repacked once per
  weight tensor pair (the last pair is cached, by identity and version), then
  moe_wna16_marlin_gemm + SiLU
  (baseline_marlin.py:140-168).

and, for the operators around the expert layer (no reference counterpart):

* ``ferret_moe::add_rms_norm(Tensor x, Tensor residual, Tensor weight, float
  eps=1e-6) -> (Tensor, Tensor)`` and ``add_rms_norm_fp8(..., bool
  use_ue8m0=False) -> (Tensor, Tensor, Tensor, Tensor)``;
* ``ferret_moe::moe_route(Tensor logits, int topk, ...) -> (Tensor weights,
  Tensor ids)`` and ``moe_balance_loss(Tensor logits, Tensor topk_ids, float
  coef, ...) -> (Tensor loss, Tensor counts, Tensor prob_sums, Tensor
  n_tokens)``, both differentiable in the logits (weights and loss; the other
  outputs carry no gradient);
* ``ferret_moe::int4_linear(Tensor x, Tensor w, Tensor w_scale, Tensor?
  w_zero=None, Tensor? bias=None) -> Tensor``.

The norms and ``int4_linear`` have no backward pass: a gradient that reaches
their results raises.
A second derivative through the router or the balance loss raises.  A
differentiable call of theirs is refused while its stream is being captured into
a CUDA graph, forward and backward: a captured backward pass that meets gradient
accumulators of an eager graph on another stream breaks the capture beyond
repair.  Captured training steps call ``ops.moe_route``,
``ops.moe_route_backward``, ``ops.moe_balance_loss`` and
``ops.moe_balance_loss_backward``, which record no autograd graph.

Every operator runs the CUDA library (CUDA tensors only); importing this
module registers them.
"""
from __future__ import annotations

import torch

from . import ops

_LIB = torch.library.Library("ferret_moe", "DEF")
_LIB.define("fp8_grouped_gemm_nt_contiguous(Tensor a, Tensor a_scale, Tensor w, Tensor w_scale, "
            "Tensor(a!) out, Tensor m_indices, bool silu=False, bool disable_ue8m0_cast=True) -> ()")
_LIB.define("per_token_cast_to_fp8(Tensor x, bool use_ue8m0=False) -> (Tensor, Tensor)")
_LIB.define("moe_align_block_size(Tensor topk_ids, int block_size, int num_experts) "
            "-> (Tensor, Tensor, Tensor)")
_LIB.define("int4_moe_w13(Tensor hidden, Tensor w_raw, Tensor w_scale, Tensor topk_ids, "
            "bool silu=True) -> Tensor")

# the last repacked INT4 weight set: (w_raw, w_scale, their versions, blob);
# holding the raw tensors keeps their memory from being reused by others
_INT4_CACHE: list = []


def _fp8_gemm(a, a_scale, w, w_scale, out, m_indices, silu=False, disable_ue8m0_cast=True):
    ops.m_grouped_fp8_gemm_nt_contiguous((a, a_scale), (w, w_scale), out, m_indices,
                                         disable_ue8m0_cast=disable_ue8m0_cast, silu=silu)


def _quant(x, use_ue8m0=False):
    return ops.per_token_cast_to_fp8(x, use_ue8m0=use_ue8m0)


def _align(topk_ids, block_size, num_experts):
    return ops.moe_align_block_size(topk_ids, block_size, num_experts)


def _int4(hidden, w_raw, w_scale, topk_ids, silu=True):
    versions = (w_raw._version, w_scale._version)
    if (_INT4_CACHE and _INT4_CACHE[0] is w_raw and _INT4_CACHE[1] is w_scale
            and _INT4_CACHE[2] == versions):
        packed = _INT4_CACHE[3]
    else:
        _INT4_CACHE.clear()          # one weight set at a time: repacks are GBs
        packed = ops.Int4W13Weights(w_raw, w_scale)
        _INT4_CACHE.extend([w_raw, w_scale, versions, packed])
    return ops.moe_wna16_w13(hidden, packed, topk_ids, silu=silu)


_LIB.impl("fp8_grouped_gemm_nt_contiguous", _fp8_gemm, "CUDA")
_LIB.impl("per_token_cast_to_fp8", _quant, "CUDA")
_LIB.impl("moe_align_block_size", _align, "CUDA")
_LIB.impl("int4_moe_w13", _int4, "CUDA")


# ----------------------------------------------------- around the expert layer

_LIB.define("add_rms_norm(Tensor x, Tensor residual, Tensor weight, float eps=1e-6) "
            "-> (Tensor, Tensor)")
_LIB.define("add_rms_norm_fp8(Tensor x, Tensor residual, Tensor weight, float eps=1e-6, "
            "bool use_ue8m0=False) -> (Tensor, Tensor, Tensor, Tensor)")
_LIB.define("moe_route(Tensor logits, int topk, str scoring='softmax', Tensor? bias=None, "
            "int n_group=1, int topk_group=1, int group_top=2, bool renormalize=False, "
            "float scale=1.0, Tensor? token_mask=None) -> (Tensor, Tensor)")
_LIB.define("moe_balance_loss(Tensor logits, Tensor topk_ids, float coef, str scoring='softmax', "
            "Tensor? token_mask=None) -> (Tensor, Tensor, Tensor, Tensor)")
_LIB.define("int4_linear(Tensor x, Tensor w, Tensor w_scale, Tensor? w_zero=None, "
            "Tensor? bias=None) -> Tensor")


def _norm(x, residual, weight, eps=1e-6):
    return ops.add_rms_norm(x, weight, residual, eps)[:2]


def _norm_fp8(x, residual, weight, eps=1e-6, use_ue8m0=False):
    return ops.add_rms_norm(x, weight, residual, eps, quant=True, use_ue8m0=use_ue8m0)


def _route(logits, topk, scoring="softmax", bias=None, n_group=1, topk_group=1, group_top=2,
           renormalize=False, scale=1.0, token_mask=None):
    return ops.moe_route(logits, topk, scoring=scoring, bias=bias, n_group=n_group,
                         topk_group=topk_group, group_top=group_top, renormalize=renormalize,
                         scale=scale, token_mask=token_mask)


def _balance(logits, topk_ids, coef, scoring="softmax", token_mask=None):
    return ops.moe_balance_loss(logits, topk_ids, coef, scoring=scoring, token_mask=token_mask)


def _int4_linear(x, w, w_scale, w_zero=None, bias=None):
    return ops.int4_linear(x, w, w_scale, w_zero=w_zero, bias=bias)


def _not_captured(name):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"torch.ops.ferret_moe.{name} does not record gradients inside a CUDA "
                           f"graph capture: capture ops.{name} and ops.{name}_backward instead")


class _Once(torch.autograd.Function):
    """A backward function's result, tied to what it was formed from.  With
    create_graph=True a second derivative through it raises; as a plain tensor it
    would count as a constant."""

    @staticmethod
    def forward(ctx, name, backward, *inputs):
        ctx.name = name
        return backward(*inputs)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"torch.ops.ferret_moe.{ctx.name} can be differentiated once only: its "
                           "backward pass has no gradient of its own")


def _route_setup(ctx, inputs, output):
    _not_captured("moe_route")
    logits, _, scoring, _, _, _, _, renormalize, scale, _ = inputs
    _, ids = output
    ctx.mark_non_differentiable(ids)
    ctx.save_for_backward(logits, ids)
    ctx.form = dict(scoring=scoring, renormalize=renormalize, scale=scale)


def _route_backward(ctx, grad_weights, _):
    _not_captured("moe_route")
    logits, ids = ctx.saved_tensors
    grad = None
    if grad_weights is not None:
        grad = _Once.apply("moe_route", lambda g, z: ops.moe_route_backward(
            g.contiguous(), z, ids, **ctx.form), grad_weights, logits)
    return grad, *[None] * 9


def _balance_setup(ctx, inputs, output):
    _not_captured("moe_balance_loss")
    logits, topk_ids, coef, scoring, token_mask = inputs
    _, counts, prob_sums, n_tokens = output
    ctx.mark_non_differentiable(counts, prob_sums, n_tokens)
    ctx.save_for_backward(logits, counts, n_tokens, token_mask)
    ctx.form = (topk_ids.shape[1], coef, scoring)


def _balance_backward(ctx, grad_loss, *_):
    _not_captured("moe_balance_loss")
    logits, counts, n_tokens, token_mask = ctx.saved_tensors
    topk, coef, scoring = ctx.form
    grad = None
    if grad_loss is not None:
        grad = _Once.apply("moe_balance_loss", lambda g, z: ops.moe_balance_loss_backward(
            g.contiguous(), z, counts, n_tokens, topk, coef, scoring=scoring,
            token_mask=token_mask), grad_loss, logits)
    return grad, None, None, None, None


def _no_backward(name):
    def backward(ctx, *_):
        raise RuntimeError(f"torch.ops.ferret_moe.{name} has no backward pass: call it under "
                           "torch.no_grad(), or on detached tensors, where no gradient has to go "
                           "through it")
    return backward


_LIB.impl("add_rms_norm", _norm, "CUDA")
_LIB.impl("add_rms_norm_fp8", _norm_fp8, "CUDA")
_LIB.impl("moe_route", _route, "CUDA")
_LIB.impl("moe_balance_loss", _balance, "CUDA")
_LIB.impl("int4_linear", _int4_linear, "CUDA")
torch.library.register_autograd("ferret_moe::moe_route", _route_backward,
                                setup_context=_route_setup, lib=_LIB)
torch.library.register_autograd("ferret_moe::moe_balance_loss", _balance_backward,
                                setup_context=_balance_setup, lib=_LIB)
for _name in ("add_rms_norm", "add_rms_norm_fp8", "int4_linear"):
    torch.library.register_autograd(f"ferret_moe::{_name}", _no_backward(_name), lib=_LIB)
