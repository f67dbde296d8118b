"""Layer norm on HIP, beside the RMSNorm of ``moe_sublayer``.

``layer_norm`` is ``torch.nn.functional.layer_norm`` over the last dimension,
forward and backward, in fp32 arithmetic; ``moe_sublayer`` calls it for a block
whose norm is a ``torch.nn.LayerNorm``. Eager calls are one autograd node in C++
(``csrc/autograd.cpp``); under ``torch.compile`` they are the custom ops
``pmoe::layer_norm_fwd`` and ``pmoe::layer_norm_bwd``, which trace without graph
breaks.
"""

from __future__ import annotations

import torch

from . import ops
from ._lib import nodes, on_device, require_gpu, stream_of
from .moe import _empty_like_none, _refuse_capture, _stage


@torch.library.custom_op("pmoe::layer_norm_fwd", mutates_args=(),
                         schema="(Tensor x, Tensor? weight, Tensor? bias, float eps, ScalarType out_dtype) -> "
                                "(Tensor, Tensor)")
def _layer_norm_fwd(x, weight, bias, eps, out_dtype):
    with _stage("layernorm"):
        return ops.layernorm_forward(x, weight, bias, eps, out_dtype)


@_layer_norm_fwd.register_fake
def _(x, weight, bias, eps, out_dtype):
    return torch.empty_like(x, dtype=out_dtype), x.new_empty(2, x.numel() // x.shape[-1], dtype=torch.float32)


@torch.library.custom_op("pmoe::layer_norm_bwd", mutates_args=(),
                         schema="(Tensor grad, Tensor x, Tensor? weight, Tensor? bias, Tensor stats, bool[] needs) -> "
                                "(Tensor, Tensor, Tensor)")
def _layer_norm_bwd(grad, x, weight, bias, stats, needs):
    _refuse_capture("layer_norm_bwd")
    dt = next((p.dtype for p in (weight, bias) if p is not None), torch.float32)
    with _stage("layernorm_bwd"):
        got = ops.layernorm_backward(grad, x, weight, stats, dt, *needs)
    return tuple(g if g is not None else _empty_like_none(x) for g in got)


@_layer_norm_bwd.register_fake
def _(grad, x, weight, bias, stats, needs):
    return tuple(torch.empty_like(t) if need else _empty_like_none(x) for need, t in zip(needs, (x, weight, bias)))


def _setup(ctx, inputs, output):
    x, weight, bias, _eps, _out_dtype = inputs
    _out, stats = output
    ctx.save_for_backward(x, weight, bias, stats)
    ctx.mark_non_differentiable(stats)
    ctx.set_materialize_grads(False)


def _autograd(ctx, grad, _gs):
    if grad is None:
        return (None,) * 5
    x, weight, bias, stats = ctx.saved_tensors
    needs = [bool(n) for n in ctx.needs_input_grad[:3]]
    got = torch.ops.pmoe.layer_norm_bwd(grad.contiguous(), x, weight, bias, stats, needs)
    return (*(g if need else None for g, need in zip(got, needs)), None, None)


_layer_norm_fwd.register_autograd(_autograd, setup_context=_setup)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``torch.nn.functional.layer_norm(x, (H,), weight, bias, eps)`` over the last
    dimension of ``x`` (..., H), any H, in fp32 arithmetic.

    ``x``, ``weight`` and ``bias`` are fp32, bf16 or fp16; parameters of two
    types are both taken in fp32. The result has ``x``'s type, or ``out_dtype``
    (16 bits from fp32 ``x``: what the 16-bit products of the block read, without
    a cast between). Unlike torch's, it does not follow autocast. Gradients reach
    ``x`` and the parameters; a second derivative and forward-mode differentiation are
    refused, and so is a backward under HIP graph capture.
    """
    assert x.dim() >= 1 and x.shape[-1] >= 1, "layer_norm expects (..., H)"
    H = x.shape[-1]
    for name, p in (("weight", weight), ("bias", bias)):
        assert p is None or tuple(p.shape) == (H,), f"layer_norm: {name} {tuple(p.shape)}, expected ({H},)"
    require_gpu(x, weight, bias)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    assert out_dtype == x.dtype or (x.dtype == torch.float32 and out_dtype in (torch.bfloat16, torch.float16)), (
        f"layer_norm: {out_dtype} from {x.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        weight, bias = weight.float(), bias.float()
    x, weight, bias = (t if t is None or t.is_contiguous() else t.contiguous() for t in (x, weight, bias))
    if torch.compiler.is_compiling():
        return torch.ops.pmoe.layer_norm_fwd(x, weight, bias, float(eps), out_dtype)[0]
    with _stage("layernorm"), on_device(x):
        return nodes().layer_norm(x, weight, bias, float(eps), out_dtype, stream_of(x))
