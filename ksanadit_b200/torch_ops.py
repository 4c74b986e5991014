"""``torch.library`` registrations of the contractions and of the operators around a gated feed-forward, so that code traced by ``torch.compile`` (KsanaDiT
breaks the graph at its attention op, ksana/operations/attention/attention_op.py:72) sees them as opaque
operators with known output shapes instead of ctypes calls it cannot trace:

    torch.ops.ksana_b200.fp8_linear(x, weight_e4m3, weight_scale, bias)  -> [..., N] in x.dtype
    torch.ops.ksana_b200.sage_attention(q, k, v)                        -> [L, H, 128] in q.dtype
    torch.ops.ksana_b200.gated_linear(x, w_gate, w_up, b_gate, b_up, act)  -> [..., F] in x.dtype
    torch.ops.ksana_b200.sandwich_norm(x, y, gate, scale, shift, post_weight, pre_weight, residual_scale, kind, eps) -> (r, h) like x
    torch.ops.ksana_b200.w4_linear(x, weight, weight_scale, weight_zero, bias, out_features) -> [..., out_features] in x.dtype

The real implementations are the CUDA kernels (no CPU implementation is registered: calling the operators on CPU tensors raises); the fake
implementations only describe shapes and dtypes.  None has an autograd formula here: gradients are those of ``ops.gated_linear`` and
``ops.sandwich_norm``, called directly.  Where ``torch.jit.trace`` or ``make_fx`` records, the last three operators have to be called in this form, and their
namesakes in ``ops`` raise; ``sandwich_norm`` has no form here without ``y`` or without the norm behind the sum.
"""

from __future__ import annotations

import torch

from . import ops


@torch.library.custom_op("ksana_b200::fp8_linear", mutates_args=(), device_types="cuda")
def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """Per-token e4m3 quantisation of ``x`` + FP8 GEMM against ``weight`` [N, K] (e4m3) with per-channel scales."""
    shape = x.shape
    x2 = x.reshape(-1, shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    xq, sx = ops.quant_fp8_rowwise(x2)
    ws = weight_scale.float()
    ws = (ws.expand(weight.shape[0]) if ws.dim() == 0 else ws.reshape(weight.shape[0])).contiguous()
    out = ops.fp8_gemm(xq, sx, weight, ws, bias, out_dtype=x.dtype)
    return out.reshape(*shape[:-1], weight.shape[0])


@fp8_linear.register_fake
def _(x, weight, weight_scale, bias=None):
    return x.new_empty(*x.shape[:-1], weight.shape[0])


@torch.library.custom_op("ksana_b200::sage_attention", mutates_args=(), device_types="cuda")
def sage_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """q [Lq, H, 128], k / v [Lk, H, 128] (bf16 / fp16) -> [Lq, H, 128]; softmax scale 128^-0.5."""
    return ops.sage_attention(q, k, v)


@sage_attention.register_fake
def _(q, k, v):
    return q.new_empty(q.shape)


@torch.library.custom_op("ksana_b200::gated_linear", mutates_args=(), device_types="cuda")
def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: torch.Tensor | None = None, b_up: torch.Tensor | None = None,
                 act: str = "silu") -> torch.Tensor:
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up)."""
    with torch.no_grad():
        return ops.gated_linear(x, w_gate, w_up, b_gate, b_up, act)


@gated_linear.register_fake
def _(x, w_gate, w_up, b_gate=None, b_up=None, act="silu"):
    return x.new_empty(*x.shape[:-1], w_gate.shape[0])


@torch.library.custom_op("ksana_b200::sandwich_norm", mutates_args=(), device_types="cuda")
def sandwich_norm(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor | None = None, scale: torch.Tensor | None = None, shift: torch.Tensor | None = None,
                  post_weight: torch.Tensor | None = None, pre_weight: torch.Tensor | None = None, residual_scale: float = 1.0, kind: str = "rms",
                  eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """r = x + residual_scale * gate * N(y) * post_weight and the modulated norm of r."""
    with torch.no_grad():
        return ops.sandwich_norm(x, y, gate=gate, scale=scale, shift=shift, post_weight=post_weight, pre_weight=pre_weight, residual_scale=residual_scale,
                                 kind=kind, eps=eps)


@sandwich_norm.register_fake
def _(x, y, gate=None, scale=None, shift=None, post_weight=None, pre_weight=None, residual_scale=1.0, kind="rms", eps=1e-6):
    return x.new_empty(x.shape), x.new_empty(x.shape)


@torch.library.custom_op("ksana_b200::w4_linear", mutates_args=(), device_types="cuda")
def w4_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, weight_zero: torch.Tensor | None, bias: torch.Tensor | None,
              out_features: int) -> torch.Tensor:
    """x times a packed 4-bit weight with group scales."""
    with torch.no_grad():
        return ops.w4_linear(x, weight, weight_scale, weight_zero, bias, out_features)


@w4_linear.register_fake
def _(x, weight, weight_scale, weight_zero, bias, out_features):
    return x.new_empty(*x.shape[:-1], out_features)
