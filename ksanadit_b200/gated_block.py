"""The gated feed-forward half of a modulated transformer block with a norm on either side of it.

    shift, scale, gate = modulation(silu(temb))                    4-bit weights: a row or a few only stream them
    h = N(x) * pre_norm * (1 + scale) + shift
    y = down(act(h w_gate^T + b_gate) * (h w_up^T + b_up))
    x = x + residual_scale * gate * N(y) * post_norm

KsanaDiT's own blocks (ksana/models/wan/wan_model.py:317-321, ksana/models/qwen/transformer.py:225-234) have a plain GELU
feed-forward and no norm behind a half: this module is for models beside them.  In a stack of halves the norm behind one and the norm
ahead of the next are one pass over the tokens.  Everything but the 4-bit modulation is differentiable (an embedding that needs a
gradient through it is refused), so the same module is fine-tuned and served; for serving, ``down`` may be a ``B200Fp8Linear``.
"""

from __future__ import annotations

import torch

from . import _lib, ops
from .w4 import B200W4Linear


class B200GatedFeedForward(torch.nn.Module):
    """``modulation``: whether the half has its own 4-bit modulation Linear (else the caller passes the three vectors)."""

    def __init__(self, dim, hidden_dim, bias=False, act="silu", kind="rms", eps=1e-6, residual_scale=1.0, modulation=True, group=128, device=None,
                 dtype=torch.bfloat16):
        super().__init__()
        if act not in ops.ACTIVATIONS:
            raise _lib.KsanaB200Error(f"act must be one of {sorted(ops.ACTIVATIONS)}, got {act!r}")
        self.dim, self.hidden_dim, self.act, self.kind, self.eps, self.residual_scale = dim, hidden_dim, act, kind, eps, residual_scale

        def parameter(*shape, dtype=dtype):
            return torch.nn.Parameter(torch.empty(*shape, device=device, dtype=dtype))

        self.w_gate, self.w_up = parameter(hidden_dim, dim), parameter(hidden_dim, dim)
        self.b_gate, self.b_up = (parameter(hidden_dim), parameter(hidden_dim)) if bias else (None, None)
        self.down = torch.nn.Linear(hidden_dim, dim, bias=bias, device=device, dtype=dtype)
        self.pre_norm, self.post_norm = (torch.nn.Parameter(torch.ones(dim, device=device, dtype=torch.float32)) for _ in range(2))
        self.modulation = B200W4Linear(dim, 3 * dim, True, group, device=device, dtype=dtype) if modulation else None

    def vectors(self, temb):
        """(shift, scale, gate), [B, 1, dim] each, of the timestep embedding [B, dim].  The 4-bit weights are frozen, and their product
        has no backward pass: an embedding that needs a gradient is refused (detach it where the gradient through the modulation is not wanted)."""
        if self.modulation is None:
            raise _lib.KsanaB200Error("this half has no modulation of its own: pass its vectors")
        return self.modulation(torch.nn.functional.silu(temb))[:, None].chunk(3, -1)

    def inner(self, h):
        """The half between its norms."""
        return self.down(ops.gated_linear(h, self.w_gate, self.w_up, self.b_gate, self.b_up, act=self.act))

    def forward(self, x, temb=None, vectors=None):
        """x [B, L, dim] -> the same after this half.  ``vectors``: (shift, scale, gate) in place of ``temb``."""
        return gated_stack([self], x, temb, None if vectors is None else [vectors])


def gated_stack(halves, x, temb=None, vectors=None):
    """Runs the halves one after the other on x [B, L, dim]; the norm behind one and the norm ahead of the next share a pass.
    ``vectors``: a (shift, scale, gate) per half, in place of ``temb``."""
    if vectors is None:
        vectors = [half.vectors(temb) for half in halves]
    if len(vectors) != len(halves):
        raise _lib.KsanaB200Error(f"{len(halves)} halves need as many (shift, scale, gate), got {len(vectors)}")
    for a, b in zip(halves, halves[1:]):
        if (a.kind, a.eps, a.dim) != (b.kind, b.eps, b.dim):
            raise _lib.KsanaB200Error("neighbouring halves share a pass: they need one kind of norm, one eps and one width")
    if not halves:
        return x
    shift, scale, gate = vectors[0]
    half = halves[0]
    x, h = ops.sandwich_norm(x, scale=scale, shift=shift, pre_weight=half.pre_norm, kind=half.kind, eps=half.eps)
    for i, half in enumerate(halves):
        y = half.inner(h)
        behind = dict(gate=gate, post_weight=half.post_norm, residual_scale=half.residual_scale, kind=half.kind, eps=half.eps)
        if i + 1 == len(halves):
            return ops.sandwich_norm(x, y, pre=False, **behind)[0]
        shift, scale, next_gate = vectors[i + 1]
        x, h = ops.sandwich_norm(x, y, scale=scale, shift=shift, pre_weight=halves[i + 1].pre_norm, **behind)
        gate = next_gate
