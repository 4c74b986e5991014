"""Linears with 4-bit weights and group scales for the one-row products of a block (timestep embedding, modulation vectors).

A product with a row or a few only streams its weight, so the time is the weight's bytes: a B200W4Linear reads a little more than
half of what the FP8 class reads, and keeps as much less in memory.  KsanaDiT has no such class; this one follows the
contract of its Linears (constructor, ``forward`` on any number of leading axes, ``reset_parameters`` that initialises nothing).
Weights are frozen: there is no backward pass.
"""

from __future__ import annotations

import torch

from . import _lib, ops

TILE_N, TILE_K, TILE_BYTES = 16, 64, 512
GROUPS = (32, 64, 128)
_ORDER = [0, 2, 4, 6, 1, 3, 5, 7]  # eight neighbouring columns as the nibbles of a 32-bit word, lowest bits first
_BACK = [0, 4, 1, 5, 2, 6, 3, 7]


def _tiles(n: int, to: int) -> int:
    return -(-n // to)


def pack_w4(q: torch.Tensor) -> torch.Tensor:
    """Values 0..15 [N, K] (uint8) -> the packed weight [ceil(N/16), ceil(K/64), 512] that ``ops.w4_linear`` reads."""
    if q.dim() != 2 or q.dtype != torch.uint8:
        raise _lib.KsanaB200Error("pack_w4 needs a 2-D uint8 tensor")
    if q.numel() and int(q.max()) > 15:  # it would change its neighbour
        raise _lib.KsanaB200Error(f"pack_w4 needs values 0 .. 15, found {int(q.max())}")
    N, K = q.shape
    nt, kt = _tiles(N, TILE_N), _tiles(K, TILE_K)
    full = torch.full((nt * TILE_N, kt * TILE_K), 8, dtype=torch.uint8, device=q.device)
    full[:N, :K] = q
    t = full.view(nt, 2, 8, kt, 2, 4, 8).permute(0, 3, 2, 5, 4, 1, 6)[..., _ORDER]
    return (t[..., 0::2] | (t[..., 1::2] << 4)).reshape(nt, kt, TILE_BYTES).contiguous()


def unpack_w4(packed: torch.Tensor, N: int, K: int) -> torch.Tensor:
    """The values 0..15 [N, K] of a packed weight."""
    nt, kt = packed.shape[:2]
    b = packed.reshape(nt, kt, 8, 4, 2, 2, 4)
    q = torch.stack([b & 15, b >> 4], -1).flatten(-2)[..., _BACK]
    return q.permute(0, 5, 2, 1, 4, 3, 6).reshape(nt * TILE_N, kt * TILE_K)[:N, :K].contiguous()


def tile_groups(v: torch.Tensor) -> torch.Tensor:
    """A value per row and group [N, K/group] -> [ceil(N/16), K/group, 16], zeros behind the last row."""
    N, groups = v.shape
    full = torch.zeros(_tiles(N, TILE_N) * TILE_N, groups, dtype=v.dtype, device=v.device)
    full[:N] = v
    return full.view(-1, TILE_N, groups).transpose(1, 2).contiguous()


def untile_groups(v: torch.Tensor, N: int) -> torch.Tensor:
    return v.transpose(1, 2).reshape(-1, v.shape[1])[:N].contiguous()


def _scales(span: torch.Tensor, levels: int, dtype) -> torch.Tensor:
    """span / levels per group in ``dtype``: a group of zeros takes the least normal number, any would do.

    Below the normal numbers a step of the type is a large part of the scale.  One that was rounded down so far that its levels no longer reach
    the group's ends is taken a step up: a value is then never more than half a level off."""
    f = torch.finfo(dtype)
    least = f.smallest_normal * f.eps
    scale = (span / levels).to(dtype)
    if not bool(scale.isfinite().all()):
        raise _lib.KsanaB200Error(f"a group's scale is not finite in {dtype}: its weights are too large, or not finite themselves")
    # a group that the least scale cannot tell from zeros: that is nothing beside weights 4096 times as large, and else the weight is lost
    lost = (scale == 0) & (span > span.amax() / 4096) if span.numel() else scale != scale
    if bool(lost.any()):
        raise _lib.KsanaB200Error(f"the weights are too small for scales of {dtype}: use bfloat16 ones")
    scale = torch.where(scale.float() * (levels + 0.5) < span, (scale.float() + least).to(dtype), scale)
    return torch.where(span == 0, torch.full_like(scale, f.smallest_normal), scale)


@torch.no_grad()
def quantize_w4(w: torch.Tensor, group: int = 128, zeros: bool = False, dtype=torch.bfloat16):
    """Rounds a weight [N, K] to 4 bits per group of ``group`` columns -> (packed, scale, zero or None) as ``ops.w4_linear`` takes them.

    Without zero points a group's values are scale * (-7 .. 7), scale = absmax / 7; with them they reach from the group's least
    value (or 0) to its largest (or 0) in 15 steps.  The scale is rounded to ``dtype`` first and the values against the
    rounded one.  Raises where ``dtype`` has no scale for the weights: fp16 ones reach down to values of some 1e-7."""
    if w.dim() != 2 or group not in GROUPS or w.shape[1] % group != 0:
        raise _lib.KsanaB200Error(f"quantize_w4 needs a [N, K] weight whose K is in whole groups of {GROUPS}, got {tuple(w.shape)} and {group}")
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"expected bfloat16 or float16 scales, got {dtype}")
    N, K = w.shape
    wf = w.float().view(N, K // group, group)
    if zeros:
        low, high = wf.amin(-1).clamp(max=0), wf.amax(-1).clamp(min=0)
        scale = _scales(high - low, 15, dtype)
        zero = torch.round(-low / scale.float()).clamp(0, 15)
    else:
        scale = _scales(wf.abs().amax(-1), 7, dtype)
        zero = torch.full_like(scale, 8, dtype=torch.float32)
    q = torch.round(wf / scale.float()[..., None] + zero[..., None]).clamp(0, 15).to(torch.uint8).view(N, K)
    return pack_w4(q), tile_groups(scale), tile_groups(zero.to(torch.uint8)) if zeros else None


def dequantize_w4(packed, scale, zero, N: int, K: int) -> torch.Tensor:
    """The fp32 weight [N, K] that a packed one stands for."""
    groups = scale.shape[1]
    z = 8.0 if zero is None else untile_groups(zero, N).float()[..., None]
    q = unpack_w4(packed, N, K).float().view(N, groups, K // groups)
    return ((q - z) * untile_groups(scale, N).float()[..., None]).view(N, K)


class B200W4Linear(torch.nn.Module):
    """Linear with a packed 4-bit ``weight``, ``weight_scale`` and, with ``zeros``, ``weight_zero`` per group, and a ``bias``."""

    def __init__(self, in_features, out_features, bias=True, group=128, zeros=False, device=None, dtype=torch.bfloat16):
        super().__init__()
        if group not in GROUPS or in_features % group != 0:
            raise _lib.KsanaB200Error(f"in_features {in_features} must be in whole groups of {GROUPS}, got groups of {group}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"expected bfloat16 or float16, got {dtype}")
        self.in_features, self.out_features, self.group, self.compute_dtype = in_features, out_features, group, dtype
        nt, groups = _tiles(out_features, TILE_N), in_features // group

        def frozen(*shape, dtype):
            return torch.nn.Parameter(torch.empty(*shape, dtype=dtype, device=device), requires_grad=False)

        self.weight = frozen(nt, _tiles(in_features, TILE_K), TILE_BYTES, dtype=torch.uint8)
        self.weight_scale = frozen(nt, groups, TILE_N, dtype=dtype)
        self.weight_zero = frozen(nt, groups, TILE_N, dtype=torch.uint8) if zeros else None
        self.bias = frozen(out_features, dtype=dtype) if bias else None

    def reset_parameters(self):
        return None

    @classmethod
    def from_float(cls, linear: torch.nn.Linear, group=128, zeros=False, dtype=torch.bfloat16):
        """Quantises a high-precision Linear."""
        m = cls(linear.in_features, linear.out_features, linear.bias is not None, group, zeros, linear.weight.device, dtype)
        packed, scale, zero = quantize_w4(linear.weight.data, group, zeros, dtype)
        m.weight.data, m.weight_scale.data = packed, scale
        if zeros:
            m.weight_zero.data = zero
        if linear.bias is not None:
            m.bias.data = linear.bias.data.to(dtype)
        return m

    def dequantized(self) -> torch.Tensor:
        return dequantize_w4(self.weight.data, self.weight_scale.data, None if self.weight_zero is None else self.weight_zero.data,
                             self.out_features, self.in_features)

    def forward(self, input: torch.Tensor) -> torch.Tensor:  # noqa: A002
        return ops.w4_linear(input, self.weight, self.weight_scale, self.weight_zero, self.bias, out_features=self.out_features)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, group={self.group}, zeros={self.weight_zero is not None}, bias={self.bias is not None}"
