"""Microscaled 4-bit tensors and the expert product that reads them.

``mx_quantize`` turns float tensors into :class:`MXTensor`: groups of 32
consecutive values share one power-of-two scale, and each value is held in 4
bits (0, 0.5, 1, 1.5, 2, 3, 4 or 6 times the scale, with a sign). Expert
weights kept this way take 17/64 of their bf16 bytes, and the sm_100a tensor
cores multiply them without unpacking, at nominally four times the bf16 rate
(measured in the product's kernel: 3.5 PFLOP/s, twice a bf16 library product's).

    w_up_mx = mx_quantize(w_up, dim=-2)         # [E, K, N], once, at load
    y = cvmm_mx(x, sel, w_up_mx)                # as cvmm(x, sel, w_up), forward only

The product quantises its input rows itself, so both sides are 4-bit; sums are
held in 32 bits. It is a serving operator: it has no backward. No reference
counterpart (the reference computes in 16 and 32 bits only).
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from ._torch_ops import calls as ops
from .api import CVMMSel, has_tangent

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


class MXTensor:
    """A microscaled 4-bit tensor of logical ``shape``, quantised along ``dim`` (-1 or -2).

    With K the size along dim, and the rows everything else (dim=-1: all
    leading axes flattened into one batch of rows; dim=-2: the last axis, one
    batch per leading index):

    data:  uint8 [*leading, rows, 16 * ceil(K / 32)], two values to a byte, the
           lower index in the lower half, zeros past K (dim=-1: leading axes
           unflattened, [*shape[:-1], 16 * ceil(K / 32)]);
    scale: uint8 [*leading, ceil(rows / 128), ceil(K / 128), 32, 4, 4], the scale
           2^(byte - 127) of row r, group j at [r // 128, j // 4, r % 32,
           r % 128 // 32, j % 4]; 255 marks a group that held an infinity or
           NaN; bytes of rows and groups that do not exist are 0.
    """

    __slots__ = ("data", "scale", "shape", "dim")

    def __init__(self, data: torch.Tensor, scale: torch.Tensor, shape, dim: int = -1):
        self.shape = shape = torch.Size(shape)
        self.data, self.scale, self.dim = data, scale, dim
        want_data, want_scale = mx_shapes(shape, dim)
        if data.shape != want_data or scale.shape != want_scale or data.dtype != torch.uint8 or scale.dtype != torch.uint8:
            raise ValueError(f"MXTensor: shape {tuple(shape)} quantised along dim {dim} has uint8 data {want_data} and "
                             f"scale {want_scale}; got {data.dtype} {tuple(data.shape)} and {scale.dtype} "
                             f"{tuple(scale.shape)}")
        if not (data.is_contiguous() and scale.is_contiguous()):
            raise ValueError("MXTensor: data and scale must be contiguous")
        if data.device != scale.device:
            raise ValueError("MXTensor: data and scale must be on one device")

    @property
    def device(self) -> torch.device:
        return self.data.device

    def to(self, device) -> "MXTensor":
        return MXTensor(self.data.to(device), self.scale.to(device), self.shape, self.dim)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values, rounded to ``dtype`` (exact in float32)."""
        if dtype not in _FLOATS:
            raise ValueError(f"MXTensor.dequantize: unsupported dtype {dtype}")
        return ops.mx_dequantize(self.data, self.scale, list(self.shape), self.dim, dtype)

    def __repr__(self) -> str:
        return f"MXTensor(shape={tuple(self.shape)}, dim={self.dim}, device={self.device})"


def mx_shapes(shape, dim: int = -1):
    """Shapes of the data and scale tensors of an MXTensor."""
    return ops.mx_shapes(shape, dim)


def mx_quantize(x: torch.Tensor, dim: int = -1) -> MXTensor:
    """Microscaled 4-bit copy of ``x`` (float32, float16 or bfloat16, any strides), groups of 32 along ``dim``.

    dim=-1 for rows, dim=-2 for expert weights [E, K, N] (the axis a product
    sums over). The scale of a group is 2^(floor(log2 max|x|) - 2); values are
    rounded to the nearest 4-bit value, ties to even, and held at 6 times the
    scale. Not differentiable: the result carries no graph."""
    if x.dtype not in _FLOATS:
        raise ValueError(f"mx_quantize: unsupported dtype {x.dtype}")
    if dim not in (-1, -2) or x.dim() < -dim:
        raise ValueError(f"mx_quantize: dim must be -1 or -2 of a tensor that has it, got {dim} for {tuple(x.shape)}")
    q = MXTensor.__new__(MXTensor)  # nothing to check
    q.data, q.scale = ops.mx_quantize(x.detach() if x.requires_grad else x, dim)
    q.shape, q.dim = x.shape, dim
    return q


def cvmm_mx(x: torch.Tensor, sel: Union[torch.Tensor, CVMMSel], keys: MXTensor,
            weights: Optional[torch.Tensor] = None) -> torch.Tensor:
    """cvmm(x, sel, keys) with 4-bit microscaled expert weights, forward only.

    x: [..., K] token rows, [..., k, K] one row per route, or [..., H, K] with k
    a multiple of H (k / H consecutive routes share a row); float32, float16 or
    bfloat16, quantised to 4 bits inside. sel: expert ids [..., k] (int32 or
    int64), or a CVMMSel, whose raw_sel and reduction_weight are used. keys:
    mx_quantize(w, dim=-2) of w [E, K, N]. weights: [..., k] route weights of the
    weighted sum over k. Returns [..., k, N], or [..., N] with weights, in
    autocast's dtype, else x's (bfloat16 for a float32 x). Route outputs and
    their weighted sum are held in 32 bits and rounded to that dtype once."""
    if isinstance(sel, CVMMSel):
        if weights is not None and sel.reduction_weight is not None:
            raise ValueError("cvmm_mx: weights given twice (argument and CVMMSel.reduction_weight)")
        weights = sel.reduction_weight if weights is None else weights
        sel = sel.raw_sel
    if not isinstance(keys, MXTensor) or len(keys.shape) != 3 or keys.dim != -2:
        raise ValueError("cvmm_mx: keys must be an MXTensor of shape [E, K, N] quantised along dim=-2")
    if x.dtype not in _FLOATS:
        raise ValueError(f"cvmm_mx: unsupported x dtype {x.dtype}")
    if sel.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"cvmm_mx: sel must be int32 or int64, got {sel.dtype}")
    E, K, N = keys.shape
    if x.dim() < 1 or x.shape[-1] != K:
        raise ValueError(f"cvmm_mx: x feature size {tuple(x.shape)[-1:]} != keys.shape[1] {K}")
    if sel.dim() < 1 or sel.shape[-1] < 1:
        raise ValueError("cvmm_mx: sel must be [..., k] with k >= 1")
    lead, k = tuple(sel.shape[:-1]), sel.shape[-1]
    rows = tuple(x.shape[:-1])
    if rows != lead and not (len(rows) == len(lead) + 1 and rows[:-1] == lead and rows[-1] > 0 and k % rows[-1] == 0):
        raise ValueError(f"cvmm_mx: x rows {rows} match neither the tokens {lead} nor the routes {(*lead, k)} of sel")
    if weights is not None and (tuple(weights.shape) != tuple(sel.shape) or weights.dtype not in _FLOATS):
        raise ValueError(f"cvmm_mx: weights must be a float tensor of sel's shape {tuple(sel.shape)}, "
                         f"got {weights.dtype} {tuple(weights.shape)}")
    device = x.device
    if sel.device != device or keys.data.device != device or (weights is not None and weights.device != device):
        raise ValueError(f"cvmm_mx: x is on {device}, sel on {sel.device}, keys on {keys.device}"
                         + ("" if weights is None else f", weights on {weights.device}"))
    if torch.is_grad_enabled() and (x.requires_grad or (weights is not None and weights.requires_grad)):
        raise RuntimeError("cvmm_mx has no backward: call it under torch.no_grad() or detach its inputs")
    if has_tangent(x) or (weights is not None and has_tangent(weights)):
        raise NotImplementedError("cvmm_mx has no forward-mode derivative")
    if torch.is_autocast_enabled("cuda"):
        out_dtype = torch.get_autocast_dtype("cuda")
    else:
        out_dtype = torch.bfloat16 if x.dtype == torch.float32 else x.dtype
    if out_dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"cvmm_mx: output dtype {out_dtype} is not a 16-bit float")
    return ops.mx_forward(x, sel, keys.data, keys.scale, K, weights, out_dtype)


__all__ = ["MXTensor", "mx_quantize", "cvmm_mx", "mx_shapes"]
