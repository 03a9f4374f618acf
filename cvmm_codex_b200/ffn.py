"""The sigma-MoE feed-forward layer on the sm_100a CVMM kernels.

The reference's caller of CVMM (benchmark_ffn_moe.py:83-100, the
feed-forward of sigma-MoE / MoEUT) is, under bf16 autocast:

    logits = x @ gate
    probs = softmax(float(logits)); weights, sel = probs.topk(k)
    weights = weights / weights.sum(-1).clamp_min(1e-20)
    sel_up = cvmm_prepare_sel2(sel)
    hidden = F.gelu(cvmm(x, sel_up, w_up))
    sel_down = cvmm_prepare_sel2(sel_up, weights, route_input=True)
    out = cvmm(hidden.view(..., k, H), sel_down, w_down)

Here the same layer runs with three fusions:
* the router (softmax, top-k, renormalisation) is one kernel
  (``api.router_topk``) instead of four torch passes over [T, E];
* one selector preparation serves both projections: the down projection
  re-wraps the up projection's sorted routes (cvmm.py:1788-1792), so the
  device sort runs once per layer;
* GELU is applied in the up projection's epilogue (``api.cvmm_gelu``), so the
  activation costs no pass of its own, and its backward is one vectorised
  elementwise kernel on the saved pre-activation.
The router matmul is a plain bf16 cuBLAS GEMM (x @ gate).

Two variants beyond the reference's layer: routing by ``router_select`` (sigmoid
scores, a balance bias, expert groups), in training as in serving, and 4-bit
microscaled expert weights (``mx_quantize``), for serving only: both products
then run on the 4-bit tensor cores and the hidden rows between them are
quantised as the input rows are.
"""
from __future__ import annotations

import math

from typing import Optional, Union

import torch

from .api import cvmm, cvmm_gelu, cvmm_prepare_sel2, router_select, router_topk
from .mx import MXTensor, cvmm_mx, mx_quantize

Weights = Union[torch.Tensor, MXTensor]


def sigma_moe_ffn(x: torch.Tensor, gate: torch.Tensor, w_up: Weights, w_down: Weights, k: int,
                  renormalize: bool = True, scoring: str = "softmax", bias: Optional[torch.Tensor] = None,
                  n_groups: int = 1, top_groups: Optional[int] = None, group_score: str = "max",
                  scale: float = 1.0) -> torch.Tensor:
    """The sigma-MoE FFN layer (benchmark_ffn_moe.py:87-98) on x [..., D]:
    gate [D, E], w_up [E, D, H], w_down [E, H, D]; returns [..., D]. Call it
    under torch.autocast(bfloat16) as the reference does.

    scoring, bias, n_groups, top_groups, group_score and scale are
    router_select's; with their defaults the router is the reference's.
    w_up and w_down may both be MXTensors (mx_quantize(w, dim=-2)): the expert
    products are then cvmm_mx's, without a backward."""
    mx = isinstance(w_up, MXTensor)
    if mx != isinstance(w_down, MXTensor):
        raise ValueError("sigma_moe_ffn: w_up and w_down must both be MXTensors or both be tensors")
    logits = x @ gate
    # Arguments that router_select refuses go to it even where router_topk would not look at them.
    plain = scoring == "softmax" and bias is None and n_groups == 1 and scale == 1.0
    if plain and top_groups in (None, 1) and group_score in ("max", "top2"):
        weights, sel = router_topk(logits, k, renormalize)
    else:
        weights, sel = router_select(logits, k, scoring=scoring, bias=bias, n_groups=n_groups, top_groups=top_groups,
                                     group_score=group_score, renormalize=renormalize, scale=scale)
    if mx:
        hidden = torch.nn.functional.gelu(cvmm_mx(x, sel, w_up))
        return cvmm_mx(hidden, sel, w_down, weights)
    sel_up = cvmm_prepare_sel2(sel)
    hidden = cvmm_gelu(x, sel_up, w_up)
    sel_down = cvmm_prepare_sel2(sel_up, weights, route_input=True)
    return cvmm(hidden.view(*x.shape[:-1], k, w_up.shape[-1]), sel_down, w_down)


class SigmaMoEFFN(torch.nn.Module):
    """sigma-MoE feed-forward block: n_experts experts of width expert_size,
    top-k routing by a softmax router, GELU, weighted combine. Parameters
    are fp32 (autocast casts them per call), initialised N(0, 1/fan_in).

    scoring, n_groups, top_groups, group_score and scale are router_select's.
    balance_bias: keep a buffer `bias` [n_experts], zero at first, that is added
    to the scores for the choice of experts alone; the caller moves it (down for
    experts that get too many tokens), it has no gradient."""

    def __init__(self, d_model: int, n_experts: int, expert_size: int, k: int, renormalize: bool = True,
                 device=None, scoring: str = "softmax", balance_bias: bool = False, n_groups: int = 1,
                 top_groups: Optional[int] = None, group_score: str = "max", scale: float = 1.0):
        super().__init__()
        self.k = int(k)
        self.renormalize = renormalize
        self.routing = dict(scoring=scoring, n_groups=n_groups, top_groups=top_groups, group_score=group_score,
                            scale=scale)
        self.register_buffer("bias", torch.zeros(n_experts, device=device) if balance_bias else None)
        self.gate = torch.nn.Parameter(torch.randn(d_model, n_experts, device=device) / math.sqrt(d_model))
        self.w_up = torch.nn.Parameter(torch.randn(n_experts, d_model, expert_size, device=device)
                                       / math.sqrt(d_model))
        self.w_down = torch.nn.Parameter(torch.randn(n_experts, expert_size, d_model, device=device)
                                         / math.sqrt(expert_size))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return sigma_moe_ffn(x, self.gate, self.w_up, self.w_down, self.k, self.renormalize, bias=self.bias,
                             **self.routing)

    def quantized(self) -> "SigmaMoEFFNMX":
        """This layer with its expert weights in 4 bits, for serving."""
        return SigmaMoEFFNMX(self)


class SigmaMoEFFNMX(torch.nn.Module):
    """A SigmaMoEFFN with 4-bit microscaled expert weights (17/128 of their fp32 bytes).

    Made by SigmaMoEFFN.quantized(), a copy of that layer as it is then. The
    weights' bytes, the gate and the bias are buffers: they move with the
    module and are in its state_dict. Forward only: an input that requires grad
    is refused while gradients are recorded, as cvmm_mx refuses it."""

    def __init__(self, layer: SigmaMoEFFN):
        super().__init__()
        self.k, self.renormalize, self.routing = layer.k, layer.renormalize, dict(layer.routing)
        self.up_shape, self.down_shape = tuple(layer.w_up.shape), tuple(layer.w_down.shape)
        self.register_buffer("gate", layer.gate.detach().clone())
        self.register_buffer("bias", None if layer.bias is None else layer.bias.clone())
        for name, w in (("up", layer.w_up), ("down", layer.w_down)):
            q = mx_quantize(w, dim=-2)
            self.register_buffer(name + "_data", q.data)
            self.register_buffer(name + "_scale", q.scale)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return sigma_moe_ffn(x, self.gate, MXTensor(self.up_data, self.up_scale, self.up_shape, dim=-2),
                             MXTensor(self.down_data, self.down_scale, self.down_shape, dim=-2), self.k,
                             self.renormalize, bias=self.bias, **self.routing)
