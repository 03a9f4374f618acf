"""router_select, mx_quantize and cvmm_mx together, as the feed-forward layer uses them: trained with a
balanced, grouped sigmoid router, then served with 4-bit expert weights."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

from cvmm_codex_b200 import (MXTensor, SigmaMoEFFN, cvmm, cvmm_prepare_sel2, mx_quantize, router_select, router_topk,
                             sigma_moe_ffn)
from oracle import router_mx_oracle as O

pytestmark = pytest.mark.gpu

ROUTING = dict(scoring="sigmoid", n_groups=4, top_groups=2, group_score="top2", scale=1.5)


def layer_and_input(T=600, D=192, H=96, E=32, k=6, balance_bias=True, **routing):
    torch.manual_seed(1)
    layer = SigmaMoEFFN(D, E, H, k, device="cuda", balance_bias=balance_bias, **routing)
    if layer.bias is not None:
        layer.bias.copy_(0.1 * torch.randn(E, device="cuda"))
    return layer, torch.randn(T, D, device="cuda").bfloat16()


def test_layer_trains_with_the_selected_routing():
    """Output and every gradient against the layer composed with a torch router at the same choice."""
    layer, x0 = layer_and_input(**ROUTING)
    grad = torch.randn_like(x0)
    x = x0.clone().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = layer(x)
    out.backward(grad)
    got = [x.grad, layer.gate.grad, layer.w_up.grad, layer.w_down.grad]
    layer.zero_grad()
    x = x0.clone().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        logits = x @ layer.gate
        _, sel = router_select(logits.detach(), 6, bias=layer.bias, **ROUTING)
        s = torch.sigmoid(logits.float()).gather(-1, sel)
        w = 1.5 * s / s.sum(-1, keepdim=True)
        su = cvmm_prepare_sel2(sel)
        hidden = F.gelu(cvmm(x, su, layer.w_up))
        ref = cvmm(hidden.view(600, 6, 96), cvmm_prepare_sel2(su, w, route_input=True), layer.w_down)
    ref.backward(grad)
    # bf16 layers that differ in the order of 32-bit sums and the last bit of the activation: one bf16 step
    # (2^-8) of the largest value at each of the three rounded stages
    for a, e in zip([out] + got, [ref, x.grad, layer.gate.grad, layer.w_up.grad, layer.w_down.grad]):
        assert (a.float() - e.float()).abs().max() <= 3 * 2.0 ** -8 * e.float().abs().max()
    assert layer.bias.grad is None


def test_default_routing_is_unchanged():
    layer, x = layer_and_input(balance_bias=False)
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        out = layer(x)
        w, sel = router_topk(x @ layer.gate, 6)
        su = cvmm_prepare_sel2(sel)
        from cvmm_codex_b200 import cvmm_gelu
        hidden = cvmm_gelu(x, su, layer.w_up)
        want = cvmm(hidden.view(600, 6, 96), cvmm_prepare_sel2(su, w, route_input=True), layer.w_down)
    assert torch.equal(out, want)


@pytest.mark.parametrize("T", [1, 37, 600])
@pytest.mark.parametrize("routing", [{}, ROUTING])
def test_served_layer_matches_64_bit(T, routing):
    """The 4-bit layer against its own stages in 64 bits, each stage from the stage before as the layer rounds it."""
    layer, x = layer_and_input(T=T, balance_bias=bool(routing), **routing)
    served = layer.quantized()
    assert {n for n, _ in served.named_buffers()} >= {"gate", "up_data", "up_scale", "down_data", "down_scale"}
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = served(x)
    assert out.dtype == torch.bfloat16 and out.shape == x.shape and not out.requires_grad
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        logits = x @ layer.gate
    w, sel = router_select(logits, 6, bias=layer.bias, **routing)
    values = lambda q: np.swapaxes(q.dequantize().double().cpu().numpy(), -1, -2)  # noqa: E731
    up, down = (mx_quantize(t, dim=-2) for t in (layer.w_up, layer.w_down))
    quant = lambda t: O.mx_values(*O.mx_quantize(t.double().cpu().numpy()), t.shape[-1])  # noqa: E731
    h, size, _ = O.mx_product(quant(x), sel.cpu().numpy(), values(up), None, 6)
    from cvmm_codex_b200 import cvmm_mx
    z = cvmm_mx(x, sel, up)
    half = 2.0 ** -8
    assert (np.abs(z.double().cpu().numpy() - h) <= half * np.abs(h) + (192 / 32 + 8) * 2.0 ** -23 * size * (1 + half)).all()
    hidden = F.gelu(z)
    y, size, routes = O.mx_product(quant(hidden.view(-1, 96)), sel.cpu().numpy(), values(down),
                                   w.double().cpu().numpy(), 1)
    route = (np.abs(routes) * np.abs(w.double().cpu().numpy())[..., None]).sum(-2)
    tol = half * (np.abs(y) + route) + (96 / 32 + 8 + 7) * 2.0 ** -23 * (size + route) + 1e-30
    assert (np.abs(out.double().cpu().numpy() - y) <= tol * (1 + half)).all()


def test_served_layer_moves_and_loads():
    layer, x = layer_and_input(T=40, **ROUTING)
    served, other = layer.quantized(), layer_and_input(T=40, **ROUTING)[0].quantized()
    other.up_data.zero_()
    other.load_state_dict(served.state_dict())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = served(x)
        assert torch.equal(other(x), want)
        assert torch.equal(served.cpu().cuda()(x.view(4, 10, -1)).view(40, -1), want)


def test_served_layer_is_captured():
    layer, x = layer_and_input(T=64, **ROUTING)
    served = layer.quantized()
    static = x.clone()
    side = torch.cuda.Stream()
    with torch.autocast("cuda", dtype=torch.bfloat16, cache_enabled=False):
        want = served(x)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            served(static)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = served(static)
    static.zero_()
    graph.replay()
    static.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_mixed_weights_are_refused():
    layer, x = layer_and_input(T=4)
    with pytest.raises(ValueError, match="both"):
        sigma_moe_ffn(x, layer.gate, mx_quantize(layer.w_up, dim=-2), layer.w_down, 6)
    assert isinstance(mx_quantize(layer.w_up, dim=-2), MXTensor)


def test_served_layer_refuses_a_gradient():
    layer, x = layer_and_input(T=20, **ROUTING)
    served = layer.quantized()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        want = served(x)
        with pytest.raises(RuntimeError, match="no backward"):
            served(x.clone().requires_grad_(True))
        with torch.no_grad():
            assert torch.equal(served(x.clone().requires_grad_(True)), want)


def test_one_token_from_a_transposed_product():
    """A [1, n] tensor of strides (1, 1) gives what its copy gives: routing and its gradient, and the expert products."""
    from cvmm_codex_b200 import cvmm_mx
    torch.manual_seed(2)
    x = torch.randn(64, 1, device="cuda").bfloat16().T
    gate, w = torch.randn(64, 16, device="cuda").bfloat16(), torch.randn(16, 64, 48, device="cuda") / 8
    logits = (gate.T @ x.T).T
    assert x.stride() == (1, 1) and logits.stride() == (1, 1)
    outs = []
    for same in (lambda t: t.detach(), lambda t: t.detach().reshape(-1).clone().view(1, -1)):
        z = same(logits).requires_grad_(True)
        weights, sel = router_select(z, 4, scoring="sigmoid", bias=torch.zeros(16, device="cuda"))
        (gz,) = torch.autograd.grad(weights, z, torch.arange(4.0, device="cuda").view(1, 4))
        t = same(x).requires_grad_(True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = cvmm(t, cvmm_prepare_sel2(sel), w)
        g = torch.linspace(-1, 1, 48, device="cuda").bfloat16().view(48, 1).T.expand(4, 48).view(1, 4, 48)
        (gx,) = torch.autograd.grad(y, t, g)
        outs.append((weights.detach(), sel, gz, y.detach(), gx, cvmm_mx(same(x), sel, mx_quantize(w, dim=-2)),
                     cvmm_mx(same(x), sel, mx_quantize(w, dim=-2), weights.detach())))
    assert all(torch.equal(a, e) for a, e in zip(*outs))
