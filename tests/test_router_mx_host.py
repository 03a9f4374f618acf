"""Refusals and host-side shapes of router_select, mx_quantize and cvmm_mx (no GPU)."""
import numpy as np
import pytest
import torch

import cvmm_codex_b200 as b
from cvmm_codex_b200 import _lib
from cvmm_codex_b200.mx import mx_shapes
from oracle import router_mx_oracle as O


@pytest.mark.parametrize("bad", [
    dict(top_k=0), dict(top_k=33), dict(top_k=9), dict(scoring="tanh"), dict(group_score="sum"), dict(n_groups=3),
    dict(n_groups=0), dict(n_groups=4, top_groups=5), dict(n_groups=4, top_groups=0),
    dict(n_groups=4, top_groups=1, top_k=3), dict(bias=torch.zeros(7)), dict(bias=torch.zeros(8, dtype=torch.int32)),
    dict(bias=torch.zeros(8, dtype=torch.float64)), dict(bias=torch.zeros(1, 8)),
])
def test_router_select_refuses(bad):
    args = dict(top_k=2)
    args.update(bad)
    with pytest.raises(ValueError, match="router_select"):
        b.router_select(torch.zeros(4, 8), **args)


@pytest.mark.parametrize("logits", [torch.zeros(4, 8, dtype=torch.float64), torch.zeros(4, 8, dtype=torch.int64),
                                    torch.zeros(()), torch.zeros(4, 1025), torch.zeros(4, 0)])
def test_router_select_refuses_logits(logits):
    with pytest.raises(ValueError, match="router_select"):
        b.router_select(logits, 1)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="CUDA"):
        b.router_select(torch.zeros(4, 8), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        b.mx_quantize(torch.zeros(4, 8))


def _keys(E=3, K=40, N=5):
    data, scale = mx_shapes((E, K, N), -2)
    return b.MXTensor(torch.zeros(data, dtype=torch.uint8), torch.zeros(scale, dtype=torch.uint8), (E, K, N), dim=-2)


def test_mx_shapes():
    assert mx_shapes((3, 40, 5), -2) == ((3, 5, 32), (3, 1, 1, 32, 4, 4))
    assert mx_shapes((2, 300, 129), -1) == ((2, 300, 80), (5, 2, 32, 4, 4))
    assert mx_shapes((7,), -1) == ((16,), (1, 1, 32, 4, 4))
    for bad in (((7,), -2), ((2, 3), 0), ((2, 3), 1)):
        with pytest.raises(ValueError):
            mx_shapes(*bad)


def test_mxtensor_refuses():
    k = _keys()
    for data, scale, shape, dim in (
            (k.data.int(), k.scale, k.shape, -2), (k.data[:2], k.scale, k.shape, -2),
            (k.data, k.scale[..., :3], k.shape, -2), (k.data, k.scale, (3, 5, 40), -1),
            (k.data.mT.contiguous().mT, k.scale, k.shape, -2)):
        with pytest.raises(ValueError, match="MXTensor|microscaled"):
            b.MXTensor(data, scale, shape, dim)
    with pytest.raises(ValueError, match="dtype"):
        k.dequantize(torch.float64)


def test_mx_quantize_refuses():
    for x, dim in ((torch.zeros(4, 8, dtype=torch.float64), -1), (torch.zeros(4, 8), 0), (torch.zeros(4, 8), 1),
                   (torch.zeros(8), -2)):
        with pytest.raises(ValueError, match="mx_quantize"):
            b.mx_quantize(x, dim)


@pytest.mark.parametrize("x,sel,weights", [
    (torch.zeros(4, 41), torch.zeros(4, 2, dtype=torch.int64), None),         # K
    (torch.zeros(4, 40), torch.zeros(5, 2, dtype=torch.int64), None),         # tokens
    (torch.zeros(4, 3, 40), torch.zeros(4, 2, dtype=torch.int64), None),      # rows that do not divide the routes
    (torch.zeros(4, 40), torch.zeros(4, 2), None),                            # float ids
    (torch.zeros(4, 40), torch.zeros(4, 0, dtype=torch.int64), None),
    (torch.zeros(4, 40), torch.zeros((), dtype=torch.int64), None),
    (torch.zeros(4, 40, dtype=torch.float64), torch.zeros(4, 2, dtype=torch.int64), None),
    (torch.zeros(4, 40), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 3)),
    (torch.zeros(4, 40), torch.zeros(4, 2, dtype=torch.int64), torch.zeros(4, 2, dtype=torch.int64)),
])
def test_cvmm_mx_refuses(x, sel, weights):
    with pytest.raises(ValueError, match="cvmm_mx"):
        b.cvmm_mx(x, sel, _keys(), weights)


def test_cvmm_mx_refuses_keys_gradients_and_two_weights():
    x, sel = torch.zeros(4, 40), torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(ValueError, match="keys"):
        b.cvmm_mx(x, sel, torch.zeros(3, 40, 5))
    data, scale = mx_shapes((3, 5, 40), -1)
    rows = b.MXTensor(torch.zeros(data, dtype=torch.uint8), torch.zeros(scale, dtype=torch.uint8), (3, 5, 40), -1)
    with pytest.raises(ValueError, match="keys"):
        b.cvmm_mx(x, sel, rows)
    with pytest.raises(RuntimeError, match="no backward"):
        b.cvmm_mx(x.clone().requires_grad_(True), sel, _keys())
    w = torch.ones(4, 2)
    s = b.CVMMSel(sel.int(), sel.int(), sel.reshape(-1), None, w)
    with pytest.raises(ValueError, match="twice"):
        b.cvmm_mx(x, s, _keys(), w)


@pytest.mark.parametrize("call,code", [
    (lambda l: l.cvmm_router_select(16, 3, 8, 4, 8, 2, 0, None, 0, 1, 1, 0, 1, 1.0, 16, 16, None), -2),
    (lambda l: l.cvmm_router_select(16, 0, 7, 4, 8, 2, 0, None, 0, 1, 1, 0, 1, 1.0, 16, 16, None), -1),
    (lambda l: l.cvmm_router_select(16, 0, 8, 4, 8, 2, 2, None, 0, 1, 1, 0, 1, 1.0, 16, 16, None), -1),
    (lambda l: l.cvmm_router_select(16, 0, 8, 4, 8, 2, 0, None, 0, 1, 1, 2, 1, 1.0, 16, 16, None), -1),
    (lambda l: l.cvmm_router_select(16, 0, 8, 4, 8, 5, 0, None, 0, 4, 2, 0, 1, 1.0, 16, 16, None), -1),
    (lambda l: l.cvmm_router_select(16, 0, 66, 4, 66, 2, 0, None, 0, 33, 2, 0, 1, 1.0, 16, 16, None), -1),
    (lambda l: l.cvmm_router_select(None, 0, 8, 4, 8, 2, 0, None, 0, 1, 1, 0, 1, 1.0, 16, 16, None), -1),
    (lambda l: l.cvmm_router_select_backward(16, 0, 8, 16, 16, 4, 8, 9, 0, 1, 1.0, 16, None), -1),
    (lambda l: l.cvmm_router_select_backward(16, 0, 8, None, 16, 4, 8, 2, 0, 1, 1.0, 16, None), -1),
    (lambda l: l.cvmm_mx_quantize(16, 3, 1, 4, 8, 0, 8, 1, 16, 16, None), -2),
    (lambda l: l.cvmm_mx_quantize(16, 0, 1, -1, 8, 0, 8, 1, 16, 16, None), -1),
    (lambda l: l.cvmm_mx_quantize(16, 0, 1, 4, 8, 0, 8, 1, 20, 16, None), -1),
    (lambda l: l.cvmm_mx_dequantize(16, 16, 1, 4, 8, 0, 8, 1, None, 0, None), -1),
    (lambda l: l.cvmm_mx_dequantize(16, 16, 1, 4, 8, 0, 8, 1, 16, 4, None), -2),
    # out must be 16-bit; x rows must divide the routes; keys 16-byte aligned; a workspace is required
    (lambda l: l.cvmm_mx_forward(16, 0, 4, 8, 16, 4, 8, 2, None, 0, 16, 16, 2, 8, 8, 16, 0, 16, 1 << 20, None), -2),
    (lambda l: l.cvmm_mx_forward(16, 0, 3, 8, 16, 4, 8, 2, None, 0, 16, 16, 2, 8, 8, 16, 2, 16, 1 << 20, None), -1),
    (lambda l: l.cvmm_mx_forward(16, 0, 4, 8, 16, 4, 8, 2, None, 0, 24, 16, 2, 8, 8, 16, 2, 16, 1 << 20, None), -1),
    (lambda l: l.cvmm_mx_forward(16, 0, 4, 8, 16, 4, 8, 2, None, 0, 16, 16, 2, 8, 8, 16, 2, None, 0, None), -4),
    (lambda l: l.cvmm_mx_forward(16, 0, 4, 8, 16, 0, 8, 2, None, 0, 16, 16, 2, 8, 8, 16, 2, 16, 1 << 20, None), -2),
])
def test_c_entries_refuse_before_any_launch(call, code):
    lib = _lib.load()
    assert call(lib) == code
    assert len(lib.cvmm_last_error()) > 0


def test_oracle_quantisation_is_nearest():
    """The oracle itself: every value is within half a step of its grid, and the scale is the format's."""
    x = np.random.default_rng(0).standard_normal((5, 70)) * np.exp(np.random.default_rng(1).standard_normal((5, 1)))
    codes, scale = O.mx_quantize(x)
    v = O.mx_values(codes, scale, 70)
    s = np.exp2(scale.astype(float) - 127).repeat(32, -1)[:, :70]
    a = np.abs(x) / s
    step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
    assert (np.abs(v - x) / s <= np.where(a > 6, a - 6, step / 2)).all()
    assert a.max() < 8


def test_router_select_refuses_a_tangent():
    """A forward-mode derivative is refused, not dropped, with gradients enabled or not."""
    z, t = torch.randn(4, 8), torch.randn(4, 8)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(z, t)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                b.router_select(dual, 2)
        with pytest.raises(RuntimeError, match="CUDA"):  # a tensor without a tangent is none of its business
            b.router_select(z, 2)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda a: b.router_select(a, 2)[0], (z,), (t,))


def test_cvmm_mx_refuses_tangents():
    x, sel, w = torch.zeros(4, 40), torch.zeros(4, 2, dtype=torch.int64), torch.ones(4, 2)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x), sel, _keys()), (dual(x), sel, _keys(), w), (x, sel, _keys(), dual(w)),
                     (x, b.CVMMSel(sel.int(), sel.int(), sel.reshape(-1), None, dual(w)), _keys())):
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                b.cvmm_mx(*args)
        with pytest.raises(RuntimeError, match="CUDA"):
            b.cvmm_mx(x, sel, _keys(), w)


@pytest.fixture
def router_on_the_cpu(monkeypatch):
    """The two router calls replaced by the 64-bit oracle, so that autograd's part runs without a GPU."""
    from cvmm_codex_b200 import api

    def select(self, logits, k, scoring, bias, n_groups, top_groups, group_score, renormalize, scale):
        w, sel = O.select(logits.detach().numpy(), k, scoring, bias, n_groups, top_groups, group_score, renormalize, scale)
        return torch.from_numpy(w).float(), torch.from_numpy(sel)

    def backward(self, logits, sel, grad_w, scoring, renormalize, scale):
        g, _ = O.select_grad(logits.detach().double().numpy(), sel.numpy(), grad_w.detach().numpy(), scoring,
                             renormalize, scale)
        return torch.from_numpy(g).to(logits.dtype)

    monkeypatch.setattr(type(api.ops), "router_select", select)
    monkeypatch.setattr(type(api.ops), "router_select_backward", backward)


def test_a_linear_loss_has_no_second_derivative_either(router_on_the_cpu):
    """The weights' gradient depends on the logits even where the loss's own does not: refused, not left out."""
    r = torch.randn(3, 2)
    for loss in (lambda w: (w * r).sum(), lambda w: w.square().sum()):
        z = torch.randn(3, 8, requires_grad=True)
        (g,) = torch.autograd.grad(loss(b.router_select(z, 2)[0]), z, create_graph=True)
        assert g.requires_grad
        with pytest.raises(RuntimeError, match="differentiable once"):
            (g.square().sum() + z.square().sum()).backward()
    z = torch.randn(3, 8, requires_grad=True)
    (g,) = torch.autograd.grad((b.router_select(z, 2)[0] * r).sum(), z)
    assert not g.requires_grad
    w, sel = b.router_select(z, 2)
    (w * r).sum().backward(create_graph=True)  # a graph that nobody differentiates
    assert torch.equal(z.grad, g)
    assert torch.autograd.grad((z.sum() * 2), z)[0].eq(2).all()


def test_the_served_layer_refuses_a_gradient(monkeypatch):
    """An input's gradient is refused, not dropped; without one, or under no_grad, the layer gets to its product."""
    from cvmm_codex_b200 import api

    def quantize(self, x, dim):
        return tuple(torch.zeros(s, dtype=torch.uint8) for s in mx_shapes(x.shape, dim))

    def topk(self, logits, k, renormalize):
        return torch.ones(*logits.shape[:-1], k), torch.zeros(*logits.shape[:-1], k, dtype=torch.int64)

    monkeypatch.setattr(type(api.ops), "mx_quantize", quantize)
    monkeypatch.setattr(type(api.ops), "router_topk", topk)
    served = b.SigmaMoEFFN(16, 4, 8, 2).quantized()
    x = torch.randn(3, 16)
    with pytest.raises(RuntimeError, match="no backward"):
        served(x.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="CUDA"):
        served(x)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        served(x.clone().requires_grad_(True))


@pytest.mark.parametrize("bad", [dict(top_groups=2), dict(top_groups=0), dict(group_score="sum"), dict(scoring="tanh"),
                                 dict(n_groups=3), dict(bias=torch.zeros(3))])
def test_the_layer_refuses_what_its_router_refuses(bad):
    x, gate = torch.zeros(5, 16), torch.zeros(16, 4)
    with pytest.raises(ValueError, match="router_select"):
        b.sigma_moe_ffn(x, gate, torch.zeros(4, 16, 8), torch.zeros(4, 8, 16), 2, **bad)
    layer = b.SigmaMoEFFN(16, 4, 8, 2, **{k: v for k, v in bad.items() if k != "bias"})
    if "bias" in bad:
        layer.bias = bad["bias"]
    with pytest.raises(ValueError, match="router_select"):
        layer(x)


@pytest.mark.parametrize("rows", [0, 1, 2])
def test_single_rows_of_any_stride_reach_the_library_with_a_whole_row_stride(rows, monkeypatch):
    """A transposed column [1, E] has strides (1, 1) and torch calls it contiguous."""
    from cvmm_codex_b200 import ops
    seen = []
    monkeypatch.setattr(ops, "_require_cuda", lambda *t: None)
    monkeypatch.setattr(ops, "_call", lambda name, fn, device, *args, **kw: seen.append((name, args)))
    x = torch.randn(40, rows).T
    sel = torch.zeros(rows, 2, dtype=torch.int64)
    if rows < 2:
        assert x.stride(0) < 40 and x.is_contiguous()
    ops.router_select(x, 2, "softmax", None, 1, 1, "max", True, 1.0)
    ops.router_select_backward(x, sel, torch.zeros(rows, 2), "softmax", True, 1.0)
    k = _keys()
    ops.mx_forward(x, sel, k.data, k.scale, 40, None, torch.bfloat16)
    ld = {"cvmm_router_select": 2, "cvmm_router_select_backward": 2, "cvmm_mx_forward": 3}
    assert len(seen) == 3 and all(args[ld[name]] >= 40 for name, args in seen)
    v = torch.arange(6.0).view(6, 1)[1:].T
    assert torch.equal(ops._rows(v), v) and ops._rows(v).stride() == (5, 1) and ops._rows(v).data_ptr() == v.data_ptr()


@pytest.mark.parametrize("routes,experts,n,columns", [
    (8, 128, 512, 64), (64, 128, 512, 256), (262144, 128, 512, 256), (65536, 64, 128, 128), (0, 8, 8, 0), (8, 8, 0, 0),
    # the shapes of test_gpu_mx.COLUMNS_128
    (4800, 8, 384, 128), (4800, 8, 370, 128), (4800, 8, 200, 128), (4800, 8, 374, 128), (9900, 8, 384, 128),
    (9900, 8, 380, 128),
])
def test_tile_columns(routes, experts, n, columns):
    assert _lib.load().cvmm_mx_tile_columns(routes, experts, n, 148) == columns


def test_launches():
    lib = _lib.load()
    assert [lib.cvmm_mx_launches(r, w) for r, w in ((0, 1), (1, 0), (4096, 1), (4097, 0), (4097, 1))] == [0, 2, 3, 3, 4]
