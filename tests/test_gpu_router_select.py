"""router_select and its gradient against a 64-bit evaluation (oracle/router_mx_oracle.py).

Tolerances. Choices are equal. Weights: expf of an argument with half an ulp of
at most 87 (5.2e-6), 2 ulp of expf, a sum of up to 1024 terms in 32 + 5
additions (2.2e-6) and the renormalising sum and division (2e-6): 1.2e-5
relative. Scores below the normal range are held to the step 2^-149, half a
step off, which a sum held at 1e-20 turns into 2^-150 / 1e-20 = 7.1e-26.
Gradients: the same 1.2e-5 twice over the sum of the magnitudes of
their terms (scores and weights each carry it), and half a step of the type."""
import numpy as np
import pytest
import torch

from cvmm_codex_b200 import router_select
from oracle import router_mx_oracle as O

pytestmark = pytest.mark.gpu

REL = 1.2e-5


def make(T, E, dtype, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    z = (1.5 * torch.randn(T, E, generator=g) + 0.5 * torch.randn(E, generator=g)).to(dtype)
    return z, (0.05 * torch.randn(E, generator=g) if bias else None)


def check(z, k, grad=True, **how):
    """Runs the rows of z and compares everything with the oracle."""
    bias = how.get("bias")
    zc = z.cuda().requires_grad_(grad)
    dev = dict(how, bias=None if bias is None else bias.cuda())
    w, sel = router_select(zc, k, **dev)
    assert w.dtype == torch.float32 and sel.dtype == torch.int64
    z64 = z.double().numpy()
    ref = dict(how, bias=None if bias is None else bias.double().numpy())
    ew, es = O.select(z64, k, **ref)
    np.testing.assert_array_equal(sel.cpu().numpy(), es)
    np.testing.assert_allclose(w.detach().cpu().double().numpy(), ew, rtol=REL, atol=how.get("scale", 1.0) * 7.1e-26)
    if grad:
        gw = torch.randn(w.shape, generator=torch.Generator().manual_seed(5))
        (gz,) = torch.autograd.grad(w, zc, gw.cuda())
        assert gz.dtype == z.dtype and gz.shape == z.shape
        args = (how.get("scoring", "softmax"), how.get("renormalize", True), how.get("scale", 1.0))
        eg, size = O.select_grad(z64, es, gw.double().numpy(), *args)
        # fp16 values below 2^-14 are rounded to a fixed step
        tol = 2 * REL * size + torch.finfo(z.dtype).eps / 2 * np.abs(eg) + (2.0 ** -25 if z.dtype == torch.float16 else 1e-37)
        # a score half a step of 2^-149 off, times at most 2 max|g| scale / 1e-20
        tol += 2 * float(gw.abs().max()) * how.get("scale", 1.0) * 7.1e-26
        err = np.abs(gz.cpu().double().numpy() - eg)
        assert (err <= tol).all(), (err - tol).max()
    return w, sel


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("T,E,k,groups,top,score", [
    (1, 64, 8, 1, 1, "max"), (37, 8, 8, 1, 1, "max"), (300, 128, 8, 8, 4, "top2"), (129, 100, 7, 5, 2, "max"),
    (65, 1, 1, 1, 1, "max"), (50, 33, 5, 1, 1, "max"), (40, 1024, 32, 32, 3, "top2"), (40, 960, 9, 3, 2, "max"),
    (70, 32, 3, 32, 5, "top2"), (61, 257, 4, 1, 1, "max"), (61, 512, 6, 16, 16, "max"), (30, 6, 2, 2, 1, "top2"),
])
def test_matches_64_bit(dtype, scoring, bias, T, E, k, groups, top, score):
    z, b = make(T, E, dtype, E + k, bias)
    check(z, k, scoring=scoring, bias=b, n_groups=groups, top_groups=top, group_score=score, renormalize=k % 2 == 0,
          scale=2.5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,score", [(1, "max"), (8, "max"), (8, "top2")])
def test_biased_scores_nearer_than_32_bits(scoring, groups, score):
    """Logits and bias that make every biased score nearly the same: only 64 bits tell them apart."""
    T, E, k = 500, 64, 6
    g = torch.Generator().manual_seed(7)
    if scoring == "sigmoid":
        s = 0.2 + 0.6 * torch.rand(T, E, generator=g, dtype=torch.float64)
        z = torch.log(s / (1 - s)).float()
        bias = torch.zeros(E)
        # one row's scores levelled by the bias; the other rows differ from it by a little
        bias = (0.9 - torch.sigmoid(z[0].double())).float()
        z = (z[0] + 2.0 ** -22 * torch.randint(-2, 3, (T, E), generator=g) * z[0].abs()).float()
    else:
        z0 = torch.randn(E, generator=g)
        bias = (0.5 - torch.softmax(z0.double(), -1)).float()
        z = (z0 + 2.0 ** -22 * torch.randint(-2, 3, (T, E), generator=g) * z0.abs()).float()
    check(z, k, scoring=scoring, bias=bias, n_groups=groups, top_groups=max(1, groups // 2), group_score=score)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups,score", [(1, "max"), (4, "max"), (4, "top2")])
def test_ties_go_to_the_lowest_index(scoring, bias, groups, score):
    g = torch.Generator().manual_seed(3)
    z = torch.randint(-2, 3, (400, 96), generator=g).float()
    z[0] = 0.25
    z[1] = -0.0
    z[1, ::3] = 0.0
    b = torch.zeros(96) if bias else None
    w, sel = check(z, 8, scoring=scoring, bias=b, n_groups=groups, top_groups=max(1, groups - 1), group_score=score)
    assert sel[0].tolist() == list(range(8)) and sel[1].tolist() == list(range(8))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("groups,score", [(1, "max"), (4, "max"), (4, "top2")])
@pytest.mark.parametrize("renorm", [False, True])
def test_masked_experts(scoring, bias, groups, score, renorm):
    """-inf logits: rows with all, all but one, half and one expert masked; the lowest finite value too."""
    g = torch.Generator().manual_seed(4)
    z = torch.randn(40, 16, generator=g)
    z[0] = -torch.inf
    z[1] = -torch.inf
    z[1, 13] = 0.3
    z[2, ::2] = -torch.inf
    z[3, 5] = -torch.inf
    z[4, 2:] = torch.finfo(torch.float32).min
    z[5] = torch.finfo(torch.float32).min
    z[6, :12] = -torch.inf
    b = 0.3 * torch.randn(16, generator=g) if bias else None
    w, sel = check(z, 4, scoring=scoring, bias=b, n_groups=groups, top_groups=max(1, groups // 2), group_score=score,
                   renormalize=renorm)
    assert torch.equal(w[0].detach().cpu(), torch.zeros(4))
    assert sel.min() >= 0 and sel.max() < 16


def test_not_a_number_and_infinity():
    z = torch.randn(6, 20, generator=torch.Generator().manual_seed(1))
    z[0, 7] = torch.nan
    z[1, 3] = torch.inf
    z[2, [4, 9]] = torch.inf
    z[3] = torch.nan
    for scoring in ("softmax", "sigmoid"):
        for bias in (None, torch.linspace(0, 1, 20)):
            w, sel = router_select(z.cuda(), 3, scoring=scoring, bias=None if bias is None else bias.cuda())
            ew, es = O.select(z.double().numpy(), 3, scoring=scoring, bias=None if bias is None else bias.double().numpy())
            np.testing.assert_array_equal(sel.cpu().numpy(), es)
            np.testing.assert_allclose(w.cpu().double().numpy(), ew, rtol=REL, atol=1e-37)


@pytest.mark.parametrize("groups,score", [(2, "max"), (4, "max"), (4, "top2")])
@pytest.mark.parametrize("bias", [False, True])
def test_not_a_number_in_groups(groups, score, bias):
    z = torch.randn(8, 20, generator=torch.Generator().manual_seed(1))
    z[0, 7] = torch.nan
    z[1, 3] = torch.inf
    z[2, 5:10] = -torch.inf
    z[2, 12] = torch.nan
    b = torch.linspace(0, 1, 20) if bias else None
    if bias:
        b[17] = torch.inf
        b[3] = -torch.inf
    for scoring in ("softmax", "sigmoid"):
        how = dict(scoring=scoring, n_groups=groups, top_groups=groups // 2, group_score=score)
        w, sel = router_select(z.cuda(), 3, bias=None if b is None else b.cuda(), **how)
        ew, es = O.select(z.double().numpy(), 3, bias=None if b is None else b.double().numpy(), **how)
        np.testing.assert_array_equal(sel.cpu().numpy(), es)
        np.testing.assert_allclose(w.cpu().double().numpy(), ew, rtol=REL, atol=1e-37)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,score", [(1, "max"), (8, "max"), (8, "top2"), (32, "top2")])
@pytest.mark.parametrize("size", [1e3, 1e6])
def test_large_biases_of_both_signs(scoring, groups, score, size):
    """Biases whose 32-bit sums with a score lose the score: groups of a large and a large negative one, nearly equal."""
    T, E = 300, 64
    g = torch.Generator().manual_seed(17)
    z = torch.randn(T, E, generator=g)
    bias = size * (1 + torch.rand(E // 2, generator=g))
    bias = torch.stack((bias, -bias), dim=1).flatten()
    check(z, 4, scoring=scoring, bias=bias, n_groups=groups, top_groups=max(1, groups // 2), group_score=score)
    off = bias.clone()
    off[::5] = -torch.inf
    check(z, 4, scoring=scoring, bias=off, n_groups=groups, top_groups=max(1, groups // 2), group_score=score)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bias_types_and_strides(dtype):
    z, b = make(50, 64, torch.float32, 12)
    check(z, 6, scoring="sigmoid", bias=b.to(dtype))
    wide = torch.zeros(64, 3, device="cuda")
    wide[:, 1] = b.cuda()
    got, want = router_select(z.cuda(), 6, bias=wide[:, 1]), router_select(z.cuda(), 6, bias=b.cuda())
    assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_zero_bias_is_no_bias():
    """A balance bias that starts at zero: bf16 logits tie often, and the choice is that without a bias."""
    z, _ = make(4000, 64, torch.bfloat16, 13)
    zero = torch.zeros(64, device="cuda")
    for scoring in ("softmax", "sigmoid"):
        got, want = (router_select(z.cuda(), 6, scoring=scoring, bias=b) for b in (zero, None))
        assert torch.equal(got[1], want[1])


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [False, True])
def test_gradient_matches_differences(scoring, renorm):
    z, b = make(9, 24, torch.float32, 2)
    zc = z.cuda().requires_grad_(True)
    w, sel = router_select(zc, 5, scoring=scoring, bias=b.cuda(), renormalize=renorm, scale=1.5)
    r = torch.randn(w.shape, generator=torch.Generator().manual_seed(8))
    (gz,) = torch.autograd.grad(w, zc, r.cuda())
    z64, s, h = z.double().numpy(), sel.cpu().numpy(), 1e-6
    for e in range(24):
        d = np.zeros_like(z64)
        d[:, e] = h
        up, dn = (O.select_weights(z64 + f * d, s, scoring, renorm, 1.5) for f in (1, -1))
        diff = ((up - dn) * r.double().numpy()).sum(-1) / (2 * h)
        # differences in 64 bits: h^2 of the third derivative and 2^-53 / h of rounding, below 1e-9
        np.testing.assert_allclose(gz[:, e].cpu().double().numpy(), diff, rtol=0, atol=2 * REL * 8 + 1e-9)


def test_held_sum_has_no_sum_term():
    """Scores whose sum is below 1e-20: the weights are s / 1e-20 and so is their gradient."""
    z = torch.full((3, 8), -100.0)
    z[:, 1] = -60.0
    z[1] = -50.0
    check(z, 2, scoring="sigmoid")


def test_shapes_strides_and_empty():
    z, b = make(30, 40, torch.float32, 9)
    want = router_select(z.cuda(), 4, bias=b.cuda())
    wide = torch.zeros(30, 64, device="cuda")
    wide[:, 8:48] = z.cuda()
    cols = torch.zeros(40, 30, device="cuda")
    cols.copy_(z.T)
    for view in (wide[:, 8:48], cols.T, z.cuda().view(5, 6, 40)):
        w, sel = router_select(view, 4, bias=b.cuda())
        assert w.shape == (*view.shape[:-1], 4)
        assert torch.equal(w.reshape(30, 4), want[0]) and torch.equal(sel.reshape(30, 4), want[1])
    one = router_select(z[0].cuda(), 4, bias=b.cuda())
    assert torch.equal(one[0], want[0][0]) and torch.equal(one[1], want[1][0])
    zero = torch.zeros(0, 40, device="cuda", requires_grad=True)
    w, sel = router_select(zero, 4)
    assert w.shape == sel.shape == (0, 4)
    assert torch.autograd.grad(w.sum(), zero)[0].shape == (0, 40)
    stretched = z[:1].cuda().expand(30, 40)
    w, sel = router_select(stretched, 4, bias=b.cuda())
    assert torch.equal(w, want[0][:1].expand(30, 4)) and torch.equal(sel, want[1][:1].expand(30, 4))


def test_gradients_of_views_and_broadcast():
    """A strided logits view and one row stretched over the tokens get their own gradients, a broadcast grad too."""
    z, _ = make(6, 16, torch.float32, 11)
    base = torch.zeros(6, 32, device="cuda")
    base[:, :16] = z.cuda()
    base.requires_grad_(True)
    w, sel = router_select(base[:, :16], 3, renormalize=False)
    w.sum().backward()
    eg, size = O.select_grad(z.double().numpy(), sel.cpu().numpy(), np.ones((6, 3)), "softmax", False, 1.0)
    assert (np.abs(base.grad[:, :16].cpu().double().numpy() - eg) <= 2 * REL * size + 2.0 ** -24 * np.abs(eg)).all()
    assert not base.grad[:, 16:].any()
    row = z[0].cuda().requires_grad_(True)
    w, sel = router_select(row.expand(6, 16), 3, renormalize=False)
    w.sum().backward()
    want = 6 * O.select_grad(z[:1].double().numpy(), sel[:1].cpu().numpy(), np.ones((1, 3)), "softmax", False, 1.0)[0][0]
    np.testing.assert_allclose(row.grad.cpu().double().numpy(), want, rtol=0, atol=6 * 4 * REL)


def test_no_second_derivative():
    z = torch.randn(3, 8, device="cuda", requires_grad=True)
    w, _ = router_select(z, 2)
    (g,) = torch.autograd.grad(w.square().sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_captured_and_on_another_stream():
    z, b = make(257, 48, torch.bfloat16, 21)
    zc, bc = z.cuda(), b.cuda()
    gw = torch.randn(257, 5, device="cuda")

    def step(t):
        t = t.detach().requires_grad_(True)
        w, sel = router_select(t, 5, scoring="sigmoid", bias=bc, n_groups=4, top_groups=2, group_score="top2")
        return w.detach(), sel, torch.autograd.grad(w, t, gw)[0]

    want = step(zc)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(zc)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, e) for a, e in zip(got, want))
    static = torch.zeros_like(zc)
    with torch.cuda.stream(side):
        step(static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for _ in range(2):
        static.copy_(zc)
        graph.replay()
        assert all(torch.equal(a, e) for a, e in zip(out, want))
        static.zero_()
        graph.replay()
        torch.cuda.synchronize()


def test_traces_without_a_graph_break():
    z, b = make(64, 32, torch.float32, 31)
    zc, bc = z.cuda().requires_grad_(True), b.cuda()

    def f(t):
        return router_select(t, 4, scoring="sigmoid", bias=bc)

    w, sel = f(zc)
    cw, cs = torch.compile(f, fullgraph=True)(zc)
    assert torch.equal(cs, sel) and torch.equal(cw, w)
    g = torch.randn_like(w)
    assert torch.equal(torch.autograd.grad(cw, zc, g)[0], torch.autograd.grad(w, zc, g)[0])


@pytest.mark.parametrize("E", [6, 64, 100, 300, 1000])
@pytest.mark.parametrize("bias", [False, True])
def test_weights_and_gradient_share_their_scores(E, bias):
    """One expert a token, no renormalising: the gradient at it is w (1 - w) of the very weight returned."""
    z, b = make(400, E, torch.float32, E, bias)
    zc = (3 * z).cuda().requires_grad_(True)
    w, sel = router_select(zc, 1, bias=None if b is None else b.cuda(), renormalize=False)
    (gz,) = torch.autograd.grad(w, zc, torch.ones_like(w))
    w = w.detach()
    assert torch.equal(gz.gather(-1, sel), w * (1 - w))


def test_compiled_and_linear_losses_have_no_second_derivative_either():
    r = torch.randn(3, 2, device="cuda")
    for fn in (lambda t: router_select(t, 2)[0], torch.compile(lambda t: router_select(t, 2)[0], fullgraph=True)):
        z = torch.randn(3, 8, device="cuda", requires_grad=True)
        with pytest.raises(RuntimeError):
            (g,) = torch.autograd.grad((fn(z) * r).sum(), z, create_graph=True)
            (g.square().sum() + z.square().sum()).backward()
