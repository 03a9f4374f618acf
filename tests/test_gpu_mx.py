"""Microscaled 4-bit tensors and the expert product against 64-bit evaluations (oracle/router_mx_oracle.py).

Quantised bytes and dequantised values are equal, bit for bit. Product: the
4-bit products are exact, the sums are held in 32 bits; with at most K / 32 + 8
roundings of at most one ulp each (a rounding per scaled group or matrix step)
the sum is within (K / 32 + 8) 2^-23 of the sum of the magnitudes; then half a
step of the output type, and for weighted outputs half a step of every route
output before the 32-bit weighted sum."""
import numpy as np
import pytest
import torch

import cvmm_codex_b200 as b
from cvmm_codex_b200 import MXTensor, _lib, cvmm_mx, cvmm_prepare_sel2, mx_quantize
from oracle import router_mx_oracle as O

pytestmark = pytest.mark.gpu

FLOATS = [torch.float32, torch.bfloat16, torch.float16]


def view3(t, dim):
    """numpy [batch, rows, K] of a tensor quantised along dim."""
    a = t.detach().cpu().double().numpy()
    if dim == -1:
        return a.reshape(1, -1, a.shape[-1])
    return np.swapaxes(a.reshape(-1, *a.shape[-2:]), -1, -2)


def check_quantize(x, dim):
    q = mx_quantize(x, dim)
    assert q.shape == x.shape and q.dim == dim
    v = view3(x, dim)
    codes, scale = O.mx_quantize(v)
    data, pieces = O.mx_pack(codes, scale)
    np.testing.assert_array_equal(q.scale.cpu().numpy().reshape(pieces.shape), pieces)
    np.testing.assert_array_equal(q.data.cpu().numpy().reshape(data.shape), data)
    want = O.mx_values(codes, scale, v.shape[-1])
    for dtype in FLOATS:
        got = q.dequantize(dtype)
        assert got.shape == x.shape and got.dtype == dtype and got.is_contiguous()
        rounded = torch.from_numpy(want).float().to(dtype)  # exact in fp32; one rounding
        np.testing.assert_array_equal(view3(got, dim), rounded.double().numpy())
    return q


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("dim", [-1, -2])
@pytest.mark.parametrize("shape", [(1, 1), (3, 32), (130, 200), (128, 128), (7, 33), (2, 129, 65), (3, 31, 257),
                                   (1, 5000), (2, 3, 40, 72)])
def test_quantize_matches_64_bit(dtype, dim, shape):
    g = torch.Generator().manual_seed(sum(shape))
    x = torch.randn(*shape, generator=g) * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=g))
    check_quantize(x.to(dtype).cuda(), dim)


@pytest.mark.parametrize("dim", [-1, -2])
def test_quantize_special_values(dim):
    """Ties, the largest and smallest numbers, zeros of both signs, infinities and NaN in single groups."""
    x = torch.zeros(12, 64)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.9, 6.0, 4.0])
    x[0, :11], x[0, 11:22] = ties, -ties
    x[0, 32:43] = ties * 2.0 ** 40
    x[1, :3] = torch.tensor([torch.finfo(torch.float32).max, 1e38, -1.0])
    x[1, 40] = torch.finfo(torch.float32).tiny
    x[2, :4] = torch.tensor([1e-45, -1e-45, 3e-45, 1e-44])
    x[2, 33] = 2.0 ** -126
    x[2, 34] = -(2.0 ** -128)
    x[3] = -0.0
    x[4, 5] = torch.inf
    x[4, 33] = 2.0
    x[5, 40] = -torch.inf
    x[6, 9] = torch.nan
    x[7, 2], x[7, 3] = torch.nan, torch.inf
    x[8] = 2.0 ** -124
    x[9, ::2] = torch.linspace(-8, 8, 32)
    check_quantize(x.cuda() if dim == -1 else x.T.contiguous().cuda(), dim)
    y = torch.zeros(2, 64, dtype=torch.float16)
    y[0, :4] = torch.tensor([65504.0, -6e-8, 1.0, 3e4])
    y[1, 3] = 6e-8
    y[1, 32:36] = torch.tensor([5 * 2.0 ** -24, 2.0 ** -24, -(2.0 ** -23), 3 * 2.0 ** -24])
    check_quantize(y.cuda() if dim == -1 else y.T.contiguous().cuda(), dim)


def test_quantize_strides():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 50, 70, generator=g).cuda()
    for view in (x[:, 3:40, 5:60], x.transpose(1, 2), x[::2], x[:, ::3, ::2], x.permute(2, 0, 1),
                 x[0, 0].expand(4, 70), x.flatten()[1:3301].view(60, 55), x.bfloat16()[:, :, 1:66]):
        for dim in (-1, -2):
            got, want = mx_quantize(view, dim), mx_quantize(view.contiguous(), dim)
            assert torch.equal(got.data, want.data) and torch.equal(got.scale, want.scale)


def test_quantize_empty():
    for shape, dim in (((0, 40), -1), ((0, 40, 8), -2), ((3, 0), -1), ((2, 0, 8), -2), ((2, 40, 0), -2)):
        q = mx_quantize(torch.zeros(shape, device="cuda"), dim)
        assert q.dequantize().shape == shape


# ------------------------------------------------------------------ product
def make(T, K, N, E, k, dtype, rows="token", seed=0):
    g = torch.Generator().manual_seed(seed)
    lead = {"token": (T,), "route": (T, k), "shared": (T, k // 2)}[rows]
    x = torch.randn(*lead, K, generator=g).to(dtype)
    keys = torch.randn(E, K, N, generator=g) / max(1, K) ** 0.5
    sel = torch.randint(0, E, (T, k), generator=g)
    return x, keys, sel, torch.rand(T, k, generator=g)


def expected(x, keys, sel, w, out_dtype):
    """(exact output, tolerance)."""
    E, K, N = keys.shape
    xv = view3(x, -1)
    xq = O.mx_values(*O.mx_quantize(xv), K)[0]
    wq = O.mx_values(*O.mx_quantize(view3(keys, -2)), K)
    per_row = sel.numel() // max(1, xq.shape[0])
    s, ww = sel.numpy(), None if w is None else w.double().numpy()
    out, size, y = O.mx_product(xq, s, wq, ww, per_row)
    half = torch.finfo(out_dtype).eps / 2
    acc = (K / 32 + 8) * 2.0 ** -23
    # fp16 results below 2^-14 are rounded to a fixed step
    low = 2.0 ** -25 if out_dtype == torch.float16 else 1e-37
    if w is None:
        return out, acc * size * (1 + half) + half * np.abs(out) + low
    route = (np.abs(y) * np.abs(ww)[..., None]).sum(-2)
    k = ww.shape[-1]
    tol = acc * size + half * route + (k + 1) * 2.0 ** -23 * route + low * (1 + np.abs(ww).sum(-1, keepdims=True))
    return out, tol * (1 + half) + half * np.abs(out)


def check_product(x, keys, sel, w=None, autocast=None):
    kq = mx_quantize(keys.cuda(), dim=-2)
    with torch.autocast("cuda", dtype=autocast or torch.bfloat16, enabled=autocast is not None):
        out = cvmm_mx(x.cuda(), sel.cuda(), kq, None if w is None else w.cuda())
    want_dtype = autocast or (torch.bfloat16 if x.dtype == torch.float32 else x.dtype)
    assert out.dtype == want_dtype
    assert out.shape == (*sel.shape[:-1], *((sel.shape[-1],) if w is None else ()), keys.shape[2])
    exact, tol = expected(x, keys, sel, w, out.dtype)
    err = np.abs(out.cpu().double().numpy() - exact)
    assert (err <= tol).all(), f"{(err / tol).max()} of the tolerance"
    assert _lib.device_status()[0] == 0
    return out


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("rows", ["token", "route", "shared"])
@pytest.mark.parametrize("T,K,N,E,k", [
    (1, 64, 64, 4, 2), (1, 512, 256, 16, 8), (3, 200, 74, 7, 4), (33, 31, 5, 3, 2), (100, 1, 1, 2, 2),
    (140, 128, 128, 5, 2), (70, 257, 129, 6, 6), (300, 96, 264, 2, 2), (20, 1056, 520, 40, 4), (17, 384, 1000, 1, 2),
])
def test_product_matches_64_bit(dtype, weighted, rows, T, K, N, E, k):
    x, keys, sel, w = make(T, K, N, E, k, dtype, rows, seed=T + K)
    check_product(x, keys, sel, w if weighted else None)


@pytest.mark.parametrize("T,K,N,E,k,weighted", [(2000, 512, 320, 8, 3, False), (1500, 256, 640, 64, 8, True),
                                                 (4, 4096, 136, 3, 2, True),
                                                 (9000, 160, 104, 8, 3, False), (9000, 544, 128, 5, 3, True)])
def test_product_larger(T, K, N, E, k, weighted):
    x, keys, sel, w = make(T, K, N, E, k, torch.bfloat16, seed=5)
    check_product(x, keys, sel, w if weighted else None)


def test_product_one_expert_takes_all_and_same_expert_twice():
    x, keys, sel, w = make(400, 160, 96, 9, 3, torch.bfloat16)
    check_product(x, keys, torch.full_like(sel, 8), w)
    sel[:, 1] = sel[:, 0]
    check_product(x, keys, sel, w)
    check_product(x, keys, sel)


def test_product_types_of_sel_and_weights_and_autocast():
    x, keys, sel, w = make(50, 96, 40, 5, 4, torch.float32)
    base = check_product(x, keys, sel, w)
    kq = mx_quantize(keys.cuda(), dim=-2)
    assert torch.equal(cvmm_mx(x.cuda(), sel.int().cuda(), kq, w.cuda()), base)
    assert torch.equal(cvmm_mx(x.cuda(), cvmm_prepare_sel2(sel.cuda(), w.cuda()), kq), base)
    for wt in (torch.bfloat16, torch.float16):
        check_product(x, keys, sel, w.to(wt))
    check_product(x, keys, sel, w, autocast=torch.float16)
    check_product(x, keys, sel, None, autocast=torch.bfloat16)
    check_product(x.half(), keys, sel, None, autocast=torch.bfloat16)


def test_product_strides():
    x, keys, sel, w = make(30, 64, 48, 4, 3, torch.bfloat16)
    kq = mx_quantize(keys.cuda(), dim=-2)
    want = cvmm_mx(x.cuda(), sel.cuda(), kq, w.cuda())
    wide = torch.zeros(30, 100, dtype=torch.bfloat16, device="cuda")
    wide[:, 3:67] = x.cuda()
    tall = x.cuda().T.contiguous().T
    selw = torch.zeros(30, 7, dtype=torch.int64, device="cuda")
    selw[:, 2:5] = sel.cuda()
    ww = torch.zeros(30, 6, device="cuda")
    ww[:, ::2] = w.cuda()
    for xv in (wide[:, 3:67], tall):
        assert torch.equal(cvmm_mx(xv, selw[:, 2:5], kq, ww[:, ::2]), want)
    x3 = x.cuda().view(5, 6, 64)
    assert torch.equal(cvmm_mx(x3, sel.cuda().view(5, 6, 3), kq, w.cuda().view(5, 6, 3)).view(30, 48), want)


def test_product_empty():
    _, keys, _, _ = make(1, 64, 48, 4, 3, torch.bfloat16)
    kq = mx_quantize(keys.cuda(), dim=-2)
    x, sel = torch.zeros(0, 64, device="cuda"), torch.zeros(0, 3, dtype=torch.int64, device="cuda")
    assert cvmm_mx(x, sel, kq).shape == (0, 3, 48)
    assert cvmm_mx(x, sel, kq, torch.zeros(0, 3, device="cuda")).shape == (0, 48)


def test_ids_out_of_range_contribute_nothing():
    x, keys, sel, w = make(60, 64, 48, 4, 3, torch.bfloat16)
    sel[3, 1], sel[10, 0], sel[11] = -1, 4, 1 << 40
    kq = mx_quantize(keys.cuda(), dim=-2)
    _lib.device_status()
    for ww in (None, w):
        out = cvmm_mx(x.cuda(), sel.cuda(), kq, None if ww is None else ww.cuda())
        assert _lib.device_status()[0] == 2
        exact, tol = expected(x, keys, sel, ww, out.dtype)
        assert (np.abs(out.cpu().double().numpy() - exact) <= tol).all()


def test_not_a_number_stays_in_its_row_and_column():
    x, keys, sel, w = make(40, 96, 48, 3, 2, torch.bfloat16)
    x[5, 70] = torch.nan
    x[6, 1] = torch.inf
    keys[1, 40, 7] = torch.nan
    out = cvmm_mx(x.cuda(), sel.cuda(), mx_quantize(keys.cuda(), dim=-2)).cpu()
    bad = torch.zeros(40, 2, 48, dtype=torch.bool)
    bad[5:7] = True
    bad[..., 7] |= sel == 1
    assert torch.equal(torch.isnan(out), bad)


def test_extreme_scales():
    """Rows and weights whose scales multiply far from one, without leaving the output's range."""
    x, keys, sel, _ = make(50, 128, 40, 3, 2, torch.float32)
    x = x * torch.exp2(torch.randint(-60, 60, (50, 1), generator=torch.Generator().manual_seed(3)).float())
    check_product(x, keys, sel)
    check_product(x * 2.0 ** -30, keys * 2.0 ** 30, sel)


def test_captured_on_other_streams_and_two_at_once():
    x, keys, sel, w = make(200, 320, 200, 12, 4, torch.bfloat16)
    x2, _, sel2, w2 = make(200, 320, 200, 12, 4, torch.bfloat16, seed=9)
    kq = mx_quantize(keys.cuda(), dim=-2)
    a, c = (x.cuda(), sel.cuda(), w.cuda()), (x2.cuda(), sel2.cuda(), w2.cuda())
    f = lambda t: cvmm_mx(t[0], t[1], kq, t[2])  # noqa: E731
    wa, wc = f(a), f(c)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            got.append((f(a), wa))
        with torch.cuda.stream(s2):
            got.append((f(c), wc))
    torch.cuda.synchronize()
    assert all(torch.equal(g, e) for g, e in got)
    static = tuple(t.clone() for t in a)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = f(static)
    with torch.cuda.graph(g2):
        o2 = f(static)
    for src, want in ((c, wc), (a, wa)):
        for t, v in zip(static, src):
            t.copy_(v)
        g1.replay()
        with torch.cuda.stream(s1):
            s1.wait_stream(torch.cuda.default_stream())
            g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(o1, want) and torch.equal(o2, want)


def test_many_routes_captured():
    """More routes than one block lists: the call's own reset of its counters is part of the graph."""
    x, keys, sel, w = make(1700, 96, 72, 40, 3, torch.bfloat16)
    kq = mx_quantize(keys.cuda(), dim=-2)
    static = (x.cuda(), sel.cuda(), w.cuda())
    want = check_product(x, keys, sel, w)
    other = check_product(x, keys, (sel + 7) % 40, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cvmm_mx(static[0], static[1], kq, static[2])
    for s, e in ((sel, want), ((sel + 7) % 40, other), (sel, want)):
        static[1].copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, e)


def test_many_experts():
    x, keys, sel, w = make(90, 40, 24, 3000, 3, torch.float16)
    check_product(x, keys, sel, w)
    x, keys, sel, w = make(2000, 40, 24, 4096, 3, torch.float16)
    check_product(x, keys, sel)
    with pytest.raises(ValueError, match="4096"):
        cvmm_mx(torch.zeros(1, 8, device="cuda"), torch.zeros(1, 1, dtype=torch.int64, device="cuda"),
                mx_quantize(torch.zeros(4097, 8, 8, device="cuda"), dim=-2))


def test_same_bits_every_time():
    x, keys, sel, w = make(900, 512, 256, 16, 4, torch.bfloat16)
    kq = mx_quantize(keys.cuda(), dim=-2)
    t = (x.cuda(), sel.cuda(), kq, w.cuda())
    want = cvmm_mx(*t)
    assert all(torch.equal(cvmm_mx(*t), want) for _ in range(5))


def test_quantize_and_product_trace_without_a_graph_break():
    x, keys, sel, w = make(64, 96, 40, 4, 2, torch.bfloat16)
    kq = mx_quantize(keys.cuda(), dim=-2)
    xc, sc, wc = x.cuda(), sel.cuda(), w.cuda()

    def f(t):
        return cvmm_mx(t, sc, kq, wc), mx_quantize(t).dequantize(torch.bfloat16)

    want = f(xc)
    got = torch.compile(f, fullgraph=True)(xc)
    assert all(torch.equal(a, e) for a, e in zip(got, want))


def test_kept_weights_round_trip():
    """An MXTensor rebuilt from its parts is the same tensor."""
    _, keys, _, _ = make(1, 72, 33, 3, 2, torch.float32)
    q = mx_quantize(keys.cuda(), dim=-2)
    r = MXTensor(q.data.cpu().cuda(), q.scale.clone(), q.shape, dim=-2)
    assert torch.equal(r.dequantize(), q.dequantize()) and r.to("cpu").device.type == "cpu"
    assert repr(r).startswith("MXTensor(") and b.MXTensor is MXTensor


# ------------------------------------------------------------------ weighted sums are rounded once
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows", ["token", "route"])
@pytest.mark.parametrize("T,K,N,E,k", [(32, 512, 1024, 128, 8), (3, 200, 74, 7, 4), (33, 31, 5, 3, 2), (500, 96, 260, 5, 3),
                                       (700, 160, 640, 4, 5), (9000, 64, 128, 5, 3), (9000, 64, 100, 5, 3)])
def test_weighted_sum_is_rounded_once(dtype, rows, T, K, N, E, k):
    """`expected`'s tolerance without half a step of every route output: the sums alone, and one rounding."""
    x, keys, sel, w = make(T, K, N, E, k, dtype, rows, seed=T + N)
    out = cvmm_mx(x.cuda(), sel.cuda(), mx_quantize(keys.cuda(), dim=-2), w.cuda())
    xq = O.mx_values(*O.mx_quantize(view3(x, -1)), K)[0]
    wq = O.mx_values(*O.mx_quantize(view3(keys, -2)), K)
    exact, size, y = O.mx_product(xq, sel.numpy(), wq, w.double().numpy(), 1 if rows == "route" else k)
    route = (np.abs(y) * w.double().numpy()[..., None]).sum(-2)
    half = torch.finfo(out.dtype).eps / 2
    low = 2.0 ** -25 if out.dtype == torch.float16 else 1e-37
    tol = ((K / 32 + 8) * size + (k + 1) * route) * 2.0 ** -23 * (1 + half) + half * np.abs(exact) + low
    err = np.abs(out.cpu().double().numpy() - exact)
    assert (err <= tol).all(), f"{(err / tol).max()} of the tolerance"


@pytest.mark.parametrize("N", [8, 36, 37, 300, 640])
def test_weighted_sum_of_routes_past_the_16_bit_range(N):
    """Two routes of 64 * 256 * 4 = 65536, which fp16 does not hold, with weights 1/4 and 1/2: 49152 exactly."""
    x = torch.full((3, 64), 256.0, dtype=torch.float16, device="cuda")
    keys = mx_quantize(torch.full((2, 64, N), 4.0, device="cuda"), dim=-2)
    sel = torch.tensor([[0, 1], [1, 0], [1, 1]], device="cuda")
    w = torch.tensor([0.25, 0.5], device="cuda").expand(3, 2)
    out = cvmm_mx(x, sel, keys, w)
    assert out.dtype == torch.float16 and torch.equal(out, torch.full((3, N), 49152.0, dtype=torch.float16, device="cuda"))
    assert torch.isinf(cvmm_mx(x, sel, keys)).all()


# T, K, N, E, k, weighted: several 128-column tiles, whole and ragged, one and two tiles an SM
COLUMNS_128 = [(1600, 160, 384, 8, 3, False), (1600, 288, 370, 8, 3, True), (1600, 96, 200, 8, 3, True),
               (1600, 31, 374, 8, 3, False), (3300, 544, 384, 8, 3, False), (3300, 160, 380, 8, 3, True)]


@pytest.mark.parametrize("T,K,N,E,k,weighted", COLUMNS_128)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_product_of_several_128_column_tiles(T, K, N, E, k, weighted, dtype):
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert _lib.load().cvmm_mx_tile_columns(T * k, E, N, sms) == 128
    x, keys, sel, w = make(T, K, N, E, k, dtype, seed=N)
    check_product(x, keys, sel, w if weighted else None)


@pytest.mark.parametrize("T,weighted", [(4, False), (4, True), (2000, False), (2000, True)])
def test_recorded_launches(T, weighted):
    from cvmm_codex_b200 import ops
    x, keys, sel, w = make(T, 64, 48, 4, 3, torch.bfloat16)
    kq, args = mx_quantize(keys.cuda(), dim=-2), (x.cuda(), sel.cuda(), w.cuda() if weighted else None)
    rec = ops.Recorder()
    with rec:
        cvmm_mx(args[0], args[1], kq, args[2])
    assert rec.launches == 2 + (T * 3 > 4096) + weighted
