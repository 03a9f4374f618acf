"""64-bit oracles (numpy, CPU) of router_select, the microscaled 4-bit format and its expert product."""
import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


# ------------------------------------------------------------------ router
def scores(z, scoring):
    z = np.asarray(z, dtype=np.float64)
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            return 1 / (1 + np.exp(-z))
        m = np.nanmax(z, axis=-1, keepdims=True) if z.size else z
        p = np.exp(z - np.where(m == -np.inf, 0.0, m))
        total = p.sum(-1, keepdims=True)
        return p / np.where(total == 0, 1.0, total)


def _ranked(v):
    """Indices by descending value, NaN first, ties to the lowest index."""
    nan = np.isnan(v)
    return sorted(range(len(v)), key=lambda i: (not nan[i], 0.0 if nan[i] else -v[i], i))


def select(z, k, scoring="softmax", bias=None, n_groups=1, top_groups=None, group_score="max", renormalize=True,
           scale=1.0):
    """(weights float64 [T, k], sel [T, k]) for logits z [T, E]."""
    z = np.asarray(z, dtype=np.float64)
    T, E = z.shape
    top_groups = n_groups if top_groups is None else top_groups
    s = scores(z, scoring)
    by = s if bias is None else s + np.asarray(bias, dtype=np.float64)
    by = np.where(z == -np.inf, -np.inf, by)
    order = z if bias is None else by
    size = E // n_groups
    sel = np.zeros((T, k), dtype=np.int64)
    for t in range(T):
        allowed = range(E)
        if n_groups > 1:
            value = []
            for g in range(n_groups):
                part = (by if group_score == "top2" else order)[t, g * size:(g + 1) * size]
                top = part[_ranked(part)]
                extra = top[1] if group_score == "top2" and size > 1 and top[1] != -np.inf else 0.0
                value.append(top[0] + extra)
            best = set(_ranked(np.array(value))[:top_groups])
            allowed = [e for e in range(E) if e // size in best]
        v = np.array([order[t, e] for e in allowed])
        sel[t] = [allowed[i] for i in _ranked(v)[:k]]
    w = np.take_along_axis(s, sel, -1)
    if renormalize:
        total = w.sum(-1, keepdims=True)
        w = w / np.where(total < 1e-20, 1e-20, total)
    return scale * w, sel


def select_weights(z, sel, scoring, renormalize, scale):
    w = np.take_along_axis(scores(z, scoring), sel, -1)
    if renormalize:
        total = w.sum(-1, keepdims=True)
        w = w / np.where(total < 1e-20, 1e-20, total)
    return scale * w


def select_grad(z, sel, grad_w, scoring, renormalize, scale):
    """(gradient, sum of the magnitudes of the terms it is made of) w.r.t. z."""
    s = scores(z, scoring)
    w = np.take_along_axis(s, sel, -1)
    g = scale * np.asarray(grad_w, dtype=np.float64)
    size = np.abs(g)
    if renormalize:
        total = w.sum(-1, keepdims=True)
        held = np.where(total < 1e-20, 1e-20, total)
        size = (size + (size * w).sum(-1, keepdims=True) / held) / held
        g = (g - np.where(total < 1e-20, 0.0, (g * w).sum(-1, keepdims=True) / held)) / held
    gs, gsize = np.zeros_like(s), np.zeros_like(s)
    np.put_along_axis(gs, sel, g, -1)
    np.put_along_axis(gsize, sel, size, -1)
    if scoring == "softmax":
        return (s * (gs - (s * gs).sum(-1, keepdims=True)), s * (gsize + (s * gsize).sum(-1, keepdims=True)))
    return gs * s * (1 - s), gsize * s


# ------------------------------------------------------------------ microscaled 4-bit values
def mx_quantize(x):
    """(codes uint8 [.., 32 * groups], scale bytes [.., groups]) of x [.., K] along its last axis."""
    x = np.asarray(x, dtype=np.float64)
    K = x.shape[-1]
    groups = -(-K // 32)
    b = np.zeros((*x.shape[:-1], groups * 32))
    b[..., :K] = x
    b = b.reshape(*x.shape[:-1], groups, 32)
    with np.errstate(all="ignore"):
        amax = np.abs(b).max(-1)
        fine = np.isfinite(amax)
        e = np.where(fine & (amax > 0), np.frexp(np.where(fine, amax, 1.0))[1] - 1 - 2, -127)
        e = np.clip(e, -127, 127)
        v = np.where(fine[..., None], b * np.exp2(-e.astype(np.float64))[..., None], 0.0)
    a = np.minimum(np.abs(v), 6.0)
    # nearest of the eight values; between two equally near the one with the even code
    d = np.abs(a[..., None] - GRID)
    near = d.min(-1, keepdims=True)
    tied = d == near
    even = np.arange(8) % 2 == 0
    code = np.where((tied & even).any(-1), np.argmax(tied & even, -1), np.argmax(tied, -1))
    code = code + 8 * (np.signbit(v) & (a >= 0))
    scale = np.where(fine, e + 127, 255).astype(np.uint8)
    return code.reshape(*x.shape[:-1], groups * 32).astype(np.uint8), scale


def mx_values(codes, scale, K):
    v = GRID[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127))
    v = v.reshape(*codes.shape[:-1], -1, 32) * s[..., None]
    return v.reshape(codes.shape)[..., :K]


def mx_pack(codes, scale):
    """The data and scale bytes of codes [B, rows, 32 * groups], scale [B, rows, groups] in the library's layout."""
    data = codes[..., 0::2] | (codes[..., 1::2] << 4)
    B, rows, groups = scale.shape
    rp, kp = -(-rows // 128), -(-groups // 4)
    out = np.zeros((B, rp, kp, 32, 4, 4), dtype=np.uint8)
    for r in range(rows):
        for j in range(groups):
            out[:, r // 128, j // 4, r % 32, r % 128 // 32, j % 4] = scale[:, r, j]
    return data, out


def mx_product(x, sel, w, weights=None, per_row=1):
    """(out, sum of magnitudes of the products, route outputs) of quantised rows x [rows, K] with w [E, N, K] values.

    per_row: routes per row of x. Ids outside [0, E) contribute zeros."""
    R = sel.size
    ids = sel.reshape(-1)
    y = np.zeros((R, w.shape[1]))
    size = np.zeros_like(y)
    for e in range(w.shape[0]):
        r = np.nonzero(ids == e)[0]
        if r.size:
            y[r] = x[r // per_row] @ w[e].T
            size[r] = np.abs(x[r // per_row]) @ np.abs(w[e]).T
    y, size = y.reshape(*sel.shape, -1), size.reshape(*sel.shape, -1)
    if weights is None:
        return y, size, y
    return (y * weights[..., None]).sum(-2), (size * np.abs(weights)[..., None]).sum(-2), y
