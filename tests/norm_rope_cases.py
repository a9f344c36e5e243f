"""Rows, tables and weights for the tests of normed and rotated heads, and their values and gradients in float64."""

from types import SimpleNamespace

import torch as t

POSITIONS = 200


def rows(n, hq, hkv, d, dtype, w_dtype=None, table_dtype=t.float32, device="cuda", seed=0, positions=None):
    """Projected rows of `n` tokens; w_dtype None: no weights. Positions lie inside and outside the tables."""
    gen = t.Generator(device="cpu").manual_seed(seed * 7919 + n * 31 + d)
    s = SimpleNamespace(n=n, hq=hq, hkv=hkv, d=d, eps=1e-5)
    s.qkv = (2.0 * t.randn(n, (hq + 2 * hkv) * d, generator=gen)).to(device).to(dtype)
    s.positions = (t.randint(-3, POSITIONS + 3, (n,), generator=gen) if positions is None else positions).to(device)
    angles = t.arange(POSITIONS, dtype=t.float64)[:, None] / 100.0 ** (t.arange(0, d, 2, dtype=t.float64) / d)
    s.cos, s.sin = angles.cos().to(table_dtype).to(device), angles.sin().to(table_dtype).to(device)
    s.q_weight = s.k_weight = None
    if w_dtype is not None:
        s.q_weight, s.k_weight = ((1.0 + 0.5 * t.randn(d, generator=gen)).to(w_dtype).to(device) for _ in range(2))
    s.grads = [t.randn(n, h, d, generator=gen).to(device).to(dtype) for h in (hq, hkv, hkv)]
    return s


def args(s):
    return (s.qkv, s.positions, s.cos, s.sin, s.hq, s.hkv, s.q_weight, s.k_weight, s.eps)


def angles_64(s):
    inside = ((s.positions >= 0) & (s.positions < len(s.cos)))[:, None, None]
    at = s.positions.clamp(0, len(s.cos) - 1).long()
    return t.where(inside, s.cos[at].double()[:, None], 1.0), t.where(inside, s.sin[at].double()[:, None], 0.0)


def turn(y, c, s, across=-1.0):
    a, b = y[..., 0::2], y[..., 1::2]
    return t.stack([c * a + across * s * b, s * a + c * b], -1).flatten(-2)


def heads_64(s):
    """(x, 1 / rms, weight) of the q and k heads, and the values."""
    x = s.qkv.double().unflatten(1, (-1, s.d))
    x, v = x[:, :s.hq + s.hkv], x[:, s.hq + s.hkv:]
    if s.q_weight is None:
        return x, t.ones_like(x[..., :1]), t.ones_like(x[:1]), v
    inv = 1.0 / t.sqrt((x * x).mean(-1, keepdim=True) + s.eps)
    w = t.cat([s.q_weight.double().expand(s.hq, -1), s.k_weight.double().expand(s.hkv, -1)])[None]
    return x, inv, w, v


def forward_64(s):
    """(q and k heads, the magnitudes that float32 rounds on the way, values)."""
    x, inv, w, v = heads_64(s)
    c, n = angles_64(s)
    y = x * inv * w
    return turn(y, c, n), turn(y.abs(), c.abs(), n.abs(), 1.0), v


def backward_64(s, grads):
    """(dx, its magnitudes, [(dw, its magnitudes)] for q and k) from gradients of q, k and v (None: zeros)."""
    x, inv, w, v = heads_64(s)
    c, n = angles_64(s)
    g = [t.zeros(s.n, h, s.d, dtype=t.float64, device=s.qkv.device) if y is None else y.double()
         for y, h in zip(grads, (s.hq, s.hkv, s.hkv))]
    up = t.cat(g[:2], 1)
    h, ha = turn(up, c, -n), turn(up.abs(), c.abs(), n.abs(), 1.0)
    if s.q_weight is None:
        return t.cat([h, g[2]], 1).flatten(1), t.cat([ha, g[2].abs()], 1).flatten(1), None
    unit = x * inv
    dx = inv * (h * w - unit * (h * w * unit).mean(-1, keepdim=True))
    da = inv * (ha * w.abs() + unit.abs() * (ha * w.abs() * unit.abs()).mean(-1, keepdim=True))
    sums = [(y[:, a:b].sum((0, 1)), z[:, a:b].sum((0, 1))) for y, z in (((h * unit), (ha * unit.abs())),)
            for a, b in ((0, s.hq), (s.hq, s.hq + s.hkv))]
    return t.cat([dx, g[2]], 1).flatten(1), t.cat([da, g[2].abs()], 1).flatten(1), sums
