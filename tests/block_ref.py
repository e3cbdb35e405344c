"""The norms around a block, the clipped step and the 8-bit product in plain 64-bit numpy, from their formulas."""
import numpy as np


def norm(v, w, b, eps, layer):
    v = v.astype(np.float64)
    m = v.mean(1, keepdims=True) if layer else 0.0
    hat = (v - m) / np.sqrt(np.square(v - m).mean(1, keepdims=True) + eps)
    return hat * w.astype(np.float64) + (0.0 if b is None else b.astype(np.float64))


def gate_rows(gate, rows):
    return np.repeat(gate.astype(np.float64), rows // gate.shape[0], axis=0)


def forward(x, h, gate, post_w, post_b, pre_w, pre_b, scale, eps, layer):
    r = x.astype(np.float64)
    if h is not None:
        u = h.astype(np.float64) if post_w is None else norm(h, post_w, post_b, eps, layer)
        r = r + scale * (u if gate is None else gate_rows(gate, x.shape[0]) * u)
    return r, None if pre_w is None else norm(r, pre_w, pre_b, eps, layer)


def norm_vjp(v, w, g, eps, layer):
    """(dv, dw, db) of norm(v) under g, from the derivative of each step: mean, spread, quotient."""
    v, g, count = v.astype(np.float64), g.astype(np.float64), v.shape[1]
    w = w.astype(np.float64)
    c = v - v.mean(1, keepdims=True) if layer else v
    spread = np.sqrt(np.square(c).mean(1, keepdims=True) + eps)
    hat, a = c / spread, g * w
    d_spread = -(a * c).sum(1, keepdims=True) / spread ** 2
    dc = a / spread + d_spread * c / (count * spread)
    dv = dc - dc.mean(1, keepdims=True) if layer else dc
    return dv, (g * hat).sum(0), g.sum(0)


def backward(r, h, gate, post_w, post_b, pre_w, scale, eps, layer, dr, dn):
    out = {"dx": np.zeros(r.shape) if dr is None else dr.astype(np.float64)}
    if pre_w is not None:
        dv, out["dpre_w"], out["dpre_b"] = norm_vjp(r, pre_w, dn, eps, layer)
        out["dx"] = out["dx"] + dv
    if h is None:
        return out
    sd = scale * out["dx"]
    du = sd if gate is None else gate_rows(gate, r.shape[0]) * sd
    if post_w is None:
        u, out["dh"] = h.astype(np.float64), du
    else:
        u = norm(h, post_w, post_b, eps, layer)
        out["dh"], out["dpost_w"], out["dpost_b"] = norm_vjp(h, post_w, du, eps, layer)
    if gate is not None:
        out["dgate"] = (sd * u).reshape(gate.shape[0], -1, r.shape[1]).sum(1)
    return out


def quantize(v):
    """Rows of v: whole numbers and scales, f32 where the definition rounds to f32."""
    v = np.asarray(v, np.float32)
    with np.errstate(all="ignore"):
        largest = np.abs(v).max(1) if v.shape[1] else np.zeros(v.shape[0], np.float32)
        scale = np.where(np.isfinite(largest), largest / np.float32(127), np.float32(np.nan)).astype(np.float32)
        q = np.rint(v.astype(np.float64) / scale.astype(np.float64)[:, None])
    q = np.where((scale > 0)[:, None], np.clip(q, -127, 127), 0.0)
    return q.astype(np.int64), scale


def int8_product(xq, xs, wq, ws, bias):
    """xq [m, k], wq [n, k]: exact sums, then the formula in 64 bits."""
    y = (xq @ wq.T).astype(np.float64) * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    return y if bias is None else y + bias.astype(np.float64)
