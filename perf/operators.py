"""What surrounds the products of a block, as cases that can be timed and compared: the norms before and after a block
with its gate and residual scale, the product in 8-bit integers, and the clipped SGD step over many tensors.

With `own` set, `run` calls the library as a host program does: `cabi.Context` on device buffers that the caller owns.
Otherwise it computes the same from elementary torch operations.  `exact` has the definitions in 64 bits.
"""
import math

import torch

own = False

NORM = ("norm_fwd", "norm_bwd")
CLIP = ("clip", "clip_step")

_contexts = {}


def _context():
    """One context for the whole process, as a host program keeps it."""
    from katsu_b200 import cabi

    device = torch.cuda.current_device()
    if device not in _contexts:
        _contexts[device] = cabi.Context(device)
    return _contexts[device]


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def _norm(kind, rows, cols, norm, gate, post=True, **more):
    """norm: rms or layer (with biases); gate: rows of the gate, 0 for none; post: a norm behind the block too."""
    return dict(kind=kind, rows=rows, cols=cols, norm=norm, gate=gate, post=post, **more)


def _clip(kind, sizes, clipped=True, **more):
    """sizes: the tensors' lengths, in groups `length x count`; clipped: whether the norm is above the limit."""
    return dict(kind=kind, sizes=sizes, clipped=clipped, **more)


def _int8(m, k, n, bias=True, **more):
    return dict(kind="int8_linear", m=m, k=k, n=n, bias=bias, **more)


def listed():
    return [
        # One token of a served model: the smallest call, all latency.
        _norm("norm_fwd", 1, 4096, "rms", 1, name="norm_fwd_1x4096"),
        # A prompt or a training batch: every token has its own gate.
        _norm("norm_fwd", 8192, 4096, "rms", 8192, name="norm_fwd_8192x4096"),
        # Backward of a training batch, the gate one value a channel (layer scale).
        _norm("norm_bwd", 16384, 2048, "rms", 1, name="norm_bwd_16384x2048"),
        # Odd sizes: layer norms with biases, seven sequences with a gate row each, rows that start on no vector boundary.
        _norm("norm_bwd", 1022, 1367, "layer", 7, name="norm_bwd_1022x1367_layer"),
        # The small CNN's parameters: three tensors, one step.
        _clip("clip_step", "864x1,18432x1,655360x1", name="clip_step_small_cnn"),
        # A stack of 24 blocks: 240 tensors, 1.2 GB of gradients.
        _clip("clip_step", "1024x96,1048576x96,4194304x48", name="clip_step_240_tensors"),
        # A flat bucket of odd tensors, as an all-reduce leaves it: clipped alone, for an optimizer of the caller's.
        _clip("clip", "333x40,70001x20,999983x9", name="clip_69_odd_tensors"),
        # A hidden layer for one token: the weights are read once.
        _int8(1, 4096, 4096, name="int8_1x4096x4096"),
        # The classifier head of the small CNN, served.
        _int8(512, 65536, 10, name="int8_512x65536x10"),
        # Sizes that are no multiple of anything.
        _int8(1021, 2047, 515, name="int8_1021x2047x515"),
        # The benchmark's square products.
        _int8(4096, 4096, 4096, bias=False, name="int8_4096"),
        _int8(8192, 8192, 8192, bias=False, name="int8_8192"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_norm(rng):
    kind = rng.choice(NORM)
    cols = _log(rng, 64, 16384)
    if rng.random() < 0.6:
        cols = max(64, cols // 64 * 64)
    rows = min(_log(rng, 1, 32768), 2 ** 25 // cols)
    gate = rng.choice([0, 1, rows])
    if rng.random() < 0.3:  # sequences of one length
        gate = rng.choice([2, 3, 5, 8, 16])
        rows = max(1, rows // gate) * gate
    return _norm(kind, rows, cols, rng.choice(["rms", "layer"]), gate, rng.random() < 0.7)


def _draw_clip(rng):
    groups, left = [], 2.0e8
    for _ in range(rng.randint(1, 4)):
        length = _log(rng, 1, 2e7)
        count = min(_log(rng, 1, 200), max(1, int(left / length)))
        left = max(1.0, left - length * count)
        groups.append("%dx%d" % (length, count))
    return _clip(rng.choice(CLIP), ",".join(groups), rng.random() < 0.8)


def _draw_int8(rng):
    m, k, n = _log(rng, 1, 8192), _log(rng, 64, 16384), _log(rng, 8, 16384)
    if rng.random() < 0.4:
        m = rng.randint(1, 16)
    if rng.random() < 0.6:
        k, n = max(64, k // 64 * 64), max(16, n // 16 * 16)
    while m * k * n > 5e11:
        m, k, n = (v // 2 + 1 if v == max(m, k, n) else v for v in (m, k, n))
    if rng.random() < 0.2:
        return dict(kind="int8_weights", k=k, n=n)
    return _int8(m, k, n, rng.random() < 0.5)


def draw(rng):
    return rng.choice([_draw_norm, _draw_norm, _draw_clip, _draw_int8, _draw_int8])(rng)


def _sizes(case):
    return [int(length) for part in case["sizes"].split(",") for length, count in [part.split("x")] for _ in range(int(count))]


def work(case):
    kind = case["kind"]
    if kind in NORM:
        values, cols = case["rows"] * case["cols"], case["cols"]
        weights = cols * (1 + case["post"]) * (1 + (case["norm"] == "layer")) + case["gate"] * cols
        if kind == "norm_fwd":  # x, h -> r, n
            return {"bytes": 4 * (4 * values + weights), "flops": 12 * values}
        return {"bytes": 4 * (6 * values + 2 * weights), "flops": 30 * values}  # r, h, dr, dn -> dx, dh
    if kind in CLIP:
        total = sum(_sizes(case))
        return {"bytes": 4 * total * (2 if kind == "clip" else 3), "flops": 4 * total}
    k, n = case["k"], case["n"]
    if kind == "int8_weights":
        return {"bytes": 5 * k * n + 4 * n, "flops": 3 * k * n}
    m = case["m"]
    return {"bytes": 4 * m * k + n * k + 4 * n * (1 + case["bias"]) + 4 * m * n, "flops": 2 * m * k * n}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rand(gen, *shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).add_(mean)


def _over_127(largest):
    """Divided by a tensor: by a number, torch multiplies with its reciprocal, which is another scale in the last bit."""
    return largest / torch.full_like(largest, 127.0)


def _quantized(w):
    """Weights [k, n] as the 8-bit product reads them: one row of whole 16-byte units per output channel, and its scale."""
    k, n = w.shape
    scale = _over_127(w.abs().amax(0))
    q = torch.zeros(n, (k + 15) // 16 * 16, device=w.device, dtype=torch.int8)
    q[:, :k] = torch.round(w.t().double() / scale.double()[:, None]).to(torch.int8)
    return q, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = case["kind"]
    state = {"case": case}
    if kind in NORM:
        rows, cols, layer = case["rows"], case["cols"], case["norm"] == "layer"
        # a residual stream has grown over the blocks before; a block's output has not
        stream = _rand(gen, rows, cols, std=3.0, mean=0.2)
        state.update(h=_rand(gen, rows, cols), scale=0.5, eps=1e-6)
        state["gate"] = _rand(gen, case["gate"], cols, std=0.3, mean=1.0) if case["gate"] else None
        for name in ("post", "pre"):
            here = name == "pre" or case["post"]
            state[name + "_w"] = _rand(gen, cols, std=0.2, mean=1.0) if here else None
            state[name + "_b"] = _rand(gen, cols, std=0.2) if here and layer else None
        if kind == "norm_fwd":
            state.update(x=stream, r=torch.empty_like(stream), n=torch.empty_like(stream))
            return state
        state.update(r=stream, dr=_rand(gen, rows, cols, std=0.01), dn=_rand(gen, rows, cols, std=0.01))
        for name in ("h", "gate", "post_w", "post_b", "pre_w", "pre_b"):
            state["d" + name] = None if state[name] is None else torch.empty_like(state[name])
        state["dx"] = torch.empty_like(stream)
        return state
    if kind in CLIP:
        sizes = _sizes(case)
        # one flat buffer, every tensor right behind the one before
        state.update(sizes=sizes, g=_rand(gen, sum(sizes), std=0.01), lr=0.05)
        state["grads"] = list(state["g"].split(sizes))
        state["max_norm"] = 0.01 * math.sqrt(sum(sizes)) * (0.3 if case["clipped"] else 3.0)
        state["norm"] = torch.empty((), device="cuda")
        if kind == "clip":
            state["out"] = torch.empty_like(state["g"])
        else:
            state["w"] = _rand(gen, sum(sizes), std=0.02)
        target = state["out"] if kind == "clip" else state["w"]
        state["targets"] = list(target.split(sizes))
        state["pointers"] = [[t.data_ptr() for t in state[name]] for name in ("grads", "targets")]
        return state
    w = _rand(gen, case["k"], case["n"], std=math.sqrt(1.0 / case["k"]))
    if kind == "int8_weights":
        state.update(w=w, q=torch.empty(case["n"], (case["k"] + 15) // 16 * 16, device="cuda", dtype=torch.int8),
                     ws=torch.empty(case["n"], device="cuda"))
        return state
    # activations with a few channels much larger than the rest
    loud = torch.where(torch.rand(case["k"], generator=gen, device="cuda") < 0.01, 8.0, 1.0)
    state["x"] = _rand(gen, case["m"], case["k"]) * loud
    state["wq"], state["ws"] = _quantized(w)
    state["bias"] = _rand(gen, case["n"], std=0.1) if case["bias"] else None
    state["y"] = torch.empty(case["m"], case["n"], device="cuda")
    return state


# ---------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------
def _hat(v, eps, layer):
    """The values without weights, and what they were multiplied by."""
    if layer:
        v = v - v.mean(1, keepdim=True)
    rstd = torch.rsqrt(v.square().mean(1, keepdim=True) + eps)
    return v * rstd, rstd


def _affine(v, w, b):
    return v * w if b is None else v * w + b


def _gate_rows(st):
    """The gate as it stands before every row: [gate rows, rows of each, cols]."""
    return st["gate"][:, None, :].expand(-1, st["h"].shape[0] // st["gate"].shape[0], -1).reshape(st["h"].shape)


def _plain_norm_fwd(st):
    layer = st["case"]["norm"] == "layer"
    u = st["h"] if st["post_w"] is None else _affine(_hat(st["h"], st["eps"], layer)[0], st["post_w"], st["post_b"])
    gated = u if st["gate"] is None else _gate_rows(st) * u
    r = st["x"] + st["scale"] * gated
    return {"r": r, "n": _affine(_hat(r, st["eps"], layer)[0], st["pre_w"], st["pre_b"])}


def _hat_vjp(g, hat, rstd, layer):
    inner = g - hat * (g * hat).mean(1, keepdim=True)
    return rstd * (inner - g.mean(1, keepdim=True) if layer else inner)


def _plain_norm_bwd(st):
    layer = st["case"]["norm"] == "layer"
    r_hat, r_rstd = _hat(st["r"], st["eps"], layer)
    dx = st["dr"] + _hat_vjp(st["dn"] * st["pre_w"], r_hat, r_rstd, layer)
    out = {"dx": dx, "dpre_w": (st["dn"] * r_hat).sum(0), "dpre_b": st["dn"].sum(0) if layer else None}
    du = st["scale"] * dx if st["gate"] is None else st["scale"] * _gate_rows(st) * dx
    u = st["h"]
    if st["post_w"] is None:
        out["dh"] = du
    else:
        h_hat, h_rstd = _hat(st["h"], st["eps"], layer)
        u = _affine(h_hat, st["post_w"], st["post_b"])
        out.update(dh=_hat_vjp(du * st["post_w"], h_hat, h_rstd, layer), dpost_w=(du * h_hat).sum(0))
        out["dpost_b"] = du.sum(0) if layer else None
    if st["gate"] is not None:
        out["dgate"] = (st["scale"] * dx * u).reshape(st["gate"].shape[0], -1, u.shape[1]).sum(1)
    return out


def _plain_clip(st):
    squares = torch.stack([g.square().sum(dtype=torch.float64) for g in st["grads"]])
    norm = squares.sum().sqrt().float()
    factor = torch.clamp(st["max_norm"] / norm, max=1.0)
    if st["case"]["kind"] == "clip":
        return {"norm": norm, "g": torch.cat([g * factor for g in st["grads"]])}
    st["w"].copy_(torch.cat([w - st["lr"] * (factor * g) for w, g in zip(st["targets"], st["grads"])]))
    return {"norm": norm, "w": st["w"]}


def _quotients(v, scale):
    """v / scale to the nearest whole number, 0 where the scale is 0; in 64 bits, where no border is missed."""
    return torch.where(scale > 0, torch.round(v.double() / scale.double()), 0.0).clamp(-127, 127).float()


def _plain_int8_linear(st):
    x = st["x"]
    xs = _over_127(x.abs().amax(1, keepdim=True))
    y = (_quotients(x, xs) @ st["wq"][:, : x.shape[1]].float().t()) * xs * st["ws"]
    return y if st["bias"] is None else y + st["bias"]


def _plain_int8_weights(st):
    scale = _over_127(st["w"].abs().amax(0))
    return {"q": _quotients(st["w"], scale).t().contiguous().to(torch.int8), "scale": scale}


# ---------------------------------------------------------------------------
# one pass: the library
# ---------------------------------------------------------------------------
def _at(t):
    return None if t is None else t.data_ptr()


def _kind(st):
    from katsu_b200 import cabi

    return cabi.NORM_LAYER if st["case"]["norm"] == "layer" else cabi.NORM_RMS


def _own_norm_fwd(st):
    c = st["case"]
    _context().block_norm_fwd(_at(st["x"]), _at(st["h"]), _at(st["gate"]), c["gate"], _at(st["post_w"]), _at(st["post_b"]),
                              _at(st["pre_w"]), _at(st["pre_b"]), st["scale"], st["eps"], _kind(st), _at(st["r"]), _at(st["n"]),
                              c["rows"], c["cols"])
    return {"r": st["r"], "n": st["n"]}


def _own_norm_bwd(st):
    c = st["case"]
    _context().block_norm_bwd(_at(st["r"]), _at(st["h"]), _at(st["gate"]), c["gate"], _at(st["post_w"]), _at(st["post_b"]),
                              _at(st["pre_w"]), st["scale"], st["eps"], _kind(st), _at(st["dr"]), _at(st["dn"]), _at(st["dx"]),
                              _at(st["dh"]), _at(st["dgate"]), _at(st["dpost_w"]), _at(st["dpost_b"]), _at(st["dpre_w"]),
                              _at(st["dpre_b"]), c["rows"], c["cols"])
    names = ["dx", "dpre_w", "dpre_b", "dh", "dpost_w", "dpost_b", "dgate"]
    return {name: st[name] for name in names if st[name] is not None}


def _own_clip(st):
    grads, targets = st["pointers"]
    if st["case"]["kind"] == "clip":
        _context().clip_grads(grads, targets, st["sizes"], st["max_norm"], _at(st["norm"]))
        return {"norm": st["norm"], "g": st["out"]}
    _context().sgd_step_clipped(targets, grads, st["sizes"], st["lr"], st["max_norm"], _at(st["norm"]))
    return {"norm": st["norm"], "w": st["w"]}


def _own_int8_linear(st):
    c = st["case"]
    _context().int8_linear(_at(st["x"]), _at(st["wq"]), _at(st["ws"]), _at(st["bias"]), _at(st["y"]), c["m"], c["k"], c["n"])
    return st["y"]


def _own_int8_weights(st):
    c = st["case"]
    _context().int8_quantize_weights(_at(st["w"]), _at(st["q"]), _at(st["ws"]), c["k"], c["n"])
    return {"q": st["q"][:, : c["k"]], "scale": st["ws"]}


_PLAIN = {"norm_fwd": _plain_norm_fwd, "norm_bwd": _plain_norm_bwd, "clip": _plain_clip, "clip_step": _plain_clip,
          "int8_linear": _plain_int8_linear, "int8_weights": _plain_int8_weights}
_OWN = {"norm_fwd": _own_norm_fwd, "norm_bwd": _own_norm_bwd, "clip": _own_clip, "clip_step": _own_clip,
        "int8_linear": _own_int8_linear, "int8_weights": _own_int8_weights}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_norm(v, w, b, eps, layer):
    m = v.sum(1, keepdim=True) / v.shape[1] if layer else torch.zeros_like(v[:, :1])
    spread = torch.sqrt(((v - m) ** 2).sum(1, keepdim=True) / v.shape[1] + eps)
    out = (v - m) / spread * w
    return out if b is None else out + b


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind in NORM:
        if case["rows"] * case["cols"] > 5e7:
            return None
        layer = case["norm"] == "layer"
        names = [k for k in ("x", "h", "gate", "post_w", "post_b", "pre_w", "pre_b") if st.get(k) is not None]
        v = {k: st[k].double().requires_grad_(kind == "norm_bwd") for k in names}
        u = v["h"]
        if case["post"]:
            u = _exact_norm(u, v["post_w"], v.get("post_b"), st["eps"], layer)
        if case["gate"]:
            row = torch.arange(case["rows"], device="cuda") // (case["rows"] // case["gate"])
            u = u * v["gate"][row]
        if kind == "norm_fwd":
            r = v["x"] + st["scale"] * u
            return {"r": r, "n": _exact_norm(r, v["pre_w"], v.get("pre_b"), st["eps"], layer)}
        # the residual stream is given behind the addition: the part that the block added moves it, from zero
        moved = torch.zeros_like(u).requires_grad_()
        r = st["r"].double() + moved
        n = _exact_norm(r, v["pre_w"], v.get("pre_b"), st["eps"], layer)
        (n * st["dn"].double() + r * st["dr"].double()).sum().backward()
        (st["scale"] * u * moved.grad).sum().backward()
        return {"dx": moved.grad, **{"d" + k: v[k].grad for k in names}}
    if kind in CLIP:
        g = st["g"].double()
        norm = math.sqrt(float((g * g).sum()))
        c = 1.0 if norm <= st["max_norm"] else st["max_norm"] / norm
        norm_out = torch.tensor(norm, dtype=torch.float64, device="cuda")
        if kind == "clip":
            return {"norm": norm_out, "g": g * c}
        return {"norm": norm_out, "w": st["w"].double() - st["lr"] * c * g}
    if kind == "int8_weights":
        w = st["w"]
        scale = w.abs().max(0).values / torch.tensor(127.0, device="cuda")
        q = (w.double() / scale.double()).round().clamp(-127, 127)
        return {"q": q.t().contiguous().to(torch.int8), "scale": scale.double()}
    x = st["x"]
    scale = (x.abs().max(1).values / torch.tensor(127.0, device="cuda")).double()
    q = (x.double() / scale[:, None]).round().clamp(-127, 127)
    y = torch.matmul(q, st["wq"][:, : case["k"]].double().t()) * scale[:, None] * st["ws"].double()[None, :]
    return y if st["bias"] is None else y + st["bias"].double()
