"""The two ends of a language model, as cases that can be timed and compared: the lookup of its tokens' rows and the gradient
of their table, the loss against a teacher's top logits with its gradient, and what a server does to logits before it picks
from them.

With `own` set, `run` calls the library as a host program does: `cabi.Context` on device buffers that the caller owns.
Otherwise it computes the same from elementary torch operations.  `exact` has the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

EMBED = ("embed_fwd", "embed_bwd", "int8_embed")
DISTILL = ("distill_fwd", "distill_bwd")

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
def _embed(kind, count, vocab, cols, **more):
    """count tokens, whose frequencies fall off as those of words do, and a table [vocab, cols]."""
    return dict(kind=kind, count=count, vocab=vocab, cols=cols, **more)


def _distill(kind, rows, vocab, top, temperature=2.0, hard=0.5, masked=0.1, **more):
    """masked: the share of rows of weight 0 (prompts, padding); hard: the share of the loss that is of the labels."""
    return dict(kind=kind, rows=rows, vocab=vocab, top=top, temperature=temperature, hard=hard, masked=masked, **more)


def _adjust(rows, vocab, history, biases=0, allowed=1.0, **more):
    """allowed: the share of the vocabulary that a grammar leaves; 1 for no grammar."""
    return dict(kind="adjust", rows=rows, vocab=vocab, history=history, biases=biases, allowed=allowed, **more)


def listed():
    return [
        # One token of a served model: the smallest call, all latency.
        _embed("embed_fwd", 1, 32768, 4096, name="embed_fwd_1x4096"),
        # A prompt or a training batch.
        _embed("embed_fwd", 8192, 65536, 4096, name="embed_fwd_8192x4096"),
        # A decoding batch of a model served in 8 bits, whose head's weights are its table too.
        _embed("int8_embed", 64, 65536, 4096, name="int8_embed_64x4096"),
        # Odd sizes; the head has left its own gradient in the table's already, and the lookup's is added.
        _embed("embed_bwd", 3001, 10007, 515, accumulate=True, name="embed_bwd_3001x515_added"),
        # A training batch: the gradient of the whole table is written.
        _embed("embed_bwd", 65536, 65536, 2048, accumulate=False, name="embed_bwd_65536x2048"),
        # The loss of four positions, as an evaluation or a small fine-tuning step asks for it.
        _distill("distill_fwd", 4, 131072, 64, masked=0.0, name="distill_fwd_4x131072"),
        # A training batch of 4096 positions: the loss alone (validation), and with its gradient (a training step).
        _distill("distill_fwd", 4096, 32768, 64, name="distill_fwd_4096x32768"),
        _distill("distill_bwd", 4096, 32768, 64, name="distill_bwd_4096x32768"),
        # Rows that start on no vector boundary, the teacher alone.
        _distill("distill_bwd", 511, 50021, 17, temperature=1.0, hard=0.0, name="distill_bwd_511x50021"),
        # One sequence that is being answered.
        _adjust(1, 32768, 500, name="adjust_1x32768"),
        # A decoding batch of long conversations under grammars, with biases.
        _adjust(64, 131072, 4096, biases=16, allowed=0.05, name="adjust_64x131072"),
        # Odd sizes, no grammar.
        _adjust(33, 50021, 1500, biases=7, name="adjust_33x50021"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _vocab(rng, lo=1000, hi=200000):
    vocab = _log(rng, lo, hi)
    return vocab // 64 * 64 if rng.random() < 0.6 else vocab


def _draw_embed(rng):
    kind = rng.choice(["embed_fwd", "embed_bwd", "embed_bwd", "int8_embed"])
    vocab, cols = _vocab(rng), _log(rng, 16, 8192)
    if rng.random() < 0.6:
        cols = max(16, cols // 32 * 32)
    cols = max(16, min(cols, 2 ** 27 // vocab))
    count = min(_log(rng, 1, 100000), 2 ** 27 // cols)
    return _embed(kind, count, vocab, cols, **({"accumulate": rng.random() < 0.4} if kind == "embed_bwd" else {}))


def _draw_distill(rng):
    vocab = _vocab(rng)
    rows = min(_log(rng, 1, 16384), 2 ** 27 // vocab)
    return _distill(rng.choice(DISTILL), rows, vocab, _log(rng, 1, 200), rng.choice([1.0, 1.5, 2.0, 4.0]),
                    rng.choice([0.0, 0.3, 0.5]), rng.choice([0.0, 0.1, 0.4]))


def _draw_adjust(rng):
    vocab = _vocab(rng)
    rows = min(_log(rng, 1, 512), 2 ** 26 // vocab)
    return _adjust(rows, vocab, _log(rng, 1, 16384), rng.choice([0, 0, 3, 40]), rng.choice([1.0, 1.0, 0.5, 0.02]))


def draw(rng):
    return rng.choice([_draw_embed, _draw_embed, _draw_distill, _draw_distill, _draw_adjust])(rng)


def _distinct(count, vocab):
    """How many different tokens `count` draws of _tokens have, on average."""
    p = np.log1p(1.0 / np.arange(1, vocab + 1)) / math.log(vocab + 1)
    return float(-np.expm1(count * np.log1p(-p)).sum())


def work(case):
    kind, vocab = case["kind"], case["vocab"]
    if kind in EMBED:
        count, cols = case["count"], case["cols"]
        rows = _distinct(count, vocab) * cols
        if kind == "embed_bwd":
            table = 8 * rows if case["accumulate"] else 4 * vocab * cols
            return {"bytes": 4 * count * cols + table + 4 * count, "flops": 2 * count * cols}
        return {"bytes": 4 * count * cols + rows * (4 if kind == "embed_fwd" else 1) + 4 * count, "flops": count * cols}
    rows = case["rows"]
    if kind in DISTILL:
        read = rows - int(rows * case["masked"])
        small = 8 * rows * (case["top"] + 2)
        if kind == "distill_fwd":
            return {"bytes": 4 * read * vocab + small, "flops": 6 * read * vocab}
        return {"bytes": 4 * (read + rows) * vocab + small, "flops": 12 * read * vocab}
    values, grammar = rows * vocab, case["allowed"] < 1
    return {"bytes": 4 * values * (1 + case["allowed"]) + (values / 8 if grammar else 0) + 4 * rows * case["history"] + 8 * rows * case["biases"],
            "flops": 2 * values}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rand(gen, *shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(std).add_(mean)


def _tokens(gen, vocab, *shape):
    """Tokens whose frequency falls with their number, as that of words in text does with their rank."""
    u = torch.rand(shape, generator=gen, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(vocab + 1)).floor() - 1).clamp_(0, vocab - 1).to(torch.int32)


def _uniform(gen, lo, hi, *shape):
    return torch.rand(shape, generator=gen, device="cuda") * (hi - lo) + lo


def _prepare_embed(case, gen, state):
    kind, count, vocab, cols = case["kind"], case["count"], case["vocab"], case["cols"]
    state.update(tokens=_tokens(gen, vocab, count), scale=math.sqrt(cols))
    if kind == "embed_bwd":
        state["dy"] = _rand(gen, count, cols, std=0.01)
        state["dtable"] = _rand(gen, vocab, cols, std=0.01) if case["accumulate"] else torch.empty(vocab, cols, device="cuda")
        return state
    if kind == "embed_fwd":
        state["table"] = _rand(gen, vocab, cols, std=0.02)
    else:
        # as the 8-bit product keeps weights: one row of whole 16-byte units per output channel, and its scale
        state["q"] = torch.zeros(vocab, (cols + 15) // 16 * 16, device="cuda", dtype=torch.int8)
        state["q"][:, :cols] = torch.randint(-127, 128, (vocab, cols), generator=gen, device="cuda", dtype=torch.int8)
        state["ws"] = _uniform(gen, 2e-4, 8e-4, vocab)
    state["y"] = torch.empty(count, cols, device="cuda")
    return state


def _prepare_distill(case, gen, state):
    rows, vocab, top = case["rows"], case["vocab"], min(case["top"], case["vocab"])
    logits = _rand(gen, rows, vocab, std=2.0)
    # a teacher that agrees with the student in part, sharper than it
    teacher, index = torch.topk(_rand(gen, rows, vocab).add_(logits).mul_(1.3), top, dim=1)
    index = index.to(torch.int32)
    index[torch.rand(rows, top, generator=gen, device="cuda") < 0.02] = -1  # lists shorter than the longest are filled up
    labels = _tokens(gen, vocab, rows)
    labels[torch.rand(rows, generator=gen, device="cuda") < 0.05] = -100
    weight = torch.full((rows,), 1.0 / rows, device="cuda")
    weight[torch.randperm(rows, generator=gen, device="cuda")[: int(rows * case["masked"])]] = 0.0
    state.update(logits=logits, teacher=teacher.contiguous(), index=index.contiguous(), labels=labels, weight=weight,
                 temperature=case["temperature"], soft=1.0 - case["hard"], hard=case["hard"], top=top)
    state["loss"] = torch.empty(rows, device="cuda")
    if case["kind"] == "distill_bwd":
        state["g"] = _uniform(gen, 0.5, 1.5, rows)
        state["dlogits"] = torch.empty(rows, vocab, device="cuda")
    return state


def _prepare_adjust(case, gen, state):
    rows, vocab, history, biases = case["rows"], case["vocab"], case["history"], case["biases"]
    lengths = torch.randint(history // 2, history + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    state.update(logits=_rand(gen, rows, vocab, std=3.0), history=_tokens(gen, vocab, rows, history), lengths=lengths,
                 prompts=(lengths * _uniform(gen, 0.0, 1.0, rows)).to(torch.int32), repetition=_uniform(gen, 1.0, 1.3, rows),
                 presence=_uniform(gen, 0.0, 1.0, rows), frequency=_uniform(gen, 0.0, 0.5, rows),
                 out=torch.empty(rows, vocab, device="cuda"), bias_tokens=None, bias=None, words=None)
    if biases:
        state["bias_tokens"] = _tokens(gen, vocab, rows, biases)
        state["bias"] = _uniform(gen, -5.0, 5.0, rows, biases)
    if case["allowed"] < 1:
        bits = torch.rand(rows, (vocab + 31) // 32, 32, generator=gen, device="cuda") < case["allowed"]
        words = (bits.long() << torch.arange(32, device="cuda")).sum(2)
        state["words"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    make = _prepare_embed if case["kind"] in EMBED else _prepare_distill if case["kind"] in DISTILL else _prepare_adjust
    return make(case, gen, {"case": case})


# ---------------------------------------------------------------------------
# one pass: the plain forms
# ---------------------------------------------------------------------------
def _plain_embed_fwd(st):
    return st["table"][st["tokens"].long()] * st["scale"]


def _plain_int8_embed(st):
    tokens = st["tokens"].long()
    return st["q"][tokens, : st["case"]["cols"]].float() * st["ws"][tokens, None] * st["scale"]


def _plain_embed_bwd(st):
    sums = torch.zeros_like(st["dtable"]).index_add_(0, st["tokens"].long(), st["dy"])
    st["dtable"].copy_(st["dtable"] + sums * st["scale"] if st["case"]["accumulate"] else sums * st["scale"])
    return st["dtable"]


def _log_softmax(v):
    v = v - v.amax(1, keepdim=True)
    return v - v.exp().sum(1, keepdim=True).log()


def _teacher(st):
    """The teacher's probabilities over its listed tokens, and these; entries without a token have none."""
    there = st["index"] >= 0
    t = torch.where(there, st["teacher"] / st["temperature"], -torch.inf)
    e = torch.where(there, (t - t.amax(1, keepdim=True)).exp(), 0.0)
    return e / e.sum(1, keepdim=True).clamp_min(1e-30), st["index"].clamp_min(0).long()


def _plain_distill_fwd(st):
    p, at = _teacher(st)
    # differences of nearly equal logarithms: in 64 bits
    log_q = _log_softmax(st["logits"] / st["temperature"]).gather(1, at).double()
    loss = st["soft"] * st["temperature"] ** 2 * torch.where(p > 0, p.double() * (p.double().log() - log_q), 0.0).sum(1)
    if st["hard"]:
        label = st["labels"].long()
        at_label = _log_softmax(st["logits"]).gather(1, label.clamp_min(0)[:, None])[:, 0]
        loss = loss + st["hard"] * torch.where(label >= 0, -at_label, 0.0)
    return torch.where(st["weight"] != 0, loss * st["weight"], 0.0).float()


def _plain_distill_bwd(st):
    """The loss of every row and the gradient of its logits."""
    p, at = _teacher(st)
    q = _log_softmax(st["logits"] / st["temperature"]).exp() * (p.sum(1, keepdim=True) > 0)
    d = q.scatter_add(1, at, -p) * (st["soft"] * st["temperature"])
    if st["hard"]:
        label = st["labels"].long()
        there = (label >= 0)[:, None].float()
        d = d + st["hard"] * there * _log_softmax(st["logits"]).exp().scatter_add(1, label.clamp_min(0)[:, None], -there)
    d = torch.where((st["weight"] != 0)[:, None], d * (st["weight"] * st["g"])[:, None], 0.0)
    return {"loss": _plain_distill_fwd(st), "dlogits": d}


def _plain_adjust(st):
    z, at = st["logits"], torch.arange(st["case"]["history"], device="cuda")
    history, one = st["history"].long(), torch.ones((), device="cuda")
    past = (at < st["lengths"][:, None]).float()
    generated = past * (at >= st["prompts"][:, None])
    seen = torch.zeros_like(z).scatter_add_(1, history, past * one)
    count = torch.zeros_like(z).scatter_add_(1, history, generated * one)
    r = st["repetition"][:, None]
    v = torch.where(seen > 0, torch.where(z > 0, z / r, z * r), z)
    v = v - torch.where(count > 0, st["frequency"][:, None] * count + st["presence"][:, None], 0.0)
    if st["bias"] is not None:
        v = v.scatter_add(1, st["bias_tokens"].long(), st["bias"])
    if st["words"] is not None:
        bits = (st["words"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        v = torch.where(bits.reshape(z.shape[0], -1)[:, : z.shape[1]] != 0, v, -torch.inf)
    return v


# ---------------------------------------------------------------------------
# one pass: the library
# ---------------------------------------------------------------------------
def _at(t):
    return None if t is None else t.data_ptr()


def _own_embed_fwd(st):
    c = st["case"]
    _context().embed_fwd(_at(st["table"]), _at(st["tokens"]), st["scale"], _at(st["y"]), c["count"], c["vocab"], c["cols"])
    return st["y"]


def _own_int8_embed(st):
    c = st["case"]
    _context().int8_embed(_at(st["q"]), _at(st["ws"]), _at(st["tokens"]), st["scale"], _at(st["y"]), c["count"], c["vocab"], c["cols"])
    return st["y"]


def _own_embed_bwd(st):
    c = st["case"]
    _context().embed_bwd(_at(st["tokens"]), _at(st["dy"]), st["scale"], _at(st["dtable"]), c["count"], c["vocab"], c["cols"],
                         int(c["accumulate"]))
    return st["dtable"]


def _own_distill_fwd(st):
    c = st["case"]
    _context().distill_fwd(_at(st["logits"]), _at(st["teacher"]), _at(st["index"]), _at(st["labels"]), _at(st["weight"]),
                           st["temperature"], st["soft"], st["hard"], _at(st["loss"]), c["rows"], c["vocab"], st["top"])
    return st["loss"]


def _own_distill_bwd(st):
    c = st["case"]
    _context().distill_bwd(_at(st["logits"]), _at(st["teacher"]), _at(st["index"]), _at(st["labels"]), _at(st["weight"]),
                           st["temperature"], st["soft"], st["hard"], _at(st["g"]), _at(st["loss"]), _at(st["dlogits"]), c["rows"],
                           c["vocab"], st["top"])
    return {"loss": st["loss"], "dlogits": st["dlogits"]}


def _own_adjust(st):
    c = st["case"]
    _context().adjust_logits(_at(st["logits"]), _at(st["history"]), _at(st["prompts"]), _at(st["lengths"]), _at(st["repetition"]),
                             _at(st["presence"]), _at(st["frequency"]), _at(st["bias_tokens"]), _at(st["bias"]), _at(st["words"]),
                             _at(st["out"]), c["rows"], c["vocab"], c["history"], c["biases"])
    return st["out"]


_PLAIN = {"embed_fwd": _plain_embed_fwd, "embed_bwd": _plain_embed_bwd, "int8_embed": _plain_int8_embed,
          "distill_fwd": _plain_distill_fwd, "distill_bwd": _plain_distill_bwd, "adjust": _plain_adjust}
_OWN = {"embed_fwd": _own_embed_fwd, "embed_bwd": _own_embed_bwd, "int8_embed": _own_int8_embed,
        "distill_fwd": _own_distill_fwd, "distill_bwd": _own_distill_bwd, "adjust": _own_adjust}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _exact_distill(st, lo, hi, grad):
    """Rows lo to hi - 1: the loss of each, or its gradient, from the formula's terms."""
    z = st["logits"][lo:hi].double()
    at, t = st["index"][lo:hi].long(), st["teacher"][lo:hi].double() / st["temperature"]
    p = torch.where(at >= 0, torch.exp(t - t.amax(1, keepdim=True)), 0.0)
    mass = p.sum(1, keepdim=True)
    p = torch.where(mass > 0, p / mass, 0.0)
    label = st["labels"][lo:hi].long()
    w = st["weight"][lo:hi].double()
    if not grad:
        log_q = torch.log_softmax(z / st["temperature"], 1).gather(1, at.clamp(min=0))
        kl = (torch.special.xlogy(p, p) - p * log_q).sum(1)
        ce = torch.where(label >= 0, -torch.log_softmax(z, 1).gather(1, label.clamp(min=0)[:, None])[:, 0], 0.0)
        return w * (st["soft"] * st["temperature"] ** 2 * kl + st["hard"] * ce)
    row = torch.arange(hi - lo, device="cuda")
    d = torch.softmax(z / st["temperature"], 1) * (mass > 0)
    d.index_put_((row[:, None].expand_as(at), at.clamp(min=0)), -p, accumulate=True)
    d *= st["soft"] * st["temperature"]
    if st["hard"]:
        there = (label >= 0).double()
        e = torch.softmax(z, 1) * there[:, None]
        e[row, label.clamp(min=0)] -= there
        d += st["hard"] * e
    return d * (w * st["g"][lo:hi].double())[:, None]


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "embed_fwd":
        return torch.index_select(st["table"], 0, st["tokens"].long()).double() * st["scale"]
    if kind == "int8_embed":
        tokens = st["tokens"].long()
        return torch.index_select(st["q"], 0, tokens)[:, : case["cols"]].double() * (st["ws"].double() * st["scale"])[tokens][:, None]
    if kind == "embed_bwd":
        # a table of double precision, a slab of columns at a time
        out = []
        for dy, before in zip(st["dy"].split(256, 1), st["dtable"].split(256, 1)):
            sums = torch.zeros(before.shape, device="cuda", dtype=torch.float64)
            sums.index_put_((st["tokens"].long(),), dy.double() * st["scale"], accumulate=True)
            out.append(sums + before.double() if case["accumulate"] else sums)
        return torch.cat(out, 1)
    if kind in DISTILL:
        step = max(1, 2 ** 25 // case["vocab"])
        runs = [(lo, min(lo + step, case["rows"])) for lo in range(0, case["rows"], step)]
        loss = torch.cat([_exact_distill(st, lo, hi, False) for lo, hi in runs])
        if kind == "distill_fwd":
            return loss
        return {"loss": loss, "dlogits": torch.cat([_exact_distill(st, lo, hi, True) for lo, hi in runs])}
    rows, vocab = case["rows"], case["vocab"]
    v = st["logits"].double()
    for i in range(rows):
        n, m = int(st["lengths"][i]), int(st["prompts"][i])
        tokens = st["history"][i, :n].long()
        seen = torch.unique(tokens)
        r = st["repetition"][i].double()
        v[i, seen] = torch.where(v[i, seen] > 0, v[i, seen] / r, v[i, seen] * r)
        count = torch.bincount(tokens[m:], minlength=vocab).double()
        v[i] -= st["frequency"][i].double() * count + st["presence"][i].double() * (count > 0)
        if st["bias"] is not None:
            v[i] += torch.bincount(st["bias_tokens"][i].long(), weights=st["bias"][i].double(), minlength=vocab)
    if st["words"] is not None:
        at = torch.arange(vocab, device="cuda")
        words = st["words"].long() & 0xFFFFFFFF
        v[((words[:, at // 32] >> (at % 32)) & 1) == 0] = -torch.inf
    return v
