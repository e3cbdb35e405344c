"""The lookup of tokens, the loss against a teacher's top logits and the adjusted logits in plain 64-bit numpy, from their
formulas, and how far f32 arithmetic may be off them."""
import numpy as np

U = 2.0 ** -24  # half a step of f32, relative to the value


def device_ints(v):
    """Whole numbers as the f32 array of the same bits, which is what the tests upload."""
    return np.ascontiguousarray(np.asarray(v, np.int32)).reshape(-1).view(np.float32)


def zipf(rng, vocab, shape):
    """Tokens whose frequency falls with their number."""
    return np.minimum(np.floor(np.exp(rng.random(shape) * np.log(vocab + 1))) - 1, vocab - 1).astype(np.int64)


def valid(tokens, vocab):
    return (tokens >= 0) & (tokens < vocab)


def embed(table, tokens, scale):
    there = valid(tokens, len(table))
    return np.where(there[:, None], table[np.where(there, tokens, 0)].astype(np.float64) * scale, 0.0)


def embed_grad(tokens, dy, scale, vocab):
    """The gradient, and what the sums of every row may be off: a value passes the additions of its piece (8 to 64 places; 256 tokens
    are one) and those of the pieces of its run, and the product with the scale rounds once more."""
    there = valid(tokens, vocab)
    want, size = np.zeros((vocab, dy.shape[1])), np.zeros((vocab, dy.shape[1]))
    np.add.at(want, tokens[there], dy[there].astype(np.float64))
    np.add.at(size, tokens[there], np.abs(dy[there].astype(np.float64)))
    run = np.bincount(tokens[there], minlength=vocab)
    roundings = np.minimum(run, 256) + np.ceil(run / 8) + 2
    return want * scale, 1.01 * U * roundings[:, None] * size * abs(scale) + 2.0 ** -149


def softmax(x):
    """Probabilities of every row and their logarithms.  A row of -inf only is NaN."""
    with np.errstate(all="ignore"):
        m = x.max(1, keepdims=True)
        d = x - m
        total = np.exp(d).sum(1, keepdims=True)
        return np.exp(d) / total, d - np.log(total)


def distill(z, teacher, index, labels, weight, T, soft, hard, g=None):
    """loss and gradient of every row, and how far off f32 may be.

    An exponential of x = (z - largest) / T is off by U (6 + 4 |x|), relatively: its function 2 ulp, and roundings of z - largest,
    1 / T and the product.  A row's sum of them has 60 further roundings on a value's way at most in joins of lanes, warps and blocks, each
    with an exponential, and those of its thread: an addition for every 1024 tokens, and a product with an exponential where the largest
    value changes, at most for every 4096.  p has the same terms with fewer additions."""
    z = z.astype(np.float64)
    rows, vocab = z.shape
    top = index.shape[1]
    w = np.ones(rows) if weight is None else weight.astype(np.float64)
    g = np.ones(rows) if g is None else g.astype(np.float64)
    loss, off = np.zeros(rows), np.zeros(rows)
    sums = 66 + vocab / 1024 + 6 * vocab / 4096
    dz, doff = np.zeros((rows, vocab)), np.zeros((rows, vocab))
    if soft == 0 or top == 0:
        soft, T = 0.0, 1.0
    with np.errstate(all="ignore"):
        q, log_q = softmax(z / T)
        s, log_s = softmax(z)
        x, x1 = np.abs((z - z.max(1, keepdims=True)) / T), np.abs(z - z.max(1, keepdims=True))
        for i in range(rows):
            if w[i] == 0:
                continue
            there = valid(index[i], vocab)
            t = np.where(there, teacher[i].astype(np.float64) / T, -np.inf)
            e = np.exp(t - t.max()) if there.any() and t.max() > -np.inf else np.zeros(top)
            taught, labelled = bool(soft != 0 and e.sum() != 0), bool(hard != 0 and labels is not None and valid(labels[i], vocab))
            spread = np.nansum(q[i] * np.where(np.isfinite(x[i]), x[i], 0))
            sum_q = U * (sums + 4 * spread)
            spread1 = np.nansum(s[i] * np.where(np.isfinite(x1[i]), x1[i], 0))
            sum_s = U * (sums + 4 * spread1)
            if taught:
                p = e / e.sum()
                at = index[i][there & (p > 0)]
                pp = p[there & (p > 0)]
                kl = np.sum(pp * (np.log(pp) - log_q[i, at]))
                loss[i] += soft * T * T * kl
                gap = np.abs(np.log(pp) - log_q[i, at])
                xt = np.abs((t - t.max())[there & (p > 0)])
                off[i] += soft * T * T * (np.sum(2 * pp * U * (6 + 4 * xt) * (gap + gap.max(initial=0))) + U * (6 + 4 * np.sum(pp * xt)) + sum_q)
                dz[i] += soft * T * q[i]
                doff[i] += soft * T * q[i] * (sum_q + U * (12 + 4 * np.where(np.isfinite(x[i]), x[i], 0)))
                for j, token in enumerate(index[i]):
                    if there[j]:
                        dz[i, token] -= soft * T * p[j]
                        xj = abs(t[j] - t.max()) if p[j] > 0 else 0.0
                        doff[i, token] += soft * T * p[j] * U * (40 + 4 * xj + 4 * np.sum(pp * xt) + top)
            if labelled:
                loss[i] -= hard * log_s[i, labels[i]]
                off[i] += hard * sum_s
                dz[i] += hard * s[i]
                doff[i] += hard * s[i] * (sum_s + U * (12 + 4 * np.where(np.isfinite(x1[i]), x1[i], 0)))
                dz[i, labels[i]] -= hard
                doff[i, labels[i]] += hard * 6 * U
            loss[i] *= w[i]
            off[i] = abs(w[i]) * off[i] + 2 * U * abs(loss[i]) + 2.0 ** -140
            dz[i] *= w[i] * g[i]
            doff[i] = abs(w[i] * g[i]) * doff[i] + 4 * U * np.abs(dz[i]) + 2.0 ** -125  # (below the smallest normal number exponentials are 0)
    return loss, off, dz, doff


def adjust(z, history, prompts, lengths, repetition, presence, frequency, bias_tokens, bias, allowed):
    """The adjusted logits and how far off f32 may be: a rounding each of the penalty, the counts' product, their sum and the biases'."""
    rows, vocab = z.shape
    v, off = z.astype(np.float64), np.zeros(z.shape)
    with np.errstate(all="ignore"):
        for i in range(rows):
            cols = history.shape[1]
            n = cols if lengths is None else min(max(int(lengths[i]), 0), cols)
            m = 0 if prompts is None else min(max(int(prompts[i]), 0), n)
            tokens = history[i, :n]
            seen = np.unique(tokens[valid(tokens, vocab)])
            r = 1.0 if repetition is None else float(repetition[i])
            v[i, seen] = np.where(v[i, seen] > 0, v[i, seen] / r, v[i, seen] * r)
            off[i, seen] += U * np.abs(v[i, seen])
            generated = tokens[m:]
            count = np.bincount(generated[valid(generated, vocab)], minlength=vocab).astype(np.float64)
            f, a = (0.0 if x is None else float(x[i]) for x in (frequency, presence))
            there = count > 0
            v[i, there] -= f * count[there] + a
            off[i, there] += 2 * U * (np.abs(f) * count[there] + abs(a)) + U * np.abs(v[i, there])
            if bias is not None:
                # (a token's biases are added up first)
                total, size, number = np.zeros(vocab), np.zeros(vocab), np.zeros(vocab)
                for token, b in zip(bias_tokens[i], bias[i]):
                    if 0 <= token < vocab:
                        total[token] += float(b)
                        size[token] += abs(float(b))
                        number[token] += 1
                on = number > 0
                v[i, on] += total[on]
                off[i, on] += U * (number * size)[on] + U * np.abs(v[i, on])
    off = 1.01 * off + 2.0 ** -149
    if allowed is not None:
        v = np.where(allowed, v, -np.inf)
    return v, off


def words_of(allowed):
    """[rows, vocab] truth values as the words of bits that the library reads."""
    rows, vocab = allowed.shape
    padded = np.zeros((rows, (vocab + 31) // 32 * 32), bool)
    padded[:, :vocab] = allowed
    return np.packbits(padded, axis=1, bitorder="little").view(np.uint32).view(np.int32)


def assert_near(got, want, off, what=""):
    """Infinities and NaNs where the formula has them, everything else within `off`."""
    got = np.asarray(got, np.float64).reshape(want.shape)
    # what rounds to f32 beyond its largest number (2^128 - 2^104; the border is half a step above it) is infinite there
    want = np.where(np.abs(want) >= 2.0 ** 128 - 2.0 ** 103, np.copysign(np.inf, want), want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (what, np.argwhere(np.isnan(got) != np.isnan(want))[:5])
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), what
    fine = np.isfinite(want)
    assert np.isfinite(got[fine]).all(), what
    bad = np.abs(got[fine] - want[fine]) > np.broadcast_to(off, want.shape)[fine]
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(fine)[bad][:5], got[fine][bad][:5], want[fine][bad][:5],
                           np.broadcast_to(off, want.shape)[fine][bad][:5])
