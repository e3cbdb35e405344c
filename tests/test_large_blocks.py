"""The norms, the 8-bit product and clipping over more than 2^32 values: rows (tokens, channels) are independent, so the last ones of the
large call must equal, bit for bit, the same ones alone."""
import numpy as np
import pytest

from parity_util import REL_L2_TOL, rel_l2

pytestmark = pytest.mark.gpu

ROWS, TAIL = 1048583, 700


@pytest.fixture
def device():
    import torch

    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)

    class Device:
        @staticmethod
        def normal(*shape):
            return torch.randn(shape, generator=gen, device="cuda")

        @staticmethod
        def empty(*shape, dtype=torch.float32):
            return torch.empty(shape, device="cuda", dtype=dtype)

        sync = staticmethod(torch.cuda.synchronize)
        equal = staticmethod(torch.equal)

    yield Device
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows,cols", [(ROWS, 4100), (ROWS * 4, 1031)])
def test_norms(ctx, device, rows, cols):
    assert rows * cols > 2 ** 32
    x, h, w = device.normal(rows, cols), device.normal(rows, cols), device.normal(cols)
    r, n, rt, nt = device.empty(rows, cols), device.empty(rows, cols), device.empty(TAIL, cols), device.empty(TAIL, cols)
    p = lambda t: t.data_ptr()  # noqa: E731
    device.sync()
    ctx.block_norm_fwd(p(x), p(h), None, 0, p(w), None, p(w), None, 0.5, 1e-6, 0, p(r), p(n), rows, cols)
    ctx.block_norm_fwd(p(x[-TAIL:]), p(h[-TAIL:]), None, 0, p(w), None, p(w), None, 0.5, 1e-6, 0, p(rt), p(nt), TAIL, cols)
    ctx.sync()
    assert device.equal(r[-TAIL:], rt) and device.equal(n[-TAIL:], nt)
    # backward of the norm behind the sum: h in the place of its gradient, dx in that of x; n is scratch for the parts
    dn, dx, dh, dw, dwt = h, x, n, device.empty(cols), device.empty(cols)
    dn_tail, parts = dn[-TAIL:].clone(), np.zeros(cols)
    device.sync()
    ctx.block_norm_bwd(p(r), None, None, 0, None, None, p(w), 1.0, 1e-6, 0, None, p(dn), p(dx), None, None, None, None, p(dw), None, rows, cols)
    ctx.block_norm_bwd(p(rt), None, None, 0, None, None, p(w), 1.0, 1e-6, 0, None, p(dn_tail), p(nt), None, None, None, None, p(dwt), None, TAIL,
                       cols)
    ctx.sync()
    assert device.equal(dx[-TAIL:], nt)
    whole = dw.double().cpu().numpy()
    for i in range(0, rows, 1 << 18):
        m = min(1 << 18, rows - i)
        ctx.block_norm_bwd(p(r) + 4 * i * cols, None, None, 0, None, None, p(w), 1.0, 1e-6, 0, None, p(dn) + 4 * i * cols, p(dh), None, None, None,
                           None, p(dw), None, m, cols)
        ctx.sync()
        parts += dw.double().cpu().numpy()
    assert rel_l2(whole, parts) <= REL_L2_TOL


def test_clipping(ctx, device):
    count, ends = 2 ** 32 + 5, 1000
    g, w, norm = device.normal(count), device.normal(count), device.empty(1)
    total = sum(float((v.double() ** 2).sum()) for v in g.split(1 << 28)) ** 0.5
    before = [(g[s].clone(), w[s].clone()) for s in (slice(0, ends), slice(2 ** 31 - 500, 2 ** 31 + 500), slice(count - ends, count))]
    device.sync()
    ctx.sgd_step_clipped([w.data_ptr()], [g.data_ptr()], [count], 0.5, total / 4, norm.data_ptr())
    ctx.clip_grads([g.data_ptr()], [g.data_ptr()], [count], total / 4, norm.data_ptr())
    ctx.sync()
    assert abs(float(norm) - total) <= 2.0 ** -22 * total
    for s, (g0, w0) in zip((slice(0, ends), slice(2 ** 31 - 500, 2 ** 31 + 500), slice(count - ends, count)), before):
        assert float((g[s] - g0 / 4).abs().max()) <= 3 * 2.0 ** -24 * float(g0.abs().max())  # factor (and its neighbour), product
        assert device.equal(w[s], w0 - 0.5 * g[s])


@pytest.mark.parametrize("m,k,n", [(ROWS, 4100, 24), (70001, 64, 65600)])
def test_tokens(ctx, device, m, k, n):
    assert max(m * k, m * n) > 2 ** 32
    row = ctx.int8_row_bytes(k) // 4
    x, w, wq, ws = device.normal(m, k), device.normal(k, n), device.empty(n, row), device.empty(n)
    y, yt = device.empty(m, n), device.empty(TAIL, n)
    device.sync()
    ctx.int8_quantize_weights(w.data_ptr(), wq.data_ptr(), ws.data_ptr(), k, n)
    ctx.int8_linear(x.data_ptr(), wq.data_ptr(), ws.data_ptr(), None, y.data_ptr(), m, k, n)
    ctx.int8_linear(x[-TAIL:].data_ptr(), wq.data_ptr(), ws.data_ptr(), None, yt.data_ptr(), TAIL, k, n)
    ctx.sync()
    assert device.equal(y[-TAIL:], yt)


def test_channels(ctx, device):
    import torch

    k, n, m = 4100, ROWS, 3
    row = ctx.int8_row_bytes(k) // 4
    w, x = device.normal(k, n), device.normal(m, k)
    wq, ws, y = device.empty(n, row), device.empty(n), device.empty(m, n)
    last = w[:, -TAIL:].contiguous()
    wqt, wst, yt = device.empty(TAIL, row), device.empty(TAIL), device.empty(m, TAIL)
    device.sync()
    for weights, q, s, out, channels in ((w, wq, ws, y, n), (last, wqt, wst, yt, TAIL)):
        ctx.int8_quantize_weights(weights.data_ptr(), q.data_ptr(), s.data_ptr(), k, channels)
        ctx.int8_linear(x.data_ptr(), q.data_ptr(), s.data_ptr(), None, out.data_ptr(), m, k, channels)
    ctx.sync()
    assert device.equal(wq[-TAIL:].view(dtype=torch.int32), wqt.view(dtype=torch.int32))
    assert device.equal(ws[-TAIL:], wst) and device.equal(y[:, -TAIL:], yt)
