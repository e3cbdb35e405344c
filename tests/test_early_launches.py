"""Launches that may start under their predecessor's end (programmatic dependent launch) are for grids whose blocks are all
resident at once (launch.cuh).  Calls are captured, not run, and the edges of the captured graph say which of their kernels start
early."""
import ctypes

import pytest

from katsu_b200 import cabi
from test_int8 import floats

PROGRAMMATIC, CLUSTER_DIMENSION, SMS = 1, 4, 16  # CU_GRAPH_DEPENDENCY_TYPE_, CU_LAUNCH_ATTRIBUTE_, CU_DEVICE_ATTRIBUTE_ of cuda.h
p, u = ctypes.c_void_p, ctypes.c_uint


class Edge(ctypes.Structure):  # CUgraphEdgeData
    _fields_ = [("ports", ctypes.c_ubyte * 2), ("type", ctypes.c_ubyte), ("reserved", ctypes.c_ubyte * 5)]


class Kernel(ctypes.Structure):  # CUDA_KERNEL_NODE_PARAMS_v2
    _fields_ = [("func", p), ("grid", u * 3), ("block", u * 3), ("shared", u), ("params", p), ("extra", p), ("kern", p), ("ctx", p)]


class Attribute(ctypes.Structure):  # CUlaunchAttribute
    _fields_ = [("id", ctypes.c_int), ("pad", ctypes.c_int), ("value", u * 16)]


class Config(ctypes.Structure):  # CUlaunchConfig
    _fields_ = [("grid", u * 3), ("block", u * 3), ("shared", u), ("stream", p), ("attrs", ctypes.POINTER(Attribute)), ("count", u)]


def early_launches(ctx, call):
    """(kernel, blocks, blocks that the device holds at once) of every kernel of `call` that starts early."""
    cuda = ctypes.CDLL("libcuda.so.1")

    def ok(name, *args):
        assert getattr(cuda, name)(*args) == 0, name

    stream, graph, count = p(), p(), ctypes.c_size_t(0)
    ctx.call("katsu_cuda_stream", ctypes.byref(stream))
    ok("cuStreamBeginCapture_v2", stream, 2)  # relaxed
    try:
        call()
    finally:
        ok("cuStreamEndCapture", stream, ctypes.byref(graph))
    ok("cuGraphGetEdges_v2", graph, None, None, None, ctypes.byref(count))
    ends, edges = [(p * count.value)() for _ in range(2)], (Edge * count.value)()
    ok("cuGraphGetEdges_v2", graph, *ends, edges, ctypes.byref(count))
    found = []
    for i in range(count.value):
        if edges[i].type != PROGRAMMATIC:
            continue
        k, value, held, sms = Kernel(), (u * 16)(), ctypes.c_int(0), ctypes.c_int(0)
        ok("cuGraphKernelNodeGetParams_v2", p(ends[1][i]), ctypes.byref(k))
        func, name = p(k.func), ctypes.c_char_p()
        if not k.func:
            ok("cuKernelGetFunction", ctypes.byref(func), p(k.kern))
        ok("cuFuncGetName", ctypes.byref(name), func)
        ok("cuGraphKernelNodeGetAttribute", p(ends[1][i]), CLUSTER_DIMENSION, value)
        blocks = k.grid[0] * k.grid[1] * k.grid[2]
        if value[0] > 1:
            dims = Attribute(CLUSTER_DIMENSION, 0, value)
            config = Config(k.grid, k.block, k.shared, None, ctypes.pointer(dims), 1)
            ok("cuOccupancyMaxActiveClusters", ctypes.byref(held), func, ctypes.byref(config))
            held.value *= value[0]
        else:
            ok("cuOccupancyMaxActiveBlocksPerMultiprocessor", ctypes.byref(held), func, ctypes.c_int(k.block[0]), ctypes.c_size_t(k.shared))
            ok("cuDeviceGetAttribute", ctypes.byref(sms), SMS, 0)
            held.value *= sms.value
        found.append((name.value.decode(), blocks, held.value))
    ok("cuGraphDestroy", graph)
    return found


def matmul(m, k, n):
    def calls(ctx, a):
        x, w, y = a(m * k), a(k * n), a(m * n)
        dx, dw = a(m * k), a(k * n)
        ctx.matmul_fwd(x, w, y, m, k, n)
        ctx.matmul_bwd(x, w, y, dx, dw, m, k, n)
    return calls


def conv(n, c, hw, k, r=3, stride=1, pad=1):
    def calls(ctx, a):
        out = (hw + 2 * pad - r) // stride + 1
        x, w, y = a(n * c * hw * hw), a(k * c * r * r), a(n * k * out * out)
        dx, dw = a(n * c * hw * hw), a(k * c * r * r)
        shape = (n, c, hw, hw, k, r, r, stride, pad)
        ctx.conv2d_fwd(x, w, y, *shape)
        ctx.conv2d_bwd(x, w, y, dx, dw, *shape)
    return calls


def norm(rows, cols, layer, gate_rows=0):
    def calls(ctx, a):
        x, h, r, n, dr, dn, dx, dh = (a(rows * cols) for _ in range(8))
        w, b, dw, db = a(cols), a(cols) if layer else None, [a(cols) for _ in range(2)], [a(cols) if layer else None for _ in range(2)]
        gate, dgate = (a(gate_rows * cols) if gate_rows else None for _ in range(2))
        ctx.block_norm_fwd(x, h, gate, gate_rows, w, b, w, b, 1.0, 1e-6, int(layer), r, n, rows, cols)
        ctx.block_norm_bwd(r, h, gate, gate_rows, w, b, w, 1.0, 1e-6, int(layer), dr, dn, dx, dh, dgate, dw[0], db[0], dw[1], db[1], rows, cols)
    return calls


def int8(m, k, n):
    def calls(ctx, a):
        x, w, wq, ws, y = a(m * k), a(k * n), a(floats(n, k)), a(n), a(m * n)
        ctx.int8_quantize_weights(w, wq, ws, k, n)
        ctx.int8_linear(x, wq, ws, None, y, m, k, n)
    return calls


def clip(sizes):
    def calls(ctx, a):
        g, w, norm_ = [a(s) for s in sizes], [a(s) for s in sizes], a(1)
        ctx.clip_grads(g, g, sizes, 1.0, norm_)
        ctx.sgd_step_clipped(w, g, sizes, 0.1, 1.0, norm_)
    return calls


CALLS = {
    "matmul 2048 x 2048 x 2048": matmul(2048, 2048, 2048), "matmul 300 x 20000 x 200": matmul(300, 20000, 200),
    "matmul 512 x 65536 x 10": matmul(512, 65536, 10), "matmul 1021 x 2047 x 515": matmul(1021, 2047, 515), "matmul 64 x 64 x 64": matmul(64, 64, 64),
    "conv 8 x 64 x 56, 64": conv(8, 64, 56, 64), "conv 4 x 512 x 14, 512": conv(4, 512, 14, 512), "conv 2 x 24 x 9, 40": conv(2, 24, 9, 40),
    "conv 16 x 128 x 56, 256": conv(16, 128, 56, 256), "conv 8 x 128 x 56, 128, stride 2": conv(8, 128, 56, 128, stride=2),
    "norm 3000 x 128": norm(3000, 128, False), "norm 4000 x 1367, layer": norm(4000, 1367, True, 5), "norm 2000 x 2048": norm(2000, 2048, False, 1),
    "norm 500 x 8192, layer": norm(500, 8192, True), "norm 300 x 16384": norm(300, 16384, False), "norm 700 x 5003": norm(700, 5003, False),
    "8 bits 2 x 4096 x 4096": int8(2, 4096, 4096), "8 bits 40 x 30000 x 24": int8(40, 30000, 24), "8 bits 2000 x 2048 x 2048": int8(2000, 2048, 2048),
    "8 bits 512 x 65536 x 10": int8(512, 65536, 10), "8 bits 30 x 131072 x 64": int8(30, 131072, 64),
    "clip a few": clip([864, 18432, 655360]), "clip many": clip([70001] * 400),
}


@pytest.mark.gpu
@pytest.mark.parametrize("which", CALLS)
def test_all_blocks_are_resident_at_once(which):
    ctx, buffers = cabi.Context(0), []

    def allocate(count):
        buffers.append(ctx.alloc(count))
        return buffers[-1]

    try:
        CALLS[which](ctx, allocate)  # (buffers, and a workspace of its size: the capture allocates nothing)
        ctx.sync()
        again = iter(buffers)
        found = early_launches(ctx, lambda: CALLS[which](ctx, lambda count: next(again)))
        assert [launch for launch in found if launch[1] > launch[2]] == []
        for pointer in buffers:
            ctx.free(pointer)
    finally:
        ctx.close()
