"""The product with 4-bit weights against its definition in 64 bits.

Tolerance, per output, before any output rounding: with S = sum_i |a_i w_i|, the kernels add at most
`adds` terms one after another in f32 (the matrix instructions' steps of 16 inputs within a group,
three of them for f32 activations, then one per group and a few across warps), each off by at
most 2^-23 of a partial sum that S bounds (the matrix unit may truncate), and an f32 activation is
represented to 2^-22. The activation function's slope is at most 1.1, its own f32 steps cost at most
2^-20 of the value. Then half a step of the output type, relative to the value; for f16 below 2^-14
half a step is 2^-25.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def types():
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def weights(ctx, n, k, group, zeros, seed):
    """A handle and the weights in 64 bits."""
    from telmo_b200 import PackedWeights, Precision
    from test_q4 import decode
    g = np.random.default_rng(seed)
    groups = -(-k // group)
    values = g.integers(0, 256, (n, -(-k // 2)), dtype=np.uint8)
    scales = ((g.random((n, groups)) + 0.5) * g.choice([0.01, 0.1, 1.0], (n, groups))).astype(np.float16)
    scales = (scales * g.choice([1, 1, 1, -1], (n, groups))).astype(np.float32)
    z = g.integers(0, 16, (n, groups), dtype=np.uint8) if zeros else None
    p = PackedWeights(n, k, Precision.Q4, values, scales, zeros=z, group=group)
    return p.upload(ctx), decode(p)


def reference(a, w, bias, act, scale, c0):
    y = a @ w.T
    if bias is not None:
        y = y + bias
    if act == "RELU":
        y = np.maximum(y, 0)
    elif act == "SILU":
        y = y / (1 + np.exp(-y))
    y = y * scale
    return y if c0 is None else y + c0


def bound(a, w, y, bias, scale, c0, group, out):
    k = a.shape[1]
    adds = 3 * group / 16 + -(-k // 128) * (128 // group) + 16
    s = np.abs(a) @ np.abs(w).T
    b = 1.1 * abs(scale) * (s * (adds * 2.0 ** -23 + 2.0 ** -22) + (0 if bias is None else np.abs(bias) * 2.0 ** -24))
    b = b + np.abs(y) * 2.0 ** -20 + (0 if c0 is None else np.abs(c0) * 2.0 ** -23)
    half = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}[out]
    return b + (np.abs(y) + b) * half + (2.0 ** -25 if out == "f16" else 1e-37)


def run(ctx, m, n, k, group=32, zeros=False, dtype="f32", out="f32", act="NONE", scale=1.0, with_bias=False,
        accumulate=False, lda=None, ldc=None, offset=0, seed=0, stream=None):
    import torch
    from telmo_b200 import Act, Epilogue, Kernels
    t = types()
    dev, w = weights(ctx, n, k, group, zeros, seed)
    g = torch.Generator().manual_seed(seed + 1)
    lda, ldc = lda or k, ldc or n
    store = torch.randn(offset + m * lda + 8, generator=g).to(t[dtype]).cuda()
    a = store[offset:offset + m * lda].view(m, lda)
    c = torch.randn((m, ldc), generator=g).to(t[out]).cuda()
    before = c.clone()
    bias = torch.randn(n, generator=g).cuda() if with_bias else None
    Kernels(ctx).matmul(a, lda, m, dev, c, ldc, Epilogue(bias=bias, act=Act[act], scale=scale, accumulate=accumulate),
                        stream=stream)
    ctx.check(stream)
    av = a[:, :k].double().cpu().numpy()
    bv = None if bias is None else bias.double().cpu().numpy()
    c0 = before[:, :n].double().cpu().numpy() if accumulate else None
    y = reference(av, w, bv, act, scale, c0)
    off = np.abs(c[:, :n].double().cpu().numpy() - y)
    assert (off <= bound(av, w, y, bv, scale, c0, group, out)).all(), float(off.max())
    assert torch.equal(c[:, n:], before[:, n:])  # what lies between the rows stays as it was
    dev.free()


ROWS = [1, 2, 3, 8, 9, 17, 31, 32, 33, 64, 65, 130, 257]


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_rows_types_groups(ctx, m, dtype, group, zeros):
    n, k = (130, 1000) if m % 2 else (257, 1024)
    run(ctx, m, n, k, group, zeros, dtype, dtype, with_bias=bool(m % 3), seed=m)


@pytest.mark.parametrize("n,k", [(1, 1), (1, 128), (7, 31), (15, 32), (16, 33), (17, 127), (31, 129), (33, 255),
                                 (129, 640), (640, 2049), (2049, 97)])
@pytest.mark.parametrize("m", [1, 5, 20, 40, 150])
@pytest.mark.parametrize("dtype,out,group,zeros", [("f32", "f32", 32, True), ("bf16", "f32", 128, False),
                                                   ("f16", "f16", 64, True), ("f32", "bf16", 64, False)])
def test_odd_sizes(ctx, n, k, m, dtype, out, group, zeros):
    run(ctx, m, n, k, group, zeros, dtype, out, seed=n + k)


@pytest.mark.parametrize("m", [1, 4, 19, 70])
@pytest.mark.parametrize("act,scale,with_bias,accumulate", [
    ("NONE", 0.5, True, True), ("RELU", 1.0, True, False), ("SILU", 2.0, True, True), ("SILU", 1.0, False, False),
    ("RELU", -1.5, False, True)])
@pytest.mark.parametrize("dtype,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
def test_epilogues(ctx, m, act, scale, with_bias, accumulate, dtype, out):
    run(ctx, m, 150, 300, 32, True, dtype, out, act, scale, with_bias, accumulate, seed=m)


@pytest.mark.parametrize("m", [1, 3, 12, 24, 50, 200])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lda,ldc,offset", [(1001, 151, 0), (1001, 150, 1), (1000, 152, 3), (1004, 150, 2),
                                            (1008, 160, 8)])
def test_strides_and_alignment(ctx, m, dtype, lda, ldc, offset):
    run(ctx, m, 150, 1000, 64, True, dtype, dtype, lda=lda, ldc=ldc, offset=offset, seed=lda)


@pytest.mark.parametrize("m,n,k,group", [(1, 4096, 4096, 128), (8, 1024, 4096, 32), (32, 2049, 1024, 64),
                                         (300, 4096, 1024, 32), (1024, 1024, 4096, 128)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_model_sizes(ctx, m, n, k, group, dtype):
    run(ctx, m, n, k, group, True, dtype, "f32", with_bias=True, seed=n)


@pytest.mark.parametrize("m", [1, 2, 8, 30, 100, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_a_row_that_is_not_finite_stays_alone(ctx, m, dtype):
    import torch
    from telmo_b200 import Kernels
    n, k = 70, 200
    dev, w = weights(ctx, n, k, 32, True, 5)
    a = torch.randn((m, k), generator=torch.Generator().manual_seed(6)).to(types()[dtype]).cuda()
    clean, c = (torch.empty((m, n), device="cuda") for _ in range(2))
    Kernels(ctx).linear(a, m, dev, clean)
    for bad in (float("nan"), float("inf"), -float("inf")):
        b = a.clone()
        b[m // 2, 77] = bad
        Kernels(ctx).linear(b, m, dev, c)
        ctx.check()
        assert not torch.isfinite(c[m // 2]).any()
        keep = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(c[keep], clean[keep])
    dev.free()


@pytest.mark.parametrize("m", [1, 16, 100])
def test_f32_activations_of_very_different_size(ctx, m):
    """Rows from 2^-100 to 2^100 and a row with one large value: each row keeps its own accuracy."""
    import torch
    from telmo_b200 import Kernels
    n, k = 64, 512
    dev, w = weights(ctx, n, k, 128, False, 9)
    a = torch.randn((m, k), generator=torch.Generator().manual_seed(1))
    a *= torch.exp2(torch.linspace(-100, 100, m))[:, None] if m > 1 else 2.0 ** -100
    a[m // 2, 3] *= 1e5
    c = torch.empty((m, n), device="cuda")
    Kernels(ctx).linear(a.cuda(), m, dev, c)
    ctx.check()
    av = a.double().numpy()
    y = av @ w.T
    off = np.abs(c.double().cpu().numpy() - y)
    assert (off <= bound(av, w, y, None, 1.0, None, 128, "f32")).all()
    dev.free()


def test_no_rows_and_refusals(ctx):
    import torch
    from telmo_b200 import Epilogue, Kernels, TelmoError, _lib
    kern = Kernels(ctx)
    dev, _ = weights(ctx, 40, 64, 32, False, 1)
    a = torch.randn((4, 64), device="cuda")
    c = torch.full((4, 40), 3.0, device="cuda")
    kern.linear(a, 0, dev, c)
    ctx.check()
    assert (c == 3).all()
    bad = [
        lambda: kern.linear(a.double(), 4, dev, c),
        lambda: kern.linear(a, 4, dev, c.double()),
        lambda: kern.linear(a.cpu(), 4, dev, c),
        lambda: kern.linear(a, 5, dev, c),
        lambda: kern.linear(a[:, :63], 4, dev, c),
        lambda: kern.matmul(a, 63, 4, dev, c, 40),
        lambda: kern.matmul(a, 64, 4, dev, c, 39),
        lambda: kern.linear(a, 4, dev, c[:, :39]),
        lambda: kern.linear(a, 4, dev, c, Epilogue(bias=torch.zeros(39, device="cuda"))),
        lambda: kern.linear(a, 4, dev, c, Epilogue(bias=torch.zeros(40, device="cuda").bfloat16())),
        lambda: kern.linear_q(c, c, 64, c, 4, dev, c, 40),
    ]
    for call in bad:
        with pytest.raises(TelmoError):
            call()
    L, h, s = _lib.load(), ctx.handle, None
    pa, pc = a.data_ptr(), c.data_ptr()
    arg = _lib.TELMO_ERR_ARGUMENT
    assert L.telmo_linear_q4(h, pa, 2, 64, 4, dev.handle, None, 0, 1.0, 0, pc, 0, 40, s) == arg
    assert L.telmo_linear_q4(h, pa, 0, 64, 4, dev.handle, None, 0, 1.0, 0, pc, 2, 40, s) == arg
    assert L.telmo_linear_q4(h, pa, 0, 64, 4, dev.handle, None, 3, 1.0, 0, pc, 0, 40, s) == arg
    assert L.telmo_linear_q4(h, pa + 2, 0, 64, 4, dev.handle, None, 0, 1.0, 0, pc, 0, 40, s) == arg
    assert L.telmo_linear_q4(h, pa, 1, 64, 4, dev.handle, None, 0, 1.0, 0, pc + 1, 1, 40, s) == arg
    assert L.telmo_linear_q4(h, None, 0, 64, 4, dev.handle, None, 0, 1.0, 0, pc, 0, 40, s) == arg
    assert L.telmo_linear_q4(h, pa, 0, 64, 4, dev.handle, None, 0, 1.0, 0, None, 0, 40, s) == arg
    assert L.telmo_linear_noalloc(h, pa, 64, 4, dev.handle, None, 0, 1.0, 0, pc, 0, 40, s) == _lib.TELMO_ERR_UNSUPPORTED
    v = np.zeros((4, 32), np.uint8)
    sc = np.ones((4, 2), np.float32)
    out = __import__("ctypes").c_void_p()

    def upload(n=4, k=64, group=32, codes=v.ctypes.data, scales=sc.ctypes.data, zeros=None):
        return L.telmo_weights_upload_q4(h, n, k, group, codes, scales, zeros, __import__("ctypes").byref(out))
    for more in ({"n": 0}, {"k": 0}, {"group": 16}, {"codes": None}, {"scales": None}):
        assert upload(**more) == arg and not out.value
    for wrong in (0.1, np.nan, np.inf, 1e6):
        s2 = sc.copy()
        s2[3, 1] = wrong
        assert upload(scales=s2.ctypes.data) == arg and not out.value
    z = np.full((4, 2), 16, np.uint8)
    assert upload(zeros=z.ctypes.data) == arg and not out.value
    assert (c == 3).all()
    dev.free()


def test_columns_and_overlaps_are_refused(ctx):
    """A bias that is a column, transposed activations, rows other than the view's, and outputs that overlap."""
    import torch
    from telmo_b200 import Epilogue, Kernels, TelmoError
    kern = Kernels(ctx)
    dev, _ = weights(ctx, 40, 64, 32, False, 1)
    store = torch.randn((64, 128), device="cuda")
    c = torch.zeros((4, 40), device="cuda")
    before = store.clone()
    for call in (lambda: kern.linear(store[:4, :64].contiguous(), 4, dev, c, Epilogue(bias=store[:40, 0])),
                 lambda: kern.matmul(store.t(), 64, 4, dev, c, 40), lambda: kern.matmul(store[:, :64], 64, 4, dev, c, 40),
                 lambda: kern.matmul(store, 128, 4, dev, store[0, 63:], 128),
                 lambda: kern.matmul(store[0, 39:], 128, 4, dev, store, 128),
                 lambda: kern.matmul(store, 128, 4, dev, store[1], 64), lambda: kern.matmul(store, 128, 1, dev, store, 40)):
        with pytest.raises(TelmoError):
            call()
    ctx.check()
    assert torch.equal(store, before) and not c.any()
    kern.matmul(store[:, :64], 128, 4, dev, c, 40)
    kern.matmul(store[:, :64], 128, 4, dev, store[:, 64:104], 128)  # side by side
    ctx.check()
    assert torch.equal(store[:4, 64:104], c) and torch.equal(store[:, 104:], before[:, 104:])
    assert torch.equal(store[:, :64], before[:, :64]) and torch.equal(store[4:], before[4:])


@pytest.mark.parametrize("m", [1, 24, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_streams_and_graphs(ctx, m, dtype):
    """On another stream; captured into two graphs that are replayed one after the other and at once."""
    import torch
    from telmo_b200 import Kernels
    n, k = 200, 515
    side = torch.cuda.Stream()
    run(ctx, m, n, k, 64, True, dtype, "f32", seed=3, stream=side)
    kern = Kernels(ctx)
    dev, w = weights(ctx, n, k, 64, True, 4)
    inputs = [torch.randn((m, k), device="cuda").to(types()[dtype]) for _ in range(2)]
    outs = [torch.zeros((m, n), device="cuda") for _ in range(2)]
    want = [torch.zeros((m, n), device="cuda") for _ in range(2)]
    for x, y in zip(inputs, want):
        kern.linear(x, m, dev, y)
    torch.cuda.synchronize()
    graphs = []
    for x, y in zip(inputs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kern.linear(x, m, dev, y)
        graphs.append(g)
    for _ in range(3):
        for y in outs:
            y.zero_()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for y, e in zip(outs, want):
            assert torch.equal(y, e)
    del graphs
    dev.free()


def test_scales_are_f16_values(ctx):
    """Every finite f16 value is taken as a scale; its f32 neighbours are not."""
    from telmo_b200 import PackedWeights, Precision, TelmoError
    bits = np.arange(1 << 16, dtype=np.uint16)
    values = bits.view(np.float16).astype(np.float32)
    values = values[np.isfinite(values)]
    k = 32 * values.size
    codes = np.zeros((1, k // 2), np.uint8)
    PackedWeights(1, k, Precision.Q4, codes, values[None, :]).upload(ctx).free()
    some = np.concatenate([values[::3001], np.float32([2.0 ** -24, 65504.0, 2.0 ** -14, -2.0 ** -24])])
    for v in some[some != 0]:
        for wrong in (np.nextafter(v, np.float32(np.inf)), np.nextafter(v, np.float32(-np.inf))):
            with pytest.raises(TelmoError):
                PackedWeights(1, 32, Precision.Q4, codes[:, :16], np.float32([[wrong]])).upload(ctx)


@pytest.mark.parametrize("m,dtype", [(1, "f32"), (20, "f32"), (100, "f32"), (100, "bf16")])
def test_a_context_first_product_is_captured(m, dtype):
    """Nothing that a capture forbids is left to a product's first call."""
    import torch
    from telmo_b200 import Context, Kernels
    own = Context(0)
    n, k = 200, 300
    dev, w = weights(own, n, k, 32, False, 4)
    a = torch.randn((m, k), device="cuda").to(types()[dtype])
    c = torch.zeros((m, n), device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        Kernels(own).linear(a, m, dev, c)
    g.replay()
    own.check()
    av = a.double().cpu().numpy()
    y = av @ w.T
    assert (np.abs(c.double().cpu().numpy() - y) <= bound(av, w, y, None, 1.0, None, 32, "f32")).all()
    del g
    dev.free()
    own.close()


@pytest.mark.parametrize("m", [1, 2, 20, 100])
def test_long_rows(ctx, m):
    """Inputs beyond what shared memory holds of a row's digits, and an odd number of them."""
    run(ctx, m, 33, 30001, 128, True, "f32", "f32", seed=m)
    run(ctx, m, 17, 20000, 32, False, "bf16", "f32", seed=m)


def test_offsets_beyond_32_bits(ctx):
    """Rows of a and c whose offsets pass 2^31 elements, in each kernel's range of rows."""
    import torch
    from telmo_b200 import Kernels
    n, k = 40, 64
    dev, w = weights(ctx, n, k, 32, False, 8)
    for m, ld in ((2, (1 << 31) + 8), (9, (1 << 28) + 8), (33, (1 << 26) + 8)):
        store = torch.zeros((m - 1) * ld + k, dtype=torch.bfloat16, device="cuda")
        out = torch.zeros((m - 1) * ld + n, dtype=torch.bfloat16, device="cuda")
        rows = torch.randn((m, k), device="cuda").bfloat16()
        for r in range(m):
            store[r * ld:r * ld + k] = rows[r]
        Kernels(ctx).matmul(store, ld, m, dev, out, ld)
        ctx.check()
        av = rows.double().cpu().numpy()
        y = av @ w.T
        got = np.stack([out[r * ld:r * ld + n].double().cpu().numpy() for r in range(m)])
        assert (np.abs(got - y) <= bound(av, w, y, None, 1.0, None, 32, "bf16")).all()
        del store, out
    torch.cuda.empty_cache()
    dev.free()


@pytest.mark.parametrize("m", [2, 24, 130, 300])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_the_same_bits_again(ctx, m, dtype):
    """No sum depends on timing."""
    import torch
    from telmo_b200 import Kernels
    n, k = 1000, 2100
    dev, _ = weights(ctx, n, k, 64, True, 2)
    a = torch.randn((m, k), device="cuda").to(types()[dtype])
    first, again = (torch.empty((m, n), device="cuda") for _ in range(2))
    Kernels(ctx).linear(a, m, dev, first)
    for _ in range(5):
        again.zero_()
        Kernels(ctx).linear(a, m, dev, again)
        ctx.check()
        assert torch.equal(first, again)
    dev.free()


def test_two_streams_at_once(ctx):
    """Products on two streams whose workspaces are live at the same time."""
    import torch
    from telmo_b200 import Kernels
    n, k, m = 512, 1024, 400
    dev, _ = weights(ctx, n, k, 64, False, 6)
    kern = Kernels(ctx)
    a = [torch.randn((m, k), device="cuda") for _ in range(2)]
    want = [torch.empty((m, n), device="cuda") for _ in range(2)]
    for x, y in zip(a, want):
        kern.linear(x, m, dev, y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[torch.zeros((m, n), device="cuda") for _ in range(10)] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(10):
        for s in range(2):
            kern.linear(a[s], m, dev, got[s][i], stream=streams[s])
    torch.cuda.synchronize()
    ctx.check()
    for s in range(2):
        assert all(torch.equal(y, want[s]) for y in got[s])
    dev.free()


@pytest.mark.parametrize("m,k,dtype", [(12, 512, "f32"), (24, 515, "f16"), (40, 515, "bf16"), (300, 512, "f32")])
def test_each_product_reads_the_one_before(ctx, m, k, dtype):
    """A chain of products, each of whose activations are the output of the one before, gives the bits that it
    gives with a wait after each; captured too. (A product starts while its activations are still prepared.)"""
    import torch
    from telmo_b200 import Epilogue, Kernels
    devs = [weights(ctx, k, k, 32, True, s)[0] for s in range(3)]
    kern, t = Kernels(ctx), types()[dtype]
    x = torch.randn((m, k), device="cuda").to(t)
    # f16's last outputs underflow (each product is about a tenth of its activations): all outputs are compared.
    want, got = ([torch.zeros((m, k), device="cuda", dtype=t) for _ in range(13)] for _ in range(2))

    def chain(to, wait):
        to[0].copy_(x)
        for i in range(12):
            kern.linear(to[i], m, devs[i % 3], to[i + 1], Epilogue(scale=1e-3))
            if wait:
                torch.cuda.synchronize()
    chain(want, True)
    assert all(y.float().abs().max() > 0 for y in want[:4]) and all(torch.isfinite(y).all() for y in want)
    for _ in range(20):
        chain(got, False)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain(got, False)
    for _ in range(5):
        for y in got:
            y.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    ctx.check()
    del graph
    for d in devs:
        d.free()


def weights_without(ctx, n, k, j, seed):
    """Weights in which input j of every output is 0: its code is the zero point."""
    from telmo_b200 import PackedWeights, Precision
    from test_q4 import decode
    g = np.random.default_rng(seed)
    z = g.integers(0, 16, (n, -(-k // 32)), dtype=np.uint8)
    q = g.integers(0, 16, (n, 2 * -(-k // 2)), dtype=np.uint8)
    q[:, j] = z[:, j // 32]
    scales = (0.5 + g.random((n, -(-k // 32)))).astype(np.float16).astype(np.float32)
    p = PackedWeights(n, k, Precision.Q4, q[:, 0::2] | (q[:, 1::2] << 4), scales, zeros=z, group=32)
    assert (decode(p)[:, j] == 0).all()
    return p.upload(ctx), decode(p)


@pytest.mark.parametrize("m", [1, 2, 4, 8, 9, 16, 24, 33, 100, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("ratio", [10, 17, 24, 30, 38])
def test_a_large_activation_without_weight(ctx, m, dtype, ratio):
    """One activation 2^ratio times the others whose weights are 0, so the others alone decide. With A the row's
    largest, an activation enters the product to 2^-55 A (one or two rows, whatever the type), as it is (up to eight
    rows, and 16-bit types), or to the larger of 2^-22 of itself, which `bound` has, and 2^-39 A (more rows of f32)."""
    import torch
    from telmo_b200 import Kernels
    n, k, j = 40, 512, 77
    dev, w = weights_without(ctx, n, k, j, 3)
    a = torch.randn((m, k), generator=torch.Generator().manual_seed(ratio)).clamp(-4, 4)
    a[:, j] = 2.0 ** ratio
    a = a.to(types()[dtype])
    c = torch.empty((m, n), device="cuda")
    Kernels(ctx).linear(a.cuda(), m, dev, c)
    ctx.check()
    av = a.double().numpy()
    y = av @ w.T
    held = 2.0 ** -55 if m <= 2 else 2.0 ** -39 if m > 8 and dtype == "f32" else 0.0
    lim = bound(av, w, y, None, 1.0, None, 32, "f32") + np.abs(av).max(axis=1)[:, None] * held * np.abs(w).sum(axis=1)
    assert (np.abs(c.double().cpu().numpy() - y) <= lim).all()
    dev.free()


@pytest.mark.parametrize("m", [1, 2, 8, 16, 30, 100, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ["RELU", "SILU"])
def test_a_row_that_is_not_finite_under_an_activation_function(ctx, m, dtype, act):
    """Sums that are not finite, in that row alone: RELU makes 0 of -infinity, and nothing else is finite."""
    import torch
    from telmo_b200 import Act, Epilogue, Kernels
    n, k = 70, 200
    dev, w = weights(ctx, n, k, 32, True, 5)
    a = torch.randn((m, k), generator=torch.Generator().manual_seed(6)).to(types()[dtype]).cuda()
    clean, c = (torch.empty((m, n), device="cuda") for _ in range(2))
    epi = Epilogue(act=Act[act])
    Kernels(ctx).linear(a, m, dev, clean, epi)
    for bad in (float("nan"), float("inf"), -float("inf")):
        b = a.clone()
        b[m // 2, 77] = bad
        Kernels(ctx).linear(b, m, dev, c, epi)
        ctx.check()
        row = c[m // 2]
        assert (~torch.isfinite(row) | ((row == 0) & (act == "RELU"))).all()
        assert not np.isnan(bad) or row.isnan().all()
        keep = torch.arange(m, device="cuda") != m // 2
        assert torch.equal(c[keep], clean[keep])
    dev.free()


@pytest.mark.parametrize("m", [9, 33])
def test_rows_of_more_pieces_than_a_grid_is_high(ctx, m):
    """16-bit rows off 16-byte boundaries are copied in pieces of 2048: rows with more than 65535 of them. A few of the
    134 million weights are not 0, in the first, the last and the pieces around the last of a grid's."""
    import torch
    from telmo_b200 import Kernels, PackedWeights, Precision
    k = 65535 * 2048 + 2049
    at = np.array([0, 5, 2047, 2048, 65535 * 2048 - 1, 65535 * 2048, 65535 * 2048 + 77, k - 2, k - 1])
    codes = np.full((1, (k + 1) // 2), 0x88, np.uint8)
    for i, q in zip(at, range(9, 16 + len(at))):
        q = q if q < 16 else q - 16
        codes[0, i // 2] = codes[0, i // 2] & (0x0f if i & 1 else 0xf0) | (q << 4 if i & 1 else q)
    w = np.stack([codes[0, at // 2] & 15, codes[0, at // 2] >> 4])[at & 1, np.arange(len(at))].astype(np.float64) - 8
    assert (w != 0).all()
    dev = PackedWeights(1, k, Precision.Q4, codes, np.ones((1, -(-k // 128)), np.float32), group=128).upload(ctx)
    a = torch.ones((m, k), dtype=torch.bfloat16, device="cuda")
    a[:, torch.from_numpy(at).cuda()] = torch.randn((m, len(at)), generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    c = torch.zeros((m, 1), device="cuda")
    Kernels(ctx).linear(a, m, dev, c)
    ctx.check()
    av = a[:, torch.from_numpy(at).cuda()].double().cpu().numpy()
    # Every other product is exactly 0, and so are the sums without these inputs.
    lim = (np.abs(av) @ np.abs(w)) * len(at) * 2.0 ** -23
    assert (np.abs(c[:, 0].double().cpu().numpy() - av @ w) <= lim).all()
    dev.free()
    del a
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m", [1, 2, 5, 9, 20, 33, 130, 200, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_behind_the_last_stay_as_they_were(ctx, m, dtype):
    """A buffer of more rows than the call names, and rows of a that are not finite behind the last."""
    import torch
    from telmo_b200 import Kernels
    n, k = 300, 520
    dev, w = weights(ctx, n, k, 64, True, 7)
    a = torch.randn((m + 300, k), generator=torch.Generator().manual_seed(8)).to(types()[dtype]).cuda()
    a[m:] = float("nan")
    c = torch.full((m + 300, n), 5.0, device="cuda")
    Kernels(ctx).linear(a, m, dev, c)
    ctx.check()
    av = a[:m].double().cpu().numpy()
    y = av @ w.T
    assert (np.abs(c[:m].double().cpu().numpy() - y) <= bound(av, w, y, None, 1.0, None, 64, "f32")).all()
    assert (c[m:] == 5).all()
    dev.free()


@pytest.mark.parametrize("m", [1, 7, 12, 50])
@pytest.mark.parametrize("out", ["f32", "bf16"])
def test_the_general_entry_takes_the_handle(ctx, m, out):
    """telmo_linear with 4-bit weights gives what telmo_linear_q4 gives; a pair of int32 sums is refused."""
    import ctypes
    import torch
    from telmo_b200 import _lib
    L, n, k = _lib.load(), 130, 200
    dev, _ = weights(ctx, n, k, 64, True, 3)
    a = torch.randn((m, k + 3), device="cuda")
    bias = torch.randn(n, device="cuda")
    one, two = (torch.randn((m, n + 1), generator=torch.Generator().manual_seed(1)).to(types()[out]).cuda() for _ in range(2))
    dtype, stream = {"f32": 0, "bf16": 1}[out], torch.cuda.current_stream().cuda_stream
    assert L.telmo_linear(ctx.handle, a.data_ptr(), k + 3, m, dev.handle, bias.data_ptr(), 2, 0.5, 1, one.data_ptr(), dtype,
                          n + 1, stream) == 0
    assert L.telmo_linear_q4(ctx.handle, a.data_ptr(), 0, k + 3, m, dev.handle, bias.data_ptr(), 2, 0.5, 1, two.data_ptr(),
                             dtype, n + 1, stream) == 0
    assert L.telmo_linear(ctx.handle, a.data_ptr(), k + 3, m, dev.handle, None, 0, 1.0, 0, one.data_ptr(), 2, n + 1,
                          stream) == _lib.TELMO_ERR_ARGUMENT
    ctx.check()
    assert torch.equal(one, two)
    rows, cols = ctypes.c_size_t(), ctypes.c_size_t()
    assert L.telmo_weights_shape(dev.handle, ctypes.byref(rows), ctypes.byref(cols)) == 0
    assert (rows.value, cols.value) == (n, k)
    dev.free()


@pytest.mark.parametrize("m", [1, 2, 5, 12, 24, 100])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [2.0 ** -130, 2.0 ** -110, 2.0 ** 100])
def test_rows_near_the_ends_of_the_range(ctx, m, dtype, size):
    """Rows of subnormal values, of the smallest normal ones and of very large ones, scaled by c's scale to about 1."""
    import torch
    from telmo_b200 import Epilogue, Kernels
    n, k = 70, 260
    dev, w = weights(ctx, n, k, 32, True, 11)
    a = (torch.randn((m, k), generator=torch.Generator().manual_seed(2)) * size).to(types()[dtype])
    scale = float(np.float32(min(1 / size, 2.0 ** 120)))
    c = torch.empty((m, n), device="cuda")
    Kernels(ctx).linear(a.cuda(), m, dev, c, Epilogue(scale=scale))
    ctx.check()
    av = a.double().numpy()
    y = av @ w.T * scale
    # Parts below 2^-126 may vanish, and sums are f32: an error of 2^-126 for each product of size 8 and scale 1 / size.
    lim = bound(av, w, y, None, scale, None, 32, "f32") + 2.0 ** -126 * scale * np.abs(w).sum(axis=1)
    assert (np.abs(c.double().cpu().numpy() - y) <= lim).all()
    dev.free()
