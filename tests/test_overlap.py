"""Whether a call's matrices share memory (telmo_b200/csrc/overlap.h) against sets of bytes, and the calls that are
refused for it."""

import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

WRAPPER = """
#include "overlap.h"
using namespace telmo;
extern "C" int shares(size_t a, size_t ap, size_t ar, size_t an, size_t b, size_t bp, size_t br, size_t bn) {
    return overlap(Span{(const void*)a, ap, ar, an}, Span{(const void*)b, bp, br, bn});
}
extern "C" int shares_other(size_t a, size_t ap, size_t ar, size_t an, size_t b, size_t bp, size_t br, size_t bn) {
    return overlaps_other_rows(Span{(const void*)a, ap, ar, an}, Span{(const void*)b, bp, br, bn});
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    (d / "w.cpp").write_text(WRAPPER)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "telmo_b200", "csrc"), "-o",
                    str(d / "w.so"), str(d / "w.cpp")], check=True)
    L = ctypes.CDLL(str(d / "w.so"))
    for f in (L.shares, L.shares_other):
        f.argtypes = [ctypes.c_size_t] * 8
    return L


def row_bytes(p, pitch, row, rows):
    return [set(range(p + r * pitch, p + r * pitch + row)) for r in range(rows)]


def test_against_sets_of_bytes(lib):
    """Matrices of one pitch are judged to the byte; of two pitches, whatever shares a byte is found."""
    g = random.Random(1)
    seen = {}
    for _ in range(30000):
        rows = g.choice([1, 1, 2, 3, 5])
        ap, bp = g.randint(1, 9), g.randint(1, 9)
        if g.random() < 0.6:
            bp = ap
        a = (g.randint(100, 140), ap, g.randint(1, ap), rows)
        b = (g.randint(100, 140), bp, g.randint(1, bp), rows)
        ra, rb = row_bytes(*a), row_bytes(*b)
        any_ = any(x & y for x in ra for y in rb)
        other = any(ra[i] & rb[j] for i in range(rows) for j in range(rows) if i != j)
        got, got_other = bool(lib.shares(*a, *b)), bool(lib.shares_other(*a, *b))
        assert got >= any_ and got_other >= other, (a, b)
        if rows == 1:
            assert got == any_ and got_other == other, (a, b)
        elif ap == bp:
            # One pitch: rows beyond the last one count as if they were there.
            far = [row_bytes(p - 60 * ap, pitch, row, rows + 120) for p, pitch, row, rows in (a, b)]
            ends = max(a[0], b[0]) < min(a[0] + (rows - 1) * ap + a[2], b[0] + (rows - 1) * bp + b[2])
            assert got == (ends and any(x & y for x in far[0][60:60 + rows] for y in far[1])), (a, b)
            assert got_other == (ends and any(x & far[1][j] for i, x in enumerate(far[0][60:60 + rows], 60)
                                              for j in range(len(far[1])) if i != j)), (a, b)
        seen[got, got_other] = seen.get((got, got_other), 0) + 1
    assert set(seen) >= {(False, False), (True, False), (True, True)}


def test_nothing_overlaps_what_is_absent(lib):
    there = (100, 8, 8, 2)
    for gone in ((0, 8, 8, 2), (100, 8, 0, 2)):
        assert not lib.shares(*there, *gone) and not lib.shares(*gone, *there)
        assert not lib.shares_other(*there, *gone) and not lib.shares_other(*gone, *there)


@pytest.mark.gpu
def test_outputs_among_inputs_are_refused(ctx):
    """Outputs that lie where other rows' inputs are, and the ones that may."""
    import numpy as np
    import torch
    from telmo_b200 import Epilogue, Kernels, LogitRules, PackedWeights, Precision, TelmoError
    k = Kernels(ctx)
    i32 = dict(dtype=torch.int32, device="cuda")
    x = torch.randn((4, 64), generator=torch.Generator().manual_seed(1)).cuda()
    history, n = torch.randint(0, 64, (4, 6), generator=torch.Generator().manual_seed(2)).int().cuda(), torch.full((4,), 5, **i32)
    theta, masks, state = torch.full((4,), 2.0, device="cuda"), torch.full((4, 2), -1, **i32), torch.zeros(4, **i32)
    bias_ids, bias = torch.zeros((4, 3), **i32), torch.zeros((4, 3), device="cuda")
    r = LogitRules(history=history, history_len=n, repetition=theta, bias_ids=bias_ids, bias=bias, allowed=masks, state=state)
    ids, lp = torch.full((4, 2), -7, **i32), torch.zeros((4, 2), device="cuda")
    tensors = (x, history, n, theta, masks, state, bias_ids, bias, ids, lp)
    before = [t.clone() for t in tensors]
    f32 = lambda t: t.view(torch.float32)
    calls = [lambda t=t: k.choose_tokens(x, 64, 4, 64, r, 2, t.view(torch.int32).flatten())
             for t in (x, history, masks, bias_ids, bias)]
    calls += [lambda t=t: k.choose_tokens(x, 64, 4, 64, r, 2, ids, f32(t).flatten()) for t in (x, history, masks, bias_ids, bias, ids)]
    calls += [lambda t=t: k.constrain_logits(x, 64, 4, 1, r, f32(t), 1) for t in (n, theta, state)]
    calls += [lambda t=t: k.constrain_logits(x, 64, 4, t.shape[1], r, f32(t), t.shape[1]) for t in (history, masks, bias_ids, bias)]
    calls += [lambda: k.constrain_logits(x, 64, 1, 6, r, f32(history), 6)]
    dev = PackedWeights.encode(np.ones((64, 32), np.float32), 64, 32, Precision.Q4).upload(ctx)
    a, c = torch.ones((4, 32), device="cuda"), torch.full((5, 64), 3.0, device="cuda")
    calls += [lambda: k.linear(a, 4, dev, c[:4], Epilogue(bias=c[0])), lambda: k.linear(a, 4, dev, c[:4], Epilogue(bias=c[3])),
              lambda: k.linear(a, 4, dev, c[:4], Epilogue(bias=c.flatten()[10:74])),
              lambda: k.linear(a, 1, dev, c[:1], Epilogue(bias=c.flatten()[1:65])),
              lambda: k.linear(a, 1, dev, c.flatten().view(torch.bfloat16)[:64], Epilogue(bias=c[0]))]
    for i, call in enumerate(calls):
        with pytest.raises(TelmoError):
            call()
            pytest.fail(f"call {i} was taken")
    ctx.check()
    assert all(torch.equal(t, b) for t, b in zip(tensors, before)) and (c == 3).all()
    dev.free()


@pytest.mark.gpu
def test_a_row_s_tokens_may_lie_among_its_own_inputs(ctx):
    """The chosen token written to the next place of the tokens so far, step after step; one of each row over what
    the row was given; a bias that becomes its row's output."""
    import numpy as np
    import torch
    from telmo_b200 import Epilogue, Kernels, LogitRules, PackedWeights, Precision
    k = Kernels(ctx)
    g = torch.Generator().manual_seed(4)
    x = torch.randn((1, 50000), generator=g).cuda()
    i32 = dict(dtype=torch.int32, device="cuda")
    history, apart = torch.full((1, 9), -1, **i32), torch.full((1, 9), -1, **i32)
    n, penalty, one = torch.zeros(1, **i32), torch.full((1,), 9.0, device="cuda"), torch.zeros((1, 1), **i32)
    for step in range(8):
        k.choose_tokens(x, 50000, 1, 50000, LogitRules(history, n, presence=penalty), 1, history[:, step:step + 1])
        k.choose_tokens(x, 50000, 1, 50000, LogitRules(apart, n, presence=penalty), 1, one)
        apart[0, step] = one[0, 0]
        n += 1
    ctx.check()
    assert torch.equal(history, apart) and len(set(history[0].tolist())) == 9 and history[0, 8] == -1
    many = torch.randn((300, 3000), generator=g).cuda()
    last, want = many.argmax(1).int()[:, None].contiguous(), torch.zeros((300, 1), **i32)
    ones, much = torch.ones(300, **i32), torch.full((300,), 9.0, device="cuda")
    k.choose_tokens(many, 3000, 300, 3000, LogitRules(last.clone(), ones, presence=much), 1, want)
    k.choose_tokens(many, 3000, 300, 3000, LogitRules(last, ones, presence=much), 1, last)
    ctx.check()
    assert torch.equal(last, want)
    dev = PackedWeights.encode(torch.randn((500, 96), generator=g).numpy(), 500, 96, Precision.Q4).upload(ctx)
    a, bias = torch.randn((1, 96), generator=g).cuda(), torch.randn(500, generator=g).cuda()
    c = torch.empty((1, 500), device="cuda")
    k.linear(a, 1, dev, c, Epilogue(bias=bias))
    k.linear(a, 1, dev, bias[None], Epilogue(bias=bias))
    ctx.check()
    assert torch.equal(c[0], bias)
    dev.free()
