"""What the entry points that take tensors check of them before a kernel gets an address: that a view
really holds the rows that the call names. The checks read no memory, so they run on host tensors here, with
a context whose device is the host's."""

import types

import pytest

import telmo_b200
from telmo_b200 import TelmoError


class Host(types.SimpleNamespace):
    device = -1  # what a host tensor's get_device() says


def accepts(t, rows, cols, ld):
    try:
        return telmo_b200._matrix(Host(), t, "t", (t.dtype,), rows, cols, ld) == t.data_ptr()
    except TelmoError:
        return False


def test_a_view_must_hold_the_rows_itself():
    import torch
    buf = torch.zeros((8, 32))
    assert accepts(buf[:2, :16], 2, 16, 32) and accepts(buf[:2, :16], 1, 16, 32) and accepts(buf[2:, 8:], 6, 24, 32)
    for rows, cols, ld in ((3, 16, 32), (8, 16, 32), (2, 17, 32), (2, 16, 16), (2, 16, 31)):
        assert not accepts(buf[:2, :16], rows, cols, ld)
    assert not accepts(buf[:, 0], 8, 1, 32) and not accepts(buf[:, 0], 1, 1, 1) and not accepts(buf.t(), 8, 8, 32)
    assert not accepts(torch.zeros((1, 4)).expand(3, 4), 3, 4, 4)


def test_leading_dimensions_must_be_rows_of_one_distance():
    import torch
    x = torch.zeros((2, 8, 16))
    cut = x[:, :5]  # a batch of which five steps of eight are meant
    assert not accepts(cut, 10, 16, 16) and not accepts(cut, 6, 16, 16)
    assert accepts(cut, 5, 16, 16)  # the first sequence alone
    narrow = x[:, :, :10]
    assert accepts(narrow, 16, 10, 16) and not accepts(narrow, 17, 10, 16) and not accepts(narrow, 16, 11, 16)
    first = x[:, :1]  # a step of each sequence: rows 128 apart
    assert accepts(first, 2, 16, 128) and not accepts(first, 2, 16, 16) and not accepts(first, 3, 16, 128)
    assert not accepts(x.transpose(0, 1), 16, 16, 16)


def test_contiguous_tensors_are_memory():
    import torch
    x = torch.zeros((4, 32))
    assert accepts(x, 8, 16, 16) and accepts(x, 3, 32, 48) and accepts(x.view(-1), 2, 40, 80)
    assert not accepts(x, 8, 17, 17) and not accepts(x, 5, 32, 32) and not accepts(x, 2, 32, 31)


@pytest.mark.gpu
def test_outputs_leave_what_lies_outside_a_view(ctx):
    """Fewer rows in the view than the call names, and a batch cut short: refused, nothing written."""
    import numpy as np
    import torch
    from telmo_b200 import Kernels, PackedWeights, Precision
    kern = Kernels(ctx)
    w = PackedWeights.encode(np.ones((16, 32), np.float32), 16, 32, Precision.Q4).upload(ctx)
    a = torch.ones((16, 32), device="cuda")
    buf = torch.full((16, 48), 7.0, device="cuda")
    cube = buf.view(2, 8, 48)
    ids = torch.full((10, 1), -9, dtype=torch.int32, device="cuda")
    for call in (lambda: kern.matmul(a, 32, 8, w, buf[:2, :16], 48), lambda: kern.matmul(a, 32, 10, w, cube[:, :5, :16], 48),
                 lambda: kern.matmul(cube[:, :5, :32], 48, 10, w, torch.empty((10, 16), device="cuda"), 16),
                 lambda: kern.constrain_logits(a, 32, 3, 32, None, buf[:2, :32], 48),
                 lambda: kern.constrain_logits(cube[:, :5, :32], 48, 10, 32, None, torch.empty((10, 32), device="cuda"), 32),
                 lambda: kern.choose_tokens(cube[:, :5], 48, 10, 48, None, 1, ids),
                 lambda: kern.choose_tokens(buf[:2, :32], 48, 3, 32, None, 1, ids)):
        with pytest.raises(TelmoError):
            call()
    ctx.check()
    assert (buf == 7).all() and (ids == -9).all()
    kern.matmul(a, 32, 5, w, cube[:, :5, :16], 48)
    kern.matmul(a, 32, 16, w, cube[:, :, 16:32], 48)
    ctx.check()
    assert (cube[0, :5, :16] != 7).all() and (cube[0, 5:, :16] == 7).all() and (cube[1, :, :16] == 7).all()
    assert (cube[:, :, 16:32] != 7).all() and (cube[:, :, 32:] == 7).all()
    w.free()
