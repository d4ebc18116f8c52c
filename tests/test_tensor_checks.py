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


def rules_of(r, rows, vocab):
    """The C structure that a call with these sizes would pass."""
    return telmo_b200._lib.LogitRules.from_buffer_copy(r._struct(Host(), rows, vocab))


def test_rules_are_read_anew_in_each_call():
    """Tensors reshaped in place between two calls, with the same address and as many elements as before."""
    import torch
    from telmo_b200 import LogitRules
    ids, bias = torch.zeros((4, 6), dtype=torch.int32), torch.zeros((4, 6))
    r = LogitRules(bias_ids=ids, bias=bias)
    s = rules_of(r, 4, 100)
    assert (s.n_bias, s.bias_ld, s.bias_ids, s.bias) == (6, 6, ids.data_ptr(), bias.data_ptr())
    ids.resize_(6, 4), bias.resize_(6, 4)
    s = rules_of(r, 4, 100)
    assert (s.n_bias, s.bias_ld) == (4, 4)
    ids.t_(), bias.t_()
    with pytest.raises(TelmoError):
        rules_of(r, 4, 100)

    history, n = torch.zeros((4, 8), dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    theta = torch.ones(8)
    r = LogitRules(history=history, history_len=n, repetition=theta)
    s = rules_of(r, 4, 100)
    assert (s.n_history, s.history_ld, s.history, s.history_len) == (8, 8, history.data_ptr(), n.data_ptr())
    assert s.repetition == theta.data_ptr() and not s.frequency and not s.presence and not s.state
    history.as_strided_((4, 4), (8, 1))
    s = rules_of(r, 4, 100)
    assert (s.n_history, s.history_ld) == (4, 8)
    theta.as_strided_((4,), (2,))
    with pytest.raises(TelmoError):
        rules_of(r, 4, 100)
    r.repetition = None
    rules_of(r, 4, 100)
    history.data = history.data.view(torch.float32)
    with pytest.raises(TelmoError):
        rules_of(r, 4, 100)

    masks, state = torch.zeros((4, 4), dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    r = LogitRules(allowed=masks, state=state)
    s = rules_of(r, 4, 128)
    assert (s.allowed, s.n_states, s.allowed_ld, s.state) == (masks.data_ptr(), 4, 4, state.data_ptr())
    masks.resize_(2, 8)
    s = rules_of(r, 4, 128)
    assert (s.n_states, s.allowed_ld) == (2, 8)
    state.resize_(3)
    with pytest.raises(TelmoError):
        rules_of(r, 4, 128)


def test_rules_on_the_host_are_refused_one_by_one():
    """Each of the nine tensors with a fault of its own."""
    import torch
    from telmo_b200 import LogitRules
    i32 = dict(dtype=torch.int32)
    table, vec, f, m = torch.zeros((4, 5), **i32), torch.zeros(4, **i32), torch.ones(4), torch.zeros((4, 4), **i32)
    good = dict(history=table, history_len=vec, repetition=f, frequency=f, presence=f, bias_ids=table,
                bias=torch.zeros((4, 5)), allowed=m, state=vec)
    rules_of(LogitRules(**good), 4, 100)
    for name, t in good.items():
        wrong = [t.double(), t[:3]]
        if t.dim() == 1:
            wrong += [torch.stack((t, t), dim=1)[:, 0]]
        else:
            wrong += [t.t().contiguous().t(), t[:1].expand(4, -1), t.flatten()]
        for bad in wrong:
            if name == "allowed" and bad.shape[0] == 3 and bad.dim() == 2:
                continue  # fewer masks than rows will do where there are states
            with pytest.raises(TelmoError):
                rules_of(LogitRules(**{**good, name: bad}), 4, 100)
    for absent in ("history", "history_len", "bias_ids", "bias", "allowed"):
        with pytest.raises(TelmoError):
            rules_of(LogitRules(**{**good, absent: None}), 4, 100)
    assert bytes(rules_of(LogitRules(), 4, 100)) == bytes(120)
    with pytest.raises(TelmoError):  # on another device than the context's
        LogitRules(**good)._struct(types.SimpleNamespace(device=0), 4, 100)


@pytest.mark.gpu
def test_rules_reshaped_between_two_calls(ctx):
    """The same lists as [4, 6] and then as [6, 4], against new ones of that shape."""
    import torch
    from telmo_b200 import Kernels, LogitRules
    k, g = Kernels(ctx), torch.Generator().manual_seed(5)
    ids = torch.randint(0, 50, (4, 6), generator=g, dtype=torch.int32).cuda()
    bias = torch.randn((4, 6), generator=g).cuda()
    x = torch.randn((4, 50), generator=g).cuda()
    got, want = torch.empty_like(x), torch.empty_like(x)
    r = LogitRules(bias_ids=ids, bias=bias)
    for shape in ((4, 6), (6, 4), (4, 6)):
        ids.resize_(shape), bias.resize_(shape)
        k.constrain_logits(x, 50, 4, 50, r, got, 50)
        k.constrain_logits(x, 50, 4, 50, LogitRules(bias_ids=ids.clone(), bias=bias.clone()), want, 50)
        ctx.check()
        assert torch.equal(got, want)
