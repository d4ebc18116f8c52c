"""4-bit weights on the host: the encoding, and what encoding and packing refuse."""

import ctypes

import numpy as np
import pytest

from telmo_b200 import PackedWeights, Precision, TelmoError, _lib


def decode(p):
    """The weights of a Q4 PackedWeights in 64 bits: (code - zero) * scale."""
    groups = -(-p.k // p.group)
    v = p.values.reshape(p.n, -1)
    q = np.stack([v & 15, v >> 4], axis=2).reshape(p.n, -1)[:, :p.k].astype(np.float64)
    z = np.full((p.n, groups), 8.0) if p.zeros is None else p.zeros.reshape(p.n, groups)
    at = np.arange(p.k) // p.group
    return (q - z[:, at]) * p.scales.reshape(p.n, groups).astype(np.float64)[:, at]


@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (5, 33), (16, 128), (17, 257), (2, 1000)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_encoding_is_within_half_a_step(n, k, group, zeros):
    g = np.random.default_rng(n * k + group)
    rows = g.standard_normal((n, k)).astype(np.float32)
    rows[0, : min(k, 5)] = 0
    p = PackedWeights.encode(rows, n, k, Precision.Q4, group=group, zeros=zeros)
    assert (p.scales == p.scales.astype(np.float16)).all()
    d = p.scales.reshape(n, -1)[:, np.arange(k) // group].astype(np.float64)
    # Half a step where the range fits. The scale is rounded to f16 (2^-11 of itself), which may
    # leave the extremes, 8 or 15 steps out, short by that much; a rounded zero point moves the
    # range by up to half a step more.
    err = np.abs(decode(p) - rows)
    bound = d * (0.5 + 15 * 2.0 ** -11 + (0.5 if zeros else 0.0) + 1e-5)
    assert (err <= bound).all()


def test_an_all_zero_group_and_extremes():
    rows = np.zeros((2, 64), np.float32)
    rows[1, 3], rows[1, 40] = 7.0, -8.0
    p = PackedWeights.encode(rows, 2, 64, Precision.Q4)
    assert (decode(p) == rows).all()
    p = PackedWeights.encode(rows, 2, 64, Precision.Q4, zeros=True)
    assert (decode(p)[0] == 0).all()


def test_encoding_refuses():
    rows = np.ones((2, 64), np.float32)
    for group in (0, 16, 48, 256):
        with pytest.raises(TelmoError):
            PackedWeights.encode(rows, 2, 64, Precision.Q4, group=group)
    for bad in (np.nan, np.inf, -np.inf, 3e38):
        r = rows.copy()
        r[1, 5] = bad
        with pytest.raises(TelmoError):
            PackedWeights.encode(r, 2, 64, Precision.Q4)
    L = _lib.load()
    buf = np.zeros(256, np.float32)
    p = buf.ctypes.data
    assert L.telmo_encode_q4(None, 1, 32, 32, p, p, None) == _lib.TELMO_ERR_ARGUMENT
    assert L.telmo_encode_q4(p, 1, 32, 32, None, p, None) == _lib.TELMO_ERR_ARGUMENT
    assert L.telmo_encode_q4(p, 1, 32, 32, p, None, None) == _lib.TELMO_ERR_ARGUMENT
    assert L.telmo_encode_q4(p, 0, 32, 32, p, p, None) == _lib.TELMO_ERR_ARGUMENT
    assert L.telmo_encode_q4(p, 1, 0, 32, p, p, None) == _lib.TELMO_ERR_ARGUMENT


def test_packing_refuses():
    v, s, z = np.zeros((4, 33), np.uint8), np.ones((4, 3), np.float32), np.zeros((4, 3), np.uint8)
    PackedWeights(4, 65, Precision.Q4, v, s, zeros=z, group=32)
    for args, more in (((4, 65, Precision.Q4, v[:, 1:], s), {}), ((4, 65, Precision.Q4, v, s[:, 1:]), {}),
                       ((4, 65, Precision.Q4, v, s), {"zeros": z[:, 1:]}),
                       ((4, 65, Precision.Q4, v, s), {"zeros": z.astype(np.int32)}),
                       ((4, 65, Precision.Q4, v.view(np.int8), s), {}),
                       ((4, 65, Precision.Q4, v, s), {"group": 33}), ((0, 65, Precision.Q4, v[:0], s[:0]), {}),
                       ((16, 2, Precision.INT8, np.zeros(32, np.int8), np.ones(16, np.float32)),
                        {"zeros": np.zeros(16, np.uint8)})):
        with pytest.raises(TelmoError):
            PackedWeights(*args, **more)


def test_null_handles_are_refused():
    L = _lib.load()
    h = ctypes.c_void_p()
    buf = np.zeros(64, np.float32)
    p = buf.ctypes.data
    assert L.telmo_weights_upload_q4(None, 1, 32, 32, p, p, None, ctypes.byref(h)) == _lib.TELMO_ERR_ARGUMENT
    assert L.telmo_linear_q4(None, p, 0, 32, 1, None, None, 0, 1.0, 0, p, 0, 1, None) == _lib.TELMO_ERR_ARGUMENT


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("largest", [2.0 ** -13, 2.0 ** -17, 3e-6, 1e-6, 2.0 ** -20, 4e-7, 2.0 ** -23, 1e-9])
def test_small_weights_keep_their_range(zeros, largest):
    """Scales below 2^-14 are multiples of 2^-24, far apart against themselves: they are rounded up, so that codes reach
    the group's largest weights. Off by half a step, and half a step more where a zero point is rounded."""
    g = np.random.default_rng(3)
    rows = (g.uniform(-1, 1, (4, 96)) * largest).astype(np.float32)
    rows[:, ::32] = largest * np.float32([[1], [-1], [1], [-1]])
    p = PackedWeights.encode(rows, 4, 96, Precision.Q4, group=32, zeros=zeros)
    d = p.scales.reshape(4, 3)[:, np.arange(96) // 32].astype(np.float64)
    assert (d == p.scales.astype(np.float16).reshape(4, 3)[:, np.arange(96) // 32]).all() and (d > 0).all()
    assert (np.abs(decode(p) - rows) <= d * (0.5 + 0.5 * zeros + 1e-5)).all()
