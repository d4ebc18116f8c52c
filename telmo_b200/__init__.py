"""telmo_b200: the B200-native (sm_100a) hot path of telmo's speech encoders.

The Python layer mirrors the reference's operator interface for this path -- ``Kernels``,
``PackedWeights``, ``Epilogue``, ``Act``, ``Precision`` (src/kernels/mod.rs, src/quant.rs) and the
model entry points -- over the C ABI of ``libtelmo_b200.so`` (include/telmo_b200.h). Device
buffers are torch CUDA tensors (torch is used for device memory and streams only); every
computation runs in the library's CUDA kernels. There is no CPU fallback: without the library
or a B200 the calls raise.
"""

from __future__ import annotations

import ctypes
import enum
import functools
from dataclasses import dataclass
from typing import Optional

import numpy as np

from . import _lib
from ._lib import TelmoError, check

__all__ = ["Act", "Context", "Epilogue", "Kernels", "LogitRules", "PackedWeights", "Precision", "TelmoError",
           "DeviceWeights"]


class Precision(enum.IntEnum):
    """How a weight matrix's values are stored (src/quant.rs:22-30)."""
    F32 = 0
    F16 = 1
    BF16 = 2
    INT8 = 3
    Q8_0 = 4
    Q4 = 5  # codes 0..15 with a scale, and if given a zero point, per group of inputs


class Act(enum.IntEnum):
    """An activation applied in the matrix product's epilogue (src/kernels/mod.rs:366-373)."""
    NONE = 0
    RELU = 1
    SILU = 2


class DType(enum.IntEnum):
    F32 = 0
    BF16 = 1
    I32_PAIR = 2
    F16 = 3


@dataclass
class Epilogue:
    """``c = (accumulate ? c : 0) + scale * act(sum + bias)`` (src/kernels/mod.rs:375-398)."""
    bias: Optional[object] = None
    act: Act = Act.NONE
    scale: float = 1.0
    accumulate: bool = False

    @staticmethod
    def with_bias(bias) -> "Epilogue":
        return Epilogue(bias=bias)


Epilogue.PLAIN = Epilogue()


def _ptr(t) -> Optional[int]:
    if t is None:
        return None
    if hasattr(t, "data_ptr"):
        return t.data_ptr()
    if isinstance(t, np.ndarray):
        return t.ctypes.data
    return int(t)


def _stream(stream) -> Optional[int]:
    if stream is None:
        import torch
        return torch.cuda.current_stream().cuda_stream
    return getattr(stream, "cuda_stream", stream)


def _refuse(message: str):
    raise TelmoError(_lib.TELMO_ERR_ARGUMENT, message)


def _matrix(ctx, t, name: str, dtypes, rows: int, cols: int, ld: int) -> int:
    """The address of a [rows, cols] matrix with rows `ld` elements apart that starts at tensor `t`,
    which must lie on the context's device, be of one of `dtypes` and reach to the last element. A
    view with gaps must have that many rows itself, `ld` apart, and their elements next to one
    another."""
    if t.get_device() != ctx.device:  # -1 in host memory
        _refuse(f"{name}: a tensor on {t.device}, the context is on cuda:{ctx.device}")
    if t.dtype not in dtypes:
        _refuse(f"{name}: {t.dtype} is not one of {', '.join(str(d) for d in dtypes)}")
    if rows > 0 and cols > 0:
        if ld < cols:
            _refuse(f"{name}: rows {ld} elements apart hold no {cols} elements")
        if t.is_contiguous():
            have = t.numel()
            if have < (rows - 1) * ld + cols:
                _refuse(f"{name}: {have} elements, {(rows - 1) * ld + cols} are needed")
        elif not _has_rows(t.shape, t.stride(), rows, cols, ld):
            _refuse(f"{name}: {list(t.shape)} with strides {list(t.stride())} has no {rows} rows of {cols} "
                    f"elements, {ld} apart")
    return t.data_ptr()


def _has_rows(shape, strides, rows: int, cols: int, ld: int) -> bool:
    """Whether a view's first `rows` rows (all its dimensions but the last, in order) lie `ld` elements
    apart and hold `cols` elements next to one another. Dimensions behind the last row that is used
    may lie anywhere."""
    if strides[-1] != 1 or cols > shape[-1]:
        return False
    have = 1  # rows that the dimensions so far hold
    for size, stride in zip(reversed(shape[:-1]), reversed(strides[:-1])):
        if have >= rows:
            break
        if size != 1 and stride != ld * have:
            return False
        have *= size
    return have >= rows


def _vector(ctx, t, name: str, dtypes, rows: int) -> int:
    """The address of a value per row, or 0 where there is no tensor."""
    if t is None:
        return 0
    if t.get_device() == ctx.device and t.dtype in dtypes and t.numel() >= rows and t.is_contiguous():
        return t.data_ptr()
    return _matrix(ctx, t, name, dtypes, 1, rows, rows)  # says what is wrong


def _table(ctx, t, name: str, dtypes, least_rows: int, least_cols: int) -> tuple:
    """The rows, address, columns and row distance of a matrix of at least that size."""
    shape, strides = t.shape, t.stride()
    if len(shape) != 2 or strides[1] != 1 or shape[0] < least_rows or shape[1] < least_cols:
        _refuse(f"{name}: a matrix of at least [{least_rows}, {least_cols}] with unit stride "
                f"along its rows, not {list(shape)}")
    rows, cols = shape
    ld = strides[0] if rows > 1 else max(cols, 1)
    if ld < cols or t.get_device() != ctx.device or t.dtype not in dtypes:
        _matrix(ctx, t, name, dtypes, rows, cols, ld)  # says what is wrong
    return rows, t.data_ptr(), cols, ld


@functools.lru_cache(maxsize=None)
def _float_types() -> dict:
    """torch dtype -> TELMO_DTYPE_* of the entry points that take f32, bf16 and f16."""
    import torch
    return {torch.float32: 0, torch.bfloat16: 1, torch.float16: 3}


@functools.lru_cache(maxsize=None)
def _f32_only() -> tuple:
    import torch
    return (torch.float32,)


@functools.lru_cache(maxsize=None)
def _i32_only() -> tuple:
    import torch
    return (torch.int32,)


@functools.lru_cache(maxsize=None)
def _mask_types() -> tuple:
    import torch
    return (torch.int32, torch.uint32)


def _stream_on(ctx, stream) -> Optional[int]:
    """The given stream, or torch's current stream on the context's device."""
    if stream is None:
        return _current_stream()(ctx.device)
    return getattr(stream, "cuda_stream", stream)


@functools.lru_cache(maxsize=None)
def _current_stream():
    """A function from a device to torch's current stream there, as an address."""
    import torch
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # without a Stream object in between
    return raw or (lambda device: torch.cuda.current_stream(device).cuda_stream)


class Context:
    """One GPU. Replaces the reference's Kernels table + thread Pool with CUDA streams."""

    def __init__(self, device: int = 0):
        lib = _lib.load()
        h = ctypes.c_void_p()
        check(lib.telmo_ctx_create(device, ctypes.byref(h)), None)
        self._h = h
        self.device = device

    @property
    def handle(self):
        return self._h

    def check(self, stream=None) -> None:
        """Waits for the stream and raises if a kernel gave up on a bounded wait."""
        check(_lib.load().telmo_ctx_check(self._h, _stream(stream)), self._h)

    def close(self) -> None:
        if getattr(self, "_h", None):
            _lib.load().telmo_ctx_destroy(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class DeviceWeights:
    """A weight matrix uploaded to one context (tensor-core layout)."""

    def __init__(self, ctx: Context, handle, n: int, k: int, precision: Precision = Precision.INT8):
        self.ctx, self._h, self.n, self.k, self.precision = ctx, handle, n, k, precision

    @property
    def handle(self):
        return self._h

    def free(self) -> None:
        if getattr(self, "_h", None):
            _lib.load().telmo_weights_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


class PackedWeights:
    """A weight matrix of ``n`` outputs and ``k`` inputs in the reference's panel layout
    (src/kernels/mod.rs:177-304): 16-output panels of int8 values with one f32 scale per output
    (Int8) or per block of 32 inputs of each output (Q8_0, src/quant.rs:8-13).

    Q4, which the reference does not have, is row-major: ``values`` holds n rows of ceil(k / 2) bytes
    (two codes 0..15 each, the even input in the low half), ``scales`` [n, ceil(k / group)] f16
    values and ``zeros``, where given, as many zero points 0..15 (8 where not), for groups of 32, 64
    or 128 inputs: ``w = (code - zero) * scale``."""

    def __init__(self, n: int, k: int, precision: Precision, values: np.ndarray,
                 scales: np.ndarray, zeros: Optional[np.ndarray] = None, group: int = 32):
        if precision == Precision.Q4:
            self._init_q4(n, k, values, scales, zeros, group)
            return
        if zeros is not None:
            _refuse(f"{precision.name}: only Q4 has zero points")
        panels = (n + 15) // 16
        if precision not in (Precision.INT8, Precision.Q8_0):
            raise TelmoError(_lib.TELMO_ERR_UNSUPPORTED,
                             f"{precision.name}: this build runs int8 weights (INT8, Q8_0) only")
        if precision == Precision.Q8_0 and k % 32:
            raise TelmoError(_lib.TELMO_ERR_ARGUMENT, "Q8_0 needs inputs in multiples of 32")
        n_scales = panels * 16 * (k // 32 if precision == Precision.Q8_0 else 1)
        if values.size != panels * 16 * k or scales.size != n_scales:
            raise TelmoError(_lib.TELMO_ERR_ARGUMENT, "panel sizes do not match n and k")
        self.n, self.k, self.precision = n, k, precision
        self.values = np.ascontiguousarray(values, dtype=np.int8)
        self.scales = np.ascontiguousarray(scales, dtype=np.float32)

    def _init_q4(self, n, k, values, scales, zeros, group) -> None:
        if group not in (32, 64, 128):
            _refuse(f"Q4: groups of 32, 64 or 128 inputs, not {group}")
        if n < 1 or k < 1:
            _refuse(f"Q4: bad sizes n={n} k={k}")
        groups = -(-k // group)
        if values.size != n * (-(-k // 2)) or scales.size != n * groups:
            _refuse("Q4: sizes do not match n, k and group")
        if zeros is not None and (zeros.size != n * groups or zeros.dtype != np.uint8):
            _refuse("Q4: zero points are uint8, one per scale")
        if values.dtype != np.uint8:
            _refuse("Q4: values are uint8, two codes to a byte")
        self.n, self.k, self.precision, self.group = n, k, Precision.Q4, group
        self.values = np.ascontiguousarray(values)
        self.scales = np.ascontiguousarray(scales, dtype=np.float32)
        self.zeros = None if zeros is None else np.ascontiguousarray(zeros)

    @staticmethod
    def encode(rows: np.ndarray, n: int, k: int, precision: Precision = Precision.INT8,
               group: int = 32, zeros: bool = False) -> "PackedWeights":
        """quant::encode (src/quant.rs:202-269) of a row-major f32 [n, k] matrix; for Q4 (groups of
        ``group`` inputs, with zero points if ``zeros``) telmo_encode_q4."""
        rows = np.ascontiguousarray(rows, dtype=np.float32).reshape(n, k)
        if precision == Precision.Q4:
            if group not in (32, 64, 128):
                _refuse(f"Q4: groups of 32, 64 or 128 inputs, not {group}")
            groups = -(-k // group)
            values = np.zeros((n, -(-k // 2)), np.uint8)
            scales = np.zeros((n, groups), np.float32)
            z = np.zeros((n, groups), np.uint8) if zeros else None
            check(_lib.load().telmo_encode_q4(rows.ctypes.data, n, k, group, values.ctypes.data,
                                              scales.ctypes.data, _ptr(z)))
            return PackedWeights(n, k, precision, values, scales, z, group)
        panels = (n + 15) // 16
        values = np.zeros(panels * 16 * k, np.int8)
        if precision == Precision.Q8_0:
            scales = np.zeros(panels * 16 * (k // 32), np.float32)
            encode = _lib.load().telmo_encode_q8_0
        else:
            scales = np.zeros(panels * 16, np.float32)
            encode = _lib.load().telmo_encode_int8
        check(encode(rows.ctypes.data, n, k, values.ctypes.data, scales.ctypes.data))
        return PackedWeights(n, k, precision, values, scales)

    def upload(self, ctx: Context) -> DeviceWeights:
        h = ctypes.c_void_p()
        if self.precision == Precision.Q4:
            check(_lib.load().telmo_weights_upload_q4(ctx.handle, self.n, self.k, self.group,
                                                      self.values.ctypes.data,
                                                      self.scales.ctypes.data, _ptr(self.zeros),
                                                      ctypes.byref(h)), ctx.handle)
            return DeviceWeights(ctx, h, self.n, self.k, self.precision)
        check(_lib.load().telmo_weights_upload(ctx.handle, int(self.precision), self.n, self.k,
                                               self.values.ctypes.data, self.scales.ctypes.data,
                                               ctypes.byref(h)), ctx.handle)
        return DeviceWeights(ctx, h, self.n, self.k, self.precision)


@dataclass
class LogitRules:
    """What a decoder lays over logits before it chooses (telmo_logit_rules): penalties for the
    row's tokens so far, biases, and the masks of a grammar's states. Tensors on the context's
    device, ``None`` for a rule left out."""
    history: Optional[object] = None      # int32 [rows, width]
    history_len: Optional[object] = None  # int32 [rows]
    repetition: Optional[object] = None   # f32 [rows], above 0
    frequency: Optional[object] = None    # f32 [rows]
    presence: Optional[object] = None     # f32 [rows]
    bias_ids: Optional[object] = None     # int32 [rows, entries <= 2^20], negative: unused
    bias: Optional[object] = None         # f32 [rows, entries]
    allowed: Optional[object] = None      # int32 (or uint32) [states, ceil(vocab / 32)] bit masks
    state: Optional[object] = None        # int32 [rows], negative: no mask; None: row r has mask r

    def _struct(self, ctx, rows: int, vocab: int) -> bytes:
        """The C structure's bytes, checked and made anew for each call: a tensor may have been reshaped
        in place since the last one (6 us with all rules; comparing what a kept one was made of would
        read as much of each tensor)."""
        i32, f32 = _i32_only(), _f32_only()
        h, ids, masks = self.history, self.bias_ids, self.allowed
        history = n_history = history_ld = said = theta = freq = pres = 0
        bias = n_bias = bias_ld = n_states = masks_ld = state = 0
        if h is not None:
            if self.history_len is None:
                _refuse("history: its lengths are missing")
            history, n_history, history_ld = _table(ctx, h, "history", i32, rows, 0)[1:]
            said = _vector(ctx, self.history_len, "history_len", i32, rows)
            theta = _vector(ctx, self.repetition, "repetition", f32, rows)
            freq = _vector(ctx, self.frequency, "frequency", f32, rows)
            pres = _vector(ctx, self.presence, "presence", f32, rows)
            if n_history == 0:  # an empty tensor has no address; without tokens no penalty applies
                history = theta = freq = pres = 0
        elif not (self.history_len is self.repetition is self.frequency is self.presence is None):
            _refuse("penalties need the tokens so far (history)")
        if ids is not None or self.bias is not None:
            if ids is None or self.bias is None or ids.shape != self.bias.shape:
                _refuse("bias_ids and bias are two matrices of one shape")
            ids, n_bias, bias_ld = _table(ctx, ids, "bias_ids", i32, rows, 0)[1:]
            bias, _, ld = _table(ctx, self.bias, "bias", f32, rows, 0)[1:]
            if ld != bias_ld:
                _refuse("bias_ids and bias must have the same stride")
        if masks is not None:
            n_states, masks, _, masks_ld = _table(ctx, masks, "allowed", _mask_types(), 1, -(-vocab // 32))
            if self.state is not None:
                state = _vector(ctx, self.state, "state", i32, rows)
            elif n_states < rows:
                _refuse(f"{n_states} masks for {rows} rows, and no states")
        elif self.state is not None:
            _refuse("state needs the masks (allowed)")
        return _lib.LOGIT_RULES.pack(history, n_history, history_ld, said, theta, freq, pres, ids or 0, bias, n_bias,
                                     bias_ld, masks or 0, n_states, masks_ld, state)


class Kernels:
    """The matrix product of src/kernels/mod.rs on the GPU: ``linear`` and ``matmul`` over
    packed int8 weights, with the reference's Epilogue. Tensors are torch CUDA tensors.

    With Q4 weights ``a`` and ``c`` may each be f32, bf16 or f16 and must lie on the context's
    device; ``stream`` defaults to torch's current stream there. What is kept of small activations
    beside large ones depends on the type and on m (telmo_linear_q4)."""

    def __init__(self, ctx: Context):
        self.ctx = ctx

    def linear(self, a, m: int, w: DeviceWeights, c, epi: Epilogue = Epilogue.PLAIN,
               stream=None) -> None:
        """``c = epilogue(a * w^T)`` with ``a`` and ``c`` contiguous (src/kernels/mod.rs:691)."""
        if w.precision == Precision.Q4 and not (a.is_contiguous() and c.is_contiguous()):
            _refuse("linear takes contiguous tensors (matmul takes strides)")
        self.matmul(a, w.k, m, w, c, w.n, epi, stream)

    def matmul(self, a, lda: int, m: int, w: DeviceWeights, c, ldc: int,
               epi: Epilogue = Epilogue.PLAIN, stream=None, out_dtype: DType = None) -> None:
        """``c[m, n] = epilogue(a[m, k] * w^T)`` with strides (src/kernels/mod.rs:657)."""
        if w.precision == Precision.Q4:
            self._matmul_q4(a, lda, m, w, c, ldc, epi, stream, out_dtype)
            return
        import torch
        if out_dtype is None:
            out_dtype = DType.BF16 if c.dtype == torch.bfloat16 else \
                DType.I32_PAIR if c.dtype == torch.int32 else DType.F32
        check(_lib.load().telmo_linear(self.ctx.handle, _ptr(a), lda, m, w.handle, _ptr(epi.bias),
                                       int(epi.act), float(epi.scale), int(epi.accumulate),
                                       _ptr(c), int(out_dtype), ldc, _stream(stream)),
              self.ctx.handle)

    def _matmul_q4(self, a, lda, m, w, c, ldc, epi, stream, out_dtype) -> None:
        types = _float_types()
        pa = _matrix(self.ctx, a, "a", types, m, w.k, lda)
        pc = _matrix(self.ctx, c, "c", types, m, w.n, ldc)
        if out_dtype is not None and out_dtype != types[c.dtype]:
            _refuse(f"c is {c.dtype}, not {out_dtype!r}")
        pb = None
        if epi.bias is not None:
            pb = _matrix(self.ctx, epi.bias, "bias", _f32_only(), 1, w.n, w.n)
        check(_lib.load().telmo_linear_q4(self.ctx.handle, pa, types[a.dtype], lda, m, w.handle, pb,
                                          int(epi.act), float(epi.scale), int(epi.accumulate), pc,
                                          types[c.dtype], ldc, _stream_on(self.ctx, stream)),
              self.ctx.handle)

    def constrain_logits(self, logits, ld: int, rows: int, vocab: int, rules: Optional[LogitRules],
                         out, out_ld: int, stream=None) -> None:
        """``rules`` laid over ``logits`` [rows, ld] (f32, bf16 or f16, ``vocab`` of each row) into
        ``out`` [rows, out_ld] of the same type, which may be ``logits`` itself
        (telmo_logits_constrain)."""
        types = _float_types()
        pl = _matrix(self.ctx, logits, "logits", types, rows, vocab, ld)
        po = _matrix(self.ctx, out, "out", (logits.dtype,), rows, vocab, out_ld)
        st = None if rules is None else rules._struct(self.ctx, rows, vocab)
        check(_lib.load().telmo_logits_constrain(self.ctx.handle, pl, types[logits.dtype], ld, rows,
                                                 vocab, st, po, out_ld, _stream_on(self.ctx, stream)),
              self.ctx.handle)

    def choose_tokens(self, logits, ld: int, rows: int, vocab: int, rules: Optional[LogitRules],
                      k: int, ids, logprobs=None, stream=None) -> None:
        """The ``k`` (1..8) best tokens of each row of ``logits`` under ``rules``, best first and the
        lowest first where several tie, into ``ids`` (int32 [rows, k], -1 where nothing is left),
        and their log-probabilities into ``logprobs`` (f32 [rows, k]) (telmo_logits_choose)."""
        types = _float_types()
        pl = _matrix(self.ctx, logits, "logits", types, rows, vocab, ld)
        pi = _matrix(self.ctx, ids, "ids", _i32_only(), rows, k, k)
        pp = None if logprobs is None else _matrix(self.ctx, logprobs, "logprobs", _f32_only(), rows, k, k)
        st = None if rules is None else rules._struct(self.ctx, rows, vocab)
        check(_lib.load().telmo_logits_choose(self.ctx.handle, pl, types[logits.dtype], ld, rows, vocab,
                                              st, k, pi, pp, _stream_on(self.ctx, stream)),
              self.ctx.handle)

    def quantize_x2(self, a, lda: int, m: int, k: int, hi, lo, ldq: int, scale,
                    stream=None) -> None:
        check(_lib.load().telmo_quantize_x2(self.ctx.handle, _ptr(a), lda, m, k, _ptr(hi),
                                            _ptr(lo), ldq, _ptr(scale), _stream(stream)),
              self.ctx.handle)

    def conv_module_rows(self, x, frames: int, channels: int, kernel: int, stride: int, w, bias,
                         out, stream=None) -> None:
        """GLU, depthwise convolution and SiLU over one utterance's rows into `out` (f32), the
        reference's glu, dwconv1d_frame and silu kernels (src/kernels/mod.rs:462-470)."""
        check(_lib.load().telmo_conv_module_rows(self.ctx.handle, _ptr(x), frames, channels, kernel,
                                                 stride, _ptr(w), _ptr(bias), _ptr(out),
                                                 _stream(stream)),
              self.ctx.handle)

    def linear_q(self, hi, lo, ldq: int, scale, m: int, w: DeviceWeights, c, ldc: int,
                 epi: Epilogue = Epilogue.PLAIN, out_dtype: DType = DType.F32,
                 stream=None) -> None:
        check(_lib.load().telmo_linear_q(self.ctx.handle, _ptr(hi), _ptr(lo), ldq, _ptr(scale),
                                         m, w.handle, _ptr(epi.bias), int(epi.act),
                                         float(epi.scale), int(epi.accumulate), _ptr(c),
                                         int(out_dtype), ldc, _stream(stream)),
              self.ctx.handle)
