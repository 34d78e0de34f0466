"""Gradients in many tensors: norm, clipping and accumulation without a flat copy.

``GradientList`` names the tensors a backward pass leaves behind (CUDA tensors of
one device, f32, bf16 or f16, contiguous or rows with a pitch) and runs the
gradient-list entry points of the C ABI on them as they lie; ``B200Adamw.step``
and its passes, and ``B200Trainer.process_batch``, take a list wherever they take
a flat gradient tensor.  Every numeric operation runs in libslmopt.so.
"""
from __future__ import annotations

import ctypes

from . import _lib

# Workspaces up to this size are kept with the results of a call.
_SHARED_BYTES = 4096
_KINDS = {"l2": _lib.NORM_L2, "max": _lib.NORM_MAX}


_CODES: dict = {}


def _dtype_codes() -> dict:
    """slm_dtype by torch dtype."""
    if not _CODES:
        import torch

        _CODES.update({torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16,
                       torch.float16: _lib.DTYPE_F16})
    return _CODES


def _rows(tensor) -> tuple[int, int, int]:
    """(rows, columns, row stride) of a tensor whose elements, in row-major
    order, are equally spaced runs; ValueError for any other layout."""
    if tensor.is_contiguous():
        n = tensor.numel()
        return 1, n, n
    dims = [(n, s) for n, s in zip(tensor.shape, tensor.stride()) if n != 1]
    columns, inner = 1, len(dims)
    while inner > 0 and dims[inner - 1][1] == columns:
        columns *= dims[inner - 1][0]
        inner -= 1
    if inner == 0:
        return 1, columns, columns
    rows, stride = dims[inner - 1]
    for n, s in reversed(dims[:inner - 1]):
        if s != stride * rows:
            raise ValueError("a gradient must be contiguous, or rows at one distance")
        rows *= n
    if stride < columns:
        raise ValueError("a gradient's elements must not overlap")
    return rows, columns, stride


class GradientNorm:
    """What a norm or clip call found, in device memory.  The properties are
    tensors: taking one does not wait on the host, it orders torch's current stream
    behind the call's stream; ``read`` waits.  (Inside a capture nothing is ordered:
    a call is captured on the capture's own stream.  A replay of a captured call
    renews the values in the replay's stream order.)

    ``values`` is one f32 tensor: the norm of all gradients divided by the loss
    scale, the clip scale, the largest magnitude, 1.0 if a gradient or the norm
    is not finite (the clip scale is then 0.0) else 0.0; and with per_tensor each
    tensor's norm, then each tensor's largest magnitude."""

    __slots__ = ("_buffer", "_count", "_tensors", "_call", "_after")

    def __init__(self, buffer, count: int, tensors: int, call: tuple):
        # f32: the values, the f64 sum of squares, and scratch of the call.
        self._buffer = buffer
        self._count = count
        self._tensors = tensors
        # The device's index, the call's stream, and an event behind the call if that
        # was not the current stream.
        self._call = call
        self._after = None  # the last stream ordered behind it

    def _ready(self):
        """The buffer, with the current stream behind the call."""
        index, stream, event = self._call
        current = _current_stream(index)
        if current != stream and current != self._after and \
                _order_behind(self._buffer, index, stream, event):
            self._after = current
        return self._buffer

    @property
    def values(self):
        return self._ready().as_strided((self._count,), (1,))

    @property
    def norm(self):
        return self._ready()[0]

    @property
    def clip_scale(self):
        return self._ready()[1]

    @property
    def max_abs(self):
        return self._ready()[2]

    @property
    def nonfinite(self):
        return self._ready()[3]

    @property
    def sum_squares(self):
        """The f64 sum of squares (0-d tensor): what ranks that hold different
        tensors add up."""
        import torch

        return self._ready()[self._count:self._count + 2].view(torch.float64)[0]

    @property
    def tensor_norms(self):
        if self._count == 4:
            raise ValueError("the call was made without per_tensor")
        return self._ready()[4:4 + self._tensors]

    @property
    def tensor_max(self):
        if self._count == 4:
            raise ValueError("the call was made without per_tensor")
        return self._ready()[4 + self._tensors:self._count]

    def read(self) -> _lib.ListNorm:
        """The four values on the host; waits for them."""
        return _lib.ListNorm(*self._ready()[:4].tolist())


class GradientList:
    """Tensors whose norm, clipping, accumulation or step is wanted together.

    The list holds references to the tensors.  Their storage is read at the
    addresses of the last construction or ``bind``: after ``tensor.data = ...``
    or a new backward pass that allocated new gradients, ``bind`` the new ones.
    Work runs on ``stream`` (None: the legacy default stream) and is ordered
    with the rest of that stream; the tensors must be ready there.  A list must
    outlive the CUDA graphs that have captured its calls."""

    def __init__(self, tensors):
        import torch

        self.lib = _lib.load()
        _free_retired()
        self._h = None
        self.tensors = tuple(tensors)
        if not self.tensors:
            raise ValueError("the list contains no tensors")
        first = self.tensors[0]
        if not isinstance(first, torch.Tensor) or not first.is_cuda:
            raise ValueError("gradients must be CUDA tensors")
        self.device = first.device
        self._shapes = [self._layout(t) for t in self.tensors]
        codes = _dtype_codes()
        views = (_lib.GradView * len(self.tensors))(
            *[(t.data_ptr(), rows, columns, stride, codes[dtype])
              for t, (dtype, rows, columns, stride) in zip(self.tensors, self._shapes)])
        h = ctypes.c_void_p()
        _lib.check(self.lib.slm_grad_list_create(views, len(self.tensors), self.device.index,
                                                 ctypes.byref(h)))
        self._h = h
        # Streams that the bound tensors are in use on: None, or for one that the
        # caller owns (and may destroy) an event behind the last call there.
        self._streams: dict = {}
        self.elements = int(self.lib.slm_grad_list_elements(h))
        self._lay_out(int(self.lib.slm_grad_list_workspace_bytes(h)))
        # What every call needs, looked up once.
        self._empty, self._f32, self._index = torch.empty, torch.float32, self.device.index
        self._tensor_type, self._strided = torch.Tensor, torch.strided
        self._norm_call, self._clip_call = self.lib.slm_grad_list_norm, self.lib.slm_grad_list_clip

    def _layout(self, t):
        """(dtype, rows, columns, row stride) of a tensor that the list can take."""
        import torch

        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError("gradients must be CUDA tensors")
        if t.device != self.device:
            raise ValueError("gradients must be on one device")
        if t.dtype not in _dtype_codes():
            raise TypeError("gradients must be float32, bfloat16 or float16")
        if t.layout != torch.strided or t.is_neg():
            raise ValueError("gradients must be dense tensors, not lazily negated views")
        if t.is_contiguous():
            n = t.numel()
            return t.dtype, 1, n, n
        return (t.dtype, *_rows(t))

    def _is(self, t, shape) -> bool:
        """Whether t has this layout (the common case, contiguous, without detours)."""
        if type(t) is self._tensor_type and t.get_device() == self._index and \
                t.dtype is shape[0] and shape[1] == 1 and t.layout is self._strided and \
                t.is_contiguous() and t.numel() == shape[2]:
            return not t.is_neg()
        return self._layout(t) == shape

    def _lay_out(self, work_bytes: int) -> None:
        """Where a call's results and workspace go: for calls without and with
        per_tensor the number of values, where the workspace begins in the results'
        allocation (in f32), and the elements of that allocation.  A small workspace
        shares it; a large one is freed with the call instead of living as long as
        the results."""
        self._work_bytes = work_bytes
        self._shared = work_bytes <= _SHARED_BYTES
        counts = (4, 4 + 2 * len(self.tensors))
        heads = [(count + 5) & ~3 for count in counts]
        self._plan = [(count, head, head + work_bytes // 4 if self._shared else head)
                      for count, head in zip(counts, heads)]

    def __len__(self) -> int:
        return len(self.tensors)

    def close(self) -> None:
        """Frees the list, once the device's outstanding work is done.  During a
        capture, which cannot be waited in (a list may be collected at any time),
        that is left to the next creation or ``close`` of a list outside."""
        h, self._h = getattr(self, "_h", None), None
        if h:
            _RETIRED.append((self.lib, h, self.tensors))
        _free_retired()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    @property
    def handle(self):
        if not self._h:
            raise ValueError("the list is closed")
        return self._h

    def bind(self, tensors, stream=None) -> None:
        """Take other tensors of the same types, sizes and strides, in order.  The
        old ones are let go; torch's allocator learns which streams calls of the
        list have used them on (calls on a stream given by its handle, other than
        torch's current one, are waited for)."""
        tensors = tuple(tensors)
        if len(tensors) != len(self._shapes) or \
                not all(self._is(t, shape) for t, shape in zip(tensors, self._shapes)):
            raise ValueError("other tensors than the list's: types, sizes and strides must agree")
        ptrs = (ctypes.c_void_p * len(tensors))(*[t.data_ptr() for t in tensors])
        _lib.check(self.lib.slm_grad_list_bind(self.handle, ptrs, len(tensors),
                                               _stream_handle(stream)))
        old, self.tensors = self.tensors, tensors
        self._streams.pop(_current_stream(self._index), None)  # ordered as it is
        while self._streams:
            handle, event = self._streams.popitem()
            if event is not None:
                event.synchronize()
                continue
            on = _torch_stream(handle, self._index)
            for t in old:
                t.record_stream(on)

    def norm(self, loss_scale: float = 1.0, max_norm: float = 1.0, kind: str = "l2",
             per_tensor: bool = False, stream=None) -> GradientNorm:
        """The norm ("l2", or "max": the largest magnitude) of all gradients
        divided by loss_scale, and the clip scale min(max_norm / norm, 1)."""
        return self._run(False, None, loss_scale, max_norm, kind, per_tensor, stream)

    def clip(self, max_norm: float = 1.0, loss_scale: float = 1.0, kind: str = "l2", out=None,
             per_tensor: bool = False, stream=None) -> GradientNorm:
        """Divide by loss_scale and scale down to max_norm, in place or into the
        tensors of the list ``out`` (same sizes, any type).  Nothing is written
        when a gradient is inf or NaN."""
        return self._run(True, out, loss_scale, max_norm, kind, per_tensor, stream)

    def _run(self, write, out, loss_scale, max_norm, kind, per_tensor, stream) -> GradientNorm:
        code = _KINDS.get(kind)
        if code is None:
            raise ValueError('kind must be "l2" or "max"')
        h = self._h or self.handle
        n = len(self.tensors)
        count, head, room = self._plan[1 if per_tensor else 0]
        # Results and workspace come from the memory of the stream that the call runs
        # on: another stream's may still be in use by what is queued there.
        s = None if stream is None else _stream_handle(stream)
        on = s or 0
        away = _current_stream(self._index) != on
        if away:
            with _on_stream(self._index, s):
                buffer, work = self._room(room)
        else:
            buffer, work = self._room(room)
        v = buffer.data_ptr()
        w = v + 4 * head if work is None else work.data_ptr()
        norms, tops = (v + 16, v + 16 + 4 * n) if per_tensor else (None, None)
        if write:
            to = None if out is None else out._h or out.handle
            st = self._clip_call(h, to, loss_scale, max_norm, code, v, norms, tops, v + 4 * count,
                                 w, self._work_bytes, s)
        else:
            st = self._norm_call(h, loss_scale, max_norm, code, v, norms, tops, v + 4 * count, w,
                                 self._work_bytes, s)
        if st:
            _lib.check(st)
        event = _event_on(self._index, on) if away else None
        self._streams[on] = owned = event if isinstance(stream, int) else None
        if out is not None:
            out._streams[on] = owned
        return GradientNorm(buffer, count, n, (self._index, on, event))

    def _room(self, elements: int):
        """Results of a call, and its workspace where they do not share, from the
        current stream's memory."""
        buffer = self._empty(elements, dtype=self._f32, device=self.device)
        return buffer, None if self._shared else self._empty(
            self._work_bytes // 4, dtype=self._f32, device=self.device)

    def accumulate(self, acc, overwrite: bool = False, stream=None) -> None:
        """acc (f32, one value per element, tensor after tensor) += the
        gradients, or acc = the gradients."""
        if acc.device != self.device or acc.dtype != self._f32 or not acc.is_contiguous() or \
                acc.numel() != self.elements:
            raise ValueError("acc must be a contiguous f32 tensor on the list's device with one "
                             "value per element")
        _lib.check(self.lib.slm_grad_list_accumulate(self.handle, acc.data_ptr(), self.elements,
                                                     1 if overwrite else 0,
                                                     _stream_handle(stream)))
        self._used(stream)

    def _used(self, stream) -> None:
        """Takes note of the stream that a call with the list has run on."""
        on = _stream_handle(stream) or 0
        away = isinstance(stream, int) and _current_stream(self._index) != on
        self._streams[on] = _event_on(self._index, on) if away else None


_RETIRED: list = []  # (library, handle, tensors) of closed lists that are still to be freed


def _free_retired() -> None:
    while _RETIRED and not _capturing():
        lib, handle, tensors = _RETIRED.pop()
        if lib.slm_grad_list_destroy(handle):
            _RETIRED.append((lib, handle, tensors))  # another thread captures
            return


def _capturing() -> bool:
    import torch

    return torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing()


def _stream_handle(stream) -> int | None:
    """The handle of a torch stream or a handle; None or 0: the legacy default stream."""
    if stream is None:
        return None
    handle = stream if isinstance(stream, int) else int(stream.cuda_stream)
    return 0 if handle == 1 else handle  # 1: cudaStreamLegacy, the same stream


def _current_stream(index: int) -> int:
    """The handle of a device's current stream; from the first call on torch's own lookup."""
    global _current_stream
    import torch

    _current_stream = torch._C._cuda_getCurrentRawStream
    return _current_stream(index)


def _torch_stream(stream: int | None, index: int):
    """torch's object for a stream handle (None or 0: the legacy default stream)."""
    import torch

    if not stream:
        return torch.cuda.default_stream(index)
    return torch.cuda.ExternalStream(stream, device=index)


def _on_stream(index: int, stream: int | None):
    """Context in which a stream is torch's current one."""
    import torch

    return torch.cuda.stream(_torch_stream(stream, index))


def _event_on(index: int, stream: int):
    """An event behind what is on a stream now; None where that is being captured
    (there is nothing to wait for outside of the graph)."""
    import torch

    with _on_stream(index, stream):
        if torch.cuda.is_current_stream_capturing():
            return None
        event = torch.cuda.Event()
        event.record()
    return event


def _order_behind(tensor, index: int, stream: int, event) -> bool:
    """Lets torch's current stream wait for the event, or without one for what is on
    ``stream``, where ``tensor`` was written, and tells the allocator that it is read
    there.  False inside a capture, which cannot wait for work outside of it."""
    import torch

    with torch.cuda.device(index):
        if torch.cuda.is_current_stream_capturing():
            return False
        current = torch.cuda.current_stream()
        if event is not None:
            current.wait_event(event)
        else:
            current.wait_stream(_torch_stream(stream, index))
        tensor.record_stream(current)
    return True
