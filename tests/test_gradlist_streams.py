"""Gradient lists and streams without a GPU: in which order the wrapper allocates,
calls, waits and reads.  The library and torch's streams are stand-ins."""
from __future__ import annotations

import contextlib
import ctypes
from types import SimpleNamespace

import pytest
import torch

from slmopt import B200Adamw, GradientList, gradlist

CURRENT, OTHER = 5, 7  # stream handles


@pytest.fixture
def log(monkeypatch):
    """What happens to streams, in order; torch's current stream is CURRENT."""
    events = []
    now = SimpleNamespace(stream=CURRENT)
    monkeypatch.setattr(gradlist, "_current_stream", lambda index: now.stream)
    monkeypatch.setattr(gradlist, "_use_on", lambda t, s: None, raising=False)

    @contextlib.contextmanager
    def on_stream(index, stream):
        before, now.stream = now.stream, stream or 0
        yield
        now.stream = before

    monkeypatch.setattr(gradlist, "_on_stream", on_stream, raising=False)

    def order(tensor, index, stream, event):
        # Behind the call's event where there is one: its stream may be gone by then.
        assert event is None or event.stream == stream
        events.append(("wait", now.stream, stream))
        return True

    monkeypatch.setattr(gradlist, "_order_behind", order, raising=False)

    def event_on(index, stream):
        return SimpleNamespace(stream=stream,
                               synchronize=lambda: events.append(("synchronize", stream)))

    monkeypatch.setattr(gradlist, "_event_on", event_on, raising=False)
    return SimpleNamespace(events=events, now=now)


def a_list(log, work_bytes=64):
    """A GradientList of two tensors whose library and allocator are stand-ins."""
    lst = GradientList.__new__(GradientList)
    lst._h = ctypes.c_void_p(1)
    lst.tensors = (torch.ones(3), torch.ones(2))
    lst.device, lst._index = torch.device("cpu"), 0
    lst._streams = {}
    lst.elements, lst._f32 = 5, torch.float32
    lst._lay_out(work_bytes)

    def empty(n, dtype, device):
        log.events.append(("allocate", log.now.stream))
        return torch.zeros(n, dtype=dtype)

    def call(h, *args):
        # The kernel is a stand-in: the norm of these tensors, written at once.
        log.events.append(("call", args[-1] or 0))
        values = args[-7]
        ctypes.memmove(values, (ctypes.c_float * 4)(5.0 ** 0.5, 0.25, 1.0, 0.0), 16)
        return 0

    lst._empty, lst._norm_call, lst._clip_call = empty, call, call
    lst.lib = SimpleNamespace(slm_grad_list_destroy=lambda h: 0)
    return lst


READS = {
    "read": lambda r: r.read().norm,
    "norm": lambda r: r.norm.item(),
    "clip_scale": lambda r: r.clip_scale.item(),
    "max_abs": lambda r: r.max_abs.item(),
    "nonfinite": lambda r: r.nonfinite.item(),
    "values": lambda r: r.values.tolist(),
    "sum_squares": lambda r: r.sum_squares.item(),
    "tensor_norms": lambda r: r.tensor_norms.tolist(),
    "tensor_max": lambda r: r.tensor_max.tolist(),
}


@pytest.mark.parametrize("stream", [OTHER, None])
@pytest.mark.parametrize("take", READS.values(), ids=READS.keys())
def test_results_are_read_behind_the_call(log, take, stream):
    lst = a_list(log)
    r = lst.norm(per_tensor=True, stream=stream)
    assert ("call", stream or 0) in log.events and not any(e[0] == "wait" for e in log.events)
    take(r)
    assert log.events[-1] == ("wait", CURRENT, stream or 0)
    take(r)  # once is enough
    assert sum(e[0] == "wait" for e in log.events) == 1
    log.now.stream = 9
    take(r)
    assert log.events[-1] == ("wait", 9, stream or 0)


def test_results_of_the_current_stream_wait_for_nothing(log):
    r = a_list(log).norm(stream=CURRENT)
    assert r.read().norm == pytest.approx(5.0 ** 0.5)
    r.values
    assert not any(e[0] == "wait" for e in log.events)
    log.now.stream = 0
    r = a_list(log).norm()  # None is the legacy default stream, torch's stream 0
    r.read()
    assert not any(e[0] == "wait" for e in log.events)


@pytest.mark.parametrize("work_bytes", [64, 1 << 20], ids=["small", "large"])
@pytest.mark.parametrize("stream", [OTHER, None, CURRENT, 1])
@pytest.mark.parametrize("call", ["norm", "clip"])
def test_results_and_workspace_come_from_the_calls_stream(log, call, stream, work_bytes):
    lst = a_list(log, work_bytes)
    getattr(lst, call)(stream=stream)
    on = 0 if stream in (None, 1) else stream
    assert log.events == [("allocate", on)] * (1 if work_bytes == 64 else 2) + [("call", on)]
    assert log.now.stream == CURRENT


def test_a_list_closed_inside_a_capture_is_freed_after_it(log, monkeypatch):
    freed, capturing, failing = [], [True], [0]

    def destroy(h):
        if failing[0]:
            return 1
        freed.append(h.value)
        return 0

    monkeypatch.setattr(gradlist, "_capturing", lambda: capturing[0], raising=False)
    lists = []
    for k in range(4):
        lst = a_list(log)
        lst._h = ctypes.c_void_p(10 + k)
        lst.lib = SimpleNamespace(slm_grad_list_destroy=destroy)
        lists.append(lst)
    lists[0].close()
    lists.pop(1).__del__()
    assert freed == []
    for call in (lists[0].norm, lists[0].clip, lambda: lists[0].handle):
        with pytest.raises(ValueError):
            call()
    capturing[0] = False
    lists[1].close()
    assert sorted(freed) == [10, 11, 12]
    failing[0] = 1  # another thread captures: the list is not lost
    lists[2].close()
    failing[0] = 0
    lists[2].close()
    lists[0].close()
    assert sorted(freed) == [10, 11, 12, 13]


@pytest.mark.parametrize("parameters", [4, 5, 6])
def test_a_handle_accumulates_lists_of_its_size_alone(log, parameters):
    opt = B200Adamw.__new__(B200Adamw)
    opt.P, opt._h = parameters, None
    lst = a_list(log)  # of 5 elements
    lst.lib.slm_grad_list_accumulate = lambda h, acc, n, overwrite, s: log.events.append(n) or 0
    acc = torch.zeros(5)
    if parameters == 5:
        opt.accumulate(acc, lst)
        assert log.events == [5]
        return
    with pytest.raises(ValueError):
        opt.accumulate(acc, lst)
    assert log.events == []


def test_tensors_let_go_by_a_bind_stay_until_their_streams_are_done(log, monkeypatch):
    monkeypatch.setattr(gradlist, "_torch_stream", lambda stream, index: stream or 0)

    class Tensor:
        def __init__(self, name):
            self.name = name

        def data_ptr(self):
            return 4096

        def record_stream(self, stream):
            log.events.append((self.name, stream))

    class Stream:  # torch's, which outlive every use
        cuda_stream = OTHER

    lst, out = a_list(log), a_list(log)
    for one in (lst, out):
        one._is = lambda t, shape: True
        one._shapes = [None, None]
        one.lib.slm_grad_list_bind = lambda h, ptrs, n, s: 0
        one.lib.slm_grad_list_accumulate = lambda h, acc, n, overwrite, s: 0
        one.bind([Tensor("a"), Tensor("b")])

    def released(which):
        log.events.clear()
        which.bind([Tensor("a"), Tensor("b")])
        return sorted(log.events)

    def stub(*args):
        return 0

    opt = B200Adamw.__new__(B200Adamw)
    opt.P, opt.device, opt._h, opt._check = 5, 0, None, lambda status: None
    opt.lib = SimpleNamespace(slm_opt_step_list=stub, slm_opt_norm_pass_list=stub,
                              slm_opt_norm_pass_accumulate_list=stub)
    monkeypatch.setattr("slmopt.optimizer._check_accumulator", lambda acc, n, device: None)
    assert released(lst) == []
    for call in (lambda **on: lst.norm(**on), lambda **on: lst.clip(out=out, **on),
                 lambda **on: lst.accumulate(torch.zeros(5), **on),
                 lambda **on: opt.step(lst, wait=False, **on),
                 lambda **on: opt.norm_pass(lst, **on),
                 lambda **on: opt.norm_pass_accumulate(torch.zeros(5), lst, **on)):
        call(stream=CURRENT)  # torch's current stream: in order by itself
        assert released(lst) == released(out) == []
        call(stream=Stream)
        call()
        assert released(lst) == [("a", 0), ("a", OTHER), ("b", 0), ("b", OTHER)]
        assert released(lst) == []
        released(out)
        call(stream=OTHER)  # a handle, whose stream its owner may destroy
        assert released(lst) == [("synchronize", OTHER)]
        released(out)
    lst.clip(out=out, stream=Stream)
    assert released(out) == released(lst) == [("a", OTHER), ("b", OTHER)]
