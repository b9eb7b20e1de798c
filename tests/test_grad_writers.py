"""The order of backward passes that write the same parameter gradients, next to a thread that captures."""
import threading
import traceback

import pytest
import torch
import torch.nn as nn

from video_classification_amd import ops


class Event:
    def __init__(self):
        self.stream = self.behind = None

    def record(self, stream):
        assert not stream.capturing, "recorded into another thread's capture"
        self.stream, self.behind = stream, list(stream.done)


class Stream:
    """A stream as the order of gradient writers sees it: `done` is what its work comes after."""

    def __init__(self, handle, foreign=False):
        self.cuda_stream, self.stream_id = handle, handle if foreign or handle == 0 else 8 * handle + 3
        self.capturing, self.done = False, []

    def record_event(self):
        e = Event()
        e.record(self)
        return e

    def wait_event(self, event):
        if event.stream.capturing:
            raise RuntimeError("HIP invalidates the capture of the event's stream")
        self.done += event.behind

    def wait_stream(self, other):
        self.wait_event(other.record_event())


@pytest.fixture
def on(monkeypatch):
    """on(stream): makes it the current one."""
    now = [None]
    monkeypatch.setattr(ops, "_last_writer", {})
    monkeypatch.setattr(ops, "_marks", {}, raising=False)
    monkeypatch.setattr(ops, "_own_stream", lambda dev: Stream(99), raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: now[0].cuda_stream, raising=False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0].capturing)
    monkeypatch.setattr(torch.cuda, "Event", Event)

    def switch(stream):
        now[0] = stream
        return stream
    return switch


def write(stream, what):
    dev = torch.device("cuda", 0)
    ops._before_grads(dev)
    stream.done.append(what)
    ops._after_grads(dev)


def test_a_writer_on_a_stream_that_is_captured_by_now(on):
    a, b = Stream(1), Stream(2)
    write(on(a), "a")
    a.capturing = True  # by another thread
    write(on(b), "b")
    assert b.done == ["a", "b"]


def test_the_order_of_several_streams(on):
    a, b, c, d = Stream(0), Stream(1), Stream(2, foreign=True), Stream(3)
    write(on(a), "a")
    write(on(b), "b")
    write(on(c), "c")
    write(on(d), "d")
    assert set(d.done) == set("abcd")
    write(on(a), "e")
    assert set(a.done) == set("abcde")
    again = Stream(2, foreign=True)  # a handle that came back
    write(on(c), "f")
    write(on(again), "g")
    assert set(again.done) == set("abcdefg")


def test_a_capture_neither_waits_nor_is_waited_for(on):
    a, b = Stream(1), Stream(2)
    write(on(a), "a")
    b.capturing = True
    write(on(b), "captured")
    assert b.done == ["captured"]
    c = Stream(3)
    write(on(c), "c")
    assert c.done == ["a", "c"]


@pytest.mark.gpu
def test_an_eager_pass_beside_a_capture_on_the_last_writers_stream(cuda):
    """One thread captures on the stream of an earlier eager pass while another thread runs an eager one elsewhere."""
    torch.manual_seed(0)
    w, b = nn.Parameter(torch.randn(40, 64, device=cuda)), nn.Parameter(torch.randn(40, device=cuda))
    x, t = torch.randn(200, 64, device=cuda), torch.randint(0, 40, (200,), device=cuda)
    gn = nn.GroupNorm(4, 64).to(cuda)
    ops.linear_cross_entropy(x, w, b, t).backward()
    ops.group_norm(x, gn).backward(x)
    once = [p.grad.clone() for p in (w, b, gn.weight, gn.bias)]
    captured, eager, errors = torch.cuda.Stream(), torch.cuda.Stream(), []
    torch.cuda.synchronize()

    def step(stream):
        with torch.cuda.stream(stream):
            ops.linear_cross_entropy(x, w, b, t).backward()
            ops.group_norm(x, gn).backward(x)

    step(eager)
    step(captured)
    torch.cuda.synchronize()

    def other():
        try:
            step(eager)
        except Exception:  # handed to the test
            errors.append(traceback.format_exc())

    graph = torch.cuda.CUDAGraph()
    y = torch.zeros(8, device=cuda)
    with torch.cuda.graph(graph, stream=captured, capture_error_mode="thread_local"):
        y.add_(1)
        thread = threading.Thread(target=other)
        thread.start()
        thread.join(60)
        y.add_(1)
    assert not thread.is_alive() and not errors, errors
    torch.cuda.synchronize()
    for p, g in zip((w, b, gn.weight, gn.bias), once):
        assert torch.allclose(p.grad, 4 * g, rtol=1e-6, atol=0)
    before = [p.grad.clone() for p in (w, b, gn.weight, gn.bias)]
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert (y == 2 * (k + 1)).all()
    for p, g in zip((w, b, gn.weight, gn.bias), before):
        assert torch.equal(p.grad, g)  # the eager pass is in no graph
