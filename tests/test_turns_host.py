"""Threads that share a handle (CPU only): binding the caller's stream and the
library call are one turn of the handle, in every operator, so that no thread's
work goes to another thread's stream or runs in another's ordered mode.  The
library is a recorder, the handle a stand-in with a handle's turn."""
import threading

import pytest
import torch

import kernix_b200 as kx
from kernix_b200 import sharded

A, B = 0xA0, 0xB0      # two threads' streams
REAL = kx._abi.lib


class Stand:
    """A handle's stream, mode and turn, without a device."""

    def __init__(self):
        self.device, self.stream, self.ordered_matmul = 0, 0, False
        self._turn = kx.Handle.adopt(kx.C.c_void_p(), 0)._turn
        self.ptr = self._h = kx.C.c_void_p(1)

    def set_stream(self, stream):
        self.stream = stream

    def set_ordered_matmul(self, ordered):
        self.ordered_matmul = ordered


class Recorder:
    """The library: shapes are the real one's; a call that enqueues, once
    inside, lets the other thread try to enqueue before it looks where it is."""

    SHAPES = ("kx_matmul_shape", "kx_conv2d_shape")

    def __init__(self, h):
        self.h, self.seen, self.inside = h, {}, threading.Event()
        self.tried = threading.Event()

    def __getattr__(self, name):
        if name in self.SHAPES:
            return getattr(REAL, name)

        def call(*_):
            mine = threading.current_thread().name
            if mine == "first":
                self.inside.set()
                self.tried.wait(5)
                # time to come in, if it can
                threading.Event().wait(0.05)
            self.seen.setdefault(mine, []).append((name, self.h.stream, self.h.ordered_matmul))
            return 0
        return call


class Binding:
    """The native binding: calls the library, or leaves the call to the general path."""

    def __init__(self, lib):
        def taking(results):
            return lambda *a: lib and (lib.from_the_binding(), *[None] * results)
        self.token_log_probs, self.token_log_probs_backward, self.grad_norm = taking(5), taking(1), taking(1)


def operators():
    x, y = torch.zeros(4, 4), torch.zeros(4, 4)
    img, w = torch.zeros(1, 1, 4, 4), torch.zeros(1, 1, 3, 3)
    t, r = torch.zeros(4, dtype=torch.int64), torch.zeros(4)
    out = lambda: torch.zeros(4, 4)  # noqa: E731
    plan = sharded.RowPlan(4, 1, 4)
    return {
        "matmul": lambda: kx.matmul(x, y),
        "matmul_into": lambda: kx.matmul_into(x, y, out()),
        "matmul_into_replicated": lambda: kx.matmul_into_replicated(x, y, out(), 4096),
        "matmul_reference": lambda: kx.matmul_reference(x, y),
        "conv2d": lambda: kx.conv2d(img, w),
        "conv2d_reference": lambda: kx.conv2d_reference(img, w),
        "tensordot": lambda: kx.tensordot(x, y, [1], [0]),
        "matmul_backward": lambda: kx.matmul_backward(x, y, out()),
        "conv2d_backward": lambda: kx.conv2d_backward(img, w, torch.zeros(1, 1, 2, 2)),
        "softmax": lambda: kx.softmax(x, -1),
        "softmax_temperature": lambda: kx.softmax_temperature(x, -1, 2.0),
        "attention": lambda: kx.attention(x, y, x, 2.0),
        "rows_sharded": lambda: sharded.rows_sharded(x, y, out(), plan, 0),
        "token_log_probs": lambda: kx.token_log_probs(x, t, top=1, entropy=True),
        "token_log_probs_into": lambda: kx.token_log_probs_into(x, t, kx.TokenLogProbs(log_probs=torch.zeros(4))),
        "token_log_probs_backward": lambda: kx.token_log_probs_backward(x, t, lse=r, grad_log_probs=r),
        "grad_norm": lambda: kx.grad_norm([x, y]),
        "clip_grad_norm": lambda: kx.clip_grad_norm([x, y], 1.0),
    }


@pytest.fixture
def shared(monkeypatch):
    h = Stand()
    lib = Recorder(h)
    streams = {"first": A, "second": B}
    monkeypatch.setattr(kx, "lib", lib)
    monkeypatch.setattr(kx._abi, "lib", lib)
    monkeypatch.setattr(kx, "_route", lambda t: h)
    monkeypatch.setattr(kx, "_device_index", lambda t: 0)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    monkeypatch.setattr(kx, "_current_stream", lambda dev: streams[threading.current_thread().name])
    monkeypatch.setattr(kx, "_native", lambda: Binding(None))
    monkeypatch.setattr(kx, "_norm_workspace", lambda: 64)
    return lib


def race(lib, first, second):
    """``first`` on stream A; while it is in the library, ``second`` on B."""
    failed = []

    def run(call, before):
        try:
            before()
            call()
        except BaseException as e:  # noqa: BLE001  (reported by the test's thread)
            failed.append(e)

    def after_the_first():
        lib.inside.wait(5)
        lib.tried.set()

    threads = [threading.Thread(target=run, args=(first, lambda: None), name="first"),
               threading.Thread(target=run, args=(second, after_the_first), name="second")]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
    assert not any(t.is_alive() for t in threads) and not failed, failed
    return lib.seen


@pytest.mark.parametrize("name", list(operators()))
def test_a_call_keeps_its_stream(shared, name):
    """Against a product and against log probabilities on the other stream."""
    ops = operators()
    for other in ("matmul", "token_log_probs"):
        shared.seen, shared.inside, shared.tried = {}, threading.Event(), threading.Event()
        seen = race(shared, ops[name], ops[other])
        assert [s for _, s, _ in seen["first"]] == [A] * len(seen["first"]), seen
        assert [s for _, s, _ in seen["second"]] == [B] * len(seen["second"]), seen


@pytest.mark.parametrize("name", ["token_log_probs", "token_log_probs_backward", "grad_norm", "clip_grad_norm"])
def test_a_call_through_the_binding_keeps_its_stream(shared, monkeypatch, name):
    monkeypatch.setattr(kx, "_native", lambda: Binding(shared))
    seen = race(shared, operators()[name], operators()["softmax"])
    assert seen == {"first": [("from_the_binding", A, False)], "second": [("kx_softmax_f32", B, False)]}


def test_ordered_mode_is_its_calls_own(shared):
    seen = race(shared, operators()["matmul_reference"], operators()["matmul"])
    assert [m for _, _, m in seen["first"]] == [True] and [m for _, _, m in seen["second"]] == [False]
    assert not shared.h.ordered_matmul


def test_host_products_take_a_turn_too(monkeypatch):
    """try_dense_matmul's staging and stream belong to the handle."""
    import numpy as np
    h = Stand()
    lib = Recorder(h)
    monkeypatch.setattr(kx, "lib", lib)
    monkeypatch.setattr(kx, "handle", lambda device=None: h)
    a = np.zeros((4, 4), np.float32)
    m = kx.MatrixInput.__new__(kx.MatrixInput)
    m.data, m._dims, m._strides, m.origin = a.reshape(-1), (4, 4), [4, 1], 0
    for call in (lambda: kx.try_dense_matmul(a, a, a.copy(), 4, 4, 4), lambda: kx.try_strided_matmul(m, m, a.copy())):
        lib.seen, lib.inside, lib.tried = {}, threading.Event(), threading.Event()
        order = []

        def second():
            with h._turn:
                order.append(list(lib.seen))

        race(lib, call, second)
        assert order == [["first"]]     # not before the product was done


def test_a_finaliser_may_call_within_a_turn():
    """The turn is its thread's: a call made while a call of the same thread
    has it goes ahead."""
    h = Stand()
    assert h._turn.acquire(timeout=1) and h._turn.acquire(timeout=1)
    h._turn.release()
    h._turn.release()


def test_threads_that_make_the_first_handle_at_once_share_it(monkeypatch):
    """Else each would have a turn, and calls of both, of its own."""
    both = threading.Barrier(2, timeout=5)

    class Slow:
        def __init__(self, device):
            both.wait()

    monkeypatch.setattr(kx, "Handle", Slow)
    monkeypatch.setattr(kx, "_handles", {})
    got = []
    threads = [threading.Thread(target=lambda: got.append(kx.handle(3))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(10)
    assert len(got) == 2 and got[0] is got[1] is kx.handle(3)


@pytest.mark.parametrize("name", ["matmul", "matmul_reference", "conv2d_reference", "token_log_probs", "grad_norm"])
def test_a_call_that_fails_gives_the_turn_back(shared, name):
    def fails(*_):
        raise kx.InvalidParameter("no")

    for broken in ("set_stream", "set_ordered_matmul"):
        if broken == "set_ordered_matmul" and "reference" not in name:
            continue
        setattr(shared.h, broken, fails)
        threading.current_thread().name, mine = "second", threading.current_thread().name
        try:
            with pytest.raises(kx.InvalidParameter):
                operators()[name]()
        finally:
            threading.current_thread().name = mine
        delattr(shared.h, broken)
        free = []
        t = threading.Thread(target=lambda: free.append(shared.h._turn.acquire(timeout=2)))
        t.start()
        t.join()
        assert free == [True]
        shared.h._turn = threading.RLock()
