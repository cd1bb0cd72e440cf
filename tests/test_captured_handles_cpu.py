"""A CUDA graph holds addresses of the scratch of the handle that it was captured with.  A longer input, another table type or
the host tier make the module take a new handle; the old one has to live on, or a replay works on freed memory.  Shown with
stand-ins for the handle and for the capture, so that nothing can be replayed."""
import gc
import weakref

import pytest
import torch

from llm720_b200 import PEER, functional, peer


class Handle:
    def __init__(self, *, max_tokens, **kw):
        self.cfg = type("Config", (), {"max_tokens": max_tokens})
        self.closed = False

    def close(self):
        self.closed = True

    def set_row_tier(self, *a):
        pass

    def forward(self, x, w, out):
        pass


@pytest.fixture
def capturing(monkeypatch):
    state = {"on": False}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["on"])
    monkeypatch.setattr(peer, "PeerOp", Handle)
    monkeypatch.setattr(functional, "PeerOp", Handle)
    monkeypatch.setattr(functional, "_OPS", {})
    return state


def _layer():
    return PEER(64, 64, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16])


@pytest.mark.parametrize("which", ["_operator", "_product_operator"])
def test_a_handle_that_was_captured_lives_on(capturing, which):
    m = _layer()
    take = getattr(m, which)
    take(torch.device("cuda", 0), torch.float32, 10)            # warm-up
    capturing["on"] = True
    held = weakref.ref(take(torch.device("cuda", 0), torch.float32, 10))
    capturing["on"] = False
    larger = take(torch.device("cuda", 0), torch.float32, 1000)
    gc.collect()
    assert held() is not None and held() is not larger and not held().closed
    m._op = m._sel_op = None                                    # what the host tier's switches do
    gc.collect()
    assert held() is not None
    del m, take, larger
    gc.collect()
    assert held() is None                                       # with the module, as its parameters


def test_a_handle_that_was_not_captured_goes(capturing):
    m = _layer()
    held = weakref.ref(m._operator(torch.device("cuda", 0), torch.float32, 10))
    m._operator(torch.device("cuda", 0), torch.float32, 1000)
    gc.collect()
    assert held() is None


@pytest.mark.parametrize("captured", [False, True])
def test_the_functional_form(capturing, captured):
    class Cuda(torch.Tensor):                                   # as far as the function looks before it asks for a handle
        device = property(lambda self: torch.device("cuda", 0))

    def call(T):
        x = torch.zeros(1, T, 64).as_subclass(Cuda)
        key = torch.zeros(16, 16)
        try:
            functional.peer_forward(x, torch.zeros(64, 64), None, key, key, torch.zeros(256, 64), torch.zeros(256, 64), 2, 256, 1, 4)
        except (RuntimeError, AssertionError):                  # no device for the output
            pass
    capturing["on"] = captured
    call(10)
    first, = functional._OPS.values()
    capturing["on"] = False
    call(1000)
    second, = functional._OPS.values()
    assert second is not first and first.closed == (not captured)
