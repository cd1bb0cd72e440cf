"""gather_eval_backward_sorted compares the shapes of what it is given with its configuration before it makes a buffer or calls
the library: the kernels take sizes from the configuration, and would read or write beyond tensors of others."""
import pytest
import torch

from llm720_b200.peer import PeerOp

T, H, K, D, DOUT, N = 5, 2, 4, 64, 48, 30


def _op():
    op = PeerOp.__new__(PeerOp)                                 # as far as the checks need one; no library, no handle
    op.device, op.handle = torch.device("cpu"), None
    op.act_dtype = op.table_dtype = torch.float32
    op.cfg = type("Config", (), dict(input_dim=D, output_dim=DOUT, num_heads=H, top_k=K, num_experts=N, expert_hidden_size=1))
    return op


def _args(**kw):
    a = dict(x=torch.zeros(T, D), grad_out=torch.zeros(T, DOUT), ids32=torch.zeros(T, H * K, dtype=torch.int32),
             weights=torch.zeros(T, H * K), down=torch.zeros(N, D), up=torch.zeros(N, DOUT))
    a.update(kw)
    return a


@pytest.mark.parametrize("bad", [
    dict(x=torch.zeros(T, D - 16)), dict(x=torch.zeros(T * D)), dict(grad_out=torch.zeros(T - 1, DOUT)),
    dict(grad_out=torch.zeros(T, D)), dict(ids32=torch.zeros(T, K, dtype=torch.int32)), dict(weights=torch.zeros(T - 1, H * K)),
    dict(down=torch.zeros(N, D // 2)), dict(up=torch.zeros(N, D)), dict(up=torch.zeros(4, DOUT)),
    dict(grad_rows=N + 1), dict(grad_rows=0), dict(grad_rows=-3)])
def test_shapes_are_compared(bad):
    with pytest.raises(ValueError, match="expected|grad_rows"):
        _op().gather_eval_backward_sorted(**_args(**bad))


@pytest.mark.parametrize("good", [dict(), dict(down=torch.zeros(N - 1, D)),      # ids beyond it are skipped
                                  dict(ids32=torch.zeros(T, H, K, dtype=torch.int32), weights=torch.zeros(T, H, K)),
                                  dict(grad_rows=7), dict(grad_rows=7, down=torch.zeros(7, D), up=torch.zeros(9, DOUT))])
def test_good_shapes_reach_the_library(good):
    with pytest.raises(AttributeError, match="lib"):            # there is none behind this stand-in
        _op().gather_eval_backward_sorted(**_args(**good))
