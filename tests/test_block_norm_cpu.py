"""Refusals of the block's entry points that come before any launch, and so without a device: a norm whose parameters are not as
long as the rows would be read beyond its end."""
import pytest
import torch

from llm720_b200 import PEER
from llm720_b200.peer import PeerOp


def _layer():
    m = PEER(64, 64, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16])
    return m, torch.randn(1, 4, 64)


class Bare(torch.nn.Module):
    """weight, bias and eps, as block_forward reads them, without a normalized_shape"""
    eps = 1e-5

    def __init__(self, n_weight, n_bias):
        super().__init__()
        self.weight = None if n_weight is None else torch.nn.Parameter(torch.ones(n_weight))
        self.bias = None if n_bias is None else torch.nn.Parameter(torch.zeros(n_bias))


@pytest.mark.parametrize("norm", [lambda: torch.nn.LayerNorm(32), lambda: torch.nn.LayerNorm(128),
                                  lambda: torch.nn.LayerNorm(32, elementwise_affine=False), lambda: torch.nn.LayerNorm((4, 64))])
def test_a_norm_of_another_width_is_refused(norm):
    m, x = _layer()
    for grad in (True, False):
        with torch.set_grad_enabled(grad), pytest.raises(ValueError, match="normalises"):
            m.block_train(x, norm())
    if norm().weight is not None:
        with torch.no_grad(), pytest.raises(ValueError, match="64"):
            m.block_forward(x, norm())


@pytest.mark.parametrize("n_weight,n_bias", [(32, 64), (64, 32), (None, 8), (1, None)])
def test_parameters_of_another_length_are_refused(n_weight, n_bias):
    m, x = _layer()
    with torch.no_grad(), pytest.raises(ValueError, match="64"):
        m.block_forward(x, Bare(n_weight, n_bias))


def test_the_operator_refuses_them_too():
    op = PeerOp.__new__(PeerOp)                                 # as far as the checks need one
    op.device, op.handle, op.cfg = torch.device("cpu"), None, type("Config", (), {"input_dim": 64})
    h, out = torch.zeros(4, 64), torch.zeros(4, 64)
    for w, b in ((torch.ones(32), None), (None, torch.ones(65))):
        with pytest.raises(ValueError, match="64"):
            op.block_forward(h, {}, w, b, 1e-5, out)


def test_the_block_norms_entry_refuses_before_any_launch():
    from llm720_b200 import _lib
    native = _lib.load()

    def call(x=16, dt=_lib.DTYPE_BF16, w=None, b=None, eps=1e-5, rows=4, dim=8, out=16, mean=16, rstd=16):
        return native.peer_block_norm(x, dt, w, b, eps, rows, dim, out, mean, rstd, None)

    for kw in (dict(x=None), dict(out=None), dict(rows=-1), dict(dim=0), dict(dim=(1 << 20) + 1), dict(dt=_lib.DTYPE_E4M3),
               dict(eps=-1.0), dict(eps=float("nan")), dict(mean=None), dict(rstd=None), dict(x=17), dict(out=17), dict(w=18),
               dict(b=18), dict(mean=18)):
        assert call(**kw) == _lib.ERR_INVALID_ARG, kw
        assert "peer_block_norm" in _lib.last_error(None)
    assert call(rows=0, x=None, out=None) == _lib.OK
