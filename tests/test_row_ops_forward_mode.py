"""Forward-mode differentiation: the operators have no such derivative, and a tangent that they would drop is refused.  The
refusal comes before the look at the device, so it is tested without one."""
import pytest
import torch
import torch.autograd.forward_ad as fw

import llm720_b200 as lib
from llm720_b200 import PEER


def _calls(device):
    x, w, b = torch.randn(4, 16, device=device), torch.ones(16, device=device), torch.zeros(16, device=device)
    ids, table = torch.tensor([1, 0, 3], device=device), torch.randn(5, 16, device=device)
    payload, scale = torch.zeros(4, 16, device=device).to(torch.float8_e4m3fn), torch.ones(4, device=device)
    dual = lambda t: fw.make_dual(t, torch.ones_like(t))
    return {
        "x": lambda: lib.layer_norm(dual(x), w, b), "weight": lambda: lib.layer_norm(x, dual(w), b),
        "bias": lambda: lib.layer_norm(x, w, dual(b)), "kept": lambda: lib.layer_norm(dual(x), checkpoint="e4m3"),
        "both modes": lambda: lib.layer_norm(dual(x.clone().requires_grad_()), w, b),
        "pack": lambda: lib.pack_rows_e4m3(dual(x)), "unpack": lambda: lib.unpack_rows_e4m3(payload, dual(scale)),
        "table": lambda: lib.embedding(ids, dual(table))}


NAMES = ["x", "weight", "bias", "kept", "both modes", "pack", "unpack", "table"]


def _refused(call):
    for guard in (torch.enable_grad, torch.no_grad):            # tangents go through no_grad
        with fw.dual_level(), guard(), pytest.raises(RuntimeError, match="forward-mode"):
            call()


@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused(name):
    _refused(_calls("cpu")[name])


def _layer():
    m = PEER(64, 64, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16])
    return m, torch.nn.LayerNorm(64), torch.randn(1, 4, 64)


def test_the_layer_refuses_tangents():
    m, ln, x = _layer()
    for frozen in (False, True):
        for p in [*m.parameters(), *ln.parameters()]:
            p.requires_grad_(not frozen)
        with fw.dual_level():
            dual = fw.make_dual(x, torch.ones_like(x))
            for call in (lambda: m(dual), lambda: m.block_train(dual, ln)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
    with fw.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
        m.block_forward(fw.make_dual(x, torch.ones_like(x)), ln)
    with fw.dual_level():                                       # a parameter's own
        ln.weight.requires_grad_(False)
        w = fw.make_dual(ln.weight.detach().clone(), torch.ones(64))
        del ln.weight
        ln.weight = w
        with pytest.raises(RuntimeError, match="forward-mode"):
            m.block_train(x, ln)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused_on_the_device(cuda_device, name):
    _refused(_calls(cuda_device)[name])


@pytest.mark.gpu
def test_with_forward_mode_off_a_tangent_is_not_looked_at(cuda_device):
    x = torch.randn(4, 16, device=cuda_device)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        with fw._set_fwd_grad_enabled(False):
            assert torch.equal(lib.layer_norm(dual), lib.layer_norm(x))
