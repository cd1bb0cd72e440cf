"""The norm in front of the layer in ``PEER.block_train`` as a module with a behaviour of its own."""
import pytest
import torch

from llm720_b200 import PEER

pytestmark = pytest.mark.gpu


class Doubled(torch.nn.LayerNorm):
    def forward(self, x):
        return 2.0 * super().forward(x)


def _case(device, dtype=torch.float32, D=64, tokens=37, seed=3):
    g = torch.Generator(device=device).manual_seed(seed)
    m = PEER(D, D, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16]).to(device).to(dtype)
    m.table_grad_sums = "sorted"
    hidden = (2 * torch.randn(1, tokens, D, generator=g, device=device) + 0.25).to(dtype)
    dy = torch.randn(1, tokens, D, generator=g, device=device).to(dtype)
    return m, hidden, dy


def _hooked(kind, D):
    ln = Doubled(D) if kind == "subclass" else torch.nn.LayerNorm(D)
    if kind == "forward hook":
        ln.register_forward_hook(lambda mod, args, out: 2.0 * out)
    if kind == "pre-hook":
        ln.register_forward_pre_hook(lambda mod, args: (args[0] + torch.linspace(0, 1, D, device=args[0].device),))
    if kind == "backward hook":
        ln.register_full_backward_hook(lambda mod, gi, go: (3.0 * gi[0],))
    if kind == "own forward":
        ln.forward = lambda x: 2.0 * torch.nn.functional.layer_norm(x, (D,), ln.weight, ln.bias, ln.eps)
    return ln


@pytest.mark.parametrize("kind", ["subclass", "forward hook", "pre-hook", "backward hook", "own forward"])
def test_what_a_norm_does_beside_its_parameters_is_done(cuda_device, kind):
    """A norm with a forward or hooks of its own is called as a module."""
    m, hidden, dy = _case(cuda_device)
    ln = _hooked(kind, 64).to(cuda_device)
    leaves = lambda h: (h, ln.weight, m.expert_down.weight)
    h = hidden.clone().requires_grad_()
    want = h + m(ln(h))
    want_grads = torch.autograd.grad(want, leaves(h), dy)
    h = hidden.clone().requires_grad_()
    got = m.block_train(h, ln)
    got_grads = torch.autograd.grad(got, leaves(h), dy)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(got_grads, want_grads))
    with torch.no_grad():
        assert torch.equal(m.block_train(hidden, ln), want)
