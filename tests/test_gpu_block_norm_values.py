"""The norm in front of the layer in ``PEER.block_train``: forward and backward pass see the same values of it."""
import pytest
import torch

from llm720_b200 import PEER, autograd

pytestmark = pytest.mark.gpu


def _case(device, dtype=torch.float32, D=64, tokens=37, seed=3):
    g = torch.Generator(device=device).manual_seed(seed)
    m = PEER(D, D, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16]).to(device).to(dtype)
    m.table_grad_sums = "sorted"
    hidden = (2 * torch.randn(1, tokens, D, generator=g, device=device) + 0.25).to(dtype)
    dy = torch.randn(1, tokens, D, generator=g, device=device).to(dtype)
    return m, hidden, dy


@pytest.mark.parametrize("dtype,D,affine", [(torch.bfloat16, 512, True), (torch.bfloat16, 136, True), (torch.float32, 64, True),
                                            (torch.float32, 1000, False), (torch.bfloat16, 2048, False)])
def test_the_backward_pass_sees_the_norm_of_the_forward_pass(cuda_device, monkeypatch, dtype, D, affine):
    """The layer's input that the backward pass forms anew gives the scores of the forward pass, bit for bit."""
    m, hidden, dy = _case(cuda_device, dtype, D, 600)
    ln = torch.nn.LayerNorm(D, elementwise_affine=affine).to(cuda_device)
    if affine:
        with torch.no_grad():
            ln.weight.copy_(torch.linspace(0.7, 1.3, D))
            ln.bias.copy_(torch.linspace(-0.2, 0.3, D))
    seen = []
    inner = autograd._layer_grads
    monkeypatch.setattr(autograd, "_layer_grads", lambda module, op, x, *rest: (seen.append(x), inner(module, op, x, *rest))[1])
    h = hidden.clone().requires_grad_()
    y = m.block_train(h, ln)
    scores = m._last_expert_scores.clone()
    torch.autograd.grad(y, (h,), dy)
    with torch.no_grad():
        m(seen[0].view(hidden.shape))
        assert torch.equal(m._last_expert_scores, scores)
        assert torch.equal(m.block_forward(hidden, ln), y)
