"""The block on a batch without tokens: the layer takes one, and so do block_forward and block_train, with gradients of zero."""
import pytest
import torch

from llm720_b200 import PEER

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sums", ["auto", "fp32", "sorted"])
@pytest.mark.parametrize("ck", [None, "e4m3"])
@pytest.mark.parametrize("shape", [(1, 0, 64), (0, 5, 64)])
def test_a_batch_without_tokens(cuda_device, shape, ck, sums):
    m = PEER(64, 64, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16]).to(cuda_device)
    m.table_grad_sums, m.activation_checkpoint = sums, ck
    ln = torch.nn.LayerNorm(64).to(cuda_device)
    h = torch.randn(shape, device=cuda_device, requires_grad=True)
    y = m.block_train(h, ln)
    assert y.shape == shape
    leaves = [h, ln.weight, ln.bias, m.query_proj.weight, m.query_layer_norm.weight, m.expert_down.weight, m.expert_up.weight]
    for leaf, g in zip(leaves, torch.autograd.grad(y, leaves, torch.ones_like(y))):
        assert g.shape == leaf.shape and not g.any()
    with torch.no_grad():
        assert m.block_forward(h, ln).shape == shape and m.block_train(h, ln).shape == shape
