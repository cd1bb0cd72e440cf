"""A captured training step, replayed after a longer input has made the module take a larger handle."""
import pytest
import torch

from llm720_b200 import PEER

pytestmark = pytest.mark.gpu


def test_a_step_is_replayed_after_the_handle_was_replaced(cuda_device):
    torch.manual_seed(5)
    m = PEER(64, 64, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16]).to(cuda_device)
    m.table_grad_sums = "sorted"
    ln = torch.nn.LayerNorm(64).to(cuda_device)
    h = torch.randn(1, 40, 64, device=cuda_device, requires_grad=True)
    dy = torch.randn(1, 40, 64, device=cuda_device)

    def step():
        y = m.block_train(h, ln)
        return [y.detach(), *torch.autograd.grad(y, (h, ln.weight, m.expert_down.weight, m.query_proj.weight), dy)]

    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    before = m._op
    with torch.no_grad():
        m.block_forward(torch.randn(2, 3000, 64, device=cuda_device), ln)
        assert m._op is not before
        h.copy_(torch.randn_like(h))
    graph.replay()
    got = [t.clone() for t in out]
    assert all(torch.equal(a, b) for a, b in zip(got, step()))
