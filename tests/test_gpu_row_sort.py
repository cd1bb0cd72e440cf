"""The one-launch sort behind the embedding's gradient while other work holds and frees SMs, so that the blocks of its cluster
start at different times.  Gradients are small whole numbers: their sums are exact in any order and compared for equality."""
import pytest
import torch

import llm720_b200 as lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,V", [(1, 1), (300, 200), (5000, 70000), (16384, 32000), (40000, (1 << 24) + 5), (65536, 257)])
def test_gradients_beside_other_work_on_the_gpu(cuda_device, n, V):
    g = torch.Generator(device=cuda_device).manual_seed(n + V)
    weight = torch.zeros(V, 1, device=cuda_device, requires_grad=True)
    jobs = []
    for _ in range(4):
        ids = torch.randint(0, V, (n,), generator=g, device=cuda_device)
        dy = torch.randint(-3, 4, (n, 1), generator=g, device=cuda_device).float()
        ref = torch.zeros(V, dtype=torch.int64, device=cuda_device).index_add_(0, ids, dy.long().squeeze(1))
        jobs.append((ids, dy, ref.float().unsqueeze(1)))
    noise = [torch.randn(s, s, generator=g, device=cuda_device) for s in (256, 700, 1500)]
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    wrong = torch.zeros((), dtype=torch.int64, device=cuda_device)
    for turn in range(60):
        with torch.cuda.stream(side):
            m = noise[turn % 3]
            torch.mm(m, m)
        ids, dy, ref = jobs[turn % 4]
        got, = torch.autograd.grad(lib.embedding(ids, weight), weight, dy)
        wrong += (got != ref).sum()
    torch.cuda.current_stream().wait_stream(side)
    assert wrong.item() == 0
