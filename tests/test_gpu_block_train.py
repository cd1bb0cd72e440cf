"""Training form of the block, ``hidden + PEER(LayerNorm(hidden))``, its 8-bit checkpoints, the expert tables' gradient by
sorted ids, and a run of all of them with the embedding below.

Tolerances: fp32 layers within 2e-5 of the largest entry of autograd through the oracle (as for the layer's own
gradients: the sums differ in order only); bf16 tables' sorted sums within half a step of bf16 of the fp32 sums plus
the order of at most n additions of fp32.  Where a kernel's result is compared with another run of the same kernels on
the same numbers, the comparison is for equality."""
import pytest
import torch

import llm720_b200 as lib
from llm720_b200 import PEER, synthetic as syn
from oracle import peer_oracle as orc
from _util import load_golden, make_op, oracle_shape, oracle_weights, rel_err

pytestmark = pytest.mark.gpu


def _module(cfg, sd, device, index_mode="reference"):
    m = PEER(**cfg.module_kwargs()).to(cfg.dtype)
    m.load_state_dict({k: v.to(cfg.dtype) for k, v in sd.items()})
    m = m.to(device).eval()
    m.index_mode = index_mode
    return m


def _ln(D, seed, device):
    ln = torch.nn.LayerNorm(D, eps=1e-5)
    g = torch.Generator().manual_seed(seed)
    with torch.no_grad():
        ln.weight.copy_(1.0 + 0.2 * torch.randn(D, generator=g))
        ln.bias.copy_(0.1 * torch.randn(D, generator=g))
    return ln.to(device)


def _grads(m, ln, hidden, dy):
    h = hidden.detach().clone().requires_grad_()
    leaves = [h, ln.weight, ln.bias] + [p for n, p in m.named_parameters() if "sub_keys" not in n]
    y = m.block_train(h, ln)
    return y.detach(), torch.autograd.grad(y, leaves, dy), ["hidden", "ln.weight", "ln.bias"] + \
        [n for n, _ in m.named_parameters() if "sub_keys" not in n]


@pytest.mark.parametrize("sums", ["auto", "sorted"])
def test_block_train_against_autograd_through_the_oracle(cuda_device, sums):
    cfg, sd, x, _ = load_golden("c1_affine")
    m = _module(cfg, sd, cuda_device)
    m.table_grad_sums = sums
    ln = _ln(cfg.input_dim, 1, cuda_device)
    hidden = x * 3.0 + 0.5
    g = torch.Generator().manual_seed(3)
    dy = torch.randn(x.shape, generator=g)
    y, grads, names = _grads(m, ln, hidden.to(cuda_device), dy.to(cuda_device))
    with torch.no_grad():
        assert torch.equal(y, m.block_forward(hidden.to(cuda_device), ln))
    leaf = {k: v.float().clone().requires_grad_() for k, v in sd.items()}
    h = hidden.clone().requires_grad_()
    cpu_ln = _ln(cfg.input_dim, 1, "cpu")
    out, ids, _ = orc.forward(cpu_ln(h), oracle_weights(leaf), oracle_shape(cfg), "reference")
    assert torch.equal(m._last_expert_indices.cpu(), ids)
    (h + out).backward(dy)
    ref = {"hidden": h.grad, "ln.weight": cpu_ln.weight.grad, "ln.bias": cpu_ln.bias.grad, **{k: v.grad for k, v in leaf.items()}}
    for n, got in zip(names, grads):
        assert rel_err(got.cpu(), ref[n]) < 2e-5, (n, rel_err(got.cpu(), ref[n]))


def _bf16_case(device, tokens=(2, 150)):
    cfg = syn.scaled(syn.CONFIGS["c2"], product_key_dim=(64, 32), batch=tokens[0], seq=tokens[1], input_dim=512, output_dim=512,
                     num_heads=4, query_dim=128)
    sd = syn.make_weights(cfg, 9, device, random_affine=True)
    m = _module(cfg, sd, device, "product")
    m.table_grad_sums = "sorted"                              # the same from run to run
    hidden = (syn.make_input(cfg, 9, device).float() * 2.0 + 0.25).to(cfg.dtype)
    g = torch.Generator(device=device).manual_seed(4)
    dy = torch.randn(hidden.shape, generator=g, device=device).to(cfg.dtype)
    return m, _ln(cfg.input_dim, 2, device), hidden, dy


def test_checkpoint_of_a_representable_input_changes_nothing(cuda_device):
    """An input that its 8-bit form holds exactly: every gradient is bit for bit that of the node that keeps the tensor."""
    m, ln, hidden, dy = _bf16_case(cuda_device)
    hidden = lib.unpack_rows_e4m3(*lib.pack_rows_e4m3(hidden), hidden.dtype)
    y0, g0, names = _grads(m, ln, hidden, dy)
    m.activation_checkpoint = "e4m3"
    y1, g1, _ = _grads(m, ln, hidden, dy)
    assert torch.equal(y0, y1)
    for n, a, b in zip(names, g0, g1):
        assert torch.equal(a, b), n


def test_checkpoint_gradients_are_those_of_the_rounded_input(cuda_device):
    """The 8-bit node against the plain node whose kept input is replaced by the rounded one behind its back."""
    m, ln, hidden, dy = _bf16_case(cuda_device)
    flat = hidden.view(-1, hidden.shape[-1])

    def rounded(t):
        is_hidden = t.shape == flat.shape and t.dtype == flat.dtype and torch.equal(t, flat)
        return lib.unpack_rows_e4m3(*lib.pack_rows_e4m3(t), t.dtype) if is_hidden else t
    with torch.autograd.graph.saved_tensors_hooks(rounded, lambda t: t):
        y0, g0, names = _grads(m, ln, hidden, dy)
    m.activation_checkpoint = "e4m3"
    y1, g1, _ = _grads(m, ln, hidden, dy)
    assert torch.equal(y0, y1)
    for n, a, b in zip(names, g0, g1):
        assert torch.equal(a, b), n
    m.activation_checkpoint = None
    _, exact, _ = _grads(m, ln, hidden, dy)
    assert not torch.equal(exact[0], g1[0])                   # the rounding is there


def test_layer_keeps_its_input_in_8_bits(cuda_device):
    """PEER.forward with activation_checkpoint: gradients of the layer at a representable input, and what is kept."""
    m, _, hidden, dy = _bf16_case(cuda_device)
    hidden = lib.unpack_rows_e4m3(*lib.pack_rows_e4m3(hidden), hidden.dtype)
    kept = []
    def keep(t):
        kept.append((t.dtype, t.shape))
        return t
    results = []
    for mode in (None, "e4m3"):
        m.activation_checkpoint = mode
        kept.clear()
        h = hidden.clone().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
            y = m(h)
        results.append((y.detach(), torch.autograd.grad(y, (h, m.expert_down.weight, m.query_proj.weight), dy)))
        rows = (hidden.shape[0] * hidden.shape[1], hidden.shape[2])
        assert ((torch.bfloat16, rows) in kept) == (mode is None)
        assert ((torch.float8_e4m3fn, rows) in kept) == (mode == "e4m3")
    assert torch.equal(results[0][0], results[1][0])
    assert all(torch.equal(a, b) for a, b in zip(results[0][1], results[1][1]))


@pytest.mark.parametrize("dtype,D,Dout,H,k,N,T,act", [
    (torch.float32, 32, 48, 2, 4, 64, 7, "gelu"), (torch.float32, 256, 256, 4, 8, 300, 65, "relu"),
    (torch.float32, 1024, 512, 2, 4, 128, 1, "gelu"), (torch.bfloat16, 2048, 2048, 8, 16, 4096, 40, "gelu"),
    (torch.bfloat16, 512, 1024, 4, 8, 50, 129, "relu"), (torch.bfloat16, 64, 64, 8, 16, 3000, 700, "gelu"),
    (torch.bfloat16, 136, 72, 3, 15, 200, 33, "gelu"), (torch.float32, 512, 512, 5, 13, 90, 600, "relu")])
def test_sorted_table_gradients(cuda_device, dtype, D, Dout, H, k, N, T, act):
    """Against the form that adds in fp32 tables (itself checked against autograd), up to 90,000 selections."""
    g = torch.Generator().manual_seed(D + T)
    cfg = syn.PeerConfig("t", D, Dout, H, 32, (N, 1), k, dtype, dtype, 1, T)
    op = make_op(cfg, cuda_device, activation=act)
    dev = lambda t: t.to(cuda_device)
    x, dy = dev(torch.randn(T, D, generator=g).to(dtype)), dev(torch.randn(T, Dout, generator=g).to(dtype))
    down = dev((torch.randn(N, D, generator=g) * D ** -0.5).to(dtype))
    up = dev((torch.randn(N, Dout, generator=g) * D ** -0.5).to(dtype))
    ids = torch.randint(0, N, (T, H * k), generator=g, dtype=torch.int32)
    ids[:, 1] = ids[:, 0]                                      # the same row twice in a token
    ids[:, 2] = 3                                              # a row that every token names
    ids = dev(ids)
    w = dev(torch.rand(T, H * k, generator=g))
    gx, gw, gd, gu = op.gather_eval_backward(x, dy, ids, w, down, up)
    sx, sw, sd_, su = op.gather_eval_backward_sorted(x, dy, ids, w, down, up)
    op.query_status()
    assert torch.equal(gx, sx) and torch.equal(gw, sw)
    step = torch.finfo(dtype).eps / 2
    for got, ref in ((sd_, gd), (su, gu)):
        assert got.dtype == dtype
        count = torch.bincount(ids.flatten().long(), minlength=N).double().unsqueeze(1).to(cuda_device)
        # order of the fp32 additions: at most count additions of terms no larger than the largest sum's
        bound = step * ref.double().abs() + (2 * count + 4) * 2.0 ** -24 * ref.double().abs().max()
        assert ((got.double() - ref.double()).abs() <= bound).all()
        assert not got[count.squeeze(1) == 0].any()
    again = op.gather_eval_backward_sorted(x, dy, ids, w, down, up)
    assert all(torch.equal(a, b) for a, b in zip(again, (sx, sw, sd_, su)))


def test_sorted_table_gradients_skip_and_refuse(cuda_device):
    cfg = syn.PeerConfig("t", 32, 32, 1, 32, (16, 1), 2, torch.float32, torch.float32, 1, 3)
    op = make_op(cfg, cuda_device)
    dev = cuda_device
    x, dy = torch.randn(3, 32, device=dev), torch.randn(3, 32, device=dev)
    down, up = torch.randn(16, 32, device=dev), torch.randn(16, 32, device=dev)
    w = torch.ones(3, 2, device=dev)
    bad = torch.tensor([[0, 1], [99, 2], [-1, 3]], dtype=torch.int32, device=dev)
    got = op.gather_eval_backward_sorted(x, dy, bad, w, down, up)
    with pytest.raises(RuntimeError, match="outside"):
        op.query_status()
    # the same without the two ids: zero weight on any row leaves dx, and adds nothing to the tables
    w0 = w.clone()
    w0[1, 0] = w0[2, 0] = 0.0
    good = bad.clone()
    good[1, 0] = good[2, 0] = 5
    ref = op.gather_eval_backward_sorted(x, dy, good, w0, down, up)
    for a, b in zip(got[::2], ref[::2]):
        assert torch.equal(a, b)
    assert torch.equal(got[3], ref[3])
    # fewer rows than the table has: ids beyond them are skipped and reported
    got = op.gather_eval_backward_sorted(x, dy, good, w, down, up, grad_rows=4)
    assert got[2].shape == (4, 32)
    with pytest.raises(RuntimeError, match="outside"):
        op.query_status()
    empty = op.gather_eval_backward_sorted(x[:0], dy[:0], good[:0], w[:0], down, up)
    assert not empty[2].any() and not empty[3].any() and empty[0].shape == (0, 32)
    wide = syn.PeerConfig("w", 4096, 4096, 2, 32, (64, 1), 4, torch.bfloat16, torch.bfloat16, 1, 9)
    wop = make_op(wide, cuda_device)
    z = torch.zeros(9, 4096, dtype=torch.bfloat16, device=dev)
    t = torch.zeros(64, 4096, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError, match="4 KB"):
        wop.gather_eval_backward_sorted(z, z, torch.zeros(9, 8, dtype=torch.int32, device=dev), torch.zeros(9, 8, device=dev), t, t)


def test_block_train_in_slices_and_with_frozen_parts(cuda_device):
    """Longer than the handle's scratch: the same gradients; and with nothing below the layer to train."""
    m, ln, hidden, dy = _bf16_case(cuda_device, (2, 700))
    y0, g0, names = _grads(m, ln, hidden, dy)
    n, _, _, _ = _bf16_case(cuda_device, (2, 700))
    n.max_slice_tokens = 512
    y1, g1, _ = _grads(n, ln, hidden, dy)
    assert torch.equal(y0, y1) and torch.equal(m._last_expert_indices, n._last_expert_indices)
    for name, a, b in zip(names, g0, g1):
        assert torch.equal(a, b), name
    for p in ln.parameters():
        p.requires_grad_(False)
    y = m.block_train(hidden, ln)                             # hidden itself without a gradient
    up, = torch.autograd.grad(y, (m.expert_up.weight,), dy)
    assert torch.equal(up, g0[names.index("expert_up.weight")])
    for p in m.parameters():
        p.requires_grad_(False)
    y = m.block_train(hidden, ln)                             # nothing to train: the inference path
    assert not y.requires_grad and torch.equal(y, y0)
    h = hidden.clone().requires_grad_()
    dh, = torch.autograd.grad(m.block_train(h, ln), (h,), dy)
    assert torch.equal(dh, g0[0])


@pytest.mark.parametrize("ck", [None, "e4m3"])
def test_block_train_captured_and_replayed(cuda_device, ck):
    m, ln, hidden, dy = _bf16_case(cuda_device)
    m.activation_checkpoint = ck
    h = hidden.clone().requires_grad_()
    leaves = [h, ln.weight, ln.bias] + [p for n, p in m.named_parameters() if "sub_keys" not in n]

    def step():
        y = m.block_train(h, ln)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (1, 2):
        g = torch.Generator(device=cuda_device).manual_seed(seed)
        with torch.no_grad():
            h.copy_(torch.randn(h.shape, generator=g, device=cuda_device).to(h.dtype))
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_block_train_with_a_norm_in_the_layers_type(cuda_device):
    m, ln, hidden, dy = _bf16_case(cuda_device)
    with torch.no_grad():
        for p in ln.parameters():
            p.copy_(p.bfloat16())
    y0, g0, names = _grads(m, ln, hidden, dy)
    y1, g1, _ = _grads(m, ln.bfloat16(), hidden, dy)          # the same values, stored in bf16
    assert torch.equal(y0, y1)
    for name, a, b in zip(names, g0, g1):
        assert torch.equal(a.bfloat16(), b), name


def test_block_train_refusals(cuda_device):
    m = PEER(64, 64, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16]).to(cuda_device)
    x = torch.randn(1, 4, 64, device=cuda_device)
    with pytest.raises(ValueError, match="normalises"):
        m.block_train(x, torch.nn.LayerNorm(32).to(cuda_device))
    with pytest.raises(TypeError, match="parameters"):
        m.block_train(x, torch.nn.LayerNorm(64).to(cuda_device).half())
    m.activation_checkpoint = "int4"
    with pytest.raises(ValueError, match="activation_checkpoint"):
        m.block_train(x, torch.nn.LayerNorm(64).to(cuda_device))
    m.activation_checkpoint = "e4m3"
    m.dropout.p = 0.1
    with pytest.raises(RuntimeError, match="dropout"):
        m.train().block_train(x, torch.nn.LayerNorm(64).to(cuda_device))
    m.activation_checkpoint = None
    y = m.block_train(x, torch.nn.LayerNorm(64).to(cuda_device))         # dropout alone: the stages as separate nodes
    y.sum().backward()
    assert torch.isfinite(m.expert_down.weight.grad).all()
    n = PEER(64, 32, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16]).to(cuda_device)
    with pytest.raises(ValueError, match="adds its input back"):
        n.block_train(x, torch.nn.LayerNorm(64).to(cuda_device))
    f = PEER(64, 64, 256, num_experts_per_tok=4, num_heads=2, query_dim=32, product_key_dim=[16, 16]).to(cuda_device).bfloat16()
    f.quantize_tables_e4m3()
    with pytest.raises(RuntimeError, match="inference-only"):
        f.block_train(x.bfloat16(), torch.nn.LayerNorm(64).to(cuda_device))
    n.table_grad_sums = "other"
    with pytest.raises(ValueError, match="sorted"):
        n(x).sum().backward()


def test_training_step_of_a_small_model(cuda_device):
    """Embedding, two blocks and a final norm, as a training program strings them together: every gradient against
    autograd through torch's embedding and LayerNorm and the oracle's layer, in fp32."""
    cfg, sd, _, _ = load_golden("c1_affine")
    D, V = cfg.input_dim, 97
    g = torch.Generator().manual_seed(11)
    ids = torch.randint(0, V, (2, 40), generator=g)
    ids[0, :3] = 0                                             # padding
    table = 0.3 * torch.randn(V, D, generator=g)
    dy = torch.randn(2, 40, D, generator=g)
    scale = 2.5
    # the reference
    leaf = {k: v.float().clone().requires_grad_() for k, v in sd.items()}
    t = table.clone().requires_grad_()
    lns = [_ln(D, s, "cpu") for s in (1, 2, 3)]
    h = scale * torch.nn.functional.embedding(ids, t, padding_idx=0)
    chosen = []
    for ln in lns[:2]:
        out, sel, _ = orc.forward(ln(h), oracle_weights(leaf), oracle_shape(cfg), "reference")
        h = h + out
        chosen.append(sel)
    lns[2](h).backward(dy)
    # the library
    m = _module(cfg, sd, cuda_device)
    m.table_grad_sums = "sorted"
    dt = table.to(cuda_device).requires_grad_()
    glns = [_ln(D, s, cuda_device) for s in (1, 2, 3)]
    h = lib.embedding(ids.to(cuda_device), dt, scale, padding_idx=0)
    for ln, sel in zip(glns[:2], chosen):
        h = m.block_train(h, ln)
        assert torch.equal(m._last_expert_indices.cpu(), sel)
    lib.layer_norm(h, glns[2].weight, glns[2].bias, glns[2].eps).backward(dy.to(cuda_device))
    assert rel_err(dt.grad.cpu(), t.grad) < 2e-5 and not dt.grad[0].any()
    for a, b in zip(glns, lns):
        assert rel_err(a.weight.grad.cpu(), b.weight.grad) < 2e-5 and rel_err(a.bias.grad.cpu(), b.bias.grad) < 2e-5
    for n, p in m.named_parameters():
        if leaf[n].grad is not None:
            assert rel_err(p.grad.cpu(), leaf[n].grad) < 2e-5, n
    # the same model with 8-bit checkpoints runs, and its gradients point the same way
    m.zero_grad()
    m.activation_checkpoint = "e4m3"
    dt2 = table.to(cuda_device).requires_grad_()
    h = lib.embedding(ids.to(cuda_device), dt2, scale, padding_idx=0)
    for ln in glns[:2]:
        h = m.block_train(h, ln)
    lib.layer_norm(h, glns[2].weight, glns[2].bias, glns[2].eps, checkpoint="e4m3").backward(dy.to(cuda_device))
    for a, b in ((dt2.grad.cpu(), t.grad), (m.expert_down.weight.grad.cpu(), leaf["expert_down.weight"].grad)):
        assert torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), dim=0) > 0.95
