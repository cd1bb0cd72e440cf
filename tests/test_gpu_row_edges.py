"""Rows at odd addresses at the very ends of their buffers, and rows closer together than 16 bytes (expanded and overlapping
views) at odd addresses.  Bounds as in test_gpu_row_ops.py."""
import pytest
import torch

import llm720_b200 as lib
from test_gpu_row_ops import DTYPES, close, embedding_reference, norm_reference, packed_reference

pytestmark = pytest.mark.gpu
NAN = float("nan")


def _view(R, D, stride, off, dtype, device, seed):
    """[R, D] rows `stride` values apart, `off` values into a buffer of NaN."""
    g = torch.Generator(device=device).manual_seed(seed)
    extent = (R - 1) * stride + D
    buf = torch.full((off + extent + 16,), NAN, device=device, dtype=dtype)
    buf[off:off + extent] = torch.randn(extent, generator=g, device=device).to(dtype)
    return buf.as_strided((R, D), (stride, 1), off)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,D", [(1100, 515), (2100, 1031), (1030, 4099), (5, 515)])
@pytest.mark.parametrize("stride", [0, 1, 3, None])
def test_rows_close_together_at_odd_addresses(cuda_device, R, D, stride, dtype):
    x = _view(R, D, D if stride is None else stride, 1, dtype, cuda_device, R + D)
    payload, scale = lib.pack_rows_e4m3(x)
    ref, ref_scale = packed_reference(x)
    assert torch.equal(scale.double(), ref_scale) and torch.equal(payload.double() * scale.double().unsqueeze(1), ref)
    dy = _view(R, D, D if stride is None else stride, 3, dtype, cuda_device, R)
    w = torch.linspace(0.5, 1.5, D, device=cuda_device).requires_grad_()
    b = torch.zeros(D, device=cuda_device, requires_grad=True)
    leaf = x.detach().requires_grad_()
    for ck in (None, "e4m3"):
        y = lib.layer_norm(leaf, w, b, checkpoint=ck)
        kept = None if ck is None else lib.unpack_rows_e4m3(payload, scale, dtype)
        want, err = norm_reference(x, w.detach(), b.detach(), 1e-5, dy, kept)
        grads = torch.autograd.grad(y, (leaf, w, b), dy)
        for got, r, e, name in zip((y.detach(), *grads), want, err, ("y", "dx", "dw", "db")):
            close(got, r, e, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 3, 5, 7, 9, 33, 515])
def test_8_bit_rows_at_odd_addresses(cuda_device, D, dtype):
    """Payload rows of a few bytes that begin anywhere."""
    R = 1300
    g = torch.Generator(device=cuda_device).manual_seed(D)
    for off in (0, 1, 5, 15):
        buf = torch.full((off + R * D + 16,), 0x7f, device=cuda_device, dtype=torch.uint8)          # NaN around
        part = torch.randint(0, 0x7f, (R * D,), generator=g, device=cuda_device, dtype=torch.uint8)
        buf[off:off + R * D] = part
        payload = buf[off:off + R * D].view(R, D).view(torch.float8_e4m3fn)
        scale = torch.exp2(torch.randint(-4, 4, (R,), generator=g, device=cuda_device).float())
        got = lib.unpack_rows_e4m3(payload, scale, dtype)
        assert torch.equal(got.float(), part.view(R, D).view(torch.float8_e4m3fn).float() * scale.unsqueeze(1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 2, 3, 5, 9, 17, 130])
@pytest.mark.parametrize("stride", [0, 1, 2, None])
def test_gradient_rows_close_together_at_odd_addresses(cuda_device, D, stride, dtype):
    """Embedding gradients whose rows share granules with the ends of their buffer, and tables of very few rows."""
    g = torch.Generator(device=cuda_device).manual_seed(D)
    for V, n, off in ((1, 1, 1), (1, 40, 3), (3, 40, 5), (3, 700, 0), (50, 33000, 1)):
        ids = torch.randint(-1, V, (n,), generator=g, device=cuda_device)
        dy = _view(n, D, D if stride is None else stride, off, dtype, cuda_device, n)
        w = _view(V, D, D, off, dtype, cuda_device, V).requires_grad_()
        out = lib.embedding(ids, w, 2.0)
        gw, = torch.autograd.grad(out, (w,), dy)
        ref, ref_grad, err = embedding_reference(ids, w.detach(), 2.0, dy, None)
        close(out.detach(), ref, 0 * ref, "out")
        close(gw, ref_grad, err, "grad")
