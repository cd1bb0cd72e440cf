"""layer_norm, pack_rows_e4m3 / unpack_rows_e4m3 and embedding against plain implementations in 64 bits.

Tolerances, from the arithmetic (u = 2^-24, half a step of fp32):
  * rounding to the output type: half a step, ``finfo.eps / 2`` of the value;
  * a sum over a row of D values adds at most D/32 + 16 numbers in a chain on any thread, so its error is at most
    ``(D/32 + 16) u`` of the sum of magnitudes; mean, variance and the two sums of the gradient are such sums;
  * a column sum over R rows has chains of at most R/64 + 600 additions;
  * packing has no arithmetic error: payload and scale are compared for equality.
The bounds below are these, with the terms written out at each check."""
import math

import pytest
import torch
import torch.utils.checkpoint

import llm720_b200 as lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):                     # results below the normal range round in steps of this size
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


# ---------------------------------------------------------------- references in 64 bits

def packed_reference(x):
    """(values the packed form of x stands for, scale) in 64 bits."""
    x = x.double()
    finite = torch.isfinite(x)
    top = torch.where(finite, x.abs(), 0.0).amax(-1, keepdim=True)
    m, e = torch.frexp(top / 448.0)
    e = torch.where(m > 0.5, e, e - 1).clamp_min(-126)
    scale = torch.where(top > 0, torch.ldexp(torch.ones_like(top), e), 1.0)
    v = torch.where(finite, x / scale, 0.0)
    octave = (torch.frexp(v)[1] - 1).clamp_min(-6)
    step = torch.ldexp(torch.ones_like(v), octave - 3)
    return torch.where(finite, torch.round(v / step) * step * scale, math.nan), scale.squeeze(-1)


def unpacked_reference(x, dtype):
    top = torch.finfo(dtype).max
    return packed_reference(x)[0].clamp(-top, top)


def norm_reference(x, w, b, eps, dy, kept=None):
    """y, dx, dw, db and the magnitudes their error bounds need, in 64 bits; ``kept``: what stands for x in the
    backward pass."""
    x, dy = x.double(), dy.double()
    D = x.shape[-1]
    w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(D, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    n = (x - mean) * r
    y = n * w + b
    nb = n if kept is None else (kept.double() - mean) * r
    g = dy * w
    m1, m2 = g.mean(-1, keepdim=True), (g * nb).mean(-1, keepdim=True)
    dx = r * (g - m1 - nb * m2)
    a = D / 32 + 16
    size = x.abs().amax(-1, keepdim=True) * r                 # rounding of the mean, seen after the scaling
    # n: mean off by a u max|x|, rstd off by a relative 2 a u (a squared deviation carries twice the mean's error)
    en = a * U * (size + 3 * n.abs())
    ey = en * w.abs() + 4 * U * (n.abs() * w.abs() + b.abs())
    enb = a * U * (size + 3 * nb.abs())
    ag = g.abs()
    em1 = a * U * ag.mean(-1, keepdim=True)
    em2 = a * U * (ag * nb.abs()).mean(-1, keepdim=True) + (ag * enb).mean(-1, keepdim=True)
    edx = r * (em1 + nb.abs() * em2 + enb * m2.abs()) + (4 + 2 * a) * U * r * (ag + m1.abs() + nb.abs() * m2.abs())
    chain = x.shape[0] / 64 + 600
    edw = chain * U * (dy * nb).abs().sum(0) + (dy.abs() * enb).sum(0)
    edb = chain * U * dy.abs().sum(0)
    return (y, dx, (dy * nb).sum(0), dy.sum(0)), (ey, edx, edw, edb)


def close(got, ref, err, what):
    assert got.shape == ref.shape, what
    bound = err + half_step(got.dtype) * (ref.abs() + err) + tiny(got.dtype)
    # IEEE rounding to nearest: a result beyond the largest finite value and half a step more is infinite (an fp16 row of
    # one value kept in 8 bits has a deviation of sqrt(eps) and a gradient of the rounding error squared over eps^1.5)
    top = torch.finfo(got.dtype).max * (1 + half_step(got.dtype))
    over = ref.abs() - bound >= top
    assert (got[over].double() == ref[over].sign() * math.inf).all(), what
    near = ref.abs() + bound >= top
    got, ref, bound = got[~near], ref[~near], bound[~near]
    off = (got.double() - ref).abs()
    worst = (off - bound).max().item() if got.numel() else 0.0
    assert worst <= 0.0, f"{what}: {off.max().item():.3g} off, {worst:.3g} over its bound"


def stream_rows(R, D, dtype, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(R, D, generator=g, device=device) * (0.25 + 2 * torch.rand(R, 1, generator=g, device=device))
    x += torch.randn(D, generator=g, device=device)
    if R > 2:
        x[1] = 0.0                                          # a padded row
        x[2] = 3.25                                         # a constant one
    return x.to(dtype)


def params(D, dtype, seed, device):
    g = torch.Generator(device=device).manual_seed(seed + 1000)
    w = (1 + 0.3 * torch.randn(D, generator=g, device=device)).to(dtype)
    return w, (0.2 * torch.randn(D, generator=g, device=device)).to(dtype)


# ---------------------------------------------------------------- layer norm

SHAPES = [(1, 1), (3, 2), (5, 31), (4, 32), (129, 33), (7, 256), (64, 1000), (300, 264), (9, 1537), (130, 2048), (33, 4096),
          (5, 4100), (3, 8192), (2, 20001), (3, 40960), (2000, 64), (4097, 8), (1, 4096), (2, 70000),
          (1500, 1537), (1100, 33), (1026, 2001), (1030, 4099), (1025, 8191), (1024, 1), (1300, 7), (1200, 1024), (1100, 1536),
          (2600, 511), (1040, 8192), (1033, 4100), (2100, 1537), (2050, 4099), (2049, 300), (2100, 8191)]


@pytest.mark.parametrize("ck", [None, "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,D", SHAPES)
def test_layer_norm_and_its_gradients(cuda_device, R, D, dtype, ck):
    x = stream_rows(R, D, dtype, R + D, cuda_device).requires_grad_()
    pdtype = dtype if (R + D) % 2 else torch.float32
    w, b = params(D, pdtype, R + D, cuda_device)
    w.requires_grad_(), b.requires_grad_()
    g = torch.Generator(device=cuda_device).manual_seed(5)
    dy = torch.randn(R, D, generator=g, device=cuda_device).to(dtype)
    y = lib.layer_norm(x, w, b, 1e-5, checkpoint=ck)
    grads = torch.autograd.grad(y, (x, w, b), dy)
    ref, err = norm_reference(x.detach(), w.detach(), b.detach(), 1e-5, dy,
                              unpacked_reference(x.detach(), dtype) if ck else None)
    for name, got, r, e in zip(("y", "dx", "dw", "db"), (y.detach(), *grads), ref, err):
        close(got, r, e, name)
    with torch.no_grad():
        assert torch.equal(lib.layer_norm(x, w, b, 1e-5), y)              # inference gives the same values
    again = torch.autograd.grad(lib.layer_norm(x, w, b, 1e-5, checkpoint=ck), (x, w, b), dy)
    assert all(torch.equal(a, c) for a, c in zip(again, grads))           # nothing depends on an order of arrival


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_layer_norm_with_parameters_missing(cuda_device, which, dtype):
    R, D = 37, 520
    x = stream_rows(R, D, dtype, 3, cuda_device).requires_grad_()
    w, b = params(D, dtype, 3, cuda_device)
    w = w.requires_grad_() if which == "weight" else None
    b = b.requires_grad_() if which == "bias" else None
    dy = torch.randn(R, D, device=cuda_device).to(dtype)
    y = lib.layer_norm(x, w, b)
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    ref, err = norm_reference(x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), 1e-5, dy)
    close(y.detach(), ref[0], err[0], "y")
    close(grads[0], ref[1], err[1], "dx")
    if w is not None:
        close(grads[1], ref[2], err[2], "dw")
    if b is not None:
        close(grads[1], ref[3], err[3], "db")


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_gradient_of_the_weight_alone(cuda_device, dtype):
    """An input without a gradient (the first norm above a frozen table)."""
    x = stream_rows(70, 192, dtype, 4, cuda_device)
    w, b = params(192, torch.float32, 4, cuda_device)
    w.requires_grad_()
    dy = torch.randn(70, 192, device=cuda_device).to(dtype)
    gw, = torch.autograd.grad(lib.layer_norm(x, w, b), (w,), dy)
    ref, err = norm_reference(x, w.detach(), b, 1e-5, dy)
    close(gw, ref[2], err[2], "dw")


@pytest.mark.parametrize("ck", [None, "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_of_strided_and_misaligned_inputs(cuda_device, dtype, ck):
    for R, D in ((6, 256), (1030, 256), (1100, 515), (2100, 515)):
        _strided(cuda_device, dtype, ck, R, D)


def _strided(cuda_device, dtype, ck, R, D):
    base = stream_rows(R * 5, D + 24, dtype, 6, cuda_device)
    flat = torch.randn(R * D + 3, device=cuda_device).to(dtype)
    w, b = params(D, torch.float32, 6, cuda_device)
    views = {"columns of wider rows": base[:R, 8:8 + D], "one element off": flat[1:1 + R * D].view(R, D),
             "odd row stride": torch.randn(R, D + 1, device=cuda_device).to(dtype)[:, :D],
             "every second row": base[:2 * R:2, :D], "transposed": torch.randn(D, R, device=cuda_device).to(dtype).t(),
             "three dimensions": torch.randn(4, R, D, device=cuda_device).to(dtype).transpose(0, 1),
             "one row repeated": base[:1, :D].expand(R, D)}
    for name, v in views.items():
        x = v.detach().requires_grad_()
        assert x.stride() == v.stride()
        for grad in (torch.randn(v.shape, device=cuda_device).to(dtype), torch.ones((), dtype=dtype, device=cuda_device).expand(v.shape),
                     torch.randn(v.shape[:-1] + (D + 8,), device=cuda_device).to(dtype)[..., :D]):
            y = lib.layer_norm(x, w, b, checkpoint=ck)
            dx, = torch.autograd.grad(y, (x,), grad)
            ref, err = norm_reference(v.reshape(-1, D), w, b, 1e-5, grad.reshape(-1, D),
                                      unpacked_reference(v.reshape(-1, D), dtype) if ck else None)
            close(y.detach().reshape(-1, D), ref[0], err[0], name + " y")
            close(dx.reshape(-1, D), ref[1], err[1], name + " dx")


def test_layer_norm_keeps_rows_apart(cuda_device):
    """A row with NaN or infinities ruins itself only; the sums over the rows are then NaN, as by the formula."""
    for dtype, R, D in [(t, *s) for t in DTYPES for s in ((40, 512), (40, 77), (1500, 512), (1500, 77), (1500, 2050), (1100, 5), (2200, 301), (2200, 2050))]:
        x = stream_rows(R, D, dtype, 8, cuda_device)
        clean = x.clone()
        x[5, D // 2], x[9, 0], x[11, D - 1] = math.nan, math.inf, -math.inf
        w, b = params(D, torch.float32, 8, cuda_device)
        dy = torch.randn(R, D, device=cuda_device).to(dtype)
        keep = [i for i in range(R) if i not in (5, 9, 11)]
        for ck in (None, "e4m3"):
            outs = []
            for t in (x, clean):
                t = t.detach().requires_grad_()
                y = lib.layer_norm(t, w, b, checkpoint=ck)
                outs.append((y.detach(), torch.autograd.grad(y, (t,), dy)[0]))
            for got, ref in zip(*outs):
                assert torch.equal(got[keep], ref[keep])
                assert got[[5, 9, 11]].isnan().any(-1).all()


def test_layer_norm_of_a_large_mean(cuda_device):
    """Values near 1000 with a deviation of 0.5: the variance is not lost to cancellation."""
    for R, D in ((64, 2048), (1100, 2048), (1100, 1999), (1030, 530)):
        x = (1000 + 0.5 * torch.randn(R, D, device=cuda_device)).requires_grad_()
        dy = torch.randn(R, D, device=cuda_device)
        y = lib.layer_norm(x)
        dx, = torch.autograd.grad(y, (x,), dy)
        ref, err = norm_reference(x.detach(), None, None, 1e-5, dy)
        close(y.detach(), ref[0], err[0], "y")
        close(dx, ref[1], err[1], "dx")
        assert (y - ref[0]).abs().max() < 2e-3                 # mean rounded to fp32: 1000 * 2^-24 / 0.5 and its sums


def test_rows_behind_two_to_the_31_elements(cuda_device):
    """Rows whose offsets pass 32 bits: the last 3000 of 1.1 million rows of 2048 (and of 2047) against a call on them
    alone, and table rows at the end of a table of that size."""
    n, tail = 1_100_000, 3000                                  # enough rows for the kernels of many rows
    for D in (2048, 2047):
        base = torch.randn(5000, D, device=cuda_device).bfloat16()
        x = base.repeat(n // 5000, 1)
        w, b = params(D, torch.float32, 7, cuda_device)
        for ck in (None, "e4m3"):
            outs = []
            for t in (x, x[-tail:].clone()):
                t = t.detach().requires_grad_()
                y = lib.layer_norm(t, w, b, checkpoint=ck)
                dx, = torch.autograd.grad(y, (t,), t.detach())
                outs.append((y.detach()[-tail:].clone(), dx[-tail:].clone()))
                del y, dx, t
            assert all(torch.equal(p, q) for p, q in zip(*outs))
        payload, scale = lib.pack_rows_e4m3(x)
        few, few_scale = lib.pack_rows_e4m3(x[-tail:])
        assert torch.equal(payload[-tail:].view(torch.uint8), few.view(torch.uint8)) and torch.equal(scale[-tail:], few_scale)
        assert torch.equal(lib.unpack_rows_e4m3(payload, scale)[-tail:], lib.unpack_rows_e4m3(few, few_scale))
        del payload, scale
        ids = torch.randint(n - 300, n, (4096,), device=cuda_device)
        table = x.requires_grad_()
        out = lib.embedding(ids, table, 2.0)
        assert torch.equal(out.detach(), (x.detach()[ids].float() * 2.0).bfloat16())
        g, = torch.autograd.grad(out, (table,), out.detach())
        small = x.detach()[n - 300:].clone().requires_grad_()
        gs, = torch.autograd.grad(lib.embedding(ids - (n - 300), small, 2.0), (small,), out.detach())
        assert torch.equal(g[n - 300:], gs) and not g[:n - 300].any()
        del x, table, out, g, small, gs, outs
        torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,D", [(5, 31), (40, 256), (1500, 77), (1500, 512), (2100, 515), (1030, 1536), (3, 20001)])
def test_gradient_of_a_residual_is_added_before_the_rounding(cuda_device, R, D, dtype):
    """The C entry's ``add``, on every kind of row: dx + add, rounded once."""
    from llm720_b200 import _lib
    x, add = stream_rows(R, D, dtype, 1, cuda_device), stream_rows(R, D, dtype, 2, cuda_device)
    dy = torch.randn(R, D, device=cuda_device).to(dtype)
    w, _ = params(D, torch.float32, 1, cuda_device)
    mean = x.double().mean(-1).float()
    rstd = (1 / torch.sqrt(x.double().var(-1, unbiased=False) + 1e-5)).float()
    out, dw = torch.empty_like(x), torch.empty(D, device=cuda_device)
    native = _lib.load()
    n = native.peer_layer_norm_workspace(R, D)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda_device)
    code = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}[dtype]
    _lib.check(native.peer_layer_norm_backward(
        dy.data_ptr(), D, x.data_ptr(), D, None, None, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), code, _lib.DTYPE_F32,
        add.data_ptr(), R, D, out.data_ptr(), dw.data_ptr(), None, ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream))
    ref, err = norm_reference(x, w, None, 1e-5, dy)
    close(out, ref[1] + add.double(), err[1] + 2 * U * (ref[1].abs() + add.double().abs()), "dx + add")
    close(dw, ref[2], err[2], "dw")


def test_layer_norm_against_differences(cuda_device):
    """dx, dw, db against central differences of sum(y * dy), y from the fp32 kernel, summed in 64 bits.  y carries
    an error of at most ~8 u |y|; through sum|dy| (~200) and h = 2^-6 that is ~2e-2; the third-order term h^2/6 is
    below 1e-2 of the gradient's norm."""
    x = torch.randn(4, 64, device=cuda_device)
    w, b = params(64, torch.float32, 9, cuda_device)
    dy = torch.randn(4, 64, device=cuda_device)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(lib.layer_norm(*leaves), leaves, dy)
    h = 2.0 ** -6
    for i in range(3):
        v = torch.randn_like(leaves[i])
        def loss(sign):
            args = [t.detach() for t in leaves]
            args[i] = args[i] + sign * h * v
            return (lib.layer_norm(*args).double() * dy.double()).sum()
        slope = ((loss(1) - loss(-1)) / (2 * h)).item()
        want = (grads[i].double() * v.double()).sum().item()
        assert abs(slope - want) <= 2e-2 + 1e-2 * (grads[i].norm() * v.norm()).item(), i


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,D", [(300, 8208), (200, 8201), (1100, 9216)])
def test_layer_norm_of_many_rows_beyond_8192_values(cuda_device, R, D, dtype):
    for ck in (None, "e4m3"):
        test_layer_norm_and_its_gradients(cuda_device, R, D, dtype, ck)
    test_gradient_of_a_residual_is_added_before_the_rounding(cuda_device, R, D, dtype)


def test_layer_norm_of_the_widest_row(cuda_device):
    D = 1 << 20
    for dtype, ck in ((torch.bfloat16, None), (torch.float32, "e4m3")):
        x = stream_rows(2, D, dtype, 12, cuda_device).requires_grad_()
        w, b = params(D, torch.float32, 12, cuda_device)
        w.requires_grad_()
        dy = torch.randn(2, D, device=cuda_device).to(dtype)
        y = lib.layer_norm(x, w, b, checkpoint=ck)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        ref, err = norm_reference(x.detach(), w.detach(), b, 1e-5, dy, unpacked_reference(x.detach(), dtype) if ck else None)
        for name, got, r, e in (("y", y.detach(), ref[0], err[0]), ("dx", dx, ref[1], err[1]), ("dw", dw, ref[2], err[2])):
            close(got, r, e, name)
        payload, scale = lib.pack_rows_e4m3(x)
        value, ref_scale = packed_reference(x.detach())
        assert torch.equal(payload.double() * scale.double().unsqueeze(-1), value) and torch.equal(scale.double(), ref_scale)


def test_layer_norm_in_inference_mode_and_recomputed(cuda_device):
    """Under torch.inference_mode, and inside torch's own recomputation of activations."""
    x = torch.randn(1200, 264, device=cuda_device, requires_grad=True)
    w, b = (t.requires_grad_() for t in params(264, torch.float32, 1, cuda_device))
    y = lib.layer_norm(x, w, b)
    with torch.inference_mode():
        assert torch.equal(lib.layer_norm(x, w, b), y)
        payload, scale = lib.pack_rows_e4m3(x)
        lib.unpack_rows_e4m3(payload, scale, torch.float32)
    dy = torch.randn_like(y)
    want = torch.autograd.grad(y, (x, w, b), dy)
    again = torch.utils.checkpoint.checkpoint(lib.layer_norm, x, w, b, use_reentrant=False)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(again, (x, w, b), dy), want))
    # part of the gradients only, and the rest later
    y = lib.layer_norm(x, w, b)
    part = torch.autograd.grad(y, (b,), dy, retain_graph=True) + torch.autograd.grad(y, (x, w), dy)
    assert all(torch.equal(p, q) for p, q in zip(part, (want[2], want[0], want[1])))


def test_an_input_changed_in_place_is_noticed(cuda_device):
    x = torch.randn(8, 16, device=cuda_device)
    w = torch.ones(16, device=cuda_device, requires_grad=True)
    y = lib.layer_norm(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = lib.layer_norm(x, w, checkpoint="e4m3")               # keeps its own copy of x
    x.add_(1)
    y.sum().backward()


def test_negated_views_are_read_with_their_signs(cuda_device):
    """The imaginary part of a conjugate is a view whose signs are in a flag, not in memory."""
    for D in (1, 40):
        z = torch.randn(6, D, dtype=torch.complex64, device=cuda_device)
        neg = z.conj().imag
        assert neg.is_neg()
        plain = -z.imag
        b = torch.randn(D, device=cuda_device, requires_grad=True)
        x = torch.randn(6, D, device=cuda_device, requires_grad=True)
        assert torch.equal(lib.layer_norm(neg, None, b), lib.layer_norm(plain, None, b))
        for got, want in zip(torch.autograd.grad(lib.layer_norm(x, None, b), (x, b), neg),
                             torch.autograd.grad(lib.layer_norm(x, None, b), (x, b), plain)):
            assert torch.equal(got, want)
        for got, want in zip(lib.pack_rows_e4m3(neg), lib.pack_rows_e4m3(plain)):
            assert torch.equal(got.float(), want.float())
        ids = torch.tensor([1, 0, 2, 2, 1, 5], device=cuda_device)
        grads = [torch.autograd.grad(lib.embedding(ids, x), (x,), dy)[0] for dy in (neg, plain)]
        assert torch.equal(*grads)
    one = torch.randn(1, dtype=torch.complex64, device=cuda_device).conj().imag
    with pytest.raises(ValueError, match="contiguous"):
        lib.layer_norm(torch.randn(3, 1, device=cuda_device), one)
    with pytest.raises(ValueError, match="contiguous"):
        lib.embedding(torch.tensor([0], device=cuda_device), one.view(1, 1))


def test_layer_norm_of_nothing(cuda_device):
    for shape in ((0, 64), (3, 0, 64)):
        x = torch.randn(shape, device=cuda_device, requires_grad=True)
        w, b = (t.requires_grad_() for t in params(64, torch.float32, 1, cuda_device))
        for ck in (None, "e4m3"):
            y = lib.layer_norm(x, w, b, checkpoint=ck)
            gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
            assert y.shape == shape and gx.shape == shape and not gw.any() and not gb.any()
    x = torch.randn(64, device=cuda_device)                   # one row without a row dimension
    ref, err = norm_reference(x.view(1, 64), None, None, 1e-5, x.view(1, 64))
    close(lib.layer_norm(x).view(1, 64), ref[0], err[0], "y")


def test_layer_norm_refusals(cuda_device):
    x = torch.randn(3, 16, device=cuda_device)
    w = torch.ones(16, device=cuda_device)
    with pytest.raises(ValueError, match="expected"):
        lib.layer_norm(x, w[:8])
    with pytest.raises(TypeError, match="parameters are"):
        lib.layer_norm(x, w.bfloat16())
    with pytest.raises(TypeError, match="one dtype"):
        lib.layer_norm(x.bfloat16(), w, w.bfloat16())
    with pytest.raises(RuntimeError, match="is on cpu"):
        lib.layer_norm(x, w.cpu())
    with pytest.raises(TypeError, match="float64"):
        lib.layer_norm(x.double())
    with pytest.raises(ValueError, match="eps"):
        lib.layer_norm(x, eps=-1e-5)
    with pytest.raises(ValueError, match="contiguous"):
        lib.layer_norm(x, torch.ones(32, device=cuda_device)[::2])
    with pytest.raises(ValueError, match="rows of at least"):
        lib.layer_norm(torch.randn((), device=cuda_device))
    with pytest.raises(ValueError, match="dim"):
        lib.layer_norm(torch.zeros(1, (1 << 20) + 1, device=cuda_device))
    y = lib.layer_norm(x.requires_grad_())
    g, = torch.autograd.grad(y.sum(), (x,), create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    g, = torch.autograd.grad(lib.layer_norm(x.detach(), w.requires_grad_(), w).sum(), (w,), create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    table = torch.randn(5, 4, device=cuda_device, requires_grad=True)
    g, = torch.autograd.grad(lib.embedding(torch.tensor([1, 2], device=cuda_device), table).sum(), (table,), create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()


# ---------------------------------------------------------------- 8-bit rows

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,D", SHAPES)
def test_packed_rows_equal_the_definition(cuda_device, R, D, dtype):
    x = stream_rows(R, D, dtype, R * 3 + D, cuda_device)
    payload, scale = lib.pack_rows_e4m3(x)
    value, ref_scale = packed_reference(x)
    assert payload.dtype == torch.float8_e4m3fn and payload.shape == x.shape
    assert torch.equal(scale.double(), ref_scale)
    assert torch.equal(payload.double() * scale.double().unsqueeze(-1), value)
    for out in DTYPES:
        top = torch.finfo(out).max
        assert torch.equal(lib.unpack_rows_e4m3(payload, scale, out), value.clamp(-top, top).to(out))
    # and the half step the format promises
    near = torch.maximum(x.double().abs(), (scale.double() * 2.0 ** -6).unsqueeze(-1)) * 2.0 ** -4
    assert ((value - x.double()).abs() <= near).all()


def test_packing_at_the_borders_of_the_format(cuda_device):
    """Every value halfway between two e4m3 values, largest magnitudes around 448 * 2^k, subnormal and topmost ones."""
    grid = torch.arange(0, 127, device=cuda_device, dtype=torch.uint8).view(torch.float8_e4m3fn).float()     # 0 .. 448
    mid = (grid[1:] + grid[:-1]) / 2
    rows = [torch.cat([grid, mid, -mid, torch.full((1,), 448.0, device=cuda_device)])]
    for k in (-130, -126, -100, 0, 60, 118):
        for m in (448.0, 448.0 * (1 + 2.0 ** -23), 448.0 * (1 - 2.0 ** -24), 511.0, 256.0, 449.0):
            r = torch.zeros_like(rows[0])
            r[0] = math.ldexp(m, k)
            r[1:100] = torch.linspace(-1, 1, 99, device=cuda_device) * r[0]
            rows.append(r)
    rows.append(torch.full_like(rows[0], 1e-45))
    rows.append(torch.full_like(rows[0], -3.4028234e38))
    x = torch.stack(rows)
    value, ref_scale = packed_reference(x)
    payload, scale = lib.pack_rows_e4m3(x)
    assert torch.equal(scale.double(), ref_scale)
    assert torch.equal(payload.double() * scale.double().unsqueeze(-1), value)
    top = torch.finfo(torch.float32).max
    assert torch.equal(lib.unpack_rows_e4m3(payload, scale, torch.float32), value.clamp(-top, top).float())
    for dtype, big in ((torch.float16, 65504.0), (torch.bfloat16, 3.3895313892515355e38)):
        x = torch.full((2, 16), big, device=cuda_device, dtype=dtype)
        x[1, 3:] = 1.0
        assert torch.isfinite(lib.unpack_rows_e4m3(*lib.pack_rows_e4m3(x), dtype)).all()
        assert torch.equal(lib.unpack_rows_e4m3(*lib.pack_rows_e4m3(x), dtype)[0], x[0])


def test_packing_infinities_and_nan(cuda_device):
    for D in (24, 256, 2048, 20001):
        for dtype in DTYPES:
            x = stream_rows(6, D, dtype, 2, cuda_device)
            x[0, 3], x[3, 0], x[4, D - 1], x[5] = math.inf, math.nan, -math.inf, math.nan
            value, ref_scale = packed_reference(x)
            payload, scale = lib.pack_rows_e4m3(x)
            assert torch.equal(scale.double(), ref_scale) and torch.isfinite(scale).all()
            got = lib.unpack_rows_e4m3(payload, scale, torch.float32).double()
            assert torch.equal(got.isnan(), ~torch.isfinite(x))
            assert torch.equal(got.nan_to_num(7.0), value.nan_to_num(7.0))


def test_packing_views_and_refusals(cuda_device):
    x = torch.randn(5, 7, 40, device=cuda_device).bfloat16()
    for v in (x[:, :, 3:20], x.transpose(0, 1), x[..., ::2], x[:, :1].expand(5, 7, 40), x[0], x[0, 0], x[:0]):
        payload, scale = lib.pack_rows_e4m3(v)
        value, ref_scale = packed_reference(v) if v.numel() else (v.double(), v[..., 0].double())
        assert payload.shape == v.shape and torch.equal(scale.double(), ref_scale)
        assert torch.equal(lib.unpack_rows_e4m3(payload, scale, torch.float32).double(), value)
    payload, scale = lib.pack_rows_e4m3(x)
    assert torch.equal(lib.unpack_rows_e4m3(payload[:, ::2], scale[:, ::2]), lib.unpack_rows_e4m3(payload, scale)[:, ::2])
    with pytest.raises(ValueError, match="belong together"):
        lib.unpack_rows_e4m3(payload, scale[:3])
    with pytest.raises(TypeError):
        lib.unpack_rows_e4m3(payload.view(torch.uint8), scale)
    with pytest.raises(TypeError):
        lib.unpack_rows_e4m3(payload, scale, torch.float64)
    with pytest.raises(RuntimeError, match="scale is on"):
        lib.unpack_rows_e4m3(payload, scale.cpu())
    with pytest.raises(TypeError):
        lib.pack_rows_e4m3(x.double())
    with pytest.raises(TypeError):
        lib.pack_rows_e4m3(payload)


# ---------------------------------------------------------------- embedding

def ids_of(kind, n, V, device, seed=0):
    g = torch.Generator(device=device).manual_seed(seed + n + V)
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=g, device=device)
    if kind == "one":
        return torch.full((n,), V // 2, device=device)
    if kind == "zipf":
        u = torch.rand(n, generator=g, device=device, dtype=torch.float64)
        return (torch.exp(u * math.log(V)) - 1).long().clamp(0, V - 1)
    if kind == "descending":
        return (V - 1 - torch.arange(n, device=device) % V)
    if kind == "none":
        return torch.full((n,), -1, device=device)
    ids = torch.randint(-3, V + 3, (n,), generator=g, device=device)               # "outside": some ids beyond the table
    ids[::3] = -1
    return ids


def embedding_reference(ids, weight, scale, dy, padding_idx):
    flat, V = ids.reshape(-1).long(), weight.shape[0]
    inside = (flat >= 0) & (flat < V)
    out = torch.zeros(flat.numel(), weight.shape[1], dtype=torch.float64, device=weight.device)
    out[inside] = weight.double()[flat[inside]] * scale
    take = inside if padding_idx is None else inside & (flat != padding_idx)
    grad = torch.zeros(weight.shape, dtype=torch.float64, device=weight.device)
    size = torch.zeros_like(grad)
    grad.index_put_((flat[take],), dy.reshape(-1, weight.shape[1])[take].double() * scale, accumulate=True)
    size.index_put_((flat[take],), dy.reshape(-1, weight.shape[1])[take].double().abs() * abs(scale), accumulate=True)
    chain = torch.zeros(V, dtype=torch.float64, device=weight.device)
    chain.index_put_((flat[take],), torch.ones(int(take.sum()), dtype=torch.float64, device=weight.device), accumulate=True)
    return out, grad, (chain.unsqueeze(1) + 1) * U * size          # at most as many additions in a chain as positions


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["uniform", "one", "zipf", "descending", "outside", "none"])
@pytest.mark.parametrize("n,V,D", [(1, 1, 1), (1, 5, 8), (7, 3, 33), (16, 16, 64), (17, 100, 7), (1000, 2, 40), (333, 5000, 136),
                                   (2049, 257, 24), (5000, 70000, 16), (12001, 500, 12),
                                   (20000, 33, 264), (33000, 300, 48), (70001, 1000, 8), (66000, 70000, 4)])
def test_embedding_and_its_gradient(cuda_device, n, V, D, kind, dtype):
    ids = ids_of(kind, n, V, cuda_device)
    if (n + V) % 2:
        ids = ids.int()
    g = torch.Generator(device=cuda_device).manual_seed(1)
    w = torch.randn(V, D, generator=g, device=cuda_device).to(dtype).requires_grad_()
    dy = torch.randn(n, D, generator=g, device=cuda_device).to(dtype)
    pad = V // 3 if (n + D) % 2 else None
    scale = 0.37
    dropped = torch.zeros(1, dtype=torch.int64, device=cuda_device)
    out = lib.embedding(ids, w, scale, padding_idx=pad, dropped=dropped)
    gw, = torch.autograd.grad(out, (w,), dy)
    ref, ref_grad, err = embedding_reference(ids, w.detach(), scale, dy, pad)
    close(out.detach(), ref, U * 2 * ref.abs(), "out")                  # scale rounded to fp32, one product
    close(gw, ref_grad, err + 2 * U * ref_grad.abs(), "grad")
    assert int(dropped) == int(((ids < 0) | (ids >= V)).sum())
    with torch.no_grad():
        assert torch.equal(lib.embedding(ids, w, scale, padding_idx=pad), out)
    again, = torch.autograd.grad(lib.embedding(ids, w, scale, padding_idx=pad), (w,), dy)
    assert torch.equal(again, gw)


def test_embedding_sums_in_the_order_of_the_positions(cuda_device):
    """Rows whose sum depends on the order of additions: the gradient is bit for bit the fp32 sum over the positions
    in order, for an id whose positions lie in one tile."""
    n, V = 12, 4
    ids = torch.tensor([2, 0, 2, 1, 2, 0, 2, 2, 1, 0, 2, 2], device=cuda_device)
    w = torch.zeros(V, 8, device=cuda_device, requires_grad=True)
    dy = torch.randn(n, 8, device=cuda_device) * torch.logspace(-6, 6, n, device=cuda_device).unsqueeze(1)
    gw, = torch.autograd.grad(lib.embedding(ids, w), (w,), dy)
    for v in range(V):
        acc = torch.zeros(8, device=cuda_device)
        for t in torch.nonzero(ids == v).flatten().tolist():
            acc = acc + dy[t]
        assert torch.equal(gw[v], acc)


@pytest.mark.parametrize("D", [1, 7, 40, 67])
@pytest.mark.parametrize("more", [0, 40000])
def test_embedding_of_ids_that_begin_and_end_anywhere_in_a_tile(cuda_device, more, D):
    """Ids with one position fewer, as many and one more than a tile of 16 or 64 (the latter behind 32,768 ids), from every
    offset in one; frequent ids next to one another."""
    repeats = [1, 15, 1, 16, 2, 17, 31, 32, 33, 3, 63, 64, 65, 5, 127, 128, 129, 16, 16, 64, 64, 17, 65, 7, 1500, 900] * 3
    for lead in (0, 1, 7, 15, 40):
        each = torch.tensor([lead] + repeats + [more], device=cuda_device)
        V = each.numel() + 2                                   # the last two without a position
        g = torch.Generator(device=cuda_device).manual_seed(lead)
        ids = torch.repeat_interleave(torch.arange(each.numel(), device=cuda_device), each)
        ids = ids[torch.randperm(ids.numel(), generator=g, device=cuda_device)]
        w = torch.randn(V, D, generator=g, device=cuda_device).bfloat16().requires_grad_()
        dy = torch.randn(ids.numel(), D, generator=g, device=cuda_device).bfloat16()
        gw, = torch.autograd.grad(lib.embedding(ids, w, 0.5), (w,), dy)
        ref, ref_grad, err = embedding_reference(ids, w.detach(), 0.5, dy, None)
        close(gw, ref_grad, err, "grad")
        assert not gw[-2:].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [1, 2, 3, 7, 9, 15, 31, 129, 514, 2051])
def test_embedding_rows_at_any_address(cuda_device, D, dtype):
    """Tables and gradients that begin at every value of 16 bytes, rows of odd widths; what lies around the rows is left
    alone and never enters them."""
    V, n = 37, 300
    g = torch.Generator(device=cuda_device).manual_seed(D)
    ids = torch.randint(-2, V, (n,), generator=g, device=cuda_device)
    nan = float("nan")
    for off in (0, 1, 3, 6):
        big = torch.full((V * D + 16,), nan, device=cuda_device, dtype=dtype)
        w = big[off:off + V * D].view(V, D).copy_(torch.randn(V, D, generator=g, device=cuda_device)).requires_grad_()
        wide = torch.full((n, D + 2 * off + 1), nan, device=cuda_device, dtype=dtype)
        dy = wide[:, off:off + D].copy_(torch.randn(n, D, generator=g, device=cuda_device))
        out = lib.embedding(ids, w, 3.0)
        gw, = torch.autograd.grad(out, (w,), dy)
        ref, ref_grad, err = embedding_reference(ids, w.detach(), 3.0, dy, None)
        close(out.detach(), ref, 0 * ref, "out")
        close(gw, ref_grad, err, "grad")


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_views_shapes_and_empty_batches(cuda_device, dtype):
    V, D = 50, 24
    w = torch.randn(V, D, device=cuda_device).to(dtype).requires_grad_()
    grid = torch.randint(0, V, (6, 5), device=cuda_device)
    for ids in (grid, grid.t(), grid[:, ::2], grid[0, 0], grid[:0], grid.int()):
        out = lib.embedding(ids, w, 2.0)
        assert out.shape == ids.shape + (D,)
        wide = torch.randn(out.shape[:-1] + (D + 5,), device=cuda_device).to(dtype)
        for dy in (wide[..., :D], wide[..., 1:D + 1], torch.ones((), device=cuda_device, dtype=dtype).expand(out.shape)):
            gw, = torch.autograd.grad(lib.embedding(ids, w, 2.0), (w,), dy)
            ref, ref_grad, err = embedding_reference(ids, w.detach(), 2.0, dy.reshape(-1, D), None)
            close(out.detach().reshape(-1, D), ref, 0 * ref, "out")
            close(gw, ref_grad, err, "grad")
    off = torch.randn(V * D + 1, device=cuda_device).to(dtype)[1:].view(V, D).requires_grad_()       # misaligned table
    out = lib.embedding(grid, off)
    close(out.detach(), off.detach()[grid].double(), 0 * out.double(), "out")


def test_embedding_against_differences(cuda_device):
    """The lookup is linear in the table: differences equal the gradient up to fp32 rounding of outputs of size ~3
    (2^-23 * 3 * sum|dy| ~ 1e-4 over h = 1)."""
    ids = torch.tensor([[3, 1, 1], [0, -1, 3]], device=cuda_device)
    w = torch.randn(5, 16, device=cuda_device, requires_grad=True)
    dy = torch.randn(2, 3, 16, device=cuda_device)
    gw, = torch.autograd.grad(lib.embedding(ids, w, 1.5), (w,), dy)
    v = torch.randn(5, 16, device=cuda_device)
    with torch.no_grad():
        f = lambda s: (lib.embedding(ids, w + s * v, 1.5).double() * dy.double()).sum()
        assert abs(((f(1) - f(-1)) / 2 - (gw.double() * v.double()).sum()).item()) < 1e-3


def test_embedding_refusals(cuda_device):
    w = torch.randn(8, 4, device=cuda_device)
    ids = torch.zeros(3, dtype=torch.int64, device=cuda_device)
    for bad, exc in ((lambda: lib.embedding(ids.float(), w), TypeError), (lambda: lib.embedding(ids.short(), w), TypeError),
                     (lambda: lib.embedding(ids.cpu(), w), RuntimeError), (lambda: lib.embedding(ids, w[0]), ValueError),
                     (lambda: lib.embedding(ids, w.t()), ValueError), (lambda: lib.embedding(ids, w, padding_idx=8), ValueError),
                     (lambda: lib.embedding(ids, w, padding_idx=-1), ValueError), (lambda: lib.embedding(ids, w.double()), TypeError),
                     (lambda: lib.embedding(ids, w, dropped=torch.zeros(1, device=cuda_device)), TypeError),
                     (lambda: lib.embedding(ids, w[:0]), ValueError)):
        with pytest.raises(exc):
            bad()


# ---------------------------------------------------------------- streams and captured graphs

def _all_outputs(x, w, b, table, ids, dy, dye):
    y = lib.layer_norm(x, w, b, checkpoint="e4m3")
    g = torch.autograd.grad(y, (x, w, b), dy)
    e = lib.embedding(ids, table, 3.0)
    ge, = torch.autograd.grad(e, (table,), dye)
    back = lib.unpack_rows_e4m3(*lib.pack_rows_e4m3(x), x.dtype)
    return [t.detach() for t in (y, *g, e, ge, back)]


def _inputs(device, seed, n, D, V):
    g = torch.Generator(device=device).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=device)
    x, table = r(n, D).bfloat16().requires_grad_(), r(V, D).bfloat16().requires_grad_()
    w, b = r(D).requires_grad_(), r(D).requires_grad_()
    ids = torch.randint(-1, V, (n,), generator=g, device=device)
    return x, w, b, table, ids, r(n, D).bfloat16(), r(n, D).bfloat16()


SIZES = [(300, 264, 90), (70000, 24, 90), (20000, 33, 5000)]       # one launch for the sort, three per digit, odd rows


@pytest.mark.parametrize("n,D,V", SIZES)
def test_two_streams_at_once(cuda_device, n, D, V):
    sets = [_inputs(cuda_device, s, n, D, V) for s in (1, 2)]
    want = [_all_outputs(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(cuda_device) for _ in sets]
    got = [[], []]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_all_outputs(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


@pytest.mark.parametrize("n,D,V", SIZES)
def test_captured_and_replayed_with_new_inputs(cuda_device, n, D, V):
    """Forward and backward in two captured graphs, replayed in turn with other inputs."""
    sets = [_inputs(cuda_device, s, n, D, V) for s in (3, 4)]
    fresh = [[t.detach().clone() for t in _inputs(cuda_device, s, n, D, V)] for s in (5, 6)]
    want = []
    for f in fresh:
        leaves = [t.clone().requires_grad_(i < 4) if t.is_floating_point() else t.clone() for i, t in enumerate(f)]
        want.append(_all_outputs(*leaves))
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in sets:
            _all_outputs(*s)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_all_outputs(*s))
        graphs.append(graph)
    for _ in range(2):
        for i in range(2):
            with torch.no_grad():
                for dst, src in zip(sets[i], fresh[i]):
                    dst.copy_(src)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))
