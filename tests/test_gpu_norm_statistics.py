"""The statistics that the layer norm hands to its backward pass, of rows whose mean is large against their deviation, against 64
bits.  The deviation must not depend on how exactly the mean can be written in fp32.

Bounds (u = 2^-24, a = D / 32 + 16 as the chains of additions in test_gpu_row_ops.py): the mean is a sum of D values, off by at most
a u of the largest magnitude; a sum of squares of deviations is off by a relative a u, and so by 2 a u at most when formed from
parts about other points than the mean (which lie within a deviation or so of it here); 1 / sqrt halves that and adds two
roundings."""
import pytest
import torch

from llm720_b200 import _lib

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
CODES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _statistics(x, pack):
    R, D = x.shape
    y, stats = torch.empty_like(x), torch.empty(2, R, device=x.device)
    payload = torch.empty(R, D, dtype=torch.uint8, device=x.device) if pack else None
    scale = torch.empty(R, device=x.device) if pack else None
    p = lambda t: None if t is None else t.data_ptr()
    _lib.check(_lib.load().peer_layer_norm(p(x), D, CODES[x.dtype], None, None, _lib.DTYPE_F32, 1e-12, R, D, p(y), p(stats),
                                           stats[1].data_ptr(), p(payload), p(scale), torch.cuda.current_stream().cuda_stream))
    return stats


def _check(x, pack):
    D = x.shape[1]
    mean, rstd = _statistics(x, pack).double()
    d = x.double()
    ref = d.mean(-1)
    ref_rstd = 1 / torch.sqrt(((d - ref.unsqueeze(1)) ** 2).mean(-1) + 1e-12)
    a = D / 32 + 16
    assert ((mean - ref).abs() <= a * U * d.abs().amax(-1)).all()
    off = (rstd / ref_rstd - 1).abs().max().item()
    assert off <= (a + 2) * U, f"1 / deviation off by {off / U:.0f} u, {a + 2:.0f} allowed"


SHAPES = [(1030, 530), (1030, 1536), (1100, 520), (1100, 1999), (1100, 2048), (1100, 8191), (1100, 8192), (3, 513), (40, 1111),
          (64, 2048), (64, 8192), (5, 4100), (900, 640), (2, 20001), (1100, 257), (3, 129)]


@pytest.mark.parametrize("pack", [False, True])
@pytest.mark.parametrize("mean", [1000.0, -30000.0])
@pytest.mark.parametrize("R,D", SHAPES)
def test_deviation_of_rows_with_a_large_mean(cuda_device, R, D, mean, pack):
    for seed in range(4):
        g = torch.Generator(device=cuda_device).manual_seed(seed)
        _check(mean + 0.5 * torch.randn(R, D, generator=g, device=cuda_device), pack)


@pytest.mark.parametrize("dtype,mean", [(torch.bfloat16, 20.0), (torch.float16, 200.0)])
@pytest.mark.parametrize("R,D", SHAPES)
def test_deviation_in_16_bits(cuda_device, R, D, dtype, mean):
    g = torch.Generator(device=cuda_device).manual_seed(R)
    _check((mean + 0.5 * torch.randn(R, D, generator=g, device=cuda_device)).to(dtype), False)


@pytest.mark.parametrize("dtype,step", [(torch.float32, 0.25), (torch.bfloat16, 4.0), (torch.float16, 1.0)])
@pytest.mark.parametrize("R,D", SHAPES)
def test_deviation_of_nearly_constant_rows(cuda_device, R, D, dtype, step):
    """1000 everywhere but for five columns: a mean of up to 100,000 deviations."""
    g = torch.Generator(device=cuda_device).manual_seed(D)
    x = torch.full((R, D), 1000.0, device=cuda_device)
    at = torch.randint(0, D, (R, 5), generator=g, device=cuda_device)
    _check(x.scatter(1, at, 1000.0 + step).to(dtype), False)


@pytest.mark.parametrize("dtype", list(CODES))
@pytest.mark.parametrize("R,D", SHAPES)
def test_infinities_nan_and_overflowing_squares(cuda_device, R, D, dtype):
    """A row with an infinity or NaN has no finite statistics, whichever warp holds it; the rows beside it are untouched.  Squares
    beyond fp32 give a deviation of infinity (1 / deviation of zero), not NaN."""
    g = torch.Generator(device=cuda_device).manual_seed(D)
    x = torch.randn(R, D, generator=g, device=cuda_device).to(dtype)
    plain = _statistics(x, False).clone()
    for at in (0, D // 2, D - 1):
        for v in (float("inf"), float("-inf"), float("nan")):
            bad = x.clone()
            bad[R // 2, at] = v
            got = _statistics(bad, False)
            assert torch.isnan(got[1, R // 2]) or got[1, R // 2] == 0
            assert not torch.isfinite(got[0, R // 2])
            rest = torch.arange(R, device=cuda_device) != R // 2
            assert torch.equal(got[:, rest], plain[:, rest])
    if dtype != torch.float16:
        huge = x.float().mul(1e30).to(dtype)
        assert (_statistics(huge, False)[1] == 0).all()
    same = torch.full_like(x, 3.25)
    got = _statistics(same, False)
    # a deviation of zero: 1 / sqrt(eps), up to a squared error of the mean beside eps = 1e-12
    assert ((got[0] - 3.25).abs() <= (D / 32 + 16) * U * 3.25).all() and (got[1] > 0).all() and (got[1] <= 1.001e6).all()
