"""unpack_rows_e4m3 of scales that pack_rows_e4m3 does not write: a caller's own, of any value and sign.  payload * scale in
fp32, clamped to the type's finite range, one rounding; the same whatever kernel a row's width and number lead to."""
import pytest
import torch

import llm720_b200 as lib

pytestmark = pytest.mark.gpu

SCALES = {torch.float16: [146.0, 146.5, 147.0, 200.0, 255.0, 300.0, -147.0, -200.0, -1e6],
          torch.bfloat16: [7.4e35, 7.6e35, 1.2e36, -1.2e36, 3e38], torch.float32: [7.5e35, 7.7e35, 1.2e36, -1.2e36, -3e38]}


@pytest.mark.parametrize("dtype", list(SCALES))
@pytest.mark.parametrize("R,D", [(3, 7), (2100, 64), (40, 2048), (1100, 515), (1030, 9001)])
def test_values_of_any_scale_are_clamped(cuda_device, dtype, R, D):
    g = torch.Generator(device=cuda_device).manual_seed(R + D)
    payload = torch.randint(0, 256, (R, D), generator=g, device=cuda_device, dtype=torch.uint8).view(torch.float8_e4m3fn)
    some = torch.tensor(SCALES[dtype] + [1.0, 0.0, float("inf"), float("nan")], device=cuda_device)
    scale = some[torch.arange(R, device=cuda_device) % some.numel()]
    got = lib.unpack_rows_e4m3(payload, scale, dtype)
    top = torch.finfo(dtype).max
    ref = (payload.float() * scale.unsqueeze(1)).clamp(-top, top).to(dtype)
    assert not torch.isinf(got).any()
    assert ((got == ref) | (torch.isnan(got) & torch.isnan(ref))).all()
