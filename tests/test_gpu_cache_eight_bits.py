"""GPU check that values kept in eight bits are the quotients by their scale to nearest: 16-bit values over a scale often lie on the
border between two of them, where a product with the scale's reciprocal, off by one last place, takes the other one now and then."""
import pytest
import torch

from vllm_espalier.attention import PagedCache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [0.03, 0.0217, 1.7, 0.5, 3e-5, 900.0])
def test_values_are_the_nearest_quotients(dev, dtype, scale):
    """Every 16-bit pattern below 2^14 of either sign, as values and (without a norm and a rotation) as keys."""
    bits = torch.cat([torch.arange(0, 0x7F81), torch.arange(0, 0x7F81) - 0x8000]).to(torch.int16)
    x = bits.view(dtype)
    T = -(-x.numel() // 256)
    x = torch.nn.functional.pad(x, (0, T * 256 - x.numel())).view(T, 2, 128).to(dev)
    cache = PagedCache.empty(-(-T // 16), 16, 2, 128, torch.float8_e4m3fn, dev, k_scale=scale, v_scale=scale)
    cache.append(x, x, x, torch.arange(T, device=dev))
    # (the quotient in 64 bits, rounded to 32, lies on a border only where the exact one does, or next to it: 32 bits hold 20 more
    # than the eight-bit values' 4)
    want = (x.double().cpu() / torch.tensor(scale, dtype=torch.float32).double()).float().clamp(-448, 448).to(torch.float8_e4m3fn)
    for c in (cache.k, cache.v):
        got = c.reshape(-1, 2, 128)[:T].cpu()
        same = (got.view(torch.uint8) == want.view(torch.uint8)) | (got.float().isnan() & want.float().isnan())
        assert bool(same.all()), int((~same).sum())
