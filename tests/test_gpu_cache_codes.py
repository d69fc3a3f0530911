"""GPU: the e4m3 cache's codes bit for bit, by the definition's f32 divisions
(scale = max(amax / 448, 2^-126), code = e4m3(x / scale), rounded to nearest even)."""
import pytest
import torch

from test_gpu_decode import E4M3, quantise

pytestmark = pytest.mark.gpu


def _written(x):
    """Codes (as bytes) and scales of x [T, H, d], written in order."""
    import computd_b200 as cb

    T, H, d = x.shape
    shape = (-(-T // 16), H, 16, d)
    k, v = (torch.full(shape, 7.0, device="cuda").to(E4M3) for _ in range(2))
    ks, vs = (torch.zeros(shape[:3], device="cuda") for _ in range(2))
    cb.kv_cache_write(x, x, k, v, torch.arange(T, device="cuda"), k_scale=ks, v_scale=vs)
    assert torch.equal(k.view(torch.uint8), v.view(torch.uint8)) and torch.equal(ks, vs)
    codes = k.view(torch.uint8).transpose(1, 2).reshape(-1, H, d)[:T]
    return codes, ks.transpose(1, 2).reshape(-1, H)[:T]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [16, 80, 128])
def test_zeros_keep_their_signs(dtype, d):
    """Zeros of both signs among numbers, in vectors of nothing else, and next to tiny numbers."""
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn((40, 3, d), device="cuda", generator=g)
    x[torch.rand(x.shape, device="cuda", generator=g) < 0.3] = -0.0
    x[torch.rand(x.shape, device="cuda", generator=g) < 0.2] = 0.0
    x[3] = -0.0
    x[4] = 0.0
    x[5, :, ::2] = -0.0
    x[6] *= 2.0 ** -120
    x[7] = torch.where(x[7] == 0, x[7], -1e-38)
    x = x.to(dtype)
    codes, scales = _written(x)
    want, want_scales = quantise(x)
    assert torch.equal(codes, want.view(torch.uint8)) and torch.equal(scales, want_scales)
    assert int((codes == 0x80).sum()) > 0 and int((codes == 0).sum()) > 0


@pytest.mark.parametrize("low,high", [(-2, 2), (-30, 30), (-126, -90), (90, 127)])
def test_codes_of_many_pairs(low, high):
    """21 million (value, scale) pairs of values 2^low to 2^high, a fifth of them next to a border
    between two codes, where a quotient that is off by its last bit gives the other code."""
    g = torch.Generator(device="cuda").manual_seed(low + 200)
    shape = (20500, 8, 128)
    e = torch.rand(shape[:2] + (1,), device="cuda", generator=g) * (high - low - 1) + low
    x = torch.randn(shape, device="cuda", generator=g).clamp(-1, 1) * torch.exp2(e)
    scale = torch.clamp(x.abs().amax(-1, keepdim=True) / 448.0, min=2.0 ** -126)
    # halfway between two codes m 2^k and (m + 1) 2^k, m of 8 to 15, and its two neighbours in f32
    border = (torch.randint(8, 16, shape, device="cuda", generator=g) + 0.5) * \
        torch.exp2(torch.randint(-9, 5, shape, device="cuda", generator=g).float()) * scale
    border = (border.view(torch.int32) + torch.randint(-1, 2, shape, device="cuda", generator=g,
                                                       dtype=torch.int32)).view(torch.float32)
    at = (torch.rand(shape, device="cuda", generator=g) < 0.2) & (border < x.abs().amax(-1, keepdim=True))
    x = torch.where(at, torch.where(x < 0, -border, border), x)
    codes, scales = _written(x)
    want, want_scales = quantise(x)
    assert torch.equal(codes, want.view(torch.uint8)) and torch.equal(scales, want_scales)
