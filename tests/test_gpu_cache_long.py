"""GPU: cache writes of more tokens than the blocks of one launch take (9472 to 18944 on 148 SMs)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [9473, 14209, 300001])
def test_repeated_slots_far_apart(dtype, src, T):
    """Each slot is named about ten times all over the list: the last token's values stay."""
    import computd_b200 as cb

    g = torch.Generator(device="cuda").manual_seed(T)
    page, pages, d = 16, T // 160, 16
    n = page * pages
    wide = torch.randint(-8, 9, (T, 3, d), device="cuda", generator=g).to(src)  # codes hold these exactly
    wide[:, :, 0] = 14.0 * 32
    k, v = wide[:, :1], wide[:, 1:2]  # strided tokens
    slots = torch.randint(-1, n, (T,), device="cuda", generator=g)
    slots[T // 2], slots[7] = n, -2
    fine = (slots >= 0) & (slots < n)
    last = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    last.scatter_reduce_(0, slots[fine], torch.arange(T, device="cuda")[fine], "amax")
    kc, vc = (torch.zeros((pages, 1, page, d), device="cuda").to(dtype) for _ in range(2))
    scales = {} if dtype is torch.bfloat16 else {name: torch.ones((pages, 1, page), device="cuda")
                                                 for name in ("k_scale", "v_scale")}
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    cb.kv_cache_write(k, v, kc, vc, slots, status=status, **scales)
    assert status.item() == 5
    for name, cache, x in (("k_scale", kc, k), ("v_scale", vc, v)):
        got = cache.float().view(n, d)
        if scales:
            got = got * scales[name].view(n, 1)
        want = torch.where(last[:, None] >= 0, x[last.clamp(min=0), 0].float(), 0.0)
        assert torch.equal(got, want)
