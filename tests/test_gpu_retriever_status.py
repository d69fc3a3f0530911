"""GPU: the status word of a retrieval plan that has not been called."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_status_before_the_first_call():
    import computd_b200 as cb

    for _ in range(3):
        junk = [torch.full((1 << 22,), 1, dtype=torch.uint8, device="cuda") for _ in range(8)]
        del junk
        keys = torch.zeros((512, 64), dtype=torch.bfloat16, device="cuda")
        r = cb.Retriever(keys, keys, 16, 8)
        assert r.status() == 0
