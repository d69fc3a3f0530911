"""CPU: the chunk attention refuses a model that is not bf16 before it writes to the cache."""
import pytest
import torch

from computd_b200.dwa_lm import CausalSelfAttention, ChunkStep

BF16 = torch.bfloat16


class Untouched:
    def __getattr__(self, name):
        raise AssertionError(f"the cache's {name} was reached")


@pytest.mark.parametrize("model,table", [(torch.float32, torch.float32), (torch.float32, BF16), (BF16, torch.float32),
                                         (torch.float16, torch.float16)])
@pytest.mark.parametrize("tree", [False, True])
def test_other_types_are_refused_before_a_write(model, table, tree):
    attn = CausalSelfAttention(32, 2, 8, "cpu", model)
    cos = torch.ones((3, 8), dtype=table)
    ints = torch.zeros(3, dtype=torch.int32)
    step = ChunkStep(Untouched(), cos, cos, torch.zeros(3, dtype=torch.int64), ints[:1, None], ints[:1], ints[:2], 3,
                     True, torch.zeros((3, 1), dtype=torch.int64) if tree else None)
    with pytest.raises(ValueError, match="bf16"):
        attn.extend(torch.zeros((1, 3, 32), dtype=model), step, 0)
    with pytest.raises(AssertionError, match="append"):  # bf16 goes on to it
        attn.to(BF16).extend(torch.zeros((1, 3, 32), dtype=BF16),
                             ChunkStep(step.cache, cos.to(BF16), cos.to(BF16), *list(vars(step).values())[3:]), 0)
