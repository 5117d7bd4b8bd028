"""Calls of the drafted tokens' operators that are refused on tensors of the GPU."""
import pytest
import torch

import llm_capi

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def test_grammars_of_no_masks(gpu):
    """An empty list of masks is not the same as no grammar, but where every row says that it has none."""
    x = torch.randn((3, 70), device="cuda")
    none = torch.zeros((0, 3), dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="mask"):
        llm_capi.logits_adjust(x, allowed=none)
    with pytest.raises(ValueError, match="mask"):
        llm_capi.logits_adjust(x, allowed=torch.zeros((2, 3), dtype=torch.int32, device="cuda"))
    got = llm_capi.logits_adjust(x, allowed=none, allowed_rows=i32([-1, 0, 5]))
    assert torch.equal(got, x)
    empty = llm_capi.logits_adjust(x[:0], allowed=none)
    assert empty.shape == (0, 70)
