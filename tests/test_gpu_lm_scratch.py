"""Scratch that the language-model operators take from the library's workspace."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_products_without_experts_take_none_for_slices():
    """No expert, so zeros and no products: nothing to cut into slices of k (32 of them would be 8 GB here)."""
    import stade_hip
    t, i, o = 63, 8192, 1 << 20
    y, x = torch.ones(t, o, dtype=torch.bfloat16, device="cuda"), torch.ones(t, i, dtype=torch.bfloat16, device="cuda")
    w, start = torch.empty(0, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    held = stade_hip.workspace_info()[0]
    print("expert_mul without experts", flush=True)
    stade_hip.expert_mul(y, x, w, start, i, o, t, 0)
    assert not y.any()
    assert stade_hip.workspace_info()[0] <= max(held, 64 << 20)
    xb = torch.ones(t, o, dtype=torch.bfloat16, device="cuda")
    stade_hip.expert_mul_b(x, None, xb, w, None, start, o, i, t, 0, add=False)
    assert not xb.any()
    assert stade_hip.workspace_info()[0] <= max(held, 64 << 20)
