"""Calls of the serving operators without tokens or heads."""
import pytest
import torch

import miniattn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


@pytest.mark.parametrize("kind", ["gqa", "mqa"])
@pytest.mark.parametrize("ragged", [False, True])
def test_module_step_without_tokens(kind, ragged):
    with torch.device(DEV):
        m = miniattn.GQA_Flash(256, 4, 2) if kind == "gqa" else miniattn.MQA_Flash(256, 4)
    m = m.to(BF16).requires_grad_(False)
    caches = [torch.ones((4, 16, 2 if kind == "gqa" else 1, 64), dtype=BF16, device=DEV) for _ in range(2)]
    table = torch.tensor([[0, 2], [3, 1]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([20, 5], dtype=torch.int32, device=DEV)
    x = torch.zeros((0, 256) if ragged else (2, 0, 256), dtype=BF16, device=DEV)
    cu = torch.zeros(3, dtype=torch.int32, device=DEV) if ragged else None
    for rope in (None, miniattn.rope_table(32, 64, device=DEV)):
        assert m.forward_paged(x, *caches, table, lens, cu_q=cu, rope=rope).shape == x.shape
    assert all(bool((c == 1).all()) for c in caches)
    miniattn.check_device_status(DEV)


def test_append_without_kv_heads():
    """Nothing would fill the rotated queries."""
    q = torch.ones((1, 1, 4, 64), dtype=BF16, device=DEV)
    none, cache = q[:, :, :0], torch.ones((4, 16, 0, 64), dtype=BF16, device=DEV)
    table, lens = torch.zeros((1, 2), dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="KV heads"):
        miniattn.paged_append(none, none, cache, cache, table, lens, q=q)
