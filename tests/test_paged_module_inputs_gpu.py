"""forward_paged where the projections are the layers' own calls: what a layer returned is not the module's to write over."""
import pytest
import torch

import miniattn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
HEADS, D, PAGE = 4, 64, 16


def _module(kind):
    gen = torch.Generator(device=DEV).manual_seed(0)
    with torch.device(DEV):
        m = miniattn.GQA_Flash(HEADS * D, HEADS, 2) if kind == "gqa" else miniattn.MQA_Flash(HEADS * D, HEADS)
    m = m.to(BF16).requires_grad_(False)
    for p in m.parameters():
        p.normal_(0.0, 0.06, generator=gen)
    return m, (m.kv, 2) if kind == "gqa" else (m.k_v, 1)


def _serving(m, kv_layer, kv_heads, ragged):
    """x, the call, and what the operators give for the same queries and keys in caches of their own."""
    B, n = 2, 5
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn((B, n, HEADS * D), generator=gen, device=DEV).to(BF16)
    if ragged:
        x = x.flatten(0, 1)
    cu = torch.tensor([0, n, 2 * n], dtype=torch.int32, device=DEV) if ragged else None
    rope = miniattn.rope_table(32, D, device=DEV)
    table = torch.tensor([[0, 2], [3, 1]], dtype=torch.int32, device=DEV)
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    new_caches = lambda: [torch.zeros((4, PAGE, kv_heads, D), dtype=BF16, device=DEV) for _ in range(2)]  # noqa: E731
    call = lambda: m.forward_paged(x, *new_caches(), table, lens, cu_q=cu, rope=rope)  # noqa: E731

    def expected(q):
        caches = new_caches()
        rows = x.shape[:-1]
        kv = kv_layer(x).view(*rows, 2, kv_heads, D)
        turned = miniattn.paged_append(kv[..., 0, :, :], kv[..., 1, :, :], *caches, table, lens, cu_q=cu,
                                       q=q.clone().view(*rows, HEADS, D), rope=rope)
        return m.w_o(miniattn.paged_attention(turned, *caches, table, lens, cu_q=cu).reshape(x.shape))
    return x, call, expected


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("kind", ["gqa", "mqa"])
def test_a_hook_keeps_the_queries_it_saw(kind, ragged):
    m, (kv_layer, kv_heads) = _module(kind)
    x, call, expected = _serving(m, kv_layer, kv_heads, ragged)
    want = m.w_q(x)
    kept = []
    m.w_q.register_forward_hook(lambda layer, args, y: kept.append(y))
    got = call()
    assert len(kept) == 1 and torch.equal(kept[0], want)
    assert torch.equal(got, expected(want))


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("kind", ["gqa", "mqa"])
def test_a_layer_that_passes_its_input_on(kind, ragged):
    m, (kv_layer, kv_heads) = _module(kind)
    m.w_q = torch.nn.Identity()
    x, call, expected = _serving(m, kv_layer, kv_heads, ragged)
    before = x.clone()
    got = call()
    assert torch.equal(x, before)
    assert torch.equal(got, expected(before))
