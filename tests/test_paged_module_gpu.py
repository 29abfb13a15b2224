"""The serving operators together, as a server would use them: forward_paged of the modules (projections, append with rotation,
attention over the pages, output projection), prompts in chunks, then token by token, eager and captured."""
import pytest
import torch

import miniattn
from miniattn.ops import linear
from paged_reference import HALF_STEP, attention, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def _module(kind, d, heads, kv_heads, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    with torch.device(DEV):
        m = miniattn.GQA_Flash(d, heads, kv_heads) if kind == "gqa" else miniattn.MQA_Flash(d, heads)
    m = m.to(dtype).requires_grad_(False)
    for p in m.parameters():
        p.normal_(0.0, d ** -0.5, generator=gen)
    return m


def _cache(B, length, page, Hkv, D, dtype, seed=1):
    pages = (length + page - 1) // page
    caches = [torch.full((B * pages + 1, page, Hkv, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
    table = torch.randperm(B * pages + 1, generator=torch.Generator().manual_seed(seed))[:B * pages]
    return caches, table.view(B, pages).to(torch.int32).to(DEV)


def _held(caches, table, b, length):
    """The first `length` keys and values of a sequence."""
    return [c[table[b].long()].flatten(0, 1)[:length] for c in caches]


def _projected(y, layer):
    """layer(y) in 64 bits for 16-bit y, and what 32-bit sums and one rounding may be off by (K additions of 2^-24, and twice
    for sums that truncate)."""
    w, b = layer.weight.double(), layer.bias.double()
    out = y.double() @ w.T + b
    size = y.double().abs() @ w.abs().T + b.abs()
    return out, 1.01 * HALF_STEP[y.dtype] * out.abs() + 2 * w.shape[1] * 2.0 ** -24 * size


@pytest.mark.parametrize("kind,dtype,heads,kv,D,window,sinks,rot", [
    ("gqa", BF16, 8, 2, 64, None, 0, 64), ("gqa", F16, 4, 4, 128, 20, 2, 32), ("mqa", BF16, 8, 1, 64, None, 0, None),
    ("mqa", F16, 4, 1, 96, 33, 0, 96)])
def test_prompt_in_chunks_then_tokens(kind, dtype, heads, kv, D, window, sinks, rot):
    """What the cache holds is what was projected and rotated, and every step's output is attention over it."""
    d, B = heads * D, 3
    m = _module(kind, d, heads, kv, dtype)
    kv_layer = m.kv if kind == "gqa" else m.k_v
    caches, table = _cache(B, 200, 16, kv, D, dtype)
    rope = miniattn.rope_table(200, rot, device=DEV) if rot else None
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(3)
    for n in (50, 37, 1, 1, 5, 1):
        x = torch.randn((B, n, d), generator=gen, device=DEV).to(dtype)
        lens += n
        before = int(lens[0]) - n
        got = m.forward_paged(x, *caches, table, lens, rope=rope, window=window, sinks=sinks)
        assert got.shape == x.shape and got.dtype == dtype
        # the same projections (same call, same bits), rotated into a cache of their own
        q, new = linear(x, m.w_q, kv_layer)
        q, new = q.view(B, n, heads, D), new.view(B, n, 2, kv, D)
        apart = [c.clone() for c in caches]
        turned = miniattn.paged_append(new[:, :, 0], new[:, :, 1], *apart, table, lens, q=q, rope=rope)
        for b in range(B):
            keys, values = _held(caches, table, b, before + n)
            keys2, values2 = _held(apart, table, b, before + n)
            assert torch.equal(keys, keys2) and torch.equal(values, values2) and bool(keys.isfinite().all())
            o, tol, *_ = attention(turned[b], keys, values, before, window, sinks)
            want, tol_w = _projected(o.reshape(n, d).to(dtype), m.w_o)
            # o itself may be off by tol and by the rounding to dtype that the reference made above
            off = (tol + HALF_STEP[dtype] * o.abs()).reshape(n, d) @ m.w_o.weight.double().abs().T
            check(got[b], want, off + tol_w, f"{n} tokens at {before}, sequence {b}")
    miniattn.check_device_status(DEV)


def test_ragged_module_call():
    """Chunks of different lengths in one call, an empty sequence among them, against one call per sequence."""
    heads, kv, D, d = 8, 2, 64, 512
    m = _module("gqa", d, heads, kv, BF16)
    news = [40, 0, 3, 1]
    rope = miniattn.rope_table(64, 64, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn((sum(news), d), generator=gen, device=DEV).to(BF16)
    caches, table = _cache(4, 64, 16, kv, D, BF16)
    lens = torch.tensor(news, dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 40, 40, 43, 44], dtype=torch.int32, device=DEV)
    got = m.forward_paged(x, *caches, table, lens, cu_q=cu, max_q=40, rope=rope)
    q, new = linear(x, m.w_q, m.kv)
    turned = miniattn.paged_append(new.view(-1, 2, kv, D)[:, 0], new.view(-1, 2, kv, D)[:, 1], *[c.clone() for c in caches], table,
                                   lens, cu_q=cu, q=q.view(-1, heads, D), rope=rope)
    at = 0
    for b, n in enumerate(news):
        if n == 0:
            continue
        o, tol, *_ = attention(turned[at:at + n], *_held(caches, table, b, n), 0)
        want, tol_w = _projected(o.reshape(n, d).to(BF16), m.w_o)
        off = (tol + HALF_STEP[BF16] * o.abs()).reshape(n, d) @ m.w_o.weight.double().abs().T
        check(got[at:at + n], want, off + tol_w, f"sequence {b}")
        at += n


def test_captured_steps():
    """A decode step as a graph, lengths counted up inside it, replayed against the same steps issued one by one."""
    heads, kv, D, d, B = 8, 2, 128, 1024, 4
    m = _module("gqa", d, heads, kv, BF16)
    rope = miniattn.rope_table(300, 128, device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(5)
    prompt = torch.randn((B, 100, d), generator=gen, device=DEV).to(BF16)
    steps = torch.randn((20, B, 1, d), generator=gen, device=DEV).to(BF16)
    outs = []
    for captured in (False, True):
        caches, table = _cache(B, 300, 16, kv, D, BF16)
        lens = torch.full((B,), 100, dtype=torch.int32, device=DEV)
        m.forward_paged(prompt, *caches, table, lens, rope=rope)
        mine = []
        if not captured:
            for x in steps:
                lens += 1
                mine.append(m.forward_paged(x, *caches, table, lens, rope=rope))
        else:
            x = steps[0].clone()
            torch.cuda.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                lens += 1
                y = m.forward_paged(x, *caches, table, lens, rope=rope)
            for step in steps:
                x.copy_(step)
                g.replay()
                mine.append(y.clone())
        outs.append(torch.stack(mine))
    assert bool(outs[0].isfinite().all()) and torch.equal(outs[0], outs[1])
    miniattn.check_device_status(DEV)
