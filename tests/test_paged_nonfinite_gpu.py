"""Keys that are no numbers: the rows that see one are NaN, for the query heads of its KV head, and nothing else is."""
import pytest
import torch

import miniattn
from paged_reference import Paged, attention, check, visible

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16
HKV, G, HEAD = 2, 4, 1   # the spoiled KV head


def _compare(out, lse, want, sees, what):
    """out (n,Hq,D), lse (Hq,n); sees (n,): rows that see a spoiled key."""
    nan = torch.zeros((out.shape[0], HKV * G), dtype=torch.bool, device=DEV)
    nan[sees, HEAD * G:(HEAD + 1) * G] = True
    assert torch.equal(out.isnan(), nan[..., None].expand(out.shape)), what
    assert torch.equal(lse.isnan(), nan.T), what
    o, t, z, tz = want
    check(torch.where(nan[..., None], 0, out.double()), torch.where(nan[..., None], 0, o), t, what)
    check(torch.where(nan.T, 0, lse.double()), torch.where(nan.T, 0, z), tz, f"lse, {what}")


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("keys", [[0], [700], [-1], [-20, 5], None])   # None: all
@pytest.mark.parametrize("n,window,sinks,D,dtype", [
    (1, None, 0, 128, BF16), (3, None, 0, 64, F16), (40, None, 0, 128, BF16), (300, None, 0, 96, F16), (1, 100, 3, 128, F16),
    (60, 100, 0, 64, BF16), (300, 257, 9, 128, BF16)])
def test_paged(n, window, sinks, D, dtype, keys, value):
    lens = [n + 5, 3000, n, 1200]
    spoiled = 1
    p = Paged(lens, [n] * 4, HKV, D, dtype, 16, window=window, sinks=sinks, seed=91)
    gen = torch.Generator().manual_seed(92)
    rows = [torch.randn((n, HKV * G, D), generator=gen).to(dtype) for _ in lens]
    length = lens[spoiled]
    where = torch.arange(length) if keys is None else torch.tensor(keys) % length
    for j in where.tolist():
        page = int(p.table[spoiled, j // 16])
        if page in range(p.k_cache.shape[0]):   # there: some row sees it
            p.k_cache[page, j % 16, HEAD] = value   # an infinity makes scores of both signs, and NaN of their sums
    sees = visible(n, length, length - n, window, sinks)[:, where].any(1)
    out, lse = miniattn.paged_attention(torch.stack(rows).to(DEV), p.k_cache, p.v_cache, p.table, p.seq_lens, window=window,
                                        sinks=sinks, return_lse=True)
    for b, want in enumerate(zip(*p.expected(rows))):
        _compare(out[b], lse[b], want, sees if b == spoiled else torch.zeros(n, dtype=torch.bool), f"sequence {b}")
    miniattn.check_device_status(DEV)


@pytest.mark.parametrize("key", [0, 500, 999])
@pytest.mark.parametrize("Nq", [1, 40, 1000])
def test_window_of_contiguous_keys(Nq, key):
    gen = torch.Generator().manual_seed(93)
    q, k, v = (torch.randn((1, m, h, 64), generator=gen).to(BF16).to(DEV) for m, h in ((Nq, HKV * G), (1000, HKV), (1000, HKV)))
    want = attention(q[0], k[0], v[0], 1000 - Nq, 129, 2)
    k[0, key, HEAD] = float("nan")
    out, lse = miniattn.flash_attn_fwd(q, k, v, causal=True, layout="bnhd", return_lse=True, q_pos0=1000 - Nq, window=129, sinks=2)
    _compare(out[0], lse[0], want, visible(Nq, 1000, 1000 - Nq, 129, 2)[:, key], f"key {key}")
