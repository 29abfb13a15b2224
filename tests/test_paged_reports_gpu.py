"""Row numbers and lengths outside a paged call's tensors are reported, also those of a sequence that has no rows by them."""
import pytest
import torch

import miniattn
from paged_reference import Paged, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("rows,Hkv,lens,cu,good", [
    # the rows behind the first sequence's belong to nobody; every page that a row could need is there
    (400, 2, [900, 900, 900, 900], [0, 400, 0, 400, 0], ()),       # fall: nobody's results are defined
    (400, 2, [900, 900, 900, 900], [0, 400, 500, 450, 450], ()),   # fall, behind the rows of q
    (400, 2, [900, 900, 900, 900], [0, 400, 401, 402, 403], (0,)),  # behind the rows of q
    (400, 2, [900, 900, 900, 900], [-4, -2, 0, 0, 400], (3,)),      # in front of them
    (400, 2, [900, -1, 900, 900], [0, 400, 400, 400, 400], (0,)),   # a length without rows
    (400, 2, [900, 900, 10 ** 9, 900], [0, 400, 400, 400, 400], (0,)),
    (4096, 8, [4096, 900, 900, 900], [0, 4096, 4097, 4098, 4099], ()),  # too many items for any to be cut
    (4096, 8, [4096, 900, 900, -7], [0, 4096, 4096, 4096, 4096], ())])
def test_chunks(rows, Hkv, lens, cu, good):
    held = [n if 0 <= n < 10 ** 6 else 900 for n in lens]
    p = Paged(held, [min(rows, n) for n in held], Hkv, 64, BF16, 32, seed=61)
    gen = torch.Generator().manual_seed(62)
    q = torch.randn((rows, 4 * Hkv, 64), generator=gen).to(BF16)
    out, lse = miniattn.paged_attention(q.to(DEV), p.k_cache, p.v_cache, p.table, _ints(lens), cu_q=_ints(cu), return_lse=True)
    with pytest.raises(RuntimeError, match="outside its tensors"):
        miniattn.check_device_status(DEV)
    for b in good:
        o, t, z, tz = (x[b] for x in p.expected([q if i == b else q[:n] for i, n in enumerate(p.news)]))
        check(out[cu[b]:cu[b + 1]], o, t, f"sequence {b}")
        check(lse[:, cu[b]:cu[b + 1]], z, tz, f"lse of sequence {b}")


def test_chunks_in_order_are_not_reported():
    p = Paged([900, 0, 40, 900], [300, 0, 0, 90], 2, 64, BF16, 32, seed=63)
    q = torch.zeros((400, 8, 64), dtype=BF16, device=DEV)
    miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=p.cu_q)
    miniattn.check_device_status(DEV)


@pytest.mark.parametrize("total", [8, 3000])   # few rows and many: a CTA to a row, a warp to a row
@pytest.mark.parametrize("cu,lens", [
    ([5, 0, 4], [9, 30]),              # fall at once: no row is the first sequence's
    ([0, 8, 4001, 4005], [9, 30, 9]),  # behind the rows: no row at all
    ([-9, -4, 8], [9, 30]),            # in front of them
    ([0, 1, 2, 3, 0], [9, 9, 9, 9]),
    ([0, 8, 8], [9, -1]), ([0, 8, 8], [9, 10 ** 6])])
def test_append(cu, lens, total):
    B = len(lens)
    caches = [torch.zeros((2 * B, 16, 2, 64), dtype=BF16, device=DEV) for _ in range(2)]
    table = torch.arange(2 * B, dtype=torch.int32, device=DEV).view(B, 2)
    k = torch.ones((total, 2, 64), dtype=BF16, device=DEV)
    miniattn.paged_append(k, k, *caches, table, _ints(lens), cu_q=_ints(cu))
    with pytest.raises(RuntimeError, match="outside its tensors"):
        miniattn.check_device_status(DEV)


@pytest.mark.parametrize("total", [8, 3000])
def test_append_in_order_is_not_reported(total):
    caches = [torch.zeros((6, 16, 2, 64), dtype=BF16, device=DEV) for _ in range(2)]
    table = torch.arange(6, dtype=torch.int32, device=DEV).view(3, 2)
    k = torch.ones((total, 2, 64), dtype=BF16, device=DEV)
    miniattn.paged_append(k, k, *caches, table, _ints([9, 32, 0]), cu_q=_ints([2, 6, 6, 8]))
    miniattn.check_device_status(DEV)
