"""miniattn.paged_attention behind a shared prefix that a launch of its own reads: what one sequence holds that is not a number,
out of range or nobody's stays its own."""
import pytest
import torch

import miniattn
from paged_reference import Paged, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16
SHARED, HKV, HQ, D, PAGE, B = 1024, 8, 32, 128, 32, 48   # 200 MB would be read without: a launch of its own
OUTSIDE = 10 ** 6                                          # no page of the cache


def _batch(lens, news, seed):
    p = Paged(lens, news, HKV, D, BF16, PAGE, shared=SHARED, seed=seed)
    gen = torch.Generator().manual_seed(seed + 1)
    return p, [torch.randn((n, HQ, D), generator=gen).to(BF16) for n in news]


def _call(p, rows, ragged, shared=SHARED):
    """Output (n,Hq,D) and lse (Hq,n) of each sequence."""
    if ragged:
        out, lse = miniattn.paged_attention(torch.cat(rows).to(DEV), p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=p.cu_q,
                                            max_q=max(p.news), shared_len=shared, return_lse=True)
        return list(out.split(p.news)), list(lse.split(p.news, 1))
    out, lse = miniattn.paged_attention(torch.stack(rows).to(DEV), p.k_cache, p.v_cache, p.table, p.seq_lens,
                                        shared_len=shared, return_lse=True)
    return list(out), list(lse)


def _right(p, rows, outs, lses, but=()):
    for b, (o, t, z, tz) in enumerate(zip(*p.expected(rows))):
        if b not in but:
            check(outs[b], o, t, f"sequence {b}")
            check(lses[b], z, tz, f"lse of sequence {b}")


@pytest.mark.parametrize("ragged", [False, True])
def test_a_row_whose_own_keys_are_nan(ragged):
    """The first token after the prefix is the only key that the launch over the rest sees of sequence 5: a NaN there is one in the
    row's result, for the query heads of that KV head, as it is without the prefix."""
    p, rows = _batch([SHARED + 1] * B, [1] * B, seed=51)
    p.k_cache[int(p.table[5, SHARED // PAGE]), 0, 3] = float("nan")
    for shared in (0, SHARED):
        outs, lses = _call(p, rows, ragged, shared)
        heads = torch.zeros(HQ, dtype=torch.bool, device=DEV)
        heads[12:16] = True
        assert torch.equal(outs[5][0].isnan(), heads[:, None].expand(HQ, D)) and torch.equal(lses[5][:, 0].isnan(), heads)
        _right(p, rows, outs, lses, but=(5,))
    o, t, z, tz = (x[5] for x in p.expected(rows))
    check(outs[5][:, ~heads], o[:, ~heads], t[:, ~heads], "the other heads")
    miniattn.check_device_status(DEV)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_values_of_the_prefix_that_are_no_numbers(value):
    """They are in the results of all who see them; a sequence of length 0 sees nothing, its rows are 0."""
    lens = [0] + [SHARED + 1 + i for i in range(B - 1)]
    p, rows = _batch(lens, [1] * B, seed=52)
    p.v_cache[int(p.table[1, 7]), 9, 2, 17] = value
    outs, lses = _call(p, rows, False)
    assert bool((outs[0] == 0).all()) and bool((lses[0] == -float("inf")).all())
    for b in range(1, B):
        odd = ~outs[b][0].isfinite()
        assert bool(odd[8:12, 17].all()) and int(odd.sum()) == 4


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("length", [10 ** 9, -3])
def test_a_length_that_is_out_of_range(length, ragged):
    """Reported; the others are right, although the spoiled slot's row of the block table holds no pages."""
    lens = [SHARED + 5 + 11 * i for i in range(B)]
    p, rows = _batch(lens, [1] * B, seed=53)
    p.seq_lens[1] = length
    p.table[1] = OUTSIDE
    outs, lses = _call(p, rows, ragged)
    with pytest.raises(RuntimeError, match="outside its tensors"):
        miniattn.check_device_status(DEV)
    _right(p, rows, outs, lses, but=(1,))


def test_a_sequence_without_rows():
    """Nobody needs its tokens: its length may be an old one, its pages somebody else's by now."""
    news = [1] * B
    news[4] = 0
    lens = [SHARED + 5 + 11 * i for i in range(B)]
    lens[4] = SHARED + 900   # the longest
    p, rows = _batch(lens, news, seed=54)
    p.table[4] = OUTSIDE
    outs, lses = _call(p, rows, True)
    _right(p, rows, outs, lses)
    miniattn.check_device_status(DEV)


def test_no_length_in_range():
    """Nothing is read; reported."""
    p, rows = _batch([SHARED + 1] * B, [1] * B, seed=55)
    p.seq_lens.fill_(-1)
    p.table.fill_(OUTSIDE)
    _call(p, rows, False)
    with pytest.raises(RuntimeError, match="outside its tensors"):
        miniattn.check_device_status(DEV)


@pytest.mark.parametrize("shared", [1056, 1120])   # the last 128 keys' second half is empty, or partly there
@pytest.mark.parametrize("at", [-1, -40, 500])
def test_a_key_of_the_prefix_that_is_nan(at, shared):
    """Every row that sees it is NaN, for the query heads of that KV head; sequences that end before it are not."""
    lens = [0, 300] + [shared + 1 + i for i in range(B - 2)]
    p = Paged(lens, [1] * B, HKV, D, BF16, 16, shared=shared, seed=56)
    rows = list(torch.randn((B, 1, HQ, D), generator=torch.Generator().manual_seed(57)).to(BF16))
    key = at % shared
    p.k_cache[int(p.table[5, key // 16]), key % 16, 3] = float("nan")
    outs, lses = _call(p, rows, False, shared)
    heads = torch.zeros(HQ, dtype=torch.bool, device=DEV)
    heads[12:16] = True
    for b, (o, t, z, tz) in enumerate(zip(*p.expected(rows))):
        nan = heads & (lens[b] > key)
        assert torch.equal(outs[b][0].isnan(), nan[:, None].expand(HQ, D)) and torch.equal(lses[b][:, 0].isnan(), nan)
        check(outs[b][:, ~nan], o[:, ~nan], t[:, ~nan], f"sequence {b}")
        check(lses[b][~nan], z[~nan], tz[~nan], f"lse of sequence {b}")
    miniattn.check_device_status(DEV)


def test_row_numbers_that_leave_the_queries():
    """Reported; the sequences before are right, rows of the last one that are there are left out or undefined."""
    p, rows = _batch([SHARED + 5 + 11 * i for i in range(B)], [1] * B, seed=58)
    p.cu_q[B] = B + 3
    outs, lses = _call(p, rows, True)
    with pytest.raises(RuntimeError, match="outside its tensors"):
        miniattn.check_device_status(DEV)
    _right(p, rows, outs, lses, but=(B - 1,))
