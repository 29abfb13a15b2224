"""Numbers of a call that come as 0-dim tensors: a call goes by what they hold then.  What is no whole number is refused."""
import numpy as np
import pytest
import torch

import miniattn
from paged_reference import Paged

DEV = "cuda:0"
BF16 = torch.bfloat16


def _paged(window=None, **kw):
    p = Paged([700, 90], [2, 2], 2, 64, BF16, 16, seed=71)
    q = torch.randn((2, 2, 4, 64), generator=torch.Generator().manual_seed(72)).to(BF16).to(DEV)
    return lambda **kw: miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, **kw)


def _contiguous():
    gen = torch.Generator().manual_seed(73)
    q, k, v = (torch.randn((1, 2, n, 64), generator=gen).to(BF16).to(DEV) for n in (40, 300, 300))
    return lambda **kw: miniattn.flash_attn_fwd(q, k, v, causal=True, **{"q_pos0": 260, **kw})


@pytest.mark.gpu
@pytest.mark.parametrize("call,name,values,rest", [
    (_paged, "window", (64, 8), {}), (_paged, "sinks", (0, 30), {"window": 5}), (_paged, "softmax_scale", (0.5, 0.01), {}),
    (_paged, "shared_len", (16, 32), {}),
    (_contiguous, "window", (64, 8), {}), (_contiguous, "sinks", (1, 30), {"window": 5}),
    (_contiguous, "softmax_scale", (0.5, 0.01), {"window": 50}), (_contiguous, "q_pos0", (260, 100), {"window": 50}),
    (_contiguous, "k_pos0", (0, 100), {"window": 50})])
def test_changed_in_place(call, name, values, rest):
    call = call()
    held = torch.tensor(values[0])
    first = call(**{name: held}, **rest)
    assert torch.equal(first, call(**{name: values[0]}, **rest))
    held.fill_(values[1])
    again = call(**{name: held}, **rest)
    assert torch.equal(again, call(**{name: values[1]}, **rest))
    assert name == "shared_len" or not torch.equal(again, first)


@pytest.mark.gpu
@pytest.mark.parametrize("name,values", [("softmax_scale", (0.5, 0.01)), ("q_pos0", (260, 100)), ("k_pos0", (0, 100))])
def test_changed_in_place_without_a_window(name, values):
    gen = torch.Generator().manual_seed(76)
    q, k, v = (torch.randn((1, 2, n, 64), generator=gen).to(BF16).to(DEV) for n in (40, 300, 300))
    out = torch.empty_like(q)
    call = lambda x: miniattn.flash_attn_fwd(q, k, v, causal=True, out=out, **{"q_pos0": 260, name: x}).clone()  # noqa: E731
    held = torch.tensor(values[0])
    first = call(held)
    assert torch.equal(first, call(values[0]))
    held.fill_(values[1])
    again = call(held)
    assert torch.equal(again, call(values[1])) and not torch.equal(again, first)


@pytest.mark.gpu
def test_max_q():
    p = Paged([700, 90], [2, 60], 2, 64, BF16, 16, seed=74)
    q = torch.randn((62, 4, 64), generator=torch.Generator().manual_seed(75)).to(BF16).to(DEV)
    most = torch.tensor(60)
    call = lambda m: miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=p.cu_q, max_q=m)  # noqa: E731
    assert torch.equal(call(most), call(60))
    most.fill_(2)
    assert torch.equal(call(most), call(2))   # the other kernel: its sums are not the same bits
    assert not torch.equal(call(60), call(2))


@pytest.mark.parametrize("name", ["window", "sinks", "shared_len", "max_q", "q_pos0", "k_pos0"])
@pytest.mark.parametrize("value", [4.5, "4", torch.tensor(4.5)])
def test_what_is_no_whole_number(name, value):
    q = torch.zeros((1, 1, 2, 64), dtype=BF16)   # refused before anything is looked at
    ints = torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match=f"{name} must be a whole number"):
        if name in ("q_pos0", "k_pos0"):
            miniattn.flash_attn_fwd(q, q, q, causal=True, window=3, **{name: value})
        else:
            miniattn.paged_attention(q, q, q, ints[None], ints, **{name: value})


def test_whole_numbers_of_other_types():
    from miniattn.ops import _as_int
    others = (3, True, 3.0, np.int64(3), np.float32(3), torch.tensor(3), torch.tensor(3.0), torch.tensor([3]))
    assert [_as_int("n", x) for x in others] == [3, 1, 3, 3, 3, 3, 3, 3]
    for x in (float("nan"), float("inf"), None, 3j):
        with pytest.raises(RuntimeError, match="whole number"):
            _as_int("n", x)
