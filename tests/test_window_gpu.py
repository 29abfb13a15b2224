"""miniattn.flash_attn_fwd with a sliding window and sinks against the definition in 64 bits."""
import pytest
import torch

import miniattn
from paged_reference import attention, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def _tensors(B, Hq, Hkv, Nq, Nk, D, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn((B, n, h, D), generator=gen).to(dtype).to(DEV) for h, n in ((Hq, Nq), (Hkv, Nk), (Hkv, Nk))]


def _compare(q, k, v, window, sinks, q_pos0=0, k_pos0=0, layout="bnhd", scale=None):
    """q, k, v: (B,N,H,D)"""
    args = (q, k, v) if layout == "bnhd" else tuple(t.transpose(1, 2).contiguous() for t in (q, k, v))
    out, lse = miniattn.flash_attn_fwd(*args, causal=True, layout=layout, return_lse=True, q_pos0=q_pos0, k_pos0=k_pos0,
                                       window=window, sinks=sinks, softmax_scale=scale)
    assert out.shape == args[0].shape
    out = out if layout == "bnhd" else out.transpose(1, 2)
    for b in range(q.shape[0]):
        o, t, z, tz = attention(q[b], k[b], v[b], q_pos0 - k_pos0, window, max(0, sinks - k_pos0), scale)
        check(out[b], o, t, f"sequence {b}, window {window}, sinks {sinks}")
        check(lse[b], z, tz, f"lse of sequence {b}, window {window}, sinks {sinks}")
    miniattn.check_device_status(DEV)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 2), (64, 4), (127, 0), (128, 128), (129, 200), (300, 4), (10000, 4)])
@pytest.mark.parametrize("D,dtype,layout", [(64, F16, "bhnd"), (96, BF16, "bnhd"), (128, BF16, "bhnd")])
def test_prefill(D, dtype, layout, window, sinks):
    _compare(*_tensors(2, 6, 2, 515, 515, D, dtype, seed=window), window, sinks, layout=layout)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (7, 7), (12, 4), (20, 4), (64, 1), (129, 1)])
def test_heads(Hq, Hkv):
    _compare(*_tensors(1, Hq, Hkv, 300, 300, 64, BF16, seed=Hq), 100, 3)


@pytest.mark.parametrize("Nq,Nk", [(1, 1), (1, 777), (3, 4000), (65, 1300), (300, 2011), (128, 128), (257, 257)])
def test_last_rows_of_a_longer_context(Nq, Nk):
    _compare(*_tensors(2, 8, 2, Nq, Nk, 128, BF16, seed=Nq), 257, 4, q_pos0=Nk - Nq)


@pytest.mark.parametrize("q_pos0,k_pos0", [(0, 0), (100, 40), (1000, 0), (500, 600), (2 ** 33, 2 ** 33), (0, 5000)])
def test_positions(q_pos0, k_pos0):
    """Keys before the window, after the row, and rows that see none; sinks count positions, not keys."""
    _compare(*_tensors(1, 4, 2, 200, 333, 64, F16, seed=3), 50, 60, q_pos0=q_pos0, k_pos0=k_pos0)


def test_long():
    _compare(*_tensors(1, 2, 1, 9001, 9001, 128, BF16, seed=4), 1024, 4)


def test_wide_window_is_plain_causal():
    q, k, v = _tensors(2, 8, 2, 700, 700, 128, BF16, seed=5)
    _compare(q, k, v, 700, 0)
    _compare(q, k, v, 2 ** 31 - 1, 2 ** 31 - 1)


def test_poison_before_the_window():
    """Keys and values that slid out of every row's window hold NaN and infinities."""
    q, k, v = _tensors(2, 8, 2, 3, 2000, 128, BF16, seed=6)
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, 4:1708], bad_v[:, 4:1708] = float("nan"), float("inf")
    out = miniattn.flash_attn_fwd(q, bad_k, bad_v, causal=True, layout="bnhd", q_pos0=1997, window=290, sinks=4)
    for b in range(2):
        o, t, *_ = attention(q[b], k[b], v[b], 1997, 290, 4)
        check(out[b], o, t, f"sequence {b}")


def test_no_keys():
    q, k, v = _tensors(1, 4, 2, 5, 0, 64, BF16)
    out, lse = miniattn.flash_attn_fwd(q, k, v, causal=True, layout="bnhd", return_lse=True, window=4)
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())


def test_refusals():
    q, k, v = _tensors(1, 4, 2, 64, 64, 64, BF16)

    def refused(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            miniattn.flash_attn_fwd(q, k, v, layout="bnhd", **{"causal": True, **kw})

    refused("causal", causal=False, window=4)
    refused("window is None", sinks=4)
    refused("window", window=0)
    refused("window", window=2 ** 31)
    refused("sinks", window=4, sinks=-1)
    refused("kernel", window=4, kernel="simple")
    refused("carried state", window=4, carry_out=True, carry=miniattn.carry_state(q, "bnhd"))
