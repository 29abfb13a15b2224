"""miniattn.paged_append against the definition in 64 bits; what it does not write stays as it was, bit for bit."""
import pytest
import torch

import miniattn
from paged_reference import check, rotate

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def _setup(lens, page, Hkv, D, dtype, seed=0, heads_first=False):
    gen = torch.Generator().manual_seed(seed)
    width = max(1, (max(lens) + page - 1) // page) + 1
    n_pages = len(lens) * width + 2
    shape = (n_pages, Hkv, page, D) if heads_first else (n_pages, page, Hkv, D)
    caches = [torch.randn(shape, generator=gen).to(dtype).to(DEV) for _ in range(2)]
    if heads_first:
        caches = [c.transpose(1, 2) for c in caches]
    table = torch.randperm(n_pages, generator=gen)[:len(lens) * width].view(len(lens), width).to(torch.int32).to(DEV)
    return caches, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def _new(news, Hq, Hkv, D, dtype, seed=1):
    gen = torch.Generator().manual_seed(seed)
    kv = torch.randn((sum(news), 2, Hkv, D), generator=gen).to(dtype).to(DEV)
    q = torch.randn((sum(news), Hq, D), generator=gen).to(dtype).to(DEV)
    return kv[:, 0], kv[:, 1], q


def _compare(lens, news, page, Hq, Hkv, D, dtype, rot=None, interleaved=False, ragged=True, heads_first=False, with_q=True):
    caches, table, seq_lens = _setup(lens, page, Hkv, D, dtype, heads_first=heads_first)
    k, v, q = _new(news, Hq, Hkv, D, dtype)
    rope = miniattn.rope_table(max(lens) + 1, rot, device=DEV) if rot else None
    want_k, want_v = (c.clone().double() for c in caches)
    tol_k = torch.zeros_like(want_k)
    want_q, tol_q = q.double().clone(), torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    at = 0
    for b, (length, n) in enumerate(zip(lens, news)):
        for i in range(n):
            pos = length - n + i
            if pos < 0:
                continue
            page_no, slot = int(table[b, pos // page]), pos % page
            want_v[page_no, slot] = v[at + i].double()
            want_k[page_no, slot] = k[at + i].double()
            if rot:
                where = torch.tensor([pos], device=DEV)
                y, t = rotate(k[at + i][None], rope, where, interleaved)
                want_k[page_no, slot], tol_k[page_no, slot] = y[0], t[0]
                y, t = rotate(q[at + i][None], rope, where, interleaved)
                want_q[at + i], tol_q[at + i] = y[0], t[0]
        at += n
    cu = torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=torch.int32, device=DEV) if ragged else None
    args = [t if ragged else t.reshape(len(lens), news[0], *t.shape[1:]) for t in (k, v, q)]
    if not ragged:  # views, as a projection gives them
        args = [t.unflatten(0, (len(lens), news[0])) for t in (k, v, q)]
    q_new = miniattn.paged_append(args[0], args[1], *caches, table, seq_lens, cu_q=cu, q=args[2] if with_q else None, rope=rope,
                                  interleaved=interleaved)
    check(caches[0], want_k, tol_k, "k_cache")
    check(caches[1], want_v, torch.zeros_like(want_v), "v_cache")
    if with_q:
        assert q_new.shape == args[2].shape and q_new.data_ptr() != args[2].data_ptr()
        check(q_new.reshape(q.shape), want_q, tol_q, "q")
    else:
        assert q_new is None
    miniattn.check_device_status(DEV)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 16), (96, 96), (96, 32), (128, 128), (128, 48), (128, None)])
def test_ragged(D, rot, interleaved, dtype):
    _compare([5, 0, 130, 64, 17, 1, 100], [5, 0, 33, 1, 4, 1, 0], 16, 6, 2, D, dtype, rot, interleaved)


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_equal(n, page):
    lens = [n, 70, 2, 1000, 0, 65]  # shorter than n: the front of a padded sequence is left out
    _compare(lens, [n] * 6, page, 32, 8, 128, BF16, 128, ragged=False)
    _compare(lens, [n] * 6, page, 5, 5, 64, F16, 32, True, ragged=False, heads_first=True, with_q=False)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 1), (40, 8), (128, 1), (7, 7)])
def test_heads(Hq, Hkv):
    _compare([300, 20], [200, 3], 32, Hq, Hkv, 128, F16, 128)


def test_many_sequences():
    lens = [(i * 13) % 90 for i in range(300)]
    _compare(lens, [min(x, i % 3) for i, x in enumerate(lens)], 16, 2, 1, 64, BF16, 64)


def test_in_place_and_rows_behind():
    caches, table, seq_lens = _setup([9, 30], 16, 2, 64, BF16)
    k, v, q = _new([40], 4, 2, 64, BF16)
    cu = torch.tensor([0, 3, 20], dtype=torch.int32, device=DEV)
    rope = miniattn.rope_table(64, 64, device=DEV)
    apart = torch.full_like(q, 3.0)
    assert miniattn.paged_append(k, v, *caches, table, seq_lens, cu_q=cu, q=q, q_out=apart, rope=rope) is apart
    behind = q[20:].clone()
    assert miniattn.paged_append(k, v, *caches, table, seq_lens, cu_q=cu, q=q, q_out=q, rope=rope) is q
    assert torch.equal(q[:20], apart[:20]) and torch.equal(q[20:], behind) and bool((apart[20:] == 3).all())


def test_rows_in_front_of_the_first_sequence():
    """They belong to no sequence: nothing of the cache is written for them, their queries stay."""
    rope = miniattn.rope_table(64, 64, device=DEV)
    k, v, q = _new([12], 4, 2, 64, BF16)
    got = []
    for skip in (0, 5):
        caches, table, seq_lens = _setup([9, 30], 16, 2, 64, BF16)
        cu = torch.tensor([5 - skip, 8 - skip, 12 - skip], dtype=torch.int32, device=DEV)
        out = torch.full_like(q[skip:], 3.0)
        miniattn.paged_append(k[skip:], v[skip:], *caches, table, seq_lens, cu_q=cu, q=q[skip:], q_out=out, rope=rope)
        got.append((*caches, out[5 - skip:]))
        assert bool((out[:5 - skip] == 3).all())
    assert all(torch.equal(x, y) for x, y in zip(*got))
    miniattn.check_device_status(DEV)


@pytest.mark.parametrize("cu,lens", [([-2, 4, 8], [9, 30]), ([0, 4, 40], [9, 30]), ([0, 6, 2], [9, 30]), ([0, 4, 8], [9, -1])])
def test_bad_rows_and_negative_lengths_are_reported(cu, lens):
    caches, table, _ = _setup([9, 30], 16, 2, 64, BF16)
    k, v, q = _new([8], 4, 2, 64, BF16)
    cu, lens = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (cu, lens))
    miniattn.paged_append(k, v, *caches, table, lens, cu_q=cu, q=q)
    with pytest.raises(RuntimeError, match="outside its tensors"):
        miniattn.check_device_status(DEV)


def test_far_positions():
    """A table made in 64 bits: position 10^6 is rotated as exactly as position 0."""
    rope = miniattn.rope_table(1_000_001, 128, theta=500.0, device=DEV)
    i = torch.arange(64, dtype=torch.float64)
    angle = 1e6 * 500.0 ** (-i / 64)
    want = torch.cat([angle.cos(), angle.sin()])
    # the angle itself is off by up to 2^-53 of 10^6 and its power's error, the table by half a step
    assert float((rope[-1].cpu().double() - want).abs().max()) < 2.0 ** -24 + 1e-8
    caches, table, seq_lens = _setup([1_000_001], 1024, 1, 128, BF16)
    k, v, q = _new([1], 2, 1, 128, BF16)
    got = miniattn.paged_append(k[None], v[None], *caches, table, seq_lens, q=q[None], rope=rope)
    y, t = rotate(q, rope, torch.tensor([1_000_000], device=DEV), False)
    check(got[0], y, t, "q")


def test_bad_pages_lengths_and_positions_are_reported():
    """The tokens concerned are left out, every other place keeps its bits."""
    rope = miniattn.rope_table(40, 64, device=DEV)
    for spoil in ("page", "length", "rotation"):
        caches, table, seq_lens = _setup([20, 30, 33], 16, 2, 64, BF16)
        k, v, q = _new([2, 2, 2], 4, 2, 64, BF16)
        k, v, q = (t.unflatten(0, (3, 2)) for t in (k, v, q))
        good = [c.clone() for c in caches]
        miniattn.paged_append(k, v, *good, table, seq_lens, rope=rope)
        if spoil == "page":
            table[1, 1] = -1
        else:
            seq_lens[1] = 10 ** 9 if spoil == "length" else 45
        before = [c.clone() for c in caches]
        miniattn.paged_append(k, v, *caches, table, seq_lens, rope=rope)
        with pytest.raises(RuntimeError, match="outside its tensors"):
            miniattn.check_device_status(DEV)
        for c, g, was in zip(caches, good, before):
            for b, length in ((0, 20), (2, 33)):
                for pos in (length - 2, length - 1):
                    page_no = int(table[b, pos // 16])
                    assert torch.equal(c[page_no, pos % 16], g[page_no, pos % 16])
                    was[page_no, pos % 16] = c[page_no, pos % 16]
            assert torch.equal(c, was)


def test_refusals():
    caches, table, seq_lens = _setup([20], 16, 2, 64, BF16)
    k, v, q = (t[None] for t in _new([1], 4, 2, 64, BF16))
    args = [k, v, *caches, table, seq_lens]

    def refused(match, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            miniattn.paged_append(*a, **kw)

    refused("CUDA tensor", k.cpu(), *args[1:])
    refused("data type", k, v.half(), *args[2:])
    refused("same shape", k, v[:, :, :1], *args[2:])
    refused("heads", k[:, :, :1], v[:, :, :1], *args[2:])
    refused("q_out without q", *args, q_out=q)
    refused("tokens and head dim", *args, q=q[:, :0])
    refused("fp32", *args, rope=torch.zeros((40, 64), dtype=torch.float64, device=DEV))
    refused("multiple of 16", *args, rope=torch.zeros((40, 24), device=DEV))
    refused("multiple of 16", *args, rope=torch.zeros((40, 80), device=DEV))
    refused("must be 3-D", *args, cu_q=torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="even"):
        miniattn.rope_table(4, 5)


def test_nothing_to_do():
    caches, table, seq_lens = _setup([0], 16, 2, 64, BF16)
    was = [c.clone() for c in caches]
    k, v, q = _new([0], 4, 2, 64, BF16)
    out = miniattn.paged_append(k, v, *caches, table, seq_lens, cu_q=torch.zeros(2, dtype=torch.int32, device=DEV), q=q)
    assert out.shape == q.shape and all(torch.equal(c, w) for c, w in zip(caches, was))
