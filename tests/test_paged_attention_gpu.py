"""miniattn.paged_attention against the definition in 64 bits.  Places that no row sees hold NaN and infinities, pages that
nobody needs lie outside the cache (paged_reference.Paged)."""
import pytest
import torch

import miniattn
from paged_reference import Paged, check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


def _queries(news, Hq, D, dtype, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn((n, Hq, D), generator=gen).to(dtype) for n in news]


def _run(p, rows, ragged, **kw):
    """Output and lse by sequence: ((n,Hq,D), (Hq,n)) of each."""
    if ragged:
        q = torch.cat(rows).to(DEV)
        out, lse = miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=p.cu_q, window=p.window,
                                            sinks=p.sinks, return_lse=True, **kw)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.dtype == torch.float32
        return list(out.split(p.news)), list(lse.split(p.news, 1))
    q = torch.stack(rows).to(DEV)
    out, lse = miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, window=p.window, sinks=p.sinks,
                                        return_lse=True, **kw)
    assert out.shape == q.shape and lse.shape == (q.shape[0], q.shape[2], q.shape[1])
    return list(out), list(lse)


def _compare(p, rows, ragged, scale=None, **kw):
    outs, lses = _run(p, rows, ragged, softmax_scale=scale, **kw)
    for b, (o, l, *want) in enumerate(zip(outs, lses, *p.expected(rows, scale))):
        check(o, want[0], want[1], f"sequence {b} of {p.lens}, {p.news} new")
        check(l, want[2], want[3], f"lse of sequence {b} of {p.lens}, {p.news} new")
    miniattn.check_device_status(DEV)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_decode(D, page, dtype):
    """One token each; lengths of 0 and 1, at and beside tiles and pages, and long enough to be cut."""
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 128, 1000, 2049, 4000]
    p = Paged(lens, [1] * len(lens), 2, D, dtype, page, seed=page + D)
    _compare(p, _queries(p.news, 8, D, dtype), False)


@pytest.mark.parametrize("G", [1, 3, 5, 8, 16, 40])
@pytest.mark.parametrize("n", [1, 2, 7])
def test_heads_and_drafts(n, G):
    lens = [n, 3, 70, 1500, 0, 200]  # 3 < 7: the front of a padded sequence sees nothing
    p = Paged(lens, [n] * len(lens), 3, 128, BF16, 32, seed=G * 10 + n)
    _compare(p, _queries(p.news, 3 * G, 128, BF16), False)


@pytest.mark.parametrize("dtype,D,G,page", [(BF16, 128, 4, 32), (F16, 64, 1, 16), (BF16, 96, 3, 64), (F16, 128, 8, 256)])
def test_ragged(dtype, D, G, page):
    news = [1, 0, 300, 5, 0, 129, 64, 1]
    lens = [900, 0, 300, 5, 40, 1500, 1063, 1]
    p = Paged(lens, news, 2, D, dtype, page, seed=D + G)
    _compare(p, _queries(news, 2 * G, D, dtype), True)
    _compare(p, _queries(news, 2 * G, D, dtype), True, max_q=300)
    _compare(p, _queries(news, 2 * G, D, dtype), True, max_q=1)  # a hint, not a bound


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 4), (64, 0), (64, 64), (100, 70), (1000, 3), (5000, 4)])
@pytest.mark.parametrize("dtype,D,G,page", [(BF16, 128, 4, 16), (F16, 64, 2, 128)])
def test_window(dtype, D, G, page, window, sinks):
    news = [1, 1, 3, 200, 1, 0, 130]
    lens = [4000, 60, 1203, 1500, 1, 0, 131]
    p = Paged(lens, news, 2, D, dtype, page, window=window, sinks=sinks, seed=window)
    _compare(p, _queries(news, 2 * G, D, dtype), True)


@pytest.mark.parametrize("window,sinks", [(1, 2), (100, 4), (1024, 0)])
@pytest.mark.parametrize("n", [1, 4])
def test_window_decode(n, window, sinks):
    lens = [n, 99, 100, 101, 1500, 3000, 0, 164]
    p = Paged(lens, [n] * len(lens), 2, 128, BF16, 16, window=window, sinks=sinks, seed=window)
    _compare(p, _queries(p.news, 8, 128, BF16), False)


@pytest.mark.parametrize("n,shared,page,D,dtype", [(1, 64, 16, 128, BF16), (1, 1024, 64, 128, F16), (4, 1008, 16, 64, F16),
                                                   (1, 4096, 128, 96, BF16), (3, 16, 16, 128, BF16)])
def test_shared_prefix(n, shared, page, D, dtype):
    lens = [shared + n + x for x in (0, 1, 30, 65, 300, 1000)] + [0, shared + n, n]
    p = Paged(lens, [n] * len(lens), 2, D, dtype, page, shared=shared, seed=shared)
    _compare(p, _queries(p.news, 8, D, dtype), False, shared_len=shared)


@pytest.mark.parametrize("dtype,D,n,Hkv,G", [(BF16, 128, 1, 8, 4), (F16, 64, 4, 16, 4), (BF16, 96, 2, 8, 3), (BF16, 128, 2, 2, 40)])
def test_shared_prefix_of_a_batch(dtype, D, n, Hkv, G):
    """Enough to be read in a launch of its own: 48 sequences, the first of them padding with nothing in its block table, some
    shorter than the prefix."""
    shared = 1024
    lens = [0, n, 700, 1] + [shared + n + 29 * i for i in range(44)]
    p = Paged(lens, [n] * len(lens), Hkv, D, dtype, 32, shared=shared, seed=D)
    _compare(p, _queries(p.news, Hkv * G, D, dtype), False, shared_len=shared)


def test_shared_prefix_longer_than_every_sequence():
    lens = [0] + [900 - i for i in range(63)]
    p = Paged(lens, [1] * 64, 8, 128, BF16, 16, shared=2048, seed=8)
    table = torch.full((64, 200), 10 ** 6, dtype=torch.int32, device=DEV)  # nothing past the sequences' ends
    table[:, :p.table.shape[1]] = p.table
    p.table = table
    _compare(p, _queries(p.news, 32, 128, BF16), False, shared_len=2048)


def test_shared_prefix_ragged_batch():
    """Ragged rows behind a prefix of a launch of its own, rows behind the last sequence, an empty sequence."""
    shared = 2048
    news = [1, 0, 4, 3, 2, 1, 4, 1] * 6
    lens = [shared + 40 * i + m for i, m in enumerate(news)]
    p = Paged(lens, news, 8, 128, BF16, 64, shared=shared, seed=9)
    rows = _queries(news, 32, 128, BF16)
    q = torch.cat(rows + [torch.full((5, 32, 128), float("nan"), dtype=BF16)]).to(DEV)
    out = torch.full_like(q, 5.0)
    _, lse = miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=p.cu_q, max_q=4, shared_len=shared,
                                      out=out, return_lse=True)
    T = sum(news)
    for b, (o, t, z, tz) in enumerate(zip(*p.expected(rows))):
        check(out[:T].split(news)[b], o, t, f"sequence {b}")
        check(lse[:, :T].split(news, 1)[b], z, tz, f"lse of sequence {b}")
    assert bool((out[T:] == 5).all())
    miniattn.check_device_status(DEV)


def test_shared_prefix_ragged():
    shared = 512
    news = [1, 0, 200, 3, 65, 1]
    lens = [shared + x for x in (1, 0, 200, 500, 66, 2000)]
    p = Paged(lens, news, 2, 128, BF16, 32, shared=shared, seed=5)
    _compare(p, _queries(news, 8, 128, BF16), True, shared_len=shared, max_q=200)


def test_one_sequence_few_heads_long():
    p = Paged([30011], [1], 1, 128, BF16, 64, seed=2)
    _compare(p, _queries([1], 8, 128, BF16), False)


def test_many_sequences():
    lens = [(i * 37) % 300 for i in range(700)]
    p = Paged(lens, [1] * 700, 1, 64, F16, 16, seed=3)
    _compare(p, _queries([1] * 700, 4, 64, F16), False)


def test_scale_and_large_scores():
    """Scores far apart, the largest last: the running maximum moves by hundreds."""
    p = Paged([700, 65], [2, 2], 1, 64, F16, 16, seed=4)
    rows = [8.0 * q for q in _queries([2, 2], 2, 64, F16)]
    _compare(p, rows, False, scale=1.0)


def test_cache_layouts_and_strides():
    """Pages laid out (pages, heads, tokens, D), a block table and queries that are views of wider tensors, an output view."""
    lens, news = [70, 1, 333], [2, 2, 2]
    p = Paged(lens, news, 2, 128, BF16, 16, seed=6, heads_first=True)
    rows = _queries([2] * 3, 8, 128, BF16)
    wide = torch.full((3, p.table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, :p.table.shape[1]] = p.table
    fused = torch.zeros((3, 2, 12, 128), dtype=BF16, device=DEV)
    fused[:, :, 2:10] = torch.stack(rows).to(DEV)
    out = torch.full((3, 2, 9, 128), 7.0, dtype=BF16, device=DEV)
    got = miniattn.paged_attention(fused[:, :, 2:10], p.k_cache, p.v_cache, wide[:, :p.table.shape[1]], p.seq_lens,
                                   out=out[:, :, :8])
    for b, (o, t, *_) in enumerate(zip(*p.expected(rows))):
        check(got[b], o, t, f"sequence {b}")
    assert bool((out[:, :, 8] == 7).all())


@pytest.mark.parametrize("lens,n,G,shared", [([3000, 1700], 1, 4, 0), ([3000, 1700], 40, 4, 0), ([900, 700], 200, 1, 0),
                                             ([1100 + 17 * i for i in range(48)], 1, 8, 1024)])
def test_result_in_place_of_the_queries(lens, n, G, shared):
    p = Paged(lens, [n] * len(lens), 4, 128, BF16, 32, seed=31, shared=shared)
    rows = _queries(p.news, 4 * G, 128, BF16)
    q = torch.stack(rows).to(DEV)
    assert miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, shared_len=shared, out=q) is q
    for b, (o, t, *_) in enumerate(zip(*p.expected(rows))):
        check(q[b], o, t, f"sequence {b}")


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("lens,n,Hkv,G,D,window", [
    ([1300, 900], 128, 2, 4, 128, None),    # Q tiles one by one
    ([1100], 513, 4, 1, 64, None),          # an odd number of them
    ([700, 2, 300], 150, 1, 3, 96, 40),     # the front of a sequence missing
    ([3000, 2500], 100, 2, 4, 128, None),   # pairs, cut along the keys
    ([640] * 10, 130, 2, 8, 64, 100),       # pairs
    ([500] * 9, 260, 7, 1, 128, 300)])      # pairs, the last wave's one by one
def test_chunks(lens, n, Hkv, G, D, window, ragged):
    p = Paged(lens, [n] * len(lens), Hkv, D, BF16, 32, window=window, sinks=3 if window else 0, seed=41)
    _compare(p, _queries(p.news, Hkv * G, D, BF16), ragged)


@pytest.mark.parametrize("n,G,D", [(1, 129, 64), (3, 129, 128), (20, 129, 128), (2, 200, 96)])
def test_more_heads_than_a_tile_has_rows(n, G, D):
    p = Paged([700, 41, 5], [n, n, n], 1, D, F16, 16, seed=32)
    rows = _queries(p.news, G, D, F16)
    out = miniattn.paged_attention(torch.stack(rows).to(DEV), p.k_cache, p.v_cache, p.table, p.seq_lens)
    for b, (o, t, *_) in enumerate(zip(*p.expected(rows))):
        check(out[b], o, t, f"sequence {b}")


@pytest.mark.parametrize("most", [1, 5, 4000])
def test_max_q_picks_the_kernel_alone(most):
    """Also where it is not what it says it is."""
    p = Paged([900, 1300, 64, 2000], [70, 1, 0, 300], 2, 64, BF16, 32, seed=33)
    rows = _queries(p.news, 8, 64, BF16)
    out, lse = miniattn.paged_attention(torch.cat(rows).to(DEV), p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=p.cu_q,
                                        max_q=most, return_lse=True)
    at = 0
    for b, (o, t, z, tz) in enumerate(zip(*p.expected(rows))):
        check(out[at:at + p.news[b]], o, t, f"sequence {b}")
        check(lse[:, at:at + p.news[b]], z, tz, f"lse of sequence {b}")
        at += p.news[b]


@pytest.mark.parametrize("n", [1, 33])
def test_queries_shared_by_the_batch(n):
    """One sequence's queries expanded over the batch, a stride of 0."""
    p = Paged([700, 300, 64], [n] * 3, 2, 128, BF16, 16, seed=34)
    rows = _queries([n], 8, 128, BF16) * 3
    q = rows[0].to(DEV).expand(3, n, 8, 128)
    out = torch.empty((3, n, 8, 128), dtype=BF16, device=DEV)
    miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, out=out)
    for b, (o, t, *_) in enumerate(zip(*p.expected(rows))):
        check(out[b], o, t, f"sequence {b}")


def test_rows_behind_the_last_sequence_stay():
    p = Paged([40, 300], [3, 100], 2, 64, BF16, 16, seed=7)
    rows = _queries([3, 100], 4, 64, BF16)
    q = torch.full((150, 4, 64), float("nan"), dtype=BF16, device=DEV)
    q[:103] = torch.cat(rows).to(DEV)
    out = torch.full_like(q, 5.0)
    miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=p.cu_q, out=out)
    for b, (o, t, *_) in enumerate(zip(*p.expected(rows))):
        check(out[:103].split([3, 100])[b], o, t, f"sequence {b}")
    assert bool((out[103:] == 5).all())


@pytest.mark.parametrize("n", [1, 100])
def test_same_bits_again(n):
    """Cut items are folded in one order whoever finishes last."""
    lens = [3000, 17, 5000, 900]
    p = Paged(lens, [n] * 4, 2, 128, BF16, 32, seed=8)
    q = torch.stack(_queries([n] * 4, 8, 128, BF16)).to(DEV)
    call = lambda: miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, return_lse=True)  # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(side):
            torch.randn(1 << 22, device=DEV)
        again = call()
        assert all(torch.equal(x, y) for x, y in zip(first, again))


@pytest.mark.parametrize("lens,n,G,shared", [([3000, 1700], 1, 4, 0), ([3000, 1700], 40, 4, 0),
                                             ([1100 + 17 * i for i in range(48)], 1, 8, 1024)])
def test_two_streams(lens, n, G, shared):
    p = Paged(lens, [n] * len(lens), 4, 128, BF16, 32, seed=9, shared=shared)
    rows = _queries(p.news, 4 * G, 128, BF16)
    q = torch.stack(rows).to(DEV)
    want = list(zip(*p.expected(rows)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, shared_len=shared))
    torch.cuda.synchronize()
    assert all(torch.equal(out, outs[0]) for out in outs)
    for b, (o, t, *_) in enumerate(want):
        check(outs[0][b], o, t, f"sequence {b}")


def test_bad_lengths_and_pages_are_reported():
    """A sequence with a page outside the cache, or longer than the block table, and one with bad row numbers: the status word
    says so, the other sequences are right.  Nothing outside the tensors is touched: the kernels look before they read."""
    lens, news = [100, 200, 64, 50], [1, 1, 1, 1]
    p = Paged(lens, news, 2, 64, BF16, 16, seed=10)
    rows = _queries(news, 4, 64, BF16)
    q = torch.stack(rows).to(DEV)
    want = list(zip(*p.expected(rows)))
    for spoil in ("page", "length", "negative"):
        table, seq_lens = p.table.clone(), p.seq_lens.clone()
        if spoil == "page":
            table[1, 3] = p.k_cache.shape[0]
        else:
            seq_lens[1] = 10 ** 9 if spoil == "length" else -5
        out = miniattn.paged_attention(q, p.k_cache, p.v_cache, table, seq_lens)
        with pytest.raises(RuntimeError, match="outside its tensors"):
            miniattn.check_device_status(DEV)
        for b in (0, 2, 3):
            check(out[b], want[b][0], want[b][1], f"sequence {b} beside a bad {spoil}")
    flat, cu = q.view(4, 4, 64), torch.tensor([0, 1, 99, 99, 99], dtype=torch.int32, device=DEV)
    miniattn.paged_attention(flat, p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=cu)
    with pytest.raises(RuntimeError, match="outside its tensors"):
        miniattn.check_device_status(DEV)


def test_captured_call_serves_longer_contexts():
    """One graph, replayed while the lengths in its tensors change; a second graph and eager calls beside it."""
    steps = [[5, 200, 0], [6, 1000, 1], [64, 4000, 33]]
    graphs = []
    for seed in (11, 12):
        whole = Paged(steps[-1], [1, 1, 1], 2, 128, BF16, 16, seed=seed)
        q = torch.zeros((3, 1, 8, 128), dtype=BF16, device=DEV)
        lens = whole.seq_lens.clone()
        miniattn.paged_attention(q, whole.k_cache, whole.v_cache, whole.table, lens)  # sizes its scratch
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = miniattn.paged_attention(q, whole.k_cache, whole.v_cache, whole.table, lens)
        graphs.append((g, whole, q, lens, out))
    for k, step in enumerate(steps):
        for g, whole, q, lens, out in graphs:
            rows = _queries([1, 1, 1], 8, 128, BF16, seed=k)
            q.copy_(torch.stack(rows))
            lens.copy_(torch.tensor(step, dtype=torch.int32))
            g.replay()
            eager = miniattn.paged_attention(q, whole.k_cache, whole.v_cache, whole.table, lens)
            torch.cuda.synchronize()
            assert torch.equal(eager, out)
            for b in range(3):
                from paged_reference import attention
                o, t, *_ = attention(rows[b].to(DEV), whole.k[b][:step[b]].to(DEV), whole.v[b][:step[b]].to(DEV), step[b] - 1)
                check(out[b], o, t, f"step {k}, sequence {b}")
    miniattn.check_device_status(DEV)


@pytest.mark.parametrize("lens,n,G,shared", [([3000, 1700], 1, 4, 0), ([3000, 2900], 40, 4, 0),
                                             ([1100 + 17 * i for i in range(48)], 1, 8, 1024)])
def test_two_graphs_at_once(lens, n, G, shared):
    """Captured calls share no scratch: replayed on two streams, with an eager call beside them, they give what they give alone."""
    p = Paged(lens, [n] * len(lens), 4, 128, BF16, 32, seed=9, shared=shared)
    q = torch.stack(_queries(p.news, 4 * G, 128, BF16)).to(DEV)
    call = lambda: miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, shared_len=shared)
    want = call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = [call() for _ in range(4)]
        graphs.append((g, out, torch.cuda.Stream()))
    for _ in range(5):
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
        eager = [call() for _ in range(4)]
    torch.cuda.synchronize()
    for out in (graphs[0][1], graphs[1][1], eager):
        assert all(torch.equal(o, want) for o in out)


def test_captured_ragged_call_serves_other_batches():
    """One graph of a ragged call, replayed for batches of other rows and lengths (its grid knows the sizes of q alone)."""
    from paged_reference import attention
    whole = Paged([1500, 900, 2100, 64], [1, 1, 1, 1], 2, 128, BF16, 16, seed=21)
    for b in range(4):  # every token of every sequence is there
        for j in range(whole.lens[b]):
            if int(whole.table[b, j // 16]) < whole.k_cache.shape[0]:
                whole.k_cache[int(whole.table[b, j // 16]), j % 16] = whole.k[b][j].to(DEV)
                whole.v_cache[int(whole.table[b, j // 16]), j % 16] = whole.v[b][j].to(DEV)
    q = torch.zeros((300, 8, 128), dtype=BF16, device=DEV)
    lens, cu = whole.seq_lens.clone(), torch.tensor([0, 1, 2, 3, 300], dtype=torch.int32, device=DEV)
    miniattn.paged_attention(q, whole.k_cache, whole.v_cache, whole.table, lens, cu_q=cu)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = miniattn.paged_attention(q, whole.k_cache, whole.v_cache, whole.table, lens, cu_q=cu, return_lse=True)
    for k, (news, now) in enumerate([([100, 0, 200, 0], [1500, 10, 2100, 0]), ([1, 290, 1, 8], [700, 900, 1, 64]),
                                     ([0, 0, 0, 60], [0, 0, 0, 64]), ([75, 75, 75, 64], [75, 900, 80, 64])]):
        rows = _queries(news, 8, 128, BF16, seed=k)
        q[:sum(news)] = torch.cat(rows).to(DEV)
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        cu.copy_(torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=torch.int32))
        g.replay()
        at = 0
        for b, n in enumerate(news):
            o, t, z, tz = attention(rows[b].to(DEV), whole.k[b][:now[b]].to(DEV), whole.v[b][:now[b]].to(DEV), now[b] - n)
            check(out[at:at + n], o, t, f"batch {k}, sequence {b}")
            check(lse[:, at:at + n], z, tz, f"lse of batch {k}, sequence {b}")
            at += n
    miniattn.check_device_status(DEV)


def test_row_numbers_that_fall_do_no_lasting_harm():
    """Overlapping rows (cu_q falls) are reported; the calls after it are right."""
    p = Paged([900, 900, 900, 900], [200, 200, 0, 0], 2, 128, BF16, 16, seed=22)
    rows = _queries([200, 200], 8, 128, BF16)
    q = torch.cat(rows).to(DEV)
    bad = torch.tensor([0, 400, 0, 400, 0], dtype=torch.int32, device=DEV)
    for _ in range(3):
        miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=bad)
        out = miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, cu_q=p.cu_q)
        for b, (o, t, *_) in enumerate(list(zip(*p.expected(rows + _queries([0, 0], 8, 128, BF16))))[:2]):
            check(out.split(200)[b], o, t, f"sequence {b}")
    with pytest.raises(RuntimeError, match="outside its tensors"):
        miniattn.check_device_status(DEV)


def test_far_into_a_large_cache():
    """Offsets past 2^31 elements: the last pages of a cache of 2.2e9 elements."""
    page, Hkv, D = 64, 8, 128
    n_pages = (1 << 31) // (page * Hkv * D) + 40
    k_cache, v_cache = (torch.zeros((n_pages, page, Hkv, D), dtype=BF16, device=DEV) for _ in range(2))
    small = Paged([1000], [2], Hkv, D, BF16, page, seed=13)
    k_cache[-small.k_cache.shape[0]:], v_cache[-small.v_cache.shape[0]:] = small.k_cache, small.v_cache
    table = torch.where((small.table >= 0) & (small.table < small.k_cache.shape[0]),
                        small.table + (n_pages - small.k_cache.shape[0]), small.table)
    rows = _queries([2], 16, D, BF16)
    out = miniattn.paged_attention(torch.stack(rows).to(DEV), k_cache, v_cache, table, small.seq_lens)
    o, t, *_ = (x[0] for x in small.expected(rows))
    check(out[0], o, t, "far pages")


def test_refusals():
    p = Paged([100], [1], 2, 64, BF16, 16, seed=14)
    q = torch.zeros((1, 1, 4, 64), dtype=BF16, device=DEV)
    args = [q, p.k_cache, p.v_cache, p.table, p.seq_lens]

    def refused(match, *a, **kw):
        with pytest.raises(RuntimeError, match=match):
            miniattn.paged_attention(*a, **kw)

    refused("CUDA tensor", q.cpu(), *args[1:])
    refused("data type", q.half(), *args[1:])
    refused("fp16 and bf16", q.float(), *args[1:])
    refused("multiple of KV heads", q[:, :, :3], *args[1:])
    refused("head dim", torch.zeros((1, 1, 4, 128), dtype=BF16, device=DEV), *args[1:])
    refused("same shape", q, p.k_cache, p.v_cache[:-1], *args[3:])
    refused("int32", *args[:3], p.table.long(), p.seq_lens)
    refused("shape", *args[:4], torch.zeros(2, dtype=torch.int32, device=DEV))
    refused("must be 3-D", *args, cu_q=torch.zeros(2, dtype=torch.int32, device=DEV))
    refused("must be 4-D", q[0], *args[1:])
    refused("sinks", *args, sinks=4)
    refused("window", *args, window=0)
    refused("do not go together", *args, window=8, shared_len=16)
    refused("multiple of the page size", *args, shared_len=8)
    refused("inside the block table", *args, shared_len=16 * 1000)
    refused("between", *args, shared_len=2 ** 32 + 16)
    refused("page size", q, p.k_cache[:, :8], p.v_cache[:, :8], *args[3:])
    refused("multiple of 8", q, *(torch.zeros((4, 16, 2, 68), dtype=BF16, device=DEV)[..., :64] for _ in range(2)), *args[3:])
    refused("match q", *args, out=torch.zeros((1, 2, 4, 64), dtype=BF16, device=DEV))
    refused("max_q", q[0], *args[1:], cu_q=torch.zeros(2, dtype=torch.int32, device=DEV), max_q=0)


def test_nothing_to_do():
    p = Paged([0, 0], [0, 0], 2, 64, BF16, 16, seed=15)
    out = miniattn.paged_attention(torch.zeros((0, 4, 64), dtype=BF16, device=DEV), p.k_cache, p.v_cache, p.table, p.seq_lens,
                                   cu_q=p.cu_q)
    assert out.shape == (0, 4, 64)
    none = torch.zeros((0, 16, 2, 64), dtype=BF16, device=DEV)
    q = torch.ones((2, 1, 4, 64), dtype=BF16, device=DEV)
    out, lse = miniattn.paged_attention(q, none, none, p.table[:, :0], p.seq_lens, return_lse=True)  # no pages at all
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())
    miniattn.check_device_status(DEV)
