"""Host threads that call at the same time on one stream.  A call behind a shared prefix is three launches that hand results on
through scratch: those of another thread must not come between them in the same scratch."""
import sys
import threading
import time
import types

import pytest
import torch

from miniattn import ops


def _in_threads(jobs):
    errors = []

    def run(job):
        try:
            job()
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=run, args=(job,)) for job in jobs]
    every = sys.getswitchinterval()
    sys.setswitchinterval(1e-5)
    try:
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(every)
    if errors:
        raise errors[0]


def test_launches_of_a_call_stay_together(monkeypatch):
    """The entry point stood in for by one that takes its time: as ctypes does, it lets other threads run meanwhile."""
    zeros = torch.zeros
    inside, seen, overlaps = {}, {True: set(), False: set()}, []

    def entry(block, scratch, nbytes, stream):
        several, n = block[:1] == b"s", inside.get(scratch, 0)
        seen[several].add(scratch)
        inside[scratch] = n + 1
        if n and several:
            overlaps.append(scratch)
        time.sleep(0.002)
        if several and inside[scratch] != 1:
            overlaps.append(scratch)
        inside[scratch] -= 1
        return 0
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **kw: zeros(*a, **kw))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(ops, "_balance_scratch", {})
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(ops, "_current_raw_stream", lambda index: 7)
    monkeypatch.setattr(ops._lib, "lib", types.SimpleNamespace(miniattn_fwd_cache=entry))
    device = types.SimpleNamespace(index=0)
    _in_threads([lambda s=s: [ops._launch_cache(b"s" if s else b"-", 1000, device, s) for _ in range(20)]
                 for s in (True, True, True, False)])
    assert not overlaps and seen[True] and seen[False]
    assert not seen[True] & seen[False]   # single launches of other threads may come between


@pytest.mark.gpu
def test_two_threads_behind_a_prefix():
    import miniattn
    from paged_reference import Paged, check
    dev = "cuda:0"
    jobs, batches = [], []
    for seed in (81, 82):
        p = Paged([1100 + 17 * i for i in range(48)], [1] * 48, 4, 128, torch.bfloat16, 32, seed=seed, shared=1024)
        rows = list(torch.randn((48, 1, 32, 128), generator=torch.Generator().manual_seed(seed + 10)).bfloat16())
        batches.append((p, rows, torch.stack(rows).to(dev), []))
    for p, rows, q, outs in batches:
        call = lambda p=p, q=q: miniattn.paged_attention(q, p.k_cache, p.v_cache, p.table, p.seq_lens, shared_len=1024)  # noqa: E731
        outs.append(call())
        jobs.append(lambda call=call, outs=outs: [outs.append(call()) for _ in range(100)])
    plain = lambda: [miniattn.paged_attention(batches[0][2], *plain_args) for _ in range(100)]  # noqa: E731
    p = batches[0][0]
    plain_args = (p.k_cache, p.v_cache, p.table, p.seq_lens)
    _in_threads(jobs + [plain])
    torch.cuda.synchronize()
    for p, rows, _, outs in batches:
        for b, (o, t, *_) in enumerate(zip(*p.expected(rows))):
            check(outs[0][b], o, t, f"sequence {b}")
        assert len(outs) == 101 and all(torch.equal(o, outs[0]) for o in outs)
    miniattn.check_device_status(dev)
