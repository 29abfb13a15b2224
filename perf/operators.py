"""The serving operators: what a program that keeps its keys and values in pages calls, and what that is measured by.

A case is a dict of plain values.  ``op`` names the public entry point:

* ``append``  ``miniattn.paged_append``: keys and values of new tokens rotated by their positions and written into the
  pages of their sequences, the queries rotated on the way
* ``attend``  ``miniattn.paged_attention``: attention of the new tokens over the pages, with a sliding window and sinks
  where ``window`` is set, and with the first ``shared`` tokens of all sequences held once
* ``window``  ``miniattn.flash_attn_fwd`` with a sliding window and sinks over contiguous keys and values

Sequence i of a paged case has ``shared + ctx_i + new_i`` tokens, ``new_i`` of them new; both numbers are spread over the
logarithm of their ranges by ``mix`` alone.  Without a window, or in its reach, every page is there; pages that slid out of
the window were given back, and their entries in the block table are -1, as are those past a sequence's end.
"""
import math
import os
import random
import sys

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _paged(name, op, B, Hq, Hkv, D, dtype, page, new, ctx, window=0, sinks=0, shared=0, lse=False, rot=0, inter=False,
           mix=1):
    c = {"op": op, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype, "page": page, "new_lo": new[0], "new_hi": new[1],
         "ctx_lo": ctx[0], "ctx_hi": ctx[1], "window": window, "sinks": sinks, "shared": shared, "lse": lse, "rot": rot,
         "inter": inter, "mix": mix}
    if name:
        c["name"] = name
    return c


def _window(name, B, Hq, Hkv, Nq, Nk, D, dtype, window, sinks, layout="bhnd", lse=False):
    c = {"op": "window", "B": B, "Hq": Hq, "Hkv": Hkv, "Nq": Nq, "Nk": Nk, "D": D, "dtype": dtype, "window": window,
         "sinks": sinks, "layout": layout, "lse": lse}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # One step of a serving loop: the next token of 32 requests goes into the cache.  The smallest call.
        _paged("append_decode_b32", "append", 32, 32, 8, 128, "bf16", 16, (1, 1), (1, 4000), rot=128),
        # The prompts of a mixed batch, lengths of all kinds, neighbouring pairs rotated.
        _paged("append_ragged", "append", 7, 32, 8, 128, "fp16", 64, (1, 4096), (0, 2000), rot=128, inter=True, mix=2),
        # Long chunks of four requests, head dim 64, half of each head rotated.
        _paged("append_chunks_d64", "append", 4, 16, 4, 64, "bf16", 32, (8192, 8192), (0, 9000), rot=32, mix=3),
        # Decode: one token of 16 requests with contexts of different lengths.
        _paged("decode_b16", "attend", 16, 32, 8, 128, "bf16", 16, (1, 1), (1001, 16001), mix=4),
        # Short contexts, head dim 64, every head with keys of its own: latency.
        _paged("decode_short_d64", "attend", 4, 12, 12, 64, "fp16", 32, (1, 1), (100, 1000), lse=True, mix=5),
        # Long contexts of which each token sees the last 4096 keys and four sinks.
        _paged("decode_window_b32", "attend", 32, 32, 8, 128, "bf16", 64, (1, 1), (3000, 30000), window=4096, sinks=4, mix=6),
        # Chunked prefill of a mixed batch: some requests bring one token, some a chunk.
        _paged("chunks_ragged", "attend", 5, 32, 8, 128, "bf16", 32, (1, 2048), (500, 16000), lse=True, mix=54),
        # 64 requests behind one system prompt, decode.
        _paged("shared_decode_b64", "attend", 64, 32, 8, 128, "bf16", 16, (1, 1), (1, 1000), shared=8192, mix=8),
        # A few requests with four draft tokens each behind a short prompt, head dim 64.
        _paged("shared_draft_b9", "attend", 9, 16, 4, 64, "fp16", 16, (4, 4), (1, 300), shared=1008, lse=True, mix=9),
        # Prefill of a long document with a sliding window.
        _window("window_16384", 1, 32, 8, 16384, 16384, 128, "bf16", 4096, 4),
        # A batch of short sequences, head dim 64, log-sum-exp for a later merge.
        _window("window_1024_d64", 4, 12, 12, 1024, 1024, 64, "fp16", 256, 4, lse=True),
        # Ragged length, an odd number of heads, head dim 96, the (B,N,H,D) layout that projections produce.
        _window("window_ragged_d96", 3, 7, 7, 2001, 2001, 96, "fp16", 301, 1, layout="bnhd"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        kind = rng.choice(["append", "append", "decode", "decode", "chunk", "shared", "window", "window"])
        dtype = rng.choice(["fp16", "bf16"])
        hkv = rng.choice([1, 2, 3, 4, 8, 12])
        g = rng.choice([1, 2, 3, 4, 8])
        D = rng.choice([64, 96, 128, 128])
        page = rng.choice([16, 32, 64, 128])
        lse, mix = rng.random() < 0.4, rng.randrange(1 << 20)
        banded = rng.random() < 0.4
        window, sinks = (_log(rng, 16, 5000), rng.choice([0, 1, 4, 100])) if banded else (0, 0)
        if kind == "append":
            n = _log(rng, 1, 8192)
            new = (n, n) if rng.random() < 0.5 else (max(1, n // 8), n)
            c = _paged("", "append", _log(rng, 1, 64), hkv * g, hkv, D, dtype, page, new, (0, 9000),
                       rot=rng.choice([32, 64, D]), inter=rng.random() < 0.5, mix=mix)
        elif kind == "decode":
            n = rng.choice([1, 1, 1, 2, 5])
            c = _paged("", "attend", _log(rng, 1, 64), hkv * g, hkv, D, dtype, page, (n, n),
                       rng.choice([(10, 1000), (1000, 16000), (4000, 60000)]), window=window, sinks=sinks, lse=lse, mix=mix)
        elif kind == "chunk":
            n = _log(rng, 16, 2048)
            c = _paged("", "attend", _log(rng, 1, 8), hkv * g, hkv, D, dtype, page, rng.choice([(1, n), (n, n)]), (1, 16000),
                       window=window, sinks=sinks, lse=lse, mix=mix)
        elif kind == "shared":
            n = rng.choice([1, 1, 4])
            c = _paged("", "attend", _log(rng, 4, 64), hkv * g, hkv, D, dtype, page, (n, n), (1, 1000),
                       shared=page * _log(rng, 4, 8192 // page), lse=lse, mix=mix)
        else:
            n = _log(rng, 100, 16384)
            nq = n if rng.random() < 0.7 else max(1, n // 7)
            c = _window("", _log(rng, 1, 4), hkv * g, hkv, nq, n, D, dtype, _log(rng, 16, 5000), rng.choice([0, 1, 4, 100]),
                        layout=rng.choice(["bhnd", "bnhd"]), lse=lse)
        w = work(c)
        if w["flops"] <= 9e11 and w["bytes"] <= 8e8:
            return c


def _tokens(case):
    """(tokens of each sequence, new tokens of each sequence) of a paged case."""
    rng = random.Random(case["mix"])
    new = [_log(rng, case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    ctx = [_log(rng, case["ctx_lo"] + 1, case["ctx_hi"] + 1) - 1 for _ in range(case["B"])]
    return [case["shared"] + c + n for c, n in zip(ctx, new)], new


def _first_seen(case, length, n):
    """The first position that the window shows to the new tokens (the sinks before it apart)."""
    return max(0, length - n + 1 - case["window"]) if case["window"] else 0


def _pairs(n, first_pos, window, sinks):
    """(query, key) pairs of ``n`` queries that sit at ``first_pos`` and after."""
    total = 0
    for p in range(first_pos, first_pos + n):
        if window and p + 1 > window:
            total += window + min(sinks, p + 1 - window)
        else:
            total += p + 1
    return total


def work(case):
    c = case
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    if c["op"] == "window":
        B, Nq, Nk = c["B"], c["Nq"], c["Nk"]
        seen = Nk
        if c["window"]:
            low = max(0, Nk - Nq + 1 - c["window"])
            seen = Nk - low + min(c["sinks"], low)
        nbytes = 2.0 * B * D * (2 * Hq * Nq + 2 * Hkv * seen) + (4.0 * B * Hq * Nq if c["lse"] else 0.0)
        return {"bytes": nbytes, "flops": 4.0 * B * Hq * D * _pairs(Nq, Nk - Nq, c["window"], c["sinks"])}
    lens, new = _tokens(c)
    T = sum(new)
    if c["op"] == "append":
        # k, v and q in and out, the rotation's rows of the table; two products and a sum for each rotated element
        return {"bytes": 2.0 * 2 * T * D * (Hq + 2 * Hkv) + 4.0 * T * c["rot"], "flops": 3.0 * T * c["rot"] * (Hq + Hkv)}
    keys = c["shared"]
    pairs = 0
    for length, n in zip(lens, new):
        low = _first_seen(c, length, n)
        keys += length - low + min(c["sinks"], low) - c["shared"]
        pairs += _pairs(n, length - n, c["window"], c["sinks"])
    nbytes = 2.0 * D * (2 * Hq * T + 2 * Hkv * keys) + (4.0 * Hq * T if c["lse"] else 0.0)
    return {"bytes": nbytes, "flops": 4.0 * Hq * D * pairs}


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=_DT[dtype])


def _package():
    pkg = os.path.join(os.getcwd(), "mini-attention_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import miniattn
    return miniattn


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    Hq, Hkv, D, dt = c["Hq"], c["Hkv"], c["D"], c["dtype"]
    if c["op"] == "window":
        B, Nq, Nk = c["B"], c["Nq"], c["Nk"]
        shape = (lambda h, n: (B, h, n, D)) if c["layout"] == "bhnd" else (lambda h, n: (B, n, h, D))
        q, k, v = (_normal(gen, shape(h, n), dt) for h, n in ((Hq, Nq), (Hkv, Nk), (Hkv, Nk)))
        return {"case": c, "q": q, "k": k, "v": v}
    lens, new = _tokens(c)
    B, P = c["B"], c["page"]
    # Which pages each sequence holds, dealt out in no order; the shared ones are the same for all.
    width = max((n + P - 1) // P for n in lens) + 2
    held = []
    for length, n in zip(lens, new):
        low = _first_seen(c, length, n)
        sink_pages = (min(c["sinks"], low) + P - 1) // P
        held.append([j for j in range((length + P - 1) // P) if j >= low // P or j < sink_pages])
    shared_pages = c["shared"] // P
    n_pages = shared_pages + sum(len([j for j in h if j >= shared_pages]) for h in held) + 3
    order = list(range(n_pages))
    random.Random(seed).shuffle(order)
    deal = iter(order)
    common = [next(deal) for _ in range(shared_pages)]
    table = [[-1] * width for _ in range(B)]
    for row, pages in zip(table, held):
        for j in pages:
            row[j] = common[j] if j < shared_pages else next(deal)
    table = torch.tensor(table, dtype=torch.int32, device="cuda")
    cache_k, cache_v = (_normal(gen, (n_pages, P, Hkv, D), dt) for _ in range(2))
    T = sum(new)
    ragged = c["new_lo"] != c["new_hi"]
    cu = torch.tensor([sum(new[:i]) for i in range(B + 1)], dtype=torch.int32, device="cuda") if ragged else None
    s = {"case": c, "k_cache": cache_k, "v_cache": cache_v, "block_table": table, "lens": lens, "new": new, "cu_q": cu,
         "seq_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "max_q": max(new)}
    rows = (T,) if ragged else (B, c["new_lo"])
    s["q"] = _normal(gen, rows + (Hq, D), dt)
    if c["op"] == "append":
        kv = _normal(gen, rows + (2, Hkv, D), dt)  # what one projection produces
        s["k"], s["v"] = kv[..., 0, :, :], kv[..., 1, :, :]
        half = c["rot"] // 2
        angle = (torch.arange(max(lens) + 1, dtype=torch.float64, device="cuda")[:, None]
                 * 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half))
        s["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float()  # what miniattn.rope_table gives
    return s


def run(state):
    c = state["case"]
    if own:
        m = _package()
        if c["op"] == "window":
            return m.flash_attn_fwd(state["q"], state["k"], state["v"], causal=True, layout=c["layout"], return_lse=c["lse"],
                                    q_pos0=c["Nk"] - c["Nq"], window=c["window"], sinks=c["sinks"])
        if c["op"] == "append":
            q = m.paged_append(state["k"], state["v"], state["k_cache"], state["v_cache"], state["block_table"],
                               state["seq_lens"], cu_q=state["cu_q"], q=state["q"], rope=state["rope"],
                               interleaved=c["inter"])
            return q, state["k_cache"], state["v_cache"]
        return m.paged_attention(state["q"], state["k_cache"], state["v_cache"], state["block_table"], state["seq_lens"],
                                 cu_q=state["cu_q"], max_q=state["max_q"], window=c["window"] or None, sinks=c["sinks"],
                                 shared_len=c["shared"], return_lse=c["lse"])
    if c["op"] == "window":
        return _plain_window(state)
    return _plain_append(state) if c["op"] == "append" else _plain_attend(state)


# ---------------------------------------------------------------------------------------------------------------------
# Plain forms: elementary operations in 32 bits, rounded once at the end.


def _plain_rows(q, k, v, q_pos, k_pos, window, sinks):
    """q (n,Hq,D), k, v (L,Hkv,D) in 32 bits, their positions -> o (n,Hq,D), lse (Hq,n).  A row that sees no key is 0."""
    n, Hq, D = q.shape
    L, Hkv = k.shape[0], k.shape[1]
    rows = q.view(n, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3).reshape(Hkv, -1, D)
    s = (rows @ k.permute(1, 2, 0)).view(Hq, n, L) * (1.0 / math.sqrt(D))
    hidden = k_pos[None, :] > q_pos[:, None]
    if window:
        hidden |= (k_pos[None, :] <= q_pos[:, None] - window) & (k_pos[None, :] >= sinks)
    s.masked_fill_(hidden, float("-inf"))
    top = s.amax(2, keepdim=True).clamp_min(-3.0e38)
    p = s.sub_(top).exp_()
    total = p.sum(2, keepdim=True)
    o = (p.view(Hkv, -1, L) @ v.transpose(0, 1)).view(Hq, n, D) / total.clamp_min(1e-38)
    return o.transpose(0, 1), (top + total.log())[:, :, 0]


def _plain_window(state):
    c = state["case"]
    q, k, v = (t if c["layout"] == "bnhd" else t.transpose(1, 2) for t in (state["q"], state["k"], state["v"]))
    B, Nq, Nk = c["B"], c["Nq"], c["Nk"]
    out = torch.empty_like(q)
    lse = torch.empty((B, c["Hq"], Nq), dtype=torch.float32, device=q.device)
    pos = torch.arange(Nk, device=q.device)
    step = 1024
    for b in range(B):
        for r0 in range(0, Nq, step):
            r1 = min(Nq, r0 + step)
            first, last = r0 + Nk - Nq, r1 + Nk - Nq
            low = max(0, first + 1 - c["window"])
            keys = torch.cat([pos[:min(c["sinks"], low)], pos[low:last]])
            o, z = _plain_rows(q[b, r0:r1].float(), k[b, keys].float(), v[b, keys].float(), pos[first:last], keys,
                               c["window"], c["sinks"])
            out[b, r0:r1] = o.to(out.dtype)
            lse[b, :, r0:r1] = z
    if c["layout"] == "bhnd":
        out = out.transpose(1, 2)
    return (out, lse) if c["lse"] else out


def _plain_attend(state):
    c = state["case"]
    q, P = state["q"], c["page"]
    Hq, D = c["Hq"], c["D"]
    flat = q.reshape(-1, Hq, D)
    out = torch.empty_like(flat)
    lse = torch.empty((Hq, flat.shape[0]), dtype=torch.float32, device=q.device)
    at = 0
    for b, (length, n) in enumerate(zip(state["lens"], state["new"])):
        for r0 in range(0, n, 512):
            r1 = min(n, r0 + 512)
            first, last = length - n + r0, length - n + r1
            low = max(0, first + 1 - c["window"]) if c["window"] else 0
            pos = torch.arange(last, device=q.device)
            keys = torch.cat([pos[:min(c["sinks"], low)], pos[low:]])
            page = state["block_table"][b, keys // P].long()
            o, z = _plain_rows(flat[at + r0:at + r1].float(), state["k_cache"][page, keys % P].float(),
                               state["v_cache"][page, keys % P].float(), pos[first:last], keys, c["window"], c["sinks"])
            out[at + r0:at + r1] = o.to(out.dtype)
            lse[:, at + r0:at + r1] = z
        at += n
    out = out.view(q.shape)
    if not c["lse"]:
        return out
    return out, lse if q.dim() == 3 else lse.view(Hq, c["B"], -1).transpose(0, 1)


def _plain_append(state):
    c = state["case"]
    D, rot, P = c["D"], c["rot"], c["page"]
    device = state["q"].device
    lens, new = state["seq_lens"].long(), state["new"]
    counts = torch.tensor(new, device=device) if state["cu_q"] is not None else torch.full_like(lens, new[0])
    seq = torch.repeat_interleave(torch.arange(c["B"], device=device), counts, output_size=sum(new))
    start = torch.cumsum(counts, 0) - counts
    pos = torch.arange(sum(new), device=device) - start[seq] + (lens - counts)[seq]
    cos, sin = (t[:, None, :] for t in state["rope"][pos].split(rot // 2, 1))

    def rotated(x):
        y = x.reshape(-1, x.shape[-2], D).float()
        if c["inter"]:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., :rot // 2], y[..., rot // 2:rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)

    page = state["block_table"][seq, pos // P].long()
    state["k_cache"][page, pos % P] = rotated(state["k"])
    state["v_cache"][page, pos % P] = state["v"].reshape(-1, c["Hkv"], D)
    return rotated(state["q"]).view(state["q"].shape), state["k_cache"], state["v_cache"]


# ---------------------------------------------------------------------------------------------------------------------
# From the definitions, in 64 bits.


def exact(case, seed):
    c = case
    if work(c)["flops"] > 2e12:
        return None
    s = prepare(c, seed)
    if c["op"] == "append":
        return _exact_append(s)
    if c["op"] == "window":
        q, k, v = s["q"], s["k"], s["v"]
        if c["layout"] == "bnhd":
            q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
        lse = torch.empty(q.shape[:3], dtype=torch.float64, device=q.device)
        for b in range(c["B"]):
            for h in range(c["Hq"]):
                g = h // (c["Hq"] // c["Hkv"])
                out[b, h], lse[b, h] = _exact_head(q[b, h], k[b, g], v[b, g], c["Nk"] - c["Nq"], c["window"], c["sinks"])
        if c["layout"] == "bnhd":
            out = out.transpose(1, 2)
        return (out, lse) if c["lse"] else out
    q = s["q"]
    flat = q.reshape(-1, c["Hq"], c["D"])
    out = torch.empty(flat.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty((c["Hq"], flat.shape[0]), dtype=torch.float64, device=q.device)
    at = 0
    for b, (length, n) in enumerate(zip(s["lens"], s["new"])):
        slots = (length + c["page"] - 1) // c["page"]
        pages = s["block_table"][b, :slots].long()
        there = (pages >= 0)[:, None, None, None]
        for g in range(c["Hkv"]):
            # every position of the sequence; what slid out of the window is not held any more and counts as 0
            k, v = ((cache[pages.clamp_min(0), :, g:g + 1].double() * there).reshape(-1, c["D"])[:length]
                    for cache in (s["k_cache"], s["v_cache"]))
            for h in range(g * (c["Hq"] // c["Hkv"]), (g + 1) * (c["Hq"] // c["Hkv"])):
                out[at:at + n, h], lse[h, at:at + n] = _exact_head(flat[at:at + n, h], k, v, length - n, c["window"], c["sinks"])
        at += n
    out = out.view(q.shape)
    if not c["lse"]:
        return out
    return out, lse if q.dim() == 3 else lse.view(c["Hq"], c["B"], -1).transpose(0, 1)


def _exact_head(q, k, v, first, window, sinks):
    """One head: q (n,D) at positions ``first`` and after, k, v (L,D) from position 0 on."""
    n, L = q.shape[0], k.shape[0]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty(n, dtype=torch.float64, device=q.device)
    j = torch.arange(L, device=q.device)
    rows = max(1, (1 << 27) // max(L, 1))
    for r in range(0, n, rows):
        p = torch.arange(r, min(n, r + rows), device=q.device) + first
        visible = j[None] <= p[:, None]
        if window:
            visible &= (p[:, None] - j[None] < window) | (j[None] < sinks)
        score = torch.einsum("id,jd->ij", q[r:r + rows].double(), k.double()) / math.sqrt(q.shape[1])
        z = torch.logsumexp(torch.where(visible, score, float("-inf")), 1)
        weight = torch.where(visible, torch.exp(score - z[:, None]), 0.0)
        out[r:r + rows] = torch.einsum("ij,jd->id", weight, v.double())
        lse[r:r + rows] = z
    return out, lse


def _exact_append(s):
    c = s["case"]
    rot, P = c["rot"], c["page"]
    k, v, q = (s[x].reshape(-1, s[x].shape[-2], c["D"]).double() for x in ("k", "v", "q"))
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    pair = torch.arange(rot // 2, device=q.device)
    one, two = (2 * pair, 2 * pair + 1) if c["inter"] else (pair, pair + rot // 2)
    at = 0
    for b, (length, n) in enumerate(zip(s["lens"], s["new"])):
        p = torch.arange(length - n, length, device=q.device)
        turn = torch.complex(s["rope"][p, :rot // 2].double(), s["rope"][p, rot // 2:].double())[:, None]
        for x in (k, q):
            z = torch.complex(x[at:at + n][..., one], x[at:at + n][..., two]) * turn
            x[at:at + n, :, one], x[at:at + n, :, two] = z.real, z.imag
        pages = s["block_table"][b].long()[p // P]
        k_cache[pages, p % P], v_cache[pages, p % P] = k[at:at + n], v[at:at + n]
        at += n
    return q.view(s["q"].shape), k_cache, v_cache
