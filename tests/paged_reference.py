"""What the tests of the paged operators compare with: attention and rotation from their definitions, in 64 bits, and the
bounds on a kernel that rounds its weights and results to 16 bits and computes in 32."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def visible(n, length, first, window, sinks):
    """(n, length) truth values: query i sits at position first + i."""
    j = torch.arange(length)[None]
    p = torch.arange(n)[:, None] + first
    seen = j <= p
    if window is not None:
        seen &= (j > p - window) | (j < sinks)
    return seen


def attention(q, k, v, first, window=None, sinks=0, scale=None):
    """q (n,Hq,D), k, v (L,Hkv,D) -> o, tolerance of o (n,Hq,D), lse, tolerance of lse (Hq,n), all in 64 bits.

    Tolerance of o, with u half a step of the type and A the weighted mean of |v|: rounding each weight is off by u A, rounding
    the result by u |o|.  A score is a sum of D products, off by at most 2 D 2^-24 of the sum of their magnitudes (a factor of
    2 for sums that truncate), and its exponential by that much and 2^-20 for the argument's rounding, the approximation and
    the sum of the weights (fewer than L / 8 additions of 2^-24 in one thread); both the sum of weights and the weighted sum
    carry it.  In fp16 a weight below 2^-14 of its reference is off by up to 2^-25, and the largest weight is 1 at least."""
    n, Hq, D = q.shape
    L, Hkv = k.shape[0], k.shape[1]
    u = HALF_STEP[q.dtype]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    rows = lambda x: x.double().transpose(0, 1)  # noqa: E731
    qd, kd, vd = rows(q), rows(k).repeat_interleave(Hq // Hkv, 0), rows(v).repeat_interleave(Hq // Hkv, 0)
    seen = visible(n, L, first, window, sinks).to(q.device)[None]
    s = (qd @ kd.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
    size = (qd.abs() @ kd.abs().transpose(1, 2) * scale).masked_fill(~seen, 0.0).amax(2) if L else s.new_zeros(Hq, n)
    top = (s.amax(2) if L else s.new_full((Hq, n), -math.inf)).clamp_min(-1e300)
    w = torch.exp(s - top[..., None])
    total = w.sum(2)
    empty = total == 0
    w = w / total.clamp_min(1e-300)[..., None]
    o, a = w @ vd, w @ vd.abs()
    lse = torch.where(empty, -math.inf, top + total.clamp_min(1e-300).log())
    off = 2 * D * 2.0 ** -24 * size + 2.0 ** -20 + L / 8 * 2.0 ** -24
    tol = 1.01 * u * (a + o.abs()) + 2 * off[..., None] * a
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (seen.double() @ vd.abs())
    tol_lse = off + 2.0 ** -22 * torch.where(empty, 0.0, lse).abs()
    return o.transpose(0, 1), tol.transpose(0, 1) + 1e-30, lse, tol_lse


def rotate(x, table, pos, interleaved):
    """x (n,H,D) -> rotated, tolerance, in 64 bits; table (positions, rot) fp32, pos (n,).  Two products and a sum in 32 bits,
    rounded once."""
    half = table.shape[1] // 2
    c, s = (t.double()[:, None] for t in table[pos].split(half, 1))
    i = torch.arange(half, device=x.device)
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y, tol = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    a, b = y[..., one].clone(), y[..., two].clone()
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    tol[..., one] = 3 * 2.0 ** -24 * ((a * c).abs() + (b * s).abs())
    tol[..., two] = 3 * 2.0 ** -24 * ((b * c).abs() + (a * s).abs())
    turned = torch.zeros(x.shape[-1], dtype=torch.bool, device=x.device)
    turned[torch.cat([one, two])] = True
    # 2^-25: half of fp16's smallest step, below which rounding is no longer relative
    tol[..., turned] += 1.01 * HALF_STEP[x.dtype] * y[..., turned].abs() + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    return y, tol


class Paged:
    """Sequences in pages: what the operators get, and what lies in them.  Every place that no query row sees holds a NaN or an
    infinity, and every entry of the block table that none needs a number outside the cache."""

    def __init__(self, lens, news, Hkv, D, dtype, page, *, window=None, sinks=0, shared=0, seed=0, device="cuda:0",
                 heads_first=False, spare=3):
        gen = torch.Generator().manual_seed(seed)
        self.lens, self.news = lens, news
        B = len(lens)
        width = max((max(lens) + page - 1) // page, 1) + 2
        prefix = torch.randn((2, shared, Hkv, D), generator=gen).to(dtype)
        self.k, self.v = [], []
        rows, needed = [], []
        for length, n in zip(lens, news):
            kv = torch.randn((2, length, Hkv, D), generator=gen).to(dtype)
            m = min(shared, length)
            kv[:, :m] = prefix[:, :m]
            self.k.append(kv[0])
            self.v.append(kv[1])
            seen = visible(n, length, length - n, window, sinks)
            needed.append(seen.any(0) if n and length else torch.zeros(length, dtype=torch.bool))
        common = shared // page
        n_pages = spare + common + sum((length + page - 1) // page for length in lens)
        order = torch.randperm(n_pages, generator=gen).tolist()
        shape = (n_pages, Hkv, page, D) if heads_first else (n_pages, page, Hkv, D)
        poison = torch.tensor([math.nan, math.inf, -math.inf])[torch.randint(3, shape, generator=gen)].to(dtype)
        caches = [poison.clone(), poison.flip(0).clone()]
        at = [c.transpose(1, 2) if heads_first else c for c in caches]
        table = torch.full((B, width), -7, dtype=torch.int32)
        table[:, 1::2] = n_pages + 11
        first = [order.pop() for _ in range(common)]
        for b, length in enumerate(lens):
            for j in range((length + page - 1) // page):
                seen = needed[b][j * page:(j + 1) * page]
                if j < common:
                    p = first[j]
                elif seen.any():
                    p = order.pop()
                else:
                    continue
                table[b, j] = p
                for i in torch.nonzero(seen)[:, 0].tolist():
                    at[0][p, i], at[1][p, i] = self.k[b][j * page + i], self.v[b][j * page + i]
        self.k_cache, self.v_cache = (c.to(device).transpose(1, 2) if heads_first else c.to(device) for c in caches)
        self.table = table.to(device)
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=device)
        self.cu_q = torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=torch.int32, device=device)
        self.window, self.sinks, self.device, self.B = window, sinks, device, B

    def expected(self, q_rows, scale=None):
        """q_rows: the rows of each sequence, (n,Hq,D) -> lists of o, tolerance, lse, tolerance."""
        out = [attention(q.to(self.device), k.to(self.device), v.to(self.device), length - n, self.window, self.sinks, scale)
               for q, k, v, length, n in zip(q_rows, self.k, self.v, self.lens, self.news)]
        return [list(x) for x in zip(*out)]


def check(got, want, tol, what):
    got = got.double()
    bad = ~((got - want).abs() <= tol) & ~((got == want) & torch.isinf(want))
    if bool(bad.any()):
        i = tuple(int(x) for x in torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: {got[i].item()} for "
                             f"{want[i].item()} +- {tol.expand(got.shape)[i].item()}")
