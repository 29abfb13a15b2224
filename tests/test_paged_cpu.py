"""The paged entry points without a GPU: parameter blocks, refusals of the C entries, and the index arithmetic that the kernels
share with the host (csrc/cache.cuh, csrc/append.cuh), compiled for the CPU and compared with the rules written out."""
import ctypes as C
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "mini-attention_b200" / "csrc"
CUDA = Path("/usr/local/cuda/include")


def test_struct_layouts_match_c(tmp_path):
    from miniattn import _lib
    pairs = [("MiniAttnCacheParams", _lib.CacheParams), ("MiniAttnAppendParams", _lib.AppendParams)]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT / "include" / "miniattn.h"}"', "int main(void){"]
    for name, mirror in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in mirror._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", str(src), "-o", str(tmp_path / "layout")], check=True)
    out = iter(subprocess.run([str(tmp_path / "layout")], check=True, capture_output=True, text=True).stdout.split())
    for name, mirror in pairs:
        assert int(next(out)) == C.sizeof(mirror), name
        for f in mirror._fields_:
            assert int(next(out)) == getattr(mirror, f[0]).offset, (name, f[0])


def _cache_params(**kw):
    from miniattn import _lib
    p = _lib.CacheParams()
    p.q = p.k = p.v = p.o = p.block_table = p.seq_lens = 0x1000   # never read: validation fails first
    p.B, p.Hq, p.Hkv, p.D, p.Nq = 2, 4, 2, 64, 1
    p.page_size, p.n_pages, p.table_width, p.table_stride = 16, 10, 4, 4
    for s in (p.q_stride, p.o_stride):
        s[:] = (256, 64, 256)
    for s in (p.k_stride, p.v_stride):
        s[:] = (16 * 128, 64, 128)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw, code, text", [
    (dict(dtype=7), -2, "dtype"), (dict(D=80), -2, "head dim"), (dict(Nq=-1), -1, "negative"), (dict(Hkv=3), -1, "multiple of Hkv"),
    (dict(Hkv=0), -1, "multiple of Hkv"), (dict(page_size=24), -2, "page size"), (dict(page_size=8), -2, "page size"),
    (dict(page_size=2048), -2, "page size"), (dict(block_table=0), -1, "must not be null"), (dict(seq_lens=0), -1, "must not be null"),
    (dict(seq_lens=0x1002), -1, "4-byte"), (dict(table_stride=3), -1, "columns"), (dict(n_pages=-1), -1, "pages"),
    (dict(window=-1), -1, "negative"), (dict(sinks=4), -1, "window is 0"), (dict(shared_len=8), -1, "multiple of the page size"),
    (dict(shared_len=80), -1, "inside the block table"), (dict(shared_len=16, window=4), -2, "do not go together"),
    (dict(page_size=0), -1, "need pages"), (dict(page_size=0, block_table=0, seq_lens=0, diag=1 << 41), -2, "2^40"),
    (dict(B=65536), -2, "65535"), (dict(Nq=1 << 30), -2, "31 bits"), (dict(q=0), -1, "q is null"), (dict(o=0x1004), -1, "aligned"),
    (dict(k_stride=(2048, 64, 130)), -1, "multiple of 8"), (dict(v_stride=(2048, 64, 32)), -1, "smaller than D"),
])
def test_attention_refuses(kw, code, text):
    from miniattn import _lib
    assert _lib.lib.miniattn_fwd_cache(C.byref(_cache_params(**kw)), None, 0, None) == code
    assert text in _lib.last_error()


def test_attention_empty_calls():
    from miniattn import _lib
    assert _lib.lib.miniattn_fwd_cache(None, None, 0, None) == -1
    for kw in (dict(B=0), dict(Nq=0), dict(Hq=0), dict(cu_q=0x1000, total_q=0)):
        assert _lib.lib.miniattn_fwd_cache(C.byref(_cache_params(**kw)), None, 0, None) == 0
        assert _lib.lib.miniattn_fwd_cache_scratch_bytes(C.byref(_cache_params(**kw))) == 0


def _append_params(**kw):
    from miniattn import _lib
    p = _lib.AppendParams()
    p.k = p.v = p.q = p.k_cache = p.v_cache = p.q_out = p.rope = p.block_table = p.seq_lens = 0x1000
    p.B, p.Hq, p.Hkv, p.D, p.n = 2, 4, 2, 64, 1
    p.rot, p.rope_rows, p.page_size, p.n_pages, p.table_width, p.table_stride = 64, 100, 16, 10, 4, 4
    for s in (p.k_stride, p.v_stride):
        s[:] = (128, 64, 128)
    for s in (p.q_stride, p.q_out_stride):
        s[:] = (256, 64, 256)
    for s in (p.k_cache_stride, p.v_cache_stride):
        s[:] = (16 * 128, 64, 128)
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(p, k)[:] = v
        else:
            setattr(p, k, v)
    return p


@pytest.mark.parametrize("kw, code, text", [
    (dict(dtype=7), -2, "dtype"), (dict(D=80), -2, "head dim"), (dict(n=-1), -1, "negative"), (dict(Hkv=0), -1, "Hkv"),
    (dict(page_size=17), -2, "page size"), (dict(block_table=0), -1, "must not be null"), (dict(seq_lens=0), -1, "must not be null"),
    (dict(rot=8), -2, "multiple of 16"), (dict(rot=24), -2, "multiple of 16"), (dict(rot=80), -2, "multiple of 16"),
    (dict(rope=0x1008), -1, "16-byte"), (dict(rope_rows=-1), -1, "negative"), (dict(interleaved=2), -1, "0 or 1"),
    (dict(k=0), -1, "k is null"), (dict(v=0x1008), -1, "aligned"), (dict(q_out=0), -1, "q_out is null"),
    (dict(k_cache=0), -1, "k_cache is null"), (dict(v_cache_stride=(2048, 64, 12)), -1, "multiple of 8"),
    (dict(Hkv=70000), -2, "65535"), (dict(n=1 << 31 - 1), -2, "31 bits"),
])
def test_append_refuses(kw, code, text):
    from miniattn import _lib
    assert _lib.lib.miniattn_paged_append(C.byref(_append_params(**kw)), None) == code
    assert text in _lib.last_error()


def test_append_empty_calls():
    from miniattn import _lib
    assert _lib.lib.miniattn_paged_append(None, None) == -1
    for kw in (dict(B=0), dict(n=0), dict(cu_q=0x1000, total=0)):
        assert _lib.lib.miniattn_paged_append(C.byref(_append_params(**kw)), None) == 0


def test_status_bit_of_paged_calls():
    from miniattn import _lib
    assert _lib.lib.miniattn_check_status(1 << 7) == _lib.EINVAL and "outside its tensors" in _lib.last_error()
    assert _lib.lib.miniattn_check_status(1 << 7 | 1) == _lib.EDEVICE_WAIT


def test_python_refuses_host_tensors():
    import miniattn
    q = torch.zeros((1, 1, 2, 64), dtype=torch.float16)
    cache, table, lens = torch.zeros((4, 16, 2, 64), dtype=torch.float16), torch.zeros((1, 4), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        miniattn.paged_attention(q, cache, cache, table, lens)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        miniattn.paged_append(q, q, cache, cache, table, lens)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        miniattn.flash_attn_fwd(q, q, q, causal=True, window=4)
    with pytest.raises(RuntimeError, match="causal"):
        miniattn.flash_attn_fwd(q, q, q, window=4)


def test_rope_table():
    import miniattn
    table = miniattn.rope_table(50, 32, theta=100.0)
    assert table.shape == (50, 32) and table.dtype == torch.float32
    for pos, i in ((0, 0), (49, 0), (17, 15), (49, 7)):
        angle = torch.tensor(pos * 100.0 ** (-2 * i / 32), dtype=torch.float64)
        assert abs(float(table[pos, i]) - float(angle.cos())) <= 2.0 ** -24
        assert abs(float(table[pos, 16 + i]) - float(angle.sin())) <= 2.0 ** -24
    assert miniattn.rope_table(0, 32).shape == (0, 32)
    with pytest.raises(RuntimeError, match="even"):
        miniattn.rope_table(4, 0)


# Every key that a row sees lies in a tile of its sequence and is read; keys that no row sees count as unseen, one by one and in
# runs; nothing lies outside the sequence, the block table or the rows of q, whatever the lengths say.
GEOMETRY = r"""
#include <cuda_runtime.h>
#include "cache.cuh"
#include <cstdio>
#include <cstdlib>
using namespace ma;
static int fail(const char* what, int n) { std::printf("%s at %d\n", what, n); return 1; }
template <int T> static bool in_tiles(const CacheTiles& t, int k) {
  for (int j = 0; j < t.n; ++j) if (t.at(j) == k / T) return true;
  return false;
}
int main() {
  std::srand(7);
  int dummy = 0;
  for (int trial = 0; trial < 40000; ++trial) {
    CacheArgs a{};
    const bool paged = std::rand() % 3, ragged = paged && std::rand() % 2;
    a.window = std::rand() % 3 ? 1 + std::rand() % 300 : 0;
    a.sinks = a.window ? std::rand() % 3 * (std::rand() % 200) : 0;
    a.Nq = 1 + std::rand() % 40;
    a.page_shift = 4 + std::rand() % 3;
    a.table_width = std::rand() % 40;
    a.total_q = 100;
    if (paged && !a.window && std::rand() % 3 == 0) a.key0 = 16 * (std::rand() % 6);
    int r0 = 0, r1 = 0, len = std::rand() % 700;
    if (std::rand() % 8 == 0) len = std::rand() % 2 ? -std::rand() : 2147483647 - std::rand() % 5;
    if (paged) a.seq_lens = &dummy;
    else { a.Nk = std::rand() % 700; a.diag = std::rand() % 900 - 300; if (std::rand() % 9 == 0) a.diag = 1ll << 40; }
    if (ragged) {
      a.cu_q = &dummy;
      r0 = std::rand() % 100;
      r1 = r0 + std::rand() % 50;
      if (std::rand() % 8 == 0) { r0 = std::rand() - 1000000000; r1 = std::rand() - 1000000000; }
    }
    const CacheSeq s = cache_seq(a, r0, r1, len);
    const long long room = paged ? static_cast<long long>(a.table_width) << a.page_shift : a.Nk;
    const int held = paged ? (len < 0 ? 0 : len > room ? (int)room : len) : a.Nk;
    if (s.nq < 0 || (ragged && (s.row0 < 0 || s.row0 + s.nq > a.total_q))) return fail("rows", trial);
    if (s.lo < 0 || s.lo > s.hi || s.hi > held || s.hi > room || s.sink_end < 0 || s.sink_end > s.lo) return fail("range", trial);
    if (paged && s.bad != (len < 0 || len > room || (ragged && (r0 < 0 || r0 > 100 || r1 < r0 || r1 > 100)))) return fail("bad", trial);
    const CacheTiles t64 = cache_tiles<64>(s.lo, s.hi, s.sink_end), t128 = cache_tiles<128>(s.lo, s.hi, s.sink_end);
    if (t64.n < 1 || t128.n < 1) return fail("no tile", trial);
    static bool seen[4096];
    for (bool& x : seen) x = false;
    for (int i = 0; i < s.nq; ++i) {
      int first, end;
      cache_row(a, s, i, &first, &end);
      const long long pos = paged ? (long long)held - s.nq + i : a.diag + i;
      for (int k = 0; k < held; ++k) {
        const bool want = k <= pos && (!a.window ? k >= a.key0 : k > pos - a.window || k < a.sinks);
        if (want != (k < end && (k >= first || k < a.sinks))) return fail("row", trial);
        seen[k] |= want;
      }
    }
    for (int k = 0; k < held; ++k) {
      if (seen[k] && (!cache_seen(s.lo, s.hi, s.sink_end, k, 1) || !in_tiles<64>(t64, k) || !in_tiles<128>(t128, k)))
        return fail("a key that a row sees is not read", trial);
      if (!seen[k] && s.nq > 0 && cache_seen(s.lo, s.hi, s.sink_end, k, 1)) return fail("an unseen key counts as seen", trial);
    }
    for (int x = 0; x < 40; ++x) {
      const int n = 16 << (std::rand() % 4), k = std::rand() % 64 * n % 1024 / n * n;
      bool any = false, all = true;
      for (int i = k; i < k + n; ++i) { const bool one = cache_seen(s.lo, s.hi, s.sink_end, i, 1); any |= one; all &= one; }
      if (any != cache_seen(s.lo, s.hi, s.sink_end, k, n)) return fail("run", trial);
      if (!all != cache_partly_seen(s.lo, s.hi, s.sink_end, k, n)) return fail("partly", trial);
    }
  }
  std::printf("ok\n");
  return 0;
}
"""

APPEND = r"""
#include <cuda_runtime.h>
#include "append.cuh"
#include <cstdio>
#include <cstdlib>
using namespace ma;
int main() {
  std::srand(3);
  static float rope[1];
  for (int trial = 0; trial < 2000000; ++trial) {
    AppendArgs a{};
    a.page_shift = 4 + std::rand() % 7;
    a.table_width = std::rand() % 9;
    a.n_pages = std::rand() % 5;
    a.rope = std::rand() % 2 ? rope : nullptr;
    a.rope_rows = std::rand() % 600;
    const long long first = std::rand() % 50, n_new = std::rand() % 50;
    const int t = std::rand() % 100;
    a.rows = std::rand() % 8 ? 100 : std::rand() % 100;
    int len = std::rand() % 700;
    if (std::rand() % 8 == 0) len = std::rand() % 2 ? -std::rand() : 2147483647 - std::rand() % 3;
    const int page = std::rand() % 8 - 2;
    int asked = -1;
    const AppendSlot s = append_slot(a, t, first, n_new, len, [&](int i) { asked = i; return page; });
    const bool rows_bad = first + n_new > a.rows || t >= first + n_new;
    if (s.none != (t < first || rows_bad)) return 5;
    if (s.none && (s.held || asked != -1 || s.bad != rows_bad)) return 6;
    if (s.none) continue;
    const long long pos = len - n_new + (t - first);
    if (asked >= a.table_width) return 1;                                    // outside the block table
    const bool room = pos >= 0 && pos < ((long long)a.table_width << a.page_shift) && (!a.rope || pos < a.rope_rows);
    if (s.held != (room && page >= 0 && page < a.n_pages)) return 2;
    if (s.bad != (pos >= 0 ? !s.held : len < 0)) return 3;
    if (s.held && (s.pos != pos || s.page != page || s.at != (pos & ((1 << a.page_shift) - 1)) || asked != (pos >> a.page_shift))) return 4;
  }
  std::printf("ok\n");
  return 0;
}
"""


@pytest.mark.skipif(not (CUDA / "cuda.h").exists(), reason="no CUDA headers")
@pytest.mark.parametrize("name", ["GEOMETRY", "APPEND"])
def test_index_arithmetic(name, tmp_path):
    src = tmp_path / "walk.cpp"
    src.write_text(globals()[name])
    subprocess.run(["g++", "-O2", "-std=c++17", f"-I{CSRC}", f"-I{CUDA}", str(src), "-o", str(tmp_path / "walk")], check=True)
    r = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", (r.returncode, r.stdout)
