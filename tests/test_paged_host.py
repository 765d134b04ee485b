"""What the paged cache entry points refuse, and the page lookup of the kernels, without a GPU."""

import ctypes as C
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 4096                                 # a well-aligned address that nothing reads: every call here is refused before a launch


@pytest.fixture(scope="module")
def hip():
    from lcm import _hip
    return _hip


def _pages(hip, **kw):
    a = dict(k=P, v=P, n_pages=8, page_size=16, n_kv_heads=2, head_dim=128, dtype=1)
    a.update(kw)
    return hip.KVPages(**a)


def _batch(hip, **kw):
    a = dict(page_table=P, seq_lens=P, q_starts=P, n_seqs=3, max_pages=4, max_q=4, max_keys=64)
    a.update(kw)
    return hip.PagedBatch(**a)


def _prefix(hip, **kw):
    a = dict(page_table=P, lens=P, group_starts=P, n_groups=1, max_pages=4, max_keys=64)
    a.update(kw)
    return hip.SharedPrefix(**a)


def _refused(hip, rc, text):
    assert rc == -1 and text in hip.lib.lcmhip_last_error(), (rc, hip.lib.lcmhip_last_error())


def _attend(hip, pages=None, batch=None, q=P, q_row=1024, q_head=128, out=P, rows=6, heads=4, scale=0.1, ws=P, ws_bytes=1 << 40, prefix=None):
    pages, batch = pages or _pages(hip), batch or _batch(hip)
    if prefix is not None:
        return hip.lib.lcmhip_shared_prefix_attention(pages, batch, prefix, q, q_row, q_head, out, rows, heads, scale, 1, ws, ws_bytes, None)
    return hip.lib.lcmhip_paged_attention(pages, batch, q, q_row, q_head, out, rows, heads, scale, 1, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,text", [
    (dict(k=None), b"null pages"), (dict(v=None), b"null pages"), (dict(k=P + 8), b"16-byte"), (dict(dtype=7), b"dtype"),
    (dict(head_dim=96), b"head_dim"), (dict(head_dim=256), b"head_dim"), (dict(page_size=8), b"page_size"), (dict(page_size=48), b"page_size"),
    (dict(page_size=0), b"page_size"), (dict(page_size=1 << 17), b"page_size"), (dict(n_kv_heads=0), b"n_kv_heads"), (dict(n_kv_heads=3), b"multiple of n_kv_heads"),
    (dict(n_pages=0), b"n_pages"), (dict(n_pages=1 << 31), b"n_pages")])
def test_refused_pages(hip, kw, text):
    _refused(hip, _attend(hip, pages=_pages(hip, **kw)), text)
    if b"multiple" not in text:
        rc = hip.lib.lcmhip_paged_append(_pages(hip, **kw), _batch(hip), P, 512, 128, P, 512, 128, None, 0, 0, None, 6, 0, None, None, None, None)
        _refused(hip, rc, text)


@pytest.mark.parametrize("kw,text", [
    (dict(page_table=None), b"null"), (dict(seq_lens=None), b"null"), (dict(n_seqs=-1), b"n_seqs"), (dict(max_pages=0), b"max_pages"),
    (dict(max_q=0), b"max_q"), (dict(max_keys=0), b"max_keys"), (dict(max_keys=65), b"max_keys"),
    (dict(max_keys=(1 << 30) + 1, max_pages=1 << 30), b"max_keys"), (dict(q_starts=None), b"one row for every sequence")])
def test_refused_batches(hip, kw, text):
    _refused(hip, _attend(hip, batch=_batch(hip, **kw)), text)
    rc = hip.lib.lcmhip_paged_append(_pages(hip), _batch(hip, **kw), P, 512, 128, P, 512, 128, None, 0, 0, None, 6, 0, None, None, None, None)
    _refused(hip, rc, text)


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), b"null"), (dict(out=None), b"null"), (dict(q=P + 2), b"16 bytes"), (dict(out=P + 4), b"16 bytes"), (dict(q_row=1025), b"16 bytes"),
    (dict(q_head=132), b"16 bytes"), (dict(rows=-1), b"rows"), (dict(heads=0), b"n_heads"), (dict(heads=5), b"n_heads"),
    (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"), (dict(scale=1e-30), b"scale"), (dict(scale=1e30), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(scale=float("inf")), b"scale")])
def test_refused_attention_arguments(hip, kw, text):
    _refused(hip, _attend(hip, **kw), text)
    _refused(hip, _attend(hip, prefix=_prefix(hip), **kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(page_table=None), b"null"), (dict(lens=None), b"null"), (dict(group_starts=None), b"null"), (dict(n_groups=0), b"n_groups"),
    (dict(max_pages=0), b"max_pages"), (dict(max_keys=0), b"max_keys"), (dict(max_keys=65), b"max_keys")])
def test_refused_prefixes(hip, kw, text):
    _refused(hip, _attend(hip, prefix=_prefix(hip, **kw)), text)


def test_refused_heads(hip):
    def call(q=P, q_row=512, k=P, k_row=512, q_out=P, qo_row=512, k_out=P, rows=4, hq=4, hk=4, d=128, norm=None, rot=None, pos=P, dtype=1):
        return hip.lib.lcmhip_head_norm_rope(q, q_row, 128, k, k_row, 128, q_out, qo_row, 128, k_out, 512, 128, rows, hq, hk, d, norm, rot,
                                             pos, dtype, None)
    rot = dict(cos=P, sin=P, n_positions=8, rotary_dim=128, style=0)
    norm = dict(q_weight=P, k_weight=P, kind=1, eps=1e-5)
    cases = [(dict(q=None, k=None), b"neither"), (dict(q_out=None), b"without its output"), (dict(k=None), b"without its output"),
             (dict(d=96), b"head_dim"), (dict(dtype=3), b"dtype"), (dict(rows=-1), b"rows"), (dict(hq=0), b"head count"), (dict(q_row=513), b"16 bytes"),
             (dict(q=P + 8, q_out=P + 8), b"16 bytes"), (dict(qo_row=1024), b"in place"),
             (dict(rot=hip.Rotary(**rot), pos=None), b"positions"), (dict(rot=hip.Rotary(**{**rot, "rotary_dim": 24})), b"rotary_dim"),
             (dict(rot=hip.Rotary(**{**rot, "rotary_dim": 144})), b"rotary_dim"), (dict(rot=hip.Rotary(**{**rot, "rotary_dim": 0})), b"rotary_dim"),
             (dict(rot=hip.Rotary(**{**rot, "style": 2})), b"style"), (dict(rot=hip.Rotary(**{**rot, "cos": None})), b"null table"),
             (dict(rot=hip.Rotary(**{**rot, "n_positions": 0})), b"empty"), (dict(rot=hip.Rotary(**{**rot, "sin": P + 4})), b"16-byte"),
             (dict(norm=hip.HeadNorm(**{**norm, "kind": 9})), b"norm kind"), (dict(norm=hip.HeadNorm(**{**norm, "k_weight": None})), b"needs weights"),
             (dict(norm=hip.HeadNorm(**{**norm, "kind": 3})), b"no weights"), (dict(norm=hip.HeadNorm(**{**norm, "q_bias": P})), b"no bias"),
             (dict(norm=hip.HeadNorm(**{**norm, "eps": -1.0})), b"eps"), (dict(norm=hip.HeadNorm(**{**norm, "eps": float("nan")})), b"eps"),
             (dict(norm=hip.HeadNorm(**{**norm, "q_weight": P + 2})), b"16-byte")]
    for kw, text in cases:
        _refused(hip, call(**kw), text)


def test_refused_append(hip):
    def call(k=P, v=P, q=None, q_out=None, heads=0, k_row=512):
        return hip.lib.lcmhip_paged_append(_pages(hip), _batch(hip), k, k_row, 128, v, 512, 128, q, 512, 128, q_out, 6, heads, None, None, None, None)
    for kw, text in [(dict(k=None), b"null"), (dict(v=None), b"null"), (dict(q=P), b"together"), (dict(q_out=P), b"together"),
                     (dict(q=P, q_out=P), b"head count"), (dict(k_row=516), b"16 bytes"), (dict(v=P + 8), b"16 bytes")]:
        _refused(hip, call(**kw), text)


def test_no_sequences_is_no_work(hip):
    """A batch without sequences is accepted with empty arrays, and nothing is launched (there is no GPU here)."""
    none = _batch(hip, n_seqs=0, page_table=None, seq_lens=None)
    assert _attend(hip, batch=none) == 0 and _attend(hip, batch=none, prefix=_prefix(hip)) == 0
    assert hip.lib.lcmhip_paged_append(_pages(hip), none, P, 512, 128, P, 512, 128, None, 0, 0, None, 6, 0, None, None, None, None) == 0
    assert _attend(hip, batch=_batch(hip, n_seqs=0, q_starts=None), rows=0) == 0


def test_workspace_sizes(hip):
    n = C.c_size_t()
    assert hip.lib.lcmhip_paged_attention_workspace(_pages(hip), _batch(hip), 6, 4, None) == -1
    assert hip.lib.lcmhip_paged_attention_workspace(_pages(hip), _batch(hip), 6, 4, C.byref(n)) == 0
    assert hip.lib.lcmhip_shared_prefix_attention_workspace(_pages(hip), _batch(hip), _prefix(hip), 6, 4, C.byref(n)) == 0
    if n.value:                            # a workspace that is too small, or missing, is refused
        _refused(hip, _attend(hip, prefix=_prefix(hip), ws_bytes=n.value - 1), b"workspace")
        _refused(hip, _attend(hip, prefix=_prefix(hip), ws=None), b"workspace")
        _refused(hip, _attend(hip, prefix=_prefix(hip), ws=P + 16), b"workspace")


def test_python_layer_refuses_host_tensors():
    from lcm.nn import paged_attention as pa
    q = torch.zeros(2, 4, 128)
    with pytest.raises(RuntimeError, match="must live on a GPU"):
        pa.head_norm_rope(q, None)
    with pytest.raises(ValueError, match="queries or keys"):
        pa.head_norm_rope(None, None)
    with pytest.raises(RuntimeError, match="must live on a GPU"):
        pa.KVPages(torch.zeros(1, 1, 16, 128), torch.zeros(1, 1, 16, 128))
    with pytest.raises(RuntimeError, match="must live on a GPU"):
        pa.PagedBatch(torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="must live on a GPU"):
        pa.RotaryTable.create(8, 64, device="cpu")
    with pytest.raises(ValueError, match="layer normalization"):
        pa.HeadNorm("batch")


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")
def test_page_lookup_never_leaves_the_pool(tmp_path):
    """PageTable::page and seq_rows, the only places where a kernel turns index arrays into addresses, as host code: every id
    outside the pool and every position behind the table answers -1, row ranges stay inside the rows."""
    src = tmp_path / "lookup.hip"
    src.write_text(r'''
#include "%s/chimera-llm_amd/csrc/paged.h"
#include <cstdio>
namespace lcmhip { int fail(int c, const std::string&) { return c; } }
int main() {
    const int32_t ids[8] = {0, 6, 7, -1, INT32_MIN, INT32_MAX, 5, 1 << 20};
    lcmhip::PageTable t{ids, 4, 4, 7};
    const int want[2][4] = {{0, 6, -1, -1}, {-1, -1, 5, -1}};
    for (int s = 0; s < 2; ++s)
        for (int p = 0; p < 4; ++p)
            for (int o = 0; o < 16; ++o)
                if (t.page(s, 16 * p + o) != want[s][p]) return printf("page %%d %%d\n", s, p), 1;
    if (t.page(0, 64) != -1 || t.page(1, INT32_MAX) != -1) return 2;
    const int32_t starts[6] = {-5, 3, 2, 9, 100, INT32_MAX};
    for (int b = 0; b < 5; ++b) {
        int64_t r0, r1;
        lcmhip::seq_rows(starts, b, 8, r0, r1);
        if (r0 < 0 || r1 < r0 || r1 > 8) return printf("rows %%d\n", b), 3;
    }
    return 0;
}
''' % ROOT)
    exe = tmp_path / "lookup"
    subprocess.run(["/opt/rocm/bin/hipcc", "-std=c++17", "-O1", "--offload-host-only", str(src), "-o", str(exe)], check=True,
                   capture_output=True, timeout=300)
    assert subprocess.run([str(exe)], capture_output=True, timeout=60).returncode == 0
