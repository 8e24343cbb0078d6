"""The paged-cache and beam entries without a GPU: refusals (the checks come
before any device work), the structures' layouts, the rope frequencies."""
import ctypes as C
import json
import math
import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import GOLDEN, ROOT
from rai_b200 import native

I = native.RAI_ERR_INVALID
U = native.RAI_ERR_UNSUPPORTED
P = 0x10000  # a pointer that nothing reads


def chunk(**kw):
    c = native.PagedChunk(k=P, v=P, k_page=1024, k_head=512, k_slot=64, v_page=1024, v_head=512, v_slot=64, table=P, kv_len=P,
                          q_start=P, table_stride=4, n_seqs=2, max_pages=4, n_pages=9, page_size=8, n_kv_heads=2, head_dim=64,
                          rows=5, max_rows=3, dtype=2)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def attn(ck=None, **kw):
    a = native.PagedAttention(chunk=chunk(**(ck or {})), q=P, out=P, q_row=256, q_head=64, out_row=256, out_head=64, n_heads=4,
                              window=0, scale=0.125, softcap=0.0, workspace=P, workspace_bytes=1 << 40)
    for k, v in kw.items():
        setattr(a, k, v)
    return native.lib().rai_gpu_paged_attention(C.byref(a), None)


CHUNK_BAD = [
    (dict(k=0), I), (dict(table=0), I), (dict(dtype=3), U), (dict(n_seqs=0), I), (dict(page_size=0), I), (dict(rows=0), I),
    (dict(head_dim=60), U), (dict(head_dim=264), U), (dict(max_rows=6), I), (dict(table_stride=3), I), (dict(k_slot=60), I),
    (dict(v_page=-64), I), (dict(k=P + 8), I), (dict(max_pages=1 << 29, table_stride=1 << 29, page_size=8), I),
    (dict(n_seqs=(1 << 30) + 1), I),
]


@pytest.mark.parametrize("bad,rc", CHUNK_BAD)
def test_attention_refuses_chunks(bad, rc):
    assert attn(bad) == rc
    assert native.last_error()


@pytest.mark.parametrize("bad", [dict(q=0), dict(out=0), dict(n_heads=0), dict(n_heads=3), dict(q_row=250), dict(out_head=4),
                                 dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(softcap=-1.0),
                                 dict(softcap=math.inf), dict(window=1 << 31)])
def test_attention_refuses_arguments(bad):
    assert attn(**bad) == I


def test_attention_refuses_small_workspaces():
    big = dict(max_pages=4000, table_stride=4000)
    a = native.PagedAttention(chunk=chunk(**big), n_heads=4)
    need = native.lib().rai_gpu_paged_attention_workspace_bytes(C.byref(a))
    assert need > 0
    assert attn(big, workspace_bytes=need - 1) == I
    assert attn(big, workspace=0) == I
    assert attn(big, workspace=P + 4) == I


def rope(ck=None, **kw):
    a = native.RopeAppend(chunk=chunk(**(ck or {})), q=P, k=P, v=P, q_out=2 * P, inv_freq=P, q_row=512, q_head=64, k_row=512,
                          k_head=64, v_row=512, v_head=64, out_row=256, out_head=64, n_heads=4, rot_dim=64, interleaved=0, in_dtype=2,
                          mscale=1.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return native.lib().rai_gpu_rope_append(C.byref(a), None)


@pytest.mark.parametrize("bad,rc", [(dict(q=0), I), (dict(inv_freq=0), I), (dict(rot_dim=0), I), (dict(rot_dim=7), I),
                                    (dict(rot_dim=66), I), (dict(in_dtype=5), U), (dict(mscale=math.nan), I), (dict(k_row=500), I),
                                    (dict(q_out=P), I), (dict(n_heads=5), I)])
def test_rope_refuses(bad, rc):
    assert rope(**bad) == rc


@pytest.mark.parametrize("bad,rc", CHUNK_BAD)
def test_rope_refuses_chunks(bad, rc):
    assert rope(bad) == rc


def table(**kw):
    t = native.PageTable(table=P, lens=P, refs=P, table_stride=6, n_seqs=3, max_pages=6, n_pages=20, page_size=16)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def pool(**kw):
    p = native.PagePool(k=P, v=P, k_layer=1 << 20, k_page=4096, v_layer=1 << 20, v_page=4096, page_bytes=4096, n_layers=2, n_pages=20)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_fork_refuses():
    L = native.lib()

    def fork(a, b, parents=P):
        return L.rai_gpu_kv_fork(C.byref(a), C.byref(b), parents, None)
    far = dict(table=P + 4096, lens=P + 8192)
    for kw in (dict(table=0), dict(n_seqs=0), dict(page_size=0), dict(table_stride=5)):
        assert fork(table(**kw), table(**far)) == I
    assert fork(table(), table(**far), 0) == I
    assert fork(table(), table(refs=2 * P, **far)) == I
    assert fork(table(), table(n_pages=21, **far)) == I
    assert fork(table(), table(page_size=8, **far)) == I
    assert fork(table(), table(max_pages=5, **far)) == I
    assert fork(table(), table(lens=P + 8192)) == I                   # one table
    assert fork(table(), table(table=P + 40, lens=P + 8192)) == I     # overlapping ones
    assert fork(table(), table(table=P + 4096)) == I                  # one vector of lengths


def test_resize_and_compact_refuse():
    L = native.lib()
    ws = L.rai_gpu_kv_resize_workspace_bytes(3)
    assert ws > 0 and L.rai_gpu_kv_resize_workspace_bytes(4097) == 0

    def resize(t=None, p=None, status=P, w=P, n=ws):
        return L.rai_gpu_kv_resize(C.byref(t or table()), C.byref(p or pool()), None, 1, status, w, n, None)
    assert resize(status=0) == I and resize(w=0) == I and resize(n=ws - 1) == I
    assert resize(table(n_seqs=4097), n=1 << 30) == U
    for kw in (dict(k=0), dict(n_pages=19), dict(page_bytes=0), dict(page_bytes=4100), dict(k_page=4000), dict(k=P + 8), dict(n_layers=0)):
        assert resize(p=pool(**kw)) == I
    cw = L.rai_gpu_kv_compact_workspace_bytes(20)
    assert L.rai_gpu_kv_compact(C.byref(table()), C.byref(pool()), None, P, cw, None) == I
    assert L.rai_gpu_kv_compact(C.byref(table()), C.byref(pool()), P, P, cw - 1, None) == I
    assert L.rai_gpu_kv_copy_pages(C.byref(pool()), None, P, 3, None) == I
    assert L.rai_gpu_kv_copy_pages(C.byref(pool()), P, P, 1 << 31, None) == I
    assert L.rai_gpu_kv_copy_pages(C.byref(pool()), None, None, 0, None) == native.RAI_OK


def test_beams_refuse():
    L = native.lib()
    need = L.rai_gpu_beam_workspace_bytes(2, 3, 100, 6)
    assert need > 0
    assert L.rai_gpu_beam_workspace_bytes(2, 33, 100, 64) == 0

    def select(**kw):
        a = native.BeamSelect(logits=P, scores=P, row_stride=100, cand_score=P, cand_beam=P, cand_token=P, score=P, parent=P, token=P,
                              batch=2, beams=3, vocab=100, keep=6, eos=-1, dtype=0, workspace=P, workspace_bytes=need)
        for k, v in kw.items():
            setattr(a, k, v)
        return L.rai_gpu_beam_select(C.byref(a), None)
    for kw in (dict(logits=0), dict(token=0), dict(batch=0), dict(vocab=0), dict(keep=2), dict(row_stride=99), dict(eos=-2),
               dict(workspace=0), dict(workspace_bytes=need - 1), dict(vocab=1 << 30, row_stride=1 << 30), dict(batch=30000),
               dict(logits=P + 2), dict(history=P), dict(history=P, hist_len=P, out_history=P, out_len=2 * P, hist_cap=4, hist_stride=4,
                                                         out_hist_stride=4),
               dict(history=P, hist_len=P, out_history=2 * P, out_len=2 * P, hist_cap=4, hist_stride=3, out_hist_stride=4)):
        assert select(**kw) == I, kw
    for kw in (dict(beams=33, keep=64), dict(keep=65), dict(dtype=9)):
        assert select(**kw) == U, kw


def test_structures_have_the_headers_layout(tmp_path):
    """Size and field offsets of the ctypes structures against a C compiler's
    reading of include/rai_gpu.h."""
    pairs = [(native.PagedChunk, "rai_paged_chunk"), (native.PagedAttention, "rai_paged_attention"), (native.RopeAppend, "rai_rope_append"),
             (native.PageTable, "rai_page_table"), (native.PagePool, "rai_page_pool"), (native.BeamSelect, "rai_beam_select")]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{ROOT}/include/rai_gpu.h"', "int main(void) {"]
    want = []
    for py, c in pairs:
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        want.append(C.sizeof(py))
        for name, _ in py._fields_:
            lines.append(f'printf("%zu\\n", offsetof({c}, {name}));')
            want.append(getattr(py, name).offset)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == want


def test_host_tensors_are_refused():
    torch = pytest.importorskip("torch")
    from rai_b200 import beams, paged
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    k = torch.zeros(3, 2, 8, 64, dtype=torch.bfloat16)
    t, n, s = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: paged.attention(q, k, k, t, n, s, 2), lambda: paged.attention(q.float(), k, k, t, n, s, 2),
                 lambda: paged.attention(q[0], k, k, t, n, s, 2), lambda: paged.attention(q.requires_grad_(), k, k, t, n, s, 2),
                 lambda: paged.fork(t, n, s, n, 16), lambda: paged.resize(t, n, s, k, k, delta=1),
                 lambda: beams.select(torch.zeros(1, 2, 9), torch.zeros(1, 2)), lambda: beams.select(torch.zeros(2, 9), torch.zeros(1, 2)),
                 lambda: beams.select(torch.zeros(1, 2, 9, dtype=torch.int32), torch.zeros(1, 2))):
        with pytest.raises(ValueError):
            call()


def test_rope_frequencies():
    from rai_b200 import paged
    f, m = paged.rope_frequencies(128, 500000.0)
    assert m == 1.0 and np.array_equal(f, (500000.0 ** (-2.0 * np.arange(64) / 128)).astype(np.float32))
    f, _ = paged.rope_frequencies(64, 10000.0, "linear", factor=4.0)
    assert np.array_equal(f, (10000.0 ** (-2.0 * np.arange(32) / 64) / 4).astype(np.float32))
    f, _ = paged.rope_frequencies(64, 10000.0, "ntk", factor=4.0)
    assert np.allclose(f, (10000.0 * 4.0 ** (64 / 62)) ** (-2.0 * np.arange(32) / 64), rtol=1e-6)
    # The reference's llama3 table (taken from transformers), within the f32 steps of its own computation.
    g = json.load(open(os.path.join(GOLDEN, "llama3_inv_freq.json")))
    f, _ = paged.rope_frequencies(64, 500000.0, "llama3", factor=32.0, low=1.0, high=4.0, original=8192.0)
    want = np.array(next(v for v in g.values() if isinstance(v, list)), np.float32)
    assert np.allclose(f, want, rtol=4e-7)
    # YaRN: the fast pairs kept, the slow ones divided, monotone between.
    plain, _ = paged.rope_frequencies(128, 10000.0)
    f, m = paged.rope_frequencies(128, 10000.0, "yarn", factor=16.0, low=1.0, high=32.0, original=4096.0)
    assert abs(m - (0.1 * math.log(16.0) + 1)) < 1e-6
    ratio = plain / f
    assert np.allclose(ratio[:20], 1.0, rtol=1e-6) and np.allclose(ratio[-16:], 16.0, rtol=1e-6) and (np.diff(ratio) >= -1e-5).all()
    import rai_b200
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=300), dict(theta=1.0), dict(kind="linear", factor=0.5),
                dict(kind="llama3", factor=2.0, low=4.0, high=1.0)):
        with pytest.raises(rai_b200.RaiError):
            paged.rope_frequencies(**{"rot_dim": 64, **bad})
    with pytest.raises(ValueError):
        paged.rope_frequencies(64, kind="cubic")


@pytest.mark.parametrize("rows", [1, 3, 9])
def test_fork_refuses_outputs_of_another_number_of_rows(rows):
    """The kernel takes the number of children from the outputs and reads as
    many parents."""
    torch = pytest.importorskip("torch")
    from rai_b200 import paged
    i32 = dict(dtype=torch.int32)
    table, lens, refs, parents = torch.zeros(2, 4, **i32), torch.ones(2, **i32), torch.ones(8, **i32), torch.zeros(2, **i32)
    with pytest.raises(ValueError, match="out_lens"):
        paged.fork(table, lens, refs, parents, 16, out_table=torch.zeros(2, 4, **i32), out_lens=torch.zeros(rows, **i32))
    with pytest.raises(ValueError, match="out_table"):
        paged.fork(table, lens, refs, parents, 16, out_table=torch.zeros(rows, 4, **i32), out_lens=torch.zeros(2, **i32))


def test_attention_workspace_of_empty_pages():
    """Pages of no tokens: refused by the call, no division by zero in the
    query before it. (In a child, which the division would end.)"""
    code = """
import ctypes as C
from rai_b200 import native
for hd in (64, 128, 256):
    for dtype in range(3):
        for page, rows in ((0, 1), (0, 500), (16, 0)):
            a = native.PagedAttention(chunk=native.PagedChunk(n_seqs=1, max_pages=400, n_pages=4, page_size=page, n_kv_heads=2, head_dim=hd,
                                                              rows=rows, max_rows=rows, dtype=dtype), n_heads=4)
            assert native.lib().rai_gpu_paged_attention_workspace_bytes(C.byref(a)) == 0
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)
    assert attn(dict(page_size=0)) == I


@pytest.mark.parametrize("cap", [1e-40, -1e-40, -0.5, math.nan])
def test_attention_refuses_caps_without_a_reciprocal(cap):
    assert attn(softcap=cap) == I


def test_tensors_with_a_gradient_are_refused():
    """The operators have no backward pass: a gradient would be lost."""
    torch = pytest.importorskip("torch")
    from rai_b200 import beams, paged
    i32 = dict(dtype=torch.int32)
    q = torch.zeros(2, 4, 64)
    kx = torch.zeros(2, 2, 64)
    k = torch.zeros(3, 2, 8, 64)
    grad = torch.zeros(3, 2, 8, 64, requires_grad=True)
    t, n, s, refs = torch.zeros(1, 2, **i32), torch.ones(1, **i32), torch.zeros(2, **i32), torch.zeros(3, **i32)
    inv = torch.zeros(32)
    calls = [lambda a, b: paged.attention(q, a, b, t, n, s, 2), lambda a, b: paged.rope_append(q, kx, kx, a, b, t, n, s, inv),
             lambda a, b: paged.resize(t, n, refs, a, b, delta=1), lambda a, b: paged.compact(t, n, refs, a, b),
             lambda a, b: paged.copy_pages(a, b, n, n)]
    for call in calls:
        for a, b in ((grad, k), (k, grad)):
            with pytest.raises(ValueError, match="no gradient"):
                call(a, b)
            with torch.no_grad(), pytest.raises(ValueError, match="device"):
                call(a, b)
    for call in (lambda: paged.rope_append(q, kx, kx, k, k, t, n, s, inv.clone().requires_grad_()),
                 lambda: paged.attention(q, k, k, t, n, s, 2, lse=torch.zeros(2, 4, requires_grad=True)),
                 lambda: beams.select(torch.zeros(1, 2, 9), torch.zeros(1, 2, requires_grad=True)),
                 lambda: beams.select(torch.zeros(1, 2, 9, requires_grad=True), torch.zeros(1, 2))):
        with pytest.raises(ValueError, match="no gradient|device"):
            call()
    with pytest.raises(ValueError, match="scores: .*no gradient"):
        beams.select(torch.zeros(1, 2, 9), torch.zeros(1, 2, requires_grad=True))
    with pytest.raises(ValueError, match="inv_freq: .*no gradient"):
        paged.rope_append(q, kx, kx, k, k, t, n, s, inv.clone().requires_grad_())


def test_written_rows_that_share_memory_are_refused():
    """Strides of 0 (expanded tensors) or below a row, where a call writes;
    reading such pages is fine."""
    assert attn(out_row=0) == I and "share" in native.last_error()
    assert attn(out_head=0) == I and "share" in native.last_error()
    assert attn(out_head=32, out_row=256) == I and "share" in native.last_error()
    assert attn(out_row=192) == I and "share" in native.last_error()
    assert rope(dict(v=2 * P), out_row=0) == I and "share" in native.last_error()
    for kw in (dict(k_head=0), dict(v_slot=0), dict(k_page=0), dict(v_page=512)):
        assert rope(dict(v=2 * P, **kw)) == I and "share" in native.last_error(), kw
    assert rope() == I and "share" in native.last_error()  # k and v pages in one memory
    L = native.lib()
    far = dict(table=P + 4096, lens=P + 8192)
    for parents in (P + 4096, P + 4100, P + 8192, P + 8200):
        assert L.rai_gpu_kv_fork(C.byref(table()), C.byref(table(**far)), parents, None) == I
    ws = L.rai_gpu_kv_resize_workspace_bytes(3)
    assert L.rai_gpu_kv_resize(C.byref(table()), C.byref(pool()), P + 4, 0, P, P, ws, None) == I
    assert "overlap" in native.last_error()


def test_rope_frequencies_by_default():
    """YaRN's ramp ends at 32 turns, Llama 3's at 4."""
    from rai_b200 import paged
    args = dict(factor=8.0, original=4096.0)
    for kind, high in (("yarn", 32.0), ("llama3", 4.0)):
        f, m = paged.rope_frequencies(128, 10000.0, kind, **args)
        g, n = paged.rope_frequencies(128, 10000.0, kind, low=1.0, high=high, **args)
        assert np.array_equal(f, g) and m == n


def test_build_without_python_headers(tmp_path, monkeypatch, capsys):
    """The library is built; the extension is left out, an older one with it."""
    pytest.importorskip("torch")
    from rai_b200 import build
    old = tmp_path / "_torch_ops.so"
    old.write_bytes(b"of another build")
    monkeypatch.setattr(build, "TORCH_OPS", str(old))
    monkeypatch.setattr(build, "python_headers", lambda: str(tmp_path / "none"))
    assert build.build_torch_ops() is None
    assert not old.exists() and "Python headers" in capsys.readouterr().err


@pytest.mark.parametrize("keep", [0, 2, 65, 1 << 40])
def test_beams_refuse_keep_before_they_allocate(keep):
    torch = pytest.importorskip("torch")
    from rai_b200 import beams
    with pytest.raises(ValueError, match="keep"):
        beams.select(torch.zeros(1, 3, 9), torch.zeros(1, 3), keep=keep)


def test_attention_refuses_scales_whose_product_overflows():
    for scale in (2.4e38, 3.4e38):
        assert attn(scale=scale) == I and "scale" in native.last_error()
