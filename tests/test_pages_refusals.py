"""What the entry points of page_bounds, select_pages and attention_pages refuse before anything reaches a GPU."""
import ctypes

import pytest

ops = pytest.importorskip("gophonic_b200.ops")


def params(**kw):
    base = dict(q=4096, q_row_stride=256, out=4096, out_row_stride=256, k_plane=4096, v_plane=4096, bounds=4096, block_table=4096, bt_stride=8, seq_slot=4096,
                seq_q_start=4096, seq_q_len=4096, seq_kv_len=4096, nseq=1, heads=4, kv_heads=2, d=64, max_q_len=1, scale=1.0, list=4096, top=4, first=1, last=2,
                planes=1, pages=8, max_slots=2, rows=1)
    base.update(kw)
    return ops._PagesParams(**base)


def refused(name, dtype, **kw):
    rc = getattr(ops._lib, name)(ctypes.byref(params(**kw)), ctypes.c_int(dtype), ctypes.c_void_p(0))
    text = ops._lib.gb_last_error().decode()
    return rc == -1 and text.startswith(name[3:] + ":"), text


BAD = {
    "gb_page_bounds": [dict(d=20), dict(d=264), dict(d=0), dict(kv_heads=0), dict(pages=0), dict(bt_stride=0), dict(max_slots=0), dict(bounds=4098),
                       dict(k_plane=4104), dict(planes=1 << 28), dict(nseq=70000)],
    "gb_select_pages": [dict(d=20), dict(heads=3), dict(heads=0), dict(first=-1), dict(last=0), dict(first=3), dict(top=2), dict(top=0), dict(bt_stride=32769),
                        dict(bounds=4098), dict(nseq=1 << 20, max_q_len=1 << 12)],
    "gb_attention_pages": [dict(d=20), dict(d=144), dict(d=272), dict(heads=3), dict(kv_heads=0), dict(top=0), dict(top=1025), dict(pages=0), dict(k_plane=4104),
                           dict(v_plane=4104), dict(q=4098), dict(q_row_stride=257)],
}


@pytest.mark.parametrize("name,kw", [(n, kw) for n, bad in BAD.items() for kw in bad if "nseq" not in kw])
def test_refused(name, kw):
    ok, text = refused(name, ops.BF16, **kw)
    assert ok, text


@pytest.mark.parametrize("name", list(BAD))
def test_unknown_dtype(name):
    ok, text = refused(name, 7)
    assert ok, text


@pytest.mark.parametrize("kw", [dict(nseq=0), dict(max_q_len=0)])
@pytest.mark.parametrize("name", list(BAD))
def test_nothing_to_do(name, kw):
    assert getattr(ops._lib, name)(ctypes.byref(params(**kw)), ctypes.c_int(ops.F32), ctypes.c_void_p(0)) == 0


def test_tensors_on_the_cpu_are_refused():
    import torch
    i = torch.zeros(1, dtype=torch.int32)
    k, b, t = torch.zeros(2, 1, 64, 16), torch.zeros(2, 1, 2, 16), torch.zeros((1, 2), dtype=torch.int32)
    q, lists = torch.zeros(1, 16), torch.zeros((1, 1, 4), dtype=torch.int32)
    for call in (lambda: ops.page_bounds(k, b, t, i, i, i, 1, 1), lambda: ops.select_pages(q, b, t, i, i, i, i, 1, 1, 1, 1, 16, lists),
                 lambda: ops.attention_pages(q, q, k, k, t, i, i, i, i, 1, 1, 1, 1, 16, 1.0, lists)):
        with pytest.raises(ops.KernelError):
            call()
