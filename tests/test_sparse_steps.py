"""Which rows of a step select pages: each sequence by what it brings itself.  What needs no GPU."""
from types import SimpleNamespace

import pytest
import torch

from gophonic_b200.cache import Cache, CacheError
from gophonic_b200.config import PageSelection
from gophonic_b200.engine.step import Engine, build_batch
from gophonic_b200.parts.base import BlockStateRequest, KVRequest, KVStateRequest, StateRequest
from gophonic_b200.parts.sparse_attention import SparseAttention


def mixer(pages=3, prompts=False):
    m = SparseAttention.__new__(SparseAttention)
    m.spec = SimpleNamespace(selection=PageSelection(pages, prompts=prompts), heads=4, kv_heads=2, head_dim=64, window=0)
    m.rt = SimpleNamespace(is_fp32=False)
    return m


def who(extents, singles=None, **kw):
    batch, _ = build_batch([(i, [5] * rows, past) for i, (past, rows) in enumerate(extents)], torch.device("cpu"), singles=singles)
    got = mixer(**kw).who_selects(batch)
    return got if isinstance(got, bool) else tuple(t.tolist() for t in got)


def test_single_tokens_alone():
    assert who([(500, 1), (20, 1)]) is True
    assert who([(191, 1), (20, 1)]) is False
    assert who([(500, 1), (20, 1)], prompts=True) is True


def test_runs_alone():
    assert who([(500, 40), (20, 2)]) is False
    assert who([(500, 40), (20, 2)], prompts=True) is True


def test_single_tokens_beside_runs():
    assert who([(500, 1), (0, 300), (20, 1), (192, 1)]) == ([1, 0, 0, 1], [0, 300, 1, 0])
    assert who([(100, 1), (0, 300)]) is False
    assert who([(500, 1), (0, 300)], prompts=True) is True


def test_a_row_that_a_pass_holds_of_a_run_is_no_single_token():
    assert who([(500, 1)], [False]) is False
    assert who([(500, 1), (600, 1)], [False, True]) == ([0, 1], [1, 0])
    assert who([(500, 1), (600, 40)], [False, False]) is False
    assert who([(500, 1)], [False], prompts=True) is True


def test_a_row_of_a_run_is_read_in_one_piece():
    batch, _ = build_batch([(0, [5], 5000)], torch.device("cpu"), singles=[False])
    assert mixer().key_splits(batch) == (1, None)


@pytest.mark.parametrize("most,lens", [(100, [301]), (100, [99, 302]), (100, [301, 1]), (4, [9, 1, 3]), (1, [3, 1])])
def test_passes_know_which_rows_are_single_tokens(monkeypatch, most, lens):
    """A long step is cut into passes; what one pass holds of a run stays part of a run."""
    seen = []
    eng = SimpleNamespace(max_rows_per_pass=most, vocab=7, device="cpu", cache=SimpleNamespace(length=lambda slot: 0))
    eng._pass = lambda pieces, want, source=None, singles=None: seen.extend((slot, first, single) for (slot, _, first), single in zip(pieces, singles))
    starts = [sum(lens[:i]) for i in range(len(lens))]
    Engine._chunked(eng, [(i, [0] * n) for i, n in enumerate(lens)], starts, [])
    assert len(seen) > len(lens)
    assert all(single == (lens[slot] == 1) for slot, _, single in seen)


def test_a_run_that_selects_reads_no_cache_without_bounds():
    """Nor one that has them only because another run of its group asked: who writes the keys keeps them."""
    plain, bounded = KVRequest(2, 16), KVRequest(2, 16, bounds=True)
    for owner in (plain, KVStateRequest(plain, StateRequest((4,), torch.float32)), BlockStateRequest(plain, StateRequest((4,), torch.float32))):
        for more in ([], [(bounded, None)]):
            with pytest.raises(CacheError, match="bounds"):
                Cache([(owner, None), (bounded, 0)] + more, 256, "cpu", torch.float32)
    c = Cache([(bounded, None), (bounded, 0), (plain, 0)], 256, "cpu", torch.float32)
    assert c.view(1).bounds.data_ptr() == c.view(0).bounds.data_ptr()


@pytest.mark.parametrize("first,last", [(2 ** 31 - 1, 1), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 30, 2 ** 30), (1, 2 ** 31 - 1)])
def test_more_pages_always_chosen_than_numbers_hold(first, last):
    """Their sum passes 31 bits: refused ahead of any launch, as every sum above the list's length is."""
    import ctypes
    ops = pytest.importorskip("gophonic_b200.ops")
    p = ops._PagesParams(q=4096, q_row_stride=256, bounds=4096, block_table=4096, bt_stride=8, seq_slot=4096, seq_q_start=4096, seq_q_len=4096,
                         seq_kv_len=4096, nseq=1, heads=4, kv_heads=2, d=64, max_q_len=1, list=4096, top=4, first=first, last=last, pages=8, max_slots=2, rows=1)
    rc = ops._lib.gb_select_pages(ctypes.byref(p), ctypes.c_int(ops.BF16), ctypes.c_void_p(0))
    assert rc == -1 and "always chosen" in ops._lib.gb_last_error().decode()
