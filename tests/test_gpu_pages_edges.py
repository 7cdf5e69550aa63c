"""Attention for runs of rows (over listed pages, and over the whole cache) beside values and scores at the edge of what the types hold:
what a row does not see weighs nothing at all, and a score that is not finite shows."""
import pytest
import torch

from tests.test_gpu_pages import BF, DEV, PAGE, Step, like_lists

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from gophonic_b200 import ops as o
    return o


def attend_all(ops, s, window=0):
    """The rows of ``s`` over everything their sequences hold."""
    out = torch.full((s.q.shape[0], s.heads * s.d), 9.0, dtype=s.dtype, device=DEV)
    slot, start, q_len, kv_len = s.seq
    ops.attention(s.q_dev, out, s.dev["k_plane"], s.dev["v_plane"], s.dev["table"], slot, start, q_len, kv_len, s.nseq, s.max_q, s.heads, s.kvh, s.d,
                  s.d ** -0.5, window, algo="prefill_tc5")
    return out


def by_head(s, out):
    """[rows, kv heads, the group's channels], float32, on the CPU."""
    return out.cpu().float().reshape(out.shape[0], s.kvh, -1)


FORMS = pytest.mark.parametrize("heads,kvh,new", [(4, 1, 150), (16, 8, 700)], ids=["shared tiles", "whole tiles"])


# ---- what a row does not see -------------------------------------------------------------------
@FORMS
@pytest.mark.parametrize("where", ["unlisted page", "another row's page", "behind the last token", "later token"])
@pytest.mark.parametrize("value", [3e38, -3e38])
def test_unseen_values_near_the_largest_weigh_nothing(ops, heads, kvh, new, where, value):
    """A weight of 2^-126 would add 3.5 a key; a weight of zero leaves every bit."""
    s = Step([(1000, new)], heads, kvh, 128, BF, seed=2)
    pages = like_lists(s, 8, 5, 12, 9)
    mine, pos = s.table[s.slots[0]], 1000 + new - 1
    sees = torch.zeros((new, kvh), dtype=torch.bool)
    v = s.dev["v_plane"]
    if where == "unlisted page":
        pages[pages == 1] = -1
    clean = s.attend(ops, pages.to(DEV)).clone()
    if where == "behind the last token":
        assert (pos + 1) % PAGE
        v[mine[pos // PAGE], :, pos % PAGE + 1:] = value
    elif where == "later token":
        v[mine[pos // PAGE], :, pos % PAGE] = value
        sees[new - 1] = (pages[new - 1] == pos // PAGE).any(-1)
    else:
        page = 1 if where == "unlisted page" else 3
        v[mine[page]] = value
        sees = (pages == page).any(-1)
        assert where == "unlisted page" or (sees.any() and not sees.all())
    got, ref = by_head(s, s.attend(ops, pages.to(DEV))), by_head(s, clean)
    assert torch.equal(got[~sees], ref[~sees])
    assert ops.tc5_status() == 0


@pytest.mark.parametrize("window,seen_by_none", [(0, []), (90, [5, 6, 7, 14, 20])], ids=["all", "window"])
@pytest.mark.parametrize("value", [3e38, -3e38])
def test_unseen_values_near_the_largest_weigh_nothing_in_a_prompt(ops, window, seen_by_none, value):
    """The same of the attention over the whole cache: later tokens' values, those ahead of the window, those behind the last token."""
    past, new = 70, 200
    s = Step([(past, new)], 4, 2, 128, BF, seed=3)
    clean = attend_all(ops, s, window)
    mine, v = s.table[s.slots[0]], s.dev["v_plane"]
    later = list(range(150, 5 * PAGE))
    for pos in seen_by_none + later:
        v[mine[pos // PAGE], :, pos % PAGE] = value
    rows = [r for r in range(new) if past + r < 150 and (not window or past + r - window >= 20)]
    assert len(rows) >= 30
    got = attend_all(ops, s, window)
    assert torch.equal(got[rows], clean[rows]) and ops.tc5_status() == 0
