"""Attention for runs of rows (over listed pages, and over the whole cache) beside values and scores at the edge of what the types hold:
what a row does not see weighs nothing at all, and a score that is not finite shows."""
import math

import pytest
import torch

from tests.test_gpu_pages import BF, DEV, F32, PAGE, Step, check_selection, like_lists, names

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


# by how many CTAs share a tile: eight, three, none
FORMS = pytest.mark.parametrize("heads,kvh,new", [(4, 1, 150), (16, 8, 700), (32, 8, 700)], ids=["eight", "three", "one"])


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


# ---- scores that are not finite ----------------------------------------------------------------
def poisoned(s, keys, page, place, score):
    """A copy of the key plane ``keys`` in which one key of a page scores ``score`` (+inf, -inf or NaN) for every row: their queries' first
    channel is positive (``looks_up``)."""
    k = keys.clone()
    k[s.table[s.slots[0], page], :, place, 0] = score
    return k


def looks_up(s):
    q = s.wide[:, :s.heads * s.d].view(-1, s.heads, s.d)
    q[:, :, 0] = q[:, :, 0].abs() + 0.25
    s.q = s.wide[:, :s.heads * s.d].cpu()


def check_places(ops, s, call, sees, clean, scores):
    """``call(key plane)`` with one key poisoned at each place of page 3: rows that see it hold no finite number, the others are as they were up
    to the rounding of their weights (a row that shares its tile may be made anew over its own keys)."""
    keys = s.dev["k_plane"]
    for place in range(PAGE):
        for score in scores:
            got = by_head(s, call(poisoned(s, keys, 3, place, score)))
            see = sees(place)
            assert see.any()
            assert got[see].isnan().all(), (place, score)
            assert got[~see].isfinite().all(), (place, score)
            assert see.all() or float((got[~see] - clean[~see]).abs().max()) <= 4 * 2.0 ** -8 * float(s.v_plane.float().abs().max()), (place, score)
    assert ops.tc5_status() == 0


def check_listed(ops, heads, kvh, new, scores):
    s = Step([(150, new)], heads, kvh, 128, BF, seed=2)
    looks_up(s)
    pages = like_lists(s, 5, 5, 12, 5)
    pos = 150 + torch.arange(new).unsqueeze(1)
    listed = (pages == 3).any(-1)
    assert listed.any() and not listed.all()
    clean = by_head(s, s.attend(ops, pages.to(DEV)))

    def call(k):
        s.dev["k_plane"] = k
        return s.attend(ops, pages.to(DEV))
    check_places(ops, s, call, lambda place: listed & (pos >= 3 * PAGE + place), clean, scores)


def check_prompt(ops, scores):
    s = Step([(150, 200)], 4, 2, 128, BF, seed=3)
    looks_up(s)
    clean = by_head(s, attend_all(ops, s))
    pos = (150 + torch.arange(200)).unsqueeze(1).expand(200, 2)

    def call(k):
        s.dev["k_plane"] = k
        return attend_all(ops, s)
    check_places(ops, s, call, lambda place: pos >= 3 * PAGE + place, clean, scores)


@FORMS
def test_a_score_beyond_all_others_shows(ops, heads, kvh, new):
    """A score of +inf makes the row's softmax inf / inf, at whichever place of its page the key stands."""
    check_listed(ops, heads, kvh, new, [math.inf])


def test_a_score_beyond_all_others_shows_in_a_prompt(ops):
    check_prompt(ops, [math.inf])


@FORMS
def test_a_score_that_is_no_number_shows(ops, heads, kvh, new):
    check_listed(ops, heads, kvh, new, [math.nan])


def test_a_score_that_is_no_number_shows_in_a_prompt(ops):
    check_prompt(ops, [math.nan])


@FORMS
def test_scores_that_are_all_the_lowest_show(ops, heads, kvh, new):
    """All scores -inf: 0 / 0.  Some of them: keys of no weight."""
    s = Step([(150, new)], heads, kvh, 128, BF, seed=2)
    looks_up(s)
    pages = like_lists(s, 5, 5, 12, 5)
    pages[pages == 0] = -1       # so that some rows list page 3 alone
    pages[60:90] = -1
    pages[60:90, :, 2] = 3
    own = (150 + torch.arange(new)).view(new, 1, 1) // PAGE
    pages[(pages == 3) & (own < 3)] = -1
    alone = (pages == 3).any(-1) & ((pages == 3) | (pages < 0)).all(-1)
    without = pages.clone()
    without[without == 3] = -1
    empty = (pages < 0).all(-1)
    want = by_head(s, s.attend(ops, without.to(DEV)))
    s.dev["k_plane"][s.table[s.slots[0], 3], :, :, 0] = -math.inf
    got = by_head(s, s.attend(ops, pages.to(DEV)))
    assert alone.any() and (~alone & (pages == 3).any(-1)).any()
    assert got[alone].isnan().all() and (got[empty] == 0).all()
    assert got[~alone].isfinite().all()
    assert float((got[~alone] - want[~alone]).abs().max()) <= 4 * 2.0 ** -8 * float(s.v_plane.float().abs().max())
    s.dev["k_plane"][:, :, :, 0] = -math.inf
    got = by_head(s, s.attend(ops, pages.to(DEV)))
    assert got[~empty].isnan().all() and (got[empty] == 0).all() and ops.tc5_status() == 0


@pytest.mark.parametrize("dtype,heads,kvh,d", [(BF, 4, 2, 128), (BF, 20, 1, 64), (F32, 4, 2, 64), (F32, 20, 1, 128)], ids=names)
def test_scores_of_single_rows_that_are_not_finite(ops, dtype, heads, kvh, d):
    """Rows one by one, their lists in one piece and in several: NaN for a score of NaN or +inf and for -inf alone, zeros for no key."""
    for top in (4, 32):
        s = Step([(2100, 1)] * 7, heads, kvh, d, dtype, seed=4)
        looks_up(s)
        pages = torch.full((7, kvh, top), -1, dtype=torch.int32)
        pages[0:3, :, 1] = 3
        pages[3:6] = torch.arange(top, dtype=torch.int32) if top == 32 else torch.tensor([0, 2, 3, 9], dtype=torch.int32)
        keys = s.dev["k_plane"]
        for i, score in [(0, math.nan), (1, math.inf), (3, math.nan), (4, math.inf)]:
            keys[s.table[s.slots[i], 3], :, 41, 0] = score
        for i in (2, 5):
            keys[s.table[s.slots[i], 3], :, :, 0] = -math.inf
        want = s.attend(ops, torch.where(pages == 3, -1, pages).to(DEV))
        got = s.attend(ops, pages.to(DEV))
        assert got[:5].isnan().all() and (got[6] == 0).all() and got[5].isfinite().all()
        assert float((got[5].float() - want[5].float()).abs().max()) <= 4 * (2.0 ** -8 if dtype == BF else 2.0 ** -17) * float(s.v_plane.float().abs().max())


def test_scores_that_are_all_the_lowest_show_in_a_prompt(ops):
    s = Step([(0, 150)], 4, 2, 128, BF, seed=3)
    looks_up(s)
    s.dev["k_plane"][:, :, :, 0] = -math.inf
    assert attend_all(ops, s).isnan().all() and ops.tc5_status() == 0


@pytest.mark.parametrize("algo", ["prefill_tc5", "prefill_mma"])
@pytest.mark.parametrize("own", [False, True], ids=["a unit", "a score a head"])
def test_a_sink_takes_all_where_the_scores_are_the_lowest(ops, algo, own):
    """0 / exp(sink): zeros, where without a sink it is 0 / 0."""
    s = Step([(0, 150)], 4, 2, 128, BF, seed=3)
    looks_up(s)
    s.dev["k_plane"][:, :, :, 0] = -math.inf
    out = torch.full((150, 512), 9.0, dtype=BF, device=DEV)
    slot, start, q_len, kv_len = s.seq
    sinks = torch.tensor([0.5, -3.0, 2.0, 0.0], device=DEV) if own else None
    ops.attention(s.q_dev, out, s.dev["k_plane"], s.dev["v_plane"], s.dev["table"], slot, start, q_len, kv_len, 1, 150, 4, 2, 128, 128 ** -0.5, algo=algo,
                  sink=True, sinks=sinks)
    assert (out == 0).all() and ops.tc5_status() == 0


# ---- scores whose sums lose most of what they add up -------------------------------------------
@pytest.mark.parametrize("big", [300.0, 2e4, 1e6])
@pytest.mark.parametrize("pages,new,d", [(300, 21, 128), (300, 9, 64), (300, 40, 48), (300, 2, 128), (100, 12, 256)])
def test_select_pages_whose_scores_cancel_late(ops, big, pages, new, d):
    """The first channel's bound carries a number through the whole sum that the last channel's takes off again."""
    s = Step([(pages * PAGE - new + 1, new)], 2, 1, d, BF, seed=pages)
    bounds = s.bounds_plane()
    mine = s.table[s.slots[0]].long()
    for side in (0, 1):
        bounds[mine, 0, side, 0] = big
        bounds[mine, 0, side, d - 1] = -big
    q = s.wide[:, :2 * d].view(-1, 2, d)
    q[:, :, 0] = q[:, :, d - 1] = 0.75
    s.q = s.wide[:, :2 * d].cpu()
    check_selection(s, s.select(ops, bounds, 17), bounds, 17, 1, 2)
