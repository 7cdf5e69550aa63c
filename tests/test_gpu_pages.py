"""page_bounds, select_pages and attention_pages against their restatement in 64 bits."""
import math

import pytest
import torch

from tests.plain import pages_plain as P

pytestmark = pytest.mark.gpu

PAGE = 64
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from gophonic_b200 import ops as o
    return o


class Step:
    """Sequences in a paged cache of shuffled pages: keys and values by position, planes, table and the rows' metadata."""

    def __init__(self, seqs, heads, kvh, d, dtype, seed=0, junk=0.0, room=0, more_rows=0, spread=0.4):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.heads, self.kvh, self.d, self.dtype = seqs, heads, kvh, d, dtype
        held = [max(1, -(-(a + b) // PAGE)) for a, b in seqs]
        self.n_pages = sum(held) + 2
        width = max(held) + room
        order = torch.randperm(self.n_pages, generator=g)
        shape = (self.n_pages, kvh, PAGE, d)
        self.k_plane = torch.full(shape, junk, dtype=dtype)
        self.v_plane = torch.full(shape, junk, dtype=dtype)
        self.slots = [int(s) for s in torch.randperm(len(seqs) + 2, generator=g)[:len(seqs)]]
        self.table = torch.zeros((len(seqs) + 2, width), dtype=torch.int32)
        self.keys, self.values, self.starts = [], [], []
        at = row = 0
        for (past, new), slot, n in zip(seqs, self.slots, held):
            self.table[slot, :n] = order[at:at + n].to(torch.int32)
            at += n
            # the keys of a page are alike in part, so that pages score differently
            topic = torch.randn((n, kvh, 1, d), generator=g) * spread
            k = (torch.randn((n, kvh, PAGE, d), generator=g) + topic).to(dtype)
            v = torch.randn((n, kvh, PAGE, d), generator=g).to(dtype)
            self.keys.append(k.transpose(1, 2).reshape(-1, kvh, d)[:past + new])
            self.values.append(v.transpose(1, 2).reshape(-1, kvh, d)[:past + new])
            for j in range(n):
                m = min(PAGE, past + new - j * PAGE)
                self.k_plane[self.table[slot, j], :, :m] = k[j, :, :m]
                self.v_plane[self.table[slot, j], :, :m] = v[j, :, :m]
            self.starts.append(row)
            row += new
        self.rows = row
        wide = torch.randn((row + more_rows, (heads + 2 * kvh) * d), generator=g).to(dtype)
        self.wide = wide.to(DEV)
        self.q = wide[:, :heads * d]
        self.meta()

    def meta(self):
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
        self.seq = (ints(self.slots), ints(self.starts), ints([b for _, b in self.seqs]), ints([a + b for a, b in self.seqs]))
        self.nseq, self.max_q = len(self.seqs), max(b for _, b in self.seqs)
        self.dev = {n: getattr(self, n).to(DEV) for n in ("k_plane", "v_plane", "table")}
        self.q_dev = self.wide[:, :self.heads * self.d]

    def bounds_plane(self, fill=0.0):
        """The bounds of all full pages, as earlier steps and this one have left them; ``fill`` elsewhere."""
        out = torch.full((self.n_pages, self.kvh, 2, self.d), fill, dtype=self.dtype)
        for slot, keys in zip(self.slots, self.keys):
            b = P.bounds_of(keys)
            out[self.table[slot, :b.shape[0]].long()] = b
        return out

    def select(self, ops, bounds, top, first=1, last=2, fill=-7):
        pages = torch.full((self.q.shape[0], self.kvh, top), fill, dtype=torch.int32, device=DEV)
        slot, start, q_len, kv_len = self.seq
        ops.select_pages(self.q_dev, bounds.to(DEV), self.dev["table"], slot, start, q_len, kv_len, self.nseq, self.max_q, self.heads, self.kvh,
                         self.d, pages, first, last)
        return pages

    def attend(self, ops, pages, out=None):
        if out is None:
            out = torch.full((self.q.shape[0], self.heads * self.d), 9.0, dtype=self.dtype, device=DEV)
        slot, start, q_len, kv_len = self.seq
        ops.attention_pages(self.q_dev, out, self.dev["k_plane"], self.dev["v_plane"], self.dev["table"], slot, start, q_len, kv_len, self.nseq,
                            self.max_q, self.heads, self.kvh, self.d, self.d ** -0.5, pages)
        return out

    def each_row(self):
        for i, (past, new) in enumerate(self.seqs):
            for j in range(new):
                yield i, past + j, self.starts[i] + j


BF, F32 = torch.bfloat16, torch.float32
GEOMETRIES = [(BF, 4, 2, 128), (BF, 14, 2, 64), (BF, 5, 1, 48), (BF, 32, 1, 128), (BF, 2, 2, 256), (BF, 3, 3, 16), (BF, 8, 8, 128), (BF, 8, 1, 112),
              (F32, 4, 2, 128), (F32, 14, 2, 64), (F32, 5, 1, 24), (F32, 20, 1, 128), (F32, 2, 1, 256)]
names = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None


# ---- page_bounds -------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,heads,kvh,d", [(BF, 2, 2, 128), (BF, 1, 1, 8), (BF, 3, 3, 24), (BF, 1, 1, 256), (BF, 1, 1, 200), (F32, 2, 2, 128),
                                               (F32, 1, 1, 4), (F32, 3, 3, 20), (F32, 1, 1, 256)], ids=names)
@pytest.mark.parametrize("seqs", [[(0, 1)], [(63, 1), (64, 1), (62, 1), (127, 1)], [(0, 64), (0, 63), (0, 65), (5, 200), (60, 4), (64, 64)], [(1, 700)]],
                         ids=["one", "tokens", "mixed", "long"])
def test_page_bounds(ops, dtype, heads, kvh, d, seqs):
    s = Step(seqs, heads, kvh, d, dtype, seed=d, junk=math.nan)
    bounds = torch.full((s.n_pages, kvh, 2, d), 5.0, dtype=dtype, device=DEV)
    slot, _, q_len, kv_len = s.seq
    ops.page_bounds(s.dev["k_plane"], bounds, s.dev["table"], slot, q_len, kv_len, s.nseq, s.max_q)
    want = torch.full_like(bounds, 5.0).cpu()
    for (past, new), sl, keys in zip(seqs, s.slots, s.keys):
        b = P.bounds_of(keys)
        for j in range(past // PAGE, (past + new) // PAGE):
            want[s.table[sl, j]] = b[j]
    assert torch.equal(bounds.cpu(), want)


def test_page_bounds_of_several_planes(ops):
    s = Step([(0, 130), (60, 10)], 2, 2, 64, BF)
    planes = torch.stack([s.dev["k_plane"], -s.dev["k_plane"], s.dev["k_plane"] * 0.5])
    bounds = torch.zeros((3, s.n_pages, 2, 2, 64), dtype=BF, device=DEV)
    one = torch.zeros_like(bounds)
    slot, _, q_len, kv_len = s.seq
    ops.page_bounds(planes, bounds, s.dev["table"], slot, q_len, kv_len, s.nseq, s.max_q)
    for i in range(3):
        ops.page_bounds(planes[i], one[i], s.dev["table"], slot, q_len, kv_len, s.nseq, s.max_q)
    assert torch.equal(bounds, one) and bool((one != 0).any())
    assert torch.equal(one[0, :, :, 0], -one[1, :, :, 1])


@pytest.mark.parametrize("dtype", [BF, F32], ids=names)
def test_page_bounds_carry_nan_and_infinities(ops, dtype):
    s = Step([(0, 64)], 1, 1, 16, dtype)
    page = int(s.table[s.slots[0], 0])
    k = s.dev["k_plane"]
    k[page, 0, 17, 3] = math.nan
    k[page, 0, 40, 5] = math.inf
    k[page, 0, 63, 6] = -math.inf
    bounds = torch.zeros((s.n_pages, 1, 2, 16), dtype=dtype, device=DEV)
    slot, _, q_len, kv_len = s.seq
    ops.page_bounds(k, bounds, s.dev["table"], slot, q_len, kv_len, 1, 64)
    b = bounds[page, 0].cpu()
    assert b[:, 3].isnan().all() and b[1, 5] == math.inf and b[0, 6] == -math.inf
    others = [c for c in range(16) if c not in (3, 5, 6)]
    ref = k[page, 0][:, others].cpu()
    assert torch.equal(b[:, others], torch.stack((ref.amin(0), ref.amax(0))))


# ---- select_pages ------------------------------------------------------------------------------
def check_selection(s, pages, bounds, top, first, last):
    got = pages.cpu().tolist()
    for i, pos, row in s.each_row():
        n = pos // PAGE + 1
        b = bounds[s.table[s.slots[i], :n].long()]
        score = P.scores(s.q[row].reshape(s.heads, s.d), b)
        for g in range(s.kvh):
            want = P.choose(score[g], n - 1, top, first, last)
            assert got[row][g] == want + [-1] * (top - len(want)), (i, pos, g)


@pytest.mark.parametrize("dtype,heads,kvh,d", GEOMETRIES + [(BF, 3, 1, 8), (BF, 2, 2, 40), (F32, 3, 1, 4)], ids=names)
@pytest.mark.parametrize("seqs,top,first,last", [
    ([(0, 1)], 4, 1, 2), ([(700, 1), (64 * 5 - 1, 1), (64 * 5, 1), (2, 1)], 5, 1, 2), ([(0, 400)], 4, 1, 2), ([(1000, 30), (333, 5), (10, 70)], 6, 2, 1),
    ([(1500, 3)], 3, 0, 3), ([(1500, 3)], 1, 0, 1), ([(1500, 3)], 23, 5, 17), ([(1500, 3)], 24, 1, 1), ([(1500, 3)], 40, 1, 1)],
    ids=["first", "tokens", "prompt", "turns", "none free", "own alone", "all but one", "all", "more than all"])
def test_select_pages(ops, dtype, heads, kvh, d, seqs, top, first, last):
    s = Step(seqs, heads, kvh, d, dtype, seed=heads * 7 + d, more_rows=2, room=3)
    bounds = s.bounds_plane(fill=math.nan)     # what no full page has may be anything
    pages = s.select(ops, bounds, top, first, last)
    check_selection(s, pages, bounds, top, first, last)
    assert (pages[s.rows:] == -7).all()


def wide_step(dtype, pages, heads=2, kvh=1, d=128, new=2):
    return Step([(pages * PAGE - new + 1, new)], heads, kvh, d, dtype, seed=pages)


@pytest.mark.parametrize("dtype,new", [(BF, 2), (F32, 2), (BF, 40), (BF, 12)], ids=names)
@pytest.mark.parametrize("pages", [300, 1400, 3300])
def test_select_pages_long(ops, dtype, new, pages):
    """Clusters of single rows; tiles of 32 rows, of 16, and contexts too long for either."""
    s = wide_step(dtype, pages, new=new)
    bounds = s.bounds_plane()
    check_selection(s, s.select(ops, bounds, 33), bounds, 33, 1, 2)


@pytest.mark.parametrize("dtype,pages,top", [(BF, 4600, 33), (F32, 4600, 90), (BF, 600, 90), (F32, 1000, 70), (BF, 4600, 4500)], ids=names)
def test_select_pages_by_all_warps(ops, dtype, pages, top):
    """Candidates in a few registers a thread, in many, and from shared memory; more wanted than a warp has lanes."""
    s = wide_step(dtype, pages, d=16)
    bounds = s.bounds_plane()
    check_selection(s, s.select(ops, bounds, top), bounds, top, 1, 2)
    bounds[s.table[s.slots[0]].long()] = bounds[s.table[s.slots[0], 3].long()].clone()
    check_selection(s, s.select(ops, bounds, top), bounds, top, 1, 2)


@pytest.mark.parametrize("dtype", [BF, F32], ids=names)
@pytest.mark.parametrize("equal", [True, False])
def test_select_pages_of_many_sequences(ops, dtype, equal):
    """More single tokens than run at once: the longest begin first, and every one gets its own."""
    g = torch.Generator().manual_seed(1)
    seqs = [(640 if equal else int(torch.randint(1, 900, (1,), generator=g)), 1) for _ in range(90)]
    s = Step(seqs, 4, 2, 16, dtype, seed=5, more_rows=1)
    bounds = s.bounds_plane()
    pages = s.select(ops, bounds, 5)
    check_selection(s, pages, bounds, 5, 1, 2)
    assert (pages[s.rows:] == -7).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=names)
@pytest.mark.parametrize("kind", ["equal", "few kinds", "zero query", "one ulp", "nan", "inf", "huge", "tiny", "nan query", "inf query", "cancel"])
@pytest.mark.parametrize("pages,new,d", [(40, 2, 128), (700, 2, 128), (40, 21, 128), (300, 9, 128), (300, 21, 48), (300, 9, 16), (100, 30, 64), (100, 9, 256), (300, 2, 48)])
def test_select_pages_near_the_border(ops, dtype, kind, pages, new, d):
    """Scores that tie, that differ in the last place of one channel, that float32 cannot hold: the choice is the 64-bit one."""
    s = wide_step(dtype, pages, new=new, d=d)
    g = torch.Generator().manual_seed(pages)
    bounds = s.bounds_plane()
    n = s.table.shape[1]
    mine = s.table[s.slots[0]].long()
    if kind == "equal":
        bounds[mine] = bounds[mine[3]].clone()
    elif kind == "few kinds":
        bounds[mine] = bounds[mine[torch.randint(0, 4, (n,), generator=g)]].clone()
    elif kind == "one ulp":
        bounds[mine] = bounds[mine[3]].clone()
        for j in range(n):
            c = int(torch.randint(0, s.d, (1,), generator=g))
            x = bounds[mine[j], 0, 1, c]
            bounds[mine[j], 0, 1, c] = x * (1 + torch.finfo(dtype).eps)
    elif kind in ("nan", "inf"):
        for j in range(0, n, 3):
            bounds[mine[j], 0, j % 2, j % s.d] = math.nan if kind == "nan" else (-math.inf, math.inf)[j % 2]
    elif kind == "huge":
        bounds[mine] = (bounds[mine].float() * 1e38).to(dtype)
    elif kind == "tiny":
        bounds[mine] = (bounds[mine].float() * 1e-30).to(dtype)
        s.wide.copy_((s.wide.float() * 1e-12).to(dtype))
    elif kind == "zero query":
        s.wide.zero_()
    elif kind in ("nan query", "inf query"):
        s.wide[0, 5] = math.nan if kind == "nan query" else math.inf
    elif kind == "cancel":      # large terms that take one another off
        s.wide[:, 0], s.wide[:, 1] = 1.0, 1.0
        bounds[mine, 0, 1, 0] = 1e6
        bounds[mine, 0, 1, 1] = -1e6
    s.q = s.wide[:, :s.heads * s.d].cpu()
    check_selection(s, s.select(ops, bounds, 17), bounds, 17, 1, 2)


# ---- attention_pages ---------------------------------------------------------------------------
def random_lists(s, top, seed, empty=False):
    """Pages of each row's past in random number, ascending, then -1; every fifth row none if ``empty``."""
    g = torch.Generator().manual_seed(seed)
    pages = torch.full((s.q.shape[0], s.kvh, top), -1, dtype=torch.int32)
    for i, pos, row in s.each_row():
        own = pos // PAGE
        for h in range(s.kvh):
            if empty and (row + h) % 5 == 2:
                continue
            m = 1 + int(torch.randint(0, min(top, own + 1), (1,), generator=g))
            pick = torch.randperm(own + 1, generator=g)[:m].sort().values
            pages[row, h, :m] = pick.to(torch.int32)
    return pages


def check_attention(s, out, pages, rows=None):
    """Errors: the weights are rounded to bfloat16 (half a step, 2^-8) before they meet the values, the result once more; sums of
    float32 terms.  A score's float32 error is at most (d + 8) 2^-24 of the sum of its terms' sizes, and moves a weight by as much,
    relative; exponentials and sums add some 2^-18."""
    got = out.cpu().double().reshape(out.shape[0], -1)[:, :s.heads * s.d].reshape(-1, s.heads, s.d)
    listed = pages.cpu().tolist()
    half = 2.0 ** -8 if s.dtype == BF else 2.0 ** -24
    for i, pos, row in s.each_row():
        if rows is not None and row not in rows:
            continue
        q = s.q[row].reshape(s.heads, s.d)
        want, size = P.attend(q, s.keys[i], s.values[i], listed[row], pos, s.d ** -0.5)
        terms = q.double().abs().sum(1).max() * s.keys[i].double().abs().max() * s.d ** -0.5
        slack = 2 * (s.d + 8) * 2.0 ** -24 * float(terms) + 2.0 ** -17
        tol = size * ((half if s.dtype == BF else 0.0) + slack) * (1 + half) + want.abs() * half + 1e-30
        bad = (got[row] - want).abs() > tol
        assert not bad.any(), (i, pos, float(((got[row] - want).abs() / tol).max()))


@pytest.mark.parametrize("dtype,heads,kvh,d", GEOMETRIES, ids=names)
@pytest.mark.parametrize("seqs,top", [([(0, 1)], 4), ([(700, 1), (64 * 5 - 1, 1), (64 * 5, 1), (2, 1)], 5), ([(0, 70), (130, 3)], 4), ([(1000, 9), (333, 1)], 11),
                                      ([(1500, 1)], 24)], ids=["first", "tokens", "prompt", "turns", "full"])
def test_attention_pages(ops, dtype, heads, kvh, d, seqs, top):
    s = Step(seqs, heads, kvh, d, dtype, seed=heads + d, junk=math.nan, more_rows=3, room=2)
    pages = random_lists(s, top, seed=heads, empty=True)
    out = s.attend(ops, pages.to(DEV))
    check_attention(s, out, pages)
    assert (out[s.rows:] == 9.0).all()
    for i, pos, row in s.each_row():
        for g in range(kvh):
            if int(pages[row, g].max()) < 0:
                G = heads // kvh
                assert (out[row, g * G * d:(g + 1) * G * d] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32], ids=names)
def test_attention_pages_passes_over_entries_that_name_nothing(ops, dtype):
    s = Step([(300, 1), (80, 2)], 4, 2, 64, dtype, junk=math.nan, room=4)
    pages = torch.full((3, 2, 6), -1, dtype=torch.int32)
    pages[0, 0] = torch.tensor([-1, 0, -5, 2, 4, 7])       # 7 lies behind the row's own page
    pages[0, 1] = torch.tensor([5, 6, 7, -1, -1, -1])
    pages[1, 0] = torch.tensor([0, 1, 2, 1000000, -1, -1])
    pages[1, 1] = torch.tensor([1, -1, -1, -1, -1, -1])
    pages[2, 0] = torch.tensor([2 ** 31 - 1, -2 ** 31, -1, -1, -1, -1])
    pages[2, 1] = torch.tensor([0, 1, -1, -1, -1, -1])
    out = s.attend(ops, pages.to(DEV))
    plain = pages.clone()
    for row, own in ((0, 4), (1, 1), (2, 1)):
        plain[row][plain[row] > own] = -1
    check_attention(s, out, plain)


@pytest.mark.parametrize("dtype", [BF, F32], ids=names)
@pytest.mark.parametrize("top", [4, 24])
def test_attention_pages_single_rows_beside_what_is_not_finite(ops, dtype, top):
    """NaN keys and infinite values of listed pages come through, also where a row sees nothing else; those of others do not."""
    s = Step([(1500, 1), (1500, 1), (1500, 1), (1500, 1)], 4, 2, 64, dtype, seed=6)
    pages = torch.full((4, 2, top), -1, dtype=torch.int32)
    pages[0, :, 0] = 5
    pages[1, :, :4] = torch.tensor([1, 5, 7, 23])
    pages[2, :, :4] = torch.tensor([1, 9, 11, 23])
    pages[3, :, :2] = torch.tensor([2, 3])
    for i, (plane, page, value) in enumerate([("k_plane", 5, math.nan), ("k_plane", 5, math.nan), ("v_plane", 9, -math.inf), ("v_plane", 4, math.nan)]):
        s.dev[plane][s.table[s.slots[i], page]] = value
    # behind the row's position, in its own page
    for i in range(4):
        s.dev["v_plane"][s.table[s.slots[i], 23], :, 1500 % PAGE + 1:] = math.nan
        s.dev["k_plane"][s.table[s.slots[i], 23], :, 1500 % PAGE + 1:] = math.nan
    out = s.attend(ops, pages.to(DEV)).cpu()
    assert out[0].isnan().all() and out[1].isnan().all() and (out[2] == -math.inf).all() and out[3].isfinite().all()
    check_attention(s, out, pages, rows={3})


def test_all_pages_equal_full_attention(ops):
    """Lists of everything: what the attention over the whole cache gives, up to the rounding of the weights."""
    s = Step([(500, 1), (63, 1), (1000, 1)], 8, 2, 128, BF, seed=3)
    top = 16
    pages = s.select(ops, s.bounds_plane(), top)
    out = s.attend(ops, pages)
    full = torch.empty_like(out)
    slot, start, q_len, kv_len = s.seq
    ops.attention(s.q_dev, full, s.dev["k_plane"], s.dev["v_plane"], s.dev["table"], slot, start, q_len, kv_len, s.nseq, 1, 8, 2, 128, 128 ** -0.5)
    assert float((out.float() - full.float()).abs().max()) <= 2 * 2.0 ** -8 * float(s.v_plane.float().abs().max())


# ---- runs of rows on the tcgen05 kernel ---------------------------------------------------------
def like_lists(s, top, seed, span, pool):
    """Lists of rows that follow one another, nearly alike: every ``span`` rows a new set of ``pool`` pages, of which a row takes some."""
    g = torch.Generator().manual_seed(seed)
    pages = torch.full((s.q.shape[0], s.kvh, top), -1, dtype=torch.int32)
    sets = {}
    for i, pos, row in s.each_row():
        own = pos // PAGE
        for h in range(s.kvh):
            key = (i, h, row // span)
            if key not in sets:
                sets[key] = torch.randperm(own + 1, generator=g)[:pool]
            some = sets[key][torch.rand(len(sets[key]), generator=g) < 0.6].tolist()
            pick = sorted(set([own] + some))[-top:]
            pages[row, h, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
    return pages


@pytest.mark.parametrize("heads,kvh", [(2, 2), (4, 2), (3, 1), (4, 1), (7, 1), (16, 2), (20, 1), (128, 1)])
@pytest.mark.parametrize("seqs,top", [([(0, 16)], 4), ([(0, 150)], 5), ([(900, 70), (333, 1), (0, 33)], 9), ([(63, 2), (2000, 17)], 12)],
                         ids=["least", "prompt", "three", "behind"])
def test_attention_pages_runs(ops, heads, kvh, seqs, top):
    s = Step(seqs, heads, kvh, 128, BF, seed=heads, more_rows=2, room=1)
    pages = like_lists(s, top, heads, 12, 10)
    out = s.attend(ops, pages.to(DEV))
    assert ops.tc5_status() == 0
    check_attention(s, out, pages, rows=set(range(0, s.rows, 3 if s.rows * heads > 500 else 1)) | {s.rows - 1})
    assert (out[s.rows:] == 9.0).all()


def test_attention_pages_runs_with_empty_lists(ops):
    s = Step([(500, 40), (0, 20)], 4, 1, 128, BF, seed=1)
    pages = random_lists(s, 6, 3, empty=True)
    pages[5:30] = -1
    out = s.attend(ops, pages.to(DEV))
    check_attention(s, out, pages)
    assert (out[5:30] == 0).all()
    out = s.attend(ops, torch.full_like(pages, -1).to(DEV))
    assert (out == 0).all() and ops.tc5_status() == 0


@pytest.mark.parametrize("heads,kvh,new", [(4, 1, 150), (16, 8, 700)], ids=["shared tiles", "whole tiles"])
@pytest.mark.parametrize("where", ["unlisted page", "another row's page", "behind the last token", "later token", "keys"])
def test_attention_pages_runs_beside_values_that_are_not_finite(ops, heads, kvh, new, where):
    """What a row does not see does not reach it, be it Inf or NaN; what it sees does."""
    s = Step([(1000, new)], heads, kvh, 128, BF, seed=2, junk=math.nan if where == "behind the last token" else 0.0)
    pages = like_lists(s, 8, 5, 12, 9)
    clean = s.attend(ops, pages.to(DEV)).clone()
    if where == "behind the last token":
        assert (1000 + new) % PAGE
        check_attention(s, clean, pages, rows={0, 3, new - 1, new - 2})
        return
    target = s.dev["k_plane"] if where == "keys" else s.dev["v_plane"]
    mine = s.table[s.slots[0]]
    if where == "later token":
        pos = 1000 + new - 1
        target[mine[pos // PAGE], :, pos % PAGE] = math.nan
        sees = torch.zeros((new, kvh), dtype=torch.bool)
        sees[new - 1] = (pages[new - 1] == pos // PAGE).any(-1)
    else:
        page = 3 if where != "unlisted page" else 1
        if where == "unlisted page":
            pages[pages == page] = -1
            clean = s.attend(ops, pages.to(DEV)).clone()
        target[mine[page]] = math.inf if where == "another row's page" else math.nan
        sees = (pages == page).any(-1)
        assert where == "unlisted page" or (sees.any() and not sees.all())
    out = s.attend(ops, pages.to(DEV))
    G = heads // kvh
    got, ref = out.cpu().float().reshape(new, kvh, G * 128), clean.cpu().float().reshape(new, kvh, G * 128)
    assert not got[sees].isfinite().any()
    # the others: the same up to the rounding of the weights
    assert float((got[~sees] - ref[~sees]).abs().max()) <= 4 * 2.0 ** -8 * float(s.v_plane.float().abs().max())
    assert got[~sees].isfinite().all() and ops.tc5_status() == 0


@pytest.mark.parametrize("width", [4000, 31500, 32768])
@pytest.mark.parametrize("dtype", [BF, F32], ids=names)
def test_wide_block_tables(ops, dtype, width):
    """Sequences that could be millions of tokens long: what stands in shared memory goes by the table's width."""
    for seqs in ([(1500, 1), (90, 1)], [(1500, 40), (90, 1)]):
        held = max(-(-(a + b) // PAGE) for a, b in seqs)
        s = Step(seqs, 8, 4, 128, dtype, seed=9, room=width - held)
        bounds = s.bounds_plane()
        pages = s.select(ops, bounds, 9)
        check_selection(s, pages, bounds, 9, 1, 2)
        check_attention(s, s.attend(ops, pages), pages, rows={0, 1, 20, s.rows - 1})


def test_attention_pages_behind_tables_too_wide_to_select_from(ops):
    s = Step([(900, 30)], 4, 4, 128, BF, seed=9, room=40000)
    pages = like_lists(s, 8, 5, 12, 9)
    check_attention(s, s.attend(ops, pages.to(DEV)), pages, rows={0, 7, 29})
    with pytest.raises(ops.KernelError):
        s.select(ops, s.bounds_plane(), 8)


# ---- the three together ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,heads,kvh,d", [(BF, 8, 2, 128), (BF, 6, 3, 32), (F32, 8, 2, 64)], ids=names)
def test_a_sequence_in_steps(ops, dtype, heads, kvh, d):
    """A context evaluated in portions of odd sizes: bounds, selection and attention of every step as over the whole."""
    total = [(0, 150), (150, 1), (151, 40), (191, 1), (192, 1), (193, 300), (493, 1)]
    whole = Step([(494, 1)], heads, kvh, d, dtype, seed=4)
    bounds = torch.zeros((whole.n_pages, kvh, 2, d), dtype=dtype, device=DEV)
    for past, new in total:
        s = whole
        s.seqs = [(past, new)]
        g = torch.Generator().manual_seed(past)
        s.wide = torch.randn((new, (heads + 2 * kvh) * d), generator=g).to(dtype).to(DEV)
        s.q, s.rows = s.wide[:, :heads * d].cpu(), new
        s.meta()
        slot, _, q_len, kv_len = s.seq
        ops.page_bounds(s.dev["k_plane"], bounds, s.dev["table"], slot, q_len, kv_len, 1, new)
        pages = s.select(ops, bounds, 4)
        check_selection(s, pages, bounds.cpu(), 4, 1, 2)
        out = s.attend(ops, pages)
        check_attention(s, out, pages)


@pytest.mark.parametrize("dtype", [BF, F32], ids=names)
def test_captured_on_another_stream_and_repeated(ops, dtype):
    """The three captured into a graph on a stream of their own: the replay follows inputs changed in place, bit for bit."""
    s = Step([(700, 1), (639, 1), (1300, 1)], 8, 2, 64, dtype, seed=8)
    bounds = s.bounds_plane().to(DEV)
    pages = torch.zeros((3, 2, 6), dtype=torch.int32, device=DEV)
    out = torch.zeros((3, 8 * 64), dtype=dtype, device=DEV)
    slot, start, q_len, kv_len = s.seq

    def call():
        ops.page_bounds(s.dev["k_plane"], bounds, s.dev["table"], slot, q_len, kv_len, 3, 1)
        ops.select_pages(s.q_dev, bounds, s.dev["table"], slot, start, q_len, kv_len, 3, 1, 8, 2, 64, pages)
        ops.attention_pages(s.q_dev, out, s.dev["k_plane"], s.dev["v_plane"], s.dev["table"], slot, start, q_len, kv_len, 3, 1, 8, 2, 64, 0.125, pages)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            call()
    for seed in (1, 2):
        g = torch.Generator(device=DEV).manual_seed(seed)
        s.wide.copy_(torch.randn(s.wide.shape, generator=g, device=DEV).to(dtype))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = (pages.clone(), out.clone())
        for _ in range(3):
            call()
            torch.cuda.synchronize()
            assert torch.equal(pages, got[0]) and torch.equal(out, got[1])


def test_two_streams_at_once(ops):
    """Calls that overlap share nothing: runs, single tokens and float32 beside one another give what they give alone."""
    steps = [Step([(2000, 300)], 8, 2, 128, BF, seed=1), Step([(3000, 1), (500, 1)], 8, 2, 128, BF, seed=2), Step([(1500, 20)], 4, 2, 64, F32, seed=3)]
    alone = []
    for s in steps:
        pages = s.select(ops, s.bounds_plane(), 8)
        alone.append((pages, s.attend(ops, pages)))
    bounds = [s.bounds_plane().to(DEV) for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, b, stream in zip(steps, bounds, streams):
            with torch.cuda.stream(stream):
                pages = s.select(ops, b, 8)
                got.append((pages, s.attend(ops, pages)))
        torch.cuda.synchronize()
        for (p0, o0), (p1, o1) in zip(alone, got):
            assert torch.equal(p0, p1) and torch.equal(o0, o1)


def test_sequences_that_bring_nothing(ops):
    """A padded batch: sequences of no rows between others."""
    s = Step([(700, 3), (300, 0), (0, 0), (500, 40)], 4, 2, 128, BF, seed=4, more_rows=2)
    bounds = s.bounds_plane()
    out_bounds = torch.full((s.n_pages, 2, 2, 128), 5.0, dtype=BF, device=DEV)
    slot, _, q_len, kv_len = s.seq
    ops.page_bounds(s.dev["k_plane"], out_bounds, s.dev["table"], slot, q_len, kv_len, 4, 40)
    done = int(s.table[s.slots[3], 7])
    assert torch.equal(out_bounds[done].cpu(), bounds[done]) and int((out_bounds != 5.0).flatten(1).any(1).sum()) == 1
    pages = s.select(ops, bounds, 5)
    check_selection(s, pages, bounds, 5, 1, 2)
    check_attention(s, s.attend(ops, pages), pages)
    assert (pages[s.rows:] == -7).all()


# ---- refusals ----------------------------------------------------------------------------------
def test_refusals(ops):
    s = Step([(100, 1)], 4, 2, 64, BF)
    slot, start, q_len, kv_len = s.seq
    bounds = s.bounds_plane().to(DEV)
    pages = torch.zeros((1, 2, 4), dtype=torch.int32, device=DEV)
    out = torch.zeros((1, 256), dtype=BF, device=DEV)
    k, v, table = s.dev["k_plane"], s.dev["v_plane"], s.dev["table"]

    def bad(fn):
        with pytest.raises(ops.KernelError):
            fn()
    select = lambda q=s.q_dev, b=bounds, t=table, p=pages, heads=4, kvh=2, d=64, sl=slot, **kw: ops.select_pages(
        q, b, t, sl, start, q_len, kv_len, 1, 1, heads, kvh, d, p, **kw)
    attend = lambda q=s.q_dev, o=out, kk=k, vv=v, p=pages, heads=4, kvh=2, d=64: ops.attention_pages(
        q, o, kk, vv, table, slot, start, q_len, kv_len, 1, 1, heads, kvh, d, 0.125, p)
    select(), attend()
    bad(lambda: select(first=3, last=2))
    bad(lambda: select(last=0))
    bad(lambda: select(first=-1))
    bad(lambda: select(heads=3))
    bad(lambda: select(b=bounds.float()))
    bad(lambda: select(b=bounds.transpose(2, 3)))
    bad(lambda: select(p=pages.long()))
    bad(lambda: select(p=pages[:, :1]))
    bad(lambda: select(q=s.q_dev.cpu()))
    bad(lambda: select(q=s.q_dev.half()))
    bad(lambda: select(sl=slot.long()))
    bad(lambda: select(sl=slot[:0]))
    bad(lambda: select(t=torch.zeros((3, 32769), dtype=torch.int32, device=DEV)))
    bad(lambda: attend(kk=k.float()))
    bad(lambda: attend(vv=v[:, :1]))
    bad(lambda: attend(o=out.float()))
    bad(lambda: attend(o=out[:, :128]))
    bad(lambda: attend(p=torch.zeros((1, 2, 1025), dtype=torch.int32, device=DEV)))
    bad(lambda: attend(p=torch.zeros((2, 2, 4), dtype=torch.int32, device=DEV)))
    bad(lambda: ops.page_bounds(k, bounds.float(), table, slot, q_len, kv_len, 1, 1))
    bad(lambda: ops.page_bounds(k, bounds[:, :1].contiguous(), table, slot, q_len, kv_len, 1, 1))
    bad(lambda: ops.page_bounds(k[0], bounds, table, slot, q_len, kv_len, 1, 1))
    odd = torch.zeros((4, 1, 64, 20), dtype=BF, device=DEV)
    bad(lambda: ops.page_bounds(odd, torch.zeros((4, 1, 2, 20), dtype=BF, device=DEV), table, slot, q_len, kv_len, 1, 1))
    shifted = torch.zeros(257, dtype=BF, device=DEV)[1:].view(1, 256)
    bad(lambda: attend(q=shifted))


def test_zz_no_kernel_met_a_bad_index_or_gave_up(ops):
    """Behind all of the above: no wait ran out and (in the checked build) no index left its bounds."""
    assert ops.tc5_status() == 0 and ops.checked_status() is None
