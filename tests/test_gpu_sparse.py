"""Models whose tokens read selected pages, through the engine: against the plain model with the same selection, against the model that
reads everything, and against themselves (captured, in portions, cut back)."""
import numpy as np
import pytest
import torch

from tests.conftest import tiny_configs
from tests.plain import pages_plain as Pages
from tests.plain import qwen3_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def engine(model_dirs):
    from gophonic_b200.config import PageSelection
    from gophonic_b200.engine import Engine, Model
    memo = {}

    def get(name, dtype, pages=None, graphs=True, **kw):
        key = (name, dtype, pages, graphs, tuple(kw.items()))
        if key not in memo:
            sel = PageSelection(pages, **kw) if pages else None
            memo[key] = Engine(Model.from_dir(model_dirs[name], dtype=dtype, selection=sel), max_tokens=4096, use_graphs=graphs)
        return memo[key]
    return get


def plain_attention(selection, tokens_from):
    """The plain model's attention with a selection: rows at positions >= tokens_from select."""
    def attend(q, k, v, scale, window=0):
        full = FULL(q, k, v, scale, window)
        T, heads, d = q.shape
        kt, vt = torch.from_numpy(k), torch.from_numpy(v)
        bounds = Pages.bounds_of(kt)
        for i in range(tokens_from, T):
            own = i // 64
            if own + 1 <= selection.pages:
                continue
            b = torch.cat((bounds, bounds.new_zeros((1,) + bounds.shape[1:])))[:own + 1]      # the row's own page may not be full
            score = Pages.scores(torch.from_numpy(q[i]), b)
            listed = [Pages.choose(score[g], own, selection.pages, selection.first, selection.last) for g in range(k.shape[1])]
            full[i] = Pages.attend(torch.from_numpy(q[i]), kt, vt, listed, i, scale)[0].numpy()
        return full
    return attend


FULL = P.causal_attention


def ids(name, n, seed):
    return np.random.default_rng(seed).integers(0, tiny_configs()[name].vocab_size, size=n).tolist()


def close(got, ref):
    """float32 logits: every row to 2e-4 of the reference's spread."""
    got, ref = got.double().cpu().numpy(), np.asarray(ref)
    return np.abs(got - ref).max() <= 2e-4 * max(1.0, np.abs(ref).max())


@pytest.mark.parametrize("name", ["A", "B", "D", "F"])
@pytest.mark.parametrize("prompts,n", [(False, 250), (True, 250), (False, 100)])
def test_against_the_plain_model(engine, plain_models, monkeypatch, name, prompts, n):
    """A prompt, then tokens one by one past several page borders, also past the one from which on they select; in float32, where no
    selection is near enough a tie to flip."""
    eng = engine(name, "float32", 3, prompts=prompts)
    sel = eng.model.spec.layers[0].mixer.selection
    toks = ids(name, 319, 5)
    cfg, w = plain_models[name]
    monkeypatch.setattr(P, "causal_attention", plain_attention(sel, 0 if prompts else n))
    ref = P.forward_logits(toks, cfg, w)
    slot = eng.new_sequence()
    got = [eng.step([(slot, toks[:n])], [[0, n // 2, n - 1]])]
    got += [eng.step([(slot, [t])]) for t in toks[n:]]
    eng.end_sequence(slot)
    assert close(torch.cat(got), np.concatenate((ref[[0, n // 2, n - 1]], ref[n:])))
    monkeypatch.setattr(P, "causal_attention", FULL)
    assert not close(torch.cat(got[1:]), P.forward_logits(toks, cfg, w)[n:])       # the selection shows


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "D"])
def test_contexts_that_are_read_in_full_give_the_same_bits(engine, name, dtype):
    dense, sparse = engine(name, dtype), engine(name, dtype, 6)
    toks = ids(name, 380, 7)
    out = []
    for eng in (dense, sparse):
        slot = eng.new_sequence()
        got = [eng.step([(slot, toks[:300])], [list(range(300))])] + [eng.step([(slot, [t])]) for t in toks[300:]]
        eng.end_sequence(slot)
        out.append(torch.cat(got))
    assert torch.equal(*out)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("prompts", [False, True])
def test_a_replayed_step_is_the_eager_one(engine, dtype, prompts):
    """Unequal sequences side by side, some of which are read in full; steps captured and not."""
    out = []
    for graphs in (True, False):
        eng = engine("D", dtype, 4, graphs=graphs, prompts=prompts)
        slots = [eng.new_sequence() for _ in range(3)]
        toks = [ids("D", n + 70, 20 + n) for n in (500, 260, 40)]
        got = [eng.step([(s, t[:-70]) for s, t in zip(slots, toks)])]
        for i in range(70, 0, -1):
            got.append(eng.step([(s, [t[-i]]) for s, t in zip(slots, toks)]))
        for s in slots:
            eng.end_sequence(s)
        eng.cache.check()
        out.append(torch.cat(got))
    assert torch.equal(*out)


def test_where_a_token_came_from_does_not_matter(engine):
    """With prompts that select too, a context in one prompt, in portions of odd sizes and token by token: the same logits but for
    rounding (float32)."""
    eng = engine("B", "float32", 3, prompts=True)
    toks = ids("B", 330, 9)
    out = []
    for cuts in ([330], [1, 64, 65, 200], list(range(150, 331))):
        slot = eng.new_sequence()
        at, got = 0, None
        for cut in cuts + ([330] if cuts[-1] != 330 else []):
            got = eng.step([(slot, toks[at:cut])])
            at = cut
        out.append(got)
        eng.end_sequence(slot)
    for other in out[1:]:
        assert float((other - out[0]).abs().max()) <= 2e-4 * max(1.0, float(out[0].abs().max()))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_cut_back_and_grown_again(engine, dtype):
    """The bounds of pages that were cut and filled with other tokens are those of the new ones."""
    eng = engine("D", dtype, 3)
    a, b = ids("D", 420, 1), ids("D", 420, 2)
    slot = eng.new_sequence()
    eng.step([(slot, a[:400])])
    mark = eng.checkpoint(slot)
    for t in a[400:]:
        eng.step([(slot, [t])])
    eng.truncate(slot, 100)
    eng.step([(slot, b[100:400])])
    got = [eng.step([(slot, [t])]) for t in b[400:]]
    eng.truncate(slot, 0)
    eng.step([(slot, a[:100] + b[100:400])])
    fresh = [eng.step([(slot, [t])]) for t in b[400:]]
    eng.end_sequence(slot)
    # the prompt in one piece or two: the same but for rounding
    worst = float((torch.cat(got) - torch.cat(fresh)).abs().max())
    if dtype == "float32":
        assert worst <= 2e-4 * max(1.0, float(torch.cat(fresh).abs().max()))
    slot = eng.new_sequence()
    eng.step([(slot, a[:400])])
    mark = eng.checkpoint(slot)
    first = [eng.step([(slot, [t])]) for t in a[400:]]
    eng.restore(slot, mark)
    again = [eng.step([(slot, [t])]) for t in a[400:]]
    eng.end_sequence(slot)
    assert torch.equal(torch.cat(first), torch.cat(again))


@pytest.mark.parametrize("fmt", ["bf16", "f32"])
def test_through_the_entry_point(model_dirs, fmt):
    import gophonic_b200 as g
    out = []
    for kw in (dict(), dict(SparsePages=3), dict(SparsePages=3, SparsePrompts=True), dict(SparsePages=12)):
        model = g.Open(model_dirs["B"], g.Options(Format=fmt, CacheTokens=4096, Batch=2, **kw))
        out.append(g.Lane(model, g.TokensGenerator).Generate([ids("B", 500, 3), ids("B", 30, 4)], g.ChatOptions(MaxTokens=40), stop_ids=[]))
        model.Close()
    assert [len(r) for replies in out for r in replies] == [40] * 8
    assert out[0] == out[3]                       # everything is read
    if fmt == "f32":      # the short context too, beside one that selects (another kernel: bfloat16 rounds its weights elsewhere)
        assert all(o[1] == out[0][1] for o in out)
    assert out[0][0] != out[1][0]


def test_heads_without_a_kernel_are_refused(model_dirs):
    from gophonic_b200.config import PageSelection
    from gophonic_b200.engine import Model
    with pytest.raises(ValueError):
        Model.from_dir(model_dirs["F"], dtype="bfloat16", selection=PageSelection(4))
