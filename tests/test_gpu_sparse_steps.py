"""What a sequence's token reads does not follow from what the step's other sequences bring, nor from how a long step is cut into passes."""
import pytest
import torch

from tests.test_gpu_sparse import close, ids

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def models(model_dirs):
    from gophonic_b200.config import PageSelection
    from gophonic_b200.engine import Model
    memo = {}

    def get(name, dtype, pages=3):
        key = (name, dtype, pages)
        if key not in memo:
            memo[key] = Model.from_dir(model_dirs[name], dtype=dtype, selection=PageSelection(pages) if pages else None)
        return memo[key]
    return get


def engine_of(model, **kw):
    from gophonic_b200.engine import Engine
    return Engine(model, max_tokens=4096, **kw)


def fresh(eng, toks):
    slot = eng.new_sequence()
    eng.step([(slot, toks)])
    return slot


@pytest.mark.parametrize("name", ["A", "B", "D"])
@pytest.mark.parametrize("run", [2, 40, 150])
def test_a_single_token_beside_a_run(models, name, run):
    """The same logits as alone (float32: but for rounding), not those of a model that reads everything; the run's rows read everything."""
    eng, dense = engine_of(models(name, "float32")), engine_of(models(name, "float32", None))
    contexts = [ids(name, n, 30 + n) for n in (300, 30, 205)]
    more, extra = ids(name, 3, 40), ids(name, run, 41)
    got = {}
    for which in (eng, dense):
        slots = [fresh(which, t) for t in contexts]
        got[which, "alone"] = torch.cat([which.step([(s, [t])]) for s, t in zip(slots, more)])
        slots = [fresh(which, t) for t in contexts]
        other = fresh(which, contexts[0][:250])
        entries = [(slots[0], [more[0]]), (other, extra), (slots[1], [more[1]]), (slots[2], [more[2]])]
        got[which, "beside"] = which.step(entries, [[0], list(range(run)), [0], [0]])
        which.cache.check()
    mixed, alone = got[eng, "beside"], got[eng, "alone"]
    singles = torch.cat((mixed[:1], mixed[1 + run:]))
    assert close(singles, alone.cpu())
    assert not close(singles, got[dense, "alone"].cpu())
    assert close(mixed[1:1 + run], got[dense, "beside"][1:1 + run].cpu())


@pytest.mark.parametrize("most", [100, 150, 75, 300, 1])
def test_a_row_that_is_left_over_of_a_prompt_reads_everything(models, most):
    """A prompt of 301 tokens in passes of which the last holds one row: the logits that a reply begins with."""
    toks = ids("B", 301, 53)
    out = []
    for model, kw in ((models("B", "float32", None), {}), (models("B", "float32"), dict(max_rows_per_pass=most))):
        eng = engine_of(model, **kw)
        out.append(eng.step([(eng.new_sequence(), toks)], [[0, 299, 300]]))
    assert close(out[1], out[0].cpu())


@pytest.mark.parametrize("most", [100, 150, 75, 299, 1])
def test_the_last_row_of_a_prompt_reads_everything(models, most):
    """A prompt of 301 tokens in passes that leave one row over (or hold one each), beside another that begins with one row of a pass."""
    toks, other, single = ids("B", 301, 50), ids("B", 260, 51), ids("B", 280, 52)
    out = []
    for eng in (engine_of(models("B", "float32")), engine_of(models("B", "float32"), max_rows_per_pass=most)):
        c = fresh(eng, single[:279])
        a, b = eng.new_sequence(), eng.new_sequence()
        out.append(eng.step([(a, toks), (b, other), (c, single[279:])], [[299, 300], [0, 100, 259], [0]]))
        out.append(eng.step([(a, [5]), (b, [6])]))
        eng.cache.check()
    assert close(out[2], out[0].cpu()) and close(out[3], out[1].cpu())
    dense = engine_of(models("B", "float32", None))
    a, b = dense.new_sequence(), dense.new_sequence()
    assert close(out[2][:5], dense.step([(a, toks), (b, other)], [[299, 300], [0, 100, 259]]).cpu())


@pytest.mark.parametrize("name", ["A", "D"])
@pytest.mark.parametrize("runs", [[2], [70, 300]], ids=["two rows", "prompts"])
def test_a_mixed_step_in_bfloat16(models, name, runs):
    """One layer's attention over the same rows: a run's rows bit for bit as without the single tokens, single tokens as without the runs up to
    the rounding of their weights and of the result (a value's size times half a bfloat16 step each)."""
    from gophonic_b200.engine.step import build_batch
    eng = engine_of(models(name, "bfloat16"))
    mixer, cache = eng.model.blocks[0].mixer, eng.cache
    g = torch.Generator(device="cuda").manual_seed(7)
    extents = [(300, 1)] + [(200, n) for n in runs] + [(40, 1), (500, 1)]
    slots = [cache.alloc_slot() for _ in extents]
    cache.reserve([(slot, past + n) for slot, (past, n) in zip(slots, extents)])
    view = cache.view(0)
    view.k.normal_(generator=g)
    view.v.normal_(generator=g)
    rows = sum(n for _, n in extents)
    width = mixer.q_dim + 2 * mixer.kv_dim
    qkv = torch.randn((rows, width), generator=g, device="cuda").bfloat16()
    starts = [sum(n for _, n in extents[:i]) for i in range(len(extents))]
    for i, (past, _) in enumerate(extents):      # the bounds of what earlier steps filled
        batch, _ = build_batch([(slots[i], [0] * past, 0)], "cuda")
        mixer._bounds(batch, view)

    def run(which):
        batch, _ = build_batch([(slots[i], [0] * extents[i][1], extents[i][0]) for i in which], "cuda")
        mine = torch.cat([qkv[starts[i]:starts[i] + extents[i][1]] for i in which])
        return mixer._attend(batch, mine, view)
    every = list(range(len(extents)))
    mixed = run(every)
    runs_only = run([i for i in every if extents[i][1] > 1])
    longest = run([0, len(extents) - 1])
    at = starts[1]
    assert torch.equal(mixed[at:at + sum(runs)], runs_only)
    singles = torch.stack((mixed[0], mixed[-1]))
    assert float((singles.float() - longest.float()).abs().max()) <= 4 * 2.0 ** -8 * float(view.v.float().abs().max())
    eng.check_kernels()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["A", "D"])
def test_bounds_follow_the_keys_through_cuts(models, name, dtype):
    """Cut back and grown with other tokens, in runs, one by one and beside other sequences, also behind a restored mark: the bounds of every full
    page are the extremes of the keys that stand there, bit for bit."""
    eng = engine_of(models(name, dtype))
    toks, other = [ids(name, 460, 60 + i) for i in range(5)], fresh(eng, ids(name, 100, 70))

    def check(slot):
        n = eng.length(slot) // 64
        at = eng.cache.block_table[slot, :n].long()
        for pos in range(len(eng.model.blocks)):
            view = eng.cache.view(pos)
            k = view.k[at]
            assert torch.equal(view.bounds[at], torch.stack((k.amin(2), k.amax(2)), 2)), (pos, n)
    slot = fresh(eng, toks[0][:400])
    check(slot)
    mark = eng.checkpoint(slot)
    for t in toks[0][400:]:
        eng.step([(slot, [t])])
    check(slot)
    eng.truncate(slot, 100)
    eng.step([(slot, toks[1][100:250]), (other, [1])])
    check(slot)
    for t in toks[1][250:460]:
        eng.step([(slot, [t])])
    check(slot)
    eng.restore(slot, mark)
    for t in toks[2][400:]:
        eng.step([(slot, [t])])
    check(slot)
    eng.truncate(slot, 130)
    for i, t in enumerate(toks[3][130:260]):
        eng.step([(slot, [t]), (other, toks[4][2 * i:2 * i + 2])])
    check(slot)
    check(other)
    eng.cache.check()
