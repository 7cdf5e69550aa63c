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


@pytest.mark.parametrize("most", [100, 150, 75, 300, 1])
def test_a_row_that_is_left_over_of_a_prompt_reads_everything(models, most):
    """A prompt of 301 tokens in passes of which the last holds one row: the logits that a reply begins with."""
    toks = ids("B", 301, 53)
    out = []
    for model, kw in ((models("B", "float32", None), {}), (models("B", "float32"), dict(max_rows_per_pass=most))):
        eng = engine_of(model, **kw)
        out.append(eng.step([(eng.new_sequence(), toks)], [[0, 299, 300]]))
    assert close(out[1], out[0].cpu())
