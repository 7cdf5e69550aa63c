"""Page selection in a model's description, in the cache and in the entry point's options: what needs no GPU."""
import pytest
import torch

import gophonic_b200 as g
from gophonic_b200.cache import Cache, CacheError
from gophonic_b200.config import AttentionSpec, PageSelection, PugalixConfig, SparseAttentionSpec, with_page_selection
from gophonic_b200.config.presets import preset
from gophonic_b200.parts.base import KVRequest
from gophonic_b200.weights import declare_model
from tests.conftest import tiny_configs


@pytest.mark.parametrize("kw", [dict(pages=2), dict(pages=4, last=0), dict(pages=4, first=-1), dict(pages=5, first=3, last=3), dict(pages=0)])
def test_a_selection_that_cannot_be(kw):
    with pytest.raises(ValueError):
        PageSelection(**kw)


def test_the_layers_change_and_nothing_else():
    spec = tiny_configs()["B"].model_spec()
    sel = PageSelection(5, first=2, last=1, prompts=True)
    got = with_page_selection(spec, sel)
    assert [d.name for d in declare_model(got)] == [d.name for d in declare_model(spec)]
    for a, b in zip(spec.layers, got.layers):
        assert type(b.mixer) is SparseAttentionSpec and b.mixer.kind == "sparse_attention" and b.mixer.selection == sel
        assert (b.mixer.heads, b.mixer.kv_heads, b.mixer.head_dim, b.mixer.scale, b.mixer.position, b.mixer.qk_norm) == (
            a.mixer.heads, a.mixer.kv_heads, a.mixer.head_dim, a.mixer.scale, a.mixer.position, a.mixer.qk_norm)
        assert b.feed_forward == a.feed_forward and b.prefix == a.prefix
    assert got.schedule == spec.schedule and got.head == spec.head
    got.validate()


def test_a_window_stays_and_a_model_without_such_layers_is_refused():
    import dataclasses
    spec = tiny_configs()["B"].model_spec()
    first = dataclasses.replace(spec.layers[0], mixer=dataclasses.replace(spec.layers[0].mixer, window=100))
    got = with_page_selection(dataclasses.replace(spec, layers=(first,) + spec.layers[1:]), PageSelection(4))
    assert type(got.layers[0].mixer) is AttentionSpec and type(got.layers[1].mixer) is SparseAttentionSpec
    raw = preset("pugalix-tiny")
    with pytest.raises(ValueError):
        with_page_selection(PugalixConfig.from_dict(raw).model_spec(), PageSelection(4))


def test_bounds_stand_beside_the_groups_that_ask():
    reqs = [(KVRequest(2, 16, bounds=True), None), (KVRequest(2, 16), None), (KVRequest(1, 16), None), (None, 0)]
    c = Cache(reqs, 256, "cpu", torch.float32, max_slots=2)
    assert tuple(c.view(0).bounds.shape) == (c.n_pages + 1, 2, 2, 16) and c.view(0).bounds.dtype == torch.float32
    assert c.view(1).bounds.data_ptr() != c.view(0).bounds.data_ptr()          # the same group, a plane of its own
    assert c.view(2).bounds is None
    assert c.view(3).bounds.data_ptr() == c.view(0).bounds.data_ptr() and not c.view(3).writable
    assert [gr["bytes_per_token"] for gr in c.groups()] == [2 * 2 * 2 * 16 * 4, 2 * 16 * 4]
    with pytest.raises(CacheError):
        c.keep_bounds(None)
    with pytest.raises(CacheError):
        Cache([(KVRequest(1, 16, value_dim=8, values_in_keys=True, bounds=True), None)], 64, "cpu", torch.float32)
    Cache([(KVRequest(1, 16), None)], 64, "cpu", torch.float32).keep_bounds(None)


@pytest.mark.parametrize("kw", [dict(SparsePages=-1), dict(SparsePages=2), dict(SparsePages=1025), dict(SparsePrompts=True)])
def test_options_refused(kw):
    with pytest.raises(ValueError):
        g.Open(g.random_model_path("tinyA"), g.Options(**kw))


def test_heads_that_the_kernels_take():
    ops = pytest.importorskip("gophonic_b200.ops")
    assert all(ops.page_attention_accepts(torch.bfloat16, d) for d in (16, 48, 64, 128, 256))
    assert not any(ops.page_attention_accepts(torch.bfloat16, d) for d in (0, 8, 24, 144, 512))
    assert all(ops.page_attention_accepts(torch.float32, d) for d in (4, 24, 128, 256)) and not ops.page_attention_accepts(torch.float32, 6)
