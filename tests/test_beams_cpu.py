"""Beam search through the engine's entry points, caches that change owners, and a cache of 4 bits' bookkeeping, with
plain kernels on the CPU."""

import json
import math

import pytest
import torch
from click.testing import CliRunner

from mlx_one_b200 import BatchingConfig, BeamResult, CacheConfig, Engine, TextGenerationOptions
from mlx_one_b200.cache import CacheCapacityError, CacheManager, CacheOwnershipError
from mlx_one_b200.engine.loading import load_model
from mlx_one_b200.parts.base import FixedState, PackedView, PagedKeyValues, PagedView
from plain_beams import BeamOps, beam_search, same_hypotheses
from plain_lfm2 import PlainModel
from tiny_models import CONFIGS, make_model_dir, prompts


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    root = tmp_path_factory.mktemp("models")
    out = {}
    for name in ("A", "C"):
        folder = make_model_dir(name, root, dtype=torch.float32)
        out[name] = (folder, load_model(folder, "float32", "cpu", ops=BeamOps()), PlainModel(folder))
    return out


def engine_of(loaded, page=4, capacity=1024, requests=6, **config):
    return Engine(loaded, cache_config=CacheConfig(block_size_tokens=page, capacity_tokens=capacity, max_requests=requests),
                  batching_config=BatchingConfig(max_sequences=requests, prefill_chunk_size=7, max_scheduled_tokens=16, **config))


@pytest.mark.parametrize("name", ["A", "C"])
@pytest.mark.parametrize("beams,length,new", [(1, 5, 6), (2, 12, 5), (4, 23, 7), (6, 40, 4)])
def test_hypotheses_are_those_of_a_plain_search(models, name, beams, length, new):
    """Convolution state, pages, a window that gives pages back; prompts in portions."""
    folder, loaded, plain = models[name]
    engine = engine_of(loaded, CONFIGS[name][2])
    vocab = CONFIGS[name][0]["vocab_size"]
    for seed in range(3):
        (prompt,) = prompts(vocab, (length,), seed=seed)
        want = beam_search(plain.logits, prompt, beams, new, ())
        if want is not None:
            break
    got = engine.generate_beams_ids(prompt, TextGenerationOptions(max_tokens=new, ignore_eos=True), beams=beams)
    same_hypotheses(got, want)
    if beams == 1:
        assert list(got[0].token_ids) == plain.greedy(prompt, new)
    assert engine.cache.stats().pages_free == engine.cache.stats().pages_total
    engine.cache.check()
    engine.close()


@pytest.mark.parametrize("penalty", [0.0, 1.0, 3.0])
def test_hypotheses_that_end(models, penalty):
    """Tokens that end a hypothesis: it competes as it is, its score and text keep the end token out."""
    folder, loaded, plain = models["A"]
    (prompt,) = prompts(512, (9,), seed=3)
    free = beam_search(plain.logits, prompt, 3, 6, ())
    spec = loaded.spec
    before = spec.eos_token_ids
    ends = (free[0][0][2], free[1][0][4])
    object.__setattr__(spec, "eos_token_ids", ends)
    try:
        engine = engine_of(loaded)
        want = beam_search(plain.logits, prompt, 3, 12, ends)
        got = engine.generate_beams_ids(prompt, max_tokens=12, beams=3, length_penalty=penalty)
        same_hypotheses(got, want, penalty)
        assert any(r.finish_reason == "stop" for r in got)
        engine.close()
    finally:
        object.__setattr__(spec, "eos_token_ids", before)


def test_beside_other_requests(models):
    """A search in the middle of a request: both get what they would get alone."""
    folder, loaded, plain = models["A"]
    one, two = prompts(512, (11, 8), seed=5)
    for pipelined in (False, True):
        engine = engine_of(loaded, pipeline_decode=pipelined)
        handle = engine.submit_ids(one, max_tokens=10, ignore_eos=True)
        for _ in range(5):
            engine.step()
        got = engine.generate_beams_ids(two, max_tokens=5, ignore_eos=True, beams=3)
        same_hypotheses(got, beam_search(plain.logits, two, 3, 5, ()))
        assert list(handle.result().token_ids) == plain.greedy(one, 10)
        engine.close()


def test_searches_that_are_refused(models):
    engine = engine_of(models["A"][1], capacity=64, requests=3)
    for options in (dict(temperature=0.5), dict(top_k=3), dict(top_p=0.5), dict(stop=("x",))):
        with pytest.raises(ValueError, match="no sampling"):
            engine.generate_beams_ids([1, 2], **options)
    for beams in (0, 33, 2.0, True):
        with pytest.raises(ValueError, match="beams"):
            engine.generate_beams_ids([1, 2], beams=beams)
    with pytest.raises(ValueError, match="prompt"):
        engine.generate_beams_ids([], beams=2)
    with pytest.raises(CacheCapacityError):
        engine.generate_beams_ids([1, 2], beams=4, max_tokens=4)          # three requests
    with pytest.raises(CacheCapacityError):
        engine.generate_beams_ids([1, 2], beams=3, max_tokens=30)         # 96 tokens of 64
    engine.cache.check()
    assert engine.cache.stats().requests == 0
    assert len(engine.generate_beams_ids([1, 2], beams=3, max_tokens=4)) == 3
    engine.close()


def test_command_line(models, monkeypatch):
    import mlx_one_b200.engine as engines
    from mlx_one_b200.cli import main

    folder, loaded, plain = models["A"]
    seen = {}

    def make(model, **how):
        seen.update(how)
        return Engine(loaded, cache_config=how.get("cache_config"))

    monkeypatch.setattr(engines, "Engine", make)
    call = ["generate", str(folder), "5 17 3", "--token-ids", "--max-tokens", "4", "--dtype", "float32"]
    want = beam_search(plain.logits, [5, 17, 3], 3, 4, ())
    result = CliRunner().invoke(main, call + ["--beams", "3"])
    assert result.exit_code == 0, result.output
    best = max(want, key=lambda c: c[1])
    assert [int(v) for v in result.output.split()] == list(best[0])
    result = CliRunner().invoke(main, call + ["--beams", "3", "--json-output"])
    rows = json.loads(result.output)
    assert [tuple(r["token_ids"]) for r in rows][0] == best[0] and len(rows) == 3 and rows[0]["score"] < 0
    assert CliRunner().invoke(main, call + ["--beams", "3", "--stream"]).exit_code != 0
    monkeypatch.setattr(engines, "Engine", lambda model, **how: (_ for _ in ()).throw(ValueError(str(how["cache_config"].bits))))
    result = CliRunner().invoke(main, call + ["--cache-bits", "4"])
    assert "4" in result.output and result.exit_code != 0


def test_penalties_and_searches_without_an_answer(models, monkeypatch):
    import mlx_one_b200.engine as engines
    from mlx_one_b200.cli import main

    folder, loaded, plain = models["A"]
    engine = engine_of(loaded)
    for penalty in (math.nan, math.inf, -11, 300.0):
        with pytest.raises(ValueError, match="length_penalty"):
            engine.generate_beams_ids([1, 2], beams=2, length_penalty=penalty)
    for penalty in (-10, 0, 10.0):
        assert len(engine.generate_beams_ids([1, 2], beams=2, max_tokens=3, length_penalty=penalty)) == 2
    monkeypatch.setattr(engine, "generate_beams_ids", lambda *a, **how: [])
    monkeypatch.setattr(engines, "Engine", lambda model, **how: engine)
    result = CliRunner().invoke(main, ["generate", str(folder), "5 17", "--token-ids", "--beams", "2"])
    assert result.exit_code == 1 and "finite score" in result.output
    engine.close()


# ------------------------------------------------------------------ the cache


def manager(bits=None, page=16, more=(), capacity=128):
    needs = {0: PagedKeyValues(2, 64), 1: PagedKeyValues(2, 64), 2: PagedKeyValues(1, 128, 20), 3: FixedState((3, 5))}
    return CacheManager({**needs, **dict(more)}, page_size=page, capacity_tokens=capacity, max_requests=4,
                        dtype=torch.float32, device="cpu", bits=bits)


def test_storage_in_4_bits():
    cache = manager(4, 32)
    assert [tuple(g.storage.shape) for g in cache.paged] == [(2, 5, 2, 2, 2, 576), (1, 5, 1, 2, 2, 1152)]
    assert all(g.storage.dtype == torch.uint8 for g in cache.paged)
    cache.open("a")
    cache.grow("a", 40)
    view = cache.view(1, [torch.zeros(1, 2, dtype=torch.int32)] * 2, [torch.zeros(1, dtype=torch.int32)])
    assert isinstance(view, PackedView) and view.kv.shape == (5, 2, 2, 2, 576) and view.page_size == 32
    assert isinstance(manager().view(1, [torch.zeros(1, 2, dtype=torch.int32)] * 2, []), PagedView)


@pytest.mark.parametrize("bits,page,more,message", [
    (8, 16, {}, "4 bits"), (4, 8, {}, "16, 32, 64 or 128"), (4, 16, {7: PagedKeyValues(1, 80)}, "32, 64, 96 or 128"),
    (4, 16, {7: PagedKeyValues(1, 64, planes=1)}, "rows per token")])
def test_caches_that_have_no_4_bits(bits, page, more, message):
    with pytest.raises(ValueError, match=message):
        manager(bits, page, more)


def test_configurations_that_are_refused(models):
    for wrong in (dict(bits=8), dict(bits=4, block_size_tokens=8)):
        with pytest.raises(ValueError, match="bits"):
            CacheConfig(**wrong)
    with pytest.raises(ValueError, match="32, 64, 96 or 128"):          # (heads of 16)
        Engine(models["A"][1], cache_config=CacheConfig(bits=4, capacity_tokens=64))


def test_owners_change(models):
    """Pages and slots go to new owners, behind the first position that differs; lengths must agree."""
    cache, ops = manager(capacity=256), BeamOps()
    names = ["a", "b", "c"]
    for name in names:
        cache.open(name)
    for group in list(cache.paged) + list(cache.states):
        group.storage.copy_(torch.randn(group.storage.shape))
    order = cache.order_of(names)
    for step, first in ((24, 0), (1, 24), (1, 24), (16, 24)):
        for name in names:
            cache.grow(name, step)
            cache.advance(name, step)
        held = [[g.storage.clone() for g in kind] for kind in (cache.paged, cache.states)]
        order.apply(ops, torch.tensor([1, 1, 0], dtype=torch.int32), first)
        caches = [cache.get(name) for name in names]
        for g, (group, before) in enumerate(zip(cache.paged, held[0])):
            want = before.clone()
            for b, parent in ((0, 1), (2, 0)):
                for block in range(first // 16, -(-caches[0].length // 16)):
                    if caches[b].tables[g][block] >= 0:
                        want[:, :, caches[b].tables[g][block]] = before[:, :, caches[parent].tables[g][block]]
            assert torch.equal(group.storage, want)
        for g, (group, before) in enumerate(zip(cache.states, held[1])):
            slots = [c.slots[g] for c in caches]
            want = before.clone()
            want[:, slots[0]], want[:, slots[2]] = before[:, slots[1]], before[:, slots[0]]
            assert torch.equal(group.storage, want)
    cache.grow("a", 1)
    cache.advance("a", 1)
    with pytest.raises(CacheOwnershipError, match="different lengths"):
        order.apply(ops, torch.tensor([0, 1, 2], dtype=torch.int32))
