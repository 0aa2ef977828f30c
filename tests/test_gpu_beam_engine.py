"""A cache held in 4 bits under the engine, and beam search through its entry points, against the plain model: with its
keys and values brought to 4 bits and back, and by recomputing every hypothesis."""

import pytest
import torch

import plain_lfm2
import plain_packed
from mlx_one_b200 import BatchingConfig, CacheConfig, Engine, TextGenerationOptions
from mlx_one_b200.cache import CacheManager
from mlx_one_b200.engine.loading import load_model
from mlx_one_b200.engine.runner import Runner, StepEntry
from plain_beams import beam_search, same_hypotheses
from plain_lfm2 import PlainModel
from tiny_models import ALL_CONFIGS, assert_close, cut, make_model_dir, mixed_schedule, prompts, replay

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


class PackedPlain(PlainModel):
    """The plain model whose attention reads keys and values as a cache of 4 bits holds them."""

    def logits(self, token_ids):
        return self._with(lambda q, k, v, window: (through(k)[0], through(v)[0]), super().logits, token_ids)

    def logits_from(self, token_ids, held, dtype):
        """The same over the keys and values that an engine's cache held, layer by layer ``held[layer]`` =
        [2, tokens, heads, dim]. They have to be what the plain model's own become in 4 bits, but where the
        projections' rounding decides. 32 bits: values are off by about 2^-20 of themselves. That turns a
        value's code where the value lies so near a border, 2^-20 * 15 * 2 of them, and a group's lowest value
        or step, whose bfloat16 borders are 2^-8 apart, in 2^-11 of the groups: of 64 values together at most
        0.3 % of the groups, of the 150 of a call 0.4; three and one in a hundred more are allowed (more come
        up once in 10^3 calls), by a step or those numbers' 2^-8. bfloat16: keys and values are off by
        several 2^-8 of the group's largest, and a code by that and a step. What went the other way does
        not count against the logits, which are computed over the engine's own."""
        layers = iter(held)

        def taken(q, k, v, window):
            mine = next(layers)
            for rows, engine in ((k, mine[0]), (v, mine[1])):
                own, step = through(rows)
                off, size = (engine - own).abs(), rows.abs().amax(-1, keepdim=True)
                if dtype == F32:
                    groups = plain_packed.groups_of(rows.shape[-1])
                    turned = (off > 1e-4 * own.abs() + 1e-5).view(-1, rows.shape[-1] // groups).any(-1)
                    assert turned.sum() <= 3 + 0.01 * turned.numel(), int(turned.sum())
                    assert (off <= 1.1 * step + 2.0 ** -7 * size).all()
                else:
                    assert (off <= 1.5 * step + 0.05 * size).all(), float((off - 1.5 * step - 0.05 * size).max())
            return mine[0], mine[1]

        return self._with(taken, super().logits, token_ids)

    def _with(self, change, logits, token_ids):
        plain = plain_lfm2.causal_attention
        plain_lfm2.causal_attention = lambda q, k, v, window=None: plain(q, *change(q, k, v, window), window)
        try:
            return logits(token_ids)
        finally:
            plain_lfm2.causal_attention = plain


def through(x):
    """x [tokens, heads, dim] to 4 bits and back, and the step of every value."""
    rows = x.reshape(-1, x.shape[-1])
    code, step, low = plain_packed.quantized(rows)
    wide = step.repeat_interleave(x.shape[-1] // step.shape[1], 1)
    return plain_packed.values_of(code, step, low).float().view(x.shape), wide.float().view(x.shape)


class Recorder:
    """Reads back what every packing call of an engine's steps wrote: {request: [layer][2, tokens, heads, dim]}."""

    def __init__(self, ops, monkeypatch, layers):
        self.layers, self.calls = layers, []
        pack = ops.pack_key_values

        def both(keys, values, *, ctx, view):
            pack(keys, values, ctx=ctx, view=view)
            read = torch.stack(ops.read_key_values(ctx=ctx, view=view, dtype=F32)).cpu()
            self.calls.append((ctx.token_request.tolist(), read))

        monkeypatch.setattr(ops, "pack_key_values", both)

    def held(self, steps):
        """``steps``: for each step the requests in their order."""
        out = {}
        for number, requests in enumerate(steps):
            for layer in range(self.layers):
                owner, read = self.calls[number * self.layers + layer]
                for r, request in enumerate(requests):
                    mine = [t for t, o in enumerate(owner) if o == r]
                    out.setdefault(request, [[] for _ in range(self.layers)])[layer].append(read[:, mine])
        return {request: [torch.cat(parts, 1) for parts in layers] for request, layers in out.items()}


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = tmp_path_factory.mktemp("models")
    return {(name, dtype): make_model_dir(name, root, dtype=dtype) for name in ("B", "D", "MID") for dtype in (F32, BF16)}


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name,page", [("B", 16), ("D", 16), ("D", 32), ("MID", 64)])
def test_portions_and_decodes(folders, name, page, dtype, monkeypatch):
    """A whole prompt, token by token, in portions, and in steps that mix several requests."""
    folder = folders[name, dtype]
    loaded = load_model(folder, dtype, DEVICE)
    plain = PackedPlain(folder)
    vocab, kinds = ALL_CONFIGS[name][0]["vocab_size"], ALL_CONFIGS[name][0]["layer_types"]
    cache = CacheManager(loaded.model.cache_needs, page_size=page, capacity_tokens=2048, max_requests=8, dtype=dtype,
                         device=DEVICE, bits=4)
    runner = Runner(loaded.model, cache)
    runner.use_graphs = False
    recorder = Recorder(loaded.model.ops, monkeypatch, sum("attention" in kind for kind in kinds))

    def check(steps, requests):
        recorder.calls.clear()
        got = replay(runner, cache, steps)
        held = recorder.held([[request for request, _ in entries] for entries, _ in steps])
        for request, tokens in requests.items():
            assert_close(got[request], plain.logits_from(tokens, held[request], dtype), dtype, str(request))

    (tokens,) = prompts(vocab, (150,), seed=2)
    check([([("w", tokens)], ["w"])], {"w": tokens})
    check([([("d", tokens[:50])], [])] + [([("d", [t])], ["d"] if i == 99 else []) for i, t in enumerate(tokens[50:])],
          {"d": tokens})
    steps = [([("p", part)], []) for part in cut(tokens, (7, 2, 33, 1, 16, 5))]
    steps[-1] = (steps[-1][0], ["p"])
    check(steps, {"p": tokens})
    requests = dict(enumerate(prompts(vocab, (40, 90, 13, 66, 5, 33), seed=4)))
    check(mixed_schedule(requests), requests)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_steps_and_stale_pages(folders, dtype):
    """Steps replayed as graphs, in fresh pages and in pages that other requests have used: the same bits. (Steps
    that are not captured may cut the keys into other parts: they know the requests' true lengths.)"""
    loaded = load_model(folders["D", dtype], dtype, DEVICE)
    requests = prompts(301, (60, 45, 77, 30), seed=6)
    results = []
    for dirty in (False, True):
        cache = CacheManager(loaded.model.cache_needs, page_size=16, capacity_tokens=512, max_requests=4, dtype=dtype,
                             device=DEVICE, bits=4)
        runner = Runner(loaded.model, cache)
        if dirty:
            for group in cache.paged:
                group.storage.fill_(0xFF)                 # (steps and lowest values that are no numbers)
        collected = []
        for i, tokens in enumerate(requests):
            cache.open(i)
            collected.append(runner.step([StepEntry(i, tokens[:-14], (len(tokens) - 15,))]).clone())
        for step in range(14):
            entries = [StepEntry(i, [tokens[len(tokens) - 14 + step]], (0,)) for i, tokens in enumerate(requests)]
            collected.append(runner.step(entries).clone())
        assert runner.graph_replays >= 10
        results.append(torch.cat(collected))
        loaded.model.ops.check_errors()
    assert not torch.isnan(results[0]).any() and torch.equal(*results)


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("name,beams,new", [("D", 4, 40), ("MID", 3, 24), ("B", 5, 20), ("D", 1, 30)])
def test_beam_search(folders, name, beams, new, bits):
    """Over pages of 32-bit values and of 4 bits: hypotheses, scores, and every page given back. (A near tie
    between hypotheses, or a code on its border, may go either way: then another prompt is taken.)"""
    folder = folders[name, F32]
    vocab = ALL_CONFIGS[name][0]["vocab_size"]
    plain = PackedPlain(folder) if bits else PlainModel(folder)
    engine = Engine(folder, execution_dtype="float32",
                    cache_config=CacheConfig(block_size_tokens=16, capacity_tokens=2048, max_requests=8, bits=bits),
                    batching_config=BatchingConfig(max_sequences=8, prefill_chunk_size=32))
    tried = 0
    for seed in range(8):
        (prompt,) = prompts(vocab, (21 + 9 * seed,), seed=seed)
        want = beam_search(plain.logits, prompt, beams, new, ())
        if want is None:
            continue
        got = engine.generate_beams_ids(prompt, TextGenerationOptions(max_tokens=new, ignore_eos=True), beams=beams)
        assert sorted((r.score for r in got), reverse=True)[0] >= max(c[1] for c in want) - 1e-2
        if bits is None or [r.token_ids for r in got] == [c[0] for c in sorted(want, key=lambda c: -c[1])]:
            same_hypotheses(got, want)
            tried += 1
            break
    assert tried == 1
    stats = engine.cache.stats()
    assert stats.pages_free == stats.pages_total and stats.requests == 0
    engine.close()


def test_beams_beside_requests(folders):
    """A search between the steps of running requests changes none of their tokens."""
    folder = folders["D", BF16]
    (one, two, three) = prompts(301, (40, 33, 70), seed=9)
    config = dict(cache_config=CacheConfig(block_size_tokens=16, capacity_tokens=2048, max_requests=8, bits=4),
                  batching_config=BatchingConfig(max_sequences=4))
    with Engine(folder, **config) as engine:
        want = [r.token_ids for r in engine.generate_batch_ids([one, two], TextGenerationOptions(max_tokens=40, ignore_eos=True))]
        alone = engine.generate_beams_ids(three, max_tokens=20, beams=4, ignore_eos=True)
    with Engine(folder, **config) as engine:
        handles = [engine.submit_ids(p, max_tokens=40, ignore_eos=True) for p in (one, two)]
        for _ in range(9):
            engine.step()
        got = engine.generate_beams_ids(three, max_tokens=20, beams=4, ignore_eos=True)
        assert [(r.token_ids, r.score) for r in got] == [(r.token_ids, r.score) for r in alone]
        assert [h.result().token_ids for h in handles] == want
        assert engine.cache_bytes_per_token() * 3.5 < sum(
            4 * need.kv_heads * need.head_dim for need in engine.model.cache_needs.values() if hasattr(need, "kv_heads"))


def test_a_search_that_fails_leaves_the_engine_usable(folders):
    """A token outside the vocabulary is refused by the step function; the next search starts afresh."""
    (prompt,) = prompts(301, (20,), seed=4)
    with Engine(folders["D", BF16], cache_config=CacheConfig(block_size_tokens=16, capacity_tokens=1024, max_requests=4,
                                                             bits=4)) as engine:
        want = [(r.token_ids, r.score) for r in engine.generate_beams_ids(prompt, max_tokens=9, beams=3)]
        with pytest.raises(ValueError, match="vocabulary"):
            engine.generate_beams_ids([*prompt, 301 + 40], max_tokens=9, beams=3)
        assert engine.cache.stats().requests == 0
        assert [(r.token_ids, r.score) for r in engine.generate_beams_ids(prompt, max_tokens=9, beams=3)] == want


ARCHITECTURES = [("galarax", "G1"), ("galarax", "G3"), ("galarax", "G5"), ("farorax", "F1"), ("farorax", "F6"),
                 ("lamisun", "L1"), ("lamisun", "L4"), ("tirudra", "T1"), ("tirudra", "T5"), ("susalorn", None),
                 ("zinizen", None)]


def rescored(engine, prompt, tokens):
    """The sum of the tokens' logarithms when prompt and tokens run through the step function at once."""
    cache, runner = engine.cache, engine.runner
    whole = list(prompt) + list(tokens)
    cache.open("again")
    logits = runner.step([StepEntry("again", whole[:-1], range(len(prompt) - 1, len(whole) - 1))])
    cache.close("again")
    logs = torch.log_softmax(logits.double(), -1)
    return float(logs[torch.arange(len(tokens)), list(tokens)].sum())


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("family,name", ARCHITECTURES)
def test_every_kind_of_state_follows_its_hypothesis(tmp_path, family, name, bits):
    """Delta rules, lightning and latent attention, convolutions, state spaces, recurrences, hashes of neighbouring
    tokens: a hypothesis has the score that its tokens get when they run at once, and one hypothesis is greedy
    decoding. With 4 bits, models whose pages are keys and values of 32, 64, 96 or 128; others are refused."""
    import importlib

    module = importlib.import_module(family + "_models")
    name = name or list(module.CONFIGS)[0]
    config = module.CONFIGS[name][0]
    folder = module.make_model_dir(name, tmp_path)
    how = dict(execution_dtype="float32", cache_config=CacheConfig(block_size_tokens=16, capacity_tokens=2048,
                                                                   max_requests=6, bits=bits),
               batching_config=BatchingConfig(max_sequences=2, prefill_chunk_size=16))
    try:
        engine = Engine(folder, **how)
    except ValueError as error:
        assert bits == 4 and ("held in 4 bits" in str(error) or "32, 64, 96 or 128" in str(error))
        return
    vocab = engine.model.spec.vocab_size
    (prompt,) = prompts(vocab, (37,), seed=3)
    greedy = engine.generate_ids(prompt, max_tokens=12, ignore_eos=True).token_ids
    found = engine.generate_beams_ids(prompt, max_tokens=12, ignore_eos=True, beams=1)
    assert found[0].token_ids == greedy
    found = engine.generate_beams_ids(prompt, max_tokens=20, ignore_eos=True, beams=min(4, vocab))
    assert len({r.token_ids for r in found}) == len(found)
    for result in found:
        # 32 bits: 20 logarithms, each within the engine's 1e-4; 4 bits: a code may go either way between
        # the two runs, by which a token's logarithm moves by a few 1e-3
        assert abs(rescored(engine, prompt, result.token_ids) - result.score) <= (4e-3 if bits is None else 0.2), config
    stats = engine.cache.stats()
    assert stats.pages_free == stats.pages_total and stats.requests == 0
    engine.close()
