"""Penalties, biases and grammars through the engine, beside requests that have none."""
import numpy as np
import pytest
import torch

import plain_draft_trees as plain
from helpers import random_tokens
from tffinfer_amd import EngineOptions, LLMEngine, SamplingConfig, log

pytestmark = pytest.mark.gpu


def packed(tokens, V):
    return plain.packed([tokens], -(-V // 32))[0].numpy()


def check_greedy(r, c, V, allowed=None):
    """Every token is the first maximum of the kept logits after the options, in float32 as the kernel rounds; where float64 finds two candidates
    closer than the rounding of a few operations (2^-20 of their size) either will do."""
    for i, (row, tok) in enumerate(zip(r.logits, r.output)):
        f = lambda x: float(torch.tensor(x, dtype=torch.float32))  # noqa: E731
        masks = None if allowed is None else [allowed(r.output[:i])]
        x, _ = plain.adjust(row.view(1, V).float(), [r.prompt + r.output[:i]], [len(r.prompt)], [f(c.repetition_penalty)], [f(c.presence_penalty)],
                            [f(c.frequency_penalty)], [[(t, f(b)) for t, b in (c.logit_bias or {}).items()]], masks,
                            None if masks is None else [0 if masks[0] is not None else -1])
        best = float(x.max())
        assert float(x[0, tok]) >= best - 2.0 ** -20 * max(1.0, abs(best)), (i, tok)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graphs", [True, False])
def test_options_through_the_engine(model_dirs, dtype, graphs):
    eng = LLMEngine.from_model_dir(model_dirs["A"], EngineOptions(dtype=dtype, kv_tokens=512, max_num_seqs=6, use_graphs=graphs))
    eng.keep_logits = True
    V = eng.model.config.vocab_size
    prompts = [random_tokens(n, V, 40 + n) for n in (4, 9, 17, 5, 6, 30)]
    even = list(range(0, V, 2))

    def alternate(out):
        return None if len(out) % 3 == 2 else (even if len(out) % 2 else list(range(1, V, 2)))
    configs = [SamplingConfig(), SamplingConfig(presence_penalty=3.0, frequency_penalty=0.5), SamplingConfig(logit_bias={7: 50.0, 3: -100.0}),
               SamplingConfig(repetition_penalty=1.7), SamplingConfig(allowed=lambda out: None if alternate(out) is None else packed(alternate(out), V)),
               SamplingConfig(repetition_penalty=1.2, frequency_penalty=1.0, logit_bias={11: 2.0}, allowed=lambda out: packed(even, V))]
    res = eng.generate(prompts, configs, max_new_tokens=20, ignore_eos=True)
    for r, c, a in zip(res, configs, (None, None, None, None, alternate, lambda out: even)):
        assert len(r.output) == 20
        check_greedy(r, c, V, a)
    assert set(res[2].output) == {7} and all(t % 2 == 0 for t in res[5].output)
    assert len(set(res[1].output)) > len(set(eng.generate([prompts[1]], max_new_tokens=20, ignore_eos=True)[0].output)) - 1
    # alone, and with the step ahead of a bias (which needs no output), the same tokens in float32
    if dtype == "float32":
        for p, c, r in zip(prompts, configs, res):
            alone = LLMEngine(eng.model, EngineOptions(dtype=dtype, kv_tokens=256, max_num_seqs=1, use_graphs=graphs))
            assert alone.generate([p], c, max_new_tokens=20, ignore_eos=True)[0].output == r.output
            assert (alone.steps_ahead > 0) == (not c.needs_output)


def test_a_draw_stays_within_the_grammar(model_dirs):
    eng = LLMEngine.from_model_dir(model_dirs["A"], EngineOptions(dtype="bfloat16", kv_tokens=256, max_num_seqs=3))
    V = eng.model.config.vocab_size
    few = [3, 40, V - 1]
    c = [SamplingConfig("random", temperature=2.0, seed=s, allowed=lambda out: packed(few, V), frequency_penalty=0.5) for s in (1, 2, 3)]
    for r in eng.generate([[1, 2], [5], [9, 9, 9]], c, max_new_tokens=24, ignore_eos=True):
        assert set(r.output) <= set(few) and len(set(r.output)) > 1
    none = eng.generate([[1, 2]], SamplingConfig(allowed=lambda out: np.zeros(-(-V // 32), dtype=np.int32)), max_new_tokens=3, ignore_eos=True)
    assert none[0].output == [0, 0, 0]


def test_a_grammar_that_fails_leaves_the_requests_where_they_stood(model_dirs):
    d = model_dirs["A"]
    eng = LLMEngine.from_model_dir(d, EngineOptions(dtype="float32", kv_tokens=256, max_num_seqs=2, page_size=8))
    V = eng.model.config.vocab_size
    fail = [False]

    def grammar(out):
        if fail[0]:
            raise RuntimeError("no grammar")
        return packed(range(0, V, 3), V)
    prompts = [[1, 2, 3, 4, 5], [8, 9]]
    configs = [SamplingConfig(allowed=grammar, repetition_penalty=1.3), SamplingConfig()]
    want = [r.output for r in eng.generate(prompts, configs, max_new_tokens=20, ignore_eos=True)]
    ids = [eng.add_request(p, c, 20, ignore_eos=True) for p, c in zip(prompts, configs)]
    steps = 0
    while eng.has_work:
        steps += 1
        if steps % 4 == 0:
            fail[0] = True
            with pytest.raises(RuntimeError, match="no grammar"):
                eng.step()
            fail[0] = False
        eng.step()
    assert [eng.pop_result(i).output for i in ids] == want
    assert all(g.pool.num_used == 0 for g in eng.runner.cache.groups)


def test_refusals(model_dirs):
    eng = LLMEngine.from_model_dir(model_dirs["A"], EngineOptions(dtype="float32", kv_tokens=64, max_num_seqs=1))
    V = eng.model.config.vocab_size
    with pytest.raises(ValueError, match="vocabulary"):
        eng.add_request([1], SamplingConfig(logit_bias={V: 1.0}))
    eng.add_request([1], SamplingConfig(allowed=lambda out: np.zeros(3, dtype=np.float32)))
    with pytest.raises(ValueError, match="allowed"):
        eng.step()


def test_penalties_change_what_is_generated(model_dirs):
    """A bias above any difference of two logits has one token come every time; a presence penalty above the two together lets none come twice, and a
    frequency penalty of a third of the bias lets that one come three times before any other."""
    eng = LLMEngine.from_model_dir(model_dirs["A"], EngineOptions(dtype="float32", kv_tokens=256, max_num_seqs=3))
    eng.keep_logits = True
    one = {7: 300.0}
    configs = [SamplingConfig(logit_bias=one), SamplingConfig(logit_bias=one, presence_penalty=1000.0),
               SamplingConfig(logit_bias=one, frequency_penalty=100.0)]
    same, once, thrice = eng.generate([[1, 2, 3]] * 3, configs, max_new_tokens=30, ignore_eos=True)
    assert max(float(row.max() - row.min()) for r in (same, once, thrice) for row in r.logits) < 100.0
    assert same.output == [7] * 30 and once.output[0] == 7 and len(set(once.output)) == 30
    assert thrice.output[:3] == [7] * 3 and set(thrice.output) != {7}


@pytest.mark.parametrize("how", ["raises", "wrong shape"])
def test_a_grammar_that_fails_says_whose_it_is(model_dirs, how):
    """The caller aborts that request, and the others end as they would have."""
    eng = LLMEngine.from_model_dir(model_dirs["A"], EngineOptions(dtype="float32", kv_tokens=256, max_num_seqs=3, page_size=8))
    V = eng.model.config.vocab_size

    def fine(out):
        return packed(range(1, V, 2), V)

    def grammar(out):
        if len(out) < 4:
            return packed(range(0, V, 3), V)
        if how == "wrong shape":
            return np.zeros(1, dtype=np.int32)
        raise KeyError("no state")
    prompts, kinds = [[1, 2, 3, 4, 5], [8, 9], [3]], [SamplingConfig(allowed=fine), SamplingConfig(allowed=grammar), SamplingConfig()]
    want = [r.output for r in eng.generate([prompts[0], prompts[2]], [kinds[0], kinds[2]], max_new_tokens=12, ignore_eos=True)]
    ids = [eng.add_request(p, c, 12, ignore_eos=True) for p, c in zip(prompts, kinds)]
    failures = 0
    while eng.has_work:
        try:
            eng.step()
        except (ValueError, KeyError) as e:
            failures += 1
            assert e.request_id == ids[1]
            eng.abort(ids[1])
    assert failures == 1
    assert [eng.pop_result(ids[0]).output, eng.pop_result(ids[2]).output] == want
    r = eng.pop_result(ids[1])
    assert len(r.output) == 4 and r.finish_reason != "length"
    assert all(g.pool.num_used == 0 for g in eng.runner.cache.groups)


def test_a_grammar_that_allows_nothing_is_told(model_dirs):
    """Token 0 stands where nothing was allowed; the result says where, the log says it once, and the other requests have nothing to tell."""
    eng = LLMEngine.from_model_dir(model_dirs["A"], EngineOptions(dtype="float32", kv_tokens=256, max_num_seqs=3))
    V = eng.model.config.vocab_size

    def dead_end(out):
        return packed([] if len(out) in (2, 3, 5) else range(1, V), V)
    before = log.counts()["W"]
    configs = [SamplingConfig(allowed=dead_end), SamplingConfig(), SamplingConfig(allowed=lambda out: packed([V - 1], V)),
               SamplingConfig("random", temperature=1.5, top_k=9, seed=4, allowed=dead_end), SamplingConfig("random", seed=5, allowed=dead_end)]
    got = eng.generate([[1, 2], [3], [4], [5], [6]], configs, max_new_tokens=8, ignore_eos=True)
    assert [r.unallowed for r in got] == [[2, 3, 5], [], [], [2, 3, 5], [2, 3, 5]]
    assert all([i for i, t in enumerate(got[r].output) if t == 0] == [2, 3, 5] for r in (0, 3, 4)) and got[2].output == [V - 1] * 8
    assert log.counts()["W"] == before + 3


def test_only_who_needs_its_tokens_has_them_gathered(model_dirs):
    """A bias alone asks for no history; a penalty and a grammar do."""
    eng = LLMEngine.from_model_dir(model_dirs["A"], EngineOptions(dtype="float32", kv_tokens=256, max_num_seqs=4))
    V = eng.model.config.vocab_size
    asked, history = [], eng._history
    eng._history = lambda r: asked.append(r.id) or history(r)
    configs = [SamplingConfig(logit_bias={5: 50.0}), SamplingConfig(frequency_penalty=0.5), SamplingConfig(),
               SamplingConfig(allowed=lambda out: packed([3], V))]
    ids = [eng.add_request([1, 2], c, 3, ignore_eos=True) for c in configs]
    while eng.has_work:
        eng.step()
    assert eng.pop_result(ids[0]).output == [5] * 3 and eng.pop_result(ids[3]).output == [3] * 3
    assert sorted(asked) == sorted([ids[1], ids[3]] * 3)
