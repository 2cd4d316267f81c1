"""Options on the logits, on the host: what a SamplingConfig takes, which tables the sampler sends, what the command line reads."""
import argparse
import math
import types

import numpy as np
import pytest
import torch

from tffinfer_amd import cli
from tffinfer_amd.sampling import Sampler, SamplingConfig, TokenLog, allowed_mask, allows_none


def test_what_a_config_takes():
    c = SamplingConfig(presence_penalty=0.5, frequency_penalty=-0.25, logit_bias={"7": 2, 3: -math.inf})
    assert c.adjusts and c.needs_output and c.logit_bias == {7: 2.0, 3: -math.inf}
    assert not SamplingConfig().adjusts and not SamplingConfig().needs_output
    assert not SamplingConfig(repetition_penalty=1.2).adjusts and SamplingConfig(repetition_penalty=1.2).needs_output
    assert SamplingConfig(logit_bias={1: 1.0}).adjusts and not SamplingConfig(logit_bias={1: 1.0}).needs_output
    assert SamplingConfig(allowed=lambda out: None).needs_output and not SamplingConfig(logit_bias={}).adjusts
    for bad in (dict(presence_penalty=math.nan), dict(frequency_penalty=math.inf), dict(logit_bias={1: math.nan}), dict(logit_bias={1: math.inf}),
                dict(logit_bias={-1: 0.0}), dict(logit_bias={1 << 31: 0.0}), dict(allowed=5)):
        with pytest.raises(ValueError):
            SamplingConfig(**bad)


def test_a_grammars_answer():
    for kind in (np.int32, np.uint32):
        got = allowed_mask(SamplingConfig(allowed=lambda out: np.arange(3, dtype=kind)), np.zeros(0, np.int32), 70)
        assert got.dtype == np.int32 and got.tolist() == [0, 1, 2]
    assert allowed_mask(SamplingConfig(allowed=lambda out: None), np.zeros(0, np.int32), 70) is None
    for bad in (np.zeros(2, np.int32), np.zeros(3, np.int64), np.zeros((1, 3), np.int32)):
        with pytest.raises(ValueError):
            allowed_mask(SamplingConfig(allowed=lambda out: bad), np.zeros(0, np.int32), 70)


def test_a_log_that_grows():
    prompt, out = list(range(300)), []
    log = TokenLog(prompt)
    assert log.update(out).tolist() == prompt
    for i in range(2000):
        out.append(i * 3)
        if i % 7 == 0 or i > 1990:
            assert log.update(out).tolist() == prompt + out
    assert log.prompt_len == 300 and TokenLog([]).update([5]).tolist() == [5]


def test_the_tables_of_a_mixed_batch(monkeypatch):
    """Rows without options, with a repetition penalty alone (its distinct tokens do), with a bias alone (no tokens sent), with everything."""
    got = {}

    def adjust(logits, *args, **kw):
        got["args"], got["kw"] = args, kw
    sampler = Sampler(torch.device("cpu"), types.SimpleNamespace(adjust_logits=adjust, argmax=lambda x: "tokens"))
    asked = []

    def grammar(out):
        asked.append(out.tolist())
        return np.full(2, 6, dtype=np.uint32)
    configs = [SamplingConfig(), SamplingConfig(repetition_penalty=1.5), SamplingConfig(logit_bias={9: 1.0, 4: -2.0}),
               SamplingConfig(repetition_penalty=1.25, presence_penalty=0.5, frequency_penalty=0.125, logit_bias={1: 3.0}, allowed=grammar),
               SamplingConfig(allowed=lambda out: None)]
    histories = [None, None, None, (np.array([5, 6, 5, 7, 7], dtype=np.int32), 2), (np.array([1], dtype=np.int32), 1)]
    logits = torch.zeros(5, 40)
    assert sampler.sample_on_device(logits, configs, [0] * 5, [None, np.array([3, 8], dtype=np.int32)] + [None] * 3, histories) == "tokens"
    history, cu, prompts, rep, pres, freq = got["args"]
    assert history.tolist() == [3, 8, 5, 6, 5, 7, 7] and cu.tolist() == [0, 0, 2, 2, 7, 7] and prompts.tolist() == [0, 2, 0, 2, 0]
    assert rep.tolist() == [1.0, 1.5, 1.0, 1.25, 1.0] and pres.tolist() == [0, 0, 0, 0.5, 0] and freq.tolist() == [0, 0, 0, 0.125, 0]
    ids, values, cub = got["kw"]["bias"]
    assert ids.tolist() == [9, 4, 1] and values.tolist() == [1.0, -2.0, 3.0] and cub.tolist() == [0, 0, 0, 2, 3, 3]
    masks, rows = got["kw"]["masks"]
    assert masks.tolist() == [[6, 6]] and rows.tolist() == [-1, -1, -1, 0, -1] and asked == [[5, 7, 7]]
    assert got["kw"]["out"] is logits
    with pytest.raises(ValueError, match="prompt and output"):
        sampler.sample_on_device(logits, configs, [0] * 5, None, None)


def test_command_line():
    a = cli.build_parser().parse_args(["m", "--presence-penalty", "0.5", "--frequency-penalty", "-1", "--logit-bias", "5:1.5,7:-100"])
    assert a.presence_penalty == 0.5 and a.frequency_penalty == -1.0 and a.logit_bias == {5: 1.5, 7: -100.0}
    assert cli.build_parser().parse_args(["m"]).logit_bias is None
    with pytest.raises(argparse.ArgumentTypeError):
        cli._parse_bias("5=1")


class EmptyGrammar:
    """Callable, and false where it stands empty: a grammar is there if it is given, whatever its truth value."""

    def __init__(self):
        self.stack = []

    def __len__(self):
        return len(self.stack)

    def __call__(self, out):
        return np.full(2, 5, dtype=np.uint32)


def test_a_grammar_whose_truth_value_is_false():
    c = SamplingConfig(allowed=EmptyGrammar())
    assert not c.allowed and c.adjusts and c.needs_output
    assert allowed_mask(c, np.zeros(0, np.int32), 40).tolist() == [5, 5]


def test_options_that_float32_does_not_hold():
    """They go to the device in float32, where 1e39 is infinite."""
    most = float(np.finfo(np.float32).max)
    for bad in (dict(presence_penalty=1e39), dict(presence_penalty=-1e39), dict(frequency_penalty=1e39), dict(frequency_penalty=-1e300),
                dict(logit_bias={1: 1e39})):
        with pytest.raises(ValueError):
            SamplingConfig(**bad)
    c = SamplingConfig(presence_penalty=-most, frequency_penalty=most, logit_bias={1: most, 2: -1e39, 3: -math.inf})
    with np.errstate(over="ignore"):
        assert np.asarray(list(c.logit_bias.values()), dtype=np.float32).tolist() == [most, -math.inf, -math.inf]


def test_masks_without_a_token():
    """Bits behind the vocabulary are nobody's."""
    for V in (1, 31, 32, 33, 64, 70):
        words = -(-V // 32)
        mask = np.zeros(words, dtype=np.int32)
        assert allows_none(mask, V)
        if V % 32:
            mask[-1] = np.uint32(0xffffffff << (V % 32) & 0xffffffff).view(np.int32)
            assert allows_none(mask, V)
        for t in (0, V - 1):
            one = mask.copy()
            one.view(np.uint32)[t // 32] |= np.uint32(1 << (t % 32))
            assert not allows_none(one, V), (V, t)


def test_a_grammar_that_fills_one_array():
    """Requests whose grammar hands out the same array, filled anew, have the mask that was theirs."""
    got, room = [], np.zeros(2, dtype=np.int32)

    def grammar(out):
        room[:] = len(out)
        return room
    sampler = Sampler(torch.device("cpu"), types.SimpleNamespace(adjust_logits=lambda *a, **kw: got.append(kw["masks"]), argmax=lambda x: x))
    c = SamplingConfig(allowed=grammar)
    histories = [(np.arange(n, dtype=np.int32), 1) for n in (4, 2, 7)]
    sampler.sample_on_device(torch.zeros(3, 40), [c] * 3, [0] * 3, None, histories)
    given = [allowed_mask(c, h[0][h[1]:], 40) for h in histories]
    sampler.sample_on_device(torch.zeros(3, 40), [c] * 3, [0] * 3, None, histories, given)
    for masks, rows in got:
        assert masks.tolist() == [[3, 3], [1, 1], [6, 6]] and rows.tolist() == [0, 1, 2]


def test_biases_below_float32s_range_are_never():
    """They become -inf where they are given; a cast at every step would warn of an overflow at every step."""
    c = SamplingConfig(logit_bias={2: -1e39, 3: -math.inf, 4: -1e38})
    assert c.logit_bias == {2: -math.inf, 3: -math.inf, 4: -1e38}
    with np.errstate(over="raise"):
        assert np.asarray(list(c.logit_bias.values()), dtype=np.float32)[0] == -math.inf
