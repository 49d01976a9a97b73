"""Penalties and biases of requests in the engine: every token is the best (or the drawn one) of its adjusted logits, with slots, retraction and chains of guesses."""

import numpy as np
import pytest
import torch
import tree_oracle
from test_engine_cpu import make_engine
from test_engine_speculative_cpu import _pair, _prompts

from slime_b200.engine.http_server import EngineServer
from slime_b200.engine.request import SamplingParams

ASKS = [dict(repetition_penalty=1.7), dict(frequency_penalty=0.6, presence_penalty=0.3), dict(), dict(logit_bias={"5": 2.5, 7: -100.0, 10**6: 3.0}),
        dict(repetition_penalty=0.8, frequency_penalty=-0.2, presence_penalty=0.5, logit_bias={3: 0.5})]  # fmt: skip


@pytest.mark.parametrize("greedy", [True, False])
def test_slots_draw_from_adjusted_logits(greedy):
    _, _, plain, spec = _pair("dense")
    cfg = plain.cfg
    prompts = _prompts(cfg, len(ASKS))
    sampling = dict(max_new_tokens=20, ignore_eos=True, **(dict(temperature=0) if greedy else dict(temperature=1.0, sampling_seed=9)))
    reqs = plain.generate(prompts, [dict(sampling, **a) for a in ASKS])
    # a step's tokens from single prefills of everything in front of them, whose logits are adjusted by the oracle
    for r, a in zip(reqs, ASKS):
        n, s = len(r.input_ids), r.sampling
        bias = {int(t): v for t, v in (a.get("logit_bias") or {}).items()}
        for i in (0, 1, 7, 19):
            ids = r.input_ids + r.output_ids[:i]
            seen = {}

            def keep(logits, reqs, chains=None, seen=seen):
                seen["x"] = logits.clone()
                return logits

            with pytest.MonkeyPatch.context() as m:
                m.setattr("slime_b200.engine.penalties.adjust", keep)
                plain.generate([ids], dict(max_new_tokens=1, ignore_eos=True))
            f = lambda x: torch.tensor([x])  # noqa: E731
            x, _ = tree_oracle.adjusted(seen["x"], torch.tensor([ids]), torch.tensor([len(ids)]), torch.tensor([n]), f(s.repetition_penalty),
                                        f(s.frequency_penalty), f(s.presence_penalty), torch.tensor([list(bias)], dtype=torch.int32) if bias else None,
                                        torch.tensor([list(bias.values())]) if bias else None)  # fmt: skip
            lp = torch.log_softmax(x[0], -1)
            assert abs(float(lp[r.output_ids[i]]) - r.output_logprobs[i]) < 2e-4
            if greedy:
                assert r.output_ids[i] == int(lp.argmax())
    # the request that asks for nothing is the one that it is alone, and what a slot was asked is forgotten with its request
    assert plain.generate([prompts[2]], dict(sampling))[0].output_ids == reqs[2].output_ids
    # chains of guesses
    for x, y in zip(reqs, spec.generate(prompts, [dict(sampling, **a) for a in ASKS])):
        assert x.output_ids == y.output_ids
        assert np.abs(np.array(x.output_logprobs) - np.array(y.output_logprobs)).max() < 2e-4


def test_a_request_that_is_put_back_keeps_its_penalties():
    ask = dict(max_new_tokens=24, ignore_eos=True, frequency_penalty=0.7, presence_penalty=0.2, repetition_penalty=1.2)
    prompts = [[i + 1] * 6 for i in range(4)]
    small, big = make_engine(pages=14, max_running=4), make_engine(pages=200, max_running=4)
    a, b = (e.generate(prompts, [dict(ask, sampling_seed=i) for i in range(4)]) for e in (small, big))
    assert [r.output_ids for r in a] == [r.output_ids for r in b]
    never = big.generate([prompts[0]], dict(max_new_tokens=30, ignore_eos=True, temperature=0, presence_penalty=1e4))[0]
    assert len(set(never.output_ids)) == 30  # no token twice


def test_biases_of_more_tokens_than_any_request_before():
    _, _, plain, _ = _pair("dense")
    prompt = _prompts(plain.cfg, 1)[0]
    for allowed in ([4], list(range(30)), [4]):
        bias = {t: -1e9 for t in range(plain.cfg.vocab_size) if t not in allowed}
        got = plain.generate([prompt, prompt], [dict(max_new_tokens=6, ignore_eos=True, logit_bias=bias), dict(max_new_tokens=6, ignore_eos=True)])
        assert set(got[0].output_ids) <= set(allowed)


def test_penalties_as_they_arrive():
    sp = SamplingParams.from_dict(dict(repetition_penalty=None, frequency_penalty=None, presence_penalty=None, logit_bias=None))
    assert not sp.adjusts and sp == SamplingParams()
    assert SamplingParams.from_dict(dict(logit_bias={"12": -3})).logit_bias == {12: -3.0}
    assert EngineServer._openai_sampling(dict(frequency_penalty=0.5, presence_penalty=1, logit_bias={"3": 1}))["frequency_penalty"] == 0.5
    _, _, plain, _ = _pair("dense")
    nan, inf = float("nan"), float("inf")
    for name, values in (("repetition_penalty", (0, -1.0, nan, inf)), ("frequency_penalty", (nan, inf)), ("presence_penalty", (nan, -inf)),
                         ("logit_bias", ({-1: 1.0}, {1 << 31: 1.0}, {3: nan}, {3: inf}))):  # fmt: skip
        for bad in values:
            with pytest.raises(ValueError, match=name):
                plain.add_request([1, 2], {name: bad})
    with pytest.raises(ValueError, match="logit_bias"):
        plain.add_request([1, 2], SamplingParams(logit_bias={"3": 1.0}))
    assert not plain.has_work()
    none = plain.generate([[1, 2, 3]], dict(max_new_tokens=4, temperature=0, ignore_eos=True, logit_bias={t: -inf for t in range(40)}))[0]
    assert min(none.output_ids) >= 40


@pytest.mark.parametrize("name, bad", [
    ("repetition_penalty", 1e-46), ("repetition_penalty", 1e-30), ("repetition_penalty", 1e39), ("repetition_penalty", 2e38), ("frequency_penalty", -3e38),
    ("frequency_penalty", 1e39), ("presence_penalty", -1e39), ("presence_penalty", 3e38), ("logit_bias", {5: 1e39}), ("logit_bias", {5: 3e38}),
    ("logit_bias", {5: -3e38}),
])  # fmt: skip
def test_penalties_that_leave_no_distribution_in_fp32_are_refused(name, bad):
    """Numbers of 64 bits that fp32 rounds to zero or infinity, or that run over when they are counted or added, are no penalties; a running request goes on."""
    _, _, plain, spec = _pair("dense")
    for engine in (plain, spec):
        with pytest.raises(ValueError, match=name):
            engine.add_request([1, 2, 3], dict(max_new_tokens=4, temperature=0, ignore_eos=True, **{name: bad}))
        assert not engine.has_work()


def test_the_largest_penalties_still_leave_a_distribution():
    _, _, plain, _ = _pair("dense")
    V, inf = plain.cfg.vocab_size, float("inf")
    base = dict(max_new_tokens=8, ignore_eos=True)
    asks = [dict(frequency_penalty=s * 1e9, presence_penalty=s * 1e9, repetition_penalty=r, logit_bias={5: s * 1e9, 6: -s * 1e9, 7: -inf})
            for s in (-1, 1) for r in (1e-9, 1e9)]  # fmt: skip
    for temperature in (0, 1.0, 0.01):
        for r in plain.generate([[1, 2, 3]] * len(asks), [dict(base, temperature=temperature, **a) for a in asks]):
            assert len(r.output_ids) == 8 and 7 not in r.output_ids and np.isfinite(r.output_logprobs).all()
    # no token is left: refused, one is: taken
    with pytest.raises(ValueError, match="logit_bias"):
        plain.add_request([1, 2, 3], dict(base, logit_bias={t: -inf for t in range(V + 3)}))
    assert not plain.has_work()
    one = plain.generate([[1, 2, 3]], dict(base, logit_bias={t: -inf for t in range(V + 3) if t != 9}))[0]
    assert one.output_ids == [9] * 8


def test_a_refused_penalty_is_a_client_error_and_nothing_of_its_body_is_queued():
    import requests

    engine = make_engine()
    srv = EngineServer(engine, "127.0.0.1", 0).start(block=False)
    try:
        url = f"http://127.0.0.1:{srv.port}"
        post = lambda path, **body: requests.post(url + path, json=body, timeout=60)  # noqa: E731
        good = dict(max_new_tokens=100, ignore_eos=True)
        for bad in (dict(repetition_penalty=0), dict(frequency_penalty=-3e38), dict(logit_bias={"x": 1}), dict(logit_bias=[1, 2]), dict(presence_penalty="much"),
                    dict(repetition_penalty=[1]), dict(logit_bias={"5": None}), dict(frequency_penalty=10**400)):  # fmt: skip
            steps = engine.stats["steps"]
            r = post("/generate", input_ids=[[1, 2], [3, 4], [5]], sampling_params=[good, dict(good, **bad), good])
            assert r.status_code == 400 and r.json()["error"], r.text
            assert post("/generate", input_ids=[1, 2], sampling_params=dict(good, **bad)).status_code == 400
            r = post("/generate", input_ids=[1, 2], sampling_params=dict(good, **bad), bootstrap_room="r", bootstrap_host="http://127.0.0.1:1", first_token=3)
            assert r.status_code == 400  # (before the keys and values are fetched)
            r = post("/v1/completions", prompt=[1, 2, 3], max_tokens=100, **bad)
            assert r.status_code == 400 and r.json()["error"]["message"]
            assert not engine.has_work() and engine.stats["steps"] == steps
        r = post("/v1/completions", prompt=[1, 2, 3], max_tokens=5, temperature=0, frequency_penalty=0.5, logit_bias={"7": -100})
        assert r.status_code == 200 and r.json()["usage"]["completion_tokens"] == 5
    finally:
        srv.shutdown()
    with pytest.raises(ValueError, match="repetition_penalty"):
        engine.generate([[1], [2]], [good, dict(good, repetition_penalty=-1)])
    assert not engine.has_work()


def test_biases_of_tokens_outside_the_vocabulary_take_no_room():
    """They count for nothing, so a request that lists many of them leaves every slot's room for biases where it was, and no list is longer than the vocabulary."""
    _, _, plain, _ = _pair("dense")
    V = plain.cfg.vocab_size
    junk = {V + i: 1.0 for i in range(5000)}
    base = dict(max_new_tokens=4, ignore_eos=True, temperature=0)
    prompts = _prompts(plain.cfg, 2)
    want = plain.generate(prompts, [dict(base, logit_bias={3: 2.0, 5: -1.0}), dict(base)])
    room = plain.runner.adjustments.bias_ids.shape[1]
    got = plain.generate(prompts, [dict(base, logit_bias={**junk, 3: 2.0, 5: -1.0}), dict(base, logit_bias=junk)])
    assert [r.output_ids for r in got] == [r.output_ids for r in want]
    assert plain.runner.adjustments.bias_ids.shape[1] == room
    plain.generate(prompts, dict(base, logit_bias={t: 0.5 for t in range(V)}))
    assert plain.runner.adjustments.bias_ids.shape[1] <= V
