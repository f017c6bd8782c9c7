"""Requests that choices and forks are made of: those that an engine refuses, and those beside them."""

import pytest
import torch

from opsagent_amd.engine import engine as engine_module
from opsagent_amd.engine.engine import LLMEngine, SamplingParams
from opsagent_amd.engine.serving import EngineLoop

PARAMS = SamplingParams(max_new_tokens=5, stop_on_eos=False)


def _engine(**kw):
    cfg = dict(model="llama3-tiny", max_batch_size=8, kv_block_size=4, max_seq_len=128, spec_decode=False)
    if torch.cuda.is_available():
        cfg.update(model="llama3-micro", kv_block_size=32, max_seq_len=1024, kv_num_blocks=300)
    return LLMEngine({**cfg, **kw})


@pytest.mark.parametrize("fork", [False, True])
def test_an_empty_prompt_is_refused_by_itself(fork):
    """It has no token to go on from; the requests beside it are answered."""
    eng = _engine(fork_choices=fork)
    with pytest.raises(ValueError, match="at least one token"):
        eng.add_request([], PARAMS)
    assert not eng.requests and not eng.waiting
    loop = EngineLoop(eng)
    try:
        other = loop.submit([3, 4, 5], PARAMS)
        empty = loop.submit_choices([], PARAMS, 3)
        more = loop.submit_choices([5, 6, 7], PARAMS, 2)
        for f in empty:
            with pytest.raises(ValueError, match="at least one token"):
                f.result(timeout=60)
        assert all(len(f.result(timeout=60)[0]) == 5 for f in [other, *more])
        tokens, last = loop.submit_stream([], PARAMS)
        assert list(tokens) == []
        with pytest.raises(ValueError, match="at least one token"):
            last.result(timeout=60)
    finally:
        loop.shutdown()


def test_options_that_do_nothing_say_so(monkeypatch):
    """Hybrid models share and fork nothing; an engine that is asked to warns, and answers."""
    said = []
    monkeypatch.setattr(engine_module.log, "warning", lambda text, *args: said.append(text % args))
    hybrid = dict(model="povazen-tiny", kv_block_size=8, max_seq_len=64, kv_num_blocks=32, max_batch_size=4)
    eng = LLMEngine({**hybrid, "fork_choices": True, "shared_prefix": True})
    assert [t.split()[0] for t in said] == ["shared_prefix", "fork_choices"]
    assert all("povazen-tiny" in t for t in said) and not eng.fork_choices and not eng.shared_prefix
    assert len(eng.generate([1, 2, 3], PARAMS)[0]) == 5
    said.clear()
    LLMEngine(hybrid)
    _engine(fork_choices=True, shared_prefix=True)
    assert not said


def test_prompts_are_compared_once():
    """A long prompt's choices wait for many steps of its prefill, and compare nothing meanwhile."""
    eng = _engine(fork_choices=True, max_prefill_chunk=2)
    prompt = [3, 4, 5, 6, 7, 8, 9, 10, 11]
    compared = []

    class Tokens(list):
        def __getitem__(self, at):
            if isinstance(at, slice) and at.start is None:
                compared.append(at)
            return list.__getitem__(self, at)

    first = eng.add_request(prompt, PARAMS)
    eng.requests[first].prompt_ids = Tokens(prompt)
    same = [eng.add_request(prompt, PARAMS, fork_of=first) for _ in range(2)]
    shorter = eng.add_request(prompt[:5], PARAMS, fork_of=first)
    other = eng.add_request(prompt[:5] + [1], PARAMS, fork_of=first)
    longer = eng.add_request(prompt + [1], PARAMS, fork_of=first)
    assert [eng.requests[i].fork_of for i in (*same, shorter, other, longer)] == [first] * 3 + [None] * 2
    assert len(compared) == 5
    ids = [first, *same, shorter, other, longer]
    for _ in range(100):
        eng.step()
        if all(eng.requests[i].finished for i in ids):
            break
    assert len(compared) == 5
    out = {i: eng.requests[i].output_ids for i in ids}
    assert all(len(t) == 5 for t in out.values()) and out[same[0]] == out[same[1]]
    assert out[first] == out[same[0]] or torch.cuda.is_available()
