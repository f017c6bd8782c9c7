"""Pools that shrink: what is left of them, memory that runs out on the way, and loops under way."""

import multiprocessing as mp

import pytest
import torch

from opsagent_amd.engine.engine import LLMEngine, SamplingParams
from opsagent_amd.engine.kv_cache import BlockAllocatorError, PagedKVCache, SequenceState
from opsagent_amd.engine.serving import EngineLoop
from test_tp_gloo import _free_port, _init_dist, _tiny_cfg

SHAPES = [None, [(2, 8, 8), None, (1, 8, 4, "prefix"), (2, 8, 6, "vheads", 1)]]


def _cache(shapes, blocks=16):
    cache = PagedKVCache(3, 1, 8, 4, blocks, "cpu", torch.float32, layer_shapes=shapes)
    for k, v in cache.layers:
        if k is not None:
            k.normal_()
            if v.data_ptr() != k.data_ptr():
                v.normal_()
    return cache


def _sequence(cache, tokens):
    seq = SequenceState(cache, tokens)
    seq.ensure_capacity(len(tokens))
    seq.num_cached = len(tokens)
    seq.publish_full_blocks()
    return seq


def _rows(cache, blocks):
    return [t[blocks].clone() for kv in cache.layers for t in kv if t is not None]


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("fails", range(1, 7))
def test_memory_that_runs_out_loses_nothing(shapes, fails, monkeypatch):
    """Whichever tensor there is no memory for: sequences keep their keys, no block is named that a layer
    lacks, and the pool goes on and shrinks later."""
    cache = _cache(shapes)
    seqs = [_sequence(cache, list(range(100 * i, 100 * i + 9))) for i in range(3)]
    seqs.pop(0).free()
    want = [_rows(cache, s.blocks) for s in seqs]
    clone, calls = torch.Tensor.clone, []

    def short(t, *args, **kw):
        calls.append(t)
        if len(calls) == fails:
            raise torch.OutOfMemoryError("no memory for a layer")
        return clone(t, *args, **kw)

    with monkeypatch.context() as m:
        m.setattr(torch.Tensor, "clone", short)
        try:
            cache.shrink(10, seqs)
        except torch.OutOfMemoryError:
            pass
    assert len(calls) >= fails or fails > 5
    assert cache.num_blocks == 10 and cache.num_free() == 4
    assert all(t.shape[0] in (10, 16) for kv in cache.layers for t in kv if t is not None)
    assert all(_same(_rows(cache, s.blocks), w) for s, w in zip(seqs, want))
    child, copy = seqs[0].fork(8)                    # the pool goes on: a fork copies in every layer
    assert max(child.blocks) < 10
    cache.copy_blocks(*[[x] for x in copy])
    assert _same([t[:3] for r in _rows(cache, child.blocks[1:]) for t in r],
                 [t[:3] for r in _rows(cache, seqs[0].blocks[1:2]) for t in r])
    child.free()
    cache.shrink(9, seqs)
    assert all(t.shape[0] == 9 for kv in cache.layers for t in kv if t is not None)
    assert all(_same(_rows(cache, s.blocks), w) for s, w in zip(seqs, want))
    for s in seqs:
        s.free()
    assert cache.num_free() == 9 and not any(cache._ref)


def test_the_same_size_is_no_copy():
    cache = _cache(None)
    seq = _sequence(cache, list(range(9)))
    before = [k.data_ptr() for k, _ in cache.layers]
    cache.shrink(16, [seq])
    assert [k.data_ptr() for k, _ in cache.layers] == before and cache.num_free() == 13
    with pytest.raises(BlockAllocatorError):
        cache.shrink(2, [seq])


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("room,hits", [(0, {0: 0, 2: 0}), (1, {0: 0, 2: 0}), (2, {0: 0, 2: 8}), (3, {0: 4, 2: 8}),
                                       (9, {0: 4, 2: 8})])
def test_what_the_prefix_cache_finds_after_a_shrink(shapes, room, hits):
    """Three blocks are cached: the first sequence's one, then the third's two. The oldest go first, so
    that with room for one it is the third's second, which nothing reaches without its first."""
    cache = _cache(shapes, blocks=24)
    tokens = [[100 * i + j for j in range(4 + 3 * i)] for i in range(5)]
    seqs = [_sequence(cache, t) for t in tokens]
    before = {i: _rows(cache, seqs[i].blocks) for i in range(5)}
    for i in (0, 2):
        seqs[i].free()
    live = [seqs[i] for i in (1, 3, 4)]
    used = len({b for s in live for b in s.blocks})
    cache.shrink(used + room, live)
    assert cache.num_free() == room and all(s.blocks and max(s.blocks) < used + room for s in live)
    for i in range(5):
        found = SequenceState(cache, tokens[i] + [7])
        reused = found.reuse_prefix()
        assert reused == (hits[i] if i in hits else len(tokens[i]) // 4 * 4)
        full = reused // 4
        assert _same(_rows(cache, found.blocks), [t[:full] for t in before[i]])
        found.free()
    assert cache.num_free() == room


# -- under a loop ----------------------------------------------------------------------------------
PARAMS = SamplingParams(max_new_tokens=40, stop_on_eos=False)


def _engine(**kw):
    cfg = dict(model="llama3-tiny", max_batch_size=4, kv_block_size=4, max_seq_len=128, kv_num_blocks=100,
               spec_decode=False)
    if torch.cuda.is_available():
        cfg.update(model="llama3-micro", kv_block_size=32, max_seq_len=1024)
    return LLMEngine({**cfg, **kw})


@pytest.mark.parametrize("device", ["any", pytest.param("gpu", marks=pytest.mark.gpu)])
def test_a_loop_shrinks_between_steps(device):
    prompts = [[(7 * i + k) % 250 for i in range(11)] for k in range(3)]
    outs = []
    for shrink in (False, True):
        eng = _engine()
        loop = EngineLoop(eng)
        started, streams = [], []
        try:
            for p in prompts:
                tokens, fut = loop.submit_stream(p, PARAMS)
                streams.append(fut)
                started.append(next(tokens))
            if shrink:
                with pytest.raises(RuntimeError, match="another thread"):
                    eng.shrink_cache(60)                # not under the loop's steps
                assert eng.kv.num_blocks == 100
                loop.shrink_cache(60)
                assert eng.kv.num_blocks == 60 and eng.kv.layers[0][0].shape[0] == 60
                with pytest.raises(ValueError, match="does not shrink"):
                    loop.shrink_cache(61)
                errors = []
                streams[0].add_done_callback(lambda f: errors.append(loop.shrink_cache(59)))
            outs.append([f.result(timeout=60)[0] for f in streams])
            if shrink:
                assert loop.generate(prompts[0], PARAMS)[0]
                loop.shrink_cache(40)                   # idle
                assert errors == [None] and eng.kv.num_blocks == 40 and loop.healthy
        finally:
            loop.shutdown()
        if shrink:
            with pytest.raises(RuntimeError, match="loop has ended"):
                loop.shrink_cache(30)
            eng.shrink_cache(30)                        # nobody else runs its steps now
            assert eng.kv.num_blocks == 30
    assert outs[0] == outs[1] or torch.cuda.is_available()
    assert all(len(o) == 40 for out in outs for o in out)


def _rank(rank, world, port, q):
    dist = _init_dist(rank, world, port)
    eng = LLMEngine(_tiny_cfg(kv_num_blocks=40))
    prompt = [(5 * i) % 250 for i in range(20)]
    if rank == 0:
        want = eng.generate(prompt, SamplingParams(max_new_tokens=8, stop_on_eos=False))[0]
        rid = eng.add_request(prompt + [1], SamplingParams(max_new_tokens=8, stop_on_eos=False))
        for _ in range(4):
            eng.step()
        with pytest.raises(BlockAllocatorError):
            eng.shrink_cache(1)                         # refused on every rank: nothing is sent
        eng.shrink_cache(12)
        with pytest.raises(ValueError):
            eng.shrink_cache(13)
        while not eng.requests[rid].finished:
            eng.step()
        after = eng.generate(prompt, SamplingParams(max_new_tokens=8, stop_on_eos=False))[0]
        eng.shutdown_followers()
        q.put((0, want == after, len(eng.requests[rid].output_ids), eng.kv.num_blocks, sorted(eng.kv._free)))
    else:
        assert eng.follower_loop() == "stop"
        q.put((1, True, 8, eng.kv.num_blocks, sorted(eng.kv._free)))
    dist.barrier()
    dist.destroy_process_group()


def test_ranks_shrink_before_the_same_step():
    ctx = mp.get_context("spawn")
    q, port = ctx.Queue(), _free_port()
    procs = [ctx.Process(target=_rank, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    try:
        got = sorted(q.get(timeout=180) for _ in procs)
    finally:
        for p in procs:
            p.join(timeout=60)
            if p.is_alive():
                p.terminate()
    assert [g[1:4] for g in got] == [(True, 8, 12)] * 2 and got[0][4] == got[1][4]
