"""Which rows of a batch share cache blocks: batches whose prefixes lie deep in each other, and wide ones."""

import random
import time
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from opsagent_amd.engine import engine as engine_module
from opsagent_amd.engine.engine import LLMEngine
from opsagent_amd.engine.kv_cache import SequenceState, shared_prefixes


def _holds(tables, full, leaders, shared, saved):
    groups = {}
    for b, lead in enumerate(leaders):
        assert leaders[lead] == lead and shared[b] <= full[b]
        assert list(tables[b][: shared[b]]) == list(tables[lead][: shared[b]])
        groups.setdefault(lead, []).append(b)
    for rows in groups.values():
        assert len({shared[b] for b in rows}) == 1 and (len(rows) > 1 or shared[rows[0]] == 0)
    assert saved == sum((len(rows) - 1) * shared[rows[0]] for rows in groups.values())


@pytest.mark.parametrize("n", [1, 2, 3, 250, 256, 257, 512])
def test_nested_prefixes(n):
    """Row i begins with the blocks of every row before it: a tree as deep as there are rows."""
    order = random.Random(n).sample(range(n), n)
    tables = [list(range(i + 1)) for i in order]
    leaders, shared, saved = shared_prefixes(tables, [len(t) for t in tables])
    _holds(tables, [len(t) for t in tables], leaders, shared, saved)
    best = [0] * (n + 1)       # rows before j, the last group of them from row i on: it shares i + 1 blocks
    for j in range(1, n + 1):
        best[j] = max(best[i] + (j - i - 1) * (i + 1) for i in range(j))
    assert saved == best[n]


@pytest.mark.parametrize("n", [64, 257, 600])
def test_one_prefix_of_many_rows(n):
    """One group, however many rows there are."""
    tables = [[7, 8, 9, 100 + b] for b in range(n)]
    assert shared_prefixes(tables, [4] * n) == ([0] * n, [3] * n, 3 * (n - 1))


def _random_tables(rng):
    n, tables = rng.randint(1, 60), []
    for b in range(n):
        if tables and rng.random() < 0.8:
            old = rng.choice(tables)
            tables.append(old[: rng.randint(0, len(old))] + [1000 * b + i for i in range(rng.randint(0, 3))])
        else:
            tables.append([1000 * b + i for i in range(rng.randint(0, 9))])
    return tables, [max(0, len(t) - rng.randint(0, 1)) for t in tables]


@pytest.mark.parametrize("seed", range(20))
def test_lists_and_a_block_table_give_the_same(seed):
    """Rows of a wider table, whatever stands behind a row's full blocks."""
    rng = random.Random(seed)
    tables, full = _random_tables(rng)
    got = shared_prefixes(tables, full)
    _holds(tables, full, *got)
    table = np.full((len(tables) + 2, max(full) + 3), 5, np.int32)
    for b, blocks in enumerate(tables):
        table[b, : full[b]] = blocks[: full[b]]
    assert shared_prefixes(table[: len(tables)], full) == got
    assert shared_prefixes(table, full) == got          # as many rows as there are numbers of blocks


def test_many_long_rows_take_no_milliseconds():
    """The host finds groups within a decode step: 0.2 ms for 128 rows of 512 common blocks."""
    table = np.tile(np.arange(520, dtype=np.int32), (128, 1))
    table[:, 512:] += 1000 * np.arange(1, 129, dtype=np.int32)[:, None]
    took = []
    for _ in range(20):
        start = time.perf_counter()
        leaders, shared, saved = shared_prefixes(table, [515] * 128)
        took.append(time.perf_counter() - start)
    assert (leaders, shared, saved) == ([0] * 128, [512] * 128, 127 * 512)
    assert min(took) < 0.002


def test_a_batch_that_cannot_save_enough_is_not_looked_at(monkeypatch):
    eng = LLMEngine(dict(model="llama3-tiny", max_batch_size=4, kv_block_size=4, max_seq_len=128, kv_num_blocks=64)
                    if not torch.cuda.is_available() else
                    dict(model="llama3-micro", max_batch_size=4, max_seq_len=1024, kv_num_blocks=64))
    calls = []
    monkeypatch.setattr(engine_module, "shared_prefixes", lambda *a: (calls.append(a), shared_prefixes(*a))[1])
    batch = []
    for b in range(3):
        seq = SequenceState(eng.kv, list(range(2 * eng.block_size)) + [b])
        seq.ensure_capacity(len(seq.token_ids))
        batch.append(SimpleNamespace(seq=seq))
        eng._h_rows[4][b, :3] = torch.tensor([1, 2, 5 + b], dtype=torch.int32)
    weight = eng.block_size * eng.spec.num_kv_heads
    monkeypatch.setattr(engine_module, "SHARED_LEAST", 4 * weight + 1)
    assert not eng._find_shared(batch) and not calls
    eng._shared_key = None
    monkeypatch.setattr(engine_module, "SHARED_LEAST", 4 * weight)
    assert eng._find_shared(batch) and len(calls) == 1
    assert eng._h_groups[:, :4].tolist() == [[0, 0, 0, 0], [2, 2, 2, 0]]
