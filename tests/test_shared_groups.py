"""Which rows of a batch share cache blocks: batches whose prefixes lie deep in each other, and wide ones."""

import random

import pytest

from opsagent_amd.engine.kv_cache import shared_prefixes


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
