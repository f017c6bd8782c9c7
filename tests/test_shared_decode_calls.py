"""Calls of shared decode attention beside those of a serving step: what is refused, long batches, plans."""

import ctypes
import os

import pytest
import torch
from torch.autograd import forward_ad

from opsagent_amd import ops
from test_shared_decode import _case, _check

gpu = pytest.mark.gpu
DEVICE = "cuda" if torch.cuda.is_available() else "cpu"


def _small():
    gen = torch.Generator().manual_seed(1)
    caches = [torch.randn(6, 8, 2, 64, generator=gen).to(DEVICE, torch.bfloat16) for _ in range(2)]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    return dict(q=torch.randn(2, 4, 64, generator=gen).to(DEVICE, torch.bfloat16), k_cache=caches[0],
                v_cache=caches[1], block_table=i32([[0, 1, 2], [0, 3, 4]]), seq_lens=i32([20, 13]),
                leaders=i32([0, 0]), shared=i32([1, 1]))


@pytest.mark.parametrize("name", ["q", "k_cache", "v_cache"])
def test_gradients_of_either_mode_are_refused(name):
    """On the CPU as on the GPU: nothing is left out of a derivative without an error."""
    c = _small()
    want = ops.attention_decode_shared(**c)
    leaf = {**c, name: c[name].clone().requires_grad_()}
    with pytest.raises(RuntimeError, match="gradients"):
        ops.attention_decode_shared(**leaf)
    with torch.no_grad():
        assert torch.equal(ops.attention_decode_shared(**leaf), want)
    with forward_ad.dual_level():
        dual = {**c, name: forward_ad.make_dual(c[name], torch.ones_like(c[name]))}
        with pytest.raises(RuntimeError, match="gradients"):
            ops.attention_decode_shared(**dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="gradients"):
            ops.attention_decode_shared(**dual)
        assert torch.equal(ops.attention_decode_shared(**c), want)


def _long_batch(n):
    """n rows, block 32: three groups that go through all of them, one led by the last row, strangers,
    and rows without keys."""
    rows = []
    for b in range(n):
        lead, pages = ((0, 3), (1, 1), (b, 0), (b, 0), (n - 1, 2), (0, 3), (0, 3))[b % 7]
        rows.append((lead, pages, 0 if b % 7 == 3 else 32 * pages + 1 + (b * 7) % 40))
    rows[0], rows[1], rows[n - 1] = (0, 3, 130), (1, 1, 33), (n - 1, 2, 64)
    return rows


@gpu
@pytest.mark.parametrize("n,Hq,Hk,D,dtype", [
    (256, 8, 2, 64, torch.bfloat16),
    (257, 8, 2, 64, torch.bfloat16),
    (300, 20, 1, 64, torch.float16),
    (1024, 4, 4, 128, torch.bfloat16),
    (1025, 6, 2, 64, torch.bfloat16),
    (2047, 32, 8, 64, torch.float16),
    (2048, 8, 2, 128, torch.bfloat16),
    (2048, 128, 1, 64, torch.bfloat16),      # a tile is one row: the most partial results
])
def test_long_batches(n, Hq, Hk, D, dtype):
    """Up to as many rows as there are: more than 256 are planned by a block of 1024 threads."""
    c = _case(_long_batch(n), Hq, Hk, D, 32, dtype, seed=n)
    got = ops.attention_decode_shared(**c)
    _check(got, c)
    plan = ops.shared_decode_plan(c["seq_lens"], c["leaders"], c["shared"], (Hq, Hk), D,
                                  c["block_table"].shape[1], 32)
    assert torch.equal(ops.attention_decode_shared(**c, plan=plan), got)


@gpu
def test_more_rows_than_a_plan_takes():
    c = _case([(b, 0, 1) for b in range(2049)], 2, 1, 64, 32, seed=1)
    with pytest.raises(ValueError, match="1 to 2048 rows"):
        ops.attention_decode_shared(**c)
    empty = {x: t[:0] if x not in ("k_cache", "v_cache") else t for x, t in c.items()}
    with pytest.raises(ValueError, match="1 to 2048 rows"):
        ops.attention_decode_shared(**empty)


@gpu
@pytest.mark.parametrize("seed", range(30))
def test_a_plan_made_by_the_launch_is_the_one_made_before(seed):
    """Up to 64 rows are planned by each block for itself, or before: the same work, bit for bit."""
    gen = torch.Generator().manual_seed(seed)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=gen))  # noqa: E731
    n, leads, rows = (1, 2, 63, 64)[seed] if seed < 4 else pick(1, 64), [], []
    span = (3, 60, 400, 1500)[pick(0, 3)]
    for b in range(n):
        kind = pick(0, 9)
        if leads and kind < 6:
            lead, pages = leads[pick(0, len(leads) - 1)]
            rows.append((lead, pages, 16 * pages + pick(0, span)))
        elif kind == 6:
            rows.append((b, 0, 0))
        else:
            pages = pick(0, span // 16 + 1)
            leads.append((b, pages))
            rows.append((b, pages, 16 * pages + pick(1, span)))
    group, Hk = pick(1, 20), pick(1, 5)
    c = _case(rows, group * Hk, Hk, (64, 128)[seed % 2], 16, (torch.bfloat16, torch.float16)[seed // 2 % 2],
              seed=200 + seed)
    got = ops.attention_decode_shared(**c)
    _check(got, c)
    plan = ops.shared_decode_plan(c["seq_lens"], c["leaders"], c["shared"], (group * Hk, Hk), c["q"].shape[2],
                                  c["block_table"].shape[1], 16)
    assert torch.equal(ops.attention_decode_shared(**c, plan=plan), got)
    assert torch.equal(ops.attention_decode_shared(**c), got)


@gpu
@pytest.mark.parametrize("columns", [4, 24, 48, 96])         # as the waves share keys and columns
@pytest.mark.parametrize("shared", [False, True])
def test_many_small_float16_weights(columns, shared):
    """One key has nearly all of the weight, and what the others have in sum is not lost: weights down
    to 2^-29 of the largest are rounded by half a step 2^-11 of each, like any other, and the output by as
    much. float32 scores and exponentials are off by 2^-12 of what they weigh, as in other tests."""
    n, D, rows = 2 ** 15, 64, 2 if shared else 1
    heads = columns // rows
    q = torch.zeros(rows, heads, D, dtype=torch.float16, device=DEVICE)
    q[..., 0] = 4.0
    k = torch.zeros(n // 64, 64, 1, D, dtype=torch.float16, device=DEVICE)
    k[0, 0, 0, 0] = 4.5                                     # the others have 2^-25.97 of its weight
    v = torch.zeros_like(k)
    v[..., 1] = 1.0
    v[0, 0, 0, 1] = 0.0
    table = torch.arange(n // 64, dtype=torch.int32, device=DEVICE).expand(rows, -1).contiguous()
    i32 = lambda x: torch.full((rows,), x, dtype=torch.int32, device=DEVICE)  # noqa: E731
    got = ops.attention_decode_shared(q, k, v, table, i32(n), i32(0), i32(n // 64), scale=1.0)
    small = torch.tensor(-18.0, dtype=torch.float64).exp()
    want = float((n - 1) * small / (1 + (n - 1) * small))
    h = 2.0 ** -11
    assert want > 2.0 ** -11 and (got[..., 1].double() - want).abs().max() <= (2 * h + h * h + 2.0 ** -12) * want
    assert torch.count_nonzero(got[..., 2:]) == 0


# -- the longest rows ----------------------------------------------------------------------------
def _last_end(keys, blocks):
    """Where the last of a group's chunks ends, as the plan works it out, before it is cut to `keys`."""
    up = lambda a, b: -(-a // b)  # noqa: E731
    sizes = up(keys, 64)
    run = max(2, up(sizes + 1, blocks))
    chunk = up(up(keys, up(sizes, run)), 128) * 128
    return up(keys, chunk) * chunk


def test_rows_whose_chunks_end_past_32_bits_are_refused():
    """The last chunk of a row of nearly 2^31 tokens ends past them; a table may have room for 2^31 - 2^20."""
    assert max(_last_end(2 ** 31 - 4096 - i, 512) for i in range(5000)) >= 2 ** 31
    most = 2 ** 31 - 2 ** 20
    assert max(_last_end(most - i, n) for i in range(3000) for n in (1, 2, 8, 64, 512)) < 2 ** 31
    ops._shared_table(1, most // 2 ** 20, 2 ** 20)
    for width, block in [(2 ** 11, 2 ** 20), (most // 16 + 1, 16), (most + 1, 1)]:
        with pytest.raises(ValueError, match="a row of more than"):
            ops._shared_table(1, width, block)
    path = os.path.join(os.path.dirname(ops.__file__), "libopsagent_kernels.so")
    if not os.path.exists(path):
        pytest.skip("kernel library not built")
    from opsagent_amd.ops import hip_lib

    lib = ctypes.CDLL(path)
    hip_lib._declare(lib)
    for width, block in [(2 ** 11, 2 ** 20), (most // 16 + 1, 16), (most + 1, 1)]:
        assert lib.oa_shared_plan(None, 16, 16, 16, 16, 1, 32, 8, 128, width, block) == -102
        n = [4096, 128, 262144, 1024, 128, 262144, 1024, 128, 9, 1, 32, 8, 128, width, 50, block, 0]
        assert lib.oa_attention_decode_shared(None, 16, 16, 16, 16, None, None, None, 16, 16, 16,
                                              (ctypes.c_int64 * 17)(*n), 0.1) == -102
