"""Decode attention that reads pages which rows of a batch share once, against float64.

Tolerance, per output: the output's own rounding, half a step h of |o|; each weight's
rounding to 16 bits before its product with the values, h of sum p|v|; float16 weights
below its normal range, off by 2^-25 of the row's largest weight each; and 2^-12 of sum p|v|
for float32 scores (128 products of at most 12 in all, to 2^-24 each of the partial sums, and
as much again for the exponential)."""

import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

from opsagent_amd import ops
from opsagent_amd.ops import torch_ref

gpu = pytest.mark.gpu
DEVICE = "cuda" if torch.cuda.is_available() else "cpu"


def _case(rows, Hq=8, Hk=2, D=128, bs=32, dtype=torch.bfloat16, seed=0, spare=3, device=None):
    """rows: (leader, shared pages, length) of each. Tables name pages in any order; what lies
    behind a row's last token, and pages of nobody, hold NaN."""
    device = device or DEVICE
    gen = torch.Generator().manual_seed(seed)
    lens = [r[2] for r in rows]
    width = max(1, max(-(-n // bs) for n in lens)) + 1
    table, taken = torch.full((len(rows), width), -7, dtype=torch.int64), 0
    for b in sorted(range(len(rows)), key=lambda b: rows[b][0] != b):          # leaders first
        lead, pages, n = rows[b]
        need = -(-n // bs)
        common = min(pages, need) if 0 <= lead < len(rows) and lead != b else 0
        if common:
            table[b, :common] = table[lead, :common]
        table[b, common:need] = torch.arange(taken, taken + need - common)
        taken += need - common
    place = torch.randperm(taken + spare, generator=gen)
    table = torch.where(table >= 0, place[table.clamp(min=0)], table)
    shape = (taken + spare, bs, Hk, D)
    k, v = torch.randn(shape, generator=gen), torch.randn(shape, generator=gen)
    seen = torch.zeros(shape[:2], dtype=torch.bool)
    for b, n in enumerate(lens):
        at = torch.arange(n)
        seen[table[b, at // bs], at % bs] = True
    k[~seen], v[~seen] = float("nan"), float("nan")
    q = 2.0 * torch.randn(len(rows), Hq, D, generator=gen)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    return dict(q=q.to(device, dtype), k_cache=k.to(device, dtype), v_cache=v.to(device, dtype),
                block_table=table.to(device, torch.int32), seq_lens=i32(lens),
                leaders=i32([r[0] for r in rows]), shared=i32([r[1] for r in rows]))


def _exact(c, scale=None):
    """(output, tolerance), float64, every row from its own row of the table."""
    q, k, v = (c[x].double().cpu() for x in ("q", "k_cache", "v_cache"))
    h = torch.finfo(c["q"].dtype).eps / 2
    B, Hq, D = q.shape
    bs, Hk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for b, n in enumerate(c["seq_lens"].tolist()):
        n = min(n, c["block_table"].shape[1] * bs)
        if n <= 0:
            continue
        pages = c["block_table"][b, : -(-n // bs)].long().cpu()
        kk = k[pages].reshape(-1, Hk, D)[:n].transpose(0, 1).contiguous()      # [Hk, n, D]
        vv = v[pages].reshape(-1, Hk, D)[:n].transpose(0, 1).contiguous()
        s = q[b].view(Hk, Hq // Hk, D) @ kk.transpose(1, 2) * scale
        w = (s - s.amax(-1, keepdim=True)).exp()
        p = w / w.sum(-1, keepdim=True)
        out[b] = (p @ vv).view(Hq, D)
        size = (p @ vv.abs()).view(Hq, D)
        small = (vv.abs().sum(1, keepdim=True) / w.sum(-1, keepdim=True) * 2.0 ** -25).view(Hq, D)
        tol[b] = h * (1 + h) * out[b].abs() + (h + 2.0 ** -12) * size
        if c["q"].dtype == torch.float16:
            tol[b] += small
    return out, tol


def _check(got, c, scale=None):
    want, tol = _exact(c, scale)
    off = (got.double().cpu() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} outputs off, the worst by {(off / tol).max():.2f} tolerances"


GROUPS = {
    "one token": [(0, 0, 1)],
    "one row": [(0, 0, 100)],
    "two rows of one page": [(0, 1, 33), (0, 1, 32)],
    "prefix is all of it": [(0, 4, 128), (0, 4, 128), (0, 4, 129)],
    "ragged": [(0, 3, 97), (0, 3, 300), (0, 3, 128), (0, 3, 200)],
    "different depths": [(0, 9, 700), (0, 5, 161), (0, 8, 350)],
    "two groups and strangers": [(0, 10, 400), (1, 0, 77), (2, 6, 193), (0, 10, 321), (2, 6, 500),
                                 (5, 0, 1), (2, 6, 192), (0, 10, 330)],
    "leader in the back": [(3, 4, 150), (1, 0, 40), (3, 4, 129), (3, 4, 400)],
    "rows without keys": [(0, 2, 70), (0, 2, 0), (2, 0, 0), (0, 2, 64), (4, 0, 5)],
    "long": [(0, 60, 2000), (0, 60, 1921), (0, 60, 1920), (0, 60, 2500)],
    "many rows": [(0, 7, 224 + i % 45) if i % 5 else (i, 0, 1 + 3 * i) for i in range(130)],
}
GROUPS["many rows"][0] = (0, 7, 260)


def _at_block(rows, bs):
    """Groups are written for pages of 32 tokens."""
    return [(lead, pages * 32 // bs, n) for lead, pages, n in rows]


@gpu
@pytest.mark.parametrize("name", list(GROUPS))
@pytest.mark.parametrize("Hq,Hk,D,bs,dtype", [
    (8, 2, 128, 32, torch.bfloat16),
    (32, 8, 128, 16, torch.bfloat16),
    (14, 2, 64, 32, torch.float16),
    (6, 6, 128, 4, torch.float16),
    (20, 1, 64, 64, torch.bfloat16),
    (70, 1, 128, 1, torch.bfloat16),
])
def test_groups(name, Hq, Hk, D, bs, dtype):
    rows = _at_block(GROUPS[name], bs)
    c = _case(rows, Hq, Hk, D, bs, dtype, seed=len(name))
    _check(ops.attention_decode_shared(**c), c)
    plan = ops.shared_decode_plan(c["seq_lens"], c["leaders"], c["shared"], (Hq, Hk), D,
                                  c["block_table"].shape[1], bs)
    _check(ops.attention_decode_shared(**c, plan=plan), c)


@gpu
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 64])
@pytest.mark.parametrize("prefix,tail", [(1, 1), (2, 31), (11, 32), (40, 33)])
def test_columns_of_a_tile(rows, prefix, tail):
    c = _case([(0, prefix, 32 * prefix + (i * 7) % (tail + 1)) for i in range(rows)], seed=rows + prefix)
    _check(ops.attention_decode_shared(**c), c)


@gpu
@pytest.mark.parametrize("leaders", [[-1, 9, 4], [1, 1, 1], [1, 2, 0], [0, 0, 1], [2, 2, 0]])
def test_leaders_that_lead_nothing(leaders):
    """A row whose leader does not lead itself is its own: its own pages are read."""
    c = _case([(0, 0, 100), (1, 0, 64), (2, 0, 70)], seed=5)
    real = [x if 0 <= x < 3 and leaders[x] == x else b for b, x in enumerate(leaders)]
    c["leaders"] = torch.tensor(leaders, dtype=torch.int32, device=DEVICE)
    c["shared"] = torch.tensor([1, 1, 1], dtype=torch.int32, device=DEVICE)
    for b, x in enumerate(real):
        if x != b:
            c["block_table"][b, :1] = c["block_table"][x, :1]
    _check(ops.attention_decode_shared(**c), c)


@gpu
@pytest.mark.parametrize("shared", [-3, 0, 2, 100])
def test_shared_pages_outside_the_row(shared):
    c = _case([(0, 2, 90), (0, 2, 64), (0, 2, 75)], seed=6)
    c["shared"] = torch.full((3,), shared, dtype=torch.int32, device=DEVICE)
    if shared > 2:                                   # as many as both rows have full pages: 2
        assert torch.equal(c["block_table"][0, :2], c["block_table"][1, :2])
    _check(ops.attention_decode_shared(**c), c)


@gpu
def test_only_the_leaders_table_is_read_for_shared_pages():
    c = _case([(0, 3, 130), (0, 3, 100), (0, 3, 97)], seed=7)
    want = ops.attention_decode_shared(**c)
    c["block_table"][1:, :3] = -1
    assert torch.equal(ops.attention_decode_shared(**c), want)


@gpu
def test_lengths_and_pages_outside_the_cache():
    """Lengths are cut to the table, pages to the cache; other rows do not change."""
    c = _case([(0, 0, 64), (1, 0, 96), (2, 0, 50)], seed=8)
    want = ops.attention_decode_shared(**c)
    c["seq_lens"][1] = 2 ** 30
    c["block_table"][1, 0] = 2 ** 31 - 1
    c["block_table"][1, 1] = -5
    got = ops.attention_decode_shared(**c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


@gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scale(scale):
    c = _case(GROUPS["ragged"], seed=9)
    _check(ops.attention_decode_shared(**c, scale=scale), c, scale)


@gpu
def test_infinite_and_nan_values_stay_in_their_rows():
    c = _case([(0, 2, 70), (0, 2, 80), (2, 0, 40)], seed=10)
    want = ops.attention_decode_shared(**c)
    page = int(c["block_table"][1, 2])
    c["v_cache"][page, 3] = float("inf")
    got = ops.attention_decode_shared(**c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    assert torch.isinf(got[1]).all()
    c["k_cache"][page, 3] = float("nan")
    got = ops.attention_decode_shared(**c)
    assert torch.equal(got[0], want[0]) and torch.isnan(got[1]).all()


@gpu
@pytest.mark.parametrize("Hq,Hk", [(8, 2), (32, 2), (32, 1), (96, 1)])        # 4, 16, 32 and 96 columns a row
@pytest.mark.parametrize("rows", [1, 3])
def test_an_infinite_last_value(Hq, Hk, rows):
    """Keys behind a chunk's last weigh nothing, whatever it holds."""
    c = _case([(0, 3, 96 + 9 * i + 1) for i in range(rows)], Hq, Hk, seed=12)
    table = c["block_table"]
    for page, at in [(int(table[0, 3]), 0), (int(table[0, 2]), 31)]:          # row 0's last; all rows' last shared
        c["v_cache"][page, at, :, 5] = float("inf")
        c["v_cache"][page, at, :, 6] = float("-inf")
        got = ops.attention_decode_shared(**c)
        finite = torch.ones(128, dtype=torch.bool, device=got.device)
        finite[5:7] = False
        assert (got[0, :, 5] == float("inf")).all() and (got[0, :, 6] == float("-inf")).all()
        assert torch.isfinite(got[..., finite]).all()
    assert (got[:, :, 5] == float("inf")).all() and (got[:, :, 6] == float("-inf")).all()


@gpu
def test_large_scores():
    c = _case(GROUPS["ragged"], seed=11)
    c["q"] = c["q"] * 60
    want, _ = _exact(c)
    got = ops.attention_decode_shared(**c).double().cpu()
    assert torch.isfinite(got).all()
    # the output's rounding and the weights', 2^-8 each; scores of up to some hundreds, in
    # float32: 2^-24 of each of 128 partial sums is at most 2^-9 of a weight
    size = c["v_cache"].nan_to_num(0).double().abs().amax().cpu()
    assert (got - want).abs().max() <= (2 * 2.0 ** -8 + 2.0 ** -9) * size


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_strides(dtype):
    """Queries inside a q | k | v row, keys and values of a page beside each other, heads outside
    tokens, rows of a wider table."""
    c = _case(GROUPS["two groups and strangers"], Hq=8, Hk=2, dtype=dtype, seed=12)
    want = ops.attention_decode_shared(**c)
    B = c["q"].shape[0]
    qkv = torch.full((B, 12, 128), float("nan"), dtype=dtype, device=DEVICE)
    qkv[:, :8] = c["q"]
    both = torch.stack([c["k_cache"], c["v_cache"]], dim=1)                    # [pages, 2, bs, Hk, D]
    heads = both.permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4)    # heads outside tokens
    wide = torch.full((B, c["block_table"].shape[1] + 5), -1, dtype=torch.int32, device=DEVICE)
    wide[:, :-5] = c["block_table"]
    for cache in (both, heads):
        got = ops.attention_decode_shared(qkv[:, :8], cache[:, 0], cache[:, 1], wide[:, :-5],
                                          c["seq_lens"], c["leaders"], c["shared"])
        assert torch.equal(got, want)


@gpu
def test_offsets_past_32_bits():
    """Keys more than 2^31 elements and 2^32 bytes into the cache."""
    bs, Hk, D = 64, 8, 128
    pages = 2 ** 31 // (bs * Hk * D) + 40
    c = _case([(0, 2, 200), (0, 2, 150), (2, 0, 90)], Hq=16, Hk=Hk, bs=bs, seed=13, spare=0)
    n = c["k_cache"].shape[0]
    big = {x: torch.empty(pages, bs, Hk, D, dtype=torch.bfloat16, device=DEVICE)
           for x in ("k_cache", "v_cache")}
    for x in big:
        big[x][pages - n:] = c[x]
    table = torch.where(c["block_table"] >= 0, c["block_table"] + (pages - n), c["block_table"])
    got = ops.attention_decode_shared(**{**c, **big, "block_table": table})
    assert torch.equal(got, ops.attention_decode_shared(**c))


@gpu
@pytest.mark.parametrize("Hq,Hk,rows", [
    (64, 64, [(0, 0, 9000)]),                             # keys shared out by the waves
    (2560, 64, [(0, 0, 9000)]),                           # columns shared out
    (64, 64, [(0, 9000, 9100), (0, 9000, 9001)]),
])
def test_more_pages_than_a_unit_lists(Hq, Hk, rows):
    """Pages of one token, and more than 1024 of them in the keys that a block takes."""
    c = _case(rows, Hq, Hk, 64, 1, seed=21)
    _check(ops.attention_decode_shared(**c), c)


@gpu
def test_more_keys_than_a_cache_holds():
    """Beyond 128 MB of them the rows' own keys are read in another way."""
    c = _case([(0, 10, 320 + 1900 + i) for i in range(12)] + [(i, 0, 2000 + i) for i in range(12, 18)],
              Hq=16, Hk=8, seed=22)
    _check(ops.attention_decode_shared(**c), c)
    plan = ops.shared_decode_plan(c["seq_lens"], c["leaders"], c["shared"], (16, 8), 128,
                                  c["block_table"].shape[1], 32)
    _check(ops.attention_decode_shared(**c, plan=plan), c)


@gpu
def test_calls_on_two_streams():
    """Calls of different batches under way together share nothing."""
    cases = [_case(GROUPS["long"], Hq=32, Hk=8, seed=23), _case(GROUPS["many rows"], seed=24)]
    want = [ops.attention_decode_shared(**c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(5):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.attention_decode_shared(**c))
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for g, w in zip(got, want) for x in g)


@gpu
def test_equals_the_paged_form_and_itself():
    c = _case(GROUPS["long"], Hq=32, Hk=8, seed=14)
    got = ops.attention_decode_shared(**c)
    paged = ops.attention_decode_paged(c["q"], c["k_cache"], c["v_cache"], c["block_table"], c["seq_lens"])
    want, tol = _exact(c)
    assert ((got.double() - paged.double()).abs().cpu() <= 2 * tol).all()
    for _ in range(3):
        assert torch.equal(ops.attention_decode_shared(**c), got)


@gpu
def test_a_plan_is_made_once_for_all_layers():
    c = _case(GROUPS["two groups and strangers"], seed=15)
    width, bs = c["block_table"].shape[1], c["k_cache"].shape[1]
    plan = ops.shared_decode_plan(c["seq_lens"], c["leaders"], c["shared"], (8, 2), 128, width, bs)
    got = [ops.attention_decode_shared(**{**c, "q": q}, plan=plan) for q in (c["q"], c["q"] * 0.5)]
    assert torch.equal(got[0], ops.attention_decode_shared(**c))
    _check(got[1], {**c, "q": c["q"] * 0.5})
    narrow = {**c, "block_table": c["block_table"][:, :-1]}
    with pytest.raises(ValueError, match="other sizes"):
        ops.attention_decode_shared(**narrow, plan=plan)


@gpu
@torch.inference_mode()      # as the engine captures: one kind of capture for a process
def test_captured_steps_follow_lengths_and_leaders():
    """Two graphs over one set of buffers, replayed in turn with other lengths, groups and eager
    work between."""
    first, second = GROUPS["two groups and strangers"], [(0, 12, 400 + i) for i in range(8)]
    cases = [_case(first, seed=16), _case(second, seed=17)]
    width = max(c["block_table"].shape[1] for c in cases)
    pages = max(c["k_cache"].shape[0] for c in cases)
    buf = {x: torch.zeros_like(cases[0][x]) for x in ("q", "seq_lens", "leaders", "shared")}
    buf["block_table"] = torch.zeros(8, width, dtype=torch.int32, device=DEVICE)
    for x in ("k_cache", "v_cache"):
        buf[x] = torch.zeros(pages, *cases[0][x].shape[1:], dtype=torch.bfloat16, device=DEVICE)

    def fill(c):
        for x, t in c.items():
            if x == "block_table":
                buf[x][:, : t.shape[1]] = t
            elif x.endswith("cache"):
                buf[x][: t.shape[0]] = t
            else:
                buf[x].copy_(t)

    fill(cases[0])
    ops.attention_decode_shared(**buf)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.attention_decode_shared(**buf)
        graphs.append((g, out))
    for turn in range(6):
        c = cases[turn % 2]
        fill(c)
        for g, out in graphs:
            g.replay()
            _check(out, c)
            eager = ops.attention_decode_shared(**{**buf, "seq_lens": buf["seq_lens"].clone()})
            assert torch.equal(eager, out)


@gpu
def test_other_stream():
    c = _case(GROUPS["ragged"], seed=18)
    want = ops.attention_decode_shared(**c)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [ops.attention_decode_shared(**c) for _ in range(4)]
    here = ops.attention_decode_shared(**c)
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in (*got, here))


@gpu
def test_random_batches():
    gen = torch.Generator().manual_seed(19)
    pick = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=gen))  # noqa: E731
    for turn in range(25):
        rows, leads = [], []
        for b in range(pick(1, 40)):
            if leads and pick(0, 3):
                lead, pages = leads[pick(0, len(leads) - 1)]
                rows.append((lead, pages, max(0, pages * 16 + pick(-20, 200))))
            else:
                pages = pick(0, 30)
                leads.append((b, pages))
                rows.append((b, pages, pages * 16 + pick(1, 200)))
        group, Hk = pick(1, 9), pick(1, 4)
        c = _case(rows, group * Hk, Hk, (64, 128)[turn % 2], 16, (torch.bfloat16, torch.float16)[turn // 2 % 2],
                  seed=100 + turn)
        print("turn", turn, len(rows), group, Hk, flush=True)
        _check(ops.attention_decode_shared(**c), c)


# -- refusals ----------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("change,what", [
    (lambda c: c.update(q=c["q"].float()), "16-bit"),
    (lambda c: c.update(v_cache=c["v_cache"].half()), "16-bit"),
    (lambda c: c.update(q=c["q"][:, :3]), "equal groups"),
    (lambda c: c.update(q=c["q"][..., :64]), "channels"),
    (lambda c: c.update(q=c["q"][0]), "B, Hq, D"),
    (lambda c: c.update(k_cache=c["k_cache"][1:]), "B, Hq, D"),
    (lambda c: c.update(block_table=c["block_table"].long()), "int32"),
    (lambda c: c.update(block_table=c["block_table"][:, ::2]), "side by side"),
    (lambda c: c.update(block_table=c["block_table"][1:]), "rows"),
    (lambda c: c.update(seq_lens=c["seq_lens"].long()), "seq_lens"),
    (lambda c: c.update(leaders=c["leaders"][1:]), "leaders"),
    (lambda c: c.update(shared=c["shared"].cpu()), "one device"),
    (lambda c: c.update(k_cache=c["k_cache"][:, :24], v_cache=c["v_cache"][:, :24]), "power of 2"),
    (lambda c: c.update(q=torch.empty(4 * 8 * 128 + 4, dtype=torch.bfloat16, device=DEVICE)[4:].view(4, 8, 128)),
     "16 bytes"),
    (lambda c: c.update(v_cache=c["v_cache"].cpu()), "one device"),
    (lambda c: c.update(block_table=torch.zeros(4, 2 ** 18, dtype=torch.int32, device=DEVICE),
                        **{x: c[x][:1, :1].expand(1, 2 ** 16, 8 // 4, 128) for x in ("k_cache", "v_cache")}), "2.35 tokens"),
])
def test_refused(change, what):
    c = _case(GROUPS["ragged"], seed=20)
    change(c)
    with pytest.raises(ValueError, match=what):
        ops.attention_decode_shared(**c)


@gpu
def test_gradients_are_refused():
    c = _case(GROUPS["ragged"], seed=20)
    c["q"].requires_grad_()
    with pytest.raises(RuntimeError, match="gradients"):
        ops.attention_decode_shared(**c)
    with torch.no_grad():
        ops.attention_decode_shared(**c)


# -- the plain form ----------------------------------------------------------------------------
@pytest.mark.parametrize("name", ["one token", "ragged", "two groups and strangers", "rows without keys"])
def test_plain_form(name):
    c = _case(GROUPS[name], 4, 2, 16, 32, torch.float32, seed=3, device="cpu")
    want, _ = _exact(c)
    got = ops.attention_decode_shared(**c)
    assert torch.allclose(got.double(), want, atol=1e-5)
    live = c["seq_lens"] > 0
    paged = torch_ref.attention_decode_paged(
        c["q"][live], c["k_cache"].nan_to_num(0), c["v_cache"].nan_to_num(0),
        c["block_table"][live].clamp(min=0), c["seq_lens"][live], None)
    assert torch.allclose(got[live], paged, atol=1e-5)
    assert ops.shared_decode_plan(c["seq_lens"], c["leaders"], c["shared"], (4, 2), 16, 9, 32) is None


# -- the library ---------------------------------------------------------------------------------
@pytest.mark.skipif(shutil.which("hipcc") is None, reason="no hipcc")
@pytest.mark.parametrize("name", ["attention_shared.hip", "kv_pages.hip"])
def test_kernels_use_no_scratch(name, tmp_path):
    """Scratch reads would wait for every transfer that is under way."""
    from opsagent_amd.ops import build

    done = subprocess.run(
        [build.HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", *build.HIP_FLAGS, "-c",
         "-Rpass-analysis=kernel-resource-usage", os.path.join(build.CSRC, name), "-o",
         str(tmp_path / "x.o")], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    scratch = re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", done.stderr)
    assert scratch and set(scratch) == {"0"}


def test_entry_points():
    lib = os.path.join(os.path.dirname(ops.__file__), "libopsagent_kernels.so")
    if not os.path.exists(lib):
        pytest.skip("kernel library not built")
    for name in ("oa_shared_plan_size", "oa_shared_plan", "oa_attention_decode_shared", "oa_kv_pages_copy"):
        assert hasattr(ctypes.CDLL(lib), name), name


def test_entries_check_what_they_are_given():
    """Sizes that no launch takes, and pointers that it would not read right, come back as errors
    before anything is launched."""
    path = os.path.join(os.path.dirname(ops.__file__), "libopsagent_kernels.so")
    if not os.path.exists(path):
        pytest.skip("kernel library not built")
    from opsagent_amd.ops import hip_lib

    lib = ctypes.CDLL(path)
    hip_lib._declare(lib)
    ints, slots = ctypes.c_int(), ctypes.c_int()
    size = lambda *s: lib.oa_shared_plan_size(*s, ctypes.byref(ints), ctypes.byref(slots))  # noqa: E731
    assert size(4, 32, 8, 128) == 0 and ints.value > 0 and slots.value > 0
    for bad in [(0, 32, 8, 128), (2049, 32, 8, 128), (4, 32, 0, 128), (4, 30, 8, 128), (4, 32, 8, 96),
                (4, 129, 1, 64), (4, 4100, 4100, 64)]:
        assert size(*bad) == -100, bad
    good = [4096, 128, 262144, 1024, 128, 262144, 1024, 128, 9, 4, 32, 8, 128, 9, 50, 32, 0]
    call = lambda n, q=16, scratch=16: lib.oa_attention_decode_shared(  # noqa: E731
        None, q, 16, 16, 16, None, None, None, 16, scratch, 16, (ctypes.c_int64 * 17)(*n), 0.1)
    for at, value, rc in [(9, 0, -100), (9, -1, -100), (13, 0, -100), (14, 0, -100), (14, 2 ** 31, -100),
                          (15, 24, -101), (15, 0, -101), (13, 2 ** 29, -102), (15, 2 ** 30, -102), (0, 4092, -103), (4, 4, -103), (3, 2 ** 23, -105),
                          (6, -8, -105)]:
        n = list(good)
        n[at] = value
        assert call(n) == rc, (at, value)
    assert call(good, q=8) == -103 and call(good, scratch=20) == -103
    assert lib.oa_shared_plan(None, 16, 16, 16, 8, 4, 32, 8, 128, 9, 32) == -103
    assert lib.oa_shared_plan(None, 16, 16, 16, 16, 4, 32, 8, 128, 0, 32) == -100
    assert lib.oa_shared_plan(None, 16, 16, 16, 16, 4, 32, 8, 128, 9, 33) == -101
    assert lib.oa_shared_plan(None, 16, 16, 16, 16, 4, 32, 8, 128, 2 ** 29, 32) == -102
    bases = (ctypes.c_uint64 * 1)(4096)
    copy = lambda b, step, row, block, pages, c: lib.oa_kv_pages_copy(  # noqa: E731
        None, b, 1, step, row, block, pages, (ctypes.c_int * 3)(*c), 1)
    assert copy(bases, 512, 24, 8, 4, (0, 1, 8)) == -100
    assert copy(bases, 520, 32, 8, 4, (0, 1, 8)) == -100
    assert copy(bases, 512, 32, 0, 4, (0, 1, 8)) == -100
    assert copy(bases, 512, 2 ** 20, 2 ** 12, 4, (0, 1, 8)) == -101
    assert copy((ctypes.c_uint64 * 1)(4100), 512, 32, 8, 4, (0, 1, 8)) == -103
    for c in [(-1, 1, 8), (4, 1, 8), (0, -1, 8), (0, 4, 8), (0, 1, 9), (0, 1, -1)]:
        assert copy(bases, 512, 32, 8, 4, c) == -104
    assert copy(bases, 512, 32, 8, 4, (0, 1, 0)) == 0        # nothing to copy: nothing is launched
