"""Copies of cache pages in all layers at once: exact, and nothing beside them changes."""

import pytest
import torch

from opsagent_amd import ops

gpu = pytest.mark.gpu


def _layers(device, shapes, pages=12, block=8, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator().manual_seed(seed)
    new = lambda h, d: torch.randn(pages, block, h, d, generator=gen).to(device, dtype)  # noqa: E731
    layers = []
    for s in shapes:
        if s is None:
            layers.append((None, None))
        elif len(s) == 3:                     # values are the first channels of the keys
            k = new(s[0], s[1])
            layers.append((k, k[..., : s[2]]))
        else:
            layers.append((new(*s), new(*s)))
    return layers


def _expect(layers, src, dst, tokens):
    want = []
    for pair in layers:
        for t in pair:
            if t is not None:
                w = t.clone()
                for i, (a, b) in enumerate(zip(src, dst)):
                    n = t.shape[1] if tokens is None else tokens[i]
                    w[b, :n] = t[a, :n]
                want.append(w)
    return want


def _run(device, shapes, src, dst, tokens=None, **kw):
    layers = _layers(device, shapes, **kw)
    want = _expect(layers, src, dst, tokens)
    ops.kv_cache_copy(ops.KVPages(layers), src, dst, tokens)
    got = [t for pair in layers for t in pair if t is not None]
    for g, w in zip(got, want):
        assert torch.equal(g.view(torch.int16) if g.dtype != torch.float32 else g,
                           w.view(torch.int16) if w.dtype != torch.float32 else w)


CASES = [
    ([3], [5], None),
    ([3], [5], [1]),
    ([3, 3, 3], [5, 0, 11], [8, 0, 7]),
    ([0, 1, 2, 3], [8, 9, 10, 11], [5, 8, 0, 1]),
    ([], [], None),
    ([2], [4], [0]),
]
SHAPES = [[(2, 128)], [(2, 16), None, (2, 16)], [(1, 64, 32), (4, 8)], [(8, 128)] * 5]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("src,dst,tokens", CASES)
def test_copies(device, shapes, src, dst, tokens):
    _run(device, shapes, src, dst, tokens)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_types(dtype):
    _run("cuda", [(2, 64)] * 3, [0, 7], [9, 3], [8, 3], dtype=dtype)


@gpu
@pytest.mark.parametrize("block,heads,dim", [(1, 1, 8), (64, 8, 128), (32, 5, 72), (256, 2, 64)])
def test_sizes_of_a_page(block, heads, dim):
    _run("cuda", [(heads, dim)] * 3, [0, 1, 1], [9, 3, 4], [block, (block + 1) // 2, 1], block=block)


@gpu
def test_more_tensors_and_copies_than_a_launch_carries():
    _run("cuda", [(1, 8)] * 101, list(range(200)), list(range(399, 199, -1)),
         [i % 5 for i in range(200)], pages=400, block=4)


@gpu
def test_pages_apart():
    """Keys and values of a page beside each other, and a cache past 2^32 bytes."""
    both = torch.randn(9, 2, 8, 2, 64, device="cuda").bfloat16()
    want = both.clone()
    want[7, :, :5] = both[2, :, :5]
    ops.kv_cache_copy(ops.KVPages([(both[:, 0], both[:, 1])]), [2], [7], [5])
    assert torch.equal(both, want)
    pages = 2 ** 32 // (64 * 8 * 128 * 2) + 9
    big = torch.zeros(pages, 64, 8, 128, dtype=torch.bfloat16, device="cuda")
    big[3] = torch.randn(64, 8, 128, device="cuda").bfloat16()
    table = ops.KVPages([(big, None)])
    ops.kv_cache_copy(table, [3], [pages - 1])
    ops.kv_cache_copy(table, [pages - 1], [1], [33])
    assert torch.equal(big[pages - 1], big[3]) and torch.equal(big[1, :33], big[3, :33])
    assert not big[1, 33:].any() and not big[pages - 2].any() and not big[0].any()


@gpu
@torch.inference_mode()      # as the engine captures: one kind of capture for a process
def test_captured():
    layers = _layers("cuda", [(2, 64)] * 2)
    table = ops.KVPages(layers)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv_cache_copy(table, [1, 2], [8, 9], [8, 3])
    for turn in range(3):
        for k, v in layers:
            k.add_(1.0)
            v.mul_(0.5)
        want = _expect(layers, [1, 2], [8, 9], [8, 3])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([t for p in layers for t in p], want))


@pytest.mark.parametrize("src,dst,tokens,error,what", [
    ([1], [2, 3], None, ValueError, "targets"),
    ([1], [2], [1, 2], ValueError, "tokens"),
    ([12], [2], None, ValueError, "outside"),
    ([-1], [2], None, ValueError, "outside"),
    ([1], [12], None, ValueError, "outside"),
    ([1], [2], [9], ValueError, "of 8 tokens"),
    ([1], [2], [-1], ValueError, "of 8 tokens"),
    ([1, 2], [3, 3], None, ValueError, "two copies"),
    ([1, 2], [2, 4], None, ValueError, "the target of another"),
    ([1], [1], None, ValueError, "the target of another"),
    ([1.0], [2], None, TypeError, "ints"),
    (torch.tensor([1]), torch.tensor([2]), None, TypeError, "ints"),
])
def test_refused(src, dst, tokens, error, what):
    layers = _layers("cpu", [(2, 16)])
    before = [t.clone() for t in layers[0]]
    with pytest.raises(error, match=what):
        ops.kv_cache_copy(ops.KVPages(layers), src, dst, tokens)
    assert all(torch.equal(a, b) for a, b in zip(before, layers[0]))


def test_tables_refused():
    k = torch.zeros(4, 8, 2, 16)
    for layers, what in [([], "without tensors"), ([(None, None)], "without tensors"),
                         ([(k, torch.zeros(5, 8, 2, 16))], "one number of pages"),
                         ([(k, torch.zeros(4, 4, 2, 16))], "one number of pages"),
                         ([(k, torch.zeros(4))], "one number of pages"),
                         ([(k.transpose(1, 2), None)], "dense"),
                         ([(k[:1].expand(4, 8, 2, 16), None)], "dense")]:
        with pytest.raises(ValueError, match=what):
            ops.KVPages(layers)


@gpu
def test_tables_refused_on_the_gpu():
    with pytest.raises(ValueError, match="2 GiB"):
        ops.KVPages([(torch.empty(1, 2 ** 27, 16, device="cuda", dtype=torch.uint8), None)])
    with pytest.raises(ValueError, match="16 bytes"):
        ops.KVPages([(torch.zeros(4, 8, 1, 6, dtype=torch.bfloat16, device="cuda"), None)])
    with pytest.raises(ValueError, match="cuda"):
        ops.KVPages([(torch.zeros(4, 8, 16), torch.zeros(4, 8, 16, device="cuda"))])


def test_same_tensor_twice_is_copied_once():
    k = torch.arange(4 * 8 * 2, dtype=torch.float32).view(4, 8, 2)
    table = ops.KVPages([(k, None), (None, k), (k, k)])
    assert len(table.tensors) == 1
