"""Paged KV cache manager with block-level prefix caching.

The hipGraph-captured decode step is re-used across multi-turn ReAct iterations:
the loop at simple.go:394-615 re-sends full history each turn, and agent-turn
latency depends on KV that persists across tool-call turns.

Mechanism: the cache is a pool of fixed-size token blocks
([num_blocks, block_size, Hk_local, D] bf16 per layer, sized against the
288 GB of HBM3E per MI355X). Each FULL block of a sequence is content-hashed
by its chain hash (hash of all token ids up to and including the block);
completed blocks are published to a hash table. A new request reuses the
longest prefix of published blocks — so when the ReAct loop re-sends the
growing conversation, only the new suffix is prefilled. Freed blocks stay
cached (refcount 0) in LRU order and are evicted on allocation pressure.
"""

from __future__ import annotations

import collections
import itertools
from typing import Dict, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from opsagent_amd import ops


class BlockAllocatorError(RuntimeError):
    pass


class PagedKVCache:
    def __init__(
        self,
        num_layers: int,
        num_kv_heads_local: int,
        head_dim: int,
        block_size: int,
        num_blocks: int,
        device: str,
        dtype: torch.dtype = torch.bfloat16,
        layer_shapes: Optional[Sequence[Optional[Tuple[int, int, int]]]] = None,
        prefix_caching: bool = True,
    ):
        """layer_shapes (optional) gives each layer's own (kv_heads, key dim,
        value dim), or None for a layer that keeps no keys and values (a
        recurrent mixer, or a layer that reads another layer's cache); a
        fourth element "prefix" says that the values ARE the first `value
        dim` channels of the keys (one key head, or several of equal key and
        value size): the value tensor is then a view of the key rows and takes
        no memory; a fourth element "vheads"
        with a fifth n says that there are n value heads (n divides kv_heads:
        key head g reads value head g mod n). Without layer_shapes every
        layer is [kv_heads, head_dim] for both. prefix_caching=False turns block publishing and reuse off: a
        model that also carries recurrent state cannot restart from cached
        keys alone."""
        assert block_size & (block_size - 1) == 0, "block_size must be a power of 2"
        self.block_size = block_size
        self.num_blocks = num_blocks
        self.device = device
        self.prefix_caching = prefix_caching
        self.layers: List[Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]] = []
        if layer_shapes is None:
            layer_shapes = [(num_kv_heads_local, head_dim, head_dim)] * num_layers
        for shape in layer_shapes:
            if shape is None:
                self.layers.append((None, None))
                continue
            hk, kdim, vdim = shape[:3]
            k = torch.zeros(num_blocks, block_size, hk, kdim, dtype=dtype, device=device)
            if len(shape) > 3 and shape[3] == "prefix":
                assert vdim == kdim or (hk == 1 and vdim < kdim)
                v = k[..., :vdim]
            elif len(shape) > 4 and shape[3] == "vheads":
                assert hk % shape[4] == 0
                v = torch.zeros(num_blocks, block_size, shape[4], vdim, dtype=dtype,
                                device=device)
            else:
                v = torch.zeros(num_blocks, block_size, hk, vdim, dtype=dtype, device=device)
            self.layers.append((k, v))
        # allocator state
        self._free: collections.deque[int] = collections.deque(range(num_blocks))
        self._ref: List[int] = [0] * num_blocks
        # prefix cache: chain_hash -> block_id; and reverse for eviction.
        # _block_tokens keeps each published block's OWN token slice so a
        # 64-bit chain-hash collision cannot silently alias wrong KV: the
        # chain hash binds the ancestry, the stored slice verifies the
        # block's content (O(block_size) per block, not O(prefix)).
        self._hash_to_block: Dict[int, int] = {}
        self._block_to_hash: List[Optional[int]] = [None] * num_blocks
        self._block_tokens: List[Optional[Tuple[int, ...]]] = [None] * num_blocks
        # LRU of refcount-0 cached blocks (evictable)
        self._evictable: "collections.OrderedDict[int, None]" = collections.OrderedDict()
        self.stats = {"reused_blocks": 0, "allocated_blocks": 0, "evictions": 0}
        self._pages: Optional[ops.KVPages] = None
        self.switched = 0       # blocks that sequences gave up for an equal published one

    # -- contents of blocks -------------------------------------------------
    def copy_blocks(self, src: Sequence[int], dst: Sequence[int],
                    tokens: Optional[Sequence[int]] = None) -> None:
        """Keys and values of blocks src to blocks dst in all layers, or of their first tokens."""
        if len(src):
            if self._pages is None:
                self._pages = ops.KVPages([(k, v) if k is None else (k[: self.num_blocks], v[: self.num_blocks])
                                           for k, v in self.layers])
            ops.kv_cache_copy(self._pages, src, dst, tokens)

    def drop_cached(self, keep: int = 0) -> int:
        """Frees blocks that only the prefix cache holds, the longest unused first, until `keep` of
        them are left. Returns how many were freed."""
        drop = max(0, len(self._evictable) - max(0, keep))
        for _ in range(drop):
            bid, _ = self._evictable.popitem(last=False)
            self._forget(bid)
            self._free.append(bid)
        return drop

    def compact(self, sequences: Sequence["SequenceState"]) -> int:
        """Moves what is in use or cached to the first blocks, so that the rest of the pool is one
        run of free blocks; returns where that begins. `sequences` are all that hold blocks: their
        lists are changed. Nothing may be reading or writing the cache on another stream."""
        held = collections.Counter(b for seq in sequences for b in seq.blocks)
        if any(seq.cache is not self for seq in sequences) or any(
                self._ref[b] != held[b] for b in range(self.num_blocks)):
            raise ValueError("compacting takes every sequence that holds blocks of the cache")
        used = [b for b in range(self.num_blocks) if self._ref[b] or b in self._evictable]
        n, taken = len(used), set(used)
        src = [b for b in used if b >= n]
        dst = [b for b in range(n) if b not in taken]
        self.copy_blocks(src, dst)
        to = dict(zip(src, dst))
        for a, b in to.items():
            self._ref[a], self._ref[b] = 0, self._ref[a]
            self._block_tokens[a], self._block_tokens[b] = None, self._block_tokens[a]
            h, self._block_to_hash[a] = self._block_to_hash[a], None
            self._block_to_hash[b] = h
            if h is not None:
                self._hash_to_block[h] = b
        self._evictable = collections.OrderedDict((to.get(b, b), None) for b in self._evictable)
        self._free = collections.deque(range(n, self.num_blocks))
        for seq in sequences:
            seq.blocks = [to.get(b, b) for b in seq.blocks]
        return n

    def check_shrink(self, num_blocks: int) -> int:
        """Blocks in use. Raises what `shrink` does, where it would."""
        if not 0 < num_blocks <= self.num_blocks:
            raise ValueError(f"a pool of {self.num_blocks} blocks does not shrink to {num_blocks}")
        live = sum(1 for r in self._ref if r)
        if live > num_blocks:
            raise BlockAllocatorError(f"{live} blocks are in use, more than {num_blocks}")
        return live

    def shrink(self, num_blocks: int, sequences: Sequence["SequenceState"]) -> None:
        """Gives memory back: the pool becomes its first `num_blocks`, compacted, cached blocks that
        find no room dropped. Layers' tensors that are longer become new ones. Raises
        BlockAllocatorError where sequences hold more blocks than that. A layer that the device has
        no memory to shorten stays as it is, and so do those behind it, while the error goes on to the
        caller: the pool is sound, and can be shrunk again."""
        self.drop_cached(num_blocks - self.check_shrink(num_blocks))
        self.compact(sequences)
        # before the tensors: nobody names a block that one of them may lack
        del self._ref[num_blocks:], self._block_to_hash[num_blocks:], self._block_tokens[num_blocks:]
        self._free = collections.deque(b for b in self._free if b < num_blocks)
        self.num_blocks = num_blocks
        self._pages = None
        for i, (k, v) in enumerate(self.layers):
            if k is None or k.shape[0] == num_blocks:
                continue
            # layer by layer: the peak is one layer more than the pool
            prefix = v.data_ptr() == k.data_ptr()
            vdim, keys = v.shape[-1], k[:num_blocks].clone()
            values = keys[..., :vdim] if prefix else v[:num_blocks].clone()
            self.layers[i] = (keys, values)
            del k, v, keys, values

    # -- low-level allocator ----------------------------------------------
    def num_free(self) -> int:
        return len(self._free) + len(self._evictable)

    def _pop_free_block(self) -> int:
        if self._free:
            return self._free.popleft()
        if self._evictable:
            bid, _ = self._evictable.popitem(last=False)  # LRU
            self._forget(bid)
            self.stats["evictions"] += 1
            return bid
        raise BlockAllocatorError("KV cache out of blocks")

    def _forget(self, bid: int) -> None:
        """Takes a block out of the prefix cache's tables."""
        h = self._block_to_hash[bid]
        if h is not None:
            del self._hash_to_block[h]
            self._block_to_hash[bid] = None
            self._block_tokens[bid] = None

    def alloc_block(self) -> int:
        bid = self._pop_free_block()
        self._ref[bid] = 1
        self.stats["allocated_blocks"] += 1
        return bid

    def retain(self, bid: int) -> None:
        if self._ref[bid] == 0:
            self._evictable.pop(bid, None)
        self._ref[bid] += 1

    def release(self, bid: int) -> None:
        assert self._ref[bid] > 0
        self._ref[bid] -= 1
        if self._ref[bid] == 0:
            if self._block_to_hash[bid] is not None:
                self._evictable[bid] = None  # keep content for prefix reuse
            else:
                self._free.append(bid)

    # -- prefix cache -------------------------------------------------------
    @staticmethod
    def chain_hash(prev: int, ids: Sequence[int]) -> int:
        return hash((prev, tuple(ids)))

    def lookup_prefix(self, token_ids: Sequence[int]) -> Tuple[List[int], int]:
        """Longest reusable prefix. Returns (block_ids retained, n_tokens).

        Never reuses the entire prompt: at least one token must be recomputed
        so the engine has a last-token hidden state to sample from.
        """
        bs = self.block_size
        blocks: List[int] = []
        h = 0
        if not self.prefix_caching:
            return blocks, 0
        max_full = (len(token_ids) - 1) // bs  # leave ≥1 token to prefill
        for i in range(max_full):
            h = self.chain_hash(h, token_ids[i * bs : (i + 1) * bs])
            bid = self._hash_to_block.get(h)
            if bid is None:
                break
            # collision guard: the hash indexes, token equality decides
            if self._block_tokens[bid] != tuple(token_ids[i * bs : (i + 1) * bs]):
                break
            blocks.append(bid)
        for bid in blocks:
            self.retain(bid)
        self.stats["reused_blocks"] += len(blocks)
        return blocks, len(blocks) * bs

    def publish_block(
        self, bid: int, chain_h: int, prefix_tokens: Tuple[int, ...]
    ) -> int:
        """Publish a full block under its chain hash. If an identical block
        (hash AND token-verified) is already cached, switch to it (dedup) and
        release ours. Returns the canonical block id."""
        existing = self._hash_to_block.get(chain_h)
        if existing is not None and existing != bid:
            if self._block_tokens[existing] == prefix_tokens:
                self.retain(existing)
                self.release(bid)
                self.switched += 1
                return existing
            # hash collision with DIFFERENT content: evict the stale entry
            self._block_to_hash[existing] = None
            self._block_tokens[existing] = None
        self._hash_to_block[chain_h] = bid
        self._block_to_hash[bid] = chain_h
        self._block_tokens[bid] = prefix_tokens
        return bid


class StateSlotPool:
    """Fixed-size per-sequence state beside the paged keys and values: the
    recurrent matrix of a delta-rule mixer and the last inputs of causal
    short convolutions. One slot per live sequence; a slot is handed out at
    admission and returned when the sequence ends or is preempted.

    A slot is NOT cleared when it is reused: every kernel that reads state
    takes the sequence's start position and treats everything before
    position 0 as zero, so stale contents are never observed (and nothing
    has to be memset inside a captured graph).

    tensors[layer][name] is [num_slots, *shape] float32.
    """

    def __init__(self, num_slots: int, layer_shapes: Sequence[Dict[str, Tuple[int, ...]]],
                 device: str):
        self.num_slots = num_slots
        self.tensors: List[Dict[str, torch.Tensor]] = []
        for shapes in layer_shapes:
            self.tensors.append({
                name: torch.zeros(num_slots, *shape, dtype=torch.float32, device=device)
                for name, shape in shapes.items()
            })
        self._free: collections.deque[int] = collections.deque(range(num_slots))

    def num_free(self) -> int:
        return len(self._free)

    def alloc(self) -> int:
        if not self._free:
            raise BlockAllocatorError("out of state slots")
        return self._free.popleft()

    def release(self, slot: int) -> None:
        assert 0 <= slot < self.num_slots and slot not in self._free
        self._free.append(slot)


def shared_prefixes(
    tables: Union[np.ndarray, Sequence[Sequence[int]]], full: Sequence[int]
) -> Tuple[List[int], List[int], int]:
    """Which rows of a batch begin with the same blocks, as ops.attention_decode_shared takes it:
    (leaders, shared, saved). `tables`: block ids of each row, lists or the rows of a block table;
    `full`: how many of them are full.
    Rows are grouped so that the blocks read once instead of once a row are as many as one level of
    groups allows; `saved` is their number."""
    n = len(full)
    leaders, shared, saved = list(range(n)), [0] * n, 0
    # as arrays: 128 rows of 512 common blocks take 0.2 ms, block by block 5
    counts = np.asarray(full, np.int64)
    ids = np.full((n, max(full, default=0)), -1, np.int32)
    for b, count in enumerate(full):
        ids[b, :count] = tables[b][:count]
    # in the order of their bytes, where rows with blocks in common are neighbours
    rows_bytes = [row.tobytes() for row in ids]
    order = sorted(range(n), key=rows_bytes.__getitem__)
    # blocks in common of neighbours in that order; of a run of rows, the least of them
    common: List[int] = []
    if n > 1 and ids.shape[1]:
        ids, counts = ids[order], counts[order]
        differ = ids[1:] != ids[:-1]
        same = np.where(differ.any(1), differ.argmax(1), ids.shape[1])
        common = np.minimum(same, np.minimum(counts[1:], counts[:-1])).tolist()

    # Runs of rows with blocks in common are a tree, run 0 all rows. Of each run: blocks in common,
    # the run around it, rows that are in no run within it; and the runs, the inner ones first.
    least, outer, own_rows = [0], [-1], [[]]
    inner_first, under = [], [0]

    def begin(blocks: int) -> None:
        under.append(len(least))
        least.append(blocks)
        outer.append(-1)
        own_rows.append([])

    for b, ahead in zip(order, [*common, 0]):
        if ahead > least[under[-1]]:
            begin(ahead)
        own_rows[under[-1]].append(b)
        while least[under[-1]] > ahead:
            run = under.pop()
            if least[under[-1]] < ahead:
                begin(ahead)            # a run that begins where this one did and goes on
            outer[run] = under[-1]
            inner_first.append(run)

    # A group reads its blocks once, and each of its rows less by as many. A run is a group or not, and
    # rows go to the nearest group around them. What a run saves hangs on the group around it: `around`
    # has the blocks of the runs that may be that, from the outside, and `saves` what its rows save in
    # a group of each, or in better ones within; the last is the run itself.
    around, saves = {0: np.zeros(1, np.int64)}, {}
    for run in reversed(inner_first):
        around[run] = np.append(around[outer[run]], least[run])
        saves[run] = len(own_rows[run]) * around[run]
    saves[0] = np.zeros(1, np.int64)
    for run in inner_first:
        saves[outer[run]] += np.maximum(saves[run][:-1], saves[run][-1] - least[run])
    # (blocks, rows) of the groups; of each run the place of its group in `around`, and the group's rows
    groups: List[Tuple[int, List[int]]] = []
    place: Dict[int, Tuple[int, List[int]]] = {0: (0, [])}
    for run in reversed(inner_first):
        at, rows = place[outer[run]]
        if saves[run][-1] - least[run] > saves[run][at]:
            at, rows = len(around[run]) - 1, []
            groups.append((least[run], rows))
        rows += own_rows[run]
        place[run] = at, rows
    for pages, rows in groups:
        if len(rows) > 1:
            saved += (len(rows) - 1) * pages
            lead = min(rows)
            for b in rows:
                leaders[b], shared[b] = lead, pages
    return leaders, shared, saved


_SERIAL = itertools.count()


class SequenceState:
    """Per-sequence cache bookkeeping."""

    def __init__(self, cache: PagedKVCache, token_ids: List[int],
                 state_pool: Optional[StateSlotPool] = None):
        self.cache = cache
        self.state_pool = state_pool
        # recurrent/convolution state slot (None for pure-attention models)
        self.state_slot: Optional[int] = (
            state_pool.alloc() if state_pool is not None else None
        )
        self.token_ids = list(token_ids)  # prompt + generated
        self.blocks: List[int] = []
        self.num_cached = 0     # tokens whose KV is in cache
        self.chain_h = 0        # chain hash over published full blocks
        self.published = 0      # number of full blocks published
        self.serial = next(_SERIAL)   # tells sequences apart, also those of one request

    def fork(self, count: int) -> Tuple["SequenceState", Optional[Tuple[int, int, int]]]:
        """A sequence of its own that begins with the first `count` tokens of this one and has the
        keys of all but the last of them: it shares the blocks that are full before that token, and
        has a copy of the block that the token lies in, which it writes into. Returns it, and that
        copy as (source, target, tokens) for PagedKVCache.copy_blocks, None where nothing is copied.
        The copy has to be made before either sequence writes keys again."""
        if self.state_pool is not None:
            raise ValueError("recurrent state does not fork")
        if not 0 < count <= min(len(self.token_ids), self.num_cached + 1):
            raise ValueError(f"a fork at token {count} of {len(self.token_ids)}, {self.num_cached} with keys")
        cache, bs = self.cache, self.cache.block_size
        keep, used = divmod(count - 1, bs)
        target = cache.alloc_block() if used else None
        child = SequenceState(cache, self.token_ids[:count])
        child.blocks = self.blocks[:keep]
        for bid in child.blocks:
            cache.retain(bid)
        child.num_cached = count - 1
        child.published = min(self.published, keep)
        for i in range(child.published):
            child.chain_h = cache.chain_hash(child.chain_h, child.token_ids[i * bs : (i + 1) * bs])
        if target is None:
            return child, None
        child.blocks.append(target)
        return child, (self.blocks[keep], target, used)

    def reuse_prefix(self) -> int:
        blocks, n = self.cache.lookup_prefix(self.token_ids)
        self.blocks = blocks
        self.num_cached = n
        self.published = len(blocks)
        h = 0
        bs = self.cache.block_size
        for i in range(len(blocks)):
            h = self.cache.chain_hash(h, self.token_ids[i * bs : (i + 1) * bs])
        self.chain_h = h
        return n

    def ensure_capacity(self, n_tokens: int) -> None:
        bs = self.cache.block_size
        need = (n_tokens + bs - 1) // bs
        while len(self.blocks) < need:
            self.blocks.append(self.cache.alloc_block())

    def slots_for(self, start: int, count: int) -> torch.Tensor:
        """Flat slot ids for token positions [start, start+count)."""
        bs = self.cache.block_size
        out = torch.empty(count, dtype=torch.int32)
        for i in range(count):
            pos = start + i
            out[i] = self.blocks[pos // bs] * bs + pos % bs
        return out

    def all_slots(self, upto: int) -> torch.Tensor:
        return self.slots_for(0, upto)

    def publish_full_blocks(self) -> None:
        """Publish newly-completed full blocks to the prefix cache."""
        if not self.cache.prefix_caching:
            return
        bs = self.cache.block_size
        full = self.num_cached // bs
        while self.published < full:
            i = self.published
            self.chain_h = self.cache.chain_hash(
                self.chain_h, self.token_ids[i * bs : (i + 1) * bs]
            )
            self.blocks[i] = self.cache.publish_block(
                self.blocks[i], self.chain_h,
                tuple(self.token_ids[i * bs : (i + 1) * bs]),
            )
            self.published += 1

    def free(self) -> None:
        for bid in self.blocks:
            self.cache.release(bid)
        self.blocks = []
        if self.state_slot is not None:
            self.state_pool.release(self.state_slot)
            self.state_slot = None
