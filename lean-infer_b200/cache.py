"""Paged KV pool and block allocator with the reference engine's layout.

Mirrors leaninfer/engine/cache_manager.py:
  * BlockAllocator (cache_manager.py:13-42): FIFO free list of block ids
    1..num_blocks-1; block 0 is the trash block that idle CUDA-graph rows
    write into (cache_manager.py:20-25).
  * BlockCache (cache_manager.py:45-76): two bf16 pools
    [num_layers, num_blocks, block_size, num_kv_heads, head_dim]; write()
    scatters k, v [B, Hkv, q_len, D] to block_table[b, col // BS], col % BS,
    col = pos[b] + t. Here write() runs the paged-write kernel instead of
    torch advanced indexing; the result is bit-identical (a copy).

Beyond the reference, whose requests never share a block, blocks may have
several holders: BlockCache.fork lets sequences share the whole blocks of a
common prefix (flash_attn_with_shared_prefix reads those once for all of
them), release gives a block back when its last holder does, and
BlockCache.compact moves the used blocks to the lowest ids. copy_blocks and
move_blocks are the device side.
"""
from __future__ import annotations

from collections import deque
from typing import Optional, Sequence

import torch

from . import _lib
from .flash_attn_interface import _check, _device_index, _raw_stream, ensure_init, error_word, paged_kv_write


def blocks_for(n_tokens: int, block_size: int) -> int:
    """Blocks needed to hold n_tokens (ceil division), cache_manager.py:7-9."""
    return -(-n_tokens // block_size)


class InsufficientBlocksError(RuntimeError, AssertionError):
    """allocate(n) with fewer than n free blocks. The reference signals this
    with an assert (cache_manager.py:38, an AssertionError); this error is an
    AssertionError too, so callers catching that keep working, and a
    RuntimeError like the package's other errors. It is raised under -O as
    well, where the reference's assert would vanish."""


class BlockAllocator:
    """FIFO free list of physical block ids; block 0 is reserved as trash.
    A block may have several holders (fork); it returns to the free list when
    the last one releases it."""

    def __init__(self, num_blocks: int) -> None:
        self.free: deque[int] = deque(range(1, num_blocks))
        self._holders: dict[int, int] = {}  # blocks handed out

    @property
    def num_free(self) -> int:
        return len(self.free)

    def allocate(self, n: int) -> list[int]:
        if n > len(self.free):
            raise InsufficientBlocksError(f"Insufficient free blocks: asked {n}, free {len(self.free)}")
        blocks = [self.free.popleft() for _ in range(n)]
        for b in blocks:
            self._holders[b] = 1
        return blocks

    def fork(self, blocks: Sequence[int]) -> None:
        """One more holder for each of `blocks`, all of which must be in use."""
        missing = [b for b in blocks if b not in self._holders]
        if missing:
            raise ValueError(f"blocks {missing} are not in use")
        for b in blocks:
            self._holders[b] += 1

    def holders(self, block: int) -> int:
        """Holders of a block: 0 for a free one."""
        return self._holders.get(block, 0)

    def release(self, blocks: list[int]) -> None:
        """One holder less for each of `blocks`; those that nobody holds any
        more go to the tail of the free list. Refused as a whole where a block
        has fewer holders than that: it would be handed out twice."""
        left: dict[int, int] = {}
        for b in blocks:
            left[b] = left.get(b, self._holders.get(b, 0)) - 1
        over = [b for b, n in left.items() if n < 0]
        if over:
            raise ValueError(f"blocks {over} are released more often than they are held")
        for b in blocks:
            self._holders[b] -= 1
            if self._holders[b] == 0:
                del self._holders[b]
                self.free.append(b)

    def compact(self) -> tuple[list[int], list[int]]:
        """Renumber the used blocks into the lowest ids: returns (src, dst),
        used blocks and the free ids below them that they take. The pages have
        to be moved and every table rewritten before either is used again
        (BlockCache.compact does both)."""
        moves = []
        for s, d in zip(sorted(self._holders, reverse=True), sorted(set(self.free))):
            if d >= s:
                break
            moves.append((s, d))
        if not moves:
            return [], []
        src, dst = (list(x) for x in zip(*moves))
        self.free = deque(sorted(set(self.free).difference(dst).union(src)))
        for s, d in moves:
            self._holders[d] = self._holders.pop(s)
        return src, dst


def _pools(k_pool: torch.Tensor, v_pool: torch.Tensor) -> tuple:
    """The pools as la_copy_blocks takes them, from [L, NB, BS, Hkv, D] or one
    layer's [NB, BS, Hkv, D]."""
    shape, stride = k_pool.shape, k_pool.stride()
    if (len(shape) not in (4, 5) or shape != v_pool.shape or stride != v_pool.stride()
            or k_pool.dtype is not v_pool.dtype or k_pool.get_device() != v_pool.get_device()):
        raise RuntimeError("k_pool and v_pool must be [num_layers, num_blocks, block_size, num_heads_k, head_dim] (or one "
                           "layer) of the same shape, strides and type on one device")
    if stride[-1] != 1:
        raise RuntimeError("the head_dim axis must be contiguous")
    if len(shape) == 4:
        return (k_pool.data_ptr(), v_pool.data_ptr(), 0, *stride[:3], 1, *shape, k_pool.element_size())
    return (k_pool.data_ptr(), v_pool.data_ptr(), *stride[:4], *shape, k_pool.element_size())


def _ids(name: str, ids: torch.Tensor, n: int, dev: int) -> int:
    if ids.dtype is not torch.int32 or ids.shape != (n,) or not ids.is_contiguous() or ids.get_device() != dev:
        raise RuntimeError(f"{name} must be a contiguous int32 [num_pairs] tensor on the pools' device")
    return ids.data_ptr()


def _check_table(block_table: torch.Tensor, device: torch.device) -> None:
    _check(block_table.dtype is torch.int32 and block_table.dim() == 2 and block_table.device == device
           and block_table.stride(1) == 1 and (block_table.shape[0] < 2 or block_table.stride(0) >= block_table.shape[1]),
           "block_table must be row-contiguous int32 [batch, max_blocks] on the pools' device")


def copy_blocks(k_pool: torch.Tensor, v_pool: torch.Tensor, src_blocks: torch.Tensor, dst_blocks: torch.Tensor,
                num_tokens: Optional[torch.Tensor] = None) -> None:
    """Copy pages inside the pools: in every layer, K and V, the first
    num_tokens[i] tokens of block src_blocks[i] (all of them without
    num_tokens) to block dst_blocks[i], in one launch.

    k_pool / v_pool: [L, NB, BS, Hkv, D] or one layer's [NB, BS, Hkv, D], of
    any type of 1, 2 or 4 bytes. src_blocks, dst_blocks, num_tokens: int32 [n]
    on the pools' device, read there. One block may be the source of several
    copies. A copy whose destination is another's source, or the destination
    of one before it, is skipped and recorded, as are ids outside the pool
    (check_device_errors)."""
    args = _pools(k_pool, v_pool)
    n = src_blocks.numel()
    dev = k_pool.get_device() if k_pool.is_cuda else _device_index(k_pool)
    src, dst = _ids("src_blocks", src_blocks, n, dev), _ids("dst_blocks", dst_blocks, n, dev)
    tokens = _ids("num_tokens", num_tokens, n, dev) if num_tokens is not None else None
    with torch.cuda.device(dev):
        ensure_init(dev)
        _lib.call("la_copy_blocks", *args, src, dst, tokens, n, error_word(dev).data_ptr(), _raw_stream(dev))


def move_blocks(k_pool: torch.Tensor, v_pool: torch.Tensor, src_blocks: torch.Tensor, dst_blocks: torch.Tensor,
                block_table: torch.Tensor) -> None:
    """Move pages inside the pools: copy_blocks of whole pages, and every entry
    src_blocks[i] of block_table (int32 [B, max_blocks] on the pools' device,
    rewritten in place) becomes dst_blocks[i]. Entries of a move that is
    skipped (see copy_blocks) stay as they are."""
    args = _pools(k_pool, v_pool)
    n = src_blocks.numel()
    dev = k_pool.get_device() if k_pool.is_cuda else _device_index(k_pool)
    src, dst = _ids("src_blocks", src_blocks, n, dev), _ids("dst_blocks", dst_blocks, n, dev)
    _check_table(block_table, k_pool.device)
    rows, cols = block_table.shape
    with torch.cuda.device(dev):
        ensure_init(dev)
        _lib.call("la_move_blocks", *args, src, dst, n,
                  block_table.data_ptr(), block_table.stride(0) if rows > 1 else cols, rows, cols,
                  error_word(dev).data_ptr(), _raw_stream(dev))


def _common_blocks(a: list[int], b: list[int]) -> int:
    """Blocks that two rows begin with."""
    n = min(len(a), len(b))
    if a[:n] == b[:n]:
        return n
    same, differ = 0, n  # a[:same] and b[:same] are the same, a[:differ] and b[:differ] differ
    while differ - same > 1:
        mid = (same + differ) // 2
        if a[same:mid] == b[same:mid]:
            same = mid
        else:
            differ = mid
    return same


def shared_prefix_groups(tables: Sequence[Sequence[int]], lengths: Sequence[int], block_size: int,
                         min_blocks: int = 1) -> tuple[list[int], list[int]]:
    """The groups that flash_attn_with_shared_prefix takes, from the rows'
    block tables: (prefix_lens, cu_prefix_rows). A group is a run of rows whose
    tables begin with the same blocks, filled by all of them; its prefix is as
    many of those as all have. Where rows share more with some neighbours than
    with others (one system prompt, several documents behind it), the rows are
    divided so that the fewest blocks are read, a prefix once for its group and
    the other blocks once for each row; every group counts as one block read
    for what it costs by itself. Every row is in a group: one that shares fewer
    than min_blocks blocks with its neighbours is a group by itself, with a
    prefix of 0."""
    least = max(min_blocks, 1)
    rows = [list(t[: max(n, 0) // block_size]) for t, n in zip(tables, lengths)]
    n = len(rows)
    # Blocks common to rows i - 1 and i; 0 where no group may reach across.
    common = [0] + [_common_blocks(a, b) for a, b in zip(rows, rows[1:])] + [0]
    common = [c if c >= least else 0 for c in common]
    # Places where the best division may have to cut. Two rows that have as much
    # in common as either has with its other neighbour stay together: of a cut
    # between them, the row beside it on the side whose group shares less goes
    # over to the other group, which goes on sharing as much, and saves no less.
    cuts = [0] + [i for i in range(1, n) if common[i] == 0 or common[i] < max(common[i - 1], common[i + 1])] + [n]
    every = 1 << 62
    inside = [min(common[a + 1:b], default=every) for a, b in zip(cuts, cuts[1:])]
    # best[j]: blocks saved, less groups made, of the rows before cuts[j]; last[j]: where their last group begins, its prefix
    best, last = [0], [(0, 0)]
    for j in range(1, len(cuts)):
        shared, saved = every, None
        for i in range(j - 1, -1, -1):
            shared, size = min(shared, inside[i]), cuts[j] - cuts[i]
            here = best[i] + (size - 1) * shared - 1
            if saved is None or here >= saved:
                saved, at, prefix = here, i, shared if size > 1 else 0
            # From further back on it shares no more than `shared`. What rows in
            # front of cuts[i] save in it they would save, but for one row, as a
            # group by themselves, and best[i] is no less than with that one.
            shared = min(shared, common[cuts[i]])
            if shared == 0 or best[i] + size * shared < saved:
                break
        best.append(saved)
        last.append((at, prefix))
    lens, cu, j = [], [n], len(cuts) - 1
    while cu[-1] > 0:
        j, prefix = last[j]
        lens.append(prefix * block_size)
        cu.append(cuts[j])
    return lens[::-1], cu[::-1]


class BlockCache:
    """K/V pools [L, NB, BS, Hkv, D] bf16 on one device."""

    def __init__(self, num_layers: int, num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                 device, dtype=torch.bfloat16, zero: bool = True) -> None:
        shape = (num_layers, num_blocks, block_size, num_kv_heads, head_dim)
        alloc = torch.zeros if zero else torch.empty
        self.k = alloc(shape, dtype=dtype, device=device)
        self.v = alloc(shape, dtype=dtype, device=device)
        self.block_size = block_size
        self.device = torch.device(device)

    def write(self, layer: int, block_tables: torch.Tensor, pos: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v: [B, Hkv, q_len, D] (the reference layout); pos: [B] int64."""
        kt = k.transpose(1, 2)  # [B, q_len, Hkv, D]
        vt = v.transpose(1, 2)
        n = kt.shape[1]
        if n > 1 and kt.stride(0) != n * kt.stride(1):
            kt = kt.contiguous()
        if n > 1 and vt.stride(0) != n * vt.stride(1):
            vt = vt.contiguous()
        paged_kv_write(kt, vt, pos, block_tables, self.k[layer], self.v[layer])

    def _upload(self, *lists: Sequence[int]) -> list[torch.Tensor]:
        """int32 device tensors of equally long lists, in one copy."""
        return list(torch.tensor(lists, dtype=torch.int32).to(self.device, non_blocking=True))

    def copy_blocks(self, src: Sequence[int], dst: Sequence[int], num_tokens: Optional[Sequence[int]] = None) -> None:
        """Copy blocks src[i] to dst[i] in every layer (the first num_tokens[i]
        tokens of each, or all): copy_blocks for ids known on the host, which
        are checked here."""
        n, nb = len(src), self.k.shape[1]
        if len(dst) != n or (num_tokens is not None and len(num_tokens) != n):
            raise ValueError("src, dst and num_tokens differ in length")
        if any(not 0 <= b < nb for b in (*src, *dst)):
            raise ValueError(f"block ids outside the pool of {nb} blocks")
        if len(set(dst)) != n or not set(dst).isdisjoint(src):
            raise ValueError("every destination must be one copy's alone and no copy's source")
        if num_tokens is not None and any(not 0 <= t <= self.block_size for t in num_tokens):
            raise ValueError(f"num_tokens outside 0..{self.block_size}")
        if n:
            copy_blocks(self.k, self.v, *self._upload(*((src, dst) if num_tokens is None else (src, dst, num_tokens))))

    def fork(self, allocator: BlockAllocator, blocks: Sequence[int], num_tokens: int, n: int = 1) -> list[list[int]]:
        """The block tables of n children of a sequence that holds num_tokens
        tokens in `blocks`: the whole blocks are shared (one more holder each),
        a last block that is partly filled is copied to one of each child's
        own, in one launch. Blocks behind num_tokens stay the parent's."""
        full, rest = divmod(num_tokens, self.block_size)
        if num_tokens < 0 or n < 0 or len(blocks) < full + (rest > 0):
            raise ValueError(f"{len(blocks)} blocks do not hold {num_tokens} tokens")
        if any(allocator.holders(b) == 0 for b in blocks[: full + (rest > 0)]):
            raise ValueError("a block that is to be shared is not in use")
        own = allocator.allocate(n) if rest else []
        for i in range(n):
            allocator.fork(blocks[:full])
        if own:
            self.copy_blocks([blocks[full]] * n, own, [rest] * n)
        return [list(blocks[:full]) + own[i:i + 1] for i in range(n)]

    def compact(self, allocator: BlockAllocator, block_table: Optional[torch.Tensor] = None) -> dict[int, int]:
        """Move the used blocks to ids 1..n: the pages, the allocator's state
        and the entries of a device block_table. Returns {old id: new id} of
        the moved blocks, for tables on the host."""
        if block_table is not None:
            _check_table(block_table, self.k.device)
        src, dst = allocator.compact()
        if src:
            s, d = self._upload(src, dst)
            if block_table is None:
                copy_blocks(self.k, self.v, s, d)
            else:
                move_blocks(self.k, self.v, s, d, block_table)
        return dict(zip(src, dst))
