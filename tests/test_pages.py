"""Shared blocks on the host: holders, forks, compaction and the grouping of
rows that share a prefix; and the refusals of the page and shared-prefix entry
points, none of which needs a GPU."""
import ctypes
import random

import pytest
import torch


def test_allocator_holders(pkg):
    a = pkg.BlockAllocator(8)
    x = a.allocate(3)
    assert [a.holders(b) for b in x] == [1, 1, 1] and a.holders(7) == 0
    a.fork(x[:2])
    a.fork(x[:1])
    a.release(x)
    assert [a.holders(b) for b in x] == [2, 1, 0] and a.num_free == 5
    a.release(x[:2])
    a.release(x[:1])
    assert a.num_free == 7 and [a.holders(b) for b in x] == [0, 0, 0]
    assert list(a.free) == [4, 5, 6, 7, 3, 2, 1]
    with pytest.raises(ValueError):
        a.fork([4])


def test_allocator_fork_takes_all_or_nothing(pkg):
    a = pkg.BlockAllocator(8)
    x = a.allocate(2)
    with pytest.raises(ValueError):
        a.fork([x[0], 6])
    assert a.holders(x[0]) == 1


@pytest.mark.parametrize("seed", range(6))
def test_allocator_compaction(pkg, seed):
    """After a compaction the used blocks are the lowest ids, no destination
    was in use, every holder count moved with its block, and blocks are handed
    out once each."""
    r = random.Random(seed)
    a = pkg.BlockAllocator(40)
    held = a.allocate(r.randint(0, 39))
    a.fork(held[::3])
    gone = r.sample(held, r.randint(0, len(held)))
    a.release(gone)
    before = {b: a.holders(b) for b in range(1, 40)}
    src, dst = a.compact()
    assert len(src) == len(dst) == len(set(src) | set(dst)) - len(src)
    assert all(before[s] > 0 and before[d] == 0 and d < s for s, d in zip(src, dst))
    to = dict(zip(src, dst))
    used = sorted(b for b in before if before[b] > 0)
    assert sorted(to.get(b, b) for b in used) == list(range(1, len(used) + 1))
    assert all(a.holders(to.get(b, b)) == before[b] for b in used)
    assert sorted(a.free) == list(range(len(used) + 1, 40))
    assert a.compact() == ([], [])


def test_shared_prefix_groups(pkg):
    bs = 16
    t = [[5, 6, 7, 1], [5, 6, 7, 2], [5, 6, 3], [9, 8], [9, 4], [10], [11]]
    n = [50, 64, 40, 32, 16, 1, 0]
    # rows 0..2 share blocks 5, 6 (block 7 of rows 0, 1 only); rows 3, 4 share block 9
    assert pkg.shared_prefix_groups(t, n, bs) == ([32, 16, 0, 0], [0, 3, 5, 6, 7])
    # a block that a row has not filled yet is not shared
    assert pkg.shared_prefix_groups(t, [50, 64, 31, 15, 16, 1, 0], bs)[1] == [0, 3, 4, 5, 6, 7]
    assert pkg.shared_prefix_groups(t, n, bs, min_blocks=2) == ([32, 0, 0, 0, 0], [0, 3, 4, 5, 6, 7])
    assert pkg.shared_prefix_groups([], [], bs) == ([], [0])
    assert pkg.shared_prefix_groups([[1, 2]], [32], bs) == ([0], [0, 1])


class _HostCache:
    """A BlockCache whose device copies run on the host."""

    def __init__(self, pkg, num_blocks, block_size):
        self.c = pkg.BlockCache(2, num_blocks, block_size, 1, 8, "cpu")
        self.copied = []

    def copy(self, src, dst, num_tokens=None):
        self.copied += list(zip(src, dst, num_tokens))


def test_cache_fork(pkg, monkeypatch):
    h = _HostCache(pkg, 12, 16)
    monkeypatch.setattr(h.c, "copy_blocks", h.copy)
    a = pkg.BlockAllocator(12)
    mine = a.allocate(3)  # 1, 2, 3
    kids = h.c.fork(a, mine, 37, n=2)  # two whole blocks and 5 tokens
    assert kids == [[1, 2, 4], [1, 2, 5]] and h.copied == [(3, 4, 5), (3, 5, 5)]
    assert [a.holders(b) for b in range(1, 6)] == [3, 3, 1, 1, 1]
    assert h.c.fork(a, mine, 32) == [[1, 2]] and len(h.copied) == 2  # nothing to copy
    assert h.c.fork(a, mine, 0, n=2) == [[], []]
    with pytest.raises(ValueError):
        h.c.fork(a, mine, 49)
    with pytest.raises(ValueError):
        h.c.fork(a, [1, 9], 20)  # block 9 is free
    with pytest.raises(RuntimeError):
        h.c.fork(a, mine, 37, n=20)  # no room: nothing taken
    assert [a.holders(b) for b in range(1, 6)] == [4, 4, 1, 1, 1]
    for t in kids + [[1, 2]]:
        a.release(t)
    a.release(mine)
    assert a.num_free == 11


def test_cache_copy_refusals(pkg):
    c = pkg.BlockCache(2, 6, 16, 1, 8, "cpu")
    for src, dst, n in (([1], [1, 2], None), ([1], [6], None), ([-1], [2], None), ([1, 2], [3, 3], None),
                        ([1, 2], [2, 3], None), ([1], [2], [17]), ([1], [2], [-1]), ([1], [2], [1, 2])):
        with pytest.raises(ValueError):
            c.copy_blocks(src, dst, n)
    c.copy_blocks([], [])


def test_cache_compaction_refuses_a_table_first(pkg):
    c = pkg.BlockCache(1, 6, 16, 1, 8, "cpu")
    a = pkg.BlockAllocator(6)
    x = a.allocate(3)
    a.release(x[:1])
    with pytest.raises(RuntimeError):
        c.compact(a, torch.zeros(2, 2, dtype=torch.int64))
    assert a.holders(3) == 1 and a.holders(1) == 0  # nothing renumbered


def test_page_functions_refuse(pkg):
    k = torch.zeros(2, 4, 16, 1, 8, dtype=torch.bfloat16)
    i = torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        pkg.copy_blocks(k, k, i, i)
    with pytest.raises(RuntimeError, match="same shape"):
        pkg.copy_blocks(k, k[:1], i, i)
    with pytest.raises(RuntimeError, match="contiguous"):
        pkg.copy_blocks(k[..., ::2], k[..., ::2], i, i)


def test_shared_prefix_refuses(pkg):
    q = torch.zeros(2, 1, 16, 128, dtype=torch.bfloat16)
    kc = torch.zeros(4, 16, 8, 128, dtype=torch.bfloat16)
    n, bt = torch.ones(2, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    p, cu = torch.zeros(1, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32)
    f = pkg.flash_attn_with_shared_prefix
    with pytest.raises(RuntimeError, match="CUDA"):
        f(q, kc, kc, n, bt, p, cu)
    with pytest.raises(RuntimeError, match="bfloat16"):
        f(q.float(), kc, kc, n, bt, p, cu)
    with pytest.raises(RuntimeError, match="q must be"):
        f(q.expand(2, 2, 16, 128), kc, kc, n, bt, p, cu)
    with pytest.raises(RuntimeError, match="prefix_lens"):
        f(q, kc, kc, n, bt, torch.zeros(2, dtype=torch.int32), cu)
    with pytest.raises(RuntimeError, match="cu_prefix_rows"):
        f(q, kc, kc, n, bt, p, cu.long())
    with pytest.raises(RuntimeError, match="cache_seqlens"):
        f(q, kc, kc, n[:1], bt, p, cu)
    with pytest.raises(RuntimeError, match="block_table"):
        f(q, kc, kc, n, bt.t().contiguous().t(), p, cu)


def test_c_entries_check_arguments(pkg):
    """Status codes before anything touches a GPU."""
    from lean_infer_b200 import _lib

    lib = _lib.load()
    null, fake = ctypes.c_void_p(0), ctypes.c_void_p(1 << 20)
    odd = ctypes.c_void_p((1 << 20) + 8)

    def copy(k=fake, block=16 * 1024, token=1024, es=2, n=4, layers=2, dim=128, src=fake, tokens=null, nb=8):
        return lib.la_copy_blocks(k, fake, 8 * 16 * 1024, block, token, 128, layers, nb, 16, 8, dim, es, src, fake,
                                  tokens, n, null, null)

    assert copy(n=0) == 0 and copy(layers=0) == 0
    assert copy(n=-1) == 1 and copy(src=null) == 1 and copy(k=null) == 1 and copy(nb=0) == 1
    assert copy(es=8) == 2
    assert copy(k=odd) == 3 and copy(token=1020) == 3 and copy(dim=4) == 3
    assert copy(tokens=ctypes.c_void_p((1 << 20) + 2)) == 3

    def move(table=fake, stride=4, rows=2, cols=4, n=0):
        return lib.la_move_blocks(fake, fake, 8 * 16 * 1024, 16 * 1024, 1024, 128, 2, 8, 16, 8, 128, 2, fake, fake, n,
                                  table, stride, rows, cols, null, null)

    assert move() == 0
    assert move(table=null) == 1 and move(stride=3) == 1 and move(rows=-1) == 1

    nbytes = ctypes.c_size_t(0)
    assert lib.la_paged_decode_shared_prefix_workspace_size(0, 4, 1, 16, 3, 128, ctypes.byref(nbytes)) == 1
    assert lib.la_paged_decode_shared_prefix_workspace_size(0, -1, 1, 16, 8, 128, ctypes.byref(nbytes)) == 1

    def prefix(q=fake, bs=16, hq=16, d=128, batch=4, qs=2048, groups=1, cu=fake, scale=0.1):
        return lib.la_paged_decode_shared_prefix(
            q, qs, 128, fake, fake, 16 * 1024, 1024, 128, 8, bs, fake, 4, 4, fake, fake, cu, groups, batch, hq, 8, d,
            ctypes.c_float(scale), fake, 2048, 128, null, null, 0, null, null)

    assert prefix(batch=0) == 0
    assert prefix(q=null) == 1 and prefix(cu=null) == 1 and prefix(groups=-1) == 1 and prefix(scale=0.0) == 1
    assert prefix(bs=24) == 2 and prefix(d=64) == 2 and prefix(hq=72) == 2
    assert prefix(q=odd) == 3 and prefix(qs=2044) == 3


def test_staged_prefix_groups(pkg):
    from lean_infer_b200 import qwen3

    buf = torch.full((qwen3.prefix_bytes(4),), 255, dtype=torch.uint8)
    lens, cu = qwen3.prefix_views(buf, 4)
    assert lens.shape == (4,) and cu.shape == (5,)
    qwen3.stage_prefix(lens, cu, ([32, 64], [0, 3, 5]), 8)
    assert lens.tolist() == [32, 64, 0, 0] and cu.tolist() == [0, 3, 5, 5, 5]
    qwen3.stage_prefix(lens, cu, None, 8)
    assert lens.tolist() == [0] * 4 and cu.tolist() == [0] * 5
    for bad in (([1] * 5, list(range(6))), ([1], [0, 9]), ([1, 1], [0, 4, 2]), ([1], [0]), ([1], [-1, 2])):
        with pytest.raises(ValueError):
            qwen3.stage_prefix(lens, cu, bad, 8)


@pytest.mark.parametrize("again", [[1], [2], [0], [9], [3, 3], [3, 1], [4, 4, 4]])
def test_allocator_refuses_a_release_too_many(pkg, again):
    """A block released more often than it is held would be handed out to two
    sequences; block 0 is nobody's. Nothing of a refused call is done."""
    a = pkg.BlockAllocator(6)
    x = a.allocate(4)  # 1, 2, 3, 4
    a.fork([4])
    a.release([1, 2])
    with pytest.raises(ValueError, match="released"):
        a.release(again)
    assert [a.holders(b) for b in x] == [0, 0, 1, 2] and list(a.free) == [5, 1, 2]
    a.release([4, 3, 4])  # its two holders in one call
    assert list(a.free) == [5, 1, 2, 3, 4] and a.compact() == ([], [])
    got = a.allocate(5)
    assert sorted(got) == [1, 2, 3, 4, 5] and a.num_free == 0


def _reads(tables, lengths, bs, groups):
    """Whole blocks that the rows read, the shared ones once for a group."""
    lens, cu = groups
    full = [n // bs for n in lengths]
    assert cu[0] == 0 and cu[-1] == len(tables) and all(a < b for a, b in zip(cu, cu[1:]))
    total = 0
    for n, a, b in zip(lens, cu, cu[1:]):
        assert n % bs == 0 and (b - a > 1 or n == 0)
        k = n // bs
        assert all(t[:k] == tables[a][:k] and f >= k for t, f in zip(tables[a:b], full[a:b]))
        total += sum(full[a:b]) - (b - a - 1) * k
    return total


def _rows(*runs):
    """Tables of (rows, blocks) runs that share a first block and, within the
    run, the rest; each row ends with a block of its own."""
    tables, ids = [], iter(range(10, 10 ** 6))
    for n, k in runs:
        mine = [1] + [next(ids) for _ in range(k - 1)]
        tables += [mine + [next(ids)] for _ in range(n)]
    return tables


@pytest.mark.parametrize("runs,min_blocks,want", [
    # a system prompt of one block in front of two documents, each asked several times
    ([(64, 128), (64, 128)], 1, ([128, 128], [0, 64, 128])),
    ([(4, 101), (4, 101)], 1, ([101, 101], [0, 4, 8])),
    # one row that shares only the system prompt, behind and in front of and between the others
    ([(64, 128), (1, 1)], 1, ([128, 0], [0, 64, 65])),
    ([(1, 1), (64, 128)], 1, ([0, 128], [0, 1, 65])),
    ([(9, 128), (1, 1), (9, 128)], 1, ([128, 0, 128], [0, 9, 10, 19])),
    # so little beside it that a group of its own is not worth it
    ([(2, 2), (6, 1)], 1, ([1], [0, 8])),
    ([(2, 2), (6, 1)], 2, ([2] + [0] * 6, [0, 2, 3, 4, 5, 6, 7, 8])),
])
def test_shared_prefix_groups_keep_what_is_shared(pkg, runs, min_blocks, want):
    tables, bs = _rows(*runs), 16
    lens, cu = pkg.shared_prefix_groups(tables, [bs * len(t) - 3 for t in tables], bs, min_blocks)
    assert ([n // bs for n in lens], cu) == want


@pytest.mark.parametrize("seed", range(60))
def test_shared_prefix_groups_against_every_division(pkg, seed):
    """No division of the rows reads fewer blocks, a group counted as one."""
    r = random.Random(seed)
    bs, n, least = 16, r.randint(1, 8), r.choice((1, 1, 2))
    tables, fresh = [], iter(range(100, 10 ** 4))
    for _ in range(n):
        keep = r.randint(0, len(tables[-1])) if tables else 0
        tables.append((tables[-1][:keep] if keep else []) + [next(fresh) for _ in range(r.randint(0, 4))])
    lengths = [r.randint(0, bs * len(t)) for t in tables]
    best = None
    for cuts in range(1 << (n - 1)):
        cu = [0] + [i + 1 for i in range(n - 1) if cuts >> i & 1] + [n]
        lens = []
        for a, b in zip(cu, cu[1:]):
            k = 0
            while all(lengths[i] // bs > k and tables[i][k] == tables[a][k] for i in range(a, b)):
                k += 1
            lens.append(k * bs if b - a > 1 else 0)
        if all(b - a == 1 or n >= least * bs for n, a, b in zip(lens, cu, cu[1:])):
            cost = _reads(tables, lengths, bs, (lens, cu)) + len(lens)
            best = cost if best is None else min(best, cost)
    got = pkg.shared_prefix_groups(tables, lengths, bs, least)
    assert _reads(tables, lengths, bs, got) + len(got[0]) == best
    assert all(k == 0 or k >= least * bs for k in got[0])


def test_shared_prefix_groups_of_lengths_below_zero(pkg):
    assert pkg.shared_prefix_groups([[1, 2], [1, 2]], [-1, -40], 16) == ([0, 0], [0, 1, 2])
