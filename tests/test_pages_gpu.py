"""Pages copied and moved on the device: bit-exact against the same indexing
in torch, every other page and token left as it was."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def _bits(t):
    return t.view({1: torch.int8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def _pool(shape, dtype, dev, seed):
    """Every bit pattern, NaN payloads among them."""
    g = torch.Generator(device=dev).manual_seed(seed)
    n = torch.empty(shape, dtype=dtype, device="meta").element_size()
    return torch.randint(0, 256, (*shape[:-1], shape[-1] * n), dtype=torch.uint8, device=dev, generator=g).view(dtype)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _expect(pool, src, dst, tokens):
    want = _bits(pool).clone()
    for i, (s, d) in enumerate(zip(src, dst)):
        n = pool.shape[-3] if tokens is None else tokens[i]
        want[..., d, :n, :, :] = want[..., s, :n, :, :]
    return want


def _ids(r, total, n):
    ids = r.sample(range(total), 2 * n)
    return ids[:n], ids[n:]


CASES = [  # layers, blocks, block size, heads, dim, pairs, partly filled
    (1, 3, 16, 1, 128, 1, False),
    (28, 5, 256, 8, 128, 1, True),
    (3, 100, 16, 8, 128, 37, True),
    (2, 41, 48, 2, 64, 20, True),
    (5, 9, 1, 1, 8, 4, False),
    (2, 700, 16, 1, 128, 333, True),
    (4, 13, 100, 3, 24, 6, True),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float8_e4m3fn])
def test_copy_blocks(pkg, cuda_dev, case, dtype):
    L, nb, bs, heads, dim, n, partial = case
    if dim * dtype.itemsize % 16:
        pytest.skip("rows of 16 bytes")
    r = random.Random(n)
    k, v = (_pool((L, nb, bs, heads, dim), dtype, cuda_dev, s) for s in (1, 2))
    src, dst = _ids(r, nb, n)
    src[-1] = src[0]  # one page, several copies
    tokens = [r.choice((0, 1, bs // 2, bs - 1, bs)) for _ in range(n)] if partial else None
    want = [_expect(x, src, dst, tokens) for x in (k, v)]
    pkg.copy_blocks(k, v, _i32(src, cuda_dev), _i32(dst, cuda_dev), None if tokens is None else _i32(tokens, cuda_dev))
    pkg.check_device_errors(cuda_dev.index)
    assert torch.equal(_bits(k), want[0]) and torch.equal(_bits(v), want[1])


def test_copy_blocks_of_one_layer_and_of_some_heads(pkg, cuda_dev):
    """Views: one layer [NB, BS, Hkv, D] of a pool, and two of its kv heads."""
    k, v = (_pool((3, 8, 32, 4, 128), torch.bfloat16, cuda_dev, s) for s in (3, 4))
    for cut in ((1,), (slice(None), slice(None), slice(None), slice(1, 3))):
        a, b = k.clone(), v.clone()
        wa, wb = (_bits(x).clone() for x in (a, b))
        _bits(wa)[cut] = _expect(a[cut].contiguous(), [2, 7], [5, 0], [9, 32])
        _bits(wb)[cut] = _expect(b[cut].contiguous(), [2, 7], [5, 0], [9, 32])
        pkg.copy_blocks(a[cut], b[cut], _i32([2, 7], cuda_dev), _i32([5, 0], cuda_dev), _i32([9, 32], cuda_dev))
        pkg.check_device_errors(cuda_dev.index)
        assert torch.equal(_bits(a), wa) and torch.equal(_bits(b), wb)


def test_copy_blocks_nothing(pkg, cuda_dev):
    k = _pool((2, 4, 16, 1, 8), torch.bfloat16, cuda_dev, 5)
    was = _bits(k).clone()
    e = _i32([], cuda_dev)
    pkg.copy_blocks(k, k, e, e)
    pkg.move_blocks(k, k, e, e, torch.zeros(2, 2, dtype=torch.int32, device=cuda_dev))
    pkg.move_blocks(k[:0], k[:0], e, e, torch.zeros(0, 2, dtype=torch.int32, device=cuda_dev))
    assert torch.equal(_bits(k), was)


@pytest.mark.parametrize("src,dst,tokens,done,code", [
    ([1, 2], [2, 3], None, [(2, 3)], "copy's destination"),              # 1 -> 2 would race with 2 -> 3
    ([1, 4, 2], [3, 3, 5], None, [(1, 3), (2, 5)], "copy's destination"),  # the first copy to a page counts
    ([1, 2], [1, 3], None, [(2, 3)], None),                                # a page to itself
    ([1, 9, -1, 2], [2, 3, 4, 99], None, [], "outside the pool"),
    ([1, 2], [3, 4], [17, 16], [(2, 4)], "sequence longer"),
    ([1, 2], [3, 4], [-1, 16], [(2, 4)], "sequence longer"),
])
def test_copies_that_are_skipped(pkg, cuda_dev, src, dst, tokens, done, code):
    k, v = (_pool((2, 8, 16, 2, 64), torch.bfloat16, cuda_dev, s) for s in (6, 7))
    # pair 1 -> 2 of the fourth case is sound unless 2 is a source, which it is there
    want = [_expect(x, [s for s, _ in done], [d for _, d in done], None) for x in (k, v)]
    pkg.copy_blocks(k, v, _i32(src, cuda_dev), _i32(dst, cuda_dev), None if tokens is None else _i32(tokens, cuda_dev))
    if code is None:
        pkg.check_device_errors(cuda_dev.index)
    else:
        with pytest.raises(RuntimeError, match=code if "outside" not in code else "outside the pool|copy's"):
            pkg.check_device_errors(cuda_dev.index)
    pkg.check_device_errors(cuda_dev.index)  # read and cleared
    assert torch.equal(_bits(k), want[0]) and torch.equal(_bits(v), want[1])


@pytest.mark.parametrize("L,nb,bs,n,rows,cols", [(28, 9, 256, 3, 8, 5), (2, 700, 16, 333, 131, 77), (3, 6, 32, 1, 1, 1),
                                                (1, 5000, 16, 2400, 5, 300)])
def test_move_blocks(pkg, cuda_dev, L, nb, bs, n, rows, cols):
    r = random.Random(n)
    k, v = (_pool((L, nb, bs, 2, 64), torch.bfloat16, cuda_dev, s) for s in (8, 9))
    src, dst = _ids(r, nb, n)
    used = [b for b in range(nb) if b not in set(dst)]
    wide = torch.tensor([[r.choice(used) for _ in range(cols + 3)] for _ in range(rows)], dtype=torch.int32, device=cuda_dev)
    to = torch.arange(nb, dtype=torch.int32, device=cuda_dev)
    to[_i32(src, cuda_dev).long()] = _i32(dst, cuda_dev)
    want_table = wide.clone()
    want_table[:, 1:cols + 1] = to[wide[:, 1:cols + 1].long()]  # a view: the columns beside it stay
    want = [_expect(x, src, dst, None) for x in (k, v)]
    pkg.move_blocks(k, v, _i32(src, cuda_dev), _i32(dst, cuda_dev), wide[:, 1:cols + 1])
    pkg.check_device_errors(cuda_dev.index)
    assert torch.equal(_bits(k), want[0]) and torch.equal(_bits(v), want[1])
    assert torch.equal(wide, want_table)


def test_skipped_moves_leave_the_table(pkg, cuda_dev):
    k, v = (_pool((2, 8, 16, 2, 64), torch.bfloat16, cuda_dev, s) for s in (6, 7))
    table = _i32([[1, 2, 4, 7], [9, -1, 0, 5]], cuda_dev)
    # 1 -> 2 meets 2 -> 3; 4 -> 6 counts, 5 -> 6 after it does not; 7 -> 8 leaves the pool
    src, dst = [1, 2, 4, 5, 7], [2, 3, 6, 6, 8]
    want = [_expect(x, [2, 4], [3, 6], None) for x in (k, v)]
    pkg.move_blocks(k, v, _i32(src, cuda_dev), _i32(dst, cuda_dev), table)
    with pytest.raises(RuntimeError):
        pkg.check_device_errors(cuda_dev.index)
    assert table.tolist() == [[1, 3, 6, 7], [9, -1, 0, 5]]
    assert torch.equal(_bits(k), want[0]) and torch.equal(_bits(v), want[1])


def test_offsets_past_32_bits(pkg, cuda_dev):
    """A pool of more than 2^32 bytes per layer and more than 2^31 elements."""
    nb, bs = 4300, 256
    k = torch.zeros(2, nb, bs, 8, 128, dtype=torch.bfloat16, device=cuda_dev)
    page = _pool((2, bs, 8, 128), torch.bfloat16, cuda_dev, 10)
    k[:, 3] = page
    pkg.copy_blocks(k, k[:], _i32([3], cuda_dev), _i32([nb - 1], cuda_dev), _i32([200], cuda_dev))
    pkg.check_device_errors(cuda_dev.index)
    assert torch.equal(_bits(k[:, nb - 1, :200]), _bits(page[:, :200])) and not k[:, nb - 1, 200:].any()
    assert not k[:, nb - 2].any() and not k[:, 4].any()


def test_copy_in_a_graph(pkg, cuda_dev):
    """Captured once, replayed with other ids and counts."""
    k, v = (_pool((2, 20, 16, 2, 64), torch.bfloat16, cuda_dev, s) for s in (11, 12))
    src, dst, n = (torch.zeros(4, dtype=torch.int32, device=cuda_dev) for _ in range(3))
    table = torch.zeros(3, 4, dtype=torch.int32, device=cuda_dev)
    pkg.copy_blocks(k, v, src, dst, n)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        pkg.copy_blocks(k, v, src, dst, n)
        pkg.move_blocks(k, v, dst, src, table)
    pkg.check_device_errors(cuda_dev.index)
    for ids in ([1, 2, 3, 4], [9, 8, 7, 19]):
        to = [b + 9 if b < 10 else 5 for b in ids]
        want = [_expect(x, ids, to, [16, 3, 0, 9]) for x in (k, v)]
        want = [_expect(x.view(torch.bfloat16), to, ids, None) for x in want]
        table.copy_(_i32([[0, to[0], to[1], ids[2]]] * 3, cuda_dev))
        src.copy_(_i32(ids, cuda_dev)), dst.copy_(_i32(to, cuda_dev)), n.copy_(_i32([16, 3, 0, 9], cuda_dev))
        g.replay()
        pkg.check_device_errors(cuda_dev.index)
        assert torch.equal(_bits(k), want[0]) and torch.equal(_bits(v), want[1])
        assert table.tolist() == [[0, ids[0], ids[1], ids[2]]] * 3


def test_cache_fork_and_compact(pkg, cuda_dev):
    """A sequence forks, the parent leaves, the pool is compacted: every
    child's tokens are the parent's throughout."""
    L, nb, bs = 3, 24, 16
    cache = pkg.BlockCache(L, nb, bs, 2, 64, cuda_dev)
    cache.k.copy_(_pool(cache.k.shape, torch.bfloat16, cuda_dev, 13))
    cache.v.copy_(_pool(cache.v.shape, torch.bfloat16, cuda_dev, 14))
    a = pkg.BlockAllocator(nb)
    other = a.allocate(5)
    mine = a.allocate(4)
    n = 3 * bs + 7

    def tokens(table):
        i = torch.tensor(table, device=cuda_dev)
        return [_bits(x)[:, i].flatten(1, 2)[:, :n].clone() for x in (cache.k, cache.v)]

    want = tokens(mine)
    kids = cache.fork(a, mine, n, n=3)
    assert all(torch.equal(x, y) for t in kids for x, y in zip(tokens(t), want))
    a.release(mine)
    a.release(other)
    bt = torch.tensor(kids, dtype=torch.int32, device=cuda_dev)
    moved = cache.compact(a, bt)
    pkg.check_device_errors(cuda_dev.index)
    kids = [[moved.get(b, b) for b in t] for t in kids]
    assert bt.tolist() == kids and sorted({b for t in kids for b in t}) == [1, 2, 3, 4, 5, 6]
    assert all(torch.equal(x, y) for t in kids for x, y in zip(tokens(t), want))
    for t in kids:
        a.release(t)
    assert a.num_free == nb - 1


def _us(f, before=lambda: None):
    """Median time of a call on the device, `before` not counted."""
    times = []
    for _ in range(7):
        before()
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1000)
    return sorted(times)[3]


def _scattered(r, total, n, dev):
    """n pages of the upper half of the ids and their places in the lower."""
    ids = sorted(r.sample(range(total), 2 * n))
    return _i32(ids[n:], dev), _i32(ids[:n], dev), [b for b in range(total) if b not in set(ids[:n])]


@pytest.mark.parametrize("n,rows,cols", [(1201, 131, 77), (6000, 128, 512)])
def test_a_table_that_names_the_pages_takes_little_beside_the_copy(pkg, cuda_dev, n, rows, cols):
    """Pages of 16 tokens in 7 layers, under a table most of whose entries name
    one that moves: no more than twice the time of the copies."""
    k, v = (torch.zeros(7, 2 * n + n // 3, 16, 8, 128, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
    src, dst, used = _scattered(random.Random(n), k.shape[1], n, cuda_dev)
    names = _i32(random.Random(1).choices(used, k=rows * cols), cuda_dev).view(rows, cols)
    table = names.clone()
    copy = _us(lambda: pkg.copy_blocks(k, v, src, dst))
    move = _us(lambda: pkg.move_blocks(k, v, src, dst, table), lambda: table.copy_(names))
    pkg.check_device_errors(cuda_dev.index)
    to = torch.arange(k.shape[1], dtype=torch.int32, device=cuda_dev)
    to[src.long()] = dst
    assert torch.equal(table, to[names.long()])
    assert move <= 2 * copy, (move, copy)


def test_many_pairs_in_one_call(pkg, cuda_dev):
    """16000 pages of 16 tokens in one call take no longer than one and a half
    times sixteen calls of 1000."""
    n = 16000
    k, v = (torch.zeros(4, 2 * n + n // 3, 16, 8, 128, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
    src, dst, _ = _scattered(random.Random(n), k.shape[1], n, cuda_dev)
    parts = list(zip(src.split(1000), dst.split(1000)))
    one = _us(lambda: pkg.copy_blocks(k, v, src, dst))
    many = _us(lambda: [pkg.copy_blocks(k, v, s, d) for s, d in parts])
    pkg.check_device_errors(cuda_dev.index)
    assert one <= 1.5 * many, (one, many)


@pytest.mark.parametrize("L,bs,heads", [(1, 16, 1), (3, 16, 8), (5, 80, 3)])
@pytest.mark.parametrize("n", [1023, 1024, 2047, 2048, 5000])
def test_copies_of_many_pairs(pkg, cuda_dev, L, bs, heads, n):
    """Numbers of pairs on both sides of those at which a CTA takes more of a
    pair, with skipped pairs and counts of tokens among them."""
    r = random.Random(n + L)
    k, v = (_pool((L, 2 * n + 7, bs, heads, 64), torch.bfloat16, cuda_dev, s) for s in (15, 16))
    src, dst = _ids(r, 2 * n + 7, n)
    tokens = [r.choice((0, 1, bs // 2, bs - 1, bs)) for _ in range(n)]
    bad = r.sample(range(n), 3)
    dst[bad[0]], tokens[bad[1]], src[bad[2]] = -1, bs + 1, 2 * n + 7
    done = [i for i in range(n) if i not in bad]
    want = [_bits(x).clone() for x in (k, v)]
    i, j, t = (torch.tensor([x[i] for i in done], device=cuda_dev) for x in (src, dst, tokens))
    page, token = (torch.arange(bs, device=cuda_dev)[None] < t[:, None]).nonzero(as_tuple=True)
    for w, x in zip(want, (k, v)):
        w[:, j[page], token] = _bits(x)[:, i[page], token]
    pkg.copy_blocks(k, v, _i32(src, cuda_dev), _i32(dst, cuda_dev), _i32(tokens, cuda_dev))
    with pytest.raises(RuntimeError, match="outside the pool|sequence longer"):
        pkg.check_device_errors(cuda_dev.index)
    pkg.check_device_errors(cuda_dev.index)
    assert torch.equal(_bits(k), want[0]) and torch.equal(_bits(v), want[1])
