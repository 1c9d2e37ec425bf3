"""Decode attention over shared prefixes against every row by itself in 64 bits.

Bounds, per output element: P is rounded to bf16 before the product with V
(half a step, 2^-8 relative, weighted by |v|) and the output once more (2^-8 of
itself); scores, exponentials and sums in fp32 add less than 2^-12 of the
weighted |v|. lse: a score is a sum of 128 fp32 products, off by at most
136 * 2^-24 of scale * sum |q_d k_d|; sums of exponentials and the logarithm
add less than 2^-18 of 1 + |lse|."""
import random

import pytest
import torch

from oracle import paged_attention as opa

pytestmark = pytest.mark.gpu


class Batch:
    """groups: (rows, prefix) of each; own: keys of each row behind its prefix
    (negative: the row ends that many keys before the end of its prefix); rows
    behind the groups are in none."""

    def __init__(self, dev, groups, own, bs, hq, hkv, seed=0, layers=1, spare=0, fill=None):
        r = random.Random(seed)
        g = torch.Generator(device=dev).manual_seed(seed)
        B, grouped = len(own), sum(n for n, _ in groups)
        shared = [p for n, p in groups for _ in range(n)] + [0] * (B - grouped)
        lens = [max(0, p + s) for p, s in zip(shared, own)]
        width = max(1, max(-(-n // bs) for n in lens + [p for _, p in groups])) + spare
        need = [p // bs for _, p in groups] + [max(0, -(-n // bs) - p // bs) for n, p in zip(lens, shared)]
        ids = list(range(1, 1 + sum(need)))
        r.shuffle(ids)
        taken = []
        for n in need:
            taken.append(ids[:n])
            ids = ids[n:]
        of = [i for i, (n, _) in enumerate(groups) for _ in range(n)] + [None] * (B - grouped)
        table = [(taken[of[b]] if of[b] is not None else []) + taken[len(groups) + b] for b in range(B)]
        self.table = torch.tensor([t + [0] * (width - len(t)) for t in table], dtype=torch.int32, device=dev)
        shape = (layers, sum(need) + 1, bs, hkv, 128)
        self.kp, self.vp = (torch.randn(shape, generator=g, device=dev).to(torch.bfloat16) for _ in range(2))
        self.k, self.v = self.kp[layers - 1], self.vp[layers - 1]
        at = 0
        for n, p in groups:  # a prefix that ends inside a page: every row's own copy of it
            if p % bs:
                for b in range(at + 1, at + n):
                    if lens[b] > p // bs * bs:
                        for x in (self.k, self.v):
                            x[self.table[b, p // bs].long(), :p % bs] = x[self.table[at, p // bs].long(), :p % bs]
            at += n
        if fill is not None:  # whatever no row sees
            seen = torch.zeros(shape[1], bs, dtype=torch.bool, device=dev)
            for b, n in enumerate(lens):
                j = torch.arange(n, device=dev)
                seen[self.table[b, j // bs].long(), j % bs] = True
            for x in (self.k, self.v):
                x[~seen] = fill
        self.q = torch.randn((B, 1, hq, 128), generator=g, device=dev).to(torch.bfloat16)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        self.lens, self.prefix = i32(lens), i32([p for _, p in groups])
        self.cu = i32([sum(n for n, _ in groups[:i]) for i in range(len(groups) + 1)])

    def call(self, pkg, **kw):
        return pkg.flash_attn_with_shared_prefix(self.q, self.k, self.v, self.lens, self.table, self.prefix, self.cu,
                                                 return_softmax_lse=True, **kw)

    def check(self, pkg, got=None, **kw):
        out, lse = self.call(pkg, **kw) if got is None else got
        pkg.check_device_errors(self.q.device.index)
        ref, rlse, absv, abss = opa.paged_decode_f64(self.q, self.k, self.v, self.table, self.lens, **kw)
        off = (out.double() - ref).abs()
        assert torch.isfinite(out).all()
        worst = (off - 2.0 ** -8 * (absv + ref.abs()) - 2.0 ** -12 * absv).amax().item() if off.numel() else 0
        assert worst <= 1e-30, f"out off by {off.max().item()}, {worst} over its bound"
        lse = lse[:, :, 0].double()
        some = torch.isfinite(rlse)
        assert torch.equal(torch.isfinite(lse), some) and bool((lse[~some] < 0).all())
        bound = abss * 136 * 2.0 ** -24 + 2.0 ** -18 * (1 + rlse.abs())
        assert bool(((lse - rlse).abs()[some] <= bound[some]).all()), (lse - rlse)[some].abs().max().item()


def own(n, lo, hi, seed=0):
    r = random.Random(seed)
    return [r.randint(lo, hi) for _ in range(n)]


CASES = {
    # groups, own keys, block size, query heads, kv heads
    "one_pair": ([(2, 256)], [1, 1], 256, 16, 8),
    "engine_batch": ([(128, 1024)], own(128, 1, 300), 256, 16, 8),
    "one_key_pages": ([(3, 16)], [1, 0, 5], 16, 16, 8),
    "nothing_but_prefix": ([(5, 512)], [0] * 5, 256, 16, 8),
    "prefix_inside_a_page": ([(7, 1000)], own(7, 1, 300), 256, 16, 8),
    "prefix_shorter_than_a_page": ([(4, 100)], own(4, 1, 300), 256, 16, 8),
    "small_pages": ([(9, 16 * 77)], own(9, 0, 40), 16, 16, 8),
    "pages_of_48": ([(9, 48 * 31)], own(9, 0, 100), 48, 16, 8),
    "pages_of_80": ([(6, 80 * 9), (6, 80)], own(12, 0, 100), 80, 8, 4),
    "pages_of_384": ([(6, 384 * 3)], own(6, 0, 500), 384, 16, 8),
    "many_groups": ([(3, 64), (1, 640), (17, 320), (2, 1280), (5, 0), (4, 63)], own(40, 0, 90), 64, 16, 8),
    "rows_that_end_early": ([(6, 512), (3, 256)], [-1, 10, -512, 0, -300, 1, -256, -255, -1], 128, 16, 8),
    "first_row_ends_early": ([(4, 512)], [-200, 30, 1, 0], 128, 16, 8),
    "empty_rows": ([(3, 256)], [-256, 4, -256, 0, 0, 77, 0], 256, 16, 8),
    "no_prefix": ([(4, 0)], [3, 0, 1000, 16], 256, 16, 8),
    "group_1": ([(70, 384)], own(70, 1, 60), 128, 8, 8),
    "group_3": ([(90, 384), (2, 128)], own(92, 1, 60), 128, 12, 4),
    "group_5": ([(131, 700)], own(131, 1, 60), 32, 5, 1),
    "group_7": ([(20, 300)], own(20, 1, 60), 32, 14, 2),
    "group_8": ([(33, 1024)], own(33, 1, 60), 256, 64, 8),
    "one_kv_head": ([(251, 2048), (5, 256)], own(260, 1, 300), 256, 2, 1),
    "many_rows": ([(600, 512), (500, 256)], own(1105, 0, 30), 256, 4, 2),
    "many_small_groups": ([(2, 64 * (1 + i % 5)) for i in range(150)], own(303, 0, 20), 64, 2, 1),
    "rows_256_groups_32": ([(8, 64 * (i % 4)) for i in range(32)], own(256, 0, 90), 64, 8, 4),
    "rows_257_groups_32": ([(8, 64 * (i % 4)) for i in range(32)], own(257, 0, 90), 64, 8, 4),
    "rows_256_groups_33": ([(7, 64 * (i % 4)) for i in range(33)], own(256, 0, 90), 64, 8, 4),
    "six_hundred_groups": ([(2, 32 * (i % 7)) for i in range(600)], own(1205, 0, 40), 32, 2, 1),
    "groups_of_nothing": ([(0, 64)] * 300 + [(5, 192)] + [(0, 0)] * 300 + [(1, 64), (30, 64)], own(40, 0, 50), 64, 16, 8),
    "halves_of_key_tiles": ([(4, 16), (4, 64), (4, 80), (4, 128), (4, 144), (40, 192), (4, 208), (4, 336)],
                            own(68, 0, 20), 16, 16, 8),
    "group_8_one_head": ([(33, 1000), (2, 512)], own(35, 0, 200), 16, 8, 1),
    "no_own_keys": ([(100, 4096)], [0] * 100, 256, 16, 8),
    "mostly_own_keys": ([(2, 16)], own(100, 500, 900), 16, 16, 8),
    "many_segments_per_cta": ([(3 + i * 5 % 11, 64 * (1 + i * 7 % 9)) for i in range(24)], own(190, 1500, 2500), 64, 16, 8),
    "pairs_and_singles_in_turn": ([(20 + i * 37 % 190, 128 * (1 + i % 5)) for i in range(9)], own(1030, 60, 200), 128, 8, 4),
    "long": ([(40, 20000)], own(40, 1, 700), 256, 16, 8),
    "long_for_two": ([(2, 30011), (3, 17)], own(5, 1, 9000), 16, 16, 8),
}


@pytest.mark.parametrize("case", CASES)
def test_shared_prefix(pkg, cuda_dev, case):
    groups, n, bs, hq, hkv = CASES[case]
    Batch(cuda_dev, groups, n, bs, hq, hkv, seed=len(case)).check(pkg)


@pytest.mark.parametrize("fill", [float("nan"), float("inf"), 3e38])
def test_slots_that_no_row_sees(pkg, cuda_dev, fill):
    """Whatever lies behind a sequence's end, in unused pages and in page 0."""
    Batch(cuda_dev, [(9, 16 * 13), (4, 500), (2, 0)], own(17, 0, 40), 16, 16, 8, seed=3, spare=3, fill=fill).check(pkg)


def test_values_of_one_row_do_not_reach_another(pkg, cuda_dev):
    """NaN in the keys and values of one row's own pages stay that row's; and a
    row that ends inside the prefix does not see what lies in the rest of it."""
    w = Batch(cuda_dev, [(4, 512)], [40, 20, -200, 100], 128, 16, 8, seed=4)
    mine = w.table[0, 4].long()
    w.k[mine, 39], w.v[mine, 39] = float("nan"), float("nan")
    rest = w.table[0, 3].long()
    w.v[rest, 100] = float("nan")  # key 484 of rows 0, 1, 3; row 2 has 312
    out, lse = w.call(pkg)
    pkg.check_device_errors(cuda_dev.index)
    assert torch.isnan(out[[0, 1, 3]]).all() and torch.isnan(lse[0]).all()
    alone = pkg.flash_attn_with_kvcache(w.q[2:3], w.k, w.v, cache_seqlens=w.lens[2:3], block_table=w.table[2:3])
    assert (out[2].double() - alone[0].double()).abs().max() <= 2.0 ** -6


def test_scale_strides_and_views(pkg, cuda_dev):
    """A given softmax scale; q as a slice of a fused projection; a layer's
    slice of the pools; some of their kv heads; a wider block table."""
    w = Batch(cuda_dev, [(11, 640)], own(13, 0, 200), 128, 16, 8, seed=5, layers=3, spare=2)
    w.check(pkg, softmax_scale=0.3)
    wide = torch.randn(13, 1, 40, 128, device=cuda_dev).to(torch.bfloat16)
    w.q = wide[:, :, 3:19]
    w.check(pkg)
    w.k, w.v, w.q = w.k[:, :, 2:6], w.v[:, :, 2:6], w.q[:, :, :8]
    w.check(pkg)
    w.table = torch.nn.functional.pad(w.table, (0, 5))[:, :-3]
    w.check(pkg)


def test_large_scores(pkg, cuda_dev):
    """Scores of some hundreds, rising and falling along the prefix."""
    w = Batch(cuda_dev, [(30, 2048)], own(30, 1, 200), 256, 16, 8, seed=6)
    w.q *= 16
    out, lse = w.call(pkg)
    pkg.check_device_errors(cuda_dev.index)
    ref, rlse, absv, abss = opa.paged_decode_f64(w.q, w.k, w.v, w.table, w.lens)
    # a score may be off by 136 * 2^-24 of sum |q k| * scale, a weight by that much relative, both sides of the mean
    e = 2 * 136 * 2.0 ** -24 * abss[:, None, :, None]
    assert bool(((out.double() - ref).abs() <= (2.0 ** -8 + e) * (absv + ref.abs()) + 2.0 ** -12 * absv).all())
    assert bool(((lse[:, :, 0].double() - rlse).abs() <= abss * 136 * 2.0 ** -24 + 2.0 ** -18 * (1 + rlse.abs())).all())


def test_rising_scores(pkg, cuda_dev):
    """Each 64 keys' scores exceed those before by ten and more powers of two, so
    that what has been summed is scaled down again and again; and the same keys
    in falling order."""
    for fall in (False, True):
        w = Batch(cuda_dev, [(40, 1536), (5, 1100)], [0] * 45, 256, 16, 8, seed=17)
        w.q.abs_()
        w.k.abs_()
        n = w.lens[0].item()
        ramp = torch.arange(n, device=cuda_dev) / 64
        for row in (0, 40):
            pages = w.table[row, :-(-w.lens[row].item() // 256)].long()
            for j, page in enumerate(pages.flip(0) if fall else pages):
                r = ramp[256 * j:256 * j + 256]
                w.k[page] *= (r.flip(0) if fall else r)[:, None, None].to(torch.bfloat16)
        out, lse = w.call(pkg)
        pkg.check_device_errors(cuda_dev.index)
        ref, rlse, absv, abss = opa.paged_decode_f64(w.q, w.k, w.v, w.table, w.lens)
        e = 2 * 136 * 2.0 ** -24 * abss[:, None, :, None]  # as in test_large_scores
        assert bool(((out.double() - ref).abs() <= (2.0 ** -8 + e) * (absv + ref.abs()) + 2.0 ** -12 * absv).all())
        assert bool(((lse[:, :, 0].double() - rlse).abs() <= abss * 136 * 2.0 ** -24 + 2.0 ** -18 * (1 + rlse.abs())).all())


def test_lengths_and_groups_written_by_the_kernel_in_front(pkg, cuda_dev):
    """The call starts beside the end of the kernel before it. That one writes the
    lengths and groups here (as bits, into pages of their own), so that what the
    call saw first is out of date."""
    a = Batch(cuda_dev, [(10, 640), (4, 128), (0, 0), (9, 64)], own(24, 0, 200, 1), 64, 16, 8, seed=18)
    b = Batch(cuda_dev, [(0, 0), (20, 320), (1, 64), (3, 64)], own(24, 0, 500, 2), 64, 16, 8, seed=19)
    nb, tokens = 64, 64 * 64
    pages = [torch.zeros(nb, 64, 8, 128, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2)]
    at = pages[0].view(torch.int32)[nb - 1, 63]
    table, pos = torch.arange(nb, dtype=torch.int32, device=cuda_dev)[None], torch.zeros(1, dtype=torch.int64, device=cuda_dev)
    news = []
    for w in (a, b):
        new = torch.zeros(1, tokens, 8, 128, dtype=torch.bfloat16, device=cuda_dev)
        bits = new.view(torch.int32)[0, -1]
        bits[0, :24], bits[1, :4], bits[2, :5] = w.lens, w.prefix, w.cu
        news.append(new)

    def both():
        got = []
        for w, new in zip((a, b), news):
            pkg.paged_kv_write(new, new, pos, table, *pages)
            got.append(pkg.flash_attn_with_shared_prefix(w.q, w.k, w.v, at[0, :24], w.table, at[1, :4], at[2, :5],
                                                         return_softmax_lse=True))
        return got

    for _ in range(10):
        for w, got in zip((a, b), both()):
            w.check(pkg, got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [both() for _ in range(4)]
    for _ in range(3):
        graph.replay()
        for x in got:
            a.check(pkg, x[0])
            b.check(pkg, x[1])


def test_same_as_plain_decode(pkg, cuda_dev):
    """flash_attn_with_kvcache on the same tables, both within their bounds."""
    w = Batch(cuda_dev, [(20, 1500), (9, 256)], own(33, 0, 400), 256, 16, 8, seed=7)
    out, lse = w.call(pkg)
    ref, rlse = pkg.flash_attn_with_kvcache(w.q, w.k, w.v, cache_seqlens=w.lens, block_table=w.table,
                                            return_softmax_lse=True)
    pkg.check_device_errors(cuda_dev.index)
    _, _, absv, _ = opa.paged_decode_f64(w.q, w.k, w.v, w.table, w.lens)
    assert bool(((out.double() - ref.double()).abs() <= 2 * (2.0 ** -7 + 2.0 ** -12) * absv).all())
    some = torch.isfinite(rlse)
    assert torch.equal(torch.isfinite(lse), some) and (lse - rlse)[some].abs().max() <= 1e-4


def test_same_bits_each_time(pkg, cuda_dev):
    w = Batch(cuda_dev, [(50, 3000), (30, 777)], own(83, 0, 400), 16, 16, 8, seed=8)
    first = [x.clone() for x in w.call(pkg)]
    for _ in range(5):
        again = w.call(pkg)
        assert all(torch.equal(a.view(torch.int16 if a.dtype == torch.bfloat16 else torch.int32),
                               b.view(torch.int16 if a.dtype == torch.bfloat16 else torch.int32))
                   for a, b in zip(first, again))


def test_empty_batch_and_no_groups(pkg, cuda_dev):
    w = Batch(cuda_dev, [(2, 256)], own(6, 1, 100), 256, 16, 8, seed=9)
    z = torch.zeros(1, dtype=torch.int32, device=cuda_dev)
    out, lse = pkg.flash_attn_with_shared_prefix(w.q[:0], w.k, w.v, w.lens[:0], w.table[:0], z[:0], z,
                                                 return_softmax_lse=True)
    assert out.shape == (0, 1, 16, 128) and lse.shape == (0, 16, 1)
    w.check(pkg, pkg.flash_attn_with_shared_prefix(w.q, w.k, w.v, w.lens, w.table, z[:0], z, return_softmax_lse=True))


def test_graph_replayed_with_other_groups(pkg, cuda_dev):
    """One captured graph, replayed for other lengths, tables and groups; two
    graphs replayed at once on two streams."""
    B, G, layout = 24, 4, dict(bs=64, hq=16, hkv=8)
    batches = [Batch(cuda_dev, g, own(B, 0, 200, i), seed=10 + i, **layout) for i, g in enumerate((
        [(10, 640), (4, 128), (0, 0), (9, 64)], [(24, 1280), (0, 0), (0, 0), (0, 0)], [(0, 0), (0, 0), (2, 192), (2, 704)],
        [(1, 640), (1, 64), (1, 64), (1, 64)]))]
    width, nb = max(b.table.shape[1] for b in batches), max(b.k.shape[0] for b in batches)
    graphs = []
    for _ in range(2):
        s = Batch(cuda_dev, [(0, 0)] * G, [0] * B, seed=1, **layout)
        s.table = torch.zeros(B, width, dtype=torch.int32, device=cuda_dev)
        s.k, s.v = (torch.zeros(nb, *s.k.shape[1:], dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
        s.call(pkg)
        torch.cuda.synchronize()
        s.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s.graph):
            s.got = s.call(pkg)
        graphs.append(s)

    def load(s, b):
        s.table.zero_()
        s.table[:, :b.table.shape[1]] = b.table
        for x, y in ((s.k, b.k), (s.v, b.v)):
            x[:y.shape[0]] = y
        for n in ("q", "lens", "prefix", "cu"):
            getattr(s, n).copy_(getattr(b, n))

    for b in batches:
        load(graphs[0], b)
        graphs[0].graph.replay()
        b.check(pkg, graphs[0].got)
    load(graphs[0], batches[0]), load(graphs[1], batches[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.graph.replay()
    torch.cuda.synchronize()
    batches[0].check(pkg, graphs[0].got)
    batches[1].check(pkg, graphs[1].got)


def test_calls_one_after_another_on_two_streams(pkg, cuda_dev):
    """Each call has its own workspace: calls on two streams do not meet, and a
    call right after one that changed its inputs sees the new ones."""
    a = Batch(cuda_dev, [(30, 2048)], own(32, 0, 300, 1), 256, 16, 8, seed=11)
    b = Batch(cuda_dev, [(3, 1024), (20, 512)], own(23, 0, 300, 2), 128, 16, 4, seed=12)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(10):
        x = a.call(pkg)
        with torch.cuda.stream(side):
            got.append((x, b.call(pkg)))
    torch.cuda.synchronize()
    for x, y in got:
        a.check(pkg, x)
        b.check(pkg, y)
    lens = a.lens.clone()
    first = a.call(pkg)
    a.lens.copy_((lens - 37).clamp(min=0))
    second = a.call(pkg)
    a.check(pkg, second)
    a.lens = lens
    a.check(pkg, first)


def test_offsets_past_32_bits(pkg, cuda_dev):
    """Pages whose element offsets exceed 2^32 bytes and 2^31 elements."""
    nb = 8300
    k, v = (torch.empty(nb, 256, 8, 128, dtype=torch.bfloat16, device=cuda_dev) for _ in range(2))
    w = Batch(cuda_dev, [(9, 1024)], own(9, 1, 300), 256, 16, 8, seed=13)
    n = w.k.shape[0]
    k[nb - n:], v[nb - n:] = w.k, w.v
    w.k, w.v, w.table = k, v, w.table + (nb - n)
    w.check(pkg)


def test_pages_outside_the_pool_are_reported(pkg, cuda_dev):
    """They read as zeros, in the shared pages and in a row's own."""
    for row, col, bad in ((0, 1, 10 ** 6), (0, 0, -1), (3, 3, 77777)):
        w = Batch(cuda_dev, [(4, 384)], [20, 30, 1, 100], 128, 16, 8, seed=14)
        w.table[row if col >= 3 else slice(0, 4), col] = bad
        w.call(pkg)
        with pytest.raises(RuntimeError, match="block id outside the pool"):
            pkg.check_device_errors(cuda_dev.index)


def test_prefix_behind_the_table_and_bad_groups(pkg, cuda_dev):
    """A prefix longer than the tables is cut; groups that run backwards or
    leave the batch are reported, and the rows of sound ones are right."""
    w = Batch(cuda_dev, [(4, 384)], [0, 0, -1, -200], 128, 16, 8, seed=15)
    w.prefix += 10 ** 6
    w.check(pkg)
    for cu in ([0, 2, 99], [0, 3, 2], [-1, 2, 4]):
        w = Batch(cuda_dev, [(2, 256), (2, 256)], own(4, 1, 100), 128, 16, 8, seed=16)
        w.cu.copy_(torch.tensor(cu, dtype=torch.int32))
        w.call(pkg)
        with pytest.raises(RuntimeError, match="prefix groups"):
            pkg.check_device_errors(cuda_dev.index)
    pkg.check_device_errors(cuda_dev.index)


def test_refusals(pkg, cuda_dev):
    w = Batch(cuda_dev, [(2, 256)], [3, 4], 256, 16, 8)
    f = pkg.flash_attn_with_shared_prefix
    with pytest.raises(RuntimeError, match="one device"):
        f(w.q, w.k, w.v, w.lens.cpu(), w.table, w.prefix, w.cu)
    with pytest.raises(RuntimeError, match="misaligned"):
        f(torch.zeros(2 * 16 * 128 + 1, dtype=torch.bfloat16, device=cuda_dev)[1:].view(2, 1, 16, 128), w.k, w.v, w.lens,
          w.table, w.prefix, w.cu)
    with pytest.raises(RuntimeError, match="unsupported"):
        f(w.q[..., :64], w.k[..., :64], w.v[..., :64], w.lens, w.table, w.prefix, w.cu)
    with pytest.raises(RuntimeError, match="invalid argument"):
        f(w.q, w.k, w.v, w.lens, w.table, w.prefix, w.cu, softmax_scale=-1.0)


@pytest.mark.parametrize("cu", [[0, 100, 50, 128], [10, 60, 20, 70, 30, 128], [0, 128, 0, 128], [0, 2, 99, 300], [-1, 64, 128]])
@pytest.mark.parametrize("more_groups,more_rows", [(0, 0), (40, 0), (600, 0), (0, 150)])
def test_rows_are_right_whatever_the_bounds(pkg, cuda_dev, cu, more_groups, more_rows):
    """Bounds that run backwards or leave the batch, some with runs of rows that
    overlap, are reported, no rows share, and every row has its own result."""
    w = Batch(cuda_dev, [(128, 512)], own(128 + more_rows, -200, 100), 128, 4, 2, seed=20)
    cu = cu + [cu[-1]] * more_groups
    w.cu = torch.tensor(cu, dtype=torch.int32, device=cuda_dev)
    w.prefix = torch.full((len(cu) - 1,), 512, dtype=torch.int32, device=cuda_dev)
    got = w.call(pkg)
    with pytest.raises(RuntimeError, match="prefix groups"):
        pkg.check_device_errors(cuda_dev.index)
    w.check(pkg, got)


@pytest.mark.parametrize("bs", [16, 256])
def test_decode_right_behind_a_move(pkg, cuda_dev, bs):
    """The pages and the table that the kernel in front has just moved and
    rewritten, to and fro, called one after another and in a graph: where a page
    lies does not change a bit."""
    w = Batch(cuda_dev, [(20, 1024), (5, 512)], own(28, 0, 300), bs, 16, 8, seed=21)
    n = w.k.shape[0]
    w.k, w.v = (torch.cat([x, torch.full_like(x, float("nan"))]) for x in (w.k, w.v))
    r = random.Random(2)
    here = torch.tensor(r.sample(range(1, n), (n - 1) // 2), dtype=torch.int32, device=cuda_dev)
    there = here + n
    first = [x.clone() for x in w.call(pkg)]
    w.check(pkg, first)

    def there_and_back():
        got = []
        for a, b in ((here, there), (there, here)):
            pkg.move_blocks(w.k, w.v, a, b, w.table)
            got.append(w.call(pkg))
        return got

    got = [x for _ in range(10) for x in there_and_back()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [x for _ in range(3) for x in there_and_back()]
    for _ in range(5):
        graph.replay()
        got += [tuple(x.clone() for x in pair) for pair in captured]
    pkg.check_device_errors(cuda_dev.index)
    for out, lse in got:
        assert torch.equal(out.view(torch.int16), first[0].view(torch.int16)) and torch.equal(lse, first[1])
