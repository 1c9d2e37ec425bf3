"""The paged-cache operators of a batch that shares prompts, as cases to be timed and compared.

  prefix  decode attention (one query token per row) where consecutive rows of the batch share the pages of a
          long prefix, which is read once for all of them: flash_attn_with_shared_prefix
  copy    whole or partly filled pages copied inside the pools of all layers: copy_blocks (the copy-on-write of
          a fork: a child takes its own copy of the last, partly filled page)
  move    pages moved to the ids that compaction gives them, and the block tables rewritten: move_blocks

`run` computes each in plain torch operations, or, with `own` set, by the calls of this package. Sizes follow
from the case alone (ragged ones through its number "mix"); values follow from the seed.
"""
import random

import torch

own = False


# ---------------------------------------------------------------- cases
def listed():
    return [
        # four samples of one short prompt, a few tokens in: the smallest step, where latency counts
        _prefix("prefix_4_samples", rows=4, groups=1, idle=0, prefix=512, suffix_lo=1, suffix_hi=64, mix=1),
        # one layer at the single-layer benchmark's batch: 8 requests behind a system prompt of three pages
        _prefix("prefix_b8", rows=8, groups=1, idle=0, prefix=768, suffix_lo=1, suffix_hi=256, mix=2),
        # the engine's batch of 128 behind one system prompt, contexts as long again
        _prefix("prefix_b128", rows=128, groups=1, idle=0, prefix=2048, suffix_lo=1, suffix_hi=1024, mix=3),
        # 128 questions about one long document
        _prefix("prefix_b128_document", rows=128, groups=1, idle=0, prefix=32768, suffix_lo=1, suffix_hi=512, mix=4),
        # several prompts, each sampled an odd number of times, with 16-token pages, rows on their own and idle rows
        _prefix("prefix_groups_pages16", rows=61, groups=5, idle=3, prefix=4000, suffix_lo=1, suffix_hi=777, mix=5, bs=16),
        # one rank of a partition by kv heads: one kv head, many rows, odd group of query heads
        _prefix("prefix_one_kv_head", rows=251, groups=3, idle=0, prefix=8192, suffix_lo=16, suffix_hi=1024, mix=6, hq=5, hkv=1),
        # one child forks: its partly filled page in all 28 layers
        _copy("copy_fork_one", pages=1, partial=1, mix=11, layers=28),
        # a single layer's pool of 16-token pages, few and odd
        _copy("copy_pages16", pages=37, partial=1, mix=12, layers=3, bs=16),
        # 64 children fork at once: one source page each, partly filled
        _copy("copy_fork_64", pages=64, partial=1, mix=13, layers=28),
        # a few pages moved, whole
        _move("move_3", pages=3, rows=8, width=5, mix=21, layers=28),
        # half a pool compacted, under the tables of the engine's batch
        _move("move_96", pages=96, rows=128, width=128, mix=22, layers=28),
        # many small pages of a pool of 16-token pages
        _move("move_pages16", pages=1201, rows=131, width=77, mix=23, layers=7, bs=16),
    ]


def _prefix(name, rows, groups, idle, prefix, suffix_lo, suffix_hi, mix, hq=16, hkv=8, bs=256):
    return {"name": name, "op": "prefix", "rows": rows, "groups": groups, "idle": idle, "prefix": prefix,
            "suffix_lo": suffix_lo, "suffix_hi": suffix_hi, "mix": mix, "hq": hq, "hkv": hkv, "bs": bs}


def _copy(name, pages, partial, mix, layers, bs=256, hkv=8):
    return {"name": name, "op": "copy", "pages": pages, "partial": partial, "mix": mix, "layers": layers, "bs": bs,
            "hkv": hkv}


def _move(name, pages, rows, width, mix, layers, bs=256, hkv=8):
    return {"name": name, "op": "move", "pages": pages, "rows": rows, "width": width, "mix": mix, "layers": layers,
            "bs": bs, "hkv": hkv}


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(("prefix", "prefix", "prefix", "copy", "move"))
    mix = rng.randrange(1 << 30)
    hkv = rng.choice((1, 2, 4, 8, 8))
    bs = rng.choice((16, 32, 48, 64, 128, 256, 256))
    if op == "prefix":
        rows = _log(rng, 1, 256)
        hi = _log(rng, 1, 1024)
        prefix = _log(rng, 16, 32768)
        # no more than the work of 128 rows of 16 heads behind 32768 keys
        group = rng.choice((1, 2, 2, 3, 4, 5, 8))
        prefix = max(16, min(prefix, 128 * 16 * 32768 // (rows * hkv * group)))
        case = _prefix("", rows, rng.randint(1, min(8, rows - rows // 8)), rng.choice((0, 0, 1, 5)), prefix, rng.randint(0, hi), hi,
                       mix, hkv * group, hkv, bs)
    elif op == "copy":
        case = _copy("", min(_log(rng, 1, 1024), 64 * 256 // bs), rng.randint(0, 1), mix, rng.randint(1, 28), bs, hkv)
    else:
        case = _move("", min(_log(rng, 1, 1024), 64 * 256 // bs), _log(rng, 1, 256), _log(rng, 1, 128), mix,
                     rng.randint(1, 28), bs, hkv)
    del case["name"]
    return case


# ---------------------------------------------------------------- sizes
HEAD_DIM = 128


def _batch(case):
    """(rows of each group, prefix of each group, own keys of each row). The rows of the groups come first; the
    rows behind them share nothing: about one in eight where there are several groups, then the idle ones, which
    have no keys."""
    r = random.Random(case["mix"])
    rows, groups = case["rows"], case["groups"]
    alone = rows // 8 if groups > 1 else 0
    cuts = sorted(r.sample(range(1, rows - alone), groups - 1)) if groups > 1 else []
    sizes = [b - a for a, b in zip([0] + cuts, cuts + [rows - alone])]
    # a fork shares whole pages: most prefixes end with a page, some inside one
    prefixes = []
    for g in range(groups):
        p = case["prefix"] if g == 0 else r.randint(max(1, case["prefix"] // 4), case["prefix"])
        prefixes.append(p if r.random() < 0.25 else max(case["bs"], p // case["bs"] * case["bs"]))
    suffix = [r.randint(case["suffix_lo"], case["suffix_hi"]) for _ in range(rows)] + [0] * case["idle"]
    return sizes, prefixes, suffix


def _tokens(case):
    """Tokens to copy of each page."""
    r = random.Random(case["mix"])
    return [r.randint(1, case["bs"]) if case["partial"] else case["bs"] for _ in range(case["pages"])]


def work(case):
    token = case["hkv"] * HEAD_DIM * 2
    if case["op"] == "prefix":
        sizes, prefixes, suffix = _batch(case)
        keys = sum(prefixes) + sum(suffix)
        seen = sum(n * p for n, p in zip(sizes, prefixes)) + sum(suffix)
        heads = len(suffix) * case["hq"]
        # every key and value once, q and the output, the statistics, the tables' entries that are read
        return {"bytes": keys * 2 * token + heads * (4 * HEAD_DIM + 4) + 4 * keys // case["bs"],
                "flops": 4 * HEAD_DIM * case["hq"] * seen}
    if case["op"] == "copy":
        return {"bytes": 2 * 2 * case["layers"] * sum(_tokens(case)) * token + 12 * case["pages"], "flops": 0}
    return {"bytes": 2 * 2 * case["layers"] * case["pages"] * case["bs"] * token + 8 * case["pages"]
            + 8 * case["rows"] * case["width"], "flops": 0}


# ---------------------------------------------------------------- inputs
def _randn(shape, g):
    out = torch.empty(shape, dtype=torch.bfloat16, device=g.device)
    return out.normal_(generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "prefix":
        return _prepare_prefix(case, seed, g)
    # pools [layers, pages, tokens, kv heads, head_dim]; page 0 is the one that idle rows write to
    n, r = case["pages"], random.Random(seed)
    total = 2 * n + 1 + n // 3
    k, v = (_randn((case["layers"], total, case["bs"], case["hkv"], HEAD_DIM), g) for _ in range(2))
    ids = r.sample(range(1, total), 2 * n)
    state = {"op": case["op"], "k": k, "v": v}
    if case["op"] == "copy":
        state["src"], state["dst"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ids[:n], ids[n:]))
        state["tokens"] = torch.tensor(_tokens(case), dtype=torch.int32, device="cuda") if case["partial"] else None
        return state
    ids.sort()  # the highest used pages go to the lowest free ones
    state["src"], state["dst"] = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ids[n:], ids[:n]))
    taken = set(ids[:n])
    used = [x for x in range(total) if x not in taken]
    table = torch.tensor(used, dtype=torch.int32)
    at = torch.randint(len(used), (case["rows"], case["width"]), generator=torch.Generator().manual_seed(seed))
    state["table"] = table[at].cuda()
    return state


def _prepare_prefix(case, seed, g):
    sizes, prefixes, suffix = _batch(case)
    bs, rows = case["bs"], len(suffix)
    shared = [p for n, p in zip(sizes, prefixes) for _ in range(n)] + [0] * (rows - sum(sizes))
    lens = [p + s for p, s in zip(shared, suffix)]
    width = max(1, max(-(-n // bs) for n in lens))
    firsts = [sum(sizes[:i]) for i in range(len(sizes))]
    group_of = [i for i, n in enumerate(sizes) for _ in range(n)] + [None] * (rows - sum(sizes))
    # whole pages of a prefix are in every row's table; the page that a prefix ends inside is each row's own copy
    need = [p // bs for p in prefixes] + [-(-n // bs) - p // bs for n, p in zip(lens, shared)]
    pages = list(range(1, 1 + sum(need)))
    random.Random(seed).shuffle(pages)
    at = [sum(need[:i]) for i in range(len(need))]
    taken = [pages[a:a + n] for a, n in zip(at, need)]
    table = [((taken[group_of[b]] if group_of[b] is not None else []) + taken[len(sizes) + b]) for b in range(rows)]
    table = torch.tensor([t + [0] * (width - len(t)) for t in table], dtype=torch.int32)
    k, v = (_randn((len(pages) + 1, bs, case["hkv"], HEAD_DIM), g) for _ in range(2))
    for i, (n, p) in enumerate(zip(sizes, prefixes)):
        if p % bs:
            to = table[firsts[i] + 1:firsts[i] + n, p // bs].long().cuda()
            for pool in (k, v):
                pool[to, :p % bs] = pool[int(table[firsts[i], p // bs]), :p % bs]
    q = _randn((rows, 1, case["hq"], HEAD_DIM), g)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"op": "prefix", "q": q, "k": k, "v": v, "table": table.cuda(), "lens": i32(lens), "prefix_lens": i32(prefixes),
            "cu_rows": i32(firsts + [sum(sizes)]), "most_rows": max(sizes), "most_prefix": max(prefixes),
            "most_own": max(1, max(suffix))}


# ---------------------------------------------------------------- one pass
def _calls():
    import __graft_entry__

    return __graft_entry__.load_package()


def run(state):
    op = state["op"]
    if own:
        la = _calls()
        if op == "prefix":
            return la.flash_attn_with_shared_prefix(state["q"], state["k"], state["v"], cache_seqlens=state["lens"],
                                                    block_table=state["table"], prefix_lens=state["prefix_lens"],
                                                    cu_prefix_rows=state["cu_rows"], return_softmax_lse=True)
        if op == "copy":
            la.copy_blocks(state["k"], state["v"], state["src"], state["dst"], num_tokens=state["tokens"])
            return state["k"], state["v"]
        la.move_blocks(state["k"], state["v"], state["src"], state["dst"], state["table"])
        return state["k"], state["v"], state["table"]
    if op == "prefix":
        return _plain_prefix(state)
    src, dst = state["src"].long(), state["dst"].long()
    if op == "copy":
        return tuple(_plain_copy(state[x], src, dst, state["tokens"]) for x in ("k", "v"))
    k, v = (_plain_copy(state[x], src, dst, None) for x in ("k", "v"))
    to = torch.arange(state["k"].shape[1], dtype=torch.int32, device=src.device)
    to[src] = state["dst"]
    state["table"].copy_(to[state["table"].long()])
    return k, v, state["table"]


def _plain_copy(pool, src, dst, tokens):
    if tokens is None:
        pool[:, dst] = pool[:, src]
    else:
        page, token = (torch.arange(pool.shape[2], device=src.device)[None, :] < tokens[:, None]).nonzero(as_tuple=True)
        pool[:, dst[page], token] = pool[:, src[page], token]
    return pool


def _plain_prefix(st):
    """Scores of the prefix keys once for all rows of a group, of each row's own keys by itself, one softmax over both."""
    q, k, v, table, lens, prefix = (st[x] for x in ("q", "k", "v", "table", "lens", "prefix_lens"))
    cu, bs, (B, _, hq, D), hkv = st["cu_rows"].long(), st["k"].shape[1], q.shape, st["k"].shape[2]
    grp, scale, inf = hq // hkv, D ** -0.5, float("inf")
    lens, prefix, dev = lens.long(), prefix.long(), q.device
    qh = q[:, 0].float().view(B, hkv, grp, D) * scale

    # rows of the groups, padded to the largest group; a row of padding stands for row B, which is dropped
    rows = cu[:-1, None] + torch.arange(st["most_rows"], device=dev)
    rows = torch.where(rows < cu[1:, None], rows, B)
    G, R = rows.shape
    safe = rows.clamp(max=B - 1)
    shared = torch.zeros(B + 1, dtype=torch.long, device=dev)
    shared[rows] = prefix[:, None].expand(G, R)
    shared = shared[:B]
    j = torch.arange(st["most_prefix"], device=dev)
    page = table[cu[:-1].clamp(max=B - 1)][:, (j // bs).clamp(max=table.shape[1] - 1)].long()
    kp, vp = (x[page, j % bs].float().permute(0, 2, 1, 3) for x in (k, v))                 # [G, hkv, P, D]
    s = qh[safe].permute(0, 2, 1, 3, 4).reshape(G, hkv, R * grp, D) @ kp.transpose(2, 3)   # [G, hkv, R * grp, P]
    sees = j < torch.minimum(shared, lens)[safe][:, :, None]                               # [G, R, P]
    s = s.view(G, hkv, R, grp, -1).masked_fill_(~sees[:, None, :, None], -inf)
    mp = s.amax(-1)
    w = torch.exp(s - torch.where(mp == -inf, 0.0, mp)[..., None])
    lp, op = w.sum(-1), (w.view(G, hkv, R * grp, -1) @ vp).view(G, hkv, R, grp, D)
    m1, l1, o1 = q.new_full((B + 1, hkv, grp), -inf, dtype=torch.float32), *(
        torch.zeros(B + 1, hkv, grp, *x, device=dev) for x in ((), (D,)))
    at = rows.reshape(-1)
    m1[at], l1[at], o1[at] = (x.transpose(1, 2).reshape(G * R, hkv, grp, *x.shape[4:]) for x in (mp, lp, op))
    m1, l1, o1 = m1[:B], l1[:B], o1[:B]

    j = shared[:, None] + torch.arange(st["most_own"], device=dev)                         # [B, S]
    page = table.gather(1, (j // bs).clamp(max=table.shape[1] - 1)).long()
    ks, vs = (x[page, j % bs].float().permute(0, 2, 1, 3) for x in (k, v))
    s = (qh @ ks.transpose(2, 3)).masked_fill_((j >= lens[:, None])[:, None, None], -inf)  # [B, hkv, grp, S]
    m2 = s.amax(-1)
    w = torch.exp(s - torch.where(m2 == -inf, 0.0, m2)[..., None])
    l2, o2 = w.sum(-1), w @ vs

    m = torch.maximum(m1, m2)
    m0 = torch.where(m == -inf, 0.0, m)
    a, b = torch.exp(m1 - m0), torch.exp(m2 - m0)
    l = l1 * a + l2 * b
    o = (o1 * a[..., None] + o2 * b[..., None]) / torch.where(l == 0, 1.0, l)[..., None]
    return o.view(B, 1, hq, D).to(q.dtype), (m0 + torch.log(l)).view(B, hq, 1)


def exact(case, seed):
    """Every row by itself in 64 bits, through its own block table. Copies compute no numbers."""
    if case["op"] != "prefix":
        return None
    st = prepare(case, seed)
    q, hkv = st["q"][:, 0].double(), case["hkv"]
    out = torch.zeros_like(q)
    lse = torch.full(q.shape[:2], -float("inf"), dtype=torch.float64, device=q.device)
    for b, n in enumerate(st["lens"].tolist()):
        if n:
            pages = st["table"][b, :-(-n // case["bs"])].long()
            keys, values = (st[x][pages].flatten(0, 1)[:n].double() for x in ("k", "v"))
            s = torch.einsum("hgd,thd->hgt", q[b].view(hkv, -1, HEAD_DIM), keys) / HEAD_DIM ** 0.5
            out[b] = torch.einsum("hgt,thd->hgd", s.softmax(-1), values).flatten(0, 1)
            lse[b] = s.logsumexp(-1).flatten()
    return out.unsqueeze(1), lse.unsqueeze(-1)
