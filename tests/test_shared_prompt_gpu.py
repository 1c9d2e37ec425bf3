"""Requests that share a prompt, from its prefill to the end: the sequence is
forked, its children decode in a captured graph that reads the prompt once,
some leave, the pool is compacted, the rest go on. Every logit against the same
children kept apart, each with a prompt of its own, in a plain decode graph.

Tolerance: both sides are bf16 models that differ by the order of sums, as in
the decoder's other tests: relative L2 of the logits <= 2 %."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


@pytest.mark.parametrize("bs,prompt,bucketed", [(64, 300, False), (64, 256, True), (16, 333, False), (256, 700, True)])
def test_fork_decode_compact(pkg, cuda_dev, bs, prompt, bucketed):
    from lean_infer_b200 import qwen3

    cfg = qwen3.ModelConfig(num_hidden_layers=2, vocab_size=4096)
    model = qwen3.random_model(cfg, cuda_dev, seed=7)
    model.rope(4096)
    L, B, steps = cfg.num_hidden_layers, 5, 9
    g = torch.Generator().manual_seed(prompt)
    ids = torch.randint(0, cfg.vocab_size, (prompt,), generator=g)
    nb = -(-(prompt + steps) // bs)
    pool = 2 + (B + 1) * nb
    caches = [pkg.BlockCache(L, pool, bs, 8, 128, cuda_dev) for _ in range(2)]
    allocs = [pkg.BlockAllocator(pool) for _ in range(2)]
    cu = torch.tensor([0, prompt], dtype=torch.int32, device=cuda_dev)

    def prefill(cache, table):
        bt = torch.tensor([table], dtype=torch.int32, device=cuda_dev)
        return model(ids.to(cuda_dev), cache, bt, torch.zeros(1, dtype=torch.long, device=cuda_dev), None,
                     cu_seqlens=cu, max_seqlen=prompt)

    # shared: one prefill, forked; apart: every child its own
    first = allocs[0].allocate(2)  # something in front, released later: the compaction has blocks to move
    parent = allocs[0].allocate(-(-prompt // bs))
    prefill(caches[0], parent)
    tables = caches[0].fork(allocs[0], parent, prompt, n=B)
    allocs[0].release(parent)
    apart = [allocs[1].allocate(nb) for _ in range(B)]
    for t in apart:
        prefill(caches[1], t)
    assert len({b for t in tables for b in t}) < len({b for t in apart for b in t})

    if bucketed:
        graphs = [qwen3.BucketedDecodeGraph(model, caches[0], [2, 8], nb, prefix_groups=3),
                  qwen3.BucketedDecodeGraph(model, caches[1], [2, 8], nb)]
    else:
        graphs = [qwen3.DecodeGraph(model, caches[0], B, nb, prefix_groups=3), qwen3.DecodeGraph(model, caches[1], B, nb)]

    def logits(dg, n):
        return (dg.logits() if bucketed else dg.logits)[:n, 0].clone()

    def stage(dg, rows, tok, pos, kw):
        """All slots of a plain graph are staged, the ones that left as idle rows."""
        n = len(rows)
        bt = torch.zeros(n if bucketed else B, nb, dtype=torch.int32)
        for i, t in enumerate(rows):
            bt[i, :len(t)] = torch.tensor(t, dtype=torch.int32)
        pad = bt.shape[0] - n
        dg.stage(torch.nn.functional.pad(tok, (0, pad)).view(-1, 1), torch.nn.functional.pad(pos, (0, pad)), bt,
                 torch.nn.functional.pad(pos + 1, (0, pad), value=1).to(torch.int32), **kw)

    tok = torch.randint(0, cfg.vocab_size, (B,), generator=g)
    pos = torch.full((B,), prompt, dtype=torch.long)
    for step in range(steps):
        if step == 5:  # two children leave, what was in front of the pool too, and the pool is compacted
            for i in (3, 1):
                allocs[0].release(tables.pop(i))
                apart.pop(i)
            keep = [0, 2, 4]
            tok, pos = tok[keep], pos[keep]
            allocs[0].release(first)
            moved = caches[0].compact(allocs[0])
            assert moved
            tables = [[moved.get(b, b) for b in t] for t in tables]
        for i, t in enumerate(tables):  # a child that has filled its blocks takes one more
            if pos[i] // bs >= len(t):
                t += allocs[0].allocate(1)
        groups = pkg.shared_prefix_groups(tables, (pos + 1).tolist(), bs)
        assert groups[0] == [prompt // bs * bs] and groups[1] == [0, len(tables)]
        stage(graphs[0], tables, tok, pos, {"prefix": groups})
        stage(graphs[1], apart, tok, pos, {})
        for dg in graphs:
            dg.step()
        pkg.check_device_errors(cuda_dev.index)
        a, b = (logits(dg, len(tables)) for dg in graphs)
        assert _rel(a, b) <= 0.02, (step, _rel(a, b))
        tok = b.argmax(-1).cpu()
        pos = pos + 1
    for dg in graphs:
        dg.release()


def test_graph_refuses_prefix_without_groups(pkg, cuda_dev):
    from lean_infer_b200 import qwen3

    cfg = qwen3.ModelConfig(num_hidden_layers=1, vocab_size=256)
    model = qwen3.random_model(cfg, cuda_dev)
    cache = pkg.BlockCache(1, 4, 16, 8, 128, cuda_dev)
    one = torch.zeros(1, dtype=torch.long)
    with pytest.raises(ValueError):
        qwen3.DecodeGraph(model, cache, 1, 2).stage(one, one, one.view(1, 1), one, prefix=([0], [0, 1]))
    with pytest.raises(ValueError):
        qwen3.DecodeGraph(model, cache, 1, 2, prefix_groups=1).stage(one, one, one.view(1, 1), one,
                                                                     prefix=([0, 0], [0, 1, 1]))
