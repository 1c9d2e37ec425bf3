"""Graphs of decode steps whose rows share blocks, captured anew."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_capture_behind_a_step_with_groups(pkg, cuda_dev):
    """The groups of the last step, of a large bucket, are not those of the
    small one that is captured next: nothing is recorded as wrong, and the step
    is the same again."""
    from lean_infer_b200 import qwen3

    bs, rows, width = 16, 8, 4
    cfg = qwen3.ModelConfig(num_hidden_layers=1, vocab_size=256)
    model = qwen3.random_model(cfg, cuda_dev)
    cache = pkg.BlockCache(1, 2 + rows, bs, 8, 128, cuda_dev)
    g = torch.Generator(device=cuda_dev).manual_seed(1)
    for x in (cache.k, cache.v):
        x.normal_(generator=g)
    alloc = pkg.BlockAllocator(2 + rows)
    tables = cache.fork(alloc, alloc.allocate(1), bs, n=rows)
    tables = [t + alloc.allocate(1) for t in tables]
    dg = qwen3.BucketedDecodeGraph(model, cache, [2, rows], width, prefix_groups=1)
    n = torch.full((rows,), bs, dtype=torch.long)
    groups = pkg.shared_prefix_groups(tables, (n + 1).tolist(), bs)
    assert groups == ([bs], [0, rows])
    dg.stage(torch.arange(rows).view(-1, 1), n, torch.tensor(tables, dtype=torch.int32), (n + 1).to(torch.int32), prefix=groups)
    dg.step()
    pkg.check_device_errors(cuda_dev.index)
    first = dg.logits().clone()
    dg.release()
    dg.step()
    pkg.check_device_errors(cuda_dev.index)
    assert torch.equal(dg.logits(), first)
    dg.capture()
    pkg.check_device_errors(cuda_dev.index)
    dg.release()
