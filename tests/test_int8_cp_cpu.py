"""8-bit integer projections and kept 8-bit activations under context parallelism, on gloo CPU ranks."""
import os
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

sys.path.insert(0, os.path.dirname(__file__))
from test_cp_cpu import _inputs, _model  # noqa: E402
from test_h3_cp_cpu import _free_port, _setup  # noqa: E402


def _h3():
    m, kw, L = _setup()
    g = torch.Generator().manual_seed(3)
    for p in m.parameters():  # heads that are not zero, norm weights that are not one
        p.data.add_(0.03 * torch.randn(p.shape, generator=g))
    m.requires_grad_(False).bfloat16().quantize_int8_()
    return m, kw, L


def _sampled(m, kw):
    with torch.no_grad():
        return [o.float() for o in m(**kw)]


def _trained(m):
    m.enable_act8()
    out, feats = m(*_inputs(False), feature_hook_block=-1)
    (out.square().sum() + feats.sum()).backward()
    return out.detach(), torch.cat([p.grad.reshape(-1) for p in m.parameters()])


def _worker(rank, world, port, train, queue):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world),
                      LOCAL_RANK=str(rank))
    try:
        from dmad_b200.parallel.cp import ContextParallel, HybridContextParallel
        from dmad_b200.parallel.dist import init_distributed

        torch.set_num_threads(1)
        init_distributed(backend="gloo", timeout_s=120)
        cp = ContextParallel(impl="nccl") if world == 2 else HybridContextParallel(ulysses_size=2)
        if train:
            m = _model()
            m.enable_context_parallel(cp)
            out, grads = _trained(m)
            dist.all_reduce(grads)
            res = [out, grads]
        else:
            m, kw, L = _h3()
            assert L % world
            m.enable_context_parallel(cp)
            res = _sampled(m, kw)
        queue.put((rank, [t.numpy() for t in res], None))
        dist.destroy_process_group()
    except Exception:  # pragma: no cover
        import traceback
        queue.put((rank, None, traceback.format_exc()))


@pytest.mark.parametrize("world,train", [(2, False), (4, False), (2, True)])
def test_sharded_matches_unsharded(world, train):
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, train, queue)) for r in range(world)]
    for p in procs:
        p.start()
    res = [queue.get(timeout=300) for _ in procs]
    for p in procs:
        p.join(timeout=60)
    want = list(_trained(_model())) if train else _sampled(*_h3()[:2])
    assert all(w.norm() > 0 for w in want)
    # The attention sums in another order.  int8 in bf16: a last bit of its output (2^-8), and a number next to a border of two
    # codes goes to the other, 2^-7 of its row's largest away.  Kept codes of fp32: one number in 10^4 within fp32's noise of
    # a border, 2^-6 of its block's largest away, which is 2^-6 / 100 in norm.
    rel = 1e-3 if train else 2e-2
    for _, out, err in res:
        assert err is None, err
        for o, w in zip(out, want):
            assert (torch.from_numpy(o) - w).norm() <= rel * w.norm()
