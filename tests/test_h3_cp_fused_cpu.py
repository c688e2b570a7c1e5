"""The fused q / k norm and the 4-bit projections under context parallelism, on gloo CPU ranks: a padded packed sequence
over 2 ranks (head exchange) and over 4 (hybrid) against the same model unsharded."""
import os
import sys

import pytest
import torch
import torch.multiprocessing as mp

sys.path.insert(0, os.path.dirname(__file__))
from test_h3_cp_cpu import _free_port, _setup  # noqa: E402


def _models():
    """(fused fp32, fused and 4-bit bf16, inputs, packed length)."""
    m, kw, L = _setup()
    g = torch.Generator().manual_seed(3)
    for p in m.parameters():  # heads that are not zero, norm weights that are not one
        p.data.add_(0.03 * torch.randn(p.shape, generator=g))
    m.requires_grad_(False).enable_fused_qk_norm()
    q, _, _ = _setup()
    q.load_state_dict(m.state_dict())
    q.requires_grad_(False).bfloat16().quantize_fp4_("nvfp4")
    return m, q, kw, L


def _worker(rank, world, port, queue):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world),
                      LOCAL_RANK=str(rank))
    try:
        import torch.distributed as dist
        from dmad_b200.parallel.cp import ContextParallel, HybridContextParallel
        from dmad_b200.parallel.dist import init_distributed

        torch.set_num_threads(1)
        init_distributed(backend="gloo", timeout_s=120)
        cp = ContextParallel(impl="nccl") if world == 2 else HybridContextParallel(ulysses_size=2)
        out = []
        *nets, kw, L = _models()
        assert L % world
        with torch.no_grad():
            for m in nets:
                m.enable_context_parallel(cp)
                out += [o.float().numpy() for o in m(**kw)]
        queue.put((rank, out, None))
        dist.destroy_process_group()
    except Exception:  # pragma: no cover
        import traceback
        queue.put((rank, None, traceback.format_exc()))


@pytest.mark.parametrize("world", [2, 4])
def test_sharded_model_matches_unsharded(world):
    ctx = mp.get_context("spawn")
    queue = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, queue)) for r in range(world)]
    for p in procs:
        p.start()
    res = [queue.get(timeout=300) for _ in procs]
    for p in procs:
        p.join(timeout=60)
    *nets, kw, _ = _models()
    with torch.no_grad():
        want = [o.float() for m in nets for o in m(**kw)]
    assert all(w.norm() > 0 for w in want)
    for _, out, err in res:
        assert err is None, err
        for o, w in zip(out[:2], want[:2]):  # fp32: the unfused model's tolerance
            torch.testing.assert_close(torch.from_numpy(o), w, rtol=1e-4, atol=1e-5)
        for o, w in zip(out[2:], want[2:]):
            # bf16 attention summed in another order: a last bit (2^-8) of its output, and a number at a border of two
            # 4-bit codes (one in a hundred within a last bit of one) goes to the other, a quarter of its size away
            assert (torch.from_numpy(o) - w).norm() <= 5e-2 * w.norm()
