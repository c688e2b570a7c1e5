"""8-bit operators called from several host threads at once, on one stream and on streams of their own, and beside replays
of a captured graph: the results of calls that are waited for."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _work(seed):
    """A thread's calls and what they give one by one."""
    from dmad_b200 import ops
    g = torch.Generator().manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).cuda()
    x, w, b = rand(700, 1000), ops.quantize_int8(rand(2600, 1000)), rand(2600)
    few, one = rand(40, 1000), rand(1, 1000)
    t = [rand(600, 512).requires_grad_(True), (rand(640, 512) * 0.05).requires_grad_(True), rand(640).requires_grad_(True)]
    gy = rand(600, 640)

    def calls():
        with torch.no_grad():
            out = [ops.int8_linear(v, w, b) for v in (x, few, one)]
            out.append(ops.dequantize_int8(ops.quantize_int8(x, 32)))
        y = ops.linear_act8(*t, "gelu_tanh")
        return out + [y.detach(), *torch.autograd.grad(y, t, gy)]

    torch.cuda.synchronize()
    want = calls()
    torch.cuda.synchronize()
    return calls, want


@pytest.mark.parametrize("own_stream", [False, True])
def test_threads(own_stream):
    from dmad_b200 import ops
    work = [_work(s) for s in range(4)]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x, w = torch.randn(300, 2000, device="cuda").bfloat16(), ops.quantize_int8(torch.randn(900, 2000, device="cuda"))
    ref = ops.int8_linear(x, w)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        y = ops.int8_linear(x, w)
    wrong, errors = [0] * len(work), []

    def run(i):
        try:
            calls, want = work[i]
            stream = torch.cuda.Stream() if own_stream else torch.cuda.default_stream()
            bad = torch.zeros((), dtype=torch.int64, device="cuda")
            stream.wait_stream(torch.cuda.default_stream())
            with torch.cuda.stream(stream):
                for _ in range(40):
                    for p, q in zip(calls(), want):
                        bad += (p != q).sum()
            stream.synchronize()
            wrong[i] = int(bad)
        except Exception as e:  # pragma: no cover
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(work))]
    for t in threads:
        t.start()
    with torch.cuda.stream(side):
        for _ in range(100):
            graph.replay()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors and wrong == [0] * len(work) and torch.equal(y, ref)
    ops.check_device_status()
