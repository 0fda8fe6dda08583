"""The 4-bit floating point products, the norm with codes and the choice of experts across contexts, streams and
captures."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty
from tests.test_gpu_mx4 import buffers, make_weight
from tests.test_gpu_select import rule_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh():
    c = rocm.Context(0)
    yield c
    c.close()


def test_two_contexts_share_a_weight_on_streams_of_their_own(ctx, fresh):
    """Calls of both contexts are under way together, each with its own workspace: the bits of each alone."""
    import torch
    rng = np.random.default_rng(51)
    n, k = 200, 2100
    w, _ = make_weight(ctx, rng, n, k)
    rows = [1, 4, 20, 90, 300, 1000]
    xs = [[dev(rng.standard_normal((m, k)).astype(np.float32)) for m in rows] for _ in range(2)]
    norm = dev(np.ones(k, np.float32))
    logits = dev(rng.standard_normal((500, 64)).astype(np.float32))
    rule = rule_of(64, 6, 1, 8, 3, 2)

    def run(context, c):
        out = []
        for x, m in zip(xs[c], rows):
            y, z = empty((m, n), torch.float32), empty((m, n), torch.bfloat16)
            q, s = buffers(m, k)
            context.mx4_linear(w, x, rocm.F32, m, y, rocm.F32)
            context.add_rmsnorm_mx4(x, x, rocm.F32, m, k, norm, 1e-6, None, q, s, zero_centered=False)
            context.mx4_linear_q4(w, q, s, m, z, rocm.BF16)
            out += [y, z]
        ids, shares = empty((500, 6), torch.int32), empty((500, 6), torch.float32)
        context.moe_select(rule, logits, rocm.F32, 500, None, ids, shares)
        return out + [ids, shares]

    alone = []
    for c in range(2):
        alone.append(run(ctx, c))
        ctx.sync()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ctx.set_stream(streams[0].cuda_stream)
    fresh.set_stream(streams[1].cuda_stream)
    try:
        for _ in range(3):
            got = [run(ctx, 0), run(fresh, 1)]
            ctx.sync()
            fresh.sync()
            for c in range(2):
                assert all(torch.equal(a, b) for a, b in zip(got[c], alone[c]))
    finally:
        ctx.set_stream(None)
        fresh.set_stream(None)
    w.free()


def test_capture_refuses_growth_and_synchronous_calls(fresh):
    """A call whose workspace does not fit yet, and calls that allocate or wait, record nothing; later they run. What
    needs no workspace records at once."""
    import torch
    rng = np.random.default_rng(52)
    n, k, m = 300, 9000, 600
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda")
    scales = torch.full((n, -(-k // 32)), 120, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    w = fresh.mx4_weight(codes, scales, n, k)
    x, y = dev(rng.standard_normal((m, k)).astype(np.float32)), empty((m, n), torch.float32)
    one, few = empty((1, n), torch.float32), empty((m, n), torch.float32)
    norm = dev(np.ones(k, np.float32))
    q, s = buffers(m, k)
    stream = torch.cuda.Stream()
    fresh.set_stream(stream.cuda_stream)
    calls = (lambda: fresh.mx4_linear(w, x, rocm.F32, m, y, rocm.F32),
             lambda: fresh.mx4_weight(codes, scales, n, k),
             lambda: fresh.mx4_weight_quantize(x, rocm.F32, 8, 8),
             lambda: w.free())
    try:
        with torch.cuda.stream(stream):
            torch.cuda.synchronize()
            for call in calls:
                graph = torch.cuda.CUDAGraph()
                with pytest.raises(rocm.DzError) as e:
                    with rocm.capture(graph, stream):
                        y.zero_()
                        call()
                assert e.value.code == "INVALID_REQUEST"
            graph = torch.cuda.CUDAGraph()
            with rocm.capture(graph, stream):  # one row, and codes already made: no workspace
                fresh.mx4_linear(w, x, rocm.F32, 1, one, rocm.F32)
                fresh.add_rmsnorm_mx4(x, None, rocm.F32, m, k, norm, 0.0, None, q, s, zero_centered=False)
                fresh.mx4_linear_q4(w, q, s, m, few, rocm.F32)
            fresh.mx4_linear(w, x, rocm.F32, m, y, rocm.F32)
            first = y.clone()
            again = torch.cuda.CUDAGraph()
            with rocm.capture(again, stream):
                fresh.mx4_linear(w, x, rocm.F32, m, y, rocm.F32)
            eager_one, eager_few = torch.empty_like(one), torch.empty_like(few)
            fresh.mx4_linear(w, x, rocm.F32, 1, eager_one, rocm.F32)
            fresh.add_rmsnorm_mx4(x, None, rocm.F32, m, k, norm, 0.0, None, q, s, zero_centered=False)
            fresh.mx4_linear_q4(w, q, s, m, eager_few, rocm.F32)
            for _ in range(3):
                for t in (y, one, few):
                    t.zero_()
                graph.replay()
                again.replay()
                torch.cuda.synchronize()
                assert torch.equal(y, first) and torch.equal(one, eager_one) and torch.equal(few, eager_few)
                assert min(float(t.abs().max()) for t in (first, one, few)) > 0
    finally:
        fresh.set_stream(None)
    w.free()


@pytest.mark.parametrize("first,then", [(3, 700), (700, 3)])
def test_calls_in_turn_on_one_workspace(ctx, first, then):
    """Products of different sizes one after the other, none waited for: each as alone."""
    import torch
    rng = np.random.default_rng(first)
    n, k = 130, 640
    w, _ = make_weight(ctx, rng, n, k)
    xs = [dev(rng.standard_normal((m, k)).astype(np.float32)) for m in (first, 20, then)]
    alone = []
    for x in xs:
        y = empty((x.shape[0], n), torch.float32)
        ctx.mx4_linear(w, x, rocm.F32, x.shape[0], y, rocm.F32)
        ctx.sync()
        alone.append(y)
    got = [empty((x.shape[0], n), torch.float32) for x in xs]
    for _ in range(3):
        for x, y in zip(xs, got):
            ctx.mx4_linear(w, x, rocm.F32, x.shape[0], y, rocm.F32)
    ctx.sync()
    assert all(torch.equal(a, b) for a, b in zip(got, alone))
    w.free()
