"""Products on e4m3 weights and the mixture-of-experts layer across contexts, streams and captures."""
import numpy as np
import pytest

from decisive_amd import rocm
from tests.gpu_util import dev, empty
from tests.test_gpu_fp8 import make_weight

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh():
    c = rocm.Context(0)
    yield c
    c.close()


def _layer(ctx, rng, experts, top, hidden, ff):
    def codes(n, k):
        made = [make_weight(rng, n, k) for _ in range(experts)]
        return dev(np.stack([c for c, _ in made])), dev(np.stack([s for _, s in made]))

    router = dev((rng.standard_normal((experts, hidden)) * hidden ** -0.5).astype(np.float32))
    cfg = rocm.MoeConfig(experts=experts, top_k=top, hidden=hidden, ff=ff, renormalize=1)
    return ctx.moe(cfg, router, rocm.F32, codes(ff, hidden), codes(ff, hidden), codes(hidden, ff))


def test_two_contexts_share_handles_on_streams_of_their_own(ctx, fresh):
    """Calls of both contexts are under way together, each with its own workspace: the bits of each alone."""
    import torch
    rng = np.random.default_rng(51)
    n, k, tokens, hidden = 200, 4100, 9, 300
    codes, scales = make_weight(rng, n, k)
    w = ctx.fp8_weight(dev(codes), dev(scales), n, k)
    moe = _layer(ctx, rng, 12, 3, hidden, 200)
    rows = [1, 20, 90, 300]
    xs = [[dev(rng.standard_normal((m, k)).astype(np.float32)) for m in rows] for _ in range(2)]
    ts = [dev(rng.standard_normal((tokens, hidden)).astype(np.float32)) for _ in range(2)]
    dtypes = [rocm.F32, rocm.BF16]
    torch_types = [torch.float32, torch.bfloat16]

    def outputs(c):
        return [empty((m, n), torch_types[c]) for m in rows], empty((tokens, hidden), torch.float32)

    def forward(context, layer, x, count, y):
        context._check(rocm.load().dz_moe_forward(context.handle, layer.handle, x.data_ptr(), rocm.F32, count,
                                                  y.data_ptr()))

    alone = []
    for c in range(2):
        ys, y = outputs(c)
        for x, m, out in zip(xs[c], rows, ys):
            ctx.fp8_linear(w, x, rocm.F32, m, out, dtypes[c])
        forward(ctx, moe, ts[c], tokens, y)
        ctx.sync()
        alone.append((ys, y))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ctx.set_stream(streams[0].cuda_stream)
    fresh.set_stream(streams[1].cuda_stream)
    try:
        for _ in range(3):
            got = [outputs(0), outputs(1)]
            for i, m in enumerate(rows):
                for c, context in enumerate((ctx, fresh)):
                    context.fp8_linear(w, xs[c][i], rocm.F32, m, got[c][0][i], dtypes[c])
            for c, context in enumerate((ctx, fresh)):
                forward(context, moe, ts[c], tokens, got[c][1])
            ctx.sync()
            fresh.sync()
            for c in range(2):
                assert all(torch.equal(a, b) for a, b in zip(got[c][0], alone[c][0]))
                assert torch.equal(got[c][1], alone[c][1])
    finally:
        ctx.set_stream(None)
        fresh.set_stream(None)
    w.free()
    moe.free()


def test_capture_refuses_growth_and_synchronous_calls(fresh):
    """A call whose workspace does not fit yet, and calls that allocate or wait, record nothing; later they run."""
    import torch
    rng = np.random.default_rng(52)
    n, k, m, hidden = 300, 9000, 400, 300
    codes, scales = dev(make_weight(rng, n, k)[0]), dev(make_weight(rng, n, k)[1])
    w = fresh.fp8_weight(codes, scales, n, k)
    moe = _layer(fresh, rng, 4, 2, hidden, 9000)
    x, y = dev(rng.standard_normal((m, k)).astype(np.float32)), empty((m, n), torch.float32)
    q, s = empty((m, 71 * 128), torch.uint8), empty((71, m), torch.float32)
    t, out = dev(rng.standard_normal((128, hidden)).astype(np.float32)), empty((128, hidden), torch.float32)
    stream = torch.cuda.Stream()
    fresh.set_stream(stream.cuda_stream)
    calls = (lambda: fresh.fp8_linear(w, x, rocm.F32, m, y, rocm.F32),
             lambda: moe.forward(t, rocm.F32, 128, out),
             lambda: fresh.fp8_weight(codes, scales, n, k),
             lambda: fresh.fp8_weight_quantize(x, rocm.F32, 8, 8),
             lambda: w.free(),
             lambda: moe.free())
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
            fresh.fp8_quantize(x, rocm.F32, m, k, q, s)
            fresh.fp8_linear(w, x, rocm.F32, m, y, rocm.F32)
            moe.forward(t, rocm.F32, 128, out)
            first, first_out = y.clone(), out.clone()
            graph = torch.cuda.CUDAGraph()
            with rocm.capture(graph, stream):
                fresh.fp8_linear(w, x, rocm.F32, m, y, rocm.F32)
                moe.forward(t, rocm.F32, 128, out)
            for _ in range(3):
                y.zero_()
                out.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(y, first) and torch.equal(out, first_out)
                assert first.abs().max() > 0 and first_out.abs().max() > 0
    finally:
        fresh.set_stream(None)
    w.free()
    moe.free()
