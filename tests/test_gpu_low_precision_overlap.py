"""Two contexts at work at once on the low-precision operators: nothing of one's stands in the other's way."""
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


def test_two_contexts_at_once(ctx, fresh):
    """Products through each context's own workspace, norms and choices, enqueued in turn with nothing allocated or waited
    for in between, behind one event: both streams' calls start together, and give the bits of each alone."""
    import torch
    rng = np.random.default_rng(51)
    n, k, tokens = 200, 2100, 500
    w, _ = make_weight(ctx, rng, n, k)
    rows = [20, 300, 5, 1000, 90, 1, 17]
    norm = dev(np.ones(k, np.float32))
    logits = [dev(rng.standard_normal((tokens, 64)).astype(np.float32)) for _ in range(2)]
    rule = rule_of(64, 6, 1, 8, 3, 2)
    xs = [[dev(rng.standard_normal((m, k)).astype(np.float32)) for m in rows] for _ in range(2)]

    def outputs():
        made = [(empty((m, n), torch.float32), empty((m, n), torch.bfloat16), *buffers(m, k)) for m in rows]
        return made, empty((tokens, 6), torch.int32), empty((tokens, 6), torch.float32)

    def row(context, c, i, out):
        x, m, (y, z, q, s) = xs[c][i], rows[i], out[0][i]
        context.mx4_linear(w, x, rocm.F32, m, y, rocm.F32)
        context.add_rmsnorm_mx4(x, x, rocm.F32, m, k, norm, 1e-6, None, q, s, zero_centered=False)
        context.mx4_linear_q4(w, q, s, m, z, rocm.BF16)
        context.moe_select(rule, logits[c], rocm.F32, tokens, None, out[1], out[2])

    def results(out):
        return [t for made in out[0] for t in made[:2]] + [out[1], out[2]]

    alone, at_once = [outputs() for _ in range(2)], [outputs() for _ in range(2)]
    contexts = [ctx, fresh]
    for c in range(2):  # each context by itself: its workspace has its size afterwards
        for i in range(len(rows)):
            row(contexts[c], c, i, alone[c])
        contexts[c].sync()
    assert not torch.equal(alone[0][0][0][0], alone[1][0][0][0])
    a = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
    b, product = torch.randn_like(a), torch.empty_like(a)
    torch.mm(a, b, out=product)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    gate = torch.cuda.Event()
    for context, stream in zip(contexts, streams):
        context.set_stream(stream.cuda_stream)
    torch.cuda.synchronize()
    try:
        for _ in range(3):
            for out in at_once:
                for t in results(out):
                    t.fill_(0)
            for _ in range(4):  # some milliseconds, in which all calls below are enqueued
                torch.mm(a, b, out=product)
            gate.record()
            for stream in streams:
                stream.wait_event(gate)
            for i in range(len(rows)):
                for c in range(2):
                    row(contexts[c], c, i, at_once[c])
            ctx.sync()
            fresh.sync()
            torch.cuda.synchronize()
            for c in range(2):
                assert all(torch.equal(u, v) for u, v in zip(results(at_once[c]), results(alone[c])))
    finally:
        torch.cuda.synchronize()
        for context in contexts:
            context.set_stream(None)
    w.free()
