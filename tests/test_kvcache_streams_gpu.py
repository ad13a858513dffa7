"""The KV cache's calls on streams of the caller's and in captured graphs: what they keep must outlive the call."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kvcache as ok
from tests.test_kvcache_gpu import Case, ctx, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def _stream(torch, ctx, kind):
    """(handle to pass, the torch stream it is)"""
    if kind == "side":
        s = torch.cuda.Stream()
        return s.cuda_stream, s
    if kind == "context":
        return 0, torch.cuda.ExternalStream(ctx.stream)
    return 1, torch.cuda.default_stream()          # the legacy default stream


@pytest.mark.parametrize("kind", ["side", "context", "legacy"])
@pytest.mark.parametrize("op", ["extend", "compact"])
def test_page_copies_wait_for_their_stream(torch, ctx, kind, op):  # noqa: F811
    """The stream is busy when the copies are asked for, and the caller's next tensors are of the ids' size."""
    from raon_npu_b200.kvcache import KvCache
    pool = ok.Pool(2, 12, 2, 64, 16, rng=np.random.default_rng(0))
    dev = torch.from_numpy(pool.data.copy()).cuda()
    cache = KvCache(ctx, 2, 2, 64, 12, page_size=16, pool=dev)
    a, b = cache.new(), cache.new()
    cache.extend([a, b], [40, 21])
    c = cache.fork(b)
    if op == "compact":
        cache.free(a)
    torch.cuda.synchronize()
    handle, stream = _stream(torch, ctx, kind)
    seqs = [b, c]
    before = cache.page_pool.table(seqs)[0]
    current = torch.cuda.Stream()
    with torch.cuda.stream(current):
        torch.zeros(1, device="cuda")              # the current stream has memory by now
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            torch.cuda._sleep(40_000_000)          # some 20 ms
        if op == "extend":
            cache.extend(seqs, 1, stream=handle)
        else:
            assert cache.compact(stream=handle) == 2
        after = cache.page_pool.table(seqs)[0]
        moved = sorted({(int(s), int(d)) for s, d in zip(before.ravel(), after.ravel()) if s != d})
        assert len(moved) == (1 if op == "extend" else 2)
        # page 11 onto itself, were these taken for the moves
        others = [torch.full((2, len(moved)), 11, dtype=torch.int32, device="cuda") for _ in range(64)]
        current.synchronize()
    torch.cuda.synchronize()
    ctx.sync()
    for s, d in moved:
        pool.data[:, d] = pool.data[:, s]
    assert np.array_equal(dev.cpu().numpy(), pool.data)
    assert all((o == 11).all() for o in others)


@pytest.mark.parametrize("d,hq,heads", [(128, 8, 2), (64, 24, 2)])
def test_captured_calls_outlive_the_growth_of_scratch(torch, ctx, d, hq, heads):  # noqa: F811
    """Batches of 1, 2, 4 and 8 sequences captured in that order, on tables that widen: every one asks for more scratch
    than the last, and the earlier graphs go on giving their bytes without touching anybody else's memory."""
    from raon_npu_b200.device import Context
    own = Context(0)                                       # with no scratch yet
    graphs = []
    for i, n in enumerate((1, 2, 4, 8)):
        c = Case(torch, own, d, heads, 16, [1500 + 17 * k for k in range(n)], seed=n, extra_cols=2 + 400 * i, layers=1)
        c.layer = 0
        q = torch.randn((n, hq, d), device="cuda").bfloat16()
        out = torch.zeros_like(q)
        c.cache.attend(0, q, c.batch, out)                 # grows what it needs
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            c.cache.attend(0, q, c.batch, out)
        graphs.append((graph, out, out.clone(), c, q))
    torch.cuda.empty_cache()
    others = [torch.full((1 << k,), 0x5A, dtype=torch.uint8, device="cuda") for k in range(9, 26) for _ in range(3)]
    for _ in range(2):
        for graph, out, want, _, _ in graphs:
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    own.sync()
    assert all((o == 0x5A).all() for o in others)
    del graphs, graph
    own.close()
