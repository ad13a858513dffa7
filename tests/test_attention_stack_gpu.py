"""The attention-stack example: the projections, the cache and its pages together."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def torch():
    import torch as _t
    return _t


@pytest.fixture(scope="module")
def ctx():
    from raon_npu_b200.build import build
    build()
    from raon_npu_b200.device import Context
    c = Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("window,sinks", [(0, 0), (48, 3)])
def test_forks_and_moved_pages_give_the_same_bytes(torch, ctx, window, sinks):
    """A fork that is fed what its parent is fed gives the parent's bytes, also after other sequences have ended and
    the pages have moved; a step taken back and repeated gives the same bytes."""
    from raon_npu_b200.examples.attention_stack import AttentionStack
    stack = AttentionStack(ctx, layers=2, hidden=512, q_heads=8, kv_heads=2, head_dim=64, pages=40, page_size=16,
                           positions=256, window=window, sinks=sinks)
    cache = stack.cache
    gen = torch.Generator("cuda").manual_seed(3)
    rows = lambda n: torch.randn((n, 512), generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    other, parent = cache.new(), cache.new()
    ys = stack.prefill([other, parent], [rows(100), rows(41)])
    assert [y.shape[0] for y in ys] == [100, 41]
    child = cache.fork(parent)
    for _ in range(9):
        x = rows(2)
        y = stack.step([other, parent, child], torch.stack([x[0], x[1], x[1]]))
        assert torch.isfinite(y.float()).all() and torch.equal(y[1], y[2]) and not torch.equal(y[0], y[1])
    cache.free(other)
    for s in (parent, child):
        cache.trim(s, 49)
    assert cache.compact() > 0
    again = stack.step([child, parent], torch.stack([x[1], x[1]]))
    assert torch.equal(again[0], y[1]) and torch.equal(again[1], y[1])
    ctx.sync()


def test_the_program_runs(torch, capsys):
    from raon_npu_b200.examples import attention_stack
    attention_stack.main(["--layers", "2", "--steps", "3", "--window", "256", "--sinks", "4"])
    said = capsys.readouterr().out
    assert "a step" in said and said.strip().endswith("finite: True")
