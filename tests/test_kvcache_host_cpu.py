"""What the KV cache does on the host around its launches, with stand-ins for tensors and streams."""

from __future__ import annotations

from types import SimpleNamespace

import pytest

from raon_npu_b200 import kvcache
from raon_npu_b200.build import build
from raon_npu_b200.kvcache import KvCache, PagePool


class Ids:
    """A tensor of page ids: which streams its memory waits for."""

    def __init__(self):
        self.streams = []

    def t(self):
        return self

    contiguous = t

    def to(self, dev):
        return self

    def record_stream(self, stream):
        self.streams.append(stream)

    def __getitem__(self, i):
        return self, i


@pytest.mark.parametrize("stream,waits_for", [(None, []), (0, ["external 777"]), (1, ["default"]), (4096, ["external 4096"])])
@pytest.mark.parametrize("op", ["extend", "compact"])
def test_the_moves_of_a_call_outlive_its_launch(monkeypatch, op, stream, waits_for):
    """The ids that extend and compact make are used on the caller's stream, so their memory has to wait for it."""
    build()
    ids, launched = Ids(), []
    cuda = SimpleNamespace(ExternalStream=lambda h, dev: f"external {h}", default_stream=lambda dev: "default")
    monkeypatch.setattr(kvcache, "torch", SimpleNamespace(tensor=lambda moves, dtype: ids, int32=None, cuda=cuda,
                                                          device=lambda kind, i: (kind, i)))
    cache = KvCache.__new__(KvCache)
    cache.ctx, cache.device, cache.handle = SimpleNamespace(device=0, stream=777, handle=None), 0, None
    cache._pages = pool = PagePool(8, 4)
    cache.move_pages = lambda src, dst, stream: launched.append((list(ids.streams), stream))
    a, b = pool.new(), pool.new()
    pool.extend([a, b], [2, 6])
    pool.fork(b)
    if op == "extend":
        cache.extend([b], 1, stream=stream)
    else:
        pool.free(a)
        assert cache.compact(stream=stream) == 1
    assert launched == [(waits_for, stream)]
