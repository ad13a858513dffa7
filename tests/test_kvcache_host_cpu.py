"""What the KV cache does on the host around its launches, with stand-ins for tensors and streams."""

from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest
import torch

from raon_npu_b200 import kvcache
from raon_npu_b200.build import build
from raon_npu_b200.kvcache import KvBatch, KvCache, PagePool


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


# ---------------------------------------------------------------- devices --
class Ints:
    """An int32 tensor on some GPU."""

    dtype, is_cuda = torch.int32, True

    def __init__(self, device, *shape, strides=None):
        self.device, self.shape = torch.device("cuda", device), torch.Size(shape)
        self.strides = strides or torch.empty(shape, device="meta").stride()

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        return self.strides if i is None else self.strides[i]

    def get_device(self):
        return self.device.index

    def data_ptr(self):
        return 16


def stand_in_cache(launched=None):
    """A cache on GPU 0 without its handle; ``launched`` takes what reaches rc_kv_move_pages."""
    cache = KvCache.__new__(KvCache)
    cache.ctx, cache.device, cache.handle = SimpleNamespace(device=0, handle=None), 0, None
    cache.lib = SimpleNamespace(rc_kv_move_pages=lambda *a: launched.append(a) or 0)
    return cache


def test_the_arrays_of_a_batch_are_on_one_gpu():
    ok = KvBatch(Ints(1, 2, 3), Ints(1, 2), Ints(1, 3), max_q=4)
    assert (ok.n_seqs, ok.columns, ok.ld) == (2, 3, 3)
    for table, kv_len, q_off in ((0, 1, None), (1, 0, 1), (0, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError, match="one device"):
            KvBatch(Ints(table, 2, 3), Ints(kv_len, 2), None if q_off is None else Ints(q_off, 3), 1)
    with pytest.raises(ValueError, match="the batch is on cuda:1"):
        stand_in_cache()._batch_args(ok, 2, "attend")


def test_the_arrays_of_a_move_are_on_the_caches_gpu():
    launched = []
    cache = stand_in_cache(launched)
    for src, dst, table in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, None)):
        with pytest.raises(ValueError, match="cuda:0"):
            cache.move_pages(Ints(src, 4), Ints(dst, 4), table=None if table is None else Ints(table, 2, 5), stream=7)
    assert not launched
    cache.move_pages(Ints(0, 4), Ints(0, 4), table=Ints(0, 2, 5, strides=(8, 1)), stream=7)
    assert launched == [(None, 16, 16, 4, 16, 2, 5, 8, 7)]


# ---------------------------------------------------------------- numbers --
@pytest.mark.parametrize("one", [3, np.int64(3), np.int32(3), np.array(3), torch.tensor(3)])
def test_counts_of_any_integer_type(one):
    build()
    pool = PagePool(8, 4)
    a, b = pool.new(), pool.new()
    pool.extend([a, b], one)
    pool.extend(np.array([a, b]), [one, 1])
    pool.extend(torch.tensor([b]), np.array([2]))
    assert [pool.tokens(a), pool.tokens(b)] == [6, 6]


@pytest.mark.parametrize("bad", [1.5, [1.0], "1", None, 2**31, [2**40]])
def test_counts_that_are_not_whole_numbers_are_refused(bad):
    build()
    pool = PagePool(8, 4)
    a = pool.new()
    with pytest.raises(ValueError):
        pool.extend([a], bad)
    with pytest.raises(ValueError):
        pool.extend([0.5], 1)
    with pytest.raises(ValueError):
        pool.table([0.5])
    assert pool.tokens(a) == 0
