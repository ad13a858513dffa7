"""The KV cache's host side: page ownership against a plain model, refusals, and the oracle's own format."""

from __future__ import annotations

import ctypes
import random

import numpy as np
import pytest

from oracle import kvcache as ok
from oracle import q4nx
from raon_npu_b200 import _lib
from raon_npu_b200.build import build


@pytest.fixture(scope="module")
def PagePool():
    build()
    from raon_npu_b200.kvcache import PagePool as P
    return P


# ------------------------------------------------------------------ pages --
class Model:
    """Sequences as lists of token values; pages as a store that copies move values between."""

    def __init__(self, pages, size):
        self.size, self.store = size, [[None] * size for _ in range(pages)]
        self.text = {}

    def copy(self, moves):
        for s, d in moves:
            self.store[d] = list(self.store[s])

    def write(self, table, lo, values):
        for i, v in enumerate(values, lo):
            self.store[table[i // self.size]][i % self.size] = v

    def read(self, table, n):
        return [self.store[table[i // self.size]][i % self.size] for i in range(n)]


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("size", [1, 4, 16])
def test_sequences_keep_their_tokens(PagePool, seed, size):
    """Random extends, forks, trims, frees and compactions: what was written to a sequence is what it holds."""
    rng = random.Random(seed)
    pages = rng.choice([3, 17, 40])
    pool, m, count = PagePool(pages, size), Model(pages, size), 0
    for _ in range(300):
        op = rng.choice(["new", "extend", "extend", "extend", "fork", "trim", "free", "compact"])
        live = list(m.text)
        if op == "new":
            m.text[pool.new()] = []
        elif op == "extend" and live:
            seqs = rng.sample(live, rng.randint(1, len(live)))
            ns = [rng.choice([0, 1, 1, 2, size, 3 * size + 1]) for _ in seqs]
            before = [(pool.tokens(s), pool.table([s])[0].tolist()) for s in live]
            try:
                moves = pool.extend(seqs, ns)
            except _lib.CacheFull:
                assert before == [(pool.tokens(s), pool.table([s])[0].tolist()) for s in live]
                continue
            assert not {s for s, _ in moves} & {d for _, d in moves}
            m.copy(moves)
            for s, n in zip(seqs, ns):
                values = list(range(count, count + n))
                count += n
                m.write(pool.table([s])[0][0], len(m.text[s]), values)
                m.text[s] = m.text[s] + values
        elif op == "fork" and live:
            s = rng.choice(live)
            m.text[pool.fork(s)] = list(m.text[s])
        elif op == "trim" and live:
            s = rng.choice(live)
            n = rng.randint(0, len(m.text[s]))
            pool.trim(s, n)
            m.text[s] = m.text[s][:n]
        elif op == "free" and live:
            s = rng.choice(live)
            pool.free(s)
            del m.text[s]
        elif op == "compact":
            moves = pool.compact()
            assert not {s for s, _ in moves} & {d for _, d in moves}
            m.copy(moves)
            free, high = pool.info()
            assert high == pages - free
        held = set()
        for s, text in m.text.items():
            table, n = pool.table([s])
            assert n[0] == len(text) and m.read(table[0], len(text)) == text
            held |= set(table[0][:-(-len(text) // size)].tolist())
        assert pool.info()[0] == pages - len(held)


def test_a_full_pool_refuses_and_a_freed_page_is_used_again(PagePool):
    pool = PagePool(2, 4)
    a, b = pool.new(), pool.new()
    assert pool.extend([a], 5) == []
    with pytest.raises(_lib.CacheFull, match="1 pages needed, 0 free"):
        pool.extend([b], 1)
    pool.trim(a, 4)
    assert pool.extend([a, b], [0, 4]) == []
    assert pool.table([a, b])[0].tolist() == [[0], [1]]


def test_a_shared_tail_is_copied_once_per_writer(PagePool):
    pool = PagePool(8, 4)
    a = pool.new()
    pool.extend([a], 6)
    b, c = pool.fork(a), pool.fork(a)
    tail = pool.table([a])[0][0, 1]
    moves = pool.extend([a, b, c], 1)          # two take pages of their own, the last keeps the page
    assert [s for s, _ in moves] == [tail, tail]
    assert pool.table([c])[0][0, 1] == tail
    assert len({int(pool.table([s])[0][0, 1]) for s in (a, b, c)}) == 3
    assert len({int(pool.table([s])[0][0, 0]) for s in (a, b, c)}) == 1


def test_page_refusals(PagePool):
    pool = PagePool(4, 16)
    s = pool.new()
    with pytest.raises(ValueError):
        PagePool(0, 16)
    with pytest.raises(KeyError):
        pool.extend([s + 1], 1)
    with pytest.raises(ValueError, match="twice"):
        pool.extend([s, s], 1)
    with pytest.raises(ValueError):
        pool.extend([s], -1)
    with pytest.raises(ValueError):
        pool.extend([s], [1, 2])
    with pytest.raises(ValueError):
        pool.extend([s], 2**31 - 1)
    with pytest.raises(ValueError):
        pool.trim(s, 1)
    pool.extend([s], 40)
    with pytest.raises(ValueError, match="3 pages"):
        pool.table([s], columns=2)
    pool.free(s)
    for call in (lambda: pool.free(s), lambda: pool.tokens(s), lambda: pool.fork(s), lambda: pool.trim(s, 0),
                 lambda: pool.table([s], columns=1)):
        with pytest.raises(KeyError):
            call()
    assert pool.info() == (4, 0)


def test_pool_sizes_and_their_refusals():
    build()
    from raon_npu_b200.kvcache import KvCache, rope_table
    assert KvCache.pool_bytes(3, 4, 128, 10, 64) == 3 * 10 * 4 * 64 * 128 * 2 * 5 // 8
    assert KvCache.pool_bytes(48, 8, 128, 100_000, 128) == 48 * 100_000 * 8 * 128 * 160
    for bad in ((0, 4, 128, 10, 64), (1, 0, 128, 10, 64), (1, 4, 96, 10, 64), (1, 4, 128, 0, 64), (1, 4, 128, 10, 24)):
        with pytest.raises(ValueError):
            KvCache.pool_bytes(*bad)
    t = rope_table(5, 8)
    assert t.shape == (5, 8) and t.dtype == np.float32 and t[0].tolist() == [1] * 4 + [0] * 4
    with pytest.raises(ValueError):
        rope_table(5, 7)


def test_null_handles_are_refused_without_a_gpu():
    build()
    lib = _lib.load()
    h = ctypes.c_void_p()
    assert lib.rc_kv_create(None, 1, 1, 1, 64, 16, None, 0, ctypes.byref(h)) == _lib.RC_ERR_INVALID
    assert lib.rc_kv_append(None, 0, None, 0, 0, 0, 0, None, 1, 1, None, None, 0, None, None, 0.0, None, 0, 0, 0, None, 0,
                            None) == _lib.RC_ERR_INVALID
    assert lib.rc_kv_attend(None, 0, None, 0, 0, 0, None, 1, 1, None, None, 0, 1, 1.0, 0, 0, None, 0,
                            None) == _lib.RC_ERR_INVALID
    assert lib.rc_kv_read(None, 0, 0, None, 1, 1, None, None, 0, None, None, None) == _lib.RC_ERR_INVALID
    assert lib.rc_kv_move_pages(None, None, None, 0, None, 0, 0, 0, None) == _lib.RC_ERR_INVALID
    assert lib.rc_pages_new(None, None) == _lib.RC_ERR_INVALID
    assert lib.rc_kv_destroy(None) == 0 and lib.rc_pages_destroy(None) == 0


# ----------------------------------------------------------------- oracle --
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["k", "v"])
def test_rows_unpack_to_what_was_packed(d, kind):
    rng = np.random.default_rng(d)
    x = rng.standard_normal((5, d)) * np.exp(rng.standard_normal((5, 1)))
    q = ok.quantise(x)
    assert np.array_equal(ok.unpack_rows(*ok.pack_rows(*q, kind), kind), ok.dequantise(*q))
    step = np.repeat(q[1], ok.GROUP, -1)
    assert (np.abs(ok.dequantise(*q) - x) <= step / 2 * (1 + 1e-12)).all()


def test_the_group_rule_is_the_weight_quantisers():
    rng = np.random.default_rng(3)
    w = (rng.standard_normal((64, 256)) * 0.3).astype(np.float32)
    w[3] = 1.5
    w[5, :32] = 0
    codes, scales, mins = q4nx.quantize(w)
    c, s, m = ok.quantise(w.astype(np.float64))
    assert np.array_equal(c.reshape(w.shape), codes) and np.array_equal(s, scales) and np.array_equal(m, mins)


def test_bf16_rounding_is_the_converters():
    rng = np.random.default_rng(4)
    x = (rng.standard_normal(4096) * np.exp(8 * rng.standard_normal(4096))).astype(np.float32)
    x[:6] = [0, 1.00390625, 1.01171875, -3.0, 1e-40, 2.0**-126]
    assert np.array_equal(ok.bf16(x), q4nx.bf16_to_f32(q4nx.f32_to_bf16(x)).astype(np.float64))
