"""The 4-bit KV cache on the device against ``oracle.kvcache`` in 64 bits.

Bars.  Keys and values are computed and quantised in 64 bits on both sides:
bytes equal.  Query rows: bf16 of a 32-bit result, within one bf16 step of the
64-bit one (half a step of rounding, and 32-bit errors that can move a value
across a rounding boundary).  Attention: an element is off by at most
2^-8 |o| (bf16 rounding is 2^-9; the rest is the normalising sum, all of it
relative) plus 8 * 2^-11 * noise, noise = sqrt(sum (p v)^2) (1 + the spread of
a score's products): weights and dequantised values are rounded to 11 bits at
least, each independently, and eight standard deviations of what that leaves
are allowed.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kvcache as ok
from oracle import q4nx as q

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


def bits(x):
    """bf16 bits of f64 values (rounded once)."""
    return (ok.bf16(x).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)


def value(b):
    return q.bf16_to_f32(np.asarray(b, np.uint16)).astype(np.float64)


class Case:
    """Sequences with random pages in a random pool, mirrored in the oracle's pool."""

    def __init__(self, torch, ctx, d, heads, page, lens, qs=None, layers=2, seed=0, spare=3, extra_cols=2, k_scale=1.0,
                 v_scale=0.5, fill=True):
        from raon_npu_b200.kvcache import KvBatch, KvCache
        rng = self.rng = np.random.default_rng(seed)
        self.torch, self.ctx, self.d, self.heads, self.page, self.lens = torch, ctx, d, heads, page, list(lens)
        self.qs = [1] * len(lens) if qs is None else list(qs)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + spare
        order = rng.permutation(pages).astype(np.int32)
        self.table = np.full((len(lens), max(need + [1]) + extra_cols), -1, np.int32)
        k = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[k:k + n]
            k += n
        self.layers, self.layer = layers, layers - 1
        self.pool = ok.Pool(layers, pages, heads, d, page, rng=rng)
        if fill:
            mean = rng.standard_normal((heads, 1, d))
            for i, n in enumerate(lens):
                for t in range(n):
                    pg, at = self.table[i, t // page], t % page
                    self.pool.store("k", self.layer, pg, at, (k_scale * (rng.standard_normal((heads, 1, d)) + mean))[:, 0])
                    self.pool.store("v", self.layer, pg, at, v_scale * rng.standard_normal((heads, d)))
        dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
        self.dev_pool = dev(self.pool.data.copy())
        self.cache = KvCache(ctx, layers, heads, d, pages, page_size=page, pool=self.dev_pool)
        self.dev_table = dev(self.table)
        self.kv_len = dev(np.asarray(lens, np.int32))
        off = np.concatenate([[0], np.cumsum(self.qs)]).astype(np.int32)
        self.off = off
        self.q_off = None if qs is None else dev(off)
        self.batch = KvBatch(self.dev_table, self.kv_len, self.q_off, max(1, max(self.qs)) if qs is not None else 1)

    def kv(self, i):
        n = -(-self.lens[i] // self.page)
        return (self.pool.rows("k", self.layer, self.table[i, :n], self.lens[i]),
                self.pool.rows("v", self.layer, self.table[i, :n], self.lens[i]))

    def attend(self, hq, q_scale=1.5, scale=None, window=0, sinks=0, q_bits=None):
        """Device output, the oracle's, and the bar."""
        torch, rows = self.torch, int(self.off[-1])
        if q_bits is None:
            q_bits = bits(q_scale * self.rng.standard_normal((rows, hq, self.d)))
        qd = torch.from_numpy(q_bits.view(np.int16)).cuda()
        out = torch.full((rows, hq, self.d), 0x7FC0, dtype=torch.int16, device="cuda")
        self.cache.attend(self.layer, qd, self.batch, out, scale=scale, window=window, sinks=sinks)
        torch.cuda.synchronize()
        self.ctx.sync()
        got = value(out.cpu().numpy().view(np.uint16))
        o, noise = np.zeros(got.shape), np.zeros(got.shape)
        for i, (n, l) in enumerate(zip(self.qs, self.lens)):
            if n:
                k, v = self.kv(i)
                a = slice(self.off[i], self.off[i] + n)
                o[a], noise[a] = ok.attend(value(q_bits[a]), k, v, l - n, scale, window, sinks)
        return got, o, 2.0**-8 * np.abs(o) + 8 * 2.0**-11 * noise + 1e-30, q_bits

    def check(self, hq, **kw):
        got, o, bar, _ = self.attend(hq, **kw)
        worst = np.max(np.abs(got - o) / bar)
        assert worst <= 1, worst


# ----------------------------------------------------------------- append --
@pytest.mark.parametrize("d,hq,heads,page", [(128, 32, 4, 64), (64, 8, 8, 16), (128, 5, 1, 128), (64, 6, 2, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rope,inter,norm", [(0, False, False), (1, False, True), (1, True, True), (2, False, False),
                                             (2, True, True)])
def test_append_stores_the_oracles_bytes(torch, ctx, d, hq, heads, page, dtype, rope, inter, norm):
    from raon_npu_b200.kvcache import rope_table
    lens, qs = [17, 64, 1, 130, 33], [5, 64, 1, 2, 0]
    c = Case(torch, ctx, d, heads, page, lens, qs, seed=d + hq, fill=False)
    rng, rows, nh = c.rng, sum(qs), hq + 2 * heads
    x = (2 * rng.standard_normal((rows, nh, d))).astype(np.float32)
    x[1, hq:, 32:64] = 0.75                       # a flat group
    x[2, hq + heads:] = np.round(x[2, hq + heads:] * 4)   # many exact ties
    xb = q.f32_to_bf16(x)
    xin = value(xb) if dtype == "bf16" else x.astype(np.float64)
    wq, wk = (bits(1 + 0.2 * rng.standard_normal((2, d)))) if norm else (None, None)
    table = rope_table(200, d // rope) if rope else None
    pad = torch.zeros((rows, nh * d + 8), dtype=torch.int16 if dtype == "bf16" else torch.float32, device="cuda")
    xd = pad[:, :nh * d]                          # rows of a wider buffer
    xd.copy_(torch.from_numpy((xb.view(np.int16) if dtype == "bf16" else x).reshape(rows, -1)))
    dev = lambda a: None if a is None else torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()  # noqa: E731
    qo = torch.zeros((rows, hq, d), dtype=torch.int16, device="cuda")
    c.cache.append(c.layer, xd, c.batch, qo, q_heads=hq, q_norm=dev(wq), k_norm=dev(wk), eps=1e-5, rope=dev(table),
                   interleaved=inter)
    k_out = torch.zeros((rows, heads, d), dtype=torch.int16, device="cuda")
    v_out = torch.zeros_like(k_out)
    c.cache.read(c.layer, c.batch, k_out, v_out)
    torch.cuda.synchronize()
    ctx.sync()

    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, qs)])
    seq = np.repeat(np.arange(len(qs)), qs)
    val = lambda w: None if w is None else value(w)  # noqa: E731
    qr = ok.norm_rope(xin[:, :hq], val(wq), 1e-5, table, pos, inter)
    kr = ok.norm_rope(xin[:, hq:hq + heads], val(wk), 1e-5, table, pos, inter)
    vr = xin[:, hq + heads:]
    for r in range(rows):
        pg, at = c.table[seq[r], pos[r] // page], pos[r] % page
        c.pool.store("k", c.layer, pg, at, kr[r])
        c.pool.store("v", c.layer, pg, at, vr[r])
    assert np.array_equal(c.dev_pool.cpu().numpy(), c.pool.data)     # nothing else was written either
    got = value(qo.cpu().numpy().view(np.uint16))
    assert (np.abs(got - qr) <= 2.0**-8 * np.abs(qr) + 1e-6).all()
    for out, rows_ in ((k_out, kr), (v_out, vr)):
        held = ok.dequantise(*ok.quantise(rows_)).astype(np.float32).astype(np.float64)
        assert np.array_equal(out.cpu().numpy().view(np.uint16), bits(held))


def test_append_without_queries_and_on_idle_slots(torch, ctx):
    c = Case(torch, ctx, 64, 2, 16, [3, 0, 20], seed=5, fill=False)
    x = c.rng.standard_normal((3, 4 * 64)).astype(np.float32)
    c.cache.append(1, torch.from_numpy(x).cuda(), c.batch)
    torch.cuda.synchronize()
    ctx.sync()
    for i, n in ((0, 3), (2, 20)):
        for kind, a in (("k", 0), ("v", 128)):
            c.pool.store(kind, 1, c.table[i, (n - 1) // 16], (n - 1) % 16, x[i, a:a + 128].reshape(2, 64).astype(np.float64))
    assert np.array_equal(c.dev_pool.cpu().numpy(), c.pool.data)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -3.4e38])     # the bf16 floor of the last is -Inf
def test_append_of_a_value_without_a_four_bit_form(torch, ctx, bad):
    """The group reads NaN, its neighbours are stored, and the next synchronising call says so."""
    c = Case(torch, ctx, 128, 2, 16, [5], seed=6, fill=False)
    x = c.rng.standard_normal((1, 4 * 128)).astype(np.float32)
    x[0, 128 + 40] = bad                          # key head 1, group 1
    c.cache.append(0, torch.from_numpy(x).cuda(), c.batch)
    k, v = (torch.zeros((1, 2, 128), dtype=torch.int16, device="cuda") for _ in range(2))
    c.cache.read(0, c.batch, k, v)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="non-finite"):
        ctx.sync()
    ctx.sync()
    k = value(k.cpu().numpy().view(np.uint16))[0]
    assert np.isnan(k[1, 32:64]).all() and np.isfinite(k[0]).all()
    assert np.isfinite(k[1, :32]).all() and np.isfinite(k[1, 64:]).all()


# ----------------------------------------------------------------- attend --
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("hq,heads", [(8, 1), (4, 4), (10, 2), (32, 2)])
def test_decode_matches_the_oracle(torch, ctx, d, page, hq, heads):
    """One row a sequence, lengths around every boundary, an idle slot, garbage past the ends."""
    c = Case(torch, ctx, d, heads, page, [1, 15, 16, 17, 0, 63, 64, 65, 127, 129, 300], seed=page + hq)
    c.check(hq)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 0), (100, 70), (37, 129), (1000, 4)])
@pytest.mark.parametrize("qs", [None, [1, 3, 40, 0, 150]])
def test_windows_and_sinks(torch, ctx, window, sinks, qs):
    c = Case(torch, ctx, 64, 2, 16, [1, 65, 130, 200, 333], qs, seed=window + sinks)
    c.check(8, window=window, sinks=sinks)


@pytest.mark.parametrize("d,hq,heads,page", [(128, 8, 1, 64), (64, 4, 4, 16), (128, 10, 2, 128), (64, 32, 2, 32)])
def test_prompts_match_the_oracle(torch, ctx, d, hq, heads, page):
    """Ragged rows: whole prompts, chunks of longer contexts, single rows and sequences without rows."""
    c = Case(torch, ctx, d, heads, page, [1, 130, 257, 40, 300, 7], [1, 130, 129, 0, 33, 2], seed=d)
    c.check(hq)


def test_a_long_context(torch, ctx):
    """Enough tokens for many partial results of one row."""
    c = Case(torch, ctx, 64, 1, 128, [9001, 4097], seed=1)
    c.check(4)


@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(1e-3, 1.0, 1e-6), (30.0, 1.0, 1e4), (1.0, 8.0, 3e7), (1.0, 1e-4, 1e-20)])
def test_magnitudes(torch, ctx, q_scale, k_scale, v_scale):
    for qs in (None, [50, 5]):
        c = Case(torch, ctx, 64, 2, 32, [150, 70], qs, seed=2, k_scale=k_scale, v_scale=v_scale)
        c.check(8, q_scale=q_scale)


def test_negative_and_zero_scale(torch, ctx):
    c = Case(torch, ctx, 64, 1, 16, [100], seed=3)
    c.check(4, scale=0.0)
    c.check(4, scale=-0.2)


@pytest.mark.parametrize("qs", [None, [20, 90]])
def test_nan_in_hidden_tokens_stays_hidden(torch, ctx, qs):
    """Groups that read NaN: rows that see such a token are NaN, rows that do not are untouched by it."""
    c = Case(torch, ctx, 64, 2, 16, [100, 90], qs, seed=4)
    for i, t in ((0, 85), (1, 3)):                      # hidden by the mask from some rows, by the window from others
        _, par = c.pool.part("v")
        par[c.layer, c.table[i, t // 16], :, t % 16, 1] = 0x7FC0
        _, par = c.pool.part("k")
        par[c.layer, c.table[i, t // 16], 1, t % 16, 0] = 0x7FC0
    c.dev_pool.copy_(torch.from_numpy(c.pool.data))
    got, o, bar, _ = c.attend(4, window=16, sinks=2)
    assert np.array_equal(np.isnan(got), np.isnan(o))
    fine = ~np.isnan(o)
    assert fine.any() and (np.abs(got - o)[fine] <= bar[fine]).all()
    if qs is not None:
        assert not fine.all()


def test_rows_beyond_the_batch_are_left_alone(torch, ctx):
    from raon_npu_b200.kvcache import KvBatch
    c = Case(torch, ctx, 64, 1, 16, [30, 20], [3, 2], seed=7)
    qd = torch.zeros((8, 4, 64), dtype=torch.int16, device="cuda")
    out = torch.full((8, 4, 64), 77, dtype=torch.int16, device="cuda")
    c.cache.attend(1, qd, c.batch, out)
    few = KvBatch(c.dev_table, c.kv_len, c.q_off, max_q=1)      # an upper bound that does not hold: an error, no fault
    torch.cuda.synchronize()
    ctx.sync()
    assert (out[5:] == 77).all() and (out[:5] != 77).any()
    out.fill_(77)
    c.cache.attend(1, qd, few, out)
    torch.cuda.synchronize()
    assert (out[5:] == 77).all()
    try:
        ctx.sync()
    except ValueError:
        pass


@pytest.mark.parametrize("qs", [None, [3, 40, 130]])
def test_a_rows_bytes_do_not_depend_on_the_batch(torch, ctx, qs):
    from raon_npu_b200.kvcache import KvBatch
    c = Case(torch, ctx, 128, 2, 64, [700, 90, 1300], qs, seed=8)
    _, _, _, qb = c.attend(16)
    qd = torch.from_numpy(qb.view(np.int16)).cuda()
    whole = torch.empty_like(qd)
    for window, sinks in ((0, 0), (128, 4)):
        c.cache.attend(c.layer, qd, c.batch, whole, window=window, sinks=sinks)
        for i in range(3):
            rows = slice(int(c.off[i]), int(c.off[i + 1]))
            alone = torch.empty_like(qd[rows])
            off = None if qs is None else torch.tensor([0, c.qs[i]], dtype=torch.int32, device="cuda")
            one = KvBatch(c.dev_table[i:i + 1], c.kv_len[i:i + 1], off, c.batch.max_q)
            c.cache.attend(c.layer, qd[rows].contiguous(), one, alone, window=window, sinks=sinks)
            again = torch.empty_like(alone)
            c.cache.attend(c.layer, qd[rows].contiguous(), one, again, window=window, sinks=sinks)
            assert torch.equal(alone, whole[rows]) and torch.equal(alone, again)
    ctx.sync()


def test_strided_rows_other_streams_and_graphs(torch, ctx):
    """q inside a wider row, out likewise; the call on a side stream and in a captured step whose lengths change."""
    c = Case(torch, ctx, 128, 2, 16, [50, 200], seed=9)
    _, o, bar, qb = c.attend(8)
    wide = torch.zeros((2, 12 * 128), dtype=torch.int16, device="cuda")
    wide[:, 128:9 * 128] = torch.from_numpy(qb.view(np.int16).reshape(2, -1)).cuda()
    out = torch.zeros((2, 8 * 128 + 64), dtype=torch.bfloat16, device="cuda")
    qv, ov = wide[:, 128:9 * 128], out[:, 64:]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.cache.attend(1, qv, c.batch, ov)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    ref = ov.clone()
    assert (np.abs(ref.double().cpu().numpy().reshape(o.shape) - o) <= bar).all()
    assert (out[:, :64] == 0).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.cache.attend(1, qv, c.batch, ov)
    c.kv_len.copy_(torch.tensor([17, 0], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert (ov[1] == 0).all() and not torch.equal(ov[0], ref[0])
    c.kv_len.copy_(torch.tensor([50, 200], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(ov, ref)
    ctx.sync()


# ------------------------------------------------------------------ pages --
@pytest.mark.parametrize("n,rows,cols", [(1, 1, 1), (7, 5, 9), (60, 33, 130), (0, 2, 2)])
def test_moves_copy_pages_and_rewrite_tables(torch, ctx, n, rows, cols):
    from raon_npu_b200.kvcache import KvCache
    rng = np.random.default_rng(n)
    pool = ok.Pool(3, 130, 3, 64, 16, rng=rng)
    dev = torch.from_numpy(pool.data.copy()).cuda()
    cache = KvCache(ctx, 3, 3, 64, 130, page_size=16, pool=dev)
    order = rng.permutation(130).astype(np.int32)
    src, dst = order[:n].copy(), order[n:2 * n].copy()
    table = rng.integers(-1, 130, (rows, cols + 3)).astype(np.int32)
    table[np.isin(table, dst)] = -1
    td = torch.from_numpy(table.copy()).cuda()
    cache.move_pages(torch.from_numpy(src).cuda(), torch.from_numpy(dst).cuda(), table=td[:, :cols])
    torch.cuda.synchronize()
    ctx.sync()
    pool.data[:, dst] = pool.data[:, src]
    to = np.arange(131, dtype=np.int32)
    to[130] = -1
    to[src] = dst
    want = table.copy()
    want[:, :cols] = to[table[:, :cols]]
    assert np.array_equal(dev.cpu().numpy(), pool.data) and np.array_equal(td.cpu().numpy(), want)


def test_more_moves_than_one_hash_holds(torch, ctx):
    from raon_npu_b200.kvcache import KvCache
    pages, n = 12000, 5500
    cache = KvCache(ctx, 1, 1, 64, pages, page_size=16)
    order = np.random.default_rng(1).permutation(pages).astype(np.int32)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").reshape(60, 200).contiguous()
    cache.move_pages(torch.from_numpy(order[:n].copy()).cuda(), torch.from_numpy(order[n:2 * n].copy()).cuda(), table=table)
    torch.cuda.synchronize()
    ctx.sync()
    want = np.arange(pages, dtype=np.int32)
    want[order[:n]] = order[n:2 * n]
    assert np.array_equal(table.cpu().numpy().ravel(), want)


def test_forked_sequences_go_their_own_ways(torch, ctx):
    """extend / append / fork / compact through the cache: every sequence reads back what was appended to it."""
    from raon_npu_b200.kvcache import KvCache
    rng = np.random.default_rng(11)
    cache = KvCache(ctx, 2, 2, 64, 24, page_size=16)
    text = {}

    def grow(seqs, ns):
        cache.extend(seqs, ns)
        x = rng.standard_normal((sum(ns), 4 * 64)).astype(np.float32)
        batch = cache.batch(seqs, rows=ns)
        for layer in (0, 1):
            cache.append(layer, torch.from_numpy(x + layer).cuda(), batch)
        at = 0
        for s, n in zip(seqs, ns):
            text[s] = np.concatenate([text[s], x[at:at + n]])
            at += n

    def check():
        for s, x in text.items():
            batch = cache.batch([s], rows=[len(x)])
            for layer in (0, 1):
                k, v = (torch.zeros((len(x), 2, 64), dtype=torch.int16, device="cuda") for _ in range(2))
                cache.read(layer, batch, k, v)
                for got, cols in ((k, slice(0, 128)), (v, slice(128, 256))):
                    y = (x + np.float32(layer))[:, cols].reshape(-1, 2, 64).astype(np.float64)
                    held = ok.dequantise(*ok.quantise(y)).astype(np.float32).astype(np.float64)
                    assert np.array_equal(got.cpu().numpy().view(np.uint16), bits(held)), s
        ctx.sync()

    a, b = cache.new(), cache.new()
    text[a] = text[b] = np.zeros((0, 256), np.float32)
    grow([a, b], [21, 40])
    c, d = cache.fork(a), cache.fork(b)
    text[c], text[d] = text[a], text[b]
    check()
    grow([a, c, d], [1, 20, 3])
    check()
    cache.free(b)
    del text[b]
    cache.trim(a, 18)
    text[a] = text[a][:18]
    e = cache.fork(a)
    text[e] = text[a]
    cache.compact()
    free, high = cache.page_pool.info()
    assert high == 24 - free
    grow([e, a, d], [2, 15, 7])
    check()
    from raon_npu_b200._lib import CacheFull
    with pytest.raises(CacheFull):
        cache.extend([a], 16 * 24)
    check()


# --------------------------------------------------------------- refusals --
def test_refusals(torch, ctx):
    from raon_npu_b200.kvcache import KvBatch, KvCache
    c = Case(torch, ctx, 64, 2, 16, [20, 30], seed=12)
    z = lambda *s, dtype=torch.int16: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    q2, o2, x2 = z(2, 256), z(2, 256), z(2, 512)
    cache, batch = c.cache, c.batch
    rope = torch.zeros((40, 64), device="cuda")
    bad = [
        lambda: cache.attend(2, q2, batch, o2),                                     # no such layer
        lambda: cache.attend(0, z(2, 192), batch, z(2, 192)),                       # 3 heads over 2
        lambda: cache.attend(0, z(2, 250), batch, z(2, 250)),                       # not whole heads
        lambda: cache.attend(0, z(3, 256), batch, z(3, 256)),                       # rows without q_off
        lambda: cache.attend(0, q2, batch, z(2, 128)),
        lambda: cache.attend(0, q2.float(), batch, o2),
        lambda: cache.attend(0, q2, batch, z(256, 2).t()),                          # values apart
        lambda: cache.attend(0, z(2, 260)[:, 4:], batch, o2),                       # not on a 16-byte boundary
        lambda: cache.attend(0, q2, batch, o2, window=-1),
        lambda: cache.attend(0, q2, batch, o2, sinks=-1),
        lambda: cache.attend(0, q2, batch, o2, scale=float("nan")),
        lambda: cache.attend(0, q2.cpu(), batch, o2),
        lambda: cache.append(0, x2, batch, q_heads=4),                              # q_out missing
        lambda: cache.append(0, x2, batch, z(3, 256), q_heads=4),
        lambda: cache.append(0, z(2, 500), batch, q2, q_heads=4),
        lambda: cache.append(0, x2, batch, q2, q_heads=4, q_norm=z(128)),
        lambda: cache.append(0, x2, batch, q2, q_heads=4, rope=rope[:, :12].contiguous()),
        lambda: cache.append(0, x2, batch, q2, q_heads=4, rope=z(40, 128, dtype=torch.float32)),
        lambda: cache.append(0, x2, batch, q2, q_heads=4, rope=rope.double()),
        lambda: cache.append(0, x2, batch, q2, q_heads=4, eps=-1.0),
        lambda: cache.read(0, batch, z(2, 2, 64), z(3, 2, 64)),
        lambda: cache.read(0, batch, z(2, 64), z(2, 64)),
        lambda: cache.move_pages(z(2, dtype=torch.int32), z(3, dtype=torch.int32)),
        lambda: cache.move_pages(z(2), z(2)),
        lambda: cache.move_pages(z(99, dtype=torch.int32), z(99, dtype=torch.int32)),
        lambda: KvBatch(c.dev_table.long(), c.kv_len),
        lambda: KvBatch(c.dev_table, c.kv_len[:1]),
        lambda: KvBatch(c.dev_table, c.kv_len, q_off=z(2, dtype=torch.int32), max_q=2),
        lambda: KvBatch(c.dev_table, c.kv_len, max_q=2),
        lambda: KvCache(ctx, 2, 2, 64, 100, page_size=16, pool=c.dev_pool),         # too small
        lambda: KvCache(ctx, 2, 2, 80, 10, page_size=16),
        lambda: KvCache(ctx, 2, 2, 64, 10, page_size=48),
    ]
    before = c.dev_pool.clone()
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"case {i} was taken")
    torch.cuda.synchronize()
    ctx.sync()
    assert torch.equal(before, c.dev_pool)


@pytest.mark.parametrize("what", ["page", "length", "rope"])
def test_ids_and_lengths_outside_are_errors_not_faults(torch, ctx, what):
    c = Case(torch, ctx, 64, 2, 16, [20, 30], seed=13)
    rope = torch.zeros((25, 64), device="cuda")
    x, qo = torch.zeros((2, 512), dtype=torch.int16, device="cuda"), torch.zeros((2, 256), dtype=torch.int16, device="cuda")
    if what == "page":
        c.dev_table[1, 1] = 10_000
    elif what == "length":
        c.kv_len[1] = 1000
    calls = [lambda: c.cache.append(0, x, c.batch, qo, q_heads=4, rope=rope if what == "rope" else None)]
    if what != "rope":
        calls += [lambda: c.cache.attend(0, qo, c.batch, torch.empty_like(qo)),
                  lambda: c.cache.read(0, c.batch, *(torch.empty((2, 2, 64), dtype=torch.int16, device="cuda") for _ in "kv"))]
    for call in calls:
        call()
        torch.cuda.synchronize()
        with pytest.raises(ValueError, match="outside"):
            ctx.sync()
    ctx.sync()
