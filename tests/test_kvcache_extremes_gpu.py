"""The 4-bit KV cache where its arguments, lengths and values are extreme, in both attention kernels (a call whose
rows x group pass 255 goes to the one for prompts).  Bars as in test_kvcache_gpu.py.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kvcache as ok
from tests.test_kvcache_gpu import Case, bits, ctx, torch, value  # noqa: F401

pytestmark = pytest.mark.gpu

INT_MAX = 2**31 - 1


# --------------------------------------------------- windows, empty rows --
@pytest.mark.parametrize("window", [INT_MAX, INT_MAX - 1, 2**30, 301])
@pytest.mark.parametrize("sinks", [0, 3, INT_MAX])
@pytest.mark.parametrize("qs", [None, [3, 8, 2, 40, 5], [3, 100, 2, 40, 200]])
def test_windows_past_every_length(torch, ctx, window, sinks, qs):  # noqa: F811
    """The largest windows hide nothing, also beside idle slots and sequences with more rows than tokens."""
    c = Case(torch, ctx, 64, 2, 16, [0, 5, 0, 300, 150], qs, seed=21)
    c.check(8, window=window, sinks=sinks)


# ------------------------------------------------------------ magnitudes --
DECODE, PROMPT = [None, [50, 5]], [[100, 5]]       # with four heads a kv head


def values_up_to_the_largest(torch, ctx, qs):  # noqa: F811
    """Scales of values past 2^122, which append stores as finite groups."""
    c = Case(torch, ctx, 64, 2, 32, [150, 105], qs, seed=22, v_scale=5e37)
    assert (c.pool.part("v")[1][c.layer, c.table[0, 0], :, :, :, 0] >> 7).max() >= 127 + 122
    c.check(8)


@pytest.mark.parametrize("qs", DECODE)
def test_values_up_to_the_largest(torch, ctx, qs):  # noqa: F811
    values_up_to_the_largest(torch, ctx, qs)


def test_large_values_over_many_partial_results(torch, ctx):  # noqa: F811
    """As many chunks of a row as are joined in two steps."""
    c = Case(torch, ctx, 64, 1, 128, [9001], seed=30, v_scale=5e37, layers=1)
    c.layer = 0
    c.check(4)


@pytest.mark.parametrize("qs", PROMPT)
def test_values_up_to_the_largest_in_prompts(torch, ctx, qs):  # noqa: F811
    values_up_to_the_largest(torch, ctx, qs)


def keys_up_to_the_largest(torch, ctx, qs):  # noqa: F811
    """Scales of keys past 2^122 under queries so small that the scores are ordinary ones."""
    c = Case(torch, ctx, 64, 2, 32, [150, 105], qs, seed=23, k_scale=3e37)
    assert (c.pool.part("k")[1][c.layer, c.table[0, 0], :, :, :, 0] >> 7).max() >= 127 + 122
    c.check(8, q_scale=1e-37)


@pytest.mark.parametrize("qs", PROMPT)
def test_keys_up_to_the_largest_in_prompts(torch, ctx, qs):  # noqa: F811
    keys_up_to_the_largest(torch, ctx, qs)


# (queries 30 times as large are left out: the weights that this kernel takes as zero then decide elements whose other
# values are exactly zero)
@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(1e-3, 1.0, 1e-6), (1.0, 8.0, 3e7), (1.0, 1e-4, 1e-20)])
def test_magnitudes_of_prompts(torch, ctx, q_scale, k_scale, v_scale):  # noqa: F811
    c = Case(torch, ctx, 64, 2, 32, [150, 105], [100, 5], seed=2, k_scale=k_scale, v_scale=v_scale)
    c.check(8, q_scale=q_scale)


@pytest.mark.parametrize("qs", DECODE)
def test_keys_up_to_the_largest(torch, ctx, qs):  # noqa: F811
    keys_up_to_the_largest(torch, ctx, qs)


@pytest.mark.parametrize("qs", [None, [3, 50], [100, 5]])
def test_zero_and_negative_scales(torch, ctx, qs):  # noqa: F811
    """A scale of zero weighs all visible tokens alike, whatever the keys are."""
    c = Case(torch, ctx, 64, 2, 16, [150, 105], qs, seed=24)
    c.check(8, scale=0.0)
    c.check(8, scale=-0.2)
    big = Case(torch, ctx, 64, 2, 16, [150, 105], qs, seed=25, k_scale=3e37)
    big.check(8, scale=0.0)


# ------------------------------------------------------------- non-finite --
def test_nan_in_hidden_tokens_of_prompts(torch, ctx):  # noqa: F811
    """The prompt kernel's rows that see a group that reads NaN are NaN, those that do not are untouched by it."""
    c = Case(torch, ctx, 64, 2, 16, [100, 190], [20, 190], seed=4)
    for i, t in ((0, 85), (1, 3), (1, 140)):
        c.pool.part("v")[1][c.layer, c.table[i, t // 16], :, t % 16, 1] = 0x7FC0
        c.pool.part("k")[1][c.layer, c.table[i, t // 16], 1, t % 16, 0] = 0x7FC0
    c.dev_pool.copy_(torch.from_numpy(c.pool.data))
    got, o, bar, _ = c.attend(8, window=16, sinks=2)
    assert np.array_equal(np.isnan(got), np.isnan(o))
    fine = ~np.isnan(o)
    assert fine.any() and not fine.all() and (np.abs(got - o)[fine] <= bar[fine]).all()


@pytest.mark.parametrize("qs", [[3, 9], [100, 9]])
@pytest.mark.filterwarnings("ignore:invalid value")
def test_queries_that_are_not_finite(torch, ctx, qs):  # noqa: F811
    """A query head with NaN or Inf gives NaN to itself alone, and nothing to a row that sees no token."""
    c = Case(torch, ctx, 64, 2, 16, [150, 4], qs, seed=26)
    q = bits(c.rng.standard_normal((sum(qs), 8, 64)))
    n = qs[0]                                              # rows n .. n + 4 stand before their sequence's first token
    for row, head, what in ((0, 1, 0x7FC0), (2, 3, 0x7F80), (1, 6, 0xFF80), (n + 1, 0, 0x7FC0), (n + 2, 5, 0x7F80),
                            (n + 4, 7, 0xFFFF), (n + 6, 2, 0x7FC0), (n + 8, 4, 0x7F80)):
        q[row, head, (5 * row + head) % 64] = what
    got, o, bar, _ = c.attend(8, q_bits=q)
    assert np.array_equal(np.isnan(got), np.isnan(o)) and (got[n:n + 5] == 0).all()
    assert np.isnan(got).all(-1).sum() == np.isnan(got).any(-1).sum() == 5
    fine = ~np.isnan(o)
    assert (np.abs(got - o)[fine] <= bar[fine]).all()


# ----------------------------------------------------------------- append --
@pytest.mark.parametrize("norm", [False, True])
def test_append_of_groups_wider_than_the_largest_number(torch, ctx, norm):  # noqa: F811
    """A group from -3e38 to 3e38 has a finite scale, 4e37: it is stored as in 64 bits, without an error."""
    c = Case(torch, ctx, 64, 2, 16, [5], seed=27, fill=False)
    x = c.rng.standard_normal((1, 4 * 64)).astype(np.float32)
    for at in (3, 40, 64 + 9, 128 + 33, 192 + 1):
        x[0, at:at + 5] = [3e38, -3e38, 1e38, -2.5e38, 0.5]
    x[0, 128 + 2:128 + 4] = [3.38e38, -3.38e38]
    w = bits(np.full(64, 1e38)) if norm else None
    k = x[:, :128].reshape(1, 2, 64).astype(np.float64)
    if norm:
        x[0, :128] = c.rng.standard_normal(128)            # its norm weight takes it there
        k = ok.norm_rope(x[:, :128].reshape(1, 2, 64), value(w))
    c.cache.append(0, torch.from_numpy(x).cuda(), c.batch, k_norm=None if w is None else torch.from_numpy(w.view(np.int16)).cuda())
    torch.cuda.synchronize()
    ctx.sync()
    page = c.table[0, 0]
    c.pool.store("k", 0, page, 4, k[0])
    c.pool.store("v", 0, page, 4, x[0, 128:].reshape(2, 64).astype(np.float64))
    assert np.array_equal(c.dev_pool.cpu().numpy(), c.pool.data)


# ---------------------------------------------------------- empty batches --
@pytest.mark.parametrize("n_seqs", [0, 3])
def test_batches_without_rows(torch, ctx, n_seqs):  # noqa: F811
    """No sequences, or sequences without rows: nothing to do, and nothing done."""
    from raon_npu_b200.kvcache import KvBatch
    c = Case(torch, ctx, 64, 2, 16, [20, 30, 7], seed=28)
    before = c.dev_pool.clone()
    empty = lambda *s: torch.empty((0, *s), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    batches = [KvBatch(c.dev_table[:n_seqs], c.kv_len[:n_seqs], torch.zeros(n_seqs + 1, dtype=torch.int32, device="cuda"))]
    if n_seqs == 0:
        batches += [KvBatch(c.dev_table[:0], c.kv_len[:0]), c.cache.batch([])]
    else:
        seqs = [c.cache.new() for _ in range(n_seqs)]
        c.cache.extend(seqs, 5)
        batches.append(c.cache.batch(seqs, rows=[0] * n_seqs))
    for batch in batches:
        c.cache.append(0, empty(8 * 64), batch, empty(4 * 64), q_heads=4)
        c.cache.attend(0, empty(4 * 64), batch, empty(4, 64))
        c.cache.read(0, batch, empty(2, 64), empty(2, 64))
    torch.cuda.synchronize()
    ctx.sync()
    assert torch.equal(before, c.dev_pool)


# ---------------------------------------------------------------- scratch --
@pytest.mark.parametrize("tokens,chunks,groups", [(131072, 171, 11), (8192, 11, 0), (896, 2, 0)])
def test_scratch_holds_what_the_table_can_ask_for(torch, ctx, tokens, chunks, groups):  # noqa: F811
    """64 sequences of 8 kv heads: room for the chunks that a sequence as long as its table row has (of six stages of 128
    tokens from 48 stages on, eight or fewer below), and no more than rounding beside it."""
    from raon_npu_b200.device import Context
    from raon_npu_b200.kvcache import KvBatch, KvCache
    own = Context(0)
    cache = KvCache(own, 1, 8, 128, 64, page_size=128)
    table = torch.arange(64, dtype=torch.int32, device="cuda").reshape(64, 1).repeat(1, tokens // 128)
    batch = KvBatch(table, torch.full((64,), 77, dtype=torch.int32, device="cuda"))
    x = torch.randn((64, 24 * 128), device="cuda").bfloat16()
    q, out = torch.zeros((64, 8 * 128), device="cuda").bfloat16(), torch.zeros((64, 8 * 128), device="cuda").bfloat16()
    cache.append(0, x, batch, q, q_heads=8)
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    cache.attend(0, q, batch, out)
    torch.cuda.synchronize()
    used = free - torch.cuda.mem_get_info()[0]
    assert used <= 64 * 8 * (chunks + groups) * 8 * 130 * 4 + (4 << 20)
    own.sync()
    cache.close()
    own.close()


# ------------------------------------------------- bounds, many, far away --
@pytest.mark.parametrize("max_q", [1, 50, 70])
def test_a_bound_of_rows_that_does_not_hold(torch, ctx, max_q):  # noqa: F811
    """More rows than max_q says: those within it are computed, the others left alone, and the next synchronising call
    says so, in both kernels."""
    from raon_npu_b200.kvcache import KvBatch
    c = Case(torch, ctx, 64, 2, 16, [120, 90], [100, 80], seed=29)
    q = torch.randn((180, 8, 64), device="cuda").bfloat16()
    whole, out = torch.zeros_like(q), torch.full_like(q, 7.0)
    c.cache.attend(1, q, c.batch, whole)
    torch.cuda.synchronize()
    ctx.sync()
    c.cache.attend(1, q, KvBatch(c.dev_table, c.kv_len, c.q_off, max_q), out)
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="outside"):
        ctx.sync()
    ctx.sync()
    for first, rows in ((0, 100), (100, 80)):
        assert (out[first + max_q:first + rows] == 7).all()
        assert torch.isfinite(out[first:first + max_q].float()).all()
        if max_q == 70:                                    # the same kernel
            assert torch.equal(out[first:first + max_q], whole[first:first + max_q])


@pytest.mark.parametrize("n,most", [(70, 1), (300, 1), (45, 9), (70, 60)])
def test_many_sequences(torch, ctx, n, most):  # noqa: F811
    """Sequences past every 32nd and 256th, of one row, a few, and enough for the prompt kernel; some without rows."""
    rng = np.random.default_rng(n + most)
    qs = rng.integers(0, most + 1, n)
    qs[[0, 31, 32]] = 0, most, 0
    lens = qs + rng.integers(0, 30, n)
    lens[5] = 0 if most == 1 else max(1, qs[5] // 2)       # idle, or rows before the first token
    c = Case(torch, ctx, 64, 1, 16, lens.tolist(), qs.tolist(), seed=31)
    c.check(8)
    c.check(8, window=9, sinks=2)


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_past_four_gigabytes(torch, ctx, rows):  # noqa: F811
    """The last pages and the last layer of a pool of 6.6 GB give what the first ones give, after an append and a move."""
    from raon_npu_b200.kvcache import KvBatch, KvCache
    pages = 20000
    cache = KvCache(ctx, 2, 8, 128, pages, page_size=128)
    kv_len = torch.tensor([300, 17 + rows], dtype=torch.int32, device="cuda")
    x = torch.randn((2 * rows, 48 * 128), device="cuda").bfloat16()
    past = torch.randn((317 + rows, 48 * 128), device="cuda").bfloat16()
    outs = []
    for layer, first in ((0, 0), (1, pages - 8)):
        table = torch.arange(first, first + 8, dtype=torch.int32, device="cuda").reshape(2, 4).flip(1).contiguous()
        q = torch.empty((317 + rows, 32 * 128), device="cuda").bfloat16()
        whole = KvBatch(table, kv_len, torch.tensor([0, 300, 317 + rows], dtype=torch.int32, device="cuda"), 300)
        cache.append(layer, past, whole, q, q_heads=32)
        batch = KvBatch(table, kv_len, torch.arange(0, 2 * rows + 1, rows, dtype=torch.int32, device="cuda"), rows)
        q = q[:2 * rows]
        cache.append(layer, x, batch, q, q_heads=32)
        out = torch.zeros_like(q)
        cache.attend(layer, q, batch, out)
        kv = [torch.zeros((317 + rows, 8, 128), device="cuda").bfloat16() for _ in "kv"]
        cache.read(layer, whole, *kv)
        other = table + (8 if first == 0 else -8)
        cache.move_pages(table.reshape(-1), other.reshape(-1).contiguous(), table=table)
        moved = torch.zeros_like(q)
        cache.attend(layer, q, batch, moved)
        assert torch.equal(table, other) and torch.equal(moved, out) and out.float().abs().sum() > 0
        outs.append([q.clone(), out, *kv])
    torch.cuda.synchronize()
    ctx.sync()
    for low, high in zip(*outs):
        assert torch.equal(low, high)
    cache.close()


# -------------------------------------------------------------- precision --
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("qs", [None, [40, 7], [150, 40]])
def test_the_noise_is_that_of_operands_of_eleven_bits(torch, ctx, d, qs):  # noqa: F811
    """The outputs' error in root mean square, against the rounding to bf16 and 2^-11 of ``noise``: weights, values and (in
    prompts) keys are each off by up to 2^-12, evenly spread, which is 2^-12 of ``noise`` for the three together, and
    twice that is allowed.  Operands of nine bits would have four times as much."""
    lens = [400, 333]
    c = Case(torch, ctx, d, 2, 64, lens, qs, seed=d)
    got, o, _, q = c.attend(4 * 2)
    noise = np.zeros_like(o)
    for i, n in enumerate(c.qs):
        a = slice(c.off[i], c.off[i] + n)
        noise[a] = ok.attend(value(q[a]), *c.kv(i), lens[i] - n)[1]
    rms = lambda x: np.sqrt((x * x).mean())  # noqa: E731
    assert rms(got - o) ** 2 <= rms(ok.bf16(o) - o) ** 2 * 1.01 + (2.0**-11 * rms(noise)) ** 2
