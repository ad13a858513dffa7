"""The 4-bit KV cache at sizes where its kernels take other paths: several heads a warp, more than 32 sequences, partial
rotations, prompts of several blocks under a window.  Bars as in test_kvcache_gpu.py: bytes equal for what is stored, a
query within one bf16 step of the 64-bit one, attention within ``Case.attend``'s bar.
"""

from __future__ import annotations

import numpy as np
import pytest

from oracle import kvcache as ok
from oracle import q4nx as q
from tests.test_kvcache_gpu import Case, bits, ctx, torch, value  # noqa: F401

pytestmark = pytest.mark.gpu


def stored_bytes_match(torch, ctx, c, hq, rope, inter):
    from raon_npu_b200.kvcache import rope_table
    rows, nh, d, heads, page = int(c.off[-1]), hq + 2 * c.heads, c.d, c.heads, c.page
    x = (2 * c.rng.standard_normal((rows, nh, d))).astype(np.float32)
    xb = q.f32_to_bf16(x)
    xin = value(xb)
    wq, wk = bits(1 + 0.2 * c.rng.standard_normal((2, d)))
    table = rope_table(max(c.lens), rope) if rope else None
    dev = lambda a: None if a is None else torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).cuda()  # noqa: E731
    qo = torch.zeros((rows, hq, d), dtype=torch.int16, device="cuda")
    c.cache.append(c.layer, dev(xb.reshape(rows, -1)), c.batch, qo, q_heads=hq, q_norm=dev(wq), k_norm=dev(wk), eps=1e-5,
                   rope=dev(table), interleaved=inter)
    torch.cuda.synchronize()
    ctx.sync()
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(c.lens, c.qs)])
    seq = np.repeat(np.arange(len(c.qs)), c.qs)
    qr = ok.norm_rope(xin[:, :hq], value(wq), 1e-5, table, pos, inter)
    kr = ok.norm_rope(xin[:, hq:hq + heads], value(wk), 1e-5, table, pos, inter)
    for r in range(rows):
        pg, at = c.table[seq[r], pos[r] // page], pos[r] % page
        c.pool.store("k", c.layer, pg, at, kr[r])
        c.pool.store("v", c.layer, pg, at, xin[r, hq + heads:])
    assert np.array_equal(c.dev_pool.cpu().numpy(), c.pool.data)
    got = value(qo.cpu().numpy().view(np.uint16))
    assert (np.abs(got - qr) <= 2.0**-8 * np.abs(qr) + 1e-6).all()


@pytest.mark.parametrize("d,hq,heads,rope,inter,n", [(64, 7, 3, 16, False, 2403), (64, 7, 3, 48, True, 1201),
                                                     (128, 5, 1, 128, False, 2405), (128, 5, 3, 80, False, 1001),
                                                     (128, 1, 3, 16, True, 2399)])
def test_append_of_many_rows(torch, ctx, d, hq, heads, rope, inter, n):  # noqa: F811
    """Rows enough for two and four units of heads a warp, odd head counts, units that hold keys and values."""
    c = Case(torch, ctx, d, heads, 64, [n + 19, 1, 333], [n, 1, 0], seed=n, fill=False)
    stored_bytes_match(torch, ctx, c, hq, rope, inter)


def test_append_of_many_sequences(torch, ctx):  # noqa: F811
    """Rows are found among sequences on both sides of every 32nd one, some without rows."""
    rng = np.random.default_rng(4)
    lens = rng.integers(1, 40, 131)
    qs = np.minimum(rng.integers(0, 4, 131), lens)
    qs[[0, 31, 32, 63, 64, 130]] = [0, 0, 1, 0, 0, 1]
    c = Case(torch, ctx, 64, 2, 16, lens.tolist(), qs.tolist(), seed=2, fill=False)
    stored_bytes_match(torch, ctx, c, 3, 64, False)


@pytest.mark.parametrize("d,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 5), (257, 140), (128, 0), (1, 1)])
def test_prompts_of_several_blocks(torch, ctx, d, page, window, sinks):  # noqa: F811
    c = Case(torch, ctx, d, 2, page, [1100, 385, 640], [300, 385, 129], seed=d + window)
    c.check(6, window=window, sinks=sinks)


def test_refusals_of_the_rotation(torch, ctx):  # noqa: F811
    from raon_npu_b200.kvcache import rope_table
    c = Case(torch, ctx, 64, 1, 16, [4], fill=False)
    x = torch.zeros((1, 3 * 64), dtype=torch.bfloat16, device="cuda")
    qo = torch.zeros((1, 64), dtype=torch.bfloat16, device="cuda")
    put = lambda rope, **k: c.cache.append(0, x, c.batch, qo, q_heads=1, rope=rope, **k)  # noqa: E731
    for dims in (8, 24, 80):
        with pytest.raises(ValueError, match="multiple of 16"):
            put(torch.from_numpy(rope_table(8, dims)).cuda())
    flat = torch.zeros(8 * 16 + 1, dtype=torch.float32, device="cuda")
    with pytest.raises(ValueError, match="aligned"):
        put(flat[1:].view(8, 16))
    with pytest.raises(ValueError, match="aligned"):
        put(None, q_norm=torch.zeros(65, dtype=torch.bfloat16, device="cuda")[1:])
    put(torch.from_numpy(rope_table(2, 16)).cuda())          # position 3 has no row in the table
    torch.cuda.synchronize()
    with pytest.raises(ValueError, match="outside"):
        ctx.sync()
    ctx.sync()
