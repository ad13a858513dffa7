"""The paged 4-bit KV cache in numpy and 64 bits: what ``rc_kv_append``, ``rc_kv_attend`` and ``rc_kv_read`` compute.

Written from the definitions in include/raon_cuda.h (the reference keeps its
attention state elsewhere, so there is nothing of it to restate): head norms
and rotation, the q4nx group rule of ``oracle.q4nx.quantize`` on 64-bit
values, and softmax attention over the dequantised rows.
"""

from __future__ import annotations

import math

import numpy as np

GROUP = 32


def bf16(x) -> np.ndarray:
    """Nearest bf16 (ties to even) of finite f64 values, as f64, with a single rounding."""
    x = np.asarray(x, np.float64)
    m, e = np.frexp(x)
    e = np.maximum(e, -125)          # bf16 subnormals start below 2^-126
    return np.ldexp(np.rint(np.ldexp(x, 8 - e)), e - 8)


def _toward(x: np.ndarray, up: bool) -> np.ndarray:
    """bf16 floor / ceiling of f64 values."""
    m, e = np.frexp(x)
    e = np.maximum(e, -125)
    y = np.ldexp(x, 8 - e)
    return np.ldexp(np.ceil(y) if up else np.floor(y), e - 8)


def quantise(x):
    """f64 [..., D] -> codes [..., D/32, 32], scales, mins [..., D/32] (all f64)."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, GROUP)
    lo, hi = g.min(-1), g.max(-1)
    mn = _toward(lo, False)
    sc = _toward((hi - mn) / 15.0, True)
    short = mn + 15.0 * sc < hi
    sc = np.where(short, _toward(np.nextafter(sc, np.inf), True), sc)
    flat = hi == mn
    sc = np.where(flat, 0.0, sc)
    code = np.clip(np.rint((g - mn[..., None]) / np.where(flat, 1.0, sc)[..., None]), 0, 15)
    return np.where(flat[..., None], 0, code), sc, mn


def dequantise(code, sc, mn) -> np.ndarray:
    v = mn[..., None] + sc[..., None] * code
    return v.reshape(*v.shape[:-2], v.shape[-2] * GROUP)


def norm_rope(x, w=None, eps=1e-6, table=None, pos=None, interleaved=False) -> np.ndarray:
    """f64 [T, H, D] heads: RMS norm with weight w [D], rotation by table [positions, R] (cos | sin) at pos [T]."""
    y = np.array(x, np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + float(np.float32(eps))) * np.asarray(w, np.float64)
    if table is not None:
        r = table.shape[1]
        t = np.asarray(table, np.float64)[pos][:, None]
        a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
        u = y[..., a] * t[..., :r // 2] - y[..., b] * t[..., r // 2:]
        v = y[..., a] * t[..., r // 2:] + y[..., b] * t[..., :r // 2]
        y[..., a], y[..., b] = u, v
    return y


def _order(d: int, kind: str) -> np.ndarray:
    """[D]: the nibble of value i within its row."""
    i = np.arange(d)
    w = 8 if kind == "k" else 4
    return ((i % GROUP) // w * (d // GROUP) + i // GROUP) * w + i % w


def pack_rows(code, sc, mn, kind: str):
    """codes uint8 [..., D/2] and params uint16 [..., D/32, 2] of quantised rows."""
    flat = code.reshape(*code.shape[:-2], code.shape[-2] * GROUP).astype(np.uint8)
    nib = np.empty_like(flat)
    nib[..., _order(flat.shape[-1], kind)] = flat
    par = np.stack([sc, mn], -1).astype(np.float32).view(np.uint32) >> 16
    return nib[..., 0::2] | (nib[..., 1::2] << 4), par.astype(np.uint16)


def unpack_rows(codes, par, kind: str) -> np.ndarray:
    """f64 [..., D] values of packed rows."""
    nib = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    c = nib[..., _order(nib.shape[-1], kind)].astype(np.float64)
    f = (par.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return dequantise(c.reshape(*c.shape[:-1], c.shape[-1] // GROUP, GROUP), f[..., 0], f[..., 1])


class Pool:
    """A pool [layers][pages][heads] of head blocks as bytes, with typed views."""

    def __init__(self, layers, pages, heads, dim, page, data=None, rng=None):
        self.dim, self.page = dim, page
        self.c, self.m = page * dim // 2, page * (dim // GROUP) * 4
        shape = (layers, pages, heads, 2 * (self.c + self.m))
        if data is None:
            data = rng.integers(0, 256, shape, dtype=np.uint8)      # bytes nothing valid was written to
        self.data = np.ascontiguousarray(data).reshape(shape)

    def part(self, kind: str):
        """(codes [layers, pages, heads, page, D/2], params uint16 [layers, pages, heads, page, D/32, 2]), views."""
        a = 0 if kind == "k" else self.c + self.m
        lead = self.data.shape[:3]
        codes = self.data[..., a:a + self.c].reshape(*lead, self.page, self.dim // 2)
        par = self.data[..., a + self.c:a + self.c + self.m].view(np.uint16)
        return codes, par.reshape(*lead, self.page, self.dim // GROUP, 2)

    def store(self, kind, layer, page, at, values) -> None:
        """values f64 [heads, D] at slot ``at`` of a page."""
        codes, par = pack_rows(*quantise(values), kind)
        a = 0 if kind == "k" else self.c + self.m
        d2, p4 = self.dim // 2, self.dim // GROUP * 4
        blk = self.data[layer, page]
        blk[:, a + at * d2:a + (at + 1) * d2] = codes
        b = a + self.c + at * p4
        blk[:, b:b + p4] = np.ascontiguousarray(par.reshape(par.shape[0], -1)).view(np.uint8)

    def rows(self, kind, layer, pages, n) -> np.ndarray:
        """f64 [heads, n, D]: the first n tokens of a sequence in ``pages``."""
        codes, par = self.part(kind)
        c = codes[layer, pages].transpose(1, 0, 2, 3).reshape(codes.shape[2], -1, self.dim // 2)[:, :n]
        p = par[layer, pages].transpose(1, 0, 2, 3, 4).reshape(codes.shape[2], -1, self.dim // GROUP, 2)[:, :n]
        return unpack_rows(c, p, kind)


def attend(q, k, v, first_pos: int, scale=None, window=0, sinks=0):
    """q f64 [n, Hq, D] at positions first_pos ..; k, v f64 [H, L, D].

    Returns (o [n, Hq, D], noise): noise = sqrt(sum_t (p_t v_t)^2) (1 + rms |q_i k_i| sqrt(D) scale), the size of
    the error that independent relative errors of one unit in p, k and v leave in o."""
    n, hq, d = q.shape
    h = k.shape[0]
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    o, noise = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    t = np.arange(k.shape[1])
    for i in range(n):
        p = first_pos + i
        see = t <= p
        if window > 0:
            see &= (t > p - window) | (t < sinks)
        if p < 0 or not see.any():
            continue
        for j in range(hq):
            kk, vv = k[j // (hq // h)][see], v[j // (hq // h)][see]
            s = kk @ q[i, j] * scale
            w = np.exp(s - s.max())
            w /= w.sum()
            o[i, j] = w @ vv
            spread = np.sqrt((w[:, None] * (kk * q[i, j]) ** 2).sum()) * abs(scale)
            noise[i, j] = np.sqrt((w[:, None] ** 2 * vv ** 2).sum(0)) * (1 + spread)
    return o, noise
