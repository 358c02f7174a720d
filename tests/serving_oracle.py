"""Plain float64 forms of the serving operators (append, gather, windowed and shared-prefix decode) on the CPU, written
from the cache layouts: byte by byte, token by token."""

from __future__ import annotations

import numpy as np

# layout name: (key bits, value bits, slot bytes)
LAYOUTS = {"soa": (4, 4, 134), "soa_k8": (8, 4, 196), "soa_k3": (3, 4, 118), "soa_k3v3": (3, 3, 102),
           "aos": (4, 4, 134), "aos_k8": (8, 4, 196), "aos_k3": (3, 4, 118), "aos_k3v3": (3, 3, 102)}
BLOCK, D = 16, 128


def places(layout: str, hk: int, t: int, h: int):
    """Byte offsets in a block of token t, head h: key codes, value codes, key norm (or None), scale, zero."""
    kb, vb, slot = LAYOUTS[layout]
    kn, vn = D * kb // 8, D * vb // 8
    if layout.startswith("aos"):
        at = (t * hk + h) * slot
        norm = None if kb == 8 else at + kn
        vat = at + kn + (0 if kb == 8 else 2)
        return at, vat, norm, vat + vn, vat + vn + 2
    at = (t * hk + h) * (kn + vn)
    fields = 2 if kb == 8 else 3
    meta = BLOCK * hk * (kn + vn) + h * fields * BLOCK * 2 + 2 * t
    m = [meta + 2 * BLOCK * i for i in range(fields)]
    return at, at + kn, (None if kb == 8 else m[0]), m[-2], m[-1]


def pack(codes: np.ndarray, bits: int) -> np.ndarray:
    out = np.zeros(D * bits // 8 + 1, np.uint8)
    for d, c in enumerate(codes):
        w = int(c) << (d * bits % 8)
        out[d * bits // 8] |= w & 255
        out[d * bits // 8 + 1] |= w >> 8
    return out[:-1]


def unpack(raw: np.ndarray, bits: int) -> np.ndarray:
    r = np.append(raw, 0).astype(np.int64)
    d = np.arange(D) * bits
    return ((r[d // 8] | (r[d // 8 + 1] << 8)) >> (d % 8)) & ((1 << bits) - 1)


def f8(raw: np.ndarray) -> np.ndarray:
    import torch

    return torch.from_numpy(np.ascontiguousarray(raw)).view(torch.float8_e4m3fn).double().numpy()


def read(cache: np.ndarray, layout: str, slots, cents):
    """(keys, values), float64 [n, Hk, 128], of the cache [blocks, 16, Hk, slot]; zeros for slots that do not exist."""
    kb, vb, _ = LAYOUTS[layout]
    nb, _, hk, _ = cache.shape
    flat = cache.reshape(nb, -1)
    k, v = np.zeros((2, len(slots), hk, D))
    for i, s in enumerate(slots):
        if s < 0 or s >= nb * BLOCK:
            continue
        page = flat[s // BLOCK]
        half = lambda at: float(page[at:at + 2].view(np.float16)[0])  # noqa: E731
        for h in range(hk):
            ka, va, norm, scale, zero = places(layout, hk, int(s) % BLOCK, h)
            if kb == 8:
                k[i, h] = f8(page[ka:ka + D])
            else:
                c = cents.astype(np.float64)[unpack(page[ka:ka + D * kb // 8], kb)]
                if layout.startswith("aos"):
                    c = c / np.sqrt((c * c).sum() + 1e-16)
                k[i, h] = c * half(norm)
            v[i, h] = unpack(page[va:va + D * vb // 8], vb) * half(scale) + half(zero)
    return k, v


def rope(x: np.ndarray, cs: np.ndarray, interleaved: bool) -> np.ndarray:
    """x float64 [n, H, 128] turned by cs [n, r] (float32 table rows)."""
    x, r = x.copy(), cs.shape[1]
    c, s = cs[:, None, : r // 2].astype(np.float64), cs[:, None, r // 2:].astype(np.float64)
    i = np.arange(r // 2)
    i, j = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    a, b = x[..., i], x[..., j]
    x[..., i], x[..., j] = a * c - b * s, b * c + a * s
    return x


def append(cache, layout, key, value, slots, positions, cos_sin, R, mids, cents, *, interleaved=False,
           norm_correction=True):
    """The cache after the append (a copy).  key, value: float32 arrays holding the inputs' exact numbers."""
    import torch

    kb, vb, _ = LAYOUTS[layout]
    cache = cache.copy()
    nb, _, hk, _ = cache.shape
    flat = cache.reshape(nb, -1)
    x = key.astype(np.float64)
    if positions is not None:
        ok = (positions >= 0) & (positions < len(cos_sin))
        x = rope(x, cos_sin[np.where(ok, positions, 0)], interleaved)
    else:
        ok = np.ones(len(key), bool)
    one, top = np.float32, (1 << vb) - 1
    for n, s in enumerate(slots):
        if s < 0 or s >= nb * BLOCK or not ok[n]:
            continue
        page = flat[s // BLOCK]
        put = lambda at, v: page.__setitem__(slice(at, at + 2), np.array([v], np.float16).view(np.uint8))  # noqa: E731
        for h in range(hk):
            ka, va, norm, scale, zero = places(layout, hk, int(s) % BLOCK, h)
            if kb == 8:
                e = torch.from_numpy(x[n, h].astype(np.float32)).clamp(-448, 448).to(torch.float8_e4m3fn)
                page[ka:ka + D] = e.view(torch.uint8).numpy()
            else:
                size = np.sqrt((x[n, h] ** 2).sum())
                y = x[n, h] @ R.astype(np.float64) / (size + 1e-8)
                code = (y[:, None] >= mids.astype(np.float64)[None]).sum(1)
                page[ka:ka + D * kb // 8] = pack(code, kb)
                if layout.startswith("soa") and norm_correction:
                    size = size / np.sqrt((cents.astype(np.float64)[code] ** 2).sum() + 1e-16)
                put(norm, size)
            v = value[n, h].astype(one)  # the store's fp32 steps
            low = v.min()
            if low == 0 and np.signbit(v[v == 0]).any():
                low = one(-0.0)  # IEEE 754-2019 minimum: -0 is below +0
            step = max(one(one(v.max() - low) / one(top)), one(1e-8))
            code = np.clip(np.trunc(((v - low) / step + one(0.5)).astype(one)), 0, top).astype(np.int64)
            page[va:va + D * vb // 8] = pack(code, vb)
            put(scale, step)
            put(zero, low)
    return cache


def attention(q, cache, layout, table, lens, cents, visible, *, scale=None, sinks=None):
    """(output [B, Hq, 128], lse [B, Hq], mean |v| under the weights [B, Hq, 128]) in float64; visible(t, L) says which
    tokens t < L each query sees.  q is in the cache's basis.  A row with nothing to see: NaN and -inf."""
    B, Hq, _ = q.shape
    hk = cache.shape[2]
    g = Hq // hk
    scale = 1 / np.sqrt(D) if scale is None else scale
    out, lse, size = np.full((B, Hq, D), np.nan), np.full((B, Hq), -np.inf), np.zeros((B, Hq, D))
    for b in range(B):
        L = min(int(lens[b]), table.shape[1] * BLOCK)
        t = np.arange(max(L, 0))
        t = t[visible(t, L)]
        if len(t) == 0:
            continue
        page = table[b][t // BLOCK].astype(np.int64)
        there = (page >= 0) & (page < len(cache))
        k, v = read(cache, layout, np.where(there, page * BLOCK + t % BLOCK, -1), cents)
        for h in range(Hq):
            s = k[:, h // g] @ q[b, h].astype(np.float64) * scale
            s[~there] = -np.inf
            vv = v[:, h // g]
            if sinks is not None:
                s, vv = np.append(s, float(sinks[h])), np.concatenate([vv, np.zeros((1, D))])
            top = s.max()
            w = np.exp(s - top)
            out[b, h] = w @ vv / w.sum()
            size[b, h] = w @ np.abs(vv) / w.sum()
            lse[b, h] = top + np.log(w.sum())
    return out, lse, size
