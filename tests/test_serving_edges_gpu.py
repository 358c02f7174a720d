"""Serving operators where numbers, sizes or alignment are at their ends, against float64 forms."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import serving_oracle as SO
import tqb
from test_serving_gpu import batch, book, cos_sin_table, cuda, half_step, no_wait_timeouts, npy, random_cache  # noqa: F401

pytestmark = pytest.mark.gpu


def put_half(cache, layout, page, t, field, value):
    """Sets a token's norm (field 2), scale (3) or zero (4), head 0."""
    at = SO.places(layout, cache.shape[2], t, 0)[field]
    cache.reshape(len(cache), -1)[page, at:at + 2] = np.array([value], np.float16).view(np.uint8)


def share(monkeypatch, chunks=None):
    monkeypatch.setattr(tqb.serving, "_shares", lambda *a: True)
    if chunks is not None:
        monkeypatch.setattr(tqb.serving, "_prefix_splits", lambda *a: chunks)


@pytest.mark.parametrize("chunks", [1, 2])
def test_prefix_of_one_token_that_outweighs_the_rest(monkeypatch, chunks):
    """A first token of value 0 that takes nearly all of the weight, the others 2^-26 of it each: the output is theirs.

    Every key is its norm times one vector c and every query a multiple of c, so the products q_i k_i are positive, and a
    score is off by at most 3 * 2^-11 of itself (q, c and c norm rounded to fp16): 0.033 for the difference of the two
    scores (20.3 and 2.25).  The small weights stand 2^-26 below the largest, which the reference keeps at 2^7 at least:
    spacing 2^-24, half of it 2^-6 of a weight.  0.049 in all, 0.06 with what the values' rounding and the sums add."""
    share(monkeypatch, chunks)
    rng = np.random.default_rng(21)
    c, _, _ = book("soa")
    cache, table, lens = batch(rng, [2048 + 5] * 4, 1, "soa", 128)
    codes = SO.pack(rng.integers(0, 16, 128), 4)
    cache[:, :, :, :] = 0
    flat = cache.reshape(len(cache), -1)
    for t in range(16):
        ka, va, _, _, _ = SO.places("soa", 1, t, 0)
        flat[:, ka:ka + 64] = codes
        flat[:, va:va + 64] = rng.integers(0, 256, (len(cache), 64))
        for page in range(len(cache)):
            put_half(cache, "soa", page, t, 2, 2.5 + 0.05 * rng.standard_normal())
            put_half(cache, "soa", page, t, 3, 20.0)
            put_half(cache, "soa", page, t, 4, 100.0)
    put_half(cache, "soa", table[0, 0], 0, 2, 22.5)
    put_half(cache, "soa", table[0, 0], 0, 3, 0.0)
    put_half(cache, "soa", table[0, 0], 0, 4, 0.0)
    d = npy(c)[SO.unpack(codes, 4)].astype(np.float64)
    q = np.broadcast_to(d / (d @ d) * (26 * np.log(2) / 20 * np.sqrt(128)), (4, 4, 128)).astype(np.float32)
    got = tqb.prefix_attention(torch.from_numpy(q.copy()).cuda(), torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(),
                               torch.from_numpy(lens).cuda(), None, cuda(c), prefix_len=2048, out_dtype=torch.bfloat16)
    ref, _, size = SO.attention(q, cache, "soa", table, lens, npy(c), lambda t, L: t >= 0)
    assert (np.abs(npy(got) - ref) <= half_step(got.dtype) * np.abs(ref) + 0.06 * size).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.7, 1.5, 2.5, 5.0])
def test_prefix_error_against_the_outputs_own_rounding(monkeypatch, dtype, spread):
    """The rms error of a batch behind a prefix, relative to the outputs' rms.

    An output rounded once is off by at most half a step, 2^-11 (fp16) or 2^-8 (bf16) of it, spread evenly: rms 1 / sqrt(3)
    of that.  fp16 outputs have no more than 1.2 times that.  bf16 ones add the shared pass: a score of standard deviation
    u carries three roundings (q, c and c norm to fp16) of rms 2^-11 / sqrt(3) at most each, so 2^-11 u, which its weight
    and with it the output follows; V and P one each, 2^-11 sqrt(2 / 3) together."""
    share(monkeypatch)
    rng = np.random.default_rng(int(10 * spread))
    c, _, R = book("soa")
    cache, table, lens = batch(rng, [1024 + n for n in (1, 9, 40, 17)], 2, "soa", 64)
    q = torch.from_numpy((spread * rng.standard_normal((4, 8, 128))).astype(np.float32)).to(dtype).cuda()
    got = tqb.prefix_attention(q, torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(),
                               cuda(R), cuda(c), prefix_len=1024)
    ref, _, _ = SO.attention(npy(q).astype(np.float64) @ npy(R).astype(np.float64), cache, "soa", table, lens, npy(c),
                             lambda t, L: t >= 0)
    error = np.sqrt(((got.double().cpu().numpy() - ref) ** 2).mean() / (ref ** 2).mean())
    own = half_step(dtype) / np.sqrt(3)
    assert error <= (1.2 * own if dtype == torch.float16 else np.sqrt(own ** 2 + 2.0 ** -22 * (spread ** 2 + 2 / 3)))


def run_append(key, R, mids, cents, layout="soa", **kw):
    """Bytes of an append of ``key`` (float32 [n, hk, 128]) without rotary positions, and the definition's."""
    rng = np.random.default_rng(len(key))
    n, hk, _ = key.shape
    cache0 = rng.integers(0, 256, (n // 16 + 1, 16, hk, SO.LAYOUTS[layout][2]), dtype=np.uint8)
    slots = rng.permutation(n).astype(np.int32)
    value = rng.standard_normal(key.shape).astype(np.float32)
    cache = torch.from_numpy(cache0).cuda()
    tqb.rope_append(torch.from_numpy(key).cuda(), torch.from_numpy(value).cuda(), cache, torch.from_numpy(slots).cuda(), None,
                    None, cuda(R), cuda(mids), cuda(cents), layout=layout, **kw)
    return cache.cpu().numpy(), SO.append(cache0, layout, key, value, slots, None, None, npy(R), npy(mids), npy(cents))


@pytest.mark.parametrize("n", [300, 2600])
def test_append_norm_of_codes_of_very_different_size(n):
    """Rows along a column of R: one code of size 1 and 127 whose square, 5.9e-8, is less than half a unit of the sum's last
    place.  The norms are spread, so that some lie next to a border between two fp16 numbers."""
    _, _, R = book("soa")
    cents = torch.tensor([-0.9, -0.8, -0.7, -0.6, -0.5, -0.4, -0.3, -0.2, 2.43e-4, 0.3, 0.4, 0.5, 0.6, 0.7, 0.8, 1.0])
    rng = np.random.default_rng(n)
    key = (npy(R)[:, 0] * rng.uniform(1, 64, (n, 4, 1))).astype(np.float32)
    got, want = run_append(key, R, tqb.get_midpoints(cents), cents)
    assert np.array_equal(got, want), f"{(got != want).sum()} bytes differ"


@pytest.mark.parametrize("n", [20, 2100])
@pytest.mark.parametrize("layout", ["soa", "aos_k3"])
def test_append_borders_closer_than_fp32_can_tell(n, layout):
    """Neighbouring fp32 numbers as borders, and keys whose coordinates all lie among them."""
    _, _, R = book(layout)
    at = np.float32(1 / np.sqrt(128))
    close = [at]
    for _ in range(3):
        close = [np.nextafter(close[0], np.float32(0)), *close, np.nextafter(close[-1], np.float32(1))]
    rest = [-0.2, -0.1, -0.05, 0.02, 0.12, 0.15, 0.18, 0.2] if layout == "soa" else []
    mids = torch.from_numpy(np.sort(np.array([*close, *rest], np.float32)))
    cents = torch.linspace(-0.2, 0.2, len(mids) + 1)
    t = np.full((n, 4, 128), 1.0) * np.random.default_rng(n).uniform(0.5, 2, (n, 4, 1))
    key = (t @ npy(R).astype(np.float64).T).astype(np.float32)
    got, want = run_append(key, R, mids, cents, layout)
    assert np.array_equal(got, want), f"{(got != want).sum()} bytes differ"


@pytest.mark.parametrize("n", [40, 2600])
@pytest.mark.parametrize("layout", ["soa", "aos", "soa_k3"])
@pytest.mark.parametrize("border", ["at zero", "beside zero", "none near"])
def test_append_rows_of_zeros(n, layout, border):
    """Zeros of both signs, rows of one tiny number (their squares vanish, the sides of zero do not), among ordinary ones."""
    c, m, R = book(layout)
    if border != "at zero":
        c = c + (1e-9 if border == "beside zero" else 0.01)
        m = tqb.get_midpoints(c)
    rng = np.random.default_rng(n)
    key = rng.standard_normal((n, 3, 128)).astype(np.float32)
    key[rng.random((n, 3)) < 0.3] = 0.0
    key[rng.random((n, 3)) < 0.1] = -0.0
    tiny = rng.random((n, 3)) < 0.02
    key[tiny] = 0.0
    key[tiny, rng.integers(0, 128)] = rng.choice(np.array([1e-45, -1e-45, 3e-39, -1e-30, 1e-22], np.float32), tiny.sum())
    got, want = run_append(key, R, m, c, layout)
    assert np.array_equal(got, want), f"{(got != want).sum()} bytes differ"


@pytest.mark.parametrize("n", [64, 2048])
def test_append_of_zeros_takes_no_longer(n):
    """Dummy inputs: at most three times as long as random ones (a hundredfold where each coordinate takes 64 bits)."""
    c, m, R = (cuda(x) for x in book("soa"))
    cache = torch.zeros(n // 16, 16, 8, 134, dtype=torch.uint8, device="cuda")
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    value = torch.randn(n, 8, 128, device="cuda")
    took = []
    for key in (torch.randn_like(value), torch.zeros_like(value)):
        best = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            tqb.rope_append(key, value, cache, slots, None, None, R, m, c)
            a.record()
            for _ in range(10):
                tqb.rope_append(key, value, cache, slots, None, None, R, m, c)
            b.record()
            b.synchronize()
            best.append(a.elapsed_time(b))
        took.append(min(best))
    assert took[1] <= 3 * took[0], took
