"""Serving operators where numbers, sizes or alignment are at their ends, against float64 forms."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import serving_oracle as SO
import tqb
from test_serving_gpu import batch, book, cos_sin_table, cuda, half_step, no_wait_timeouts, npy, run_prefix  # noqa: F401

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


@pytest.mark.parametrize("n", [20, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_append_queries_of_any_size(n, dtype):
    """Rows whose squares leave fp32's range, beside ordinary ones and rows of zeros: 2^-17 |q|, as for every query."""
    c, m, R = book("soa")
    rng = np.random.default_rng(n)
    q = rng.standard_normal((n, 8, 128)) * np.exp2(rng.choice([-110, -80, -62, -55, 0, 0, 0, 55, 62, 63, 64, 80, 110], (n, 8, 1)))
    q[rng.random((n, 8)) < 0.1] = 0
    q = torch.from_numpy(q.astype(np.float32)).to(dtype).cuda()
    k = torch.from_numpy(rng.standard_normal((n, 4, 128)).astype(np.float32)).to(dtype).cuda()
    cache = torch.zeros(n // 16 + 1, 16, 4, 134, dtype=torch.uint8, device="cuda")
    cs, pos = cos_sin_table(500, 64), rng.integers(0, 500, n)
    got = tqb.rope_append(k, k, cache, torch.arange(n, dtype=torch.int32, device="cuda"), torch.from_numpy(pos).cuda(),
                          torch.from_numpy(cs).cuda(), cuda(R), cuda(m), cuda(c), query=q)
    x = SO.rope(npy(q).astype(np.float64), cs[pos], False)
    off = np.abs(got.double().cpu().numpy() - x @ npy(R).astype(np.float64))
    assert (off <= 2.0 ** -17 * np.linalg.norm(x, axis=-1, keepdims=True)).all()


def test_append_keys_beyond_fp32_write_the_same_in_both_forms():
    """|x|^2 above fp32's range, infinities and NaN: a norm of inf or NaN and codes of 0, however many rows there are."""
    c, m, R = (cuda(x) for x in book("soa"))
    rng = np.random.default_rng(5)
    n = 1700
    key = rng.standard_normal((n, 4, 128)).astype(np.float32)
    bad = rng.random((n, 4)) < 0.2
    key[bad] *= np.float32(2.0 ** 80)
    key[rng.random(key.shape) < 1e-4] = np.inf
    key[rng.random(key.shape) < 1e-4] = np.nan
    key = torch.from_numpy(key).cuda()
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    caches = [torch.zeros(n // 16 + 1, 16, 4, 134, dtype=torch.uint8, device="cuda") for _ in range(2)]
    value = torch.randn(n, 4, 128, device="cuda")
    tqb.rope_append(key, value, caches[0], slots, None, None, R, m, c)
    for i in range(0, n, 100):
        tqb.rope_append(key[i:i + 100], value[i:i + 100], caches[1], slots[i:i + 100], None, None, R, m, c)
    assert torch.equal(*caches)
    flat = caches[0].cpu().numpy().reshape(len(caches[0]), -1)
    for t, h in zip(*np.nonzero(bad)):
        ka, _, norm, _, _ = SO.places("soa", 4, t % 16, h)
        assert not np.isfinite(flat[t // 16, norm:norm + 2].view(np.float16)[0]) and (flat[t // 16, ka:ka + 64] == 0).all()


@pytest.mark.parametrize("rows,chunks", [(4, 4), (160, 2)])
def test_prefix_partials_of_empty_sequences(monkeypatch, rows, chunks):
    """Lengths of 0 and below: every split of the prefix is written with O 0 and an LSE of -inf."""
    share(monkeypatch, chunks)
    rng = np.random.default_rng(31)
    c, _, _ = book("soa")
    cache, table, lens = batch(rng, [512 + 3] * (rows // 4), 1, "soa", 32)
    lens[:] = rng.choice([0, -1, -2 ** 31, -2 ** 31 + 200], len(lens))
    lens[0] = -2 ** 31
    q = torch.from_numpy(rng.standard_normal((rows // 4, 4, 128)).astype(np.float32)).cuda()
    mid = torch.full((rows // 4, 4, chunks + 1, 129), 7.0, device="cuda")
    out = tqb.prefix_attention(q, torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(),
                               None, cuda(c), prefix_len=512, out_dtype=torch.bfloat16, mid_o=mid, num_splits=1)
    assert torch.isnan(out).all()
    assert (mid[:, :, :chunks, :128] == 0).all() and torch.isneginf(mid[:, :, :chunks, 128]).all()


@pytest.mark.parametrize("layout", ["soa", "soa_k8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_queries_of_any_alignment(layout, dtype):
    """Contiguous queries that begin one element into a buffer, in the cache's basis: the numbers of an aligned copy."""
    rng = np.random.default_rng(41)
    c, _, _ = book(layout)
    cache, table, lens = (torch.from_numpy(x).cuda() for x in batch(rng, [200, 77, 150], 2, layout, 4))
    q = torch.randn(1 + 3 * 8 * 128, device="cuda").to(dtype)[1:].view(3, 8, 128)
    for query in (q, q.transpose(0, 1).contiguous().transpose(0, 1), q[..., :].expand(3, 8, 128)):
        for call in (lambda x: tqb.window_attention(x, cache, table, lens, None, cuda(c), window=64, layout=layout),
                     lambda x: tqb.prefix_attention(x, cache, table, lens, None, cuda(c), prefix_len=64, layout=layout)):
            assert torch.equal(call(query), call(query.clone()))


@pytest.mark.parametrize("scale", [0.0, -1.0, float("nan"), float("inf"), 1e39, 10 ** 400, "x"])
def test_scales_that_are_refused(scale):
    rng = np.random.default_rng(1)
    c, _, _ = book("soa")
    cache, table, lens = (torch.from_numpy(x).cuda() for x in batch(rng, [40], 1, "soa", 1))
    q = torch.zeros(1, 4, 128, device="cuda")
    for call in (lambda: tqb.window_attention(q, cache, table, lens, None, cuda(c), window=9, scale=scale),
                 lambda: tqb.prefix_attention(q, cache, table, lens, None, cuda(c), prefix_len=16, scale=scale)):
        with pytest.raises(tqb.TqbError, match="scale"):
            call()


@pytest.mark.parametrize("layout", sorted(SO.LAYOUTS))
@pytest.mark.parametrize("hq", [4, 8])
def test_window_values_that_cancel(layout, hq):
    """Every value is the middle code times its scale less as much, 0 exactly, whatever the scales: errors go by the mean
    |v|, so the output is 0."""
    rng = np.random.default_rng(hq)
    c, _, _ = book(layout)
    kb, vb, _ = SO.LAYOUTS[layout]
    cache, table, lens = batch(rng, [300, 41, 17], 1, layout)
    middle = SO.pack(np.full(128, 1 << (vb - 1)), vb)
    flat = cache.reshape(len(cache), -1)
    for t in range(16):
        va = SO.places(layout, 1, t, 0)[1]
        flat[:, va:va + len(middle)] = middle
        for page in range(len(cache)):
            scale = np.float16(0.3 * np.exp(0.2 * rng.standard_normal()))
            put_half(cache, layout, page, t, 3, scale)
            put_half(cache, layout, page, t, 4, -scale * np.float16(1 << (vb - 1)))
    q = torch.from_numpy(1.5 * rng.standard_normal((3, hq, 128)).astype(np.float32)).cuda()
    got = tqb.window_attention(q, torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(),
                               None, cuda(c), window=200, layout=layout)
    assert (got == 0).all()


@pytest.mark.parametrize("layout", ["soa", "soa_k3v3", "aos_k8"])
@pytest.mark.parametrize("above", [20, 30])
@pytest.mark.parametrize("kernel", ["ring", "regs"])
def test_window_behind_a_first_token_that_outweighs_it(monkeypatch, layout, above, kernel):
    """A first token of value 0 with 2^above times the weight of each of the others: the output is theirs.  The bar is the
    decode calls' 2e-3, of the mean |v| here."""
    if kernel == "regs":
        monkeypatch.setenv("TQB_STAGE1_KERNEL", "regs")
    rng = np.random.default_rng(above)
    c, _, _ = book(layout)
    kb, vb, _ = SO.LAYOUTS[layout]
    cache, table, lens = batch(rng, [500, 260], 1, layout)
    flat = cache.reshape(len(cache), -1)
    if kb == 8:
        d = rng.standard_normal(128)
        raw = torch.from_numpy(d.astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
        d = SO.f8(raw)
        grow = 8  # exact in e4m3: three exponents up
        big = torch.from_numpy((d * grow).astype(np.float32)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    else:
        raw = big = SO.pack(rng.integers(0, 1 << kb, 128), kb)
        d = npy(c)[SO.unpack(raw, kb)].astype(np.float64)
        grow = 8
    for t in range(16):
        ka = SO.places(layout, 1, t, 0)[0]
        flat[:, ka:ka + len(raw)] = raw
        for page in range(len(cache)):
            if kb != 8:
                put_half(cache, layout, page, t, 2, 3.0)
    for row in table:
        ka = SO.places(layout, 1, 0, 0)[0]
        flat[row[0], ka:ka + len(big)] = big
        if kb != 8:
            put_half(cache, layout, row[0], 0, 2, 3.0 * grow)
        put_half(cache, layout, row[0], 0, 3, 0.0)
        put_half(cache, layout, row[0], 0, 4, 0.0)
    size = (1.0 if kb == 8 else 3.0) * (d @ d)
    if layout.startswith("aos") and kb != 8:
        size /= np.sqrt(d @ d)
    q = np.broadcast_to(d * (above * np.log(2) * np.sqrt(128) / (size * (grow - 1))), (2, 4, 128)).astype(np.float32)
    args = (torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(), None, cuda(c))
    for dtype in (torch.float32, torch.bfloat16):
        got = tqb.window_attention(torch.from_numpy(q.copy()).cuda(), *args, window=200, first_tokens=1, layout=layout,
                                   out_dtype=dtype, num_splits=1)
        ref, _, mean = SO.attention(q, cache, layout, table, lens, npy(c), lambda t, L: (t < 1) | (t >= L - 200))
        assert (np.abs(got.double().cpu().numpy() - ref) <= half_step(dtype) * np.abs(ref) + 2e-3 * mean).all()


@pytest.mark.parametrize("layout", sorted(SO.LAYOUTS))
@pytest.mark.parametrize("kernel", ["ring", "regs"])
def test_window_values_of_any_size(monkeypatch, layout, kernel):
    """Scales and zeros times 2^-8, exactly: outputs times 2^-8.  Both are fp32 sums of the same products, of weights good to
    2^-22: 2^-20 of the mean |v|, 2 here."""
    if kernel == "regs":
        monkeypatch.setenv("TQB_STAGE1_KERNEL", "regs")
    rng = np.random.default_rng(3)
    c, _, _ = book(layout)
    cache, table, lens = batch(rng, [300, 41, 999], 1, layout)
    q = torch.from_numpy(1.5 * rng.standard_normal((3, 5, 128)).astype(np.float32)).cuda()
    outs = []
    for f in (1.0, 2.0 ** -8):
        now = cache.copy()
        flat = now.reshape(len(now), -1)
        for t in range(16):
            for at in SO.places(layout, 1, t, 0)[3:]:
                flat[:, at:at + 2] = (np.ascontiguousarray(flat[:, at:at + 2]).view(np.float16) * np.float16(f)).view(np.uint8)
        out = tqb.window_attention(q, torch.from_numpy(now).cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda(),
                                   None, cuda(c), window=400, layout=layout)
        outs.append(out.double() / f)
    assert (outs[0] - outs[1]).abs().max().item() <= 2.0 ** -20 * 2


@pytest.mark.parametrize("layout", sorted(SO.LAYOUTS))
@pytest.mark.parametrize("own,hq,chunks", [([1, 9, 30] * 12, 8, 1), ([4, 60], 16, 2)])
def test_prefix_pass_of_many_tiles_on_every_layout(layout, own, hq, chunks):
    """bf16 outputs, one stream over every tile and two over every other one."""
    run_prefix(layout, torch.bfloat16, own, 720, hq, 2, seed=chunks, chunks=chunks)
