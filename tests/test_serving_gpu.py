"""Append, gather, windowed and shared-prefix decode on the GPU against their float64 forms.

Bars, derived before the first run.  Bytes of an append: equal (the codes are those of exact arithmetic, the values'
steps are the store's).  Rotated queries: 128 fp32 products, each partial sum off by at most 2^-24 of |x| (Cauchy-Schwarz
on a unit column), 2^-17 |x| in all.  Gather: the output type's half step, and 2^-20 for the fp32 product (AoS: the fp32
length of the centroids).  Decode: the repository's 1e-4 + 2e-3 |ref|, and the output type's half step.

The shared pass over a prefix (16-bit outputs) rounds its operands to fp16, 2^-11 at most each, so its errors go by the
mean A = sum p |v| of what is summed and not by |ref|, which may cancel.  V and P: 2 * 2^-11 A.  Scores: q_i k_i carries
three roundings (q, c, c norm) of rms at most 2^-11 / sqrt(3), 2^-11 together; over 128 products that is sigma = 2^-11
scale sqrt(sum q_i^2 k_i^2) = 2^-11 * 1.5 = 7.3e-4 for the rows here (|q| = 1.5 sqrt(128), |k| = sqrt(128)), and a score's
error moves the output by at most that times A; 4 sigma A = 3e-3 A.  Together 4e-3 A in place of 2e-3 |ref|; for rows of
another size, |q| = u sqrt(128), (2^-10 + 4 * 2^-11 u) A.  That takes the roundings for independent, which the codebook's
are not: a token has 16 different ones (8 of a symmetric codebook), so sum q_i k_i d(c_i) has the mean s * d, |d| <= 2^-11,
besides its spread.  Scores far above a row's 4 sigma need that term, 2^-11 |s| A with |s| at most the row's LSE."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import serving_oracle as SO
import tqb
from tqb import _lib

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def no_wait_timeouts(cuda_device):
    tqb.wait_timeouts(reset=True)
    yield
    torch.cuda.synchronize()
    assert tqb.wait_timeouts(reset=True) == 0, "a bounded device wait gave up"


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def book(layout):
    kb = SO.LAYOUTS[layout][0]
    if kb == 8:
        return None, None, None
    c = tqb.get_centroids(128, kb)
    R = np.linalg.qr(np.random.default_rng(7).standard_normal((128, 128)))[0].astype(np.float32)
    return c, tqb.get_midpoints(c), torch.from_numpy(R)


def cuda(x):
    return None if x is None else x.cuda()


def npy(x):
    return None if x is None else x.detach().float().cpu().numpy()


def cos_sin_table(n, r):
    a = np.arange(n)[:, None] * 10000.0 ** (-np.arange(0, r, 2) / r)
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def projections(rng, n, hq, hk, dtype, pad=0):
    """Query, key and value as slices of one [n, heads * 128 (+ pad)] projection."""
    x = torch.from_numpy(rng.standard_normal((n, (hq + 2 * hk) * 128 + pad)).astype(np.float32)).to(dtype).cuda()
    part = lambda a, b: x[:, a * 128:b * 128].unflatten(-1, (b - a, 128))  # noqa: E731
    return part(0, hq), part(hq, hq + hk), part(hq + hk, hq + 2 * hk)


def run_append(layout, dtype, n, hq, hk, rotary, interleaved, *, seed=0, pad=0, pos64=True, pad_slots=0, norm_correction=True,
               scale=1.0, codes=None, poison=False):
    rng = np.random.default_rng(seed)
    c, m, R = book(layout)
    if codes is not None:
        c, m = codes, tqb.get_midpoints(codes)
    nb = -(-n // 16) + 2
    cache0 = rng.integers(0, 256, (nb, 16, hk, SO.LAYOUTS[layout][2]), dtype=np.uint8)
    slots = rng.permutation(nb * 16)[:n].astype(np.int32)
    slots[rng.permutation(n)[:pad_slots]] = -1
    q, k, v = projections(rng, n, hq, hk, dtype, pad)
    if scale != 1.0:
        k, v = k * scale, v * scale
    if poison:  # what has no place may hold anything
        for x, bad in ((q, np.nan), (k, np.nan), (v, np.inf)):
            x[torch.from_numpy(np.flatnonzero(slots < 0)).cuda()] = bad
    table = cos_sin_table(500, rotary) if rotary else None
    pos = rng.integers(0, 500, n) if rotary else None
    cache = torch.from_numpy(cache0).cuda()
    got_q = tqb.rope_append(
        k, v, cache, torch.from_numpy(slots).cuda(),
        None if pos is None else torch.from_numpy(pos.astype(np.int64 if pos64 else np.int32)).cuda(),
        None if table is None else torch.from_numpy(table).cuda(), cuda(R), cuda(m), cuda(c), layout=layout,
        interleaved=interleaved, query=q if hq else None, norm_correction=norm_correction)
    want = SO.append(cache0, layout, npy(k), npy(v), slots, pos, table, npy(R), npy(m), npy(c), interleaved=interleaved,
                     norm_correction=norm_correction)
    got = cache.cpu().numpy()
    assert np.array_equal(got, want), f"{(got != want).sum()} of {got.size} bytes differ"
    if hq:
        x = npy(q).astype(np.float64)
        if rotary:
            x = SO.rope(x, table[pos], interleaved)
        ref = x if R is None else x @ npy(R).astype(np.float64)
        tol = (2.0 ** -17 if R is not None else 2.0 ** -24) * np.linalg.norm(x, axis=-1, keepdims=True)
        live = np.flatnonzero(slots >= 0) if poison else slice(None)
        assert (np.abs(npy(got_q) - ref) <= tol)[live].all()


@pytest.mark.parametrize("layout", sorted(SO.LAYOUTS))
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_append_writes_the_definitions_bytes(layout, dtype):
    run_append(layout, DT[dtype], 45, 8, 2, 128, False, seed=1, pad_slots=4)


@pytest.mark.parametrize("n,hq,hk,rotary,interleaved,pad,pos64", [
    (1, 32, 8, 128, False, 0, True), (1, 1, 1, 64, True, 0, False), (17, 0, 8, 96, False, 8, True),
    (129, 5, 1, 2, True, 3, True), (300, 16, 2, 34, False, 1, False), (64, 4, 4, 0, False, 0, True),
    (200, 24, 3, 126, False, 0, True), (520, 8, 8, 128, True, 0, True)])
def test_append_shapes(n, hq, hk, rotary, interleaved, pad, pos64):
    """Single tokens, odd heads, partial rotary dims of every alignment, no rotary step, odd row strides."""
    for layout in ("soa", "aos_k3v3", "soa_k8"):
        run_append(layout, torch.bfloat16, n, hq, hk, rotary, interleaved, seed=n, pad=pad, pos64=pos64)


@pytest.mark.parametrize("scale", [0.0, 1e-6, 3000.0])
def test_append_extreme_norms(scale):
    """All-zero keys sit on the codebook's middle border; large norms near the end of fp16."""
    run_append("soa", torch.float32, 37, 0, 2, 64, False, seed=3, scale=scale)
    run_append("aos_k3", torch.float32, 37, 0, 2, 64, False, seed=3, scale=scale)


def test_append_without_norm_correction():
    run_append("soa_k3", torch.bfloat16, 33, 0, 2, 128, False, seed=4, norm_correction=False)


def test_append_large_batch_bytes():
    """Enough coordinates (2 M) that some lie next to every border."""
    run_append("soa", torch.bfloat16, 2048, 0, 8, 128, False, seed=5)


def test_append_skips_what_has_no_place():
    """Out-of-range slots and positions: nothing stored, and NaN queries for the positions."""
    rng = np.random.default_rng(9)
    c, m, R = book("soa")
    cache = torch.from_numpy(rng.integers(0, 256, (3, 16, 2, 134), dtype=np.uint8)).cuda()
    before = cache.clone()
    q, k, v = projections(rng, 4, 4, 2, torch.bfloat16)
    out = tqb.rope_append(k, v, cache, torch.tensor([48, -7, 5, 6], dtype=torch.int32).cuda(),
                          torch.tensor([1, 2, 500, -1]).cuda(), torch.from_numpy(cos_sin_table(500, 128)).cuda(), cuda(R),
                          cuda(m), cuda(c), query=q)
    assert torch.equal(cache, before)
    assert torch.isfinite(out[:2]).all() and torch.isnan(out[2:]).all()


# Thousands of rows, queries and keys together, that are aligned to four elements take the tensor-core form.
LLOYD_MAX = [x for x in sorted(SO.LAYOUTS) if not x.endswith("k8")]


@pytest.mark.parametrize("layout", LLOYD_MAX)
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_append_many_rows(layout, dtype):
    run_append(layout, DT[dtype], 613, 12, 3, 128, False, seed=6, pad_slots=40, poison=True)


@pytest.mark.parametrize("n,hq,hk,rotary,interleaved,pad,pos64", [
    (8193, 0, 1, 128, True, 0, True), (2100, 0, 4, 64, True, 8, False), (1201, 5, 3, 96, False, 0, True),
    (1100, 16, 2, 2, True, 0, False), (700, 12, 4, 34, False, 0, True), (1030, 8, 1, 0, False, 0, True),
    (1100, 6, 2, 64, False, 3, True), (9000, 1, 1, 126, True, 0, True)])
def test_append_many_rows_shapes(n, hq, hk, rotary, interleaved, pad, pos64):
    """Few and many heads, partial and unaligned rotary dims, the last tile's ends, and rows that are not aligned."""
    run_append("soa_k3", torch.bfloat16, n, hq, hk, rotary, interleaved, seed=n, pad=pad, pos64=pos64)


@pytest.mark.parametrize("scale", [0.0, 1e-6, 3000.0])
def test_append_many_rows_of_extreme_norms(scale):
    run_append("soa", torch.float32, 2100, 0, 4, 64, False, seed=3, scale=scale)


@pytest.mark.parametrize("n", [40, 2100])
def test_append_codebooks_of_any_spacing(n):
    """Borders next to one another, equal ones and one far out, beside ordinary ones; no norm correction."""
    codes = torch.tensor([-9.0, -0.2, -0.2, -0.1, -1e-3, -1e-4, -1e-5, 0, 1e-7, 1e-6, 2e-6, 0.05, 0.05003, 0.1, 0.3, 0.31])
    run_append("soa", torch.bfloat16, n, 0, 4, 128, False, seed=n, codes=codes)
    run_append("soa", torch.float32, n, 0, 4, 128, False, seed=n, codes=codes, norm_correction=False)


@pytest.mark.parametrize("n", [17, 2100])
def test_append_poisoned_rows(n):
    for layout in ("aos", "soa_k8"):
        run_append(layout, torch.bfloat16, n, 4, 4, 128, True, seed=n, pad_slots=n // 3, poison=True)


def test_append_many_rows_without_a_place():
    """Half the tokens without a slot or a position, spread over every tile."""
    rng = np.random.default_rng(10)
    c, m, R = book("soa")
    n = 3000
    cache0 = rng.integers(0, 256, (n // 16 + 1, 16, 2, 134), dtype=np.uint8)
    slots = rng.permutation(n).astype(np.int32)
    slots[::5] = rng.choice([-1, -2 ** 31, len(cache0) * 16, 2 ** 31 - 1], len(slots[::5]))
    pos = rng.integers(0, 500, n)
    pos[::3] = rng.choice([-1, 500, 2 ** 40, -2 ** 40], len(pos[::3]))
    cs = cos_sin_table(500, 128)
    q, k, v = projections(rng, n, 2, 2, torch.bfloat16)
    cache = torch.from_numpy(cache0).cuda()
    out = tqb.rope_append(k, v, cache, torch.from_numpy(slots).cuda(), torch.from_numpy(pos).cuda(),
                          torch.from_numpy(cs).cuda(), cuda(R), cuda(m), cuda(c), query=q)
    want = SO.append(cache0, "soa", npy(k), npy(v), slots, pos, cs, npy(R), npy(m), npy(c))
    assert np.array_equal(cache.cpu().numpy(), want)
    assert np.array_equal(np.isnan(npy(out)).all((1, 2)), (pos < 0) | (pos >= 500))
    assert np.array_equal(np.isnan(npy(out)).any((1, 2)), (pos < 0) | (pos >= 500))


def test_append_empty():
    c, m, R = book("soa")
    cache = torch.zeros(2, 16, 2, 134, dtype=torch.uint8, device="cuda")
    e = torch.empty(0, 2, 128, device="cuda")
    out = tqb.rope_append(e, e, cache, torch.empty(0, dtype=torch.int32, device="cuda"), None, None, cuda(R), cuda(m),
                          cuda(c), query=e)
    assert out.shape == (0, 2, 128)


@pytest.mark.parametrize("layout", sorted(SO.LAYOUTS))
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,hk", [(1, 1), (53, 3), (131, 8)])
def test_gather(layout, dtype, n, hk):
    rng = np.random.default_rng(n)
    c, _, _ = book(layout)
    cache = random_cache(rng, 12, hk, layout)
    slots = rng.integers(0, 12 * 16, n).astype(np.int32)  # repeated slots may be read
    slots[n // 2:n // 2 + 1] = rng.choice([-1, 12 * 16, slots[0]])
    k, v = tqb.gather_kv(torch.from_numpy(cache).cuda(), torch.from_numpy(slots).cuda(), cuda(c), layout=layout,
                         dtype=DT[dtype])
    assert k.dtype == DT[dtype]
    rk, rv = SO.read(cache, layout, slots, npy(c))
    tol = half_step(DT[dtype]) + 2.0 ** -20
    for got, ref in ((k, rk), (v, rv)):
        assert (np.abs(got.double().cpu().numpy() - ref) <= tol * np.abs(ref) + 2.0 ** -25).all()


def test_gather_into_strided_outputs():
    rng = np.random.default_rng(2)
    c, _, _ = book("soa")
    cache = torch.from_numpy(random_cache(rng, 4, 2, "soa")).cuda()
    slots = torch.arange(40, dtype=torch.int32, device="cuda")
    k, v = tqb.gather_kv(cache, slots, cuda(c))
    buf = torch.zeros(40, 2, 2 * 128 + 3, dtype=torch.bfloat16, device="cuda")
    tqb.gather_kv(cache, slots, cuda(c), key=buf[..., :128], value=buf[..., 129:257])
    assert torch.equal(buf[..., :128], k) and torch.equal(buf[..., 129:257], v)
    assert (buf[..., 128] == 0).all() and (buf[..., 257:] == 0).all()


def random_cache(rng, nb, hk, layout):
    """Every byte a valid code, norms, scales and zeros of ordinary size."""
    kb, vb, slot = SO.LAYOUTS[layout]
    cache = rng.integers(0, 256, (nb, 16, hk, slot), dtype=np.uint8)
    flat = cache.reshape(nb, -1)
    for t in range(16):
        for h in range(hk):
            ka, va, norm, scale, zero = SO.places(layout, hk, t, h)
            if kb == 8:
                e = torch.from_numpy(rng.standard_normal((nb, 128)).astype(np.float32)).to(torch.float8_e4m3fn)
                flat[:, ka:ka + 128] = e.view(torch.uint8).numpy()
            put = lambda at, v: flat.__setitem__((slice(None), slice(at, at + 2)),  # noqa: E731
                                                 v.astype(np.float16)[:, None].view(np.uint8))
            if norm is not None:
                put(norm, 11.3 * np.exp(0.2 * rng.standard_normal(nb)))
            put(scale, 0.3 * np.exp(0.2 * rng.standard_normal(nb)))
            put(zero, -2 + 0.3 * rng.standard_normal(nb))
    return cache


def batch(rng, lens, hk, layout, shared=0):
    """Cache, block table and lengths; the first ``shared`` pages are everyone's."""
    pages = [max(0, -(-n // 16) - shared) for n in lens]
    nb = shared + sum(pages) + 2
    order = rng.permutation(nb).astype(np.int32)
    table = np.zeros((len(lens), max(1, shared + max(pages))), np.int32)
    table[:, :shared] = order[:shared]
    at = shared
    for b, n in enumerate(pages):
        table[b, shared:shared + n] = order[at:at + n]
        at += n
    return random_cache(rng, nb, hk, layout), table, np.asarray(lens, np.int32)


def check_decode(got, lse, ref, ref_lse, dtype, size=None, rel=4e-3):
    """``size``: the mean |v| that the shared pass's bar goes by."""
    got, lse = got.double().cpu().numpy(), lse.double().cpu().numpy()
    dead = np.isnan(ref)
    assert np.array_equal(np.isnan(got), dead)
    bar = 1e-4 + half_step(dtype) * np.abs(ref) + (2e-3 * np.abs(ref) if size is None else rel * size)
    assert (np.abs(got - ref)[~dead] <= bar[~dead]).all()
    assert np.array_equal(np.isneginf(lse), np.isneginf(ref_lse))
    live = np.isfinite(ref_lse)
    assert (np.abs(lse[live] - ref_lse[live]) <= 1e-4 + 2e-3 * np.abs(ref_lse[live])).all()


def run_window(layout, dtype, lens, hq, hk, window, first, *, seed=0, sinks=False, raw=True, **kw):
    rng = np.random.default_rng(seed)
    c, _, R = book(layout)
    cache, table, lens = batch(rng, lens, hk, layout)
    q = torch.from_numpy(rng.standard_normal((len(lens), hq, 128)).astype(np.float32) * 1.5).to(dtype).cuda()
    raw = raw and R is not None
    s = torch.from_numpy(rng.standard_normal(hq).astype(np.float32) * 2).cuda() if sinks else None
    lse = torch.empty(len(lens), hq, device="cuda")
    got = tqb.window_attention(q, torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(),
                               torch.from_numpy(lens).cuda(), cuda(R) if raw else None, cuda(c), window=window,
                               first_tokens=first, layout=layout, sinks=s, lse=lse, **kw)
    x = npy(q).astype(np.float64)
    x = x @ npy(R).astype(np.float64) if raw else x
    ref, ref_lse, _ = SO.attention(x, cache, layout, table, lens, npy(c), lambda t, L: (t < first) | (t >= L - window),
                                scale=kw.get("scale"), sinks=npy(s))
    assert got.dtype == kw.get("out_dtype", dtype)
    check_decode(got, lse, ref, ref_lse, got.dtype)


RAGGED = [1, 0, 15, 16, 17, 40, 99, 100, 101, 104, 105, 160, 333]


@pytest.mark.parametrize("layout", sorted(SO.LAYOUTS))
@pytest.mark.parametrize("window,first", [(100, 4), (37, 0), (1, 1)])
def test_window_layouts(layout, window, first):
    run_window(layout, torch.bfloat16, RAGGED, 8, 2, window, first, seed=window)


@pytest.mark.parametrize("hq,hk", [(32, 8), (64, 8), (5, 1), (6, 3), (10, 10), (40, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_window_heads_and_types(hq, hk, dtype):
    run_window("soa", DT[dtype], [1, 70, 200, 129], hq, hk, 64, 17, seed=hq, sinks=True)


@pytest.mark.parametrize("window,first,num_splits", [(1, 0, 1), (1, 0, 7), (16, 16, 3), (333, 0, 5), (1000, 50, 2),
                                                     (5, 400, 4), (320, 13, 64), (2 ** 30, 2 ** 30, None)])
def test_window_splits(window, first, num_splits):
    """More splits than tokens, windows and first tokens beyond the sequence, first tokens that meet the window."""
    run_window("soa", torch.float32, RAGGED, 4, 1, window, first, seed=1, num_splits=num_splits, sinks=True)


def test_window_register_kernel(monkeypatch):
    monkeypatch.setenv("TQB_STAGE1_KERNEL", "regs")
    for layout in ("soa", "aos", "soa_k8"):
        run_window(layout, torch.bfloat16, RAGGED, 8, 2, 50, 5, seed=2)


def test_window_in_the_caches_basis_and_other_arguments():
    run_window("soa", torch.float32, RAGGED, 8, 2, 50, 3, seed=3, raw=False, scale=0.05, out_dtype=torch.float16)


def test_lengths_below_zero_are_empty():
    run_window("soa", torch.bfloat16, [40, -1, 17, -2 ** 31], 4, 2, 20, 2, seed=1)
    for shared in (True, False):
        run_prefix("soa", torch.bfloat16, [4] * 3, 128, 4, 2, seed=1, short=[(1, -1), (2, -2 ** 31)], shared=shared)


def test_window_many_sequences():
    """More items than one round of the grid, ragged lengths: the weight cut with a split of first tokens."""
    rng = np.random.default_rng(4)
    run_window("soa", torch.bfloat16, list(rng.integers(1, 300, 90)), 8, 8, 128, 4, seed=5, num_splits=6)


def test_window_covering_everything_equals_the_decode_call():
    """The same splits and products; only where P V is added up differs.  A split of 10 tokens lies in two pages at most,
    so its sum of weights times codes times scales, at most 15 * 0.3 e^0.8 = 10 (the largest of 6000 scales lies below 4
    sigma), is truncated twice at 2^-23 of it by the decode call: 2.4e-6, and a rounding or two of the merge beside it."""
    rng = np.random.default_rng(8)
    c, _, R = book("soa")
    cache, table, lens = batch(rng, [5, 300, 77], 2, "soa")
    q = torch.from_numpy(rng.standard_normal((3, 8, 128)).astype(np.float32)).cuda()
    args = (torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(), torch.from_numpy(lens).cuda())
    a = tqb.window_attention(tqb.rotate_query(q, cuda(R)), *args, None, cuda(c), window=10 ** 6, num_splits=32)
    b = tqb.triton_turboquant_decode_attention(q, *args, cuda(R).T.contiguous(), cuda(c), 128 ** -0.5, 4, 66, 4)
    assert (a - b).abs().max().item() <= 2.0 ** -18


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows", [1, 15, 16, 17, 50])
def test_rotation_beside_stage1(dtype, rows):
    """The queries that a ranged call rotates on the way: 2^-17 |q| for the fp32 sums, as in the append, for rows of
    every size that their type holds (the split into parts keeps the range)."""
    rng = np.random.default_rng(rows)
    c, _, R = book("soa")
    cache, table, lens = batch(rng, [3] * rows, 1, "soa")
    q = torch.from_numpy(rng.standard_normal((rows, 1, 128)).astype(np.float32) * np.exp2(rng.integers(-9, 12, (rows, 1, 1))))
    q = q.to(DT[dtype]).cuda()
    a, r = _lib.Stage1Args(), _lib.RotateArgs()
    out = torch.full((rows, 1, 128), np.nan, device="cuda")
    mid = torch.empty(rows, 1, 1, 129, device="cuda")
    dev = [torch.from_numpy(x).cuda() for x in (cache, table, lens)] + [cuda(c), cuda(R)]
    a.q_rot = r.q_rot = out.data_ptr()
    a.q_stride_b = a.q_stride_h = r.out_stride_b = r.out_stride_h = 128
    a.kv_cache, a.block_table, a.seq_lens, a.centroids, r.rotation = (x.data_ptr() for x in dev)
    a.cache_stride_block, a.num_blocks = dev[0].stride(0), dev[0].shape[0]
    a.block_table_stride = a.max_blocks_per_seq = table.shape[1]
    a.n_centroids, a.mid_o, a.mid_stride_b, a.mid_stride_h, a.mid_stride_s = 16, mid.data_ptr(), 129, 129, 129
    a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim, a.block_size, a.num_splits = rows, 1, 1, 128, 16, 1
    r.query, r.q_stride_b, r.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
    r.query_dtype = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[q.dtype]
    r.batch, r.num_q_heads, r.head_dim = rows, 1, 128
    _lib.check(_lib.load().tqb_stage1_range(a, r, _lib.RangeArgs(0, 0, 0, 16), torch.cuda.current_stream().cuda_stream))
    x = q.double().cpu().numpy()
    tol = 2.0 ** -17 * np.linalg.norm(x, axis=-1, keepdims=True)
    assert (np.abs(out.cpu().numpy() - x @ npy(R).astype(np.float64)) <= tol).all()


def run_prefix(layout, dtype, own, prefix, hq, hk, *, seed=0, sinks=False, raw=True, short=(), scale_q=1.5, shared=True,
               chunks=None, bad=(), **kw):
    """``shared`` None: as the call decides; else whether a prefix of 128 tokens or more takes the shared pass.
    ``chunks``: its splits.  ``bad``: (entry, page id) pairs of the prefix in every row of the table."""
    with pytest.MonkeyPatch.context() as mp:
        if shared is not None:
            mp.setattr(tqb.serving, "_shares", lambda batch, rows, heads, prefix_len: shared and prefix_len >= 128)
        if chunks is not None:
            mp.setattr(tqb.serving, "_prefix_splits", lambda rows, heads, prefix_len: chunks)
        return run_prefix_as_set(layout, dtype, own, prefix, hq, hk, seed, sinks, raw, short, scale_q, bad, kw)


def run_prefix_as_set(layout, dtype, own, prefix, hq, hk, seed, sinks, raw, short, scale_q, bad, kw):
    rng = np.random.default_rng(seed)
    c, _, R = book(layout)
    cache, table, lens = batch(rng, [prefix + n for n in own], hk, layout, prefix // 16)
    for b, n in short:
        lens[b] = n
    for at, page in bad:
        table[:, at] = page
    q = torch.from_numpy(rng.standard_normal((len(lens), hq, 128)).astype(np.float32) * scale_q).to(dtype).cuda()
    raw = raw and R is not None
    s = torch.from_numpy(rng.standard_normal(hq).astype(np.float32) * 2).cuda() if sinks else None
    lse = torch.empty(len(lens), hq, device="cuda")
    got = tqb.prefix_attention(q, torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(),
                               torch.from_numpy(lens).cuda(), cuda(R) if raw else None, cuda(c), prefix_len=prefix,
                               layout=layout, sinks=s, lse=lse, **kw)
    x = npy(q).astype(np.float64)
    x = x @ npy(R).astype(np.float64) if raw else x
    ref, ref_lse, size = SO.attention(x, cache, layout, table, lens, npy(c), lambda t, L: t >= 0, scale=kw.get("scale"),
                                      sinks=npy(s))
    check_decode(got, lse, ref, ref_lse, got.dtype, size if got.dtype != torch.float32 and prefix >= 128 else None,
                 2.0 ** -10 + 2.0 ** -9 * scale_q + (2.0 ** -11 * ref_lse[..., None] if scale_q > 4 else 0))
    return got


@pytest.mark.parametrize("layout", sorted(SO.LAYOUTS))
def test_prefix_layouts(layout):
    run_prefix(layout, torch.bfloat16, [1, 0, 20, 63], 400, 8, 2, seed=1)


@pytest.mark.parametrize("hq,hk", [(32, 8), (16, 2), (5, 1), (6, 3)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
def test_prefix_heads_and_types(hq, hk, dtype):
    run_prefix("soa", DT[dtype], [3, 40, 17], 160, hq, hk, seed=hq, sinks=True)


@pytest.mark.parametrize("prefix", [0, 16, 112, 128, 144, 640])
@pytest.mark.parametrize("batch_size", [1, 2, 37, 70])
def test_prefix_lengths_and_batches(prefix, batch_size):
    rng = np.random.default_rng(prefix + batch_size)
    run_prefix("soa", torch.bfloat16, list(rng.integers(1, 50, batch_size)), prefix, 4, 1, seed=prefix)


def test_prefix_rows_shorter_than_the_prefix():
    """Padded rows of a batch (length 0) and rows that end inside the prefix, at a page's and a tile's edges."""
    run_prefix("soa", torch.bfloat16, [9] * 8, 320, 4, 1, seed=2, short=[(0, 0), (2, 1), (3, 128), (4, 129), (5, 320), (6, 255)])


@pytest.mark.parametrize("rows,chunks", [(20, 1), (20, 2), (20, 4), (128, 2), (129, 1), (160, 2), (256, 1), (257, 3), (560, 1)])
def test_prefix_of_many_tiles_to_a_block(rows, chunks):
    """One stream, two streams of one row block, the same rows over even and odd tiles, several row blocks."""
    hq = 8 if rows % 8 == 0 else 4 if rows % 4 == 0 else 1
    run_prefix("soa", torch.bfloat16, [5] * (rows // hq), 1296, hq, 1, seed=rows, chunks=chunks, sinks=True)


@pytest.mark.parametrize("layout", sorted(SO.LAYOUTS))
def test_prefix_layouts_of_many_tiles(layout):
    run_prefix(layout, torch.float16, [1, 9, 30] * 12, 720, 8, 2, seed=7, chunks=1)


@pytest.mark.parametrize("own,chunks", [([5] * 8, 2), ([5] * 40, 1)])
def test_prefix_scores_that_outgrow_their_reference(own, chunks):
    """Scores of a standard deviation of 12: later tiles' maxima exceed the first ones' by far more than 2^8."""
    run_prefix("soa", torch.bfloat16, own, 1280, 4, 1, seed=12, scale_q=12.0, chunks=chunks)


@pytest.mark.parametrize("shared", [True, False])
def test_prefix_pages_that_do_not_exist(shared):
    """Single ones, a tile of them, and a prefix of nothing else."""
    bad = [(3, -1), (11, 10 ** 6), (19, -2 ** 31)] + [(i, 2 ** 31 - 1) for i in range(24, 32)]
    run_prefix("soa", torch.bfloat16, [9] * 6, 640, 4, 1, seed=3, bad=bad, shared=shared)
    run_prefix("soa", torch.bfloat16, [9] * 6, 256, 4, 1, seed=3, bad=[(i, -1) for i in range(16)], shared=shared)


@pytest.mark.parametrize("batch_size,prefix", [(1, 640), (8, 128), (12, 16384), (64, 1024), (300, 512)])
def test_prefix_as_the_call_decides(batch_size, prefix):
    run_prefix("soa", torch.bfloat16, [3] * batch_size, prefix, 2, 2, seed=prefix, shared=None)


@pytest.mark.parametrize("layout", ["soa", "aos_k3"])
def test_prefix_keys_that_are_not_finite_stay_where_they_are_seen(layout):
    """Norms of inf and NaN behind two rows' ends: those rows have their own numbers, the others none."""
    rng = np.random.default_rng(14)
    c, _, R = book(layout)
    cache, table, lens = batch(rng, [300] * 6, 1, layout, 16)
    lens[1], lens[4] = 100, 200
    for t, bad in ((200, np.nan), (230, np.inf), (255, -np.inf)):
        _, _, norm, _, _ = SO.places(layout, 1, t % 16, 0)
        cache.reshape(len(cache), -1)[table[0, t // 16], norm:norm + 2] = np.array([bad], np.float16).view(np.uint8)
    q = torch.from_numpy(rng.standard_normal((6, 4, 128)).astype(np.float32)).to(torch.bfloat16).cuda()
    with pytest.MonkeyPatch.context() as mp:
        mp.setattr(tqb.serving, "_shares", lambda *a: True)
        got = tqb.prefix_attention(q, torch.from_numpy(cache).cuda(), torch.from_numpy(table).cuda(),
                                   torch.from_numpy(lens).cuda(), cuda(R), cuda(c), prefix_len=256, layout=layout)
    x = npy(q).astype(np.float64) @ npy(R).astype(np.float64)
    ref, _, size = SO.attention(x[[1, 4]], cache, layout, table[[1, 4]], lens[[1, 4]], npy(c), lambda t, L: t >= 0)
    assert (np.abs(npy(got)[[1, 4]] - ref) <= 1e-4 + half_step(got.dtype) * np.abs(ref) + 4e-3 * size).all()
    assert np.isnan(npy(got)[[0, 2, 3, 5]]).all()


def test_prefix_into_given_workspaces_and_outputs():
    """Partials of 129 floats, a strided output, and the same numbers as with the call's own."""
    a = run_prefix("aos_k3", torch.bfloat16, [20] * 5, 400, 6, 2, seed=5, num_splits=3)
    buf = torch.zeros(5, 6, 130, dtype=torch.bfloat16, device="cuda")
    mid = torch.full((6, 7, 11, 129), np.nan, device="cuda")
    b = run_prefix("aos_k3", torch.bfloat16, [20] * 5, 400, 6, 2, seed=5, num_splits=3, output=buf[..., :128], mid_o=mid)
    assert torch.equal(a, b) and (buf[..., 128:] == 0).all()
    assert torch.isnan(mid[5:]).all() and torch.isnan(mid[:, 6:]).all()


def test_prefix_empty_batch():
    c, _, R = book("soa")
    q = torch.empty(0, 4, 128, device="cuda")
    cache = torch.zeros(9, 16, 2, 134, dtype=torch.uint8, device="cuda")
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    out = tqb.prefix_attention(q, cache, none.reshape(0, 9), none, cuda(R), cuda(c), prefix_len=128)
    assert out.shape == (0, 4, 128)


def serving_calls(seed):
    """The four calls on inputs of their own, large enough for the tensor-core forms: a function and its results' names."""
    rng = np.random.default_rng(seed)
    c, m, R = (cuda(x) for x in book("soa"))
    cache_np, table, lens = batch(rng, [640 + n for n in rng.integers(1, 60, 64)], 4, "soa", 40)
    cache, table, lens = (torch.from_numpy(x).cuda() for x in (cache_np, table, lens))
    n = 1100
    store = torch.zeros(n // 16 + 1, 16, 4, 134, dtype=torch.uint8, device="cuda")
    slots = torch.from_numpy(rng.permutation(n).astype(np.int32)).cuda()
    q, k, v = projections(rng, n, 16, 4, torch.bfloat16)
    cs, pos = torch.from_numpy(cos_sin_table(500, 128)).cuda(), torch.from_numpy(rng.integers(0, 500, n)).cuda()

    def run(**kw):
        qr = tqb.rope_append(k, v, store, slots, pos, cs, R, m, c, query=q, **kw)
        gk, gv = tqb.gather_kv(store, slots, c, **kw)
        w = tqb.window_attention(q[:64], cache, table, lens, R, c, window=200, first_tokens=4, **kw)
        return qr, gk, gv, w, tqb.prefix_attention(q[:64], cache, table, lens, R, c, prefix_len=640, **kw), store

    return run


@pytest.fixture
def shared_prefix(monkeypatch):
    monkeypatch.setattr(tqb.serving, "_shares", lambda *a: True)


def test_calls_on_two_streams_at_once(shared_prefix):
    """Two threads' worth of calls in flight on two streams, by the current stream and by ``stream``: the same bits as
    alone, every time."""
    runs = [serving_calls(1), serving_calls(2)]
    alone = [[x.clone() for x in run()] for run in runs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(6):
        for run, st in zip(runs, streams):
            if i % 2:
                got.append(run(stream=st.cuda_stream))
            else:
                with torch.cuda.stream(st):
                    got.append(run())
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        for a, b in zip(out, alone[i % 2]):
            assert torch.equal(a, b)


def test_calls_in_two_graphs_replayed_at_once(shared_prefix):
    runs = [serving_calls(3), serving_calls(4)]
    alone = [[x.clone() for x in run()] for run in runs]
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for run, g in zip(runs, graphs):
        with torch.cuda.graph(g):
            outs.append(run())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for out in outs:
            for x in out:
                x.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for out, ref in zip(outs, alone):
            for a, b in zip(out, ref):
                assert torch.equal(a, b)


def test_step_append_then_attend_on_a_side_stream_and_in_a_graph():
    """Append, then both decode calls, as a step runs them: on a side stream, captured and replayed on new inputs."""
    rng = np.random.default_rng(11)
    c, m, R = (cuda(x) for x in book("soa"))
    cache_np, table, lens = batch(rng, [64 + n for n in (5, 30, 17)], 2, "soa", 4)
    cache, table, lens = (torch.from_numpy(x).cuda() for x in (cache_np, table, lens))
    cs = torch.from_numpy(cos_sin_table(500, 128)).cuda()
    q, k, v = projections(rng, 3, 8, 2, torch.bfloat16)
    slots = (table.gather(1, (lens[:, None].long() - 1) // 16) * 16 + (lens[:, None] - 1) % 16).flatten().int()
    pos = lens.long() - 1

    def step():
        qr = tqb.rope_append(k, v, cache, slots, pos, cs, R, m, c, query=q)
        w = tqb.window_attention(qr, cache, table, lens, None, c, window=40, first_tokens=4, out_dtype=q.dtype)
        return w, tqb.prefix_attention(qr, cache, table, lens, None, c, prefix_len=64, out_dtype=q.dtype)

    def ref():
        x = SO.rope(npy(q).astype(np.float64), npy(cs)[pos.cpu().numpy()], False) @ npy(R).astype(np.float64)
        t, l, ca = table.cpu().numpy(), lens.cpu().numpy(), cache.cpu().numpy()
        return [SO.attention(x, ca, "soa", t, l, npy(c), f)[0] for f in (lambda t, L: (t < 4) | (t >= L - 40), lambda t, L: t >= 0)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    for a, b in zip(got, ref()):
        assert (np.abs(npy(a) - b) <= 1e-4 + (2e-3 + half_step(q.dtype)) * np.abs(b)).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    q.copy_(torch.randn_like(q))
    k.copy_(torch.randn_like(k))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, ref()):
        assert (np.abs(npy(a) - b) <= 1e-4 + (2e-3 + half_step(q.dtype)) * np.abs(b)).all()
