"""Serving steps around the paged cache: append, gather, windowed and shared-prefix decode.

A decode step of a model with rotary positions is two calls::

    q_rot = tqb.rope_append(k, v, kv_cache, slots, positions, cos_sin, PiT, midpoints, centroids, query=q)
    out = tqb.window_attention(q_rot, kv_cache, block_table, seq_lens, None, centroids, window=1024,
                               first_tokens=4, out_dtype=q.dtype)

and a later chunk of a prefill reads its context back with ``gather_kv``.  All run on the tensors' device and its
current stream (or ``stream``), launch asynchronously and can be captured into CUDA graphs; outputs and the split
partials are allocated by torch unless they are given.  A workspace (``mid_o``) that two calls share serialises
nothing: calls that may overlap need one each.  Errors raise ``TqbError``.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._lib import AppendArgs, GatherArgs, RangeArgs
from .layout import BLOCK_SIZE, FP8_KEY_LAYOUTS, HEAD_DIM, KEY3_LAYOUTS, SLOT_BYTES, layout_id
from .ops import (_DTYPE_ID, _SOA_FAMILY, _block_dense, _cuda, _require, _stage1_args, _stage2_args, _stream)

_SPLIT_TOKENS = 64    # shortest split worth its partial rows (516 bytes written and read per query head)
_SPLIT_ITEMS = 2368   # (sequence, KV head, split) items of one round of the Stage1 grid: 148 CTAs x 2 groups x 8 warps


def _same_device(**tensors) -> torch.device:
    devs = {t.device for t in tensors.values() if t is not None}
    _require(len(devs) == 1, f"all tensors must be on one device, got {sorted(map(str, devs))}")
    return devs.pop()


def _check_cache(kv_cache: torch.Tensor, lay: int) -> None:
    _cuda(kv_cache, "kv_cache", torch.uint8)
    _require(kv_cache.dim() == 4 and kv_cache.shape[1] == BLOCK_SIZE and kv_cache.stride(3) == 1,
             "kv_cache must be [num_blocks, 16, Hk, slot] bytes")
    _require(kv_cache.shape[3] >= SLOT_BYTES[lay], f"this layout has slots of {SLOT_BYTES[lay]} bytes, "
             f"kv_cache has {kv_cache.shape[3]}")
    if lay in _SOA_FAMILY:
        _require(_block_dense(kv_cache), "SoA cache needs each block's bytes contiguous")


def _check_centroids(centroids: Optional[torch.Tensor], lay: int) -> int:
    n = 8 if lay in KEY3_LAYOUTS else 16
    if lay not in FP8_KEY_LAYOUTS:
        _cuda(centroids, "centroids", torch.float32)
        _require(centroids.shape == (n,) and centroids.is_contiguous(), f"centroids must be a contiguous [{n}] tensor")
    return n


def _rows(t: torch.Tensor, name: str, n: int) -> None:
    _require(isinstance(t, torch.Tensor) and t.is_cuda and t.dtype in _DTYPE_ID,
             f"{name} must be a float32/float16/bfloat16 CUDA tensor")
    _require(t.dim() == 3 and t.shape[0] == n and t.shape[2] == HEAD_DIM and (t.stride(2) == 1 or t.numel() == 0),
             f"{name} must be [{n}, heads, 128] with unit stride over the last dim")


def rope_append(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor, slot_mapping: torch.Tensor,
                positions: Optional[torch.Tensor], cos_sin: Optional[torch.Tensor],
                rotation: Optional[torch.Tensor], midpoints: Optional[torch.Tensor],
                centroids: Optional[torch.Tensor], *, layout="soa", norm_correction: bool = True,
                interleaved: bool = False, query: Optional[torch.Tensor] = None,
                q_rot: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> Optional[torch.Tensor]:
    """Append raw ``key``/``value`` ``[N, Hk, 128]`` to the cache: rotary positions, rotation and quantised store in
    one kernel (``tqb_append``), and with ``query [N, Hq, 128]`` the rotated queries ``rope(query) @ rotation`` into
    ``q_rot`` (float32 ``[N, Hq, 128]``, allocated when None), which is returned.

    ``cos_sin`` is float32 ``[max_pos, rotary_dim]``, the cosines of ``rotary_dim / 2`` angles and then their sines;
    pairs are ``(i, i + rotary_dim / 2)``, or ``(2i, 2i + 1)`` with ``interleaved``.  ``positions`` (int32 or int64
    ``[N]``) None leaves the rotary step out.  ``rotation`` is the orthogonal ``Pi^T`` of ``rotate_query``; FP8-key
    layouts use neither it nor ``midpoints``/``centroids``.  ``key``, ``value`` and ``query`` may be slices of one
    projection's output (any strides but the last).  Key codes are those of exact arithmetic, whatever the order of the
    kernel's sums; value codes are ``store``'s, byte for byte.  ``norm_correction`` folds ``1/|c|`` into the stored
    norm of the SoA Lloyd-Max layouts; the other layouts have none to fold.

    Tokens with a negative or out-of-range slot, or a position outside the table, are not stored (the latter's
    ``q_rot`` rows are NaN).  Slots must be distinct."""
    lay = layout_id(layout)
    k8 = lay in FP8_KEY_LAYOUTS
    _check_cache(kv_cache, lay)
    _cuda(slot_mapping, "slot_mapping", torch.int32)
    _require(slot_mapping.dim() == 1 and slot_mapping.is_contiguous(), "slot_mapping must be a contiguous [N] tensor")
    N, Hk = slot_mapping.shape[0], kv_cache.shape[2]
    _rows(key, "key", N)
    _rows(value, "value", N)
    _require(key.shape[1] == Hk and value.shape[1] == Hk, f"key and value must have the cache's {Hk} heads")
    _require(value.dtype == key.dtype, "key and value must have one dtype")
    n = _check_centroids(centroids, lay)
    if not k8:
        _cuda(midpoints, "midpoints", torch.float32)
        _require(midpoints.shape == (n - 1,) and midpoints.is_contiguous(),
                 f"midpoints must be a contiguous [{n - 1}] tensor")
        _cuda(rotation, "rotation", torch.float32)
        _require(tuple(rotation.shape) == (HEAD_DIM, HEAD_DIM) and rotation.is_contiguous(),
                 "rotation must be a contiguous [128, 128] matrix")
    a = AppendArgs()
    if positions is not None:
        _require(isinstance(positions, torch.Tensor) and positions.is_cuda and
                 positions.dtype in (torch.int32, torch.int64), "positions must be an int32 or int64 CUDA tensor")
        _require(positions.shape == (N,) and positions.is_contiguous(), "positions must be a contiguous [N] tensor")
        _cuda(cos_sin, "cos_sin", torch.float32)
        _require(cos_sin.dim() == 2 and cos_sin.stride(1) == 1, "cos_sin must be [max_pos, rotary_dim] row-major")
        a.positions, a.positions_are_64 = positions.data_ptr(), int(positions.dtype == torch.int64)
        a.cos_sin, a.cos_sin_stride = cos_sin.data_ptr(), max(cos_sin.stride(0), cos_sin.shape[1])
        a.max_pos, a.rotary_dim = cos_sin.shape
        _require(cos_sin.shape[0] <= 1 or cos_sin.stride(0) >= cos_sin.shape[1], "cos_sin rows must not overlap")
    a.interleaved = int(bool(interleaved))
    if query is not None:
        _rows(query, "query", N)
        _require(query.dtype == key.dtype, "query must have the key's dtype")
        if q_rot is None:
            q_rot = torch.empty(query.shape, dtype=torch.float32, device=query.device)
        _cuda(q_rot, "q_rot", torch.float32)
        _require(q_rot.shape == query.shape and q_rot.stride(2) == 1, "q_rot must have the query's shape")
        a.query, a.q_stride_n, a.q_stride_h = query.data_ptr(), query.stride(0), query.stride(1)
        a.q_rot, a.q_rot_stride_n, a.q_rot_stride_h = q_rot.data_ptr(), q_rot.stride(0), q_rot.stride(1)
        a.num_q_heads = query.shape[1]
    else:
        _require(q_rot is None, "q_rot is the output of query")
    dev = _same_device(key=key, value=value, kv_cache=kv_cache, slot_mapping=slot_mapping, positions=positions,
                       cos_sin=cos_sin, rotation=rotation, midpoints=midpoints, centroids=centroids, query=query,
                       q_rot=q_rot)
    a.key, a.value, a.dtype = key.data_ptr(), value.data_ptr(), _DTYPE_ID[key.dtype]
    a.k_stride_n, a.k_stride_h = key.stride(0), key.stride(1)
    a.v_stride_n, a.v_stride_h = value.stride(0), value.stride(1)
    if not k8:
        a.rotation, a.midpoints, a.centroids = rotation.data_ptr(), midpoints.data_ptr(), centroids.data_ptr()
    a.slot_mapping, a.kv_cache, a.layout = slot_mapping.data_ptr(), kv_cache.data_ptr(), lay
    a.cache_stride_block, a.cache_stride_pos, a.cache_stride_head = kv_cache.stride()[:3]
    a.num_blocks, a.block_size = kv_cache.shape[0], kv_cache.shape[1]
    a.num_tokens, a.num_kv_heads, a.head_dim, a.n_centroids = N, Hk, HEAD_DIM, n
    a.norm_correction = int(bool(norm_correction) and lay in _SOA_FAMILY and not k8)
    with torch.cuda.device(dev):
        _lib.check(_lib.load().tqb_append(a, stream if stream is not None else _stream(dev)))
    return q_rot


def gather_kv(kv_cache: torch.Tensor, slot_mapping: torch.Tensor, centroids: Optional[torch.Tensor], *, layout="soa",
              dtype: torch.dtype = torch.bfloat16, key: Optional[torch.Tensor] = None,
              value: Optional[torch.Tensor] = None, stream: Optional[int] = None):
    """Keys and values ``[N, Hk, 128]`` that the cache holds in ``slot_mapping``'s slots (int32 ``[N]``), in ``dtype``
    (or into ``key``/``value``), one rounding each: what a later chunk of a prefill attends to
    (reference/soa_decode_v1.py:322-454).  Lloyd-Max keys stay in the rotated basis, where the chunk's queries are taken
    too (:func:`rotate_query`).  Rows of negative or out-of-range slots are zeros."""
    lay = layout_id(layout)
    _check_cache(kv_cache, lay)
    _cuda(slot_mapping, "slot_mapping", torch.int32)
    _require(slot_mapping.dim() == 1 and slot_mapping.is_contiguous(), "slot_mapping must be a contiguous [N] tensor")
    n = _check_centroids(centroids, lay)
    N, Hk = slot_mapping.shape[0], kv_cache.shape[2]
    _require((key is None) == (value is None), "key and value go together")
    if key is None:
        _require(dtype in _DTYPE_ID, "dtype must be float32, float16 or bfloat16")
        key, value = (torch.empty(N, Hk, HEAD_DIM, dtype=dtype, device=kv_cache.device) for _ in range(2))
    _rows(key, "key", N)
    _rows(value, "value", N)
    _require(key.shape[1] == Hk and value.shape[1] == Hk and key.dtype == value.dtype,
             f"key and value must be [{N}, {Hk}, 128] tensors of one dtype")
    dev = _same_device(kv_cache=kv_cache, slot_mapping=slot_mapping, centroids=centroids, key=key, value=value)
    a = GatherArgs()
    a.kv_cache, a.layout = kv_cache.data_ptr(), lay
    a.cache_stride_block, a.cache_stride_pos, a.cache_stride_head = kv_cache.stride()[:3]
    a.num_blocks, a.block_size = kv_cache.shape[0], kv_cache.shape[1]
    a.slot_mapping = slot_mapping.data_ptr()
    a.centroids = centroids.data_ptr() if lay not in FP8_KEY_LAYOUTS else None
    a.key, a.value, a.out_dtype = key.data_ptr(), value.data_ptr(), _DTYPE_ID[key.dtype]
    a.k_stride_n, a.k_stride_h = key.stride(0), key.stride(1)
    a.v_stride_n, a.v_stride_h = value.stride(0), value.stride(1)
    a.num_tokens, a.num_kv_heads, a.head_dim, a.n_centroids = N, Hk, HEAD_DIM, n
    with torch.cuda.device(dev):
        _lib.check(_lib.load().tqb_gather(a, stream if stream is not None else _stream(dev)))
    return key, value


def _splits(items: int, tokens: int) -> int:
    """Splits of ``tokens`` for ``items`` (sequence, KV head) pairs: enough items for one round of the Stage1 grid, none
    under ``_SPLIT_TOKENS`` tokens."""
    return max(1, min(-(-_SPLIT_ITEMS // max(items, 1)), -(-tokens // _SPLIT_TOKENS)))


def _decode_args(query, kv_cache, block_table, seq_lens, rotation, centroids, lay, sinks, output, lse, out_dtype, mid_o):
    """What both decode calls check and allocate: the rows that Stage1 reads, the raw query when it rotates them, and
    the outputs."""
    _require(isinstance(query, torch.Tensor) and query.is_cuda and query.dim() == 3 and query.shape[2] == HEAD_DIM and
             query.dtype in _DTYPE_ID, "query must be a [B, Hq, 128] float32/float16/bfloat16 CUDA tensor")
    _check_cache(kv_cache, lay)
    _require(rotation is None or lay not in FP8_KEY_LAYOUTS, "FP8 keys are not rotated: rotation must be None")
    _require(isinstance(block_table, torch.Tensor) and block_table.dim() == 2 and block_table.shape[1] > 0,
             "block_table must be [B, max_blocks]")
    B, Hq, D = query.shape
    _require(Hq > 0 and Hq % kv_cache.shape[2] == 0, "query heads must be a multiple of the cache's")
    raw = None
    if rotation is not None:
        raw = query if query.stride(2) == 1 else query.contiguous()
        rows = torch.empty(B, Hq, D, dtype=torch.float32, device=query.device)
    else:
        rows = query.float().contiguous()
    if output is None:
        output = torch.empty(B, Hq, D, dtype=out_dtype or query.dtype, device=query.device)
    if lse is None:
        lse = torch.empty(B, Hq, dtype=torch.float32, device=query.device)
    if sinks is not None:
        _cuda(sinks, "sinks", torch.float32)
        _require(sinks.shape == (Hq,) and sinks.is_contiguous(), "sinks must be a contiguous [Hq] tensor")
    _same_device(query=query, kv_cache=kv_cache, block_table=block_table, seq_lens=seq_lens, rotation=rotation,
                 centroids=centroids, sinks=sinks, output=output, lse=lse, mid_o=mid_o)
    return rows, raw, output, lse


def _partials(mid_o, B, Hq, S, device) -> torch.Tensor:
    if mid_o is None:
        return torch.empty(B, Hq, S, HEAD_DIM + 1, dtype=torch.float32, device=device)
    _cuda(mid_o, "mid_o", torch.float32)
    _require(mid_o.dim() == 4 and mid_o.shape[0] >= B and mid_o.shape[1] >= Hq and mid_o.shape[2] >= S and
             mid_o.shape[3] == HEAD_DIM + 1, f"mid_o must hold [{B}, {Hq}, {S}, 129] partials")
    return mid_o[:B, :Hq, :S]


def window_attention(query: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                     rotation: Optional[torch.Tensor], centroids: Optional[torch.Tensor], *, window: int,
                     first_tokens: int = 0, scale: Optional[float] = None, layout="soa",
                     sinks: Optional[torch.Tensor] = None, num_splits: Optional[int] = None,
                     output: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                     lse: Optional[torch.Tensor] = None, mid_o: Optional[torch.Tensor] = None,
                     stream: Optional[int] = None) -> torch.Tensor:
    """Decode attention of each query ``[B, Hq, 128]`` over the last ``window`` tokens of its sequence and its first
    ``first_tokens`` ones, on any cache layout; returns ``output`` (allocated in ``out_dtype`` or the query's dtype).

    ``rotation`` is the ``[128, 128]`` matrix of ``rotate_query``, applied on the way; None for queries that are in the
    cache's basis already (``rope_append``'s ``q_rot``; FP8 keys).  ``sinks`` (float32 ``[Hq]``) adds one token of that
    logit and value 0 per head.  ``lse`` (float32 ``[B, Hq]``) receives the log-sum-exp.  Only the pages that hold
    visible tokens are read.  A sequence of length 0 gets NaN and an LSE of -inf, as in ``stage2``.  Sequences longer
    than the block table's rows are cut there.

    The first tokens are a split of their own and the window is shared by the others; ``num_splits`` counts the latter.
    ``mid_o`` may hold the partials: float32 ``[>= B, >= Hq, >= splits, 129]``, with one split more than ``num_splits``
    when ``first_tokens > 0``.  Calls with a ``rotation`` must not overlap in time on one device (``tqb_stage1_rotated``'s
    rule); with ``rotation=None`` they may."""
    lay = layout_id(layout)
    _require(isinstance(window, int) and window >= 1, "window must be at least 1")
    _require(isinstance(first_tokens, int) and first_tokens >= 0, "first_tokens must not be negative")
    _require(num_splits is None or num_splits >= 1, "num_splits must be positive")
    rows, raw, output, lse = _decode_args(query, kv_cache, block_table, seq_lens, rotation, centroids, lay, sinks, output,
                                          lse, out_dtype, mid_o)
    B, Hq, _ = query.shape
    if B == 0:
        return output
    most = block_table.shape[1] * BLOCK_SIZE
    window, first_tokens = min(window, most), min(first_tokens, most)
    S = (num_splits or _splits(B * kv_cache.shape[2], window)) + (1 if first_tokens else 0)
    mid = _partials(mid_o, B, Hq, S, query.device)
    rng = RangeArgs(window, first_tokens, 0, most)
    _ranged(rows, raw, kv_cache, block_table, seq_lens, rotation, centroids, mid, mid, rng, 0, scale, lay, sinks, output,
            lse, stream)
    return output


def _ranged(rows, raw, kv_cache, block_table, seq_lens, rotation, centroids, mid, mid_stage1, rng, lead, scale, lay, sinks,
            output, lse, stream):
    """Stage1 of ``rng`` into ``mid_stage1`` (the splits of ``mid`` from ``lead`` on) and the merge of all of ``mid``."""
    _require(seq_lens.dim() == 1 and seq_lens.shape[0] == rows.shape[0], "seq_lens must be a contiguous [B] tensor")
    a, r = _stage1_args(rows, kv_cache, block_table, seq_lens, centroids, mid_stage1, layout=lay, attn_scale=scale,
                        query=raw, rotation=rotation)
    b = _stage2_args(mid, seq_lens, output, lse)
    lib = _lib.load()
    with torch.cuda.device(output.device):
        st = stream if stream is not None else _stream(output.device)
        _lib.check(lib.tqb_stage1_range(a, r, rng, st))
        _lib.check(lib.tqb_stage2_range(b, rng, lead, sinks.data_ptr() if sinks is not None else None,
                                        _DTYPE_ID[output.dtype], output.data_ptr(), st))


def prefix_attention(query: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                     rotation: Optional[torch.Tensor], centroids: Optional[torch.Tensor], *, prefix_len: int,
                     scale: Optional[float] = None, layout="soa", sinks: Optional[torch.Tensor] = None,
                     num_splits: Optional[int] = None, output: Optional[torch.Tensor] = None,
                     out_dtype: Optional[torch.dtype] = None, lse: Optional[torch.Tensor] = None,
                     mid_o: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
    """Decode attention ``[B, Hq, 128]`` of a batch whose sequences begin with the same ``prefix_len`` tokens, a
    multiple of 16: the first ``prefix_len / 16`` entries of every row of ``block_table`` are the same pages.
    ``seq_lens`` and ``block_table`` describe whole sequences, prefix included; a sequence shorter than the prefix sees
    its own tokens only.  The other arguments are :func:`window_attention`'s."""
    lay = layout_id(layout)
    _require(isinstance(prefix_len, int) and prefix_len >= 0 and prefix_len % BLOCK_SIZE == 0,
             "prefix_len must be a multiple of 16")
    _require(num_splits is None or num_splits >= 1, "num_splits must be positive")
    rows, raw, output, lse = _decode_args(query, kv_cache, block_table, seq_lens, rotation, centroids, lay, sinks, output,
                                          lse, out_dtype, mid_o)
    B, Hq, _ = query.shape
    _require(prefix_len <= block_table.shape[1] * BLOCK_SIZE, "the block table's rows do not hold the prefix")
    if B == 0:
        return output
    most = block_table.shape[1] * BLOCK_SIZE
    S = num_splits or _splits(B * kv_cache.shape[2], most)
    mid = _partials(mid_o, B, Hq, S, query.device)
    rng = RangeArgs(0, 0, 0, most)
    _ranged(rows, raw, kv_cache, block_table, seq_lens, rotation, centroids, mid, mid, rng, 0, scale, lay, sinks, output,
            lse, stream)
    return output
