"""Serving steps around the paged cache: append, gather, windowed and shared-prefix decode.

A decode step of a model with rotary positions is two calls::

    q_rot = tqb.rope_append(k, v, kv_cache, slots, positions, cos_sin, PiT, midpoints, centroids, query=q)
    out = tqb.window_attention(q_rot, kv_cache, block_table, seq_lens, None, centroids, window=1024,
                               first_tokens=4, out_dtype=q.dtype)

and a later chunk of a prefill reads its context back with ``gather_kv``.  All run on the tensors' device and its
current stream, launch asynchronously and can be captured into CUDA graphs; outputs and the split partials are allocated
by torch unless they are given.  ``stream``, a ``cuda_stream`` handle, makes a call one that is made inside
``torch.cuda.stream`` of it: what it allocates belongs to that stream.  A workspace (``mid_o``) that two calls share serialises
nothing: calls that may overlap need one each.  Errors raise ``TqbError``.
"""

from __future__ import annotations

import ctypes
import functools
import math
import operator
import struct
from typing import Optional

import torch

from . import _lib
from ._lib import AppendArgs, GatherArgs, RangeArgs, RotateArgs, Stage1Args, Stage2Args, TqbError
from .layout import (BLOCK_SIZE, FP8_KEY_LAYOUTS, HEAD_DIM, KEY3_LAYOUTS, LAYOUT_SOA, LAYOUT_SOA_K3, LAYOUT_SOA_K3V3,
                     SLOT_BYTES, layout_id)
from .ops import _DTYPE_ID, _SOA_FAMILY, _block_dense

_F32, _U8, _I32, _I64 = torch.float32, torch.uint8, torch.int32, torch.int64
_FOLDED = (LAYOUT_SOA, LAYOUT_SOA_K3, LAYOUT_SOA_K3V3)  # the stored norm may hold the norm correction
_PITCH = HEAD_DIM + 4  # floats of a partial row in the calls' own workspace: 129, and rows of whole 16 bytes
# Shortest split worth its partial rows (516 bytes written and read per query head).  1024 tokens of one sequence and 8
# heads take 16.6, 16.0, 19.3 and 23.0 us with 16, 32, 64 and 128; 4096 take 22.3, 18.7, 19.7 and 24.9.
_SPLIT_TOKENS = 32
_SMS = 148  # of a B200, the only GPU that the library is built for


# The step's calls are launches of a few microseconds, so their arguments are packed into the C structs' bytes at once
# (a third of the time that setting the fields of a ctypes structure takes) and every check reads a property once.
def packer(cls):
    """``struct.Struct.pack`` of a flat C argument struct, in the native layout with its tail padding."""
    code = {ctypes.c_void_p: "P", ctypes.c_int32: "i", ctypes.c_int64: "q", ctypes.c_float: "f"}
    fields = [t for _, t in cls._fields_]
    return struct.Struct("@" + "".join(code[t] for t in fields) + "0" + code[max(fields, key=ctypes.sizeof)])


_APPEND, _GATHER, _STAGE1, _STAGE2, _ROTATE, _RANGE = map(
    packer, (AppendArgs, GatherArgs, Stage1Args, Stage2Args, RotateArgs, RangeArgs))
_calls = {}


def _call(name: str, *args) -> None:
    """A library call whose structs are given as bytes (None: NULL)."""
    f = _calls.get(name)
    if f is None:
        f = _lib.load()[name]  # a function object of its own, apart from _lib's
        f.argtypes = {"tqb_append": [ctypes.c_char_p, ctypes.c_void_p],
                      "tqb_gather": [ctypes.c_char_p, ctypes.c_void_p],
                      "tqb_stage1_range": [ctypes.c_char_p] * 3 + [ctypes.c_void_p],
                      "tqb_prefix": [ctypes.c_char_p, ctypes.c_int, ctypes.c_void_p],
                      "tqb_stage2_range": [ctypes.c_char_p] * 2 + [ctypes.c_int, ctypes.c_void_p, ctypes.c_int,
                                                                   ctypes.c_void_p, ctypes.c_void_p]}[name]
        f.restype = ctypes.c_int
        _calls[name] = f
    status = f(*args)
    if status:
        _lib.check(status)


def _no(msg: str):
    raise TqbError(_lib.TQB_ERR_INVALID_ARG, msg)


def _int(x, name: str) -> int:
    try:
        return operator.index(x)
    except TypeError:
        _no(f"{name} must be an integer")


def _split_count(x) -> Optional[int]:
    if x is None:
        return None
    x = _int(x, "num_splits")
    if not 1 <= x <= 1 << 20:
        _no("num_splits must be positive (and at most 2^20)")
    return x


def _on(t, name: str, dtype, dev: int = -1) -> int:
    """The CUDA device of tensor ``t`` of ``dtype``: device ``dev`` if that is given."""
    if not isinstance(t, torch.Tensor):
        _no(f"{name} must be a torch.Tensor")
    d = t.get_device()
    if d < 0:
        _no(f"{name} must be a CUDA tensor")
    if t.dtype is not dtype:
        _no(f"{name} must be {dtype}, got {t.dtype}")
    if dev >= 0 and d != dev:
        _no(f"all tensors must be on one device: {name} is on cuda:{d}, others on cuda:{dev}")
    return d


def _vector(t, name: str, n: int, dtype, dev: int) -> int:
    """Address of a contiguous [n] tensor."""
    _on(t, name, dtype, dev)
    if t.shape != (n,) or not t.is_contiguous():
        _no(f"{name} must be a contiguous [{n}] tensor")
    return t.data_ptr()


def _float_rows(t, name: str, dev: int = -1):
    """(device, dtype id, shape, strides) of a [N, heads, 128] tensor of float32, float16 or bfloat16."""
    d = t.get_device() if isinstance(t, torch.Tensor) else -1
    kind = _DTYPE_ID.get(t.dtype) if d >= 0 else None
    if kind is None:
        _no(f"{name} must be a float32/float16/bfloat16 CUDA tensor")
    if dev >= 0 and d != dev:
        _no(f"all tensors must be on one device: {name} is on cuda:{d}, others on cuda:{dev}")
    shape = t.shape
    if len(shape) != 3 or shape[2] != HEAD_DIM:
        _no(f"{name} must be [N, heads, 128], got {tuple(shape)}")
    stride = t.stride()
    if stride[2] != 1 and shape[0] and shape[1]:
        _no(f"{name} must have unit stride over the last dim")
    return d, kind, shape, stride


def _cache(kv_cache, lay: int, dev: int = -1):
    """(device, shape, strides in bytes) of the paged cache."""
    d = _on(kv_cache, "kv_cache", _U8, dev)
    shape, stride = kv_cache.shape, kv_cache.stride()
    if len(shape) != 4 or shape[0] < 1 or shape[1] != BLOCK_SIZE or shape[2] < 1 or stride[3] != 1:
        _no("kv_cache must be [num_blocks, 16, Hk, slot] bytes of at least one block")
    if shape[3] < SLOT_BYTES[lay]:
        _no(f"this layout has slots of {SLOT_BYTES[lay]} bytes, kv_cache has {shape[3]}")
    if lay in _SOA_FAMILY and not (stride[1] == shape[2] * shape[3] and stride[2] == shape[3]) and not _block_dense(kv_cache):
        _no("SoA cache needs each block's bytes contiguous")
    return d, shape, stride


def _stream(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)


def _on_stream(call):
    """``call`` with its ``stream`` made the current one, so that its workspaces are that stream's too."""
    @functools.wraps(call)
    def on(*args, stream: Optional[int] = None, **kw):
        if stream is None:
            return call(*args, **kw)
        at = next((x.device for x in (*args, *kw.values()) if isinstance(x, torch.Tensor) and x.is_cuda), None)
        if at is None or stream == _stream(at.index):
            return call(*args, **kw)
        with torch.cuda.stream(torch.cuda.ExternalStream(stream, at) if stream else torch.cuda.default_stream(at)):
            return call(*args, **kw)
    return on


@_on_stream
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
    dev, kind, kshape, ks = _float_rows(key, "key")
    _, vkind, vshape, vs = _float_rows(value, "value", dev)
    _, cshape, cs = _cache(kv_cache, lay, dev)
    N, Hk, _ = kshape
    if vshape != kshape or Hk != cshape[2] or vkind != kind:
        _no(f"key and value must be [N, {cshape[2]}, 128] tensors of one shape and dtype")
    slots = _vector(slot_mapping, "slot_mapping", N, _I32, dev)
    n = 8 if lay in KEY3_LAYOUTS else 16
    rot = mids = cents = 0
    if not k8:
        cents = _vector(centroids, "centroids", n, _F32, dev)
        mids = _vector(midpoints, "midpoints", n - 1, _F32, dev)
        _on(rotation, "rotation", _F32, dev)
        if rotation.shape != (HEAD_DIM, HEAD_DIM) or not rotation.is_contiguous():
            _no("rotation must be a contiguous [128, 128] matrix")
        rot = rotation.data_ptr()
    pos = pos64 = table = table_stride = max_pos = rotary = 0
    if positions is not None:
        pos64 = isinstance(positions, torch.Tensor) and positions.dtype is _I64
        pos = _vector(positions, "positions", N, _I64 if pos64 else _I32, dev)
        _on(cos_sin, "cos_sin", _F32, dev)
        if cos_sin.dim() != 2 or cos_sin.stride(1) != 1:
            _no("cos_sin must be [max_pos, rotary_dim] row-major")
        (max_pos, rotary), table_stride, table = cos_sin.shape, cos_sin.stride(0), cos_sin.data_ptr()
        if max_pos == 1:
            table_stride = rotary
    q = out = Hq = 0
    qs = os = (0, 0, 1)
    if query is not None:
        _, qkind, qshape, qs = _float_rows(query, "query", dev)
        if qshape[0] != N or qkind != kind:
            _no(f"query must be [{N}, Hq, 128] in the key's dtype")
        if q_rot is None:
            q_rot = torch.empty(qshape, dtype=_F32, device=query.device)
            os = (qshape[1] * HEAD_DIM, HEAD_DIM)
        else:
            _on(q_rot, "q_rot", _F32, dev)
            os = q_rot.stride()
            if q_rot.shape != qshape or os[2] != 1:
                _no("q_rot must have the query's shape and unit stride over the last dim")
        q, out, Hq = query.data_ptr(), q_rot.data_ptr(), qshape[1]
    elif q_rot is not None:
        _no("q_rot is the output of query")
    _call("tqb_append", _APPEND.pack(
        key.data_ptr(), value.data_ptr(), q, kind, ks[0], ks[1], vs[0], vs[1], qs[0], qs[1], pos, bool(pos64), table,
        table_stride, max_pos, rotary, bool(interleaved), rot, mids, cents, slots, kv_cache.data_ptr(), lay, cs[0], cs[1],
        cs[2], cshape[0], out, os[0], os[1], N, Hq, Hk, HEAD_DIM, BLOCK_SIZE, n, bool(norm_correction) and lay in _FOLDED),
        _stream(dev))
    return q_rot


@_on_stream
def gather_kv(kv_cache: torch.Tensor, slot_mapping: torch.Tensor, centroids: Optional[torch.Tensor], *, layout="soa",
              dtype: torch.dtype = torch.bfloat16, key: Optional[torch.Tensor] = None,
              value: Optional[torch.Tensor] = None, stream: Optional[int] = None):
    """Keys and values ``[N, Hk, 128]`` that the cache holds in ``slot_mapping``'s slots (int32 ``[N]``), in ``dtype``
    (or into ``key``/``value``), one rounding each: what a later chunk of a prefill attends to
    (reference/soa_decode_v1.py:322-454).  Lloyd-Max keys stay in the rotated basis, where the chunk's queries are taken
    too (:func:`rotate_query`).  Rows of negative or out-of-range slots are zeros."""
    lay = layout_id(layout)
    dev, cshape, cs = _cache(kv_cache, lay)
    if not isinstance(slot_mapping, torch.Tensor):
        _no("slot_mapping must be a torch.Tensor")
    N, Hk = slot_mapping.numel(), cshape[2]
    slots = _vector(slot_mapping, "slot_mapping", N, _I32, dev)
    n = 8 if lay in KEY3_LAYOUTS else 16
    cents = 0 if lay in FP8_KEY_LAYOUTS else _vector(centroids, "centroids", n, _F32, dev)
    if key is None and value is None:
        kind = _DTYPE_ID.get(dtype)
        if kind is None:
            _no("dtype must be float32, float16 or bfloat16")
        key = torch.empty((N, Hk, HEAD_DIM), dtype=dtype, device=kv_cache.device)
        value = torch.empty((N, Hk, HEAD_DIM), dtype=dtype, device=kv_cache.device)
        ks = vs = (Hk * HEAD_DIM, HEAD_DIM)
    else:
        _, kind, kshape, ks = _float_rows(key, "key", dev)
        _, vkind, vshape, vs = _float_rows(value, "value", dev)
        if kshape != (N, Hk, HEAD_DIM) or vshape != kshape or kind != vkind:
            _no(f"key and value must be [{N}, {Hk}, 128] tensors of one dtype")
    _call("tqb_gather", _GATHER.pack(
        kv_cache.data_ptr(), lay, cs[0], cs[1], cs[2], cshape[0], slots, cents, key.data_ptr(), value.data_ptr(), kind,
        ks[0], ks[1], vs[0], vs[1], N, Hk, HEAD_DIM, BLOCK_SIZE, n), _stream(dev))
    return key, value


def _splits(items: int, tokens: int, group: int) -> int:
    """Splits of ``tokens`` for ``items`` (sequence, KV head) pairs of ``group`` query heads each.  Stage1 walks tiles of 8
    (item, split) pairs with a group of warps each, two groups to an SM with up to 4 query heads and one with more, so a
    split count that just exceeds a whole round of the groups costs another round: of the counts that fill one to four
    rounds, the one with the least time, a round taking its split's tokens and the start and end of a tile (about 48
    tokens' time).  Splits of the longest sequence that ``tokens`` allows stay above ``_SPLIT_TOKENS`` tokens.

    Measured, us by splits (one round's in brackets): 4 heads, 64 sequences x 8, 1024 tokens: 2 63, [4 44], 5 54, 9 45;
    8 heads, the same: 1 88, [2 57], 3 72, 4 62; 8 heads, 37 x 8, 777 tokens: 3 39, [4 36], 5 46, 8 39; 5 heads, 8 x 8,
    2048 tokens: 14 25, [16 23, 18 26], 20 34, 32 29; 8 heads, 16 x 8, 3000 tokens: 8 36, [9 34], 10 52, 18 38."""
    most = max(1, -(-tokens // _SPLIT_TOKENS))
    round_ = _SMS * (16 if group <= 4 else 8)
    best = (float("inf"), 1)
    for rounds in (1, 2, 3, 4):
        s = min(most, round_ * rounds // items)
        if s:
            used = -(-items * s // round_)
            best = min(best, (used * (-(-tokens // s) + 48), s))
    pages = -(-tokens // BLOCK_SIZE)  # the fewest splits of as many whole pages
    return -(-pages // -(-pages // best[1]))


class _Step:
    """One decode call: its checked arguments, its workspace (rotated queries, split partials, LSE where the caller gives
    none, in one allocation) and its outputs."""

    def __init__(self, query, kv_cache, block_table, seq_lens, rotation, centroids, layout, scale, sinks, output, out_dtype,
                 lse, mid_o):
        self.lay = lay = layout_id(layout)
        dev, self.kind, (self.B, self.Hq, _), self.qs = _float_rows(query, "query")
        self.dev, self.query = dev, query
        _, self.cshape, self.cs = _cache(kv_cache, lay, dev)
        self.cache, self.Hk = kv_cache.data_ptr(), self.cshape[2]
        if self.Hq < 1 or self.Hq % self.Hk:
            _no(f"query heads must be a multiple of the cache's {self.Hk}")
        self.seq_lens = _vector(seq_lens, "seq_lens", self.B, _I32, dev)
        _on(block_table, "block_table", _I32, dev)
        tshape, tstride = block_table.shape, block_table.stride()
        if len(tshape) != 2 or tshape[0] != self.B or tshape[1] < 1 or tstride[1] != 1:
            _no(f"block_table must be [{self.B}, max_blocks] row-major")
        self.table, self.blocks = block_table.data_ptr(), tshape[1]
        self.table_stride = tstride[0] if self.B > 1 else max(tstride[0], tshape[1])
        self.n = 8 if lay in KEY3_LAYOUTS else 16
        self.cents = 0 if lay in FP8_KEY_LAYOUTS else _vector(centroids, "centroids", self.n, _F32, dev)
        self.rot = 0
        if rotation is not None:
            if lay in FP8_KEY_LAYOUTS:
                _no("FP8 keys are not rotated: rotation must be None")
            _on(rotation, "rotation", _F32, dev)
            if rotation.shape != (HEAD_DIM, HEAD_DIM) or not rotation.is_contiguous():
                _no("rotation must be a contiguous [128, 128] matrix")
            self.rot = rotation.data_ptr()
        self.sinks = None if sinks is None else _vector(sinks, "sinks", self.Hq, _F32, dev)
        try:
            self.scale = 1.0 / math.sqrt(HEAD_DIM) if scale is None else float(scale)
        except (TypeError, ValueError, OverflowError):
            _no("scale must be a number")
        if not 0 < self.scale < 2.0 ** 127:
            _no("scale must be positive and an fp32 number")
        if output is None:
            output = torch.empty((self.B, self.Hq, HEAD_DIM), dtype=out_dtype or query.dtype, device=query.device)
            self.os = (self.Hq * HEAD_DIM, HEAD_DIM)
            self.out_kind = _DTYPE_ID.get(output.dtype)
            if self.out_kind is None:
                _no("out_dtype must be float32, float16 or bfloat16")
        else:
            _, self.out_kind, oshape, self.os = _float_rows(output, "output", dev)
            if oshape != query.shape:
                _no("output must have the query's shape")
        self.output = output
        self.lse, self.lse_stride = 0, self.Hq
        if lse is not None:
            _on(lse, "lse", _F32, dev)
            if lse.shape != (self.B, self.Hq) or lse.stride(1) != 1:
                _no(f"lse must be [{self.B}, {self.Hq}] with unit stride over the heads")
            self.lse, self.lse_stride = lse.data_ptr(), lse.stride(0)
        self.mid_o = mid_o
        if mid_o is not None:
            _on(mid_o, "mid_o", _F32, dev)

    def workspace(self, S: int) -> None:
        """Room for S splits; the query rows that Stage1 reads."""
        rows = self.B * self.Hq
        need = 0 if self.mid_o is not None else rows * S * _PITCH
        lse_at, need = need, need + (0 if self.lse else rows)
        q_at = need = (need + 31) // 32 * 32
        # queries that need no rotation are read as they are where Stage1 can (fp32, 16-byte aligned rows)
        q, qs = self.query, self.qs
        direct = not self.rot and q.dtype is _F32 and not (q.data_ptr() | qs[0] * 4 | qs[1] * 4) & 15 and qs[0] >= 0 <= qs[1]
        if not direct and self.rot:
            need += rows * HEAD_DIM
        self.keep = ws = torch.empty(max(need, 1), dtype=_F32, device=q.device)
        base = ws.data_ptr()
        if self.mid_o is None:
            self.mid, self.ms = base, (self.Hq * S * _PITCH, S * _PITCH, _PITCH)
        else:
            m = self.mid_o
            if m.dim() != 4 or m.shape[0] < self.B or m.shape[1] < self.Hq or m.shape[2] < S or \
                    m.shape[3] != HEAD_DIM + 1 or m.stride(3) != 1:
                _no(f"mid_o must hold [{self.B}, {self.Hq}, {S}, 129] partials with unit inner stride")
            self.mid, self.ms = m.data_ptr(), m.stride()
        if not self.lse:
            self.lse = base + 4 * lse_at
        if direct:
            self.rows, self.rs = q.data_ptr(), qs
        elif self.rot:
            self.rows, self.rs = base + 4 * q_at, (self.Hq * HEAD_DIM, HEAD_DIM)
        else:
            self.query = q = torch.empty(q.shape, dtype=_F32, device=q.device).copy_(q)  # fp32 ones too: they are not aligned
            self.rows, self.rs = q.data_ptr(), q.stride()

    def stage1(self, at: int, S: int) -> bytes:
        """Stage1 arguments for S splits from split ``at`` on."""
        ms, rs, cs = self.ms, self.rs, self.cs
        return _STAGE1.pack(
            self.rows, rs[0], rs[1], self.cache, self.lay, cs[0], cs[1], cs[2], self.cshape[0], self.table,
            self.table_stride, self.blocks, self.seq_lens, self.cents, self.n, 0, 0, self.mid + 4 * ms[2] * at, ms[0],
            ms[1], ms[2], self.B, self.Hq, self.Hk, HEAD_DIM, BLOCK_SIZE, S, self.scale)

    def launch(self, rng: bytes, lead: int, S: int, prefix_len: int = 0) -> torch.Tensor:
        """Stage1 of the range into the splits from ``lead`` on, the shared prefix into those before, the merge of all
        S."""
        st = _stream(self.dev)
        ms, rs = self.ms, self.rs
        _call("tqb_stage1_range", self.stage1(lead, S - lead),
              None if not self.rot else _ROTATE.pack(self.query.data_ptr(), self.kind, self.qs[0], self.qs[1], self.rot,
                                                     self.rows, rs[0], rs[1], self.B, self.Hq, HEAD_DIM), rng, st)
        if lead:  # after Stage1, which rotates the queries
            _call("tqb_prefix", self.stage1(0, lead), prefix_len, st)
        out = self.output.data_ptr()
        _call("tqb_stage2_range", _STAGE2.pack(
            self.mid, ms[0], ms[1], ms[2], self.seq_lens, 0, out, self.os[0], self.os[1], self.lse, self.lse_stride,
            self.B, self.Hq, HEAD_DIM, S), rng, lead, self.sinks, self.out_kind, out, st)
        return self.output


def _prefix_splits(rows: int, heads: int, prefix_len: int) -> int:
    """Splits of the shared prefix for ``rows`` queries of each of ``heads`` KV heads: chunks of 128-token tiles that
    fill the SMs in as few rounds as pay (a CTA starts and ends in about the time of three tiles)."""
    tiles, units = -(-prefix_len // 128), heads * -(-rows // 256)
    best = (float("inf"), 1)
    for rounds in (1, 2, 3):
        chunks = min(tiles, _SMS * rounds // units)
        if chunks:
            best = min(best, (rounds * (-(-tiles // chunks) + 3), chunks))
    return best[1] * (2 if rows <= 128 else 1)


def _shares(batch: int, rows: int, heads: int, prefix_len: int) -> bool:
    """Whether one pass over the prefix for all rows is faster than Stage1 of every sequence.  The pass and its extra
    merge cost about 8.5 us before the first tile and, per block of 256 rows, the time that Stage1 takes for the prefix
    of five sequences.  Measured with 8 KV heads and 32 query heads, us, pass : Stage1 at (batch, prefix): (64, 512)
    35.6 : 31.2, (64, 2048) 37.0 : 59.2, (32, 2048) 31.7 : 36.0, (16, 2048) 30.7 : 27.1, (16, 8192) 39.3 : 54.6, (8, 8192)
    39.0 : 37.2, (8, 32768) 75 : 90, (4, 32768) 74 : 57, (64, 32768) 70 : 607."""
    return (batch - 5 * -(-rows // 256)) * prefix_len * heads > 1 << 18 and rows <= 1 << 22


@_on_stream
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

    ``num_splits`` splits share the tokens of the pages that hold a sequence's visible ones; ``mid_o`` may hold their partials: float32
    ``[>= B, >= Hq, >= num_splits, 129]``."""
    window, first_tokens = _int(window, "window"), _int(first_tokens, "first_tokens")
    if window < 1:
        _no("window must be at least 1")
    if first_tokens < 0:
        _no("first_tokens must not be negative")
    num_splits = _split_count(num_splits)
    s = _Step(query, kv_cache, block_table, seq_lens, rotation, centroids, layout, scale, sinks, output, out_dtype, lse,
              mid_o)
    if s.B == 0:
        return s.output
    most = s.blocks * BLOCK_SIZE
    window, first_tokens = min(window, most), min(first_tokens, most)
    S = num_splits or _splits(s.B * s.Hk, min(window + first_tokens, most), s.Hq // s.Hk)
    s.workspace(S)
    return s.launch(_RANGE.pack(window, first_tokens, 0, most), 0, S)


@_on_stream
def prefix_attention(query: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                     rotation: Optional[torch.Tensor], centroids: Optional[torch.Tensor], *, prefix_len: int,
                     scale: Optional[float] = None, layout="soa", sinks: Optional[torch.Tensor] = None,
                     num_splits: Optional[int] = None, output: Optional[torch.Tensor] = None,
                     out_dtype: Optional[torch.dtype] = None, lse: Optional[torch.Tensor] = None,
                     mid_o: Optional[torch.Tensor] = None, stream: Optional[int] = None) -> torch.Tensor:
    """Decode attention ``[B, Hq, 128]`` of a batch whose sequences begin with the same ``prefix_len`` tokens, a
    multiple of 16: the first ``prefix_len / 16`` entries of every row of ``block_table`` are the same pages, of short and
    empty sequences too (the shared pass reads the first row's).  All its tokens are written: a value that is not finite
    may reach every row there, also one that ends before it.
    ``seq_lens`` and ``block_table`` describe whole sequences, prefix included; a sequence shorter than the prefix sees
    its own tokens only.  The other arguments are :func:`window_attention`'s.

    With bf16 outputs, a prefix that is long enough for the batch is read once for all rows, with fp16 operands: it adds
    0.4e-3 to 1.1e-3 of the outputs' rms for scores of a standard deviation of 0.7 to 2.5, 1.9e-3 for 10, beside a bf16
    output's own rounding of 1.65e-3.  A short prefix, and fp16 and fp32 outputs, go sequence by sequence, in fp32.
    ``mid_o`` holds the partials of the prefix too then: ``num_splits + 2 ceil(prefix_len / 128)`` splits are always
    enough.  ``num_splits`` is the splits of each sequence's own tokens; without it their count goes by the block table's
    width, which suits tables of about the longest sequence's length."""
    prefix_len = _int(prefix_len, "prefix_len")
    if prefix_len < 0 or prefix_len % BLOCK_SIZE:
        _no("prefix_len must be a multiple of 16")
    num_splits = _split_count(num_splits)
    s = _Step(query, kv_cache, block_table, seq_lens, rotation, centroids, layout, scale, sinks, output, out_dtype, lse,
              mid_o)
    most = s.blocks * BLOCK_SIZE
    if prefix_len > most:
        _no("the block table's rows do not hold the prefix")
    if s.B == 0:
        return s.output
    lead, rows = 0, s.B * (s.Hq // s.Hk)
    if s.out_kind == _lib.TQB_DTYPE_BF16 and _shares(s.B, rows, s.Hk, prefix_len):
        lead = _prefix_splits(rows, s.Hk, prefix_len)
    else:
        prefix_len = 0
    S = (num_splits or _splits(s.B * s.Hk, max(1, most - prefix_len), s.Hq // s.Hk)) + lead
    s.workspace(S)
    return s.launch(_RANGE.pack(0, 0, prefix_len, most), lead, S, prefix_len)
