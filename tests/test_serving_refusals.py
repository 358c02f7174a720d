"""What the serving entry points refuse, on the host, before anything is launched (CPU only)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import tqb
from tqb import _build, _lib


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return _lib.load()


def append_args(**kw):
    a = _lib.AppendArgs()
    a.num_tokens, a.num_kv_heads, a.head_dim, a.block_size, a.n_centroids = 1, 2, 128, 16, 16
    for name in ("key", "value", "rotation", "midpoints", "centroids", "slot_mapping", "kv_cache"):
        setattr(a, name, 0x1000)
    a.cache_stride_block = 16 * 2 * 134
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,status", [
    (dict(head_dim=64), _lib.TQB_ERR_UNSUPPORTED), (dict(block_size=32), _lib.TQB_ERR_UNSUPPORTED),
    (dict(layout=9), _lib.TQB_ERR_INVALID_ARG), (dict(dtype=5), _lib.TQB_ERR_INVALID_ARG),
    (dict(n_centroids=8), _lib.TQB_ERR_UNSUPPORTED), (dict(num_tokens=-1), _lib.TQB_ERR_INVALID_ARG),
    (dict(layout=_lib.TQB_LAYOUT_SOA_K8, norm_correction=1), _lib.TQB_ERR_INVALID_ARG),
    (dict(positions=0x1000, rotary_dim=129, max_pos=4, cos_sin_stride=130), _lib.TQB_ERR_INVALID_ARG),
    (dict(positions=0x1000, rotary_dim=130, max_pos=4, cos_sin_stride=130), _lib.TQB_ERR_INVALID_ARG),
    (dict(positions=0x1000, rotary_dim=64, max_pos=0, cos_sin_stride=64), _lib.TQB_ERR_INVALID_ARG),
    (dict(positions=0x1000, rotary_dim=64, max_pos=4, cos_sin_stride=63), _lib.TQB_ERR_INVALID_ARG),
    (dict(positions=0x1000, rotary_dim=64, max_pos=4, cos_sin_stride=64), _lib.TQB_ERR_INVALID_ARG),  # no table
    (dict(positions=0x1004, positions_are_64=1, rotary_dim=64, max_pos=4, cos_sin_stride=64, cos_sin=0x1000),
     _lib.TQB_ERR_ALIGNMENT),
    (dict(query=0x1000), _lib.TQB_ERR_INVALID_ARG), (dict(query=0x1000, num_q_heads=4), _lib.TQB_ERR_INVALID_ARG),
    (dict(key=0), _lib.TQB_ERR_INVALID_ARG), (dict(slot_mapping=0), _lib.TQB_ERR_INVALID_ARG),
    (dict(dtype=_lib.TQB_DTYPE_F32, key=0x1002), _lib.TQB_ERR_ALIGNMENT), (dict(rotation=0x1008), _lib.TQB_ERR_ALIGNMENT),
    (dict(kv_cache=0x1001), _lib.TQB_ERR_ALIGNMENT), (dict(cache_stride_block=16 * 2 * 134 - 2), _lib.TQB_ERR_INVALID_ARG),
    (dict(layout=_lib.TQB_LAYOUT_AOS, cache_stride_pos=134, cache_stride_head=134), _lib.TQB_ERR_INVALID_ARG),
    (dict(num_tokens=2 ** 30, num_kv_heads=2), _lib.TQB_ERR_UNSUPPORTED)])
def test_append(lib, kw, status):
    assert lib.tqb_append(ctypes.byref(append_args(**kw)), None) == status


def test_append_null_and_empty(lib):
    assert lib.tqb_append(None, None) == _lib.TQB_ERR_INVALID_ARG
    assert lib.tqb_append(ctypes.byref(append_args(num_tokens=0, key=0)), None) == _lib.TQB_OK


@pytest.mark.parametrize("kw,status", [
    (dict(head_dim=64), _lib.TQB_ERR_UNSUPPORTED), (dict(block_size=8), _lib.TQB_ERR_UNSUPPORTED),
    (dict(layout=-1), _lib.TQB_ERR_INVALID_ARG), (dict(out_dtype=3), _lib.TQB_ERR_INVALID_ARG),
    (dict(layout=_lib.TQB_LAYOUT_AOS_K3), _lib.TQB_ERR_UNSUPPORTED), (dict(key=0), _lib.TQB_ERR_INVALID_ARG),
    (dict(centroids=0), _lib.TQB_ERR_INVALID_ARG), (dict(key=0x1002), _lib.TQB_ERR_ALIGNMENT),
    (dict(cache_stride_block=1000), _lib.TQB_ERR_INVALID_ARG)])
def test_gather(lib, kw, status):
    a = _lib.GatherArgs()
    a.num_tokens, a.num_kv_heads, a.head_dim, a.block_size, a.n_centroids = 1, 2, 128, 16, 16
    for name in ("key", "value", "centroids", "slot_mapping", "kv_cache"):
        setattr(a, name, 0x1000)
    a.cache_stride_block = 16 * 2 * 134
    for k, v in kw.items():
        setattr(a, k, v)
    assert lib.tqb_gather(ctypes.byref(a), None) == status
    a.num_tokens = 0
    assert lib.tqb_gather(None, None) == _lib.TQB_ERR_INVALID_ARG


def stage1_args():
    a = _lib.Stage1Args()
    a.batch, a.num_q_heads, a.num_kv_heads, a.head_dim, a.block_size, a.n_centroids, a.num_splits = 1, 4, 1, 128, 16, 16, 4
    for name in ("q_rot", "kv_cache", "block_table", "seq_lens", "centroids", "mid_o"):
        setattr(a, name, 0x1000)
    a.q_stride_b, a.q_stride_h = 512, 128
    a.cache_stride_block = 16 * 134
    a.block_table_stride = a.max_blocks_per_seq = 8
    a.mid_stride_b, a.mid_stride_h, a.mid_stride_s = 4 * 4 * 129, 4 * 129, 129
    return a


@pytest.mark.parametrize("rng,splits", [
    ((-1, 0, 0, 128), 4), ((8, -1, 0, 128), 4), ((8, 0, -16, 128), 4), ((8, 0, 0, 0), 4), ((8, 0, 0, 129), 4),
    ((8, 4, 16, 128), 4), ((8, 0, 8, 128), 4)])
def test_ranges(lib, rng, splits):
    a = stage1_args()
    a.num_splits = splits
    assert lib.tqb_stage1_range(ctypes.byref(a), None, ctypes.byref(_lib.RangeArgs(*rng)), None) == _lib.TQB_ERR_INVALID_ARG


def test_ranged_calls(lib):
    a, ok = stage1_args(), _lib.RangeArgs(8, 0, 0, 128)
    assert lib.tqb_stage1_range(ctypes.byref(a), None, None, None) == _lib.TQB_ERR_INVALID_ARG
    a.num_splits_per_seq = 0x1000
    assert lib.tqb_stage1_range(ctypes.byref(a), None, ctypes.byref(ok), None) == _lib.TQB_ERR_INVALID_ARG
    b = _lib.Stage2Args()
    b.batch, b.num_q_heads, b.head_dim, b.num_splits = 1, 4, 128, 4
    b.mid_o = b.seq_lens = b.lse = 0x1000
    for lead in (-1, 4):
        assert lib.tqb_stage2_range(ctypes.byref(b), ctypes.byref(ok), lead, None, 0, 0x1000, None) == _lib.TQB_ERR_INVALID_ARG
    assert lib.tqb_stage2_range(ctypes.byref(b), ctypes.byref(ok), 0, None, 7, 0x1000, None) == _lib.TQB_ERR_INVALID_ARG


def test_python_calls_refuse_host_tensors_and_bad_numbers():
    q, cache = torch.zeros(1, 4, 128), torch.zeros(2, 16, 1, 134, dtype=torch.uint8)
    table, lens, slots = (torch.zeros(s, dtype=torch.int32) for s in ((1, 2), (1,), (1,)))
    for call in (lambda: tqb.window_attention(q, cache, table, lens, None, None, window=0),
                 lambda: tqb.window_attention(q, cache, table, lens, None, None, window=4, first_tokens=-1),
                 lambda: tqb.window_attention(q, cache, table, lens, None, None, window=4, num_splits=0),
                 lambda: tqb.window_attention(q, cache, table, lens, None, None, window=4),
                 lambda: tqb.prefix_attention(q, cache, table, lens, None, None, prefix_len=8),
                 lambda: tqb.prefix_attention(q, cache, table, lens, None, None, prefix_len=-16),
                 lambda: tqb.prefix_attention(q, cache, table, lens, None, None, prefix_len=16),
                 lambda: tqb.gather_kv(cache, slots, None),
                 lambda: tqb.rope_append(q[:, :1], q[:, :1], cache, slots, None, None, None, None, None)):
        with pytest.raises(tqb.TqbError):
            call()


def test_structs_match_the_header(tmp_path):
    import subprocess

    from conftest import ROOT

    structs = {"tqb_range": _lib.RangeArgs, "tqb_append_args": _lib.AppendArgs, "tqb_gather_args": _lib.GatherArgs}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "tqb.h"', "int main(void) {"]
    for c, py in structs.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", "-I/usr/local/cuda/include", str(src), "-o", str(exe)],
                   check=True)
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for c, py in structs.items():
        assert int(got[c]) == ctypes.sizeof(py), c
        for f, _ in py._fields_:
            assert int(got[f"{c}.{f}"]) == getattr(py, f).offset, f"{c}.{f}"
