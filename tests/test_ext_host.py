"""Refusals and host-side arithmetic of the extended cache operators (no GPU)."""

from __future__ import annotations

import ctypes
import re
import subprocess

import numpy as np
import pytest
import torch

from _ops64 import F8, e4m3, needed_scale
from conftest import REPO
from llm_serving_runtime_b200 import _lib
from llm_serving_runtime_b200.device_pages import _view
from llm_serving_runtime_b200.paged_attention import describe_device_errors, device_error
from llm_serving_runtime_b200.score_modifiers import ScoreModifiers


def test_the_plain_e4m3_rounding_is_torchs():
    x = torch.cat([torch.linspace(-500, 500, 20001), torch.randn(20000) * 0.01, torch.tensor([2.0**-10, 3 * 2.0**-10])])
    x = x.clamp(-448, 448)
    assert np.array_equal(e4m3(x.numpy()), x.to(F8).double().numpy())


@pytest.mark.parametrize("top,e", [(448.0, 0), (448.1, 1), (1.75, -8), (1.76, -7), (0.0, -100), (3.3e38, 120)])
def test_the_plain_scale(top, e):
    assert needed_scale(np.array([top, -top / 2, np.inf, np.nan], dtype=np.float32)) == np.float32(2.0**e)


_PROBE = r"""
#include <stdio.h>
#include <stddef.h>
#include "paged_attention_b200.h"
#define F(T, f) printf(#T "." #f " %zu\n", offsetof(T, f));
#define S(T) printf(#T " %zu\n", sizeof(T));
int main(void) {
  S(pa_cache_scales) F(pa_cache_scales, value_scales) F(pa_cache_scales, value_stride_head)
  S(pa_score_modifiers) F(pa_score_modifiers, window) F(pa_score_modifiers, alibi_slopes)
  F(pa_score_modifiers, key_starts) F(pa_score_modifiers, key_starts_stride_t) F(pa_score_modifiers, prefix_lens)
  S(pa_page_view) F(pa_page_view, segment_bytes)
  S(pa_page_tables) F(pa_page_tables, num_seqs) F(pa_page_tables, seq_lens) F(pa_page_tables, num_blocks)
  F(pa_page_tables, scratch) F(pa_page_tables, error_flags)
  return 0;
}
"""


def test_struct_layouts(tmp_path):
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text(_PROBE)
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    classes = {"pa_cache_scales": _lib.CacheScalesArgs, "pa_score_modifiers": _lib.ScoreModifiersArgs,
               "pa_page_view": _lib.PageViewArgs, "pa_page_tables": _lib.PageTablesArgs}
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n"):
        if not line:
            continue
        key, val = line.rsplit(" ", 1)
        struct, _, field = key.partition(".")
        cls = classes[struct]
        assert (getattr(cls, field).offset if field else ctypes.sizeof(cls)) == int(val), key
    text = (REPO / "include" / "paged_attention_b200.h").read_text()
    assert int(re.search(r"#define PA_MAX_PAGE_VIEWS (\d+)", text).group(1)) == _lib.PA_MAX_PAGE_VIEWS


def _decode_args():
    a = _lib.DecodeArgs()
    a.batch, a.q_len, a.num_q_heads, a.num_kv_heads = 1, 1, 8, 2
    a.head_dim, a.block_size, a.dtype = 64, 16, _lib.PA_DTYPE_BFLOAT16
    return a


def test_ext_argument_errors():
    lib = _lib.load()
    a, sc, sm = _decode_args(), _lib.CacheScalesArgs(), _lib.ScoreModifiersArgs()
    assert lib.pa_decode_ext(None, None, None, None, None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert lib.pa_decode_ext(ctypes.byref(a), ctypes.byref(sc), None, None, None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert "key_scales" in _lib.last_error()
    sc.key_scales = sc.value_scales = 256
    a.dtype = _lib.PA_DTYPE_FLOAT32
    assert lib.pa_decode_ext(ctypes.byref(a), ctypes.byref(sc), None, None, None) == _lib.PA_ERR_UNSUPPORTED
    a.dtype = _lib.PA_DTYPE_BFLOAT16
    for cap in (-1.0, float("nan"), float("inf")):
        sm.softcap = cap
        assert lib.pa_decode_ext(ctypes.byref(a), None, ctypes.byref(sm), None, None) == _lib.PA_ERR_INVALID_ARGUMENT
        assert "softcap" in _lib.last_error()
    sm.softcap, sm.window = 0.0, -1
    assert lib.pa_decode_ext(ctypes.byref(a), None, ctypes.byref(sm), None, None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert "window" in _lib.last_error()
    a.batch, sm.window = 0, 0
    assert lib.pa_decode_ext(ctypes.byref(a), ctypes.byref(sc), ctypes.byref(sm), None, None) == _lib.PA_OK


def _append_args(**kw):
    a = _lib.KvAppendArgs()
    a.key = a.value = 4096
    for v in (a.key_cache, a.value_cache):
        v.data, v.num_blocks, v.stride_block, v.stride_head, v.stride_token = 8192, 4, 2048, 1024, 64
    a.slot_mapping = 4096
    a.batch, a.q_len, a.num_kv_heads, a.head_dim, a.block_size, a.dtype = 1, 1, 2, 64, 16, _lib.PA_DTYPE_BFLOAT16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,word", [({"head_dim": 72}, "multiple of 16"), ({"block_size": 24}, "power-of-two"),
                                         ({"block_size": 4}, "power-of-two"), ({"block_size": 512}, "power-of-two"),
                                         ({"batch": 1 << 20, "q_len": 1 << 12}, "too large"),
                                         ({"dtype": 3}, "dtype"), ({"key": None}, "key and value")])
def test_append8_argument_errors(change, word):
    lib = _lib.load()
    sc = _lib.CacheScalesArgs()
    sc.key_scales = sc.value_scales = 4096
    a = _append_args(**change)
    assert lib.pa_kv_append_8bit(ctypes.byref(a), ctypes.byref(sc), None) in (_lib.PA_ERR_UNSUPPORTED,
                                                                              _lib.PA_ERR_INVALID_ARGUMENT)
    assert word in _lib.last_error()


def test_append8_alignment_and_nulls():
    lib = _lib.load()
    sc = _lib.CacheScalesArgs()
    a = _append_args()
    assert lib.pa_kv_append_8bit(ctypes.byref(a), None, None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert lib.pa_kv_append_8bit(ctypes.byref(a), ctypes.byref(sc), None) == _lib.PA_ERR_INVALID_ARGUMENT
    sc.key_scales = sc.value_scales = 4096
    a.value_cache.stride_token = 72
    assert lib.pa_kv_append_8bit(ctypes.byref(a), ctypes.byref(sc), None) == _lib.PA_ERR_UNSUPPORTED
    a.value_cache.stride_token = 64
    a.key_cache.data = 8200
    assert lib.pa_kv_append_8bit(ctypes.byref(a), ctypes.byref(sc), None) == _lib.PA_ERR_UNSUPPORTED
    assert lib.pa_kv_append_8bit(ctypes.byref(_append_args(batch=0)), ctypes.byref(sc), None) == _lib.PA_OK


def test_page_argument_errors():
    lib = _lib.load()
    t = _lib.PageTablesArgs(4096, 8, 4, 8, 4096, 4096, 16, 16, 4096, None)
    views = (_lib.PageViewArgs * 9)()
    word = ctypes.c_int32()
    assert lib.pa_pages_free(None, None, 0, None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert lib.pa_pages_free(ctypes.byref(t), None, 1, None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert lib.pa_pages_free(ctypes.byref(t), 4096, 5, None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert lib.pa_pages_free(ctypes.byref(t), None, 0, None) == _lib.PA_OK
    assert lib.pa_pages_fork(ctypes.byref(t), 4096, 4096, 1, views, 9, None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert lib.pa_pages_reserve(ctypes.byref(t), 4096, None, 1, None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert lib.pa_pages_compact(ctypes.byref(t), None, 0, None, None) == _lib.PA_ERR_INVALID_ARGUMENT
    views[0].segments, views[0].segment_bytes = 1, -4
    assert lib.pa_pages_copy(views, 1, 16, 4096, 4096, 1, None, None) == _lib.PA_ERR_INVALID_ARGUMENT
    views[0].segment_bytes = 1 << 30
    views[0].data = 4096
    assert lib.pa_pages_copy(views, 1, 16, 4096, 4096, 1, None, None) == _lib.PA_ERR_UNSUPPORTED
    views[0].segment_bytes = 64
    assert lib.pa_pages_copy(views, 1, 16, None, None, 0, None, None) == _lib.PA_OK
    assert lib.pa_pages_copy(views, 1, 16, None, None, 2, None, None) == _lib.PA_ERR_INVALID_ARGUMENT
    t.block_table_stride = 7
    assert lib.pa_pages_free(ctypes.byref(t), 4096, 1, None) == _lib.PA_ERR_INVALID_ARGUMENT
    t.block_table_stride, t.scratch = 8, None
    assert lib.pa_pages_compact(ctypes.byref(t), None, 0, ctypes.addressof(word), None) == _lib.PA_ERR_INVALID_ARGUMENT
    assert lib.pa_pages_scratch_words(4, 16) == 3 * 4 + 2 * 16 + 8
    assert lib.pa_pages_scratch_words(0, 16) == 0


def _fields(t):
    v = _view(t)
    return v.stride_block, v.segments, v.stride_segment, v.segment_bytes


def test_page_views():
    pool = torch.zeros(10, 4, 2, 16, 64, dtype=torch.bfloat16)
    assert _fields(pool) == (4 * 2 * 16 * 64 * 2, 1, 0, 4 * 2 * 16 * 64 * 2)
    assert _fields(pool[:, 1]) == (4 * 2 * 16 * 64 * 2, 1, 0, 2 * 16 * 64 * 2)
    assert _fields(pool[:, ::2]) == (4 * 2 * 16 * 64 * 2, 2, 2 * 2 * 16 * 64 * 2, 2 * 16 * 64 * 2)
    assert _fields(pool[:, :, :, :8]) == (4 * 2 * 16 * 64 * 2, 8, 16 * 64 * 2, 8 * 64 * 2)
    assert _fields(torch.zeros(10, 3)) == (12, 1, 0, 12)
    assert _fields(torch.zeros(10)) == (4, 1, 0, 4)
    assert _fields(torch.zeros(10, 6, 4).transpose(1, 2)) == (96, 1, 0, 96)  # another order, the same bytes
    # stored layer by layer: a page is a run of each layer, the pages interleave
    assert _fields(torch.zeros(4, 10, 6).transpose(0, 1)) == (24, 4, 240, 24)
    with pytest.raises(ValueError, match="overlap"):
        _view(torch.zeros(400).as_strided((10, 4, 6), (6, 50, 1)))
    with pytest.raises(ValueError, match="one strided"):
        _view(torch.zeros(10, 4, 8, 8)[:, ::2, ::2, ::2])
    with pytest.raises(ValueError, match="overlap"):
        _view(torch.zeros(1, 3).expand(5, 3))
    with pytest.raises(ValueError, match="overlap"):
        _view(torch.zeros(5, 1, 3).expand(5, 4, 3))


def test_score_modifier_refusals():
    dev = torch.device("cpu")

    def args(**kw):
        return ScoreModifiers(**kw).to_args(2, 4, 3, dev)

    for bad in ({"softcap": -1.0}, {"softcap": float("nan")}, {"softcap": float("inf")}, {"softcap": 1e-31}, {"window": -1},
                {"window": 2**31}, {"alibi_slopes": torch.zeros(3)}, {"alibi_slopes": torch.zeros(4).double()},
                {"alibi_slopes": torch.zeros(8)[::2]}, {"key_starts": torch.zeros(2)},
                {"key_starts": torch.zeros(2, 2, dtype=torch.int32)}, {"key_starts": torch.zeros(3, dtype=torch.int32)},
                {"prefix_lens": torch.zeros(2)}, {"prefix_lens": torch.zeros(4, dtype=torch.int32)[::2]}):
        with pytest.raises(ValueError):
            args(**bad)
    a = args(softcap=30.0, window=7, key_starts=torch.zeros(2, 3, dtype=torch.int32))
    assert (a.softcap, a.window, a.key_starts_stride_b, a.key_starts_stride_t) == (30.0, 7, 3, 1)
    a = args(key_starts=torch.zeros(2, dtype=torch.int32))
    assert (a.key_starts_stride_b, a.key_starts_stride_t) == (1, 0)
    half = ScoreModifiers(key_starts=torch.arange(6).reshape(2, 3).int(), prefix_lens=torch.tensor([4, 5]).int()).rows(1, 2)
    assert half.key_starts.tolist() == [[3, 4, 5]] and half.prefix_lens.tolist() == [5]


def test_error_texts():
    assert "two places" in describe_device_errors(_lib.PA_DEVERR_BLOCK_CONFLICT)
    assert isinstance(device_error(_lib.PA_DEVERR_BLOCK_CONFLICT), IndexError)
    assert isinstance(device_error(_lib.PA_DEVERR_SEQUENCE), IndexError)
    assert isinstance(device_error(_lib.PA_DEVERR_PAGES_EXHAUSTED), RuntimeError)
