"""The 4-bit cache without a GPU: null and argument guards of its C entry points, and the binding's own checks."""
import ctypes

import numpy as np
import pytest

from tinymetalagent_b200 import runtime as R

BAD = R.TE_STATUS_INVALID_ARGUMENT


def test_null_guards(lib):
    assert lib.te_kv4_cache_create(None, None, None) == BAD
    lib.te_kv4_cache_free(None)
    assert lib.te_kv4_cache_seq_reset(None, 0, 0) == BAD
    assert lib.te_kv4_cache_seq_truncate(None, 0, 0) == BAD
    assert lib.te_kv4_cache_seq_length(None, 0, None) == BAD
    assert lib.te_kv4_cache_reserve(None, 0, 1) == BAD
    assert lib.te_kv4_cache_set_qkv_bias(None, 0, 1, 8, None, None, None) == BAD
    assert lib.te_kv4_append(None, 0, 1, 0, None, None, 1, 0, None, None, 0) == BAD
    assert lib.te_kv4_cache_read(None, 0, 1, 0, 0, 1, None, None, 0) == BAD
    assert lib.te_kv4_cache_write_q4_0(None, 0, 1, 0, 0, 1, None, None) == BAD
    assert lib.te_kv4_cache_read_q4_0(None, 0, 1, 0, 0, 1, None, None) == BAD
    assert lib.te_kv4_attention_decode(None, 0, 1, None, 1, None, None, None, None, 8, None, 0) == BAD


def bare_cache():
    import torch
    cache = object.__new__(R.KV4Cache)
    cache.kv_heads, cache.head_dim, cache._device = 2, 64, -1  # host tensors pass for the device's here
    cache._dtypes = {"float32": torch.float32, "float16": torch.float16, "uint8": torch.uint8}
    return cache


def test_row_views_the_append_takes():
    import torch
    c = bare_cache()
    wide = torch.zeros((3, 5, 512))
    assert c._new_rows(wide[0, :, 128:256], "k", 1, 5, "float32") == (wide.data_ptr() + 512, 512)
    assert c._new_rows(wide[:, :, :128], "k", 3, 5, "float32") == (wide.data_ptr(), 512)
    assert c._new_rows(torch.zeros((3, 5, 2, 64)), "k", 3, 5, "float32")[1] == 128
    heads = torch.zeros((5, 7, 64))
    assert c._new_rows(heads[:, 2:4], "k", 1, 5, "float32") == (heads.data_ptr() + 2 * 64 * 4, 448)
    assert c._new_rows(wide[:, :1, :128], "k", 3, 1, "float32")[1] == 5 * 512
    for x in (wide[:, :4, :128],                       # layers not evenly spaced after 4 of 5 tokens
              wide[0, :, 0:256:2],                     # a row's values are not contiguous
              torch.zeros((5, 64, 2)).transpose(1, 2),  # rows transposed
              wide[0, :, :64],                         # half a row
              wide[0, :3, :128]):                      # too few rows
        with pytest.raises(ValueError):
            c._new_rows(x, "k", 3 if x.dim() == 3 and x.shape[0] == 3 else 1, 5, "float32")
    with pytest.raises(ValueError):
        c._new_rows(wide[0, :, :128].half(), "k", 1, 5, "float32")


def test_tensor_checks_of_the_binding():
    import torch
    c = bare_cache()
    x = torch.zeros((4, 128))
    assert c._tensor(x, "x", 512, "float32") == x.data_ptr()
    assert c._tensor(None, "x", 512, "float32") is None and c._tensor(1234, "x", 512, "float32") == 1234
    for args in ((x, "x", 511, "float32"), (x, "x", 512, "float16"), (x.T, "x", 512, "float32")):
        with pytest.raises(ValueError):
            c._tensor(*args)
    c._device = 0
    with pytest.raises(ValueError):
        c._tensor(x, "x", 512, "float32")
    with pytest.raises(TypeError):
        c._tensor(np.zeros(512, np.float32), "x", 512, "float32")


def test_bias_shapes_are_checked_before_the_library():
    c = bare_cache()
    with pytest.raises(ValueError):
        c.set_qkv_bias(0, 8, np.zeros((2, 8 * 64 + 1), np.float32))
    with pytest.raises(ValueError):
        c.set_qkv_bias(0, 8)


def test_flag_value():
    import re
    from pathlib import Path
    text = (Path(__file__).resolve().parents[1] / "include" / "tinyengine_attn.h").read_text()
    assert int(re.search(r"#define TE_ATTN_OUTPUT_F16\s+\(1u << (\d+)\)", text).group(1)) == 11
    assert R.TE_ATTN_OUTPUT_F16 == 1 << 11
    assert ctypes.sizeof(R.KVCacheDesc) == 40
