"""What the 4-bit cache's binding refuses before the library sees an address, without a GPU."""
import pytest

from tinymetalagent_b200 import runtime as R


def bare_cache(device=-1):
    """A KV4Cache without a library behind it; host tensors pass for the device's (device -1)."""
    import torch
    cache = object.__new__(R.KV4Cache)
    cache.kv_heads, cache.head_dim, cache._device = 2, 64, device
    cache._dtypes = {"float32": torch.float32, "float16": torch.float16, "uint8": torch.uint8}
    return cache


def test_rows_that_share_memory_are_refused():
    """An expanded row has a token stride of 0, which the library reads as contiguous rows: it would read
    n_tokens rows from one row's memory.  Overlapping rows are no layout of the cache's either."""
    import torch
    c = bare_cache()
    row = torch.zeros((1, 128))
    for x in (row.expand(5, 128), torch.zeros((2, 64)).expand(5, 2, 64), torch.zeros((1, 1, 128)).expand(3, 5, 128),
              torch.zeros(1024).as_strided((5, 128), (64, 1)), torch.zeros((3, 1, 128)).expand(3, 5, 128)):
        with pytest.raises(ValueError):
            c._new_rows(x, "k", 3 if x.dim() == 3 and x.shape[0] == 3 else 1, 5, "float32")
    # one token, expanded or not, has no stride
    assert c._new_rows(row.expand(1, 128), "k", 1, 1, "float32") == (row.data_ptr(), 128)


class FakeLibrary:
    """Records the call that would reach the library."""

    def __init__(self):
        self.calls = []

    def te_kv4_append(self, *args):
        self.calls.append(args)
        return R.TE_STATUS_OK


def fake_cache():
    c = bare_cache()
    c.handle, c.lib = 1, FakeLibrary()
    c._c = lambda status: None
    return c, c.lib.calls


def test_append_takes_a_stride_only_with_addresses():
    """A token stride beside tensors has to be the tensors' own: another one walks past their ends or takes the wrong
    rows."""
    import torch
    c, calls = fake_cache()
    k, v = torch.zeros((5, 128)), torch.zeros((5, 128))
    wide = torch.zeros((5, 512))
    for kk, vv, stride in ((k, v, 1024), (k, v, 512), (wide[:, :128], wide[:, 128:256], 1024),
                           (wide[:, :128], wide[:, 128:256], 128), (wide.data_ptr(), v, 512), (k, wide.data_ptr(), 512)):
        with pytest.raises(ValueError):
            c.append(0, 1, 0, kk, vv, 5, token_stride=stride)
    assert calls == []
    c.append(0, 1, 0, k, v, 5, token_stride=128)
    c.append(0, 1, 0, wide[:, :128], wide[:, 128:256], 5, token_stride=512)
    c.append(0, 1, 0, wide.data_ptr(), wide[:, 128:256], 5, token_stride=512)
    c.append(0, 1, 0, wide.data_ptr(), wide.data_ptr() + 512, 5, token_stride=512)
    c.append(0, 1, 0, wide[:, :128], wide[:, 128:256], 5)
    c.append(0, 1, 0, wide.data_ptr(), wide.data_ptr() + 512, 5)
    assert [a[7] for a in calls] == [128, 512, 512, 512, 512, 128]


def test_append_refuses_what_is_no_tensor():
    """Host arrays are refused by type, and a missing operand is the library's to refuse, as in the other calls."""
    import numpy as np
    import torch
    c, calls = fake_cache()
    k = torch.zeros((5, 128))
    for kk, vv in ((np.zeros((5, 128), np.float32), k), (k, np.zeros((5, 128), np.float32))):
        with pytest.raises(TypeError):
            c.append(0, 1, 0, kk, vv, 5)
    assert calls == []
    c.append(0, 1, 0, None, k, 5)
    assert calls[0][4] is None and calls[0][5] == k.data_ptr()
