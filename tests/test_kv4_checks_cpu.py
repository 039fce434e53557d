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
