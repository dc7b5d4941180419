"""The paged 8-bit cache without a GPU: what its host code does where something is wrong."""

from types import SimpleNamespace

import pytest
import torch

CONFIG = SimpleNamespace(num_hidden_layers=2, num_key_value_heads=2, head_dim=64, rope_theta=10000.0)


@pytest.fixture(scope="module")
def L():
    from glorcq_b200 import _build, _lib
    _build.build()
    return _lib.lib()


class FakeDevice:
    """torch.cuda.device without a GPU"""

    def __init__(self, device):
        pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


def test_a_wait_that_ran_out_is_raised(L, monkeypatch):
    """The library's word is replaced by one that a kernel would have left."""
    from glorcq_b200 import _lib
    from glorcq_b200.paged_cache import PagedKVCache
    words = [[131, 5, 1, (7 << 32) | 64], [0, 0, 0, 0]]

    def error(out, clear):
        assert clear
        out[:] = words[0]
        words.pop(0)
        return 0
    monkeypatch.setattr(_lib, "lib", lambda: SimpleNamespace(glq_paged_error=error))
    monkeypatch.setattr(torch.cuda, "device", FakeDevice)
    c = PagedKVCache(CONFIG, 1, 32, "cpu", page_size=16)
    with pytest.raises(RuntimeError, match="code 131, thread 64 of block 7"):
        c.raise_on_error()
    c.raise_on_error()
    assert L.glq_paged_error(None, 1) == -1
