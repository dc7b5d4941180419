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


def test_a_snapshot_leaves_out_what_is_no_page():
    """The page table may hold any number where there is no page; indexing by such a one is an error (on a GPU, a fault)."""
    from glorcq_b200.paged_cache import PagedKVCache
    c = PagedKVCache(CONFIG, 2, 48, "cpu", page_size=16)
    for t in (c.k.view(torch.uint8), c.v.view(torch.uint8)):
        t.copy_(torch.randint(0, 256, t.shape, dtype=torch.uint8))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.rand(t.shape))
    c.page_table[0, 0], c.page_table[1, 1] = c.k.shape[1], 1 << 30
    before = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    kept = c.snapshot(20)
    assert sorted(kept[0].tolist()) == sorted(c.page_table[[0, 1], [1, 0]].tolist())
    for t in (c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale):
        t[:, kept[0]] = 0
    c.restore(kept)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip((c.k, c.v, c.k_scale, c.v_scale), before))
