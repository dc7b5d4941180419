"""The paged 8-bit cache without a GPU: what its entry points refuse, who has which pages, and the plain implementation that the GPU
tests compare with."""

import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from tests import paged_ref


@pytest.fixture(scope="module")
def L():
    from glorcq_b200 import _build, _lib
    _build.build()
    return _lib.lib()


BUF = C.create_string_buffer(4096)
PTR = (C.addressof(BUF) + 255) // 256 * 256


def descriptors(**change):
    from glorcq_b200 import _lib
    kv = _lib.PagedKv(PTR, PTR, PTR, PTR, PTR, 4, _lib.KV_I8, 8, 2, 64, 16, 4)
    rows = _lib.PagedRows(PTR, None, 1, 2, 6, 3)
    for name, value in change.items():
        setattr(kv if hasattr(kv, name) else rows, name, value)
    return kv, rows


def calls(L, kv, rows):
    """status of append, attention and read"""
    k, r = C.byref(kv) if kv else None, C.byref(rows) if rows else None
    return (L.glq_paged_append(k, r, PTR, 256, PTR, 128, PTR, 128, PTR, 256, 4, PTR, PTR, 64, None, None, 1e-6, None),
            L.glq_paged_attention(k, r, PTR, 256, PTR, 256, 4, 0.125, PTR, 1 << 40, None),
            L.glq_paged_read(k, r, PTR, PTR, None))


@pytest.mark.parametrize("change,status", [
    (dict(k_pages=None), -1), (dict(v_pages=None), -1), (dict(k_scale=None), -1), (dict(v_scale=None), -1), (dict(table=None), -1),
    (dict(start=None), -1), (dict(dtype=2), -3), (dict(dtype=-1), -3), (dict(head_dim=96), -3), (dict(head_dim=0), -3), (dict(page=8), -3),
    (dict(page=48), -3), (dict(n_pages=0), -1), (dict(n_kv=0), -1), (dict(max_pages=0), -1), (dict(table_stride=3), -1),
    (dict(max_pages=1 << 26, table_stride=1 << 26), -3), (dict(B=-1), -1), (dict(rows=-2), -1), (dict(rows=7), -1), (dict(start_stride=2), -1),
    (dict(k_pages=PTR + 8), -2), (dict(v_pages=PTR + 4), -2)])
def test_descriptors_are_checked_on_the_host(L, change, status):
    assert calls(L, *descriptors(**change)) == (status,) * 3


def test_arguments_are_checked_on_the_host(L):
    kv, rows = descriptors()
    assert calls(L, None, rows) == calls(L, kv, None) == (-1,) * 3
    k, r = C.byref(kv), C.byref(rows)

    def append(q=PTR, ldq=256, k_=PTR, ldk=128, v=PTR, ldv=128, qo=PTR, ldqo=256, heads=4, cos=PTR, sin=PTR, n=64, qn=None, kn=None):
        return L.glq_paged_append(k, r, q, ldq, k_, ldk, v, ldv, qo, ldqo, heads, cos, sin, n, qn, kn, 1e-6, None)
    for bad in (dict(k_=None), dict(v=None), dict(qo=None), dict(heads=0), dict(cos=None), dict(sin=None), dict(n=63), dict(qn=PTR), dict(kn=PTR),
                dict(ldk=120), dict(ldv=120), dict(ldq=248), dict(ldqo=248)):
        assert append(**bad) == -1, bad
    for bad in (dict(ldk=132), dict(ldv=132), dict(ldq=260), dict(ldqo=260), dict(k_=PTR + 2), dict(q=PTR + 8), dict(qo=PTR + 8), dict(v=PTR + 4),
                dict(cos=PTR + 4, sin=PTR), dict(qn=PTR + 2, kn=PTR)):
        assert append(**bad) == -2, bad

    def attention(q=PTR, ldq=256, out=PTR, ldo=256, heads=4, r=r):
        return L.glq_paged_attention(k, r, q, ldq, out, ldo, heads, 0.125, PTR, 1 << 40, None)
    for bad in (dict(q=None), dict(out=None), dict(heads=0), dict(heads=3), dict(ldq=248), dict(ldo=248)):
        assert attention(**bad) == -1, bad
    for bad in (dict(ldq=260), dict(ldo=260), dict(q=PTR + 8), dict(out=PTR + 8)):
        assert attention(**bad) == -2, bad
    for scale in (-0.125, float("nan"), float("inf")):
        assert L.glq_paged_attention(k, r, PTR, 256, PTR, 256, 4, scale, PTR, 1 << 40, None) == -1, scale
    # rows times tokens that 32 bits do not count
    many = descriptors(max_pages=1 << 25, table_stride=1 << 25, rows=1 << 20, max_new=1 << 20)
    assert L.glq_paged_attention(C.byref(many[0]), C.byref(many[1]), PTR, 256, PTR, 256, 4, 0.125, PTR, 1 << 40, None) == -3
    ragged = descriptors(q_start=PTR, max_new=-1)[1]
    assert attention(r=C.byref(ragged)) == -1
    assert L.glq_paged_read(k, r, None, PTR, None) == L.glq_paged_read(k, r, PTR, None, None) == -1
    assert L.glq_paged_read(k, r, PTR + 8, PTR, None) == -2
    # nothing to do: no launch
    assert calls(L, *descriptors(rows=0)) == calls(L, *descriptors(B=0, rows=0)) == (0,) * 3


def test_native_calls_refuse_what_is_not_on_the_gpu(L):
    from glorcq_b200.paged_cache import paged_append, paged_attention, paged_read
    cache = paged_ref.make_cache(1, "int8", 2, 64, 16, [20], "cpu")
    q, k = torch.zeros(1, 4, 64).half(), torch.zeros(1, 2, 64).half()
    start = torch.tensor([20])
    for call in (lambda: paged_append(q, k, k, None, None, *cache, start), lambda: paged_attention(q, *cache, start),
                 lambda: paged_read(*cache, start, None, 1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="k_pages must be torch.int8 or torch.float8_e4m3fn"):
        paged_attention(q, cache[0].float(), *cache[1:], start)
    with pytest.raises(RuntimeError, match="q must be a tensor"):
        paged_attention(3, *cache, start, scale=1.0)


CONFIG = SimpleNamespace(num_hidden_layers=2, num_key_value_heads=2, head_dim=64, rope_theta=10000.0)


def test_pages_are_handed_out_and_taken_back():
    from glorcq_b200.paged_cache import PagedKVCache
    c = PagedKVCache(CONFIG, 3, 100, "cpu", page_size=16, num_pages=9)
    assert (c.page_table == -1).all() and c.k.shape == (2, 9, 2, 16, 64) and c.cos.shape == (112, 32)
    c.reserve(0, 33)
    c.reserve(2, 96)
    c.reserve(0, 20)                       # has them
    used = [p for row in c.page_table.tolist() for p in row if p >= 0]
    assert len(used) == len(set(used)) == 9 and (c.page_table[0] >= 0).sum() == 3 and (c.page_table[2] >= 0).sum() == 6
    with pytest.raises(RuntimeError, match="1 pages are wanted and 0 are free"):
        c.reserve(1, 1)
    with pytest.raises(RuntimeError, match="more than 112"):
        c.reserve(0, 113)
    c.release(2)
    assert (c.page_table[2] == -1).all()
    c.reserve(1, 90)
    used = [p for row in c.page_table.tolist() for p in row if p >= 0]
    assert len(used) == len(set(used)) == 9
    full = PagedKVCache(CONFIG, 2, 100, "cpu", dtype="e4m3", page_size=32)
    assert (full.page_table >= 0).all() and full.k.dtype == torch.float8_e4m3fn
    with pytest.raises(RuntimeError, match="3 sequences are more than 2"):
        full.layer(0, 3)


@pytest.mark.parametrize("bad", [dict(dtype="fp8"), dict(page_size=8), dict(config=SimpleNamespace(**{**vars(CONFIG), "head_dim": 80}))])
def test_caches_that_the_kernels_do_not_have_are_refused(bad):
    from glorcq_b200.paged_cache import PagedKVCache
    with pytest.raises(RuntimeError, match="paged cache"):
        PagedKVCache(**{**dict(config=CONFIG, max_batch_size=1, max_cache_len=64, device="cpu"), **bad})


def test_rope_tables_keep_far_angles():
    from glorcq_b200.paged_cache import rope_tables
    import math
    cos, sin = rope_tables(64, 131073, 1e6, "cpu")
    for i in (0, 1, 31):
        a = 131072 * 1e6 ** (-2 * i / 64)
        assert abs(cos[131072, i].item() - math.cos(a)) < 1e-7 and abs(sin[131072, i].item() - math.sin(a)) < 1e-7


@pytest.mark.parametrize("dtype", ["int8", "e4m3"])
def test_plain_append_keeps_its_error(dtype):
    """The plain implementation itself: token by token or at once, values are within a code's step of what was appended, also
    where a block's scale was doubled."""
    g = torch.Generator().manual_seed(3)
    cache = paged_ref.make_cache(2, dtype, 1, 32, 16, [0], "cpu", width=3)
    cache[4][0] = torch.tensor([2, 0, 1])
    x = torch.randn(40, 1, 32, generator=g) * torch.logspace(-1, 1, 40)[:, None, None]
    for cuts in ([40], [1] * 40, [3, 30, 7]):
        pages, at = paged_ref.Pages(cache), 0
        for n in cuts:
            pages.append(0, 0, at, x[at:at + n])
            at += n
        for t, v in enumerate(pages.values(0, 0, 0, 40)):
            s = pages.scale[0][pages.phys(0, t // 16), 0]
            # int8: half a step, and as much for each time the scale doubled, halved each time: one step; e4m3: doubling loses only what is subnormal
            tol = (0.5 if len(cuts) == 1 else 1.0) * s if dtype == "int8" else x[t].abs() * 2.0 ** -4 + s * 2.0 ** -9
            assert ((v - x[t]).abs() <= tol * (1 + 1e-5)).all()
