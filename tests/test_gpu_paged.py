"""The paged 8-bit cache on the GPU against its plain implementation (tests/paged_ref.py): codes and scales equal where no sum's order
decides, attention within a bound that counts the kernel's roundings."""

import math

import pytest
import torch

from tests import paged_ref
from tests.paged_ref import Pages, make_cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    from glorcq_b200 import _build
    _build.build()
    return torch.device("cuda:0")


def i64(v, dev):
    return torch.tensor(v, dtype=torch.int64, device=dev)


def q_starts(new, dev, at=0):
    return torch.tensor([at + sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=dev)


def tables(D, n, dev):
    from glorcq_b200.paged_cache import rope_tables
    return rope_tables(D, n, 10000.0, dev)


def check_attention(got, cache, start, new, q, rows=None, scale=None):
    """rows: first row of each sequence (as by their numbers)"""
    pages = Pages(cache)
    at = 0
    for b, n in enumerate(new):
        r = at if rows is None else rows[b]
        ref, tol = paged_ref.attention(pages, b, min(max(start[b], 0), pages.table.shape[1] * pages.P), q[r:r + n].cpu(), scale)
        err = (got[r:r + n].cpu().double() - ref).abs()
        assert (err <= tol).all(), f"sequence {b}: {(err / tol.clamp(min=1e-30)).max()} of the bound"
        at += n
    from glorcq_b200 import tiled
    assert tiled.debug_error() is None          # no wait ran out


# ---- attention -----------------------------------------------------------------------------------------------------------

DECODE = [  # dtype, heads, kv heads, D, page, tokens held
    ("int8", 16, 16, 128, 64, [512]), ("e4m3", 32, 8, 128, 32, [0, 1, 15, 16, 17, 255, 700]), ("int8", 32, 4, 128, 16, [129, 3, 1000]),
    ("e4m3", 8, 1, 128, 128, [2500]), ("int8", 3, 1, 64, 16, [0, 40]), ("e4m3", 5, 5, 64, 64, [100, 63]), ("int8", 14, 2, 64, 32, [333]),
    ("e4m3", 16, 1, 128, 64, [90, 5]), ("int8", 24, 1, 64, 16, [77]), ("int8", 6, 2, 256, 64, [65, 300]), ("e4m3", 24, 2, 256, 128, [130]),
    ("int8", 4, 2, 32, 16, [0, 63]), ("e4m3", 9, 1, 32, 32, [200]), ("int8", 2, 1, 128, 64, [9000]), ("e4m3", 8, 8, 128, 16, [64] * 70)]


@pytest.mark.parametrize("dtype,heads,kv,D,P,held", DECODE)
def test_attention_of_a_decoded_token(dev, dtype, heads, kv, D, P, held):
    from glorcq_b200.paged_cache import paged_attention
    cache = make_cache(len(held) + heads, dtype, kv, D, P, [n + 1 for n in held], dev)
    q = torch.randn(len(held), heads, D, generator=torch.Generator().manual_seed(D)).half().to(dev)
    got = paged_attention(q, *cache, i64(held, dev))
    check_attention(got, cache, held, [1] * len(held), q)
    assert torch.equal(got, paged_attention(q, *cache, i64(held, dev)))
    # a table with room for long sequences: the work is shared out evenly instead of a cluster taking a sequence and head
    long = wide(cache, 40000)
    got = paged_attention(q, *long, i64(held, dev))
    check_attention(got, cache, held, [1] * len(held), q)
    assert torch.equal(got, paged_attention(q, *long, i64(held, dev)))


MUCH = 1 << 22              # tokens of room at which more than 32 rows a head go to the kernel of prompts, however few


def wide(cache, tokens):
    """The cache with a table of that many tokens a sequence, the new places empty: kernels are chosen by its room."""
    table = torch.full((cache[4].shape[0], tokens // cache[0].shape[2] + 1), -1, dtype=torch.int32, device=cache[4].device)
    table[:, : cache[4].shape[1]] = cache[4]
    return [*cache[:4], table]


CHUNKS = [  # dtype, heads, kv heads, D, page, held, new
    ("int8", 4, 2, 128, 16, [0], [1]), ("e4m3", 8, 2, 128, 64, [0, 100], [64, 3]), ("int8", 4, 4, 128, 32, [7, 0, 50], [130, 0, 1]),
    ("e4m3", 16, 1, 128, 16, [33, 250], [9, 17]), ("int8", 8, 8, 64, 128, [0, 190], [200, 65]), ("e4m3", 6, 2, 64, 16, [1, 300], [31, 129]),
    ("int8", 7, 1, 128, 64, [600], [19]), ("e4m3", 4, 2, 256, 32, [0, 40], [33, 70]), ("int8", 4, 2, 32, 16, [10, 0], [90, 2]),
    ("int8", 2, 1, 128, 64, [1500], [300]), ("e4m3", 12, 1, 64, 32, [0], [257]), ("int8", 4, 1, 128, 128, [0, 5, 9, 0], [2, 2, 4, 0])]


@pytest.mark.parametrize("dtype,heads,kv,D,P,held,new", CHUNKS)
def test_attention_of_several_tokens(dev, dtype, heads, kv, D, P, held, new):
    from glorcq_b200.paged_cache import paged_attention
    cache = make_cache(heads + P, dtype, kv, D, P, [a + n for a, n in zip(held, new)], dev)
    q = torch.randn(sum(new), heads, D, generator=torch.Generator().manual_seed(D)).half().to(dev)
    got = paged_attention(q, *cache, i64(held, dev), q_starts(new, dev), max_new=max(new))
    check_attention(got, cache, held, new, q)
    assert torch.equal(got, paged_attention(q, *cache, i64(held, dev), q_starts(new, dev), max_new=max(new)))
    # the most rows of a sequence not told: perhaps another kernel
    check_attention(paged_attention(q, *cache, i64(held, dev), q_starts(new, dev)), cache, held, new, q)
    for room in (40000, MUCH):
        check_attention(paged_attention(q, *wide(cache, room), i64(held, dev), q_starts(new, dev), max_new=max(new)), cache, held, new, q)
    if len(set(new)) == 1:
        assert torch.equal(got, paged_attention(q, *cache, i64(held, dev)))


@pytest.mark.parametrize("dtype,D", [("e4m3", 128), ("int8", 64), ("int8", 256)])
def test_blocks_with_one_tile_of_rows_and_with_two_in_turn(dev, dtype, D):
    """Sequences whose last block of 256 rows has rows in its first tile alone, for many steps, and then blocks that have both: the results are
    right and the same every time."""
    from glorcq_b200.paged_cache import paged_attention
    held, new = [700, 1500, 300, 900, 1300, 0], [40, 90, 31, 100, 20, 70]
    cache = make_cache(D, dtype, 4, D, 16, [a + n for a, n in zip(held, new)], dev)
    q = torch.randn(sum(new), 16, D, generator=torch.Generator().manual_seed(D)).half().to(dev)
    want = paged_attention(q, *cache, i64(held, dev), q_starts(new, dev), max_new=max(new))
    check_attention(want, cache, held, new, q)
    many = 24                                        # the sequences again and again: every CTA has several blocks
    table, q = cache[4].repeat(many, 1), q.repeat(many, 1, 1)
    first = paged_attention(q, *cache[:4], table, i64(held * many, dev), q_starts(new * many, dev), max_new=max(new))
    for _ in range(10):
        assert torch.equal(first, paged_attention(q, *cache[:4], table, i64(held * many, dev), q_starts(new * many, dev), max_new=max(new)))
    for i in (0, 7, many - 1):
        check_attention(first[i * sum(new):(i + 1) * sum(new)], cache, held, new, q[:sum(new)])


@pytest.mark.parametrize("heads,D,new", [(4, 128, 1), (2, 128, 150), (4, 64, 1), (4, 64, 70), (2, 256, 1), (2, 256, 30), (2, 256, 50)])
def test_rows_of_no_sequence_are_left_as_they_were(dev, heads, D, new):
    from glorcq_b200.paged_cache import paged_attention
    held, counts = [20, 0, 35], [new, 0, max(1, new // 2)]
    cache = make_cache(5, "int8", 2, D, 16, [a + n for a, n in zip(held, counts)], dev)
    n = 3 + sum(counts) + 5
    q = torch.randn(n, heads, D, generator=torch.Generator().manual_seed(1)).half().to(dev)
    for c in (cache, wide(cache, MUCH)):
        out = torch.full((n, heads, D), 7.0, dtype=torch.float16, device=dev)
        paged_attention(q, *c, i64(held, dev), q_starts(counts, dev, at=3), max_new=new, out=out)
        assert (out[:3] == 7).all() and (out[3 + sum(counts):] == 7).all()
        check_attention(out, cache, held, counts, q, rows=[3, 3 + new, 3 + new])


@pytest.mark.parametrize("D,new", [(128, 1), (128, 140), (64, 40), (32, 1)])
def test_pages_that_are_not_there_are_hidden(dev, D, new):
    from glorcq_b200.paged_cache import paged_attention
    held = [100, 60, 30]
    cache = make_cache(6, "e4m3", 2, D, 16, [a + new for a in held], dev)
    table = cache[4]
    table[0, 1], table[0, 3] = -1, 1 << 30            # two pages inside
    table[1, 0] = cache[0].shape[0]                   # the first
    table[2] = -1                                     # all of them: nothing to see
    q = torch.randn(3 * new, 4, D, generator=torch.Generator().manual_seed(1)).half().to(dev)
    for c in (cache, wide(cache, MUCH)):
        got = paged_attention(q, *c, i64(held, dev))
        assert not got[2 * new:].any()
        check_attention(got, cache, held, [new] * 3, q)


@pytest.mark.parametrize("new", [1, 50, 1100])
def test_positions_outside_the_table(dev, new):
    """A length below zero counts as none, one behind the table as the table's: such rows see all that is."""
    from glorcq_b200.paged_cache import paged_append, paged_attention
    cache = make_cache(8, "int8", 2, 64, 16, [32, 32], dev, width=2)
    q = torch.randn(2 * new, 4, 64, generator=torch.Generator().manual_seed(1)).half().to(dev)
    start = [-5, 1 << 40]
    got = paged_attention(q, *cache, i64(start, dev))
    check_attention(got, cache, start, [new] * 2, q)
    before = [t.clone() for t in cache]
    k = torch.randn(2 * new, 2, 64, generator=torch.Generator().manual_seed(2)).half().to(dev)
    cos, sin = tables(64, 32, dev)
    paged_append(None, k, k, cos, sin, *cache, i64(start, dev))
    used = cache[4][1].long()
    for a, b in zip(cache[:4], before[:4]):
        assert torch.equal(a.view(torch.uint8)[used], b.view(torch.uint8)[used])


@pytest.mark.parametrize("new", [1, 90])
def test_attention_takes_rows_of_any_distance_and_its_scale(dev, new):
    from glorcq_b200.paged_cache import paged_attention
    cache = make_cache(9, "int8", 2, 128, 32, [40 + new, 7 + new], dev)
    both = torch.randn(2 * new, 12, 128, generator=torch.Generator().manual_seed(4)).half().to(dev)
    q, out = both[:, 4:8], torch.zeros(2 * new, 9, 128, dtype=torch.float16, device=dev)
    for c in (cache, wide(cache, MUCH)):
        out[:, 2:6] = 1
        paged_attention(q, *c, i64([40, 7], dev), scale=0.21, out=out[:, 2:6])
        check_attention(out[:, 2:6], cache, [40, 7], [new] * 2, q, scale=0.21)
        assert not out[:, :2].any() and not out[:, 6:].any()


@pytest.mark.parametrize("new", [1, 33])
def test_scales_of_any_size(dev, new):
    """Blocks that are zero (scale 0), tiny and large beside one another."""
    from glorcq_b200.paged_cache import paged_attention
    cache = make_cache(10, "int8", 1, 64, 16, [96 + new], dev)
    table = cache[4][0].tolist()
    for i, t in enumerate(cache[2:4]):
        t[table[0]] *= 1e-9
        t[table[2]] *= 30.0 if i else 4.0
        t[table[3]] = 0.0
        cache[i].view(torch.uint8)[table[3]] = 0
    q = torch.randn(new, 4, 64, generator=torch.Generator().manual_seed(4)).half().to(dev)
    for c in (cache, wide(cache, MUCH)):
        check_attention(paged_attention(q, *c, i64([96], dev)), cache, [96], [new], q)


@pytest.mark.parametrize("dtype,D,new", [("int8", 128, 1), ("e4m3", 128, 12), ("int8", 128, 40), ("e4m3", 64, 40), ("int8", 256, 40), ("int8", 32, 20)])
def test_what_lies_behind_the_tokens_does_not_matter(dev, dtype, D, new):
    """Pages that are a sequence's already but hold nothing yet, and the slots behind its last token: any codes, any scales."""
    from glorcq_b200.paged_cache import paged_attention
    held = [21, 100]
    clean = make_cache(6, dtype, 2, D, 16, [a + new for a in held], dev, width=16, pool=32)
    q = torch.randn(2 * new, 4, D, generator=torch.Generator().manual_seed(4)).half().to(dev)
    dirty = [t.clone() for t in clean]
    spare = [p for p in range(32) if p not in sum(clean[4].tolist(), [])]
    for b, a in enumerate(held):
        used = (a + new + 15) // 16
        for j in range(used, min(used + 5, 16)):
            dirty[4][b, j] = spare.pop()
        if (a + new) % 16:
            for t in dirty[:2]:
                t.view(torch.uint8)[dirty[4][b, used - 1], :, (a + new) % 16:] = 0xff
    for x in (float("nan"), float("inf"), -1.0, 1e-42, 1e30):
        for p in range(32):
            if p not in sum(clean[4].tolist(), []):
                for t in dirty[:2]:
                    t.view(torch.uint8)[p] = 0x7f
                for t in dirty[2:4]:
                    t[p] = x
        for room in (0, 40000, MUCH):
            a, b = ([*c[:4], wide(c, room)[4] if room else c[4]] for c in (clean, dirty))
            assert torch.equal(paged_attention(q, *b, i64(held, dev)), paged_attention(q, *a, i64(held, dev))), (x, room)
    check_attention(paged_attention(q, *dirty, i64(held, dev)), clean, held, [new] * 2, q)


@pytest.mark.parametrize("new", [1, 40])
def test_a_scale_of_zero_means_the_mean(dev, new):
    from glorcq_b200.paged_cache import paged_attention
    cache = make_cache(6, "int8", 2, 128, 16, [90 + new], dev)
    q = torch.randn(new, 4, 128, generator=torch.Generator().manual_seed(4)).half().to(dev)
    for c in (cache, wide(cache, 40000), wide(cache, MUCH)):
        check_attention(paged_attention(q, *c, i64([90], dev), scale=0.0), cache, [90], [new], q, scale=0.0)
    for bad in (-1.0, float("nan"), float("inf")):
        with pytest.raises(RuntimeError):
            paged_attention(q, *cache, i64([90], dev), scale=bad)


@pytest.mark.parametrize("room", [0, 40000, MUCH])
@pytest.mark.parametrize("new", [1, 20])
def test_not_a_number_in_a_query_stays_in_its_row(dev, new, room):
    from glorcq_b200.paged_cache import paged_attention
    cache = make_cache(11, "e4m3", 2, 128, 32, [70 + new] * 2, dev)
    if room:
        cache = wide(cache, room)
    q = torch.randn(2 * new, 4, 128, generator=torch.Generator().manual_seed(4)).half().to(dev)
    want = paged_attention(q, *cache, i64([70], dev))
    q[0, 1, 5] = float("nan")
    got = paged_attention(q, *cache, i64([70], dev))
    assert got[0, 1].isnan().all()
    got[0, 1] = want[0, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("new", [1, 40])
def test_pages_behind_two_gigabytes_and_shared_ones(dev, new):
    """A pool above 2^31 bytes; two sequences share the pages of their beginning."""
    from glorcq_b200.paged_cache import paged_attention
    P, kv, D = 128, 16, 128
    pool = (1 << 31) // (P * kv * D) + 300
    small = make_cache(12, "int8", kv, D, P, [300 + new, 300 + new], dev, pool=8)
    far = torch.arange(pool - 8, pool, device=dev)
    cache = [torch.zeros(pool, kv, P, D, dtype=torch.int8, device=dev) for _ in range(2)] + [torch.zeros(pool, kv, device=dev) for _ in range(2)]
    for t, s in zip(cache, small):
        t[far] = s
    small[4][1, :2] = small[4][0, :2]
    cache.append(torch.where(small[4] >= 0, small[4] + pool - 8, small[4]).to(torch.int32))
    q = torch.randn(2 * new, 16, D, generator=torch.Generator().manual_seed(4)).half().to(dev)
    for room in (40000, MUCH):
        assert torch.equal(paged_attention(q, *wide(cache, room), i64([300], dev)), paged_attention(q, *wide(small, room), i64([300], dev)))
    got = paged_attention(q, *cache, i64([300], dev))
    assert torch.equal(got, paged_attention(q, *small, i64([300], dev)))
    check_attention(got[:, :1], [t[:, :1] if t.dim() > 2 or t.shape[1] == kv else t for t in small], [300, 300], [new] * 2, q[:, :1])


# ---- append ----------------------------------------------------------------------------------------------------------------

APPEND = [  # dtype, heads, kv heads, D, page, held, new
    ("int8", 16, 16, 128, 64, [512], [1]), ("e4m3", 32, 4, 128, 32, [0, 31, 32, 70], [1, 1, 1, 1]), ("int8", 4, 2, 64, 16, [0, 5, 15, 40], [50, 3, 18, 0]),
    ("e4m3", 4, 1, 256, 128, [130, 0], [200, 129]), ("int8", 3, 3, 32, 16, [1, 0], [40, 7]), ("e4m3", 4, 2, 64, 64, [10], [300]),
    ("int8", 8, 1, 256, 16, [3, 3], [2, 40]), ("int8", 1, 1, 128, 128, [0], [257])]


def rows_for(new, heads, kv, D, dev, seed=1):
    g = torch.Generator().manual_seed(seed)
    n = sum(new)
    grow = torch.logspace(-0.5, 0.5, max(n, 1))[:n, None, None]           # later tokens are larger: blocks outgrow their scales
    return [(torch.randn(n, h, D, generator=g) * grow).half().to(dev) for h in (heads, kv, kv)]


def want_append(pages, start, new, k, v, cos, sin, k_norm=None, eps=1e-6):
    at = 0
    for b, n in enumerate(new):
        pos = torch.arange(start[b], start[b] + n)
        x = k[at:at + n].cpu().float()
        if k_norm is not None:
            x = paged_ref.normed(x, k_norm.cpu(), eps)
        pages.append(0, b, start[b], paged_ref.rotated(x, cos.cpu()[:, None], sin.cpu()[:, None], pos))
        pages.append(1, b, start[b], v[at:at + n].cpu().float())
        at += n


def same_pages(cache, pages, start, new, every=True):
    """codes of all live slots and all scales equal"""
    for i in range(2):
        for b, n in enumerate(new):
            for j in range((start[b] + n + pages.P - 1) // pages.P):
                p, live = int(pages.table[b, j]), min(pages.P, start[b] + n - j * pages.P)
                assert torch.equal(cache[2 + i][p].cpu(), pages.scale[i][p]), (i, b, j)
                assert torch.equal(cache[i][p, :, :live].cpu().float(), pages.codes[i][p, :, :live]), (i, b, j)


@pytest.mark.parametrize("dtype,heads,kv,D,P,held,new", APPEND)
def test_append_writes_the_codes_of_the_definition(dev, dtype, heads, kv, D, P, held, new):
    from glorcq_b200.paged_cache import paged_append
    cache = make_cache(D + P, dtype, kv, D, P, held, dev, width=1 + max((a + n + P - 1) // P for a, n in zip(held, new)), pool=4 + sum((a + n + P - 1) // P for a, n in zip(held, new)))
    free = [p for p in range(cache[0].shape[0]) if p not in sum(cache[4].tolist(), [])]
    for b, (a, n) in enumerate(zip(held, new)):
        for j in range((a + P - 1) // P, (a + n + P - 1) // P):
            cache[4][b, j] = free.pop()
    cos, sin = tables(D, cache[4].shape[1] * P, dev)
    q, k, v = rows_for(new, heads, kv, D, dev)
    pages = Pages(cache)
    before = [t.clone() for t in cache]
    want_append(pages, held, new, k, v, cos, sin)
    got = paged_append(q, k, v, cos, sin, *cache, i64(held, dev), q_starts(new, dev))
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(held, new)])
    assert torch.equal(got.cpu(), paged_ref.rotated(q.cpu().float(), cos.cpu()[:, None], sin.cpu()[:, None], pos).half())
    same_pages(cache, pages, held, new)
    # nothing else changed: pages of nobody, slots behind the last token
    written = {(int(pages.table[b, j]), s) for b, (a, n) in enumerate(zip(held, new)) for j in range(a // P, (a + n + P - 1) // P)
               for s in range(P) if j * P + s < a + n}
    for i in range(2):
        keep = torch.ones(cache[0].shape[0], P, dtype=torch.bool)
        for p, s in written:
            keep[p, s] = False
        keep = keep.to(dev)
        assert torch.equal(cache[i].view(torch.uint8).transpose(1, 2)[keep], before[i].view(torch.uint8).transpose(1, 2)[keep])
    # the same call again changes nothing: scales cover the values now
    again = [t.clone() for t in cache]
    paged_append(None, k, v, cos, sin, *cache, i64(held, dev), q_starts(new, dev))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(again, cache))


def test_append_token_by_token_and_at_once(dev):
    """Growing blocks: 70 calls of one token, each beside its plain form; start as one number for all."""
    from glorcq_b200.paged_cache import paged_append
    for dtype in ("int8", "e4m3"):
        cache = make_cache(3, dtype, 2, 64, 32, [0, 0], dev, width=3, pool=7)
        cache[4].copy_(torch.tensor([[6, 2, 4], [0, 5, 1]]))
        cos, sin = tables(64, 96, dev)
        pages = Pages(cache)
        for t in range(70):
            _, k, v = rows_for([1, 1], 1, 2, 64, dev, seed=t)
            k, v = k * 1.05 ** t, v * (1.0 if t % 32 else 1e-3)
            want_append(pages, [t, t], [1, 1], k, v, cos, sin)
            paged_append(None, k, v, cos, sin, *cache, i64([t], dev))
        same_pages(cache, pages, [70, 70], [0, 0])


@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_append_with_norms(dev, D):
    """The norm's sum has an order of its own (D + 8 roundings of 2^-24, of which the root takes half): values against 64 bits."""
    from glorcq_b200.paged_cache import paged_append, paged_read
    held, new = [0, 37], [21, 40]
    cache = make_cache(3, "int8", 2, D, 16, [0, 37], dev, width=6, pool=12)
    free = [p for p in range(12) if p not in sum(cache[4].tolist(), [])]
    for b, (a, n) in enumerate(zip(held, new)):
        for j in range((a + 15) // 16, (a + n + 15) // 16):
            cache[4][b, j] = free.pop()
    cos, sin = tables(D, 96, dev)
    q, k, v = rows_for(new, 4, 2, D, dev)
    g = torch.Generator().manual_seed(5)
    qw, kw = ((torch.rand(D, generator=g) + 0.5).half().to(dev) for _ in range(2))
    got = paged_append(q, k, v, cos, sin, *cache, i64(held, dev), q_starts(new, dev), q_norm=qw, k_norm=kw, eps=1e-5)
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(held, new)])

    def exact(x, w):
        x = x.cpu().double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-5) * w.cpu().double()
        return paged_ref.rotated(x, cos.cpu().double()[:, None], sin.cpu().double()[:, None], pos), x.abs()
    ref, mag = exact(q, qw)
    rel = (D + 24) * 2.0 ** -24
    size = mag + torch.cat((mag[..., D // 2:], mag[..., : D // 2]), -1)
    assert ((got.cpu().double() - ref).abs() <= 2.0 ** -11 * ref.abs() + rel * size + 2.0 ** -25).all()
    ref, mag = exact(k, kw)
    size = mag + torch.cat((mag[..., D // 2:], mag[..., : D // 2]), -1)
    kk, _ = paged_read(*cache, i64(held, dev), q_starts(new, dev), sum(new))
    step = torch.stack([cache[2][cache[4][b, p // 16]].cpu() for b, a, n in zip((0, 1), held, new) for p in range(a, a + n)])[:, :, None]
    # half a step of the block (its scale may have doubled after the row was written only in the same call: then codes are of the final scale), fp16 of the read
    assert ((kk.cpu().double() - ref).abs() <= (0.5 + 2.0 ** -10) * step.double() + 2.0 ** -11 * ref.abs() + rel * size).all()


@pytest.mark.parametrize("heads,D", [(17, 128), (5, 256), (3, 64), (32, 32)])
def test_append_of_many_rows_turns_queries_as_of_few(dev, heads, D):
    """A CTA takes more rows of queries where there are many: the same values as from calls of 300 rows each."""
    from glorcq_b200.paged_cache import paged_append
    n = 1250 * max(1, 128 // (D // 16) // heads) + 37
    held, new = [3, 50], [n - 401, 401]
    pages = [(a + m + 127) // 128 for a, m in zip(held, new)]
    cache = make_cache(3, "int8", 1, D, 128, [0, 0], dev, width=max(pages), pool=sum(pages) + 1)
    cache[4].fill_(-1)
    cache[4][0, :pages[0]] = torch.arange(pages[0])
    cache[4][1, :pages[1]] = torch.arange(pages[0], sum(pages))
    cos, sin = tables(D, max(pages) * 128, dev)
    g = torch.Generator().manual_seed(D)
    q, k = (torch.randn(n + 5, h, D, generator=g).half().to(dev) for h in (heads, 1))
    qw, kw = ((torch.rand(D, generator=g) + 0.5).half().to(dev) for _ in range(2))
    for norms in ({}, dict(q_norm=qw, k_norm=kw)):
        out = torch.full_like(q, 7.0)
        paged_append(q, k, k, cos, sin, *cache, i64(held, dev), q_starts(new, dev, at=2), q_out=out, **norms)
        assert (out[:2] == 7).all() and (out[2 + n:] == 7).all()
        for b, first in ((0, 2), (1, 2 + new[0])):
            for i in range(0, new[b], 300):
                m = min(300, new[b] - i)
                rows = slice(first + i, first + i + m)
                one = [*cache[:4], cache[4][b:b + 1]]
                got = paged_append(q[rows], k[rows], k[rows], cos, sin, *one, i64([held[b] + i], dev), **norms)
                assert torch.equal(got, out[rows]), (b, i)


def test_append_of_values_that_are_not_finite(dev):
    from glorcq_b200.paged_cache import paged_append
    for dtype in ("int8", "e4m3"):
        cache = make_cache(3, dtype, 1, 64, 16, [0], dev, width=2, pool=4)
        cache[4][0] = torch.tensor([1, 3])
        v = torch.randn(20, 1, 64, generator=torch.Generator().manual_seed(5)).half().to(dev)
        v[3, 0, 7], v[4, 0, 8], v[5, 0, 9] = float("inf"), float("-inf"), float("nan")
        v[16:] = 0
        v[17, 0, 3] = float("inf")
        pages = Pages(cache)
        pages.append(0, 0, 0, v.cpu().float())
        pages.append(1, 0, 0, v.cpu().float())
        paged_append(None, v, v, None, None, *cache, i64([0], dev))
        same_pages(cache, pages, [20], [0])
        assert cache[0][1, 0, 3, 7].float() == paged_ref.QMAX[dtype] and cache[0][1, 0, 5, 9].float() == 0 and cache[2][3, 0] == 0


def test_append_rows_of_any_distance_in_place_and_left_out(dev):
    from glorcq_b200.paged_cache import paged_append
    cache = make_cache(3, "int8", 2, 64, 16, [20, 3], dev, width=3)
    plain = [t.clone() for t in cache]
    cos, sin = tables(64, 48, dev)
    qkv = torch.randn(9, 8, 64, generator=torch.Generator().manual_seed(5)).half().to(dev)
    q, k, v = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
    counts = q_starts([4, 2], dev, at=2)
    want = paged_append(q.contiguous(), k.contiguous(), v.contiguous(), cos, sin, *plain, i64([20, 3], dev), counts)
    rest = qkv.clone()
    got = paged_append(q, k, v, cos, sin, *cache, i64([20, 3], dev), counts, q_out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(q[2:8], want[2:8])
    assert torch.equal(qkv[:2], rest[:2]) and torch.equal(qkv[8:], rest[8:]) and torch.equal(qkv[:, 4:], rest[:, 4:])
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(plain, cache))


# ---- read --------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,kv,D,P", [("int8", 4, 128, 64), ("e4m3", 1, 64, 16), ("int8", 3, 32, 32), ("e4m3", 2, 256, 128)])
def test_read(dev, dtype, kv, D, P):
    from glorcq_b200.paged_cache import paged_read
    held = [200, 5, 90]
    cache = make_cache(4, dtype, kv, D, P, held, dev)
    first, count = [3, 0, 80], [197, 5, 30]             # the last asks for positions that have no page
    cache[4][0, 0] = -1
    k, v = paged_read(*cache, i64(first, dev), q_starts(count, dev), sum(count))
    pages, at = Pages(cache), 0
    for b, (f, n) in enumerate(zip(first, count)):
        for i, t in ((0, k), (1, v)):
            for r, x in enumerate(pages.values(i, b, f, n)):
                if x is None:
                    assert not t[at + r].any()
                elif f + r < held[b]:
                    assert torch.equal(t[at + r].cpu(), x.float().half())
        at += n
    one = paged_read(*cache[:4], cache[4][1:2], i64([1], dev), None, 4)
    assert torch.equal(one[0], k[198:202]) and torch.equal(one[1], v[198:202])
    assert paged_read(*cache, i64([0], dev), None, 0)[0].shape == (0, kv, D)


# ---- refusals, streams, graphs, use together ---------------------------------------------------------------------------------------

def test_refusals(dev):
    from glorcq_b200.paged_cache import paged_append, paged_attention, paged_read
    cache = make_cache(1, "int8", 2, 64, 16, [20, 20], dev)
    q, k = torch.zeros(2, 4, 64, device=dev).half(), torch.zeros(2, 2, 64, device=dev).half()
    start = i64([19], dev)
    cos, sin = tables(64, cache[4].shape[1] * 16, dev)

    def swapped(i, t):
        return [t if n == i else x for n, x in enumerate(cache)]
    bad_caches = [swapped(0, cache[0].half()), swapped(0, cache[0][..., ::2]), swapped(1, cache[1].view(torch.float8_e4m3fn)), swapped(1, cache[1][:1]),
                  swapped(2, cache[2][:1]), swapped(3, cache[3].double()), swapped(4, cache[4].long()), swapped(4, cache[4][0]), swapped(4, cache[4].cpu()),
                  swapped(0, cache[0].view(-1, 2, 8, 128)), swapped(4, cache[4].t())]
    for bad in bad_caches:
        for call in (lambda: paged_append(q, k, k, cos, sin, *bad, start), lambda: paged_attention(q, *bad, start),
                     lambda: paged_read(*bad, start, None, 2)):
            with pytest.raises(RuntimeError):
                call()
    for args in (dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q.transpose(0, 1)), dict(q=torch.zeros(3, 4, 64, device=dev).half()),
                 dict(start=start.int()), dict(start=i64([1, 2, 3], dev)), dict(q_start=i64([0, 1, 2], dev)), dict(q_start=q_starts([2], dev)), dict(out=q[:1]),
                 dict(q=torch.zeros(2, 4, 65, device=dev).half()[..., 1:])):
        with pytest.raises(RuntimeError):
            a = {**dict(q=q, start=start), **args}
            paged_attention(a["q"], *cache, a["start"], a.get("q_start"), out=a.get("out"))
    for args in (dict(cos=None), dict(cos=cos[:8], sin=sin[:8]), dict(cos=cos.half(), sin=sin.half()), dict(k=q), dict(v=k[:1]), dict(q_norm=cos[0].half()),
                 dict(q_norm=torch.ones(32, device=dev).half(), k_norm=torch.ones(32, device=dev).half()), dict(q_out=k), dict(k=k.cpu())):
        with pytest.raises(RuntimeError):
            a = {**dict(q=q, k=k, v=k, cos=cos, sin=sin), **args}
            paged_append(a["q"], a["k"], a["v"], a["cos"], a["sin"], *cache, start, None, a.get("q_norm"), a.get("k_norm"), 1e-6, a.get("q_out"))
    with pytest.raises(RuntimeError):
        paged_read(*cache, start, None, 3)
    with pytest.raises(RuntimeError):
        paged_read(*cache, start, None, -1)
    with pytest.raises(RuntimeError, match="not supported"):             # rows times tokens beyond 32 bits
        paged_attention(torch.zeros(1 << 16, 64, 64, device=dev).half(), *cache[:4], torch.full((2, 1 << 24), -1, dtype=torch.int32, device=dev), start)
    with pytest.raises(RuntimeError, match="multiple of the cache's heads"):
        paged_attention(torch.zeros(2, 3, 64, device=dev).half(), *cache, start)
    torch.cuda.synchronize()


def test_calls_run_without_the_interpreter_lock(dev):
    """The library's entry points are replaced by PyGILState_Check: 0, a success, when the calling thread does not hold the interpreter lock, and by
    Py_IsInitialized, which is 1, an unknown status."""
    import ctypes as C
    from glorcq_b200 import _lib
    from glorcq_b200.paged_cache import paged_append, paged_attention, paged_read
    cache = make_cache(1, "int8", 2, 64, 16, [20], dev)
    q = torch.zeros(1, 4, 64, dtype=torch.float16, device=dev)
    start = i64([19], dev)
    calls = {"glq_paged_append": lambda: paged_append(None, q[:, :2], q[:, :2], None, None, *cache, start),
             "glq_paged_attention": lambda: paged_attention(q, *cache, start), "glq_paged_read": lambda: paged_read(*cache, start, None, 1)}
    nat = _lib.native()
    real = {e: C.cast(getattr(_lib.lib(), e), C.c_void_p).value for e in nat.paged_names()}
    assert set(real) == {*calls, "glq_paged_attention_workspace_bytes"} and not set(real) & set(nat.names())
    probe, fails = (C.cast(f, C.c_void_p).value for f in (C.pythonapi.PyGILState_Check, C.pythonapi.Py_IsInitialized))
    try:
        for e, call in calls.items():
            nat.paged_bind({**real, e: probe})
            call()
            nat.paged_bind({**real, e: fails})
            with pytest.raises(RuntimeError):
                call()
    finally:
        nat.paged_bind(real)


def step(cache, q, k, v, cos, sin, start):
    from glorcq_b200.paged_cache import paged_append, paged_attention
    return paged_attention(paged_append(q, k, v, cos, sin, *cache, start), *cache, start)


@pytest.mark.parametrize("new,width", [(1, 32), (30, 32), (30, 2500)])
def test_captured_calls_follow_lengths_and_pages(dev, new, width):
    """Two graphs over one cache replayed on two streams, lengths and table changed in between: as eager calls, also while those run
    on a third stream."""
    cache = make_cache(1, "e4m3", 2, 128, 16, [400, 300], dev, width=width, pool=70)
    spare = [p for p in range(70) if p not in sum(cache[4].tolist(), [])]
    cos, sin = tables(128, 16 * width, dev)
    q, k, v = rows_for([new, new], 8, 2, 128, dev)
    for j, b in ((25, 0), (26, 0), (27, 0), (19, 1), (20, 1), (21, 1)):
        cache[4][b, j] = spare.pop()
    start = i64([399, 300], dev)
    from glorcq_b200.paged_cache import paged_attention
    step([t.clone() for t in cache], q, k, v, cos, sin, start)
    graphs, outs, q2 = [], [], q * 0.5
    for x in (q, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(cache, x, k, v, cos, sin, start))
        graphs.append(g)
    for s in ([399, 300], [400, 301], [17, 0]):
        start.copy_(torch.tensor(s))
        twin = [t.clone() for t in cache]
        want = [step(twin, x, k, v, cos, sin, start) for x in (q, q2)]
        for g in graphs:                     # (one after another first: both append)
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
        check_attention(outs[0], cache, s, [new, new], _rotated(q, s, new, cos, sin))
    # attention alone, side by side on three streams
    alone, res = [], []
    for x in (q, q2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res.append(paged_attention(x, *cache, start))
        alone.append(g)
    want = [paged_attention(x, *cache, start) for x in (q, q2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for g, st in zip(alone, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            third = paged_attention(q, *cache, start)
        torch.cuda.synchronize()
        assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1]) and torch.equal(third, want[0])


def _rotated(q, start, new, cos, sin):
    pos = torch.cat([torch.arange(a, a + new) for a in start])
    return paged_ref.rotated(q.cpu().float(), cos.cpu()[:, None], sin.cpu()[:, None], pos).half()


def test_a_prompt_and_decoded_tokens_together(dev):
    """Two prompts of their own lengths in pieces, then tokens one by one through PagedKVCache: pages, attention and read agree with the
    plain implementation at every step."""
    from types import SimpleNamespace
    from glorcq_b200.paged_cache import PagedKVCache
    cfg = SimpleNamespace(num_hidden_layers=2, num_key_value_heads=2, head_dim=128, rope_theta=10000.0)
    c = PagedKVCache(cfg, 2, 200, dev, dtype="int8", page_size=16, num_pages=30)
    cos, sin = c.cos, c.sin
    held = [0, 0]
    plain = None
    for n, pieces in enumerate(([50, 17], [23, 40], [1, 1], [1, 1], [5, 0], [1, 1])):
        for b in range(2):
            c.reserve(b, held[b] + pieces[b])
        q, k, v = rows_for(pieces, 8, 2, 128, dev, seed=n)
        cache = list(c.layer(1, 2))
        now = Pages(cache)
        if plain is not None:
            now.codes, now.scale = plain.codes, plain.scale
        plain = now
        want_append(plain, held, pieces, k, v, cos, sin)
        start, qs = i64(held, dev), q_starts(pieces, dev)
        q = c.append(1, q, k, v, start, 2, q_start=qs)
        y = c.attend(1, q, start, 2, q_start=qs, max_new=max(pieces))
        same_pages(cache, plain, held, pieces)
        check_attention(y, cache, held, pieces, q)
        held = [a + p for a, p in zip(held, pieces)]
    kk, vv = c.read(1, 0, 3, 60)
    ref = torch.stack(plain.values(1, 0, 3, 60)).float().half()
    assert torch.equal(vv.cpu(), ref)
    assert not c.k[0].view(torch.uint8).any()                     # the other layer was not touched
    c.release(0)
    assert (c.page_table[0] == -1).all()


SMALL = dict(hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64, vocab_size=512, num_experts=4,
             num_experts_per_tok=4, moe_intermediate_size=128, norm_topk_prob=True, rms_norm_eps=1e-6, rope_theta=10000.0, max_position_embeddings=128)


@pytest.mark.parametrize("kv_cache", ["int8", "e4m3"])
def test_decoder_over_the_paged_cache(dev, kv_cache):
    """Graph replay equals eager calls; sequences at positions of their own equal the same sequences alone; and the logits stay near those over
    the fp16 cache.  All experts are chosen, so that no routing flips.  A stored value is off by amax / 254 (int8: 1 % of a block's standard deviation, whose
    largest of 1000 to 4000 values is about 4 of them; e4m3: 2^-4 / sqrt(3) = 4 % at most), keys and values both, two layers, and the MoE block behind may
    double it: 6 % and 24 % at the very most."""
    from glorcq_b200.decoder import StaticKVCache
    from glorcq_b200.graph_wrapper import GLoRCQGraphWrapper
    from glorcq_b200.paged_cache import PagedKVCache
    from glorcq_b200.synthetic import make_decoder
    m = make_decoder(SMALL, dev, seed=3, rank=16, attn_rank=16)
    ids = torch.randint(0, 512, (2, 40), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        w = GLoRCQGraphWrapper(m, max_batch_size=2, max_seq_len=100, kv_cache=kv_cache, page_size=16)
        out, _ = w.generate(ids, max_new_tokens=12)
        again, _ = w.generate(ids, max_new_tokens=12)
        assert torch.equal(out, again) and out.shape == (2, 52)
        cache = PagedKVCache(m.config, 2, 100, dev, dtype=kv_cache, page_size=16)
        static = StaticKVCache(m.config, 2, 100, dev)
        logits = m(input_ids=ids, cache_position=torch.arange(40, device=dev), past_key_values=cache)[0]
        ref = m(input_ids=ids, cache_position=torch.arange(40, device=dev), past_key_values=static)[0]
        far = 0.06 if kv_cache == "int8" else 0.24
        assert (logits.float() - ref.float()).norm() <= far * ref.float().norm()
        for t in range(40, 51):
            logits = m(input_ids=out[:, t:t + 1], cache_position=torch.tensor([t], device=dev), past_key_values=cache)[0]
            assert torch.equal(logits[:, -1].argmax(-1), out[:, t + 1])
        # positions of their own: sequence 1 is ten tokens behind
        ragged = PagedKVCache(m.config, 2, 100, dev, dtype=kv_cache, page_size=16)
        for b, n in ((0, 40), (1, 30)):
            one = PagedKVCache(m.config, 1, 100, dev, dtype=kv_cache, page_size=16)
            one.k, one.v, one.k_scale, one.v_scale, one.page_table = ragged.k, ragged.v, ragged.k_scale, ragged.v_scale, ragged.page_table[b:b + 1]
            m(input_ids=ids[b:b + 1, :n], cache_position=torch.arange(n, device=dev), past_key_values=one)
        both = m(input_ids=torch.stack((ids[0, :1], ids[1, 30:31])), cache_position=torch.tensor([40, 30], device=dev), past_key_values=ragged)[0]
        for b, n in ((0, 40), (1, 30)):
            alone = PagedKVCache(m.config, 1, 100, dev, dtype=kv_cache, page_size=16)
            m(input_ids=ids[b:b + 1, :n], cache_position=torch.arange(n, device=dev), past_key_values=alone)
            tok = ids[0, :1] if b == 0 else ids[1, 30:31]
            want = m(input_ids=tok[None], cache_position=torch.tensor([n], device=dev), past_key_values=alone)[0]
            # (one and two rows take different sums in the experts' products: 2^-10 a rounding)
            assert (both[b].float() - want[0].float()).norm() <= 1e-2 * want.float().norm()
        # a graph at those positions
        g = w.replay(torch.stack((out[0, 51:52], out[1, 51:52])), [51, 51])
        assert g.shape == (2, 1, 512) and g.isfinite().all()
    with pytest.raises(RuntimeError):
        m(input_ids=ids, cache_position=torch.arange(7, device=dev), past_key_values=cache)
    with pytest.raises(RuntimeError):
        m(input_ids=ids.repeat(1, 4), past_key_values=cache)
