"""The paged 8-bit cache where it is easily got wrong: prompts behind contexts that take long, blocks and rows of which little is left."""

import pytest
import torch

from glorcq_b200.paged_cache import paged_attention
from tests.paged_ref import TYPES, make_cache
from tests.test_gpu_paged import MUCH, i64, wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    from glorcq_b200 import _build
    _build.build()
    return torch.device("cuda:0")


def q_starts(new, dev):
    return torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device=dev)


def long_cache(dtype, kv, D, P, tokens, dev):
    """One sequence's `tokens` tokens in pages in random order: keys of about one in size, values of about one half."""
    g = torch.Generator(device=dev).manual_seed(D + kv)
    n = -(-tokens // P)
    size = 80.0 if dtype == "int8" else 160.0
    codes = [(torch.randn(n, kv, P, D, generator=g, device=dev) * size / 2.5).clamp(-size, size) for _ in range(2)]
    codes = [(t.round() if dtype == "int8" else t).to(TYPES[dtype]) for t in codes]
    scale = [(0.75 + 0.5 * torch.rand(n, kv, generator=g, device=dev)) * 2.5 / size * x for x in (1.0, 0.5)]
    return [*codes, *scale, torch.randperm(n, generator=g, device=dev).to(torch.int32)[None]]


def exact_rows(cache, b, held, q, rows):
    """Attention in 64 bits of the rows `rows` of sequence b's q (n, heads, D), the first of which is at position `held`, and the bound of a kernel's
    error: that of paged_ref.attention, and for as many tokens one rounding of 2^-23 of the sum so far for every 16 tokens that are added to it, which
    counts for the sum of the values as for that of the weights."""
    k_pages, v_pages, k_scale, v_scale, table = cache
    D, heads, kv, P = q.shape[-1], q.shape[1], k_pages.shape[1], k_pages.shape[2]
    pages = table[b].long()
    total = min(held + len(q), len(pages) * P)
    out, tol = (torch.zeros(len(rows), heads, D, dtype=torch.float64, device=q.device) for _ in range(2))
    for h in range(kv):
        k, v = ((t[pages, h].double() * s[pages, h].double()[:, None, None]).reshape(-1, D)[:total] for t, s in ((k_pages, k_scale), (v_pages, v_scale)))
        vs = v_scale[pages, h].double().repeat_interleave(P)[:total]
        for i, r in enumerate(rows):
            n = min(held + r + 1, total)
            x = q[r, h * heads // kv:(h + 1) * heads // kv].double()
            p = torch.softmax(x @ k[:n].T * D ** -0.5, dim=1)
            size = (x.abs() @ k[:n].abs().T).amax(dim=1) * D ** -0.5
            rel = 2.0 ** -11 + 2 * ((D + 16) * 2.0 ** -23 * size + 2.0 ** -18) + 2 * n / 16 * 2.0 ** -23
            y, mag = p @ v[:n], p @ v[:n].abs()
            codes = (v[:n] / torch.where(vs > 0, vs, torch.ones_like(vs))[:n, None]).abs()
            floor = 2.0 ** -25 * (p * vs[:n]).amax(dim=1)[:, None] * codes.sum(dim=0)
            at = slice(h * heads // kv, (h + 1) * heads // kv)
            out[i, at], tol[i, at] = y, 2.0 ** -11 * y.abs() + rel[:, None] * mag + floor + 2.0 ** -25
    return out, tol


def check_rows(got, cache, b, held, q, rows):
    ref, tol = exact_rows(cache, b, held, q, rows)
    err = (got[rows].double() - ref).abs()
    assert (err <= tol).all(), f"sequence {b}: {(err / tol).max()} of the bound"
    # (the rows tell their keys apart: a result that has missed some of them, or that nobody wrote, is not within the bound)
    assert tol.max() < 0.2 * ref.abs().max()


LONG = [  # dtype, heads, kv heads, D, sequences that share the pages, tokens held, new tokens of each
    ("int8", 32, 8, 128, 1, 131072, 4096), ("e4m3", 16, 8, 256, 1, 65536, 4096), ("int8", 8, 8, 128, 50, 200000, 100), ("e4m3", 8, 8, 128, 20, 200000, 300)]


@pytest.mark.parametrize("dtype,heads,kv,D,batch,held,new", LONG)
def test_prompts_behind_contexts_that_take_long(dev, dtype, heads, kv, D, batch, held, new):
    """Pieces of the work that take milliseconds each: no wait for one of them runs out, and no row is left out.  (Many keys, few of which weigh: q is
    large, so that the scores' deviation is 3.)"""
    from glorcq_b200 import tiled
    cache = long_cache(dtype, kv, D, 128, held + new, dev)
    cache[4] = cache[4].repeat(batch, 1)
    q = (torch.randn(batch * new, heads, D, generator=torch.Generator(device=dev).manual_seed(1), device=dev) * 3).half()
    out = torch.full_like(q, 7.0)
    paged_attention(q, *cache, i64([held], dev), max_new=new, out=out)
    torch.cuda.synchronize()
    assert tiled.debug_error() is None
    assert not (out == 7.0).all(dim=-1).any()
    for b in {0, batch // 2, batch - 1}:
        rows = sorted({0, 31, new // 2, new - 30, new - 1})
        check_rows(out[b * new:(b + 1) * new], cache, b, held, q[b * new:(b + 1) * new], rows)


def test_prompts_among_thousands_of_sequences_without_rows(dev):
    """What finds a CTA's next rows looks at every sequence in between; who waits for it does not give up."""
    from glorcq_b200 import tiled
    B, held = 8000, 1000
    cache = long_cache("int8", 2, 128, 64, held + 40, dev)
    cache[4] = cache[4].repeat(B, 1)
    new = [0] * B
    for b in (0, 1, 4000, B - 1):
        new[b] = 40
    q = (torch.randn(sum(new), 4, 128, generator=torch.Generator(device=dev).manual_seed(1), device=dev) * 3).half()
    out = torch.full_like(q, 7.0)
    paged_attention(q, *cache, i64([held], dev), q_starts(new, dev), max_new=40, out=out)
    torch.cuda.synchronize()
    assert tiled.debug_error() is None
    for i in range(4):
        check_rows(out[40 * i:40 * i + 40], cache, 0, held, q[40 * i:40 * i + 40], [0, 17, 39])


SMALL = dict(hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64, vocab_size=512, num_experts=4,
             num_experts_per_tok=4, moe_intermediate_size=128, norm_topk_prob=True, rms_norm_eps=1e-6, rope_theta=10000.0, max_position_embeddings=128)


def test_generate_looks_for_waits_that_ran_out(dev, monkeypatch):
    from glorcq_b200.graph_wrapper import GLoRCQGraphWrapper
    from glorcq_b200.synthetic import make_decoder
    w = GLoRCQGraphWrapper(make_decoder(SMALL, dev, seed=3, rank=16, attn_rank=16), max_batch_size=1, max_seq_len=64, kv_cache="int8", page_size=16)
    ids = torch.arange(20, device=dev)[None]
    w.generate(ids, max_new_tokens=4)                       # nothing is wrong: the word of this device is clear

    def found():
        raise RuntimeError("a wait ran out")
    monkeypatch.setattr(w.static_cache, "raise_on_error", found)
    with pytest.raises(RuntimeError, match="a wait ran out"):
        w.generate(ids, max_new_tokens=4)


# ---- blocks and rows of which little is left ------------------------------------------------------------------------------------

ROOMS = (0, 40000, MUCH)


@pytest.mark.parametrize("new", [1, 12, 40])
@pytest.mark.parametrize("dtype,D", [("int8", 128), ("e4m3", 128), ("e4m3", 64), ("int8", 256), ("int8", 32)])
@pytest.mark.parametrize("size", [1e-3, 1e-4])
def test_values_of_zero_beside_small_ones_keep_the_others_bits(dev, dtype, D, size, new):
    """Pages whose values are all zero (scale 0) take their part of the softmax and nothing else: values of 1e-3 and 1e-4 in the other pages, none larger,
    come out as exactly as without them.  Sequences that share pages: as many as give every warp several tiles of 16 tokens."""
    held, batch = 2000, 24
    cache = long_cache(dtype, 2, D, 16, held + new, dev)
    cache[3] *= 2 * size
    empty = cache[4][0, torch.randperm(held // 16, generator=torch.Generator().manual_seed(D))[:30].to(dev)].long()
    cache[3][empty] = 0.0
    cache[1].view(torch.uint8)[empty] = 0
    cache[4] = cache[4].repeat(batch, 1)
    q = torch.randn(batch * new, 4, D, generator=torch.Generator().manual_seed(4)).half().to(dev)
    for room in ROOMS:
        got = paged_attention(q, *(wide(cache, room) if room else cache), i64([held], dev))
        for b in (0, batch - 1):
            ref, tol = exact_rows(cache, b, held, q[b * new:(b + 1) * new], [0, new // 2, new - 1])
            err = (got[[b * new, b * new + new // 2, b * new + new - 1]].double() - ref).abs()
            assert (err <= tol).all(), (room, b, (err / tol).max())

def test_rows_that_see_no_key_are_zero_whatever_lies_behind_them(dev):
    """The rows' own page is not there, and the one behind them has keys of zero or nearly: they are behind the rows all the same."""
    for dtype, D in (("int8", 128), ("e4m3", 64), ("int8", 256)):
        cache = make_cache(3, dtype, 1, D, 16, [100], dev)
        q = torch.randn(16, 4, D, generator=torch.Generator().manual_seed(4)).half().to(dev)
        first, second = int(cache[4][0, 0]), int(cache[4][0, 1])
        cache[4][0, 0] = -1
        for k_scale in (0.0, 1e-30, 1e-10, 1.0):
            cache[2][second] = k_scale
            for scale in (None, 0.0):
                for room in ROOMS:
                    c = wide(cache, room) if room else cache
                    assert not paged_attention(q, *c, i64([0], dev), scale=scale).any(), (dtype, D, k_scale, scale, room)


def test_keys_behind_a_row_stay_hidden_however_low_its_scores_are(dev):
    """Scores of -6e10, and behind the rows keys of zero, whose scores would be 0: the results are those without them.  (What the results are is not asked:
    at 6e10 a score in fp32 is rounded by 2^-24 of it, 4000, and log2 of the values' scale, which is added to it, is lost.)"""
    cache = make_cache(3, "int8", 1, 128, 16, [40], dev)
    table = cache[4][0].tolist()
    for p in table[:2]:
        cache[0][p], cache[2][p] = -127, 500.0
    cache[0][table[2]], cache[2][table[2]] = 0, 0.0
    q = torch.full((32, 4, 128), 60000.0, dtype=torch.float16, device=dev)
    for room in ROOMS:
        c = wide(cache, room) if room else cache
        without = [*c[:4], c[4].clone()]
        without[4][0, 2] = -1
        got = paged_attention(q, *c, i64([0], dev))
        assert got.any() and torch.equal(got, paged_attention(q, *without, i64([0], dev))), room


@pytest.mark.parametrize("new", [1, 12, 70])
@pytest.mark.parametrize("dtype,D", [("int8", 128), ("e4m3", 64), ("int8", 256)])
@pytest.mark.parametrize("size", [1e3, 1e6, 1e7, 3e8])
def test_scores_so_large_that_one_key_takes_all(dev, dtype, D, size, new):
    """Scores with a deviation of `size`: where the two largest are further apart than fp32 can be wrong about them (D + 16 roundings of 2^-23 of the sum of
    magnitudes, for either) by 12 at least, which leaves the second 2^-17, the row is the largest one's value.  Its weight w is rounded to fp16 as the
    product's operand and not in the sum, both of which have it relative to a maximum that may be up to 2^8 below: off by 2^-11 w / w, then by the
    exponential's and the quotient's few roundings of 2^-22 (2^-18 together), and the result by its own rounding to fp16, 2^-11."""
    held = 300
    cache = long_cache(dtype, 1, D, 32, held + new, dev)
    width = min(15000.0, size ** 0.5)
    cache[2] *= size / width
    q = (torch.randn(new, 4, D, generator=torch.Generator().manual_seed(4)).clamp(-4, 4) * width).half().to(dev)
    page = cache[4][0].long()
    k, v = ((t[page].double() * s[page].double()[:, :, None, None]).reshape(-1, D) for t, s in ((cache[0], cache[2]), (cache[1], cache[3])))
    e = torch.einsum("nhd,td->nht", q.double(), k) * D ** -0.5
    far = torch.einsum("nhd,td->nht", q.double().abs(), k.abs()).amax(dim=-1) * D ** -0.5 * (D + 16) * 2.0 ** -23 * 2 + 12
    e = e.masked_fill(torch.arange(len(k), device=dev) > held + torch.arange(new, device=dev)[:, None, None], -torch.inf)
    top = e.topk(2, dim=-1)
    sure = top.values[..., 0] - top.values[..., 1] > far
    assert sure.double().mean() > 0.8
    want = v[top.indices[..., 0]]
    # (what the second and all others add: 2^-17 of 400 values of one, at the very most; nothing at all from 1e6 on)
    bound = (2 * 2.0 ** -11 + 2.0 ** -18) * want.abs() + 2.0 ** -25 + (2.0 ** -17 * 2 * v.abs().amax() if size < 1e6 else 0.0)
    for room in ROOMS:
        got = paged_attention(q, *(wide(cache, room) if room else cache), i64([held], dev))
        assert got.isfinite().all() and ((got.double() - want).abs() <= bound)[sure].all(), room


def test_keys_behind_a_row_stay_hidden_however_low_its_scores_are(dev):
    """Scores of -6e10, and behind the rows keys of zero, whose scores would be 0: the results are those without them.  (What the results are is not asked:
    at 6e10 a score in fp32 is rounded by 2^-24 of it, 4000, and log2 of the values' scale, which is added to it, is lost.)"""
    cache = make_cache(3, "int8", 1, 128, 16, [40], dev)
    table = cache[4][0].tolist()
    for p in table[:2]:
        cache[0][p], cache[2][p] = -127, 500.0
    cache[0][table[2]], cache[2][table[2]] = 0, 0.0
    q = torch.full((32, 4, 128), 60000.0, dtype=torch.float16, device=dev)
    for room in ROOMS:
        c = wide(cache, room) if room else cache
        without = [*c[:4], c[4].clone()]
        without[4][0, 2] = -1
        got = paged_attention(q, *c, i64([0], dev))
        assert got.any() and torch.equal(got, paged_attention(q, *without, i64([0], dev))), room


# ---- host side -------------------------------------------------------------------------------------------------------------------

def test_a_cache_without_heads_is_refused(dev):
    from glorcq_b200.paged_cache import paged_append, paged_read
    cache = [torch.zeros(4, 0, 16, 64, dtype=torch.int8, device=dev) for _ in range(2)] + [torch.zeros(4, 0, device=dev) for _ in range(2)] + \
            [torch.zeros(1, 4, dtype=torch.int32, device=dev)]
    for n in (0, 1):
        q, k = torch.zeros(n, 4, 64, device=dev).half(), torch.zeros(n, 0, 64, device=dev).half()
        for call in (lambda: paged_attention(q, *cache, i64([0], dev)), lambda: paged_append(q, k, k, None, None, *cache, i64([0], dev)),
                     lambda: paged_read(*cache, i64([0], dev), None, n)):
            with pytest.raises(RuntimeError, match="one head or more"):
                call()


@pytest.mark.parametrize("kv_cache", ["static", "int8", "e4m3"])
def test_capturing_a_step_leaves_the_cache_as_it_was(dev, kv_cache):
    """A prompt in the cache, then capture_graph(): its warm-up steps write positions 0 and 10, the first of which gives a block a new scale."""
    from glorcq_b200.graph_wrapper import GLoRCQGraphWrapper
    from glorcq_b200.synthetic import make_decoder
    m = make_decoder(SMALL, dev, seed=3, rank=16, attn_rank=16)
    w = GLoRCQGraphWrapper(m, max_batch_size=2, max_seq_len=64, kv_cache=kv_cache, page_size=16)
    ids = torch.randint(0, 512, (2, 30), generator=torch.Generator().manual_seed(1)).to(dev)
    with torch.no_grad():
        m(input_ids=ids, cache_position=torch.arange(30, device=dev), past_key_values=w.static_cache)
        c = w.static_cache
        tensors = [c.k, c.v] if kv_cache == "static" else [c.k.view(torch.uint8), c.v.view(torch.uint8), c.k_scale, c.v_scale]
        before = [t.clone() for t in tensors]
        w.capture_graph()
        assert all(torch.equal(a, b) for a, b in zip(tensors, before))
        # and the captured step reads that prompt
        got = w.replay(ids[:, :1], 30).clone()
        for t, x in zip(tensors, before):
            t.copy_(x)
        want = m(input_ids=ids[:, :1], cache_position=torch.tensor([30], device=dev), past_key_values=c)[0]
        assert torch.equal(got, want)


def test_numbers_of_rows_that_go_back_and_forth_end_the_call(dev):
    """q_start must not decrease, and lies on the device: a call that is given such numbers ends, and writes nothing outside its rows and its pages."""
    import random
    from glorcq_b200 import tiled
    from glorcq_b200.paged_cache import paged_append, paged_read
    r = random.Random(1)
    cache = long_cache("int8", 2, 128, 16, 640, dev)
    spare = cache[0].shape[0]
    cache = [torch.cat((t, t[:1])) for t in cache[:4]] + [cache[4]]
    kept = [t[spare].clone() for t in cache[:4]]
    for n in range(60):
        B, N = r.choice([2, 9, 30, 700]), r.choice([20, 100, 400])
        qs = torch.tensor([r.randint(-5, N + 5) for _ in range(B + 1)], dtype=torch.int32, device=dev)
        table = cache[4].repeat(B, 1)
        start = i64([r.randint(0, 600) for _ in range(B)], dev)
        q = torch.randn(N, 4, 128, device=dev).half()
        for room in ROOMS[:2 if B > 100 else 3]:
            out = torch.full((N + 20, 4, 128), 7.0, dtype=torch.float16, device=dev)
            c = [*cache[:4], table]
            paged_attention(q, *(wide(c, room) if room else c), start, qs, max_new=r.choice([None, N]), out=out[10:-10])
            assert (out[:10] == 7).all() and (out[-10:] == 7).all()
        out = torch.full((N + 20, 4, 128), 7.0, dtype=torch.float16, device=dev)
        paged_append(q, q[:, :2], q[:, 2:], None, None, *c, start, qs, q_out=out[10:-10])
        assert (out[:10] == 7).all() and (out[-10:] == 7).all()
        paged_read(*c, start, qs, N)
    assert all(torch.equal(t[spare].view(torch.uint8), k.view(torch.uint8)) for t, k in zip(cache[:4], kept))
    assert tiled.debug_error() is None
