"""The operators of the paged 8-bit key/value cache, as cases that can be timed and compared.

Three kinds, each through the entry point a program calls:

  append   new keys and values of a batch into the cache, position rotation (and the per-head norms of some models) applied on
           the way, queries rotated too; the rows of the pages that changed are read back
  attend   attention of the new tokens over the cache: one token a sequence, or a part of a prompt behind what is there
  read     rows of the cache as fp16

A page holds `page` tokens of every key/value head as (heads, tokens, channels) codes, int8 or e4m3, with one fp32 scale for
the keys and one for the values of each (page, head).  Sequence b holds start[b] tokens before the call and gets
q_start[b] .. q_start[b + 1] of the batch's rows; pages are handed out in no order.

A block's scale is the largest finite magnitude of its values over the code's largest value (127 or 448).  A block that a call adds to
keeps its scale while that covers the new values, and otherwise has it doubled until it does, the codes that are there halved with it."""

import math
import random

import torch

own = False

QMAX = {"int8": 127.0, "e4m3": 448.0}
EPS = 1e-6


def _case(name, kind, heads, kv, dim, page, dtype, batch, tokens, context, ragged=False, norm=False):
    return {"name": name, "kind": kind, "heads": heads, "kv": kv, "dim": dim, "page": page, "dtype": dtype, "batch": batch, "tokens": tokens,
            "context": context, "ragged": ragged, "norm": norm}


def listed():
    return [
        # one layer of a decoded token, 16 heads with their own keys, after a 512-token prompt: the smallest calls
        _case("append-decode-1", "append", 16, 16, 128, 64, "int8", 1, 1, 512),
        _case("attend-decode-1", "attend", 16, 16, 128, 64, "int8", 1, 1, 512),
        # a decode batch of sequences of their own lengths: 32 heads on 4, per-head norms; 32 heads on 8
        _case("append-decode-64", "append", 32, 4, 128, 32, "e4m3", 64, 1, 2048, ragged=True, norm=True),
        _case("attend-decode-16", "attend", 32, 8, 128, 32, "e4m3", 16, 1, 1024, ragged=True),
        # a serving batch over long caches, and one sequence over a very long one
        _case("attend-decode-64-long", "attend", 32, 4, 128, 64, "int8", 64, 1, 8192, ragged=True),
        _case("attend-decode-1-long", "attend", 32, 8, 128, 64, "int8", 1, 1, 131000),
        # a long prompt into an empty cache
        _case("append-prompt-4096", "append", 32, 8, 128, 64, "int8", 1, 4096, 0),
        _case("attend-prompt-4096", "attend", 32, 4, 128, 64, "int8", 1, 4096, 0),
        # the benchmark's prompt length
        _case("attend-prompt-512", "attend", 16, 16, 128, 64, "int8", 1, 512, 0),
        # pieces of prompts, odd in length, behind what four sequences hold already
        _case("attend-chunk-4", "attend", 32, 8, 128, 16, "e4m3", 4, 700, 2900, ragged=True),
        # one sequence's cache handed on as fp16 rows; a few rows of many sequences
        _case("read-4096", "read", 32, 8, 128, 64, "int8", 1, 4096, 0),
        _case("read-33", "read", 32, 4, 128, 16, "e4m3", 33, 19, 300, ragged=True),
    ]


def lengths(case):
    """([tokens a sequence holds before the call], [new tokens]): they go by the case alone."""
    if not case["ragged"]:
        return [case["context"]] * case["batch"], [case["tokens"]] * case["batch"]
    rng = random.Random(case["batch"] * 1000003 + case["context"] * 31 + case["tokens"])
    start = [int(case["context"] * rng.uniform(0.1, 1.0)) for _ in range(case["batch"])]
    new = [case["tokens"] if case["tokens"] == 1 else rng.randint(1, case["tokens"]) for _ in range(case["batch"])]
    return start, new


def _spread(rng, lo, hi):
    """From lo to hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _fits(case):
    """No more than the largest listed cases read, compute and (in the plain form) hold."""
    start, new = lengths(case)
    held = [s + n for s, n in zip(start, new)]
    if case["kind"] != "attend":
        return sum(new) * (case["heads"] + 2 * case["kv"]) * case["dim"] <= 4096 * 48 * 128 and sum(held) * case["kv"] * case["dim"] <= 1 << 27
    padded = case["batch"] * case["heads"] * max(new) * max(held)
    return work(case)["flops"] <= 137e9 and sum(held) * case["kv"] * case["dim"] <= 131001 * 8 * 128 \
        and padded <= 5.4e8 and case["batch"] * max(held) * case["kv"] * case["dim"] <= 2.8e8


def draw(rng):
    while True:
        kind = rng.choice(("append", "attend", "attend", "attend", "read"))
        kv, group = rng.choice((1, 2, 4, 8, 16)), rng.choice((1, 2, 3, 4, 5, 6, 7, 8, 12, 16))
        if kv * group > 64:
            continue
        case = {"kind": kind, "heads": kv * group, "kv": kv, "dim": rng.choice((64, 128, 128, 128, 256)), "page": rng.choice((16, 32, 64, 128)),
                "dtype": rng.choice(("int8", "e4m3")), "batch": _spread(rng, 1, 128), "ragged": rng.random() < 0.7, "norm": kind == "append" and rng.random() < 0.3}
        if rng.random() < 0.5:
            case |= {"tokens": 1, "context": _spread(rng, 1, 131000)}
        else:
            case |= {"tokens": _spread(rng, 2, 4096), "context": rng.choice((0, _spread(rng, 1, 8192)))}
        if kind == "read" and case["tokens"] == 1:
            continue
        if _fits(case):
            return case


def _quantized(x, dtype):
    """(codes, scales) of blocks (pages, heads, tokens, channels)."""
    s = x.abs().amax(dim=(2, 3)).float() / QMAX[dtype]
    y = x * (1.0 / s).clamp(max=1e30)[:, :, None, None]
    return (y.round().to(torch.int8) if dtype == "int8" else y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)), s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    D, P, KV, H, B = case["dim"], case["page"], case["kv"], case["heads"], case["batch"]
    start, new = lengths(case)
    pages = [(s + n + P - 1) // P for s, n in zip(start, new)]
    width, pool = max(pages) + 1, sum(pages) + 3
    order = random.Random(seed).sample(range(pool), pool)
    table = torch.zeros(B, width, dtype=torch.int32)
    at = 0
    for b in range(B):
        table[b, : pages[b]] = torch.tensor(order[at : at + pages[b]], dtype=torch.int32)
        at += pages[b]

    def rows(n, heads, width=1.0):
        # a few channels are larger than the others, as in trained models
        c = torch.exp(0.5 * torch.randn(heads, D, generator=g, device=dev))
        return (torch.randn(n, heads, D, generator=g, device=dev) * c * width).half()

    def blocks():
        c = torch.exp(0.5 * torch.randn(KV, 1, D, generator=g, device=dev))
        codes = torch.empty(pool, KV, P, D, dtype=torch.int8 if case["dtype"] == "int8" else torch.float8_e4m3fn, device=dev)
        scale = torch.empty(pool, KV, dtype=torch.float32, device=dev)
        step = max(1, (1 << 26) // (KV * P * D))
        for i in range(0, pool, step):
            n = min(step, pool - i)
            codes[i : i + n], scale[i : i + n] = _quantized(torch.randn(n, KV, P, D, generator=g, device=dev) * c, case["dtype"])
        return codes, scale

    N = sum(new)
    s = {"case": dict(case), "B": B, "P": P, "qmax": QMAX[case["dtype"]], "table": table.to(dev), "max_new": max(new)}
    s["k_pages"], s["k_scale"] = blocks()
    s["v_pages"], s["v_scale"] = blocks()
    s["start"] = torch.tensor(start, dtype=torch.int64, device=dev)
    s["q_start"] = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev)
    seq = torch.tensor([b for b in range(B) for _ in range(new[b])], dtype=torch.int64, device=dev)
    s["seq"], s["pos"] = seq, torch.tensor([start[b] + i for b in range(B) for i in range(new[b])], dtype=torch.int64, device=dev)
    if case["kind"] == "attend":
        s["q"] = rows(N, H, 0.8)
        s["held"] = max(a + n for a, n in zip(start, new))
    elif case["kind"] == "read":
        s["rows"] = N
    else:
        s["q"], s["k"], s["v"] = rows(N, H), rows(N, KV), rows(N, KV)
        if case["norm"]:
            s["q_norm"], s["k_norm"] = ((1 + 0.2 * torch.randn(D, generator=g, device=dev)).half() for _ in range(2))
        angle = torch.arange(width * P, dtype=torch.float64, device=dev)[:, None] * 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        # the pages that the call changes, the first slot in each that it writes, and whose page each new row lands in
        touched = [(b, j) for b in range(B) for j in range(start[b] // P, (start[b] + new[b] + P - 1) // P)]
        index = {t: i for i, t in enumerate(touched)}
        s["touched"] = torch.tensor([int(table[b, j]) for b, j in touched], dtype=torch.int64, device=dev)
        s["begins"] = torch.tensor([max(0, start[b] - j * P) for b, j in touched], dtype=torch.int64, device=dev)
        s["row_page"] = torch.tensor([index[b, (start[b] + i) // P] for b in range(B) for i in range(new[b])], dtype=torch.int64, device=dev)
        # rows read back: from the beginning of the first changed page on
        first = [a // P * P for a in start]
        count = [a + n - f for a, n, f in zip(start, new, first)]
        s["first"] = torch.tensor(first, dtype=torch.int64, device=dev)
        s["first_start"] = torch.tensor([sum(count[:b]) for b in range(B + 1)], dtype=torch.int32, device=dev)
        s["rows"] = sum(count)
        s["back_seq"] = torch.tensor([b for b in range(B) for _ in range(count[b])], dtype=torch.int64, device=dev)
        s["back_pos"] = torch.tensor([first[b] + i for b in range(B) for i in range(count[b])], dtype=torch.int64, device=dev)
    return s


def _values(s, name, seq, pos):
    page = s["table"][seq, pos // s["P"]].long()
    return (s[name + "_pages"][page, :, pos % s["P"]].float() * s[name + "_scale"][page][:, :, None]).half()


def _normed(x, w):
    return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w.float()


def _rotated(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _add_rows(s, name, x):
    """The rows x (N, heads, channels) into the pages of `name`."""
    pages, scales, at, qmax = s[name + "_pages"], s[name + "_scale"], s["touched"], s["qmax"]
    size = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(dim=-1)
    need = torch.zeros(at.numel(), x.shape[1], device=x.device).scatter_reduce_(0, s["row_page"][:, None].expand_as(size), size, "amax") / qmax
    old = scales[at]
    fresh = (s["begins"] == 0)[:, None] | (old <= 0)
    m0, e0 = torch.frexp(old)
    m1, e1 = torch.frexp(need)
    k = torch.where(fresh | (need <= old), torch.zeros_like(e0), e1 - e0 + (m1 > m0).int())
    scale = torch.where(fresh, need, torch.ldexp(old, k))
    kept = torch.ldexp(pages[at].float(), -k[:, :, None, None])
    inv = torch.where(scale > 0, 1.0 / scale, torch.zeros_like(scale))
    y = (x * inv[s["row_page"]][:, :, None]).clamp(-qmax, qmax)
    y = torch.where(y.isnan(), torch.zeros_like(y), y)
    if pages.dtype == torch.int8:
        kept, y = kept.round(), y.round()
    codes = torch.where((torch.arange(s["P"], device=x.device) < s["begins"][:, None])[:, None, :, None], kept.to(pages.dtype).float(), pages[at].float())
    codes[s["row_page"], :, s["pos"] % s["P"]] = y.to(pages.dtype).float()
    pages[at] = codes.to(pages.dtype)
    scales[at] = scale


def _append(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if "q_norm" in s:
        q, k = _normed(q, s["q_norm"]), _normed(k, s["k_norm"])
    cos, sin = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
    _add_rows(s, "k", _rotated(k, cos, sin))
    _add_rows(s, "v", v)
    return _rotated(q, cos, sin).half(), _values(s, "k", s["back_seq"], s["back_pos"]), _values(s, "v", s["back_seq"], s["back_pos"])


def _attend(s):
    c, P = s["case"], s["P"]
    B, KV, D, G = c["batch"], c["kv"], c["dim"], c["heads"] // c["kv"]
    table = s["table"][:, : (s["held"] + P - 1) // P].long()

    def held(name):
        x = s[name + "_pages"][table].float() * s[name + "_scale"][table][..., None, None]
        return x.transpose(1, 2).reshape(B, KV, table.shape[1] * P, D)

    step = s["pos"] - s["start"][s["seq"]]
    q = torch.zeros(B, s["max_new"], KV, G, D, device=table.device)
    q[s["seq"], step] = s["q"].float().view(-1, KV, G, D)
    q = q.permute(0, 2, 1, 3, 4).reshape(B, KV, s["max_new"] * G, D)
    score = torch.matmul(q, held("k").transpose(2, 3)).mul_(D ** -0.5).view(B, KV, s["max_new"], G, -1)
    last = s["start"][:, None] + torch.arange(s["max_new"], device=table.device)
    hidden = torch.arange(score.shape[-1], device=table.device) > last[:, :, None]
    score.masked_fill_(hidden[:, None, :, None], -math.inf)
    score.sub_(score.amax(dim=-1, keepdim=True)).exp_()
    score.div_(score.sum(dim=-1, keepdim=True))
    y = torch.matmul(score.view(B, KV, s["max_new"] * G, -1), held("v")).view(B, KV, s["max_new"], G, D)
    return y[s["seq"], :, step].reshape(-1, KV * G, D).half()


def run(s):
    kind = s["case"]["kind"]
    if own:
        from glorcq_b200.paged_cache import paged_append, paged_attention, paged_read
        cache = (s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"], s["table"])
        if kind == "append":
            q = paged_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], *cache, s["start"], s["q_start"], q_norm=s.get("q_norm"),
                             k_norm=s.get("k_norm"), eps=EPS)
            return (q, *paged_read(*cache, s["first"], s["first_start"], s["rows"]))
        if kind == "attend":
            return paged_attention(s["q"], *cache, s["start"], s["q_start"], max_new=s["max_new"])
        return paged_read(*cache, s["start"], s["q_start"], s["rows"])
    if kind == "append":
        return _append(s)
    if kind == "attend":
        return _attend(s)
    return _values(s, "k", s["seq"], s["pos"]), _values(s, "v", s["seq"], s["pos"])


def work(case):
    start, new = lengths(case)
    D, KV, H, P, N = case["dim"], case["kv"], case["heads"], case["page"], sum(new)
    if case["kind"] == "read":
        return {"bytes": 2 * N * KV * D * 3, "flops": 2 * N * KV * D}
    if case["kind"] == "append":
        back = sum(a + n - a // P * P for a, n in zip(start, new))
        touched = sum((a + n + P - 1) // P - a // P for a, n in zip(start, new))
        positions = len({p for a, n in zip(start, new) for p in range(a, a + n)})
        return {"bytes": 4 * N * H * D + 6 * N * KV * D + 4 * positions * D + 16 * touched * KV + 6 * back * KV * D,
                "flops": 4 * N * (H + KV) * D + 4 * N * KV * D + 2 * back * KV * D}
    pairs = sum(n * a + n * (n + 1) // 2 for a, n in zip(start, new))
    held = sum(a + n for a, n in zip(start, new))
    pages = sum((a + n + P - 1) // P for a, n in zip(start, new))
    return {"bytes": 2 * held * KV * D + 8 * pages * KV + 4 * pages + 4 * N * H * D, "flops": 4 * pairs * H * D}


# ---- the same from the definitions, in 64 bits --------------------------------------------------------------------------------


def _to_code(y, dtype):
    if dtype == "int8":
        return torch.round(y).clamp(-127, 127)
    unit = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)     # three bits behind the leading one, none below 2^-6
    return (torch.round(y / unit) * unit).clamp(-448, 448)


def _exact_append(case, s, start, new):
    P, dtype, D = case["page"], case["dtype"], case["dim"]

    def turned(x, weight, pos):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS) * weight.double()
        cos, sin = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
        y = torch.empty_like(x)
        y[..., : D // 2] = x[..., : D // 2] * cos - x[..., D // 2 :] * sin
        y[..., D // 2 :] = x[..., D // 2 :] * cos + x[..., : D // 2] * sin
        return y

    q = turned(s["q"], s.get("q_norm"), s["pos"])
    keys, out, at = turned(s["k"], s.get("k_norm"), s["pos"]), {"k": [], "v": []}, 0
    for b in range(case["batch"]):
        for name, x in (("k", keys), ("v", s["v"].double())):
            for page in range(start[b] // P, (start[b] + new[b] + P - 1) // P):
                lo, hi = max(start[b], page * P), min(start[b] + new[b], (page + 1) * P)
                rows = x[at + lo - start[b] : at + hi - start[b]].transpose(0, 1)               # heads, tokens, channels
                need = rows.abs().amax(dim=(1, 2)) / QMAX[dtype]
                scale = need
                if lo > page * P:
                    phys = int(s["table"][b, page])
                    old = s[name + "_scale"][phys].double()
                    doubled = torch.ceil(torch.log2(need / old)).clamp(min=0)
                    scale = torch.where(old > 0, old * torch.exp2(doubled), need)
                    codes = _to_code(s[name + "_pages"][phys, :, : lo - page * P].double() * (old / scale)[:, None, None], dtype)
                    out[name].append((codes * scale[:, None, None]).transpose(0, 1))
                out[name].append((_to_code(rows / scale[:, None, None], dtype) * scale[:, None, None]).transpose(0, 1))
        at += new[b]
    return q, torch.cat(out["k"]), torch.cat(out["v"])


def _exact_attend(case, s, start, new):
    P, KV, G = case["page"], case["kv"], case["heads"] // case["kv"]
    out, at = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device), 0
    for b in range(case["batch"]):
        n, held = new[b], start[b] + new[b]
        ids = s["table"][b, : (held + P - 1) // P].long()
        for h in range(KV):
            k, v = ((s[x + "_pages"][ids, h].double() * s[x + "_scale"][ids, h].double()[:, None, None]).reshape(-1, case["dim"])[:held] for x in "kv")
            step = max(1, (1 << 26) // (held * G))
            for i in range(0, n, step):
                m = min(step, n - i)
                q = s["q"][at + i : at + i + m, h * G : (h + 1) * G].double()
                e = torch.einsum("ngd,td->ngt", q, k) / math.sqrt(case["dim"])
                e = e.masked_fill((torch.arange(held, device=k.device)[None] > start[b] + i + torch.arange(m, device=k.device)[:, None])[:, None], -math.inf)
                out[at + i : at + i + m, h * G : (h + 1) * G] = torch.einsum("ngt,td->ngd", torch.softmax(e, dim=-1), v)
        at += n
    return out


def exact(case, seed):
    s = prepare(case, seed)
    start, new = lengths(case)
    if case["kind"] == "append":
        return _exact_append(case, s, start, new)
    if case["kind"] == "attend":
        return _exact_attend(case, s, start, new)
    P, out = case["page"], {"k": [], "v": []}
    for b in range(case["batch"]):
        for page in range(start[b] // P, (start[b] + new[b] + P - 1) // P):
            phys, lo, hi = int(s["table"][b, page]), max(start[b] - page * P, 0), min(start[b] + new[b] - page * P, P)
            for name in "kv":
                out[name].append((s[name + "_pages"][phys, :, lo:hi].double() * s[name + "_scale"][phys].double()[:, None, None]).transpose(0, 1))
    return torch.cat(out["k"]), torch.cat(out["v"])
