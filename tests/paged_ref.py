"""The paged 8-bit cache from its definitions (include/glorcq_b200.h), plainly and on the CPU: a class that holds pages and does one token
and one head at a time what the kernels do, in 32 bits where codes are decided, in 64 bits elsewhere."""

import math

import torch

QMAX = {"int8": 127.0, "e4m3": 448.0}
TYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def to_code(y, dtype):
    """fp32 values / scale -> codes as fp32 numbers."""
    y = torch.nan_to_num(y.clamp(-QMAX[dtype], QMAX[dtype]), nan=0.0)
    return y.round() if dtype == "int8" else y.to(torch.float8_e4m3fn).float()


def rotated(x, cos, sin, pos):
    """fp32 rows (..., D) at the positions pos (...), products and sums rounded one by one."""
    h = x.shape[-1] // 2
    c, s = cos[pos], sin[pos]
    a, b = x[..., :h], x[..., h:]
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def normed(x, w, eps):
    x = x.double()
    return (x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()).float()


class Pages:
    """codes (fp32 numbers) and scales of keys and values, CPU copies of a cache's tensors."""

    def __init__(self, cache):
        self.dtype = "int8" if cache[0].dtype == torch.int8 else "e4m3"
        self.codes = [t.cpu().float() for t in cache[:2]]
        self.scale = [t.cpu().clone() for t in cache[2:4]]
        self.table = cache[4].cpu()
        self.P = self.codes[0].shape[2]

    def phys(self, b, j):
        p = int(self.table[b, j]) if j < self.table.shape[1] else -1
        return p if 0 <= p < self.codes[0].shape[0] else None

    def append(self, which, b, start, rows):
        """rows (n, heads, D) fp32 at positions start, start + 1, ..."""
        if len(rows) == 0:
            return
        for j in range(start // self.P, (start + len(rows) + self.P - 1) // self.P):
            p = self.phys(b, j)
            if p is None:
                continue
            lo, hi = max(start - j * self.P, 0), min(start + len(rows) - j * self.P, self.P)
            new = rows[j * self.P + lo - start: j * self.P + hi - start]
            for h in range(new.shape[1]):
                x, codes = new[:, h], self.codes[which][p, h]
                size = torch.where(x.isfinite(), x.abs(), torch.zeros(()))
                need, old = size.max() / QMAX[self.dtype], self.scale[which][p, h].clone()
                s = need
                if lo > 0 and old > 0:
                    s, n = old, 0
                    while s < need:
                        s, n = s * 2, n + 1
                    if n:
                        codes[:lo] = to_code(codes[:lo] * 2.0 ** -n, self.dtype)
                inv = 1 / s if s > 0 else torch.zeros(())
                codes[lo:hi] = to_code(x * inv, self.dtype)
                self.scale[which][p, h] = s

    def values(self, which, b, first, count):
        """(count, heads, D) 64-bit values of positions first .., None where there is no page."""
        out = []
        for t in range(first, first + count):
            p = self.phys(b, t // self.P)
            out.append(None if p is None else self.codes[which][p, :, t % self.P].double() * self.scale[which][p].double()[:, None])
        return out


def attention(pages, b, start, q, scale=None, capacity=None):
    """(n, heads, D) fp16 rows at positions start .. -> (64-bit result, bound of a kernel's error) for rows that see a key.

    The bound: one rounding of the result to fp16 (2^-11 of it) and one of each probability (2^-11 of what it contributes), and a relative error of
    each probability by those of its score -- fp32 sums of D exact products and a few fp32 roundings, (D + 16) 2^-23 of the sum of magnitudes --
    and of the exponential and the sums, 2^-18, each of them twice, since they are in the normaliser too.  A probability is rounded as what it
    weighs, p vs, relative to the largest of these, which is at least 1 when a number of fp16 may be subnormal: half of its step, 2^-25, is
    the least error whatever the probability, times the code that it multiplies."""
    D, heads = q.shape[-1], q.shape[1]
    scale = D ** -0.5 if scale is None else scale
    capacity = pages.table.shape[1] * pages.P if capacity is None else capacity
    total = min(start + len(q), capacity)
    k, v = (pages.values(i, b, 0, total) for i in (0, 1))
    there = [t for t in range(total) if k[t] is not None]
    out, tol = torch.zeros(len(q), heads, D, dtype=torch.float64), torch.zeros(len(q), heads, D, dtype=torch.float64)
    if not there:
        return out, tol
    K, V, at = torch.stack([k[t] for t in there]), torch.stack([v[t] for t in there]), torch.tensor(there)
    VS = torch.stack([pages.scale[1][pages.phys(b, t // pages.P)].double() for t in there])
    for h in range(heads):
        kh, vh = K[:, h // (heads // K.shape[1])], V[:, h // (heads // K.shape[1])]
        x = q[:, h].double()
        e = x @ kh.T * scale
        e = e.masked_fill(at[None] > (start + torch.arange(len(q)))[:, None], -math.inf)
        seen = e.isfinite().any(dim=1)
        p = torch.softmax(e[seen], dim=1)
        out[seen, h] = p @ vh
        size = (x.abs() @ kh.abs().T).max(dim=1).values[seen] * scale
        rel = 2.0 ** -11 + 2 * ((D + 16) * 2.0 ** -23 * size + 2.0 ** -18)
        vs = VS[:, h // (heads // K.shape[1])]
        codes = (vh / torch.where(vs > 0, vs, torch.ones(()))[:, None]).abs()
        floor = 2.0 ** -25 * (p * vs).max(dim=1).values[:, None] * ((p > 0).double() @ codes)
        tol[seen, h] = 2.0 ** -11 * out[seen, h].abs() + rel[:, None] * (p @ vh.abs()) + floor + 2.0 ** -25
    return out, tol


def make_cache(seed, dtype, kv, D, P, lengths, dev, spare=3, width=None, pool=None, order=None):
    """A cache that holds `lengths` random tokens: pages in random order, unused pages and slots full of bytes that stand for nothing."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + P - 1) // P for n in lengths]
    pool = sum(need) + spare if pool is None else pool
    width = max(need + [1]) + 1 if width is None else width
    ids = torch.randperm(pool, generator=g).tolist() if order is None else order
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    codes = [torch.randint(0, 256, (pool, kv, P, D), generator=g, dtype=torch.uint8) for _ in range(2)]
    scale = [torch.full((pool, kv), float("nan")) for _ in range(2)]
    at = 0
    for b, n in enumerate(lengths):
        for j in range(need[b]):
            p = ids[at]
            at += 1
            table[b, j] = p
            for i in range(2):
                x = torch.randn(kv, P, D, generator=g) * (0.5 + torch.rand(kv, 1, 1, generator=g))
                s = x.abs().amax(dim=(1, 2)) / QMAX[dtype]
                live = min(P, n - j * P)
                y = to_code(x / s[:, None, None], dtype).to(TYPES[dtype]).view(torch.uint8)
                codes[i][p, :, :live] = y[:, :live]
                scale[i][p] = s
    return [codes[0].to(dev).view(TYPES[dtype]), codes[1].to(dev).view(TYPES[dtype]), scale[0].to(dev), scale[1].to(dev), table.to(dev)]
