"""Plain 64-bit restatements of the serving operators, and random paged caches to run them on (CPU tensors)."""
import math

import torch

U32 = 2.0 ** -24            # half a step of fp32, relative
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U32}


def up(a, b):
    return -(-a // b)


def plan_ref(lens, new, table, ring, pool, page, max_tokens):
    """The rules of one step in plain Python, one request after another.  Lists in, a dict of lists out."""
    n, (head, count), width = len(ring), pool, len(table[0])
    status, taken, given, tokens = 0, 0, 0, 0
    for length, add in zip(lens, new):
        if length < 0:
            status |= 8
        elif length > width * page or (add >= 0 and length + add > width * page):
            status |= 2
        elif add < 0:
            given += up(length, page)
        else:
            taken += up(length + add, page) - up(length, page)
            tokens += add
    if not 0 <= head < n or not 0 <= count <= n or count + given > n:
        status |= 8
    status |= (1 if taken > count else 0) | (4 if tokens > max_tokens else 0)
    if status:
        return dict(table=table, ring=ring, lens=lens, pool=pool, q_start=[0] * (len(lens) + 1), slots=[-1] * max_tokens,
                    positions=[0] * max_tokens, status=status)
    table, ring = [list(r) for r in table], list(ring)
    after, q_start, slots, positions = [], [0], [], []
    k = g = 0
    for b, (length, add) in enumerate(zip(lens, new)):
        if add < 0:
            for j in range(up(length, page)):
                ring[(head + count + g) % n] = table[b][j]
                g += 1
        else:
            for j in range(up(length, page), up(length + add, page)):
                table[b][j] = ring[(head + k) % n]
                k += 1
            for t in range(length, length + add):
                slots.append(table[b][t // page] * page + t % page)
                positions.append(t)
        after.append(0 if add < 0 else length + add)
        q_start.append(q_start[-1] + max(add, 0))
    pad = max_tokens - len(slots)
    return dict(table=table, ring=ring, lens=after, pool=[(head + k) % n, count - k + g], q_start=q_start, slots=slots + [-1] * pad,
                positions=positions + [0] * pad, status=0)


class Cache:
    """Random pages for requests of the given lengths; whatever belongs to nobody holds ``filler``."""

    def __init__(self, lens, H, D, page, dtype, g, *, filler=float("nan"), layout="heads", spare=3, width=None):
        used = sum(up(n, page) for n in lens)
        self.lens, self.page = lens, page
        n_pages = used + spare
        order = torch.randperm(n_pages, generator=g).to(torch.int32)
        width = width or max(1, max(up(n, page) for n in lens))
        self.table = torch.full((len(lens), width), -7, dtype=torch.int32)
        shape = (n_pages, 2, H, page, D) if layout == "heads" else (n_pages, H, 2, page, D)
        kv = torch.full(shape, filler, dtype=dtype)
        self.kv = kv
        self.k_pages, self.v_pages = (kv[:, 0], kv[:, 1]) if layout == "heads" else (kv[:, :, 0], kv[:, :, 1])
        self.k, self.v, at = [], [], 0
        for b, n in enumerate(lens):
            ids = order[at:at + up(n, page)]
            at += len(ids)
            self.table[b, :len(ids)] = ids
            k, v = torch.randn(n, H, D, generator=g).to(dtype), torch.randn(n, H, D, generator=g).to(dtype)
            self.k.append(k)
            self.v.append(v)
            for j in range(n):
                self.k_pages[ids[j // page], :, j % page] = k[j]
                self.v_pages[ids[j // page], :, j % page] = v[j]

    def views(self, dev):
        """(k_pages, v_pages) of a copy on the GPU, with the same strides."""
        kv = self.kv.to(dev)
        return (kv[:, 0], kv[:, 1]) if self.k_pages.stride(1) == kv.stride(2) else (kv[:, :, 0], kv[:, :, 1])


def attn_ref(q, k, v, scale, causal, dtype):
    """q [n, Hq, D], k / v [L, Hk, D] of one request -> (o, bound) in fp64.  The bound on |result - o| follows the kernel's
    roundings: a score is a sum of D products (D + 3 half steps of fp32 of the sum of their magnitudes, scaled), the
    exponential adds four half steps, the sums over L keys L + D each, and bf16 rounds every probability and the result."""
    n, Hq, D = q.shape
    L, Hk = k.shape[:2]
    q, k, v = q.double(), k.double(), v.double()
    o, bound = torch.zeros(n, Hq, D, dtype=torch.float64), torch.zeros(n, Hq, D, dtype=torch.float64)
    half = HALF[dtype]
    see = torch.ones(n, L, dtype=torch.bool)
    if causal:
        see = torch.arange(L)[None] <= (L - n + torch.arange(n))[:, None]
    for h in range(Hq):
        kh, vh = k[:, h * Hk // Hq], v[:, h * Hk // Hq]
        if L == 0:
            continue
        x = (q[:, h] @ kh.t()) * scale
        x = x.masked_fill(~see, -math.inf)
        alive = see.any(1)
        p = torch.where(alive[:, None], torch.softmax(x, 1), torch.zeros_like(x))
        val = torch.where(see[:, :, None], vh[None], torch.zeros_like(vh[None]))            # unseen keys count for nothing
        mag = torch.where(see, (q[:, h].abs() @ kh.abs().t()) * abs(scale), torch.zeros_like(x))
        e = ((D + 3) * U32 * mag).amax(1, keepdim=True) + 4 * U32
        o[:, h] = torch.bmm(p[:, None], val)[:, 0]
        pv = torch.bmm(p[:, None], val.abs())[:, 0]
        probs = half if dtype == torch.bfloat16 else 0.0
        bound[:, h] = (2 * e + 2 * (L + D) * U32 + probs) * pv + half * o[:, h].abs() + 1e-30
    return o, bound * 1.01
