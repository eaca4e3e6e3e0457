"""The operators a decoder is served with, as measured cases: the plan of a paged key / value cache, the write into its
pages, attention of new tokens over them, and products with 4-bit weights.

``run`` computes a case with elementary torch operations in 32 bits, or with ``own`` through the framework's entry points;
``exact`` computes the same outputs from their definitions in 64 bits."""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------- cases ----
def listed():
    return [
        # one token for each of eight requests: what every layer stack of a small decoder waits for before it starts
        dict(name="plan 8 requests", op="plan", B=8, page=16, lo=1, hi=440, width=28, prompts=0, chunk=0, ends=0, idle=0, short=False),
        # a full server: most requests add a token, some bring a prompt, some end and give their pages back
        dict(name="plan 512 requests", op="plan", B=512, page=32, lo=1, hi=3000, width=96, prompts=64, chunk=400, ends=48, idle=20, short=False),
        # the keys and values of one token for eight requests (d_model 384: 6 heads)
        dict(name="write 8 tokens", op="write", B=8, lo=1, hi=1, H=6, D=64, page=16, dtype="bf16"),
        # the encoder's keys and values of 32 clips of 1500 frames going into the cross-attention's pages (20 heads)
        dict(name="write 32 clips", op="write", B=32, lo=1500, hi=1500, H=20, D=64, page=64, dtype="bf16"),
        # a small decoder's self-attention of one token: latency
        dict(name="attn token 8x6", op="attn", B=8, Hq=6, Hk=6, D=64, page=16, qlo=1, qhi=1, lo=5, hi=440, causal=True, dtype="bf16"),
        # the largest configuration's cross-attention of one token per request over 1500 encoder frames: a cache read
        dict(name="attn frames 64x20", op="attn", B=64, Hq=20, Hk=20, D=64, page=64, qlo=1, qhi=1, lo=1500, hi=1500, causal=False, dtype="bf16"),
        # few requests, long contexts, query heads that share keys: the work of one row has to be split over its keys
        dict(name="attn long 4x32", op="attn", B=4, Hq=32, Hk=8, D=128, page=128, qlo=1, qhi=1, lo=7001, hi=32700, causal=True, dtype="bf16"),
        # prompts in chunks on top of what is cached: matrix products
        dict(name="attn chunk 6x16", op="attn", B=6, Hq=16, Hk=4, D=64, page=64, qlo=513, qhi=2048, lo=1100, hi=8190, causal=True, dtype="bf16"),
        # 32-bit activations, ragged prompts beside single tokens
        dict(name="attn mixed f32", op="attn", B=24, Hq=8, Hk=8, D=64, page=16, qlo=1, qhi=60, lo=60, hi=448, causal=True, dtype="f32"),
        # the fused q|k|v product of a small decoder for one token
        dict(name="w4 1x1152x384", op="w4", M=1, N=1152, K=384, group=32, act=False, res=False, dtype="bf16", out="bf16"),
        # the vocabulary of a served batch, logits in 32 bits
        dict(name="w4 16x51865x1280", op="w4", M=16, N=51865, K=1280, group=64, act=False, res=False, dtype="bf16", out="f32"),
        # a wide layer for one row: the weights' bytes
        dict(name="w4 1x16384x8192", op="w4", M=1, N=16384, K=8192, group=128, act=True, res=False, dtype="bf16", out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "write", "attn", "attn", "w4", "w4"])
    if op == "plan":
        B = _log(rng, 1, 2048)
        page = rng.choice([16, 32, 64, 128, 256])
        hi = _log(rng, 4, 4000)
        prompts = rng.randint(0, B // 4)
        chunk = _log(rng, 2, max(3, min(2000, 60000 // max(1, prompts))))
        return dict(op=op, B=B, page=page, lo=1, hi=hi, width=-(-(hi + chunk) // page) + rng.randint(0, 3), prompts=prompts,
                    chunk=chunk, ends=rng.randint(0, B // 8), idle=rng.randint(0, B // 6), short=rng.random() < 0.15)
    if op == "write":
        H, D, dtype = _log(rng, 1, 32), rng.choice([64, 128]), rng.choice(["bf16", "bf16", "f32"])
        B = _log(rng, 1, 256)
        hi = _log(rng, 1, max(1, (48000 if dtype == "bf16" else 24000) * 1280 // (B * H * D)))
        return dict(op=op, B=B, lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi, H=H, D=D, page=rng.choice([16, 32, 64, 128, 256]), dtype=dtype)
    if op == "attn":
        Hk, D = _log(rng, 1, 20), rng.choice([64, 64, 128])
        Hq, dtype = Hk * rng.choice([1, 1, 2, 4, 7]), rng.choice(["bf16", "bf16", "f32"])
        kind = rng.choice(["token", "token", "few", "chunk"])
        B = _log(rng, 1, 128 if kind != "chunk" else 8)
        most = 60_000_000 // (B * Hk * D) if kind != "chunk" else 8000
        hi = _log(rng, 8, max(9, min(32000, most)))
        qhi = {"token": 1, "few": _log(rng, 2, 40), "chunk": _log(rng, 41, 1200)}[kind]
        qhi = min(qhi, hi)
        if kind == "chunk":       # no more products than the largest listed one's
            hi = max(qhi, min(hi, (250_000_000 if dtype == "bf16" else 60_000_000) // (B * qhi * Hq * (D // 64))))
        return dict(op=op, B=B, Hq=Hq, Hk=Hk, D=D, page=rng.choice([16, 32, 64, 128, 256]), qlo=1 if kind != "chunk" else (qhi + 1) // 2, qhi=qhi,
                    lo=max(qhi, hi // rng.choice([1, 2, 16])), hi=hi, causal=rng.random() < 0.7, dtype=dtype)
    K, group = _log(rng, 64, 8192), rng.choice([32, 64, 128])
    if rng.random() < 0.7:
        K = -(-K // group) * group
    M = _log(rng, 1, 64)
    N = _log(rng, 64, min(52000, 134_000_000 // K, 1_060_000_000 // (M * K)))
    res = rng.random() < 0.3
    return dict(op=op, M=M, N=N, K=K, group=group, act=rng.random() < 0.3, res=res,
                dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]), out="f32" if res else rng.choice(["bf16", "f32"]))


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, spread over their logarithm: the same for every seed, so that the work is."""
    return [int(round(lo * (hi / lo) ** ((i + 0.5) / n))) for i in range(n)] if n > 1 else [hi]


def _lens(case, rng):
    """(lengths with the new tokens, new tokens) of an attention case, in an order of the seed's."""
    pairs = list(zip(_spread(case["B"], case["lo"], case["hi"]), reversed(_spread(case["B"], case["qlo"], case["qhi"]))))
    rng.shuffle(pairs)
    return [max(a, b) for a, b in pairs], [b for _, b in pairs]


def _news(case, rng):
    """(lengths, new tokens) of a plan case: -1 for a request that ends, 0 for one that waits or for a place that is empty."""
    B, p, e, w = case["B"], case["prompts"], case["ends"], case["idle"]
    new = ([-1] * e + [0] * w + (_spread(p, 2, case["chunk"]) if p else []) + [1] * B)[:B]
    lens = _spread(B, case["lo"], case["hi"])
    lens[e:e + w:2] = [0] * len(lens[e:e + w:2])
    pairs = list(zip(lens, new))
    rng.shuffle(pairs)
    return [a for a, _ in pairs], [b for _, b in pairs]


def _up(a, b):
    return -(-a // b)


# ------------------------------------------------------------------ inputs ----
def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cdf(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _cached(case, lens, g):
    """Pages in an order of the seed's, and the table over them; a tenth of the pool belongs to nobody."""
    page, D = case["page"], case["D"]
    H = case.get("Hk", case.get("H"))
    width = max(_up(n, page) for n in lens)
    used = sum(_up(n, page) for n in lens)
    n_pages = used + max(1, used // 10)
    order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
    table = torch.zeros((len(lens), width), dtype=torch.int32, device=DEV)
    mine = (torch.arange(width, device=DEV)[None] < _i32([_up(n, page) for n in lens])[:, None])
    table[mine] = order[:used]
    kv = torch.randn((n_pages, 2, H, page, D), dtype=torch.float32 if case["dtype"] == "f32" else torch.bfloat16, device=DEV, generator=g)
    return kv[:, 0], kv[:, 1], table


def prepare(case, seed):
    rng = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    s = dict(case)
    if op == "plan":
        lens, new = _news(case, rng)
        page = case["page"]
        have = [_up(n, page) for n in lens]
        need = [_up(n + m, page) - h if m >= 0 else 0 for n, m, h in zip(lens, new, have)]
        spare = max(0, sum(need) - 1) if case["short"] else sum(need) + 37
        n_pages = sum(have) + spare
        order = torch.randperm(n_pages, device=DEV, generator=g).to(torch.int32)
        table = torch.full((case["B"], case["width"]), -1, dtype=torch.int32, device=DEV)
        mine = torch.arange(case["width"], device=DEV)[None] < _i32(have)[:, None]
        table[mine] = order[:sum(have)]
        head = rng.randrange(max(1, n_pages))
        ring = torch.full((n_pages,), -1, dtype=torch.int32, device=DEV)
        ring[(head + torch.arange(spare, device=DEV)) % n_pages] = order[sum(have):]
        tokens = sum(max(0, m) for m in new)
        s.update(lens=_i32(lens), new=_i32(new), table=table, ring=ring, pool=_i32([head, spare]),
                 lens_out=torch.zeros(case["B"], dtype=torch.int32, device=DEV), pool_out=torch.zeros(2, dtype=torch.int32, device=DEV),
                 max_tokens=_up(max(1, tokens), 8) * 8)
    elif op == "write":
        n = _spread(case["B"], case["lo"], case["hi"])
        rng.shuffle(n)
        H, D, page, dt = case["H"], case["D"], case["page"], TYPES[case["dtype"]]
        k_pages, v_pages, table = _cached(case, n, g)
        pos = torch.cat([torch.arange(x, device=DEV) for x in n])
        req = torch.repeat_interleave(torch.arange(len(n), device=DEV), torch.tensor(n, device=DEV))
        slots = (table[req, pos // page] * page + pos % page).to(torch.int32)
        qkv = torch.randn((sum(n), 3 * H * D), dtype=dt, device=DEV, generator=g)
        s.update(k_pages=k_pages, v_pages=v_pages, slots=slots, k=qkv[:, H * D:2 * H * D].unflatten(1, (H, D)), v=qkv[:, 2 * H * D:].unflatten(1, (H, D)))
    elif op == "attn":
        lens, new = _lens(case, rng)
        k_pages, v_pages, table = _cached(case, lens, g)
        q = torch.randn((sum(new), case["Hq"], case["D"]), dtype=TYPES[case["dtype"]], device=DEV, generator=g)
        s.update(k_pages=k_pages, v_pages=v_pages, table=table, lens=_i32(lens), q_start=_i32(_cdf(new)), q=q, max_q=max(new), max_k=max(lens),
                 scale=case["D"] ** -0.5)
    else:
        M, N, K, group = case["M"], case["N"], case["K"], case["group"]
        T, C = _up(N, 16), _up(K, 128)
        # 4-bit values around zero as rounded weights have them, two of a word's nibbles 16 bits apart
        q = torch.randn((N, K), device=DEV, generator=g).mul_(2.7).round_().clamp_(-8, 7).to(torch.int8)
        full = torch.zeros((T * 16, C * 128), dtype=torch.int8, device=DEV)
        full[:N, :K] = q
        e = (full.to(torch.int32) + 8).view(T, 16, C, 4, 4, 8).permute(0, 2, 4, 1, 3, 5)          # tile, chunk, k/8%4, row, k/32%4, k%8
        place = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=DEV, dtype=torch.int32)
        packed = torch.bitwise_left_shift(e, place).sum(-1).to(torch.int32).contiguous()
        scales = torch.zeros((T * 16, C * 128 // group), device=DEV)
        scales[:N, :_up(K, group)] = (0.5 + torch.rand((N, _up(K, group)), device=DEV, generator=g)) * (0.4 * K ** -0.5)
        scales = scales.to(torch.bfloat16).view(T, 16, -1).permute(0, 2, 1).contiguous()
        x = torch.randn((M, K), device=DEV, generator=g).to(TYPES[case["dtype"]])
        s.update(packed=packed, scales=scales, x=x, bias=torch.randn(N, device=DEV, generator=g) * 0.1, dt=TYPES[case["out"]],
                 residual=torch.randn((M, N), device=DEV, generator=g) if case["res"] else None)
    return s


# -------------------------------------------------------------- plain forms ----
def _plain_plan(s):
    lens, new, table, ring, page = s["lens"].long(), s["new"].long(), s["table"], s["ring"], s["page"]
    B, P = table.shape
    n, head, count, cap = ring.numel(), s["pool"][0].long(), s["pool"][1].long(), s["max_tokens"]
    have = (lens + page - 1) // page
    more = new.clamp_min(0)
    after = torch.where(new < 0, torch.zeros_like(lens), lens + more)
    need = torch.where(new < 0, torch.zeros_like(lens), (after + page - 1) // page - have)
    give = torch.where(new < 0, have, torch.zeros_like(have))
    first, back = need.cumsum(0) - need, give.cumsum(0) - give
    start = torch.cat([torch.zeros_like(more[:1]), more.cumsum(0)])
    status = (need.sum() > count) * 1 + (after > P * page).any() * 2 + (start[-1] > cap) * 4
    ok = status == 0
    j = torch.arange(P, device=DEV)[None]
    fresh = ok & (j >= have[:, None]) & (j < (have + need)[:, None])
    took = torch.where(fresh, ring[((head + first[:, None] + j - have[:, None]) % n)], table)
    gone = ok & (j < give[:, None])
    place = torch.where(gone, (head + count + back[:, None] + j) % n, torch.full_like(j, n))
    kept = torch.cat([ring, ring[:1]]).index_put((place.reshape(-1),), table.reshape(-1))[:n]
    start = torch.where(ok, start, torch.zeros_like(start))
    t = torch.arange(cap, device=DEV)
    real = t < start[-1]
    b = (torch.searchsorted(start, t, right=True) - 1).clamp(0, B - 1)
    pos = torch.where(real, lens[b] + t - start[b], torch.zeros_like(t))
    slot = torch.where(real, took[b, (pos // page).clamp_max(P - 1)].long() * page + pos % page, torch.full_like(t, -1))
    pool = torch.where(ok, torch.stack([(head + need.sum()) % n, count - need.sum() + give.sum()]), s["pool"].long())
    i = torch.int32
    return dict(table=took, ring=kept, lens=torch.where(ok, after, lens).to(i), pool=pool.to(i), q_start=start.to(i),
                slots=slot.to(i), positions=pos.to(i), status=status.to(i).reshape(1))


def _plain_write(s):
    slots, page = s["slots"].long(), s["page"]
    s["k_pages"][slots // page, :, slots % page] = s["k"]
    s["v_pages"][slots // page, :, slots % page] = s["v"]
    return s["k_pages"], s["v_pages"]


def _plain_attn(s):
    q, lens, start, page = s["q"], s["lens"].long(), s["q_start"].long(), s["page"]
    N, Hq, D = q.shape
    B, Hk, mq, mk = lens.numel(), s["Hk"], s["max_q"], s["max_k"]
    t = torch.arange(N, device=DEV)
    b = torch.searchsorted(start, t, right=True) - 1
    i = t - start[b]
    rows = torch.zeros((B, mq, Hq, D), dtype=torch.float32, device=DEV)
    rows[b, i] = q.float()
    rows = rows.view(B, mq, Hk, Hq // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    pages = s["table"][:, :_up(mk, page)].long()
    k, v = (p[pages].transpose(1, 2).reshape(B, Hk, -1, D)[:, :, :mk].float() for p in (s["k_pages"], s["v_pages"]))
    x = torch.matmul(rows, k.transpose(2, 3)) * s["scale"]
    key = torch.arange(mk, device=DEV)
    last = lens[:, None] - (start[1:] - start[:-1])[:, None] + torch.arange(mq, device=DEV)[None] if s["causal"] else (lens - 1)[:, None].expand(B, mq)
    seen = (key[None, None] <= last[:, :, None]) & (key[None, None] < lens[:, None, None])
    x = x.view(B, Hk, Hq // Hk, mq, mk).masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hk, -1, mk), v).view(B, Hq, mq, D).transpose(1, 2)
    return o[b, i].to(q.dtype)


def _unpacked(s, ft):
    """[N, K] weights of the packed words and their scales."""
    T, C = s["packed"].shape[:2]
    place = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], device=DEV, dtype=torch.int32)
    q = (torch.bitwise_right_shift(s["packed"][..., None], place) & 15) - 8
    q = q.view(T, C, 4, 16, 4, 8).permute(0, 3, 1, 4, 2, 5).reshape(T * 16, C * 128).to(ft)
    w = q.view(T * 16, -1, s["group"]) * s["scales"].to(ft).permute(0, 2, 1).reshape(T * 16, -1, 1)
    return w.view(T * 16, -1)[:s["N"], :s["K"]]


def _plain_w4(s):
    y = torch.matmul(s["x"].float(), _unpacked(s, torch.float32).t()) + s["bias"]
    if s["act"]:
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if s["res"]:
        y = y + s["residual"]
    return y.to(s["dt"])


# --------------------------------------------------- the framework's entries ----
def _own(s):
    from mocov2_whisper_flamingo_amd import ops
    if s["op"] == "plan":
        p = ops.paged_plan(s["lens"], s["new"], s["table"], s["ring"], s["pool"], s["page"], s["max_tokens"],
                           lens_out=s["lens_out"], pool_out=s["pool_out"])
        return dict(table=s["table"], ring=s["ring"], lens=s["lens_out"], pool=s["pool_out"], q_start=p.q_start, slots=p.slots,
                    positions=p.positions, status=p.status)
    if s["op"] == "write":
        ops.paged_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["slots"])
        return s["k_pages"], s["v_pages"]
    if s["op"] == "attn":
        return ops.paged_attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["q_start"], max_q=s["max_q"], max_k=s["max_k"],
                              scale=s["scale"], causal=s["causal"])
    w = ops.W4Weight(s["packed"], s["scales"], s["N"], s["K"], s["group"])
    return ops.w4_matmul(s["x"], w, bias=s["bias"], act=ops.ACT_GELU if s["act"] else ops.ACT_NONE, residual=s["residual"], out_dtype=s["dt"])


def run(state):
    if own:
        return _own(state)
    return {"plan": _plain_plan, "write": _plain_write, "attn": _plain_attn, "w4": _plain_w4}[state["op"]](state)


# -------------------------------------------------------------------- work ----
def work(case):
    op = case["op"]
    rng = random.Random(0)
    if op == "plan":
        lens, new = _news(case, rng)
        page, tokens = case["page"], sum(max(0, m) for m in new)
        moved = sum(_up(n + m, page) - _up(n, page) if m >= 0 else _up(n, page) for n, m in zip(lens, new))
        return {"bytes": 16 * case["B"] + 8 * moved + 12 * tokens, "flops": 0}
    if op == "write":
        n = sum(_spread(case["B"], case["lo"], case["hi"]))
        return {"bytes": n * (4 * case["H"] * case["D"] * (4 if case["dtype"] == "f32" else 2) + 4), "flops": 0}
    if op == "attn":
        lens, new = _lens(case, rng)
        size = 4 if case["dtype"] == "f32" else 2
        seen = sum(q * n - (q * (q - 1) // 2 if case["causal"] else 0) for n, q in zip(lens, new))
        return {"bytes": size * case["D"] * (2 * case["Hq"] * sum(new) + 2 * case["Hk"] * sum(lens)) + 4 * sum(_up(n, case["page"]) for n in lens),
                "flops": 4 * case["D"] * case["Hq"] * seen}
    M, N, K = case["M"], case["N"], case["K"]
    return {"bytes": N * K // 2 + 2 * N * _up(K, case["group"]) + 4 * N + M * K * (4 if case["dtype"] == "f32" else 2)
            + M * N * ((4 if case["out"] == "f32" else 2) + (4 if case["res"] else 0)), "flops": 2 * M * N * K}


# ------------------------------------------------------------------- exact ----
def exact(case, seed):
    if case["op"] in ("plan", "write"):       # whole numbers, and values that are only moved
        return None
    s = prepare(case, seed)
    if case["op"] == "attn":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        lens, start, G = s["lens"].tolist(), s["q_start"].tolist(), case["Hq"] // case["Hk"]
        for b, n in enumerate(lens):
            ids = s["table"][b, :_up(n, case["page"])].long()
            keys, values = (p[ids].double().permute(0, 2, 1, 3).reshape(-1, case["Hk"], case["D"])[:n] for p in (s["k_pages"], s["v_pages"]))
            rows = s["q"][start[b]:start[b + 1]].double()
            for h in range(case["Hq"]):
                x = rows[:, h] @ keys[:, h // G].t().contiguous() * s["scale"]
                if case["causal"]:
                    at = n - rows.shape[0] + torch.arange(rows.shape[0], device=DEV)
                    x = x.masked_fill(torch.arange(n, device=DEV)[None] > at[:, None], -math.inf)
                out[start[b]:start[b + 1], h] = torch.softmax(x, -1) @ values[:, h // G].contiguous()
        return out
    N, K, group = case["N"], case["K"], case["group"]
    y = torch.zeros((case["M"], N), dtype=torch.float64, device=DEV)
    x = s["x"].double()
    for k0 in range(0, K, group):              # one group of columns after another, each with its rows' scales
        k = torch.arange(k0, min(K, k0 + group), device=DEV)
        words = s["packed"][:, (k // 128)[None], (k // 8 % 4)[None], torch.arange(16, device=DEV)[:, None], (k // 32 % 4)[None]]
        nib = torch.bitwise_right_shift(words, (k % 8 // 2 * 4 + k % 2 * 16).to(torch.int32)) & 15
        part = x[:, k] @ (nib.reshape(-1, k.numel())[:N].double() - 8).t().contiguous()
        y += part * s["scales"][:, k0 // group].reshape(-1)[:N].double()
    y += s["bias"].double()
    if case["act"]:
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if case["res"]:
        y += s["residual"].double()
    return y
