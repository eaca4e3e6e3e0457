"""The serving operators (paged cache plan, page writes, attention over pages, 4-bit products) against their 64-bit
restatements in tests/serving_ref.py."""
import math
import random

import pytest
import torch

from mocov2_whisper_flamingo_amd import _lib, ops
from tests.serving_ref import Cache, HALF, U32, attn_ref, plan_ref, up

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------ plan ----
def run_plan(dev, lens, new, table, ring, pool, page, max_tokens, in_place):
    t, r, l, p = i32(table, dev), i32(ring, dev), i32(lens, dev), i32(pool, dev)
    kw = {} if in_place else dict(lens_out=torch.full_like(l, 77), pool_out=torch.full_like(p, 77))
    plan = ops.paged_plan(l, i32(new, dev), t, r, p, page, max_tokens, **kw)
    if not in_place:
        assert l.tolist() == lens and p.tolist() == pool
    lo, po = kw.get("lens_out", l), kw.get("pool_out", p)
    return dict(table=t.tolist(), ring=r.tolist(), lens=lo.tolist(), pool=po.tolist(), q_start=plan.q_start.tolist(),
                slots=plan.slots.tolist(), positions=plan.positions.tolist(), status=plan.status.item())


@pytest.mark.parametrize("B,page,width,n,max_tokens,longest,steps", [
    (1, 16, 1, 1, 4, 2, 6), (6, 16, 5, 20, 64, 40, 40), (7, 256, 3, 9, 600, 300, 20), (130, 32, 4, 300, 3000, 60, 12),
    (1024, 64, 2, 1500, 8192, 20, 4), (1024, 64, 2, 1500, 8193, 20, 4), (1025, 16, 3, 2000, 4000, 9, 4), (3000, 16, 2, 4000, 20000, 15, 3),
    (3, 64, 400, 700, 30000, 12000, 3)])
def test_plan_over_many_steps(dev, B, page, width, n, max_tokens, longest, steps):
    """Random steps of a server, one after another: tokens, prompts, idle places, ends, shortages; every output is equal."""
    rng = random.Random(B * 1000 + page)
    lens, table, pool = [0] * B, [[-1] * width for _ in range(B)], [rng.randrange(n), n]
    ring = list(range(n))
    rng.shuffle(ring)
    seen = set()
    for step in range(steps):
        new = [rng.choice([-1, 0, 1, 1, 1, rng.randint(1, longest)]) for _ in range(B)]
        want = plan_ref(lens, new, table, ring, pool, page, max_tokens)
        got = run_plan(dev, lens, new, table, ring, pool, page, max_tokens, in_place=step % 2 == 0)
        assert got == want, (step, want["status"])
        seen.add(want["status"])
        lens, table, ring, pool = want["lens"], want["table"], want["ring"], want["pool"]
    assert 0 in seen


@pytest.mark.parametrize("B", [5, 1500])
@pytest.mark.parametrize("what,status", [("pool", 1), ("row", 2), ("tokens", 4), ("negative", 8), ("head", 8), ("count", 8), ("end row", 2)])
def test_plan_refuses_a_step_as_a_whole(dev, B, what, status):
    lens, new, width, page = [20] * B, [1] * B, 4, 16
    table = [[2 * b, 2 * b + 1, -1, -1] for b in range(B)]
    n = 2 * B + 3
    ring, pool, cap = list(range(n)), [0, 3], B
    if what == "pool":
        new[:4] = [20] * 4
        cap = 2 * B + 100
    if what == "row":
        new[B - 1], cap = 45, B + 50
        pool = [0, 3]
    if what == "tokens":
        cap = B - 1
    if what == "negative":
        lens[2] = -1
    if what == "head":
        pool = [n, 3]
    if what == "count":
        pool = [0, n + 1]
    if what == "end row":
        lens[1], new[1] = 65, -1
    want = plan_ref(lens, new, table, ring, pool, page, cap)
    assert want["status"] == status and want["slots"] == [-1] * cap
    for in_place in (True, False):
        assert run_plan(dev, lens, new, table, ring, pool, page, cap, in_place) == want


@pytest.mark.parametrize("n", [100, (1 << 20) + 5])
def test_plan_sums_that_leave_32_bits(dev, n):
    """Wide table rows (never touched) and requests of millions of pages: the status of exact sums, and nothing is written."""
    B, page, width = 40, 16, 1 << 23
    table = torch.zeros(B, width, dtype=torch.int32, device=dev)
    for lens, new, status in (([0] * B, [1 << 27] * B, 1 | 4), ([1 << 27] * B, [-1] * B, 8), ([1 << 27] * B, [0] * B, 0), ([0] * B, [2 ** 31 - 1] * B, 2)):
        held, pool = i32(lens, dev), i32([0, 90], dev)
        plan = ops.paged_plan(held, i32(new, dev), table, torch.zeros(n, dtype=torch.int32, device=dev), pool, page, 64)
        assert plan.status.item() == status
        assert held.tolist() == lens and pool.tolist() == [0, 90] and plan.q_start.tolist() == [0] * (B + 1)


def test_plan_takes_rows_of_a_wider_table(dev):
    wide = torch.full((4, 9), -5, dtype=torch.int32, device=dev)
    lens, ring, pool = i32([0, 3, 16, 0], dev), torch.arange(8, dtype=torch.int32, device=dev), i32([0, 6], dev)
    wide[1, 2], wide[2, 2] = 6, 7
    ops.paged_plan(lens, i32([17, 1, 1, 0], dev), wide[:, 2:5], ring, pool, 16, 19)
    assert wide.tolist() == [[-5, -5, 0, 1, -5, -5, -5, -5, -5], [-5, -5, 6, -5, -5, -5, -5, -5, -5], [-5, -5, 7, 2, -5, -5, -5, -5, -5], [-5] * 9]
    assert lens.tolist() == [17, 4, 17, 0] and pool.tolist() == [3, 3]


# ----------------------------------------------------------------- write ----
@pytest.mark.parametrize("it,pt", [(BF, BF), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("N,H,D,page,layout", [(1, 1, 64, 16, "heads"), (37, 6, 64, 16, "heads"), (200, 5, 128, 32, "keys"), (3, 20, 64, 256, "keys"),
                                               (1031, 3, 64, 64, "heads")])
def test_write(dev, it, pt, N, H, D, page, layout):
    g = torch.Generator().manual_seed(N)
    n_pages = up(N, page) + 4
    c = Cache([5], H, D, page, pt, g, filler=-3.0, layout=layout, spare=n_pages - 1)
    kp, vp = c.views(dev)
    slots = torch.randperm(n_pages * page, generator=g)[:N].to(torch.int32)
    slots[::5] = -1                                            # padding of a step
    if N > 3:
        slots[2] = n_pages * page                              # beyond the pool: left out
    qkv = torch.randn(N, 3, H, D, generator=g).to(it)
    src = qkv.to(dev)
    ops.paged_write(src[:, 1], src[:, 2], kp, vp, slots.to(dev))
    wk, wv = c.k_pages.clone(), c.v_pages.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < n_pages * page:
            wk[s // page, :, s % page] = qkv[t, 1].to(pt)
            wv[s // page, :, s % page] = qkv[t, 2].to(pt)
    assert torch.equal(kp.cpu(), wk) and torch.equal(vp.cpu(), wv)
    ops.paged_write(src[:0, 1], src[:0, 2], kp, vp, slots[:0].to(dev))


def test_write_takes_heads_of_any_stride(dev):
    kp, vp = (torch.zeros(2, 4, 16, 64, device=dev) for _ in range(2))
    x = torch.randn(3, 64, 8, 2, device=dev).permute(3, 0, 2, 1).contiguous().permute(1, 2, 3, 0)       # [3, 8, 64, 2]
    rows = torch.randn(3, 8, 68, device=dev)[:, ::2, :64]
    ops.paged_write(rows, rows, kp, vp, i32([31, 0, 5], dev))
    assert torch.equal(kp[1, :, 15], rows[0]) and torch.equal(vp[0, :, 0], rows[1]) and torch.equal(kp[0, :, 5], rows[2]) and x.shape[0] == 3


def test_strides_of_a_dimension_of_one_do_not_count(dev):
    """Views of one row, one head or one page whose stride there is any number: PyTorch leaves it free."""
    def odd(x):
        return x.as_strided(x.shape, [13 if n == 1 else s for n, s in zip(x.shape, x.stride())])

    g = torch.Generator().manual_seed(1)
    for shape in ((1, 3), (4, 1), (1, 1)):
        k = torch.randn(*shape, 64, generator=g).to(BF).to(dev)
        slots = i32(list(range(shape[0])), dev)
        a, b = torch.zeros(2, 1, shape[1], 16, 64, dtype=BF, device=dev), torch.zeros(2, 1, shape[1], 16, 64, dtype=BF, device=dev)
        ops.paged_write(k, k, a[0], a[1], slots)
        ops.paged_write(odd(k), odd(k), odd(b[0]), odd(b[1]), slots)
        assert torch.equal(a, b) and a.any()
        tail = (i32([[0]], dev), i32([shape[0]], dev), i32([0, shape[0]], dev))
        want = ops.paged_attn(k, a[0], a[1], *tail, scale=0.125)
        assert torch.equal(ops.paged_attn(odd(k), odd(a[0]), odd(a[1]), *tail, scale=0.125, out=odd(torch.zeros_like(k))), want)


# ------------------------------------------------------------- attention ----
def attend_and_check(dev, lens, news, Hq, Hk, D, page, dtype, causal, *, seed=0, layout="heads", scale=None, edit=None, **kw):
    g = torch.Generator().manual_seed(seed)
    scale = D ** -0.5 if scale is None else scale
    c = Cache(lens, Hk, D, page, dtype, g, layout=layout)
    if edit:
        edit(c)
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    N = start[-1] + 3                                          # rows behind the last request stay as they are
    wide = torch.randn(N, Hq, 2 * D, generator=g).to(dtype)
    q = wide[:, :, D:]
    kp, vp = c.views(dev)
    out = torch.full((N, Hq, D), 5.0, dtype=dtype, device=dev)
    got = ops.paged_attn(wide.to(dev)[:, :, D:], kp, vp, c.table.to(dev), i32(lens, dev), i32(start, dev), scale=scale, causal=causal, out=out,
                         **kw)
    assert got.data_ptr() == out.data_ptr()
    got = got.cpu()
    assert torch.all(got[start[-1]:] == 5.0)
    worst = 0.0
    for b, n in enumerate(lens):
        rows = slice(start[b], start[b + 1])
        if news[b] == 0:
            continue
        o, bound = attn_ref(q[rows], c.k[b], c.v[b], scale, causal, dtype)
        err = (got[rows].double() - o).abs()
        assert torch.isfinite(got[rows].float()).all(), b
        worst = max(worst, float((err / bound).max()))
    assert worst <= 1.0, worst
    return got[:start[-1]]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_attn_single_tokens(dev, dtype, D, page, causal):
    """One token per request: contexts of one key, around the ends of a tile and of a page, and long ones."""
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 128, 255, 256, 257, 700]
    attend_and_check(dev, lens, [1] * len(lens), 3, 3, D, page, dtype, causal, max_q=1)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("Hq,Hk", [(1, 1), (4, 2), (7, 1), (20, 20), (24, 3), (40, 1)])
def test_attn_shared_heads(dev, dtype, Hq, Hk):
    attend_and_check(dev, [40, 1, 333, 90], [1, 1, 1, 1], Hq, Hk, 64, 32, dtype, True, max_q=1, layout="keys")
    attend_and_check(dev, [40, 3, 333, 90], [2, 3, 5, 9], Hq, Hk, 64, 32, dtype, True, max_q=9)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("causal", [True, False])
def test_attn_chunks(dev, dtype, D, page, causal):
    """Chunks of many lengths beside single tokens and requests that wait, on nothing and on long contexts."""
    lens = [70, 65, 1, 300, 129, 0, 515, 64, 40, 200]
    news = [70, 64, 1, 129, 1, 0, 260, 0, 17, 66]
    attend_and_check(dev, lens, news, 4, 2, D, page, dtype, causal)
    attend_and_check(dev, lens, news, 2, 2, D, page, dtype, causal, max_q=260, max_k=515)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B", [64, 65, 150])
@pytest.mark.parametrize("causal", [True, False])
def test_attn_chunks_of_many_requests(dev, dtype, D, B, causal):
    """Around 64 requests the tiles are dealt out in another way: prompts on both sides of a tile's 128 rows (64 tokens of two
    heads), single tokens and requests that wait between them."""
    rng = random.Random(B + D)
    news = [rng.choice([0, 0, 1, 1, 2, 31, 33, 63, 64, 65, 130]) for _ in range(B)]
    news[0], news[-1] = 65, 129
    lens = [n + rng.choice([0, 0, 5, 64, 190]) for n in news]
    attend_and_check(dev, lens, news, 2, 1, D, 32, dtype, causal, seed=B)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,news", [([40, 300, 7], [1, 1, 1]), ([300, 200, 64, 3], [130, 70, 1, 3]), ([9000], [1])])
def test_attn_into_its_own_queries(dev, dtype, lens, news):
    """out may be q: a row's queries are read before its result is written, in each kernel, whole and split."""
    g = torch.Generator().manual_seed(8)
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    c = Cache(lens, 2, 64, 64, dtype, g)
    kp, vp = c.views(dev)
    q = torch.randn(start[-1], 4, 64, generator=g).to(dtype).to(dev)
    tail = (kp, vp, c.table.to(dev), i32(lens, dev), i32(start, dev))
    want = ops.paged_attn(q, *tail, scale=0.125)
    assert torch.equal(ops.paged_attn(q, *tail, scale=0.125, out=q), want) and torch.equal(q, want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,news", [([300, 200, 64, 3], [130, 70, 1, 3]), ([4000] * 6, [200] * 6), ([2000] * 80, [1] * 80), ([9000, 30], [2, 1])])
def test_attn_repeats_bit_for_bit(dev, dtype, D, lens, news):
    """Nothing in a call depends on timing: no order of atomics, no score read before its matrix instruction is done."""
    g = torch.Generator(device=dev).manual_seed(10)
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    W = up(max(lens), 64)
    kv = torch.randn(len(lens) * W, 2, 2, 64, D, generator=g, device=dev).to(dtype)
    table = torch.arange(len(lens) * W, dtype=torch.int32, device=dev).view(-1, W)
    q = 4 * torch.randn(start[-1], 4, D, generator=g, device=dev).to(dtype)
    call = lambda: ops.paged_attn(q, kv[:, 0], kv[:, 1], table, i32(lens, dev), i32(start, dev), scale=D ** -0.5)
    want = call()
    assert torch.isfinite(want.float()).all()
    for _ in range(20):
        assert torch.equal(call(), want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("news", [[3, 2], [70, 90], [200, 40]])
@pytest.mark.parametrize("G", [1, 3])
def test_attn_values_that_are_not_finite_inside_a_chunk(dev, dtype, D, news, G):
    """An infinite value in the middle of the new tokens: rows before it are as without it, rows from it on are infinite in its column."""
    g = torch.Generator().manual_seed(9)
    lens = [n + 37 for n in news]
    c = Cache(lens, 2, D, 16, dtype, g)
    kp, vp = c.views(dev)
    q = torch.randn(sum(news), 2 * G, D, generator=g).to(dtype)
    hit = [37 + n // 2 for n in news]
    for b in range(2):
        vp[c.table[b, hit[b] // 16].item(), 1, hit[b] % 16, 5] = float("inf")
    got = ops.paged_attn(q.to(dev), kp, vp, c.table.to(dev), i32(lens, dev), i32([0, news[0], sum(news)], dev), scale=D ** -0.5).cpu()
    for b in range(2):
        rows = got[sum(news[:b]):sum(news[:b + 1])].double()
        o, bound = attn_ref(q[sum(news[:b]):sum(news[:b + 1])], c.k[b], c.v[b], D ** -0.5, True, dtype)
        seen = torch.zeros_like(rows, dtype=torch.bool)
        seen[hit[b] - 37:, G:, 5] = True
        assert torch.isinf(rows[seen]).all() and (rows[seen] > 0).all()
        assert ((rows - o).abs() <= bound)[~seen].all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attn_one_request(dev, dtype):
    attend_and_check(dev, [200], [200], 2, 1, 64, 16, dtype, True)
    attend_and_check(dev, [33], [33], 1, 1, 64, 16, dtype, True)
    attend_and_check(dev, [1], [1], 1, 1, 128, 16, dtype, True)


@pytest.mark.parametrize("dtype,D,B,L", [(BF, 64, 2, 9001), (BF, 128, 1, 20011), (F32, 64, 1, 6500)])
def test_attn_long_context_is_split(dev, dtype, D, B, L):
    attend_and_check(dev, [L - 7 * b for b in range(B)], [1] * B, 2, 1, D, 128, dtype, True, max_q=1)
    attend_and_check(dev, [L - 7 * b for b in range(B)], [3] * B, 2, 1, D, 128, dtype, False, max_q=3)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,news,Hq", [([300, 40, 3], [1, 1, 1], 2), ([300, 120, 90], [80, 30, 7], 2), ([2000, 1999], [2, 1], 4)])
def test_attn_hints_change_no_result(dev, dtype, lens, news, Hq):
    """max_q and max_k only choose the grid: too small or too large ones still give every row."""
    for mq in (1, 3, 100, None):
        for mk in (1, 200, 5000, None):
            attend_and_check(dev, lens, news, Hq, 2, 64, 16, dtype, True, max_q=mq, max_k=mk)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [5, 2, 70, 3]])
def test_attn_rows_that_see_nothing_are_zero(dev, dtype, news):
    """Empty requests (no keys), and more new tokens than keys: the rows before the first key see nothing."""
    g = torch.Generator().manual_seed(1)
    lens = [0, 40, 30, 2]
    c = Cache(lens, 2, 64, 16, dtype, g)
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    q = torch.randn(start[-1], 2, 64, generator=g).to(dtype)
    kp, vp = c.views(dev)
    for causal in (True, False):
        got = ops.paged_attn(q.to(dev), kp, vp, c.table.to(dev), i32(lens, dev), i32(start, dev), scale=0.125, causal=causal).cpu()
        for b, n in enumerate(lens):
            rows = got[start[b]:start[b + 1]]
            if n == 0:
                assert torch.equal(rows, torch.zeros_like(rows))
                continue
            o, bound = attn_ref(q[start[b]:start[b + 1]], c.k[b], c.v[b], 0.125, causal, dtype)
            assert ((rows.double() - o).abs() <= bound).all()
            if causal and news[b] > n:
                assert torch.equal(rows[:news[b] - n], torch.zeros_like(rows[:news[b] - n]))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("chunk", [4, 100])
def test_attn_unseen_keys_have_no_influence(dev, dtype, bad, chunk):
    """The last new token's key and value are not finite: only its own row may notice."""
    g = torch.Generator().manual_seed(2)
    L = 150
    c = Cache([L], 2, 64, 32, dtype, g)
    start = [0, chunk]
    q = torch.randn(chunk, 2, 64, generator=g).to(dtype)
    for where in ("k", "v"):
        kp, vp = c.views(dev)
        pages = kp if where == "k" else vp
        pages[c.table[0, (L - 1) // 32].item(), :, (L - 1) % 32] = bad
        got = ops.paged_attn(q.to(dev), kp, vp, c.table.to(dev), i32([L], dev), i32(start, dev), scale=0.125).cpu()
        o, bound = attn_ref(q, c.k[0], c.v[0], 0.125, True, dtype)
        assert ((got[:-1].double() - o[:-1]).abs() <= bound[:-1]).all()
        if where == "v":
            assert not torch.isfinite(got[-1]).any()


def test_attn_pages_that_do_not_exist_are_not_read(dev):
    """A table entry outside the pool hides its keys: the same result as without them."""
    g = torch.Generator().manual_seed(3)
    c = Cache([96, 96], 1, 64, 16, BF, g)
    q = torch.randn(2, 2, 64, generator=g).to(BF)
    kp, vp = c.views(dev)
    table = c.table.clone()
    table[0, 2], table[1, 0], table[1, 5] = -1, kp.shape[0], 2 ** 31 - 1
    got = ops.paged_attn(q.to(dev), kp, vp, table.to(dev), i32([96, 96], dev), i32([0, 1, 2], dev), scale=0.125).cpu()
    keep = [torch.cat([torch.arange(32), torch.arange(48, 96)]), torch.arange(16, 80)]
    for b in range(2):
        o, bound = attn_ref(q[b:b + 1], c.k[b][keep[b]], c.v[b][keep[b]], 0.125, True, BF)
        assert ((got[b:b + 1].double() - o).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_attn_scales_and_large_scores(dev, dtype):
    """A negative and a zero scale, and scores that leave one key (softmax far from uniform)."""
    for scale in (-0.125, 0.0, 4.0):
        attend_and_check(dev, [90, 200], [3, 70], 2, 2, 64, 16, dtype, True, scale=scale)


def test_attn_lengths_beyond_the_table_are_cut(dev):
    g = torch.Generator().manual_seed(4)
    c = Cache([64], 1, 64, 16, F32, g)
    q = torch.randn(1, 1, 64, generator=g)
    kp, vp = c.views(dev)
    got = ops.paged_attn(q.to(dev), kp, vp, c.table.to(dev), i32([5000], dev), i32([0, 1], dev), scale=0.125).cpu()
    o, bound = attn_ref(q, c.k[0], c.v[0], 0.125, True, F32)
    assert ((got.double() - o).abs() <= bound).all()


def test_attn_offsets_past_32_bits(dev):
    """Pages beyond 2^32 bytes and 2^31 values from the pool's start."""
    H, page, D = 4, 256, 128
    n = (1 << 32) // (2 * H * page * D) + 20                   # keys and values interleaved: the last page starts beyond 2^32 values
    kv = torch.empty((n, 2, H, page, D), dtype=BF, device=dev)
    g = torch.Generator().manual_seed(6)
    k, v, q = (torch.randn(s, H, D, generator=g).to(BF) for s in (500, 500, 2))
    ids = [n - 1, n - 7]
    kp, vp = kv[:, 0], kv[:, 1]
    slots = i32([ids[j // page] * page + j % page for j in range(500)], dev)
    ops.paged_write(k.to(dev), v.to(dev), kp, vp, slots)
    got = ops.paged_attn(q.to(dev), kp, vp, i32([ids], dev), i32([500], dev), i32([0, 2], dev), scale=0.1).cpu()
    o, bound = attn_ref(q, k, v, 0.1, True, BF)
    assert ((got.double() - o).abs() <= bound).all()
    del kv, kp, vp
    torch.cuda.empty_cache()


# ------------------------------------------------------------------- w4 ----
def w4_check(dev, M, N, K, group, xt, ot, *, act=ops.ACT_NONE, bias=True, residual=False, pad=0, seed=0):
    g = torch.Generator().manual_seed(seed + N + K)
    q = torch.randint(-8, 8, (N, K), generator=g)
    s = (torch.rand(N, up(K, group), generator=g) + 0.1).to(BF)
    x = torch.randn(M, K + pad, generator=g).to(xt)[:, :K]
    b = torch.randn(N, generator=g) if bias else None
    r = torch.randn(M, N + pad, generator=g).to(ot)[:, :N] if residual else None
    w = ops.w4_pack(q.to(dev), s.to(dev), group)
    xd = torch.zeros(M, K + pad, dtype=xt, device=dev)[:, :K]
    xd.copy_(x)
    out = None
    if pad:
        out = torch.full((M, N + pad), 9.0, dtype=ot, device=dev)[:, :N]
    got = ops.w4_matmul(xd, w, bias=None if b is None else b.to(dev), act=act, residual=None if r is None else r.to(dev), out=out, out_dtype=ot)
    if pad:
        assert torch.all(got.as_strided((M, pad), (N + pad, 1), N) == 9.0)
    sk = s.double().repeat_interleave(group, 1)[:, :K]
    wd = q.double() * sk
    y = x.double() @ wd.t()
    # K accumulations of fp32 (and as many of the -24 x that start them), each within half a step of what is summed up;
    # the sums of magnitudes: (16 + 15 + 24) |x| scale
    worst = 2 * (K + 8) * U32 * 55 * (x.double().abs() @ sk.t())
    if b is not None:
        y = y + b.double()
        worst = worst + U32 * y.abs()
    if act == ops.ACT_GELU:
        y, worst = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5))), 1.2 * worst + 8 * U32 * y.abs()      # |gelu'| < 1.13
    elif act == ops.ACT_RELU:
        y = y.clamp_min(0)
    if r is not None:
        y = y + r.double()
        worst = worst + U32 * y.abs()
    got = got.cpu().double()
    err = (got - y).abs()
    assert (err <= worst + HALF[ot] * (y.abs() + worst) + 1e-30).all()
    # and as a whole: the roundings are independent, about sqrt(K / 32) of them on sums of up to 24 sqrt(group) |x| scale,
    # against |y| = 4.6 sqrt(K) |x| scale: below 40 half steps; the result's own rounding is uniform, HALF / sqrt(3)
    # - of many values.  Fewer than 16 different ones are no average: n copies of one value y have n times one error of up to
    # HALF |y|, so that |err| / |y| <= HALF (20 rows of one column whose weight is 0 are 20 times the bias: 1.2456 is 2.73e-3 of
    # itself away from the next bf16, HALF 3.91e-3).
    one = 0.6 if y.unique().numel() >= 16 else 1.0
    assert err.norm() <= (40 * U32 + HALF[ot] * one + 1e-7) * y.norm()


@pytest.mark.parametrize("xt,ot", [(BF, BF), (BF, F32), (F32, F32), (F32, BF)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 16, 128), (1, 1, 1), (3, 50, 384), (16, 33, 200), (17, 64, 1000), (40, 100, 96), (64, 31, 257), (65, 48, 512),
                                   (130, 20, 160)])
def test_w4_sizes(dev, xt, ot, group, M, N, K):
    w4_check(dev, M, N, K, group, xt, ot)


@pytest.mark.parametrize("xt", [BF, F32])
@pytest.mark.parametrize("M,N,K", [(1, 17000, 640), (20, 16400, 256), (50, 16390, 384)])
def test_w4_wide(dev, xt, M, N, K):
    w4_check(dev, M, N, K, 64, xt, F32)


@pytest.mark.parametrize("xt,ot", [(BF, BF), (F32, F32)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K,pad", [(3, 16400, 200, 0), (5, 16385, 1000, 0), (16, 16400, 333, 5), (4, 16384, 4480, 0), (33, 16390, 1160, 0), (70, 16384, 130, 0)])
def test_w4_wide_through_lds(dev, xt, ot, group, M, N, K, pad):
    """Wide layers: x in one block and in several, rows that are not aligned, more rows than a workgroup takes."""
    w4_check(dev, M, N, K, group, xt, ot, pad=pad, residual=bool(pad), act=ops.ACT_GELU if pad else ops.ACT_NONE)


@pytest.mark.parametrize("xt,ot", [(BF, BF), (F32, F32)])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K,pad", [(17, 1280, 4500, 0), (40, 640, 9000, 0), (33, 300, 2333, 5), (64, 5120, 300, 0), (100, 4000, 1290, 0), (200, 2600, 130, 3),
                                       (18, 40, 16500, 0), (40, 16400, 2200, 0), (20, 1, 1, 0)])
def test_w4_layers_through_lds(dev, xt, ot, group, M, N, K, pad):
    """More than 16 rows: one way to eight that share the columns, one block of x and several, more columns than a block, fewer
    than a chunk, last tiles and rows that are not whole."""
    w4_check(dev, M, N, K, group, xt, ot, pad=pad, residual=bool(pad), act=ops.ACT_GELU if pad else ops.ACT_NONE)


@pytest.mark.parametrize("act", [ops.ACT_NONE, ops.ACT_GELU, ops.ACT_RELU])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("xt,ot", [(BF, BF), (BF, F32), (F32, F32)])
def test_w4_epilogue(dev, act, residual, xt, ot):
    w4_check(dev, 5, 70, 256, 32, xt, ot, act=act, residual=residual)
    w4_check(dev, 5, 70, 250, 32, xt, ot, act=act, residual=residual, bias=False, pad=3)        # rows of odd strides


def test_w4_adds_onto_its_own_output(dev):
    g = torch.Generator().manual_seed(8)
    w = ops.w4_quantize(torch.randn(96, 128, generator=g).to(dev), 32)
    x, y = torch.randn(7, 128, generator=g).to(dev), torch.randn(7, 96, generator=g).to(dev)
    want = ops.w4_matmul(x, w, residual=y)
    assert torch.equal(ops.w4_matmul(x, w, residual=y, out=y), want) and torch.equal(y, want)


@pytest.mark.parametrize("xt", [BF, F32])
def test_w4_no_rows_and_large_values(dev, xt):
    """No rows, also into a given output; and the largest values allowed, whose sums on the way stay finite."""
    w = ops.w4_pack(torch.full((20, 256), -8, dtype=torch.int32), torch.full((20, 2), 2.0 ** -10), 128)
    w = w._replace(packed=w.packed.to(dev), scales=w.scales.to(dev))
    x = torch.full((1, 256), 2.0 ** 112, dtype=xt, device=dev)                       # 5.2e33
    none = ops.w4_matmul(x[:0], w, out=torch.empty(0, 20, dtype=xt, device=dev), residual=torch.empty(0, 20, dtype=xt, device=dev))
    assert none.shape == (0, 20) and ops.w4_matmul(x[:0], w).shape == (0, 20)
    assert torch.equal(ops.w4_matmul(x, w).cpu(), torch.full((1, 20), -(2.0 ** 113), dtype=xt))         # 256 * 2^112 * -8 * 2^-10


def test_w4_rows_do_not_mix(dev):
    """A row that is not finite is NaN throughout and leaves the others alone, and a row's result does not depend on how many
    rows stand beside it in its tile."""
    g = torch.Generator().manual_seed(9)
    w = ops.w4_quantize(torch.randn(80, 256, generator=g).to(dev), 64)
    x = torch.randn(9, 256, generator=g).to(dev)
    clean = ops.w4_matmul(x, w)
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[4, 17] = bad
        got = ops.w4_matmul(y, w)
        assert torch.isnan(got[4]).all()
        keep = [0, 1, 2, 3, 5, 6, 7, 8]
        assert torch.equal(got[keep], clean[keep])
    assert torch.equal(ops.w4_matmul(x[:1], w), clean[:1])
    assert ops.w4_matmul(x[:0], w).shape == (0, 80)


def test_w4_fp32_activations_keep_their_last_bit(dev):
    """Values with all 24 bits and of every magnitude, through one weight of 1: the result is the activation itself."""
    g = torch.Generator().manual_seed(10)
    x = torch.randn(16, 32, generator=g) * torch.exp2(torch.randint(-60, 60, (16, 32), generator=g).float())
    for k in range(32):
        q = torch.zeros(16, 32, dtype=torch.int32)
        q[:, k] = 1
        one = torch.zeros_like(x)
        one[:, k] = x[:, k]
        got = ops.w4_matmul(one.to(dev), ops.w4_pack(q.to(dev), torch.ones(16, 1, device=dev), 32)).cpu()
        # 17 x - 24 x + ... : two sums around 24 |x| of half a step each, three pieces each
        assert ((got - one[:, k:k + 1]).abs() <= 6 * 24 * U32 * one[:, k:k + 1].abs()).all()


# ------------------------------------------------------------ embed, graph ----
def test_embed_tokens_at(dev):
    g = torch.Generator().manual_seed(11)
    table, pos = torch.randn(50, 64, generator=g), torch.randn(20, 64, generator=g)
    ids, at = torch.randint(0, 50, (13,), generator=g), torch.randint(0, 20, (13,), generator=g).to(torch.int32)
    got = ops.embed_tokens_at(ids.to(dev), table.to(dev), pos.to(dev), at.to(dev)).cpu()
    assert torch.equal(got, table[ids] + pos[at.long()])
    for bad_ids, bad_at in ((50, 0), (-1, 0), (0, 20), (0, -1)):
        i2, a2 = ids.clone(), at.clone()
        i2[3], a2[3] = bad_ids, bad_at
        with pytest.raises(IndexError):
            ops.embed_tokens_at(i2.to(dev), table.to(dev), pos.to(dev), a2.to(dev))
        flag = torch.zeros(1, dtype=torch.int32, device=dev)
        ops.embed_tokens_at(i2.to(dev), table.to(dev), pos.to(dev), a2.to(dev), bad=flag)
        assert flag.item() == 1


def test_calls_on_two_streams_at_once(dev):
    """Split attention, a mixed batch, products and a plan on two streams, each with operands of its own: what one stream alone gives."""
    g = torch.Generator(device=dev).manual_seed(12)

    def work(k):
        lens, news = [(9000, 700, 40), (5000, 64, 333)][k], [(1, 130, 3), (2, 1, 70)][k]
        W = up(max(lens), 64)
        kv = torch.randn(3 * W, 2, 2, 64, 64, generator=g, device=dev).to(BF)
        table = torch.arange(3 * W, dtype=torch.int32, device=dev).view(3, W)
        q = torch.randn(sum(news), 4, 64, generator=g, device=dev).to(BF)
        w = ops.w4_quantize(torch.randn(1000, 2200, generator=g, device=dev))
        x = torch.randn(24, 2200, generator=g, device=dev)
        state = (i32(list(lens), dev), i32(list(news), dev), i32([0, news[0], news[0] + news[1], sum(news)], dev))
        ring, pool = torch.arange(3 * W, dtype=torch.int32, device=dev), i32([0, 3 * W], dev)

        def call():
            lo, po = torch.empty_like(state[0]), torch.empty_like(pool)
            plan = ops.paged_plan(torch.zeros_like(state[0]), state[1], table.clone(), ring.clone(), pool, 64, 300, lens_out=lo, pool_out=po)
            return (ops.paged_attn(q, kv[:, 0], kv[:, 1], table, state[0], state[2], scale=0.125),
                    ops.paged_attn(q[:1], kv[:, 0], kv[:, 1], table[:1], state[0][:1], i32([0, 1], dev), max_q=1, scale=0.125),
                    ops.w4_matmul(x, w), ops.w4_matmul(x[:3], w), plan.slots, plan.q_start, lo, po)
        return call

    calls = [work(0), work(1)]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                got.append(c())
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_serving_step_captured_and_replayed(dev):
    """Plan, write and attention of a step in a graph: every replay moves the cache on by a token, as eager calls do."""
    g = torch.Generator().manual_seed(12)
    B, H, D, page, W, n = 5, 3, 64, 16, 12, 70

    def fresh():
        return dict(lens=i32([0, 4, 15, 16, 33], dev), table=torch.tensor([[j + 10 * b for j in range(W)] for b in range(B)], dtype=torch.int32, device=dev),
                    ring=torch.arange(n, dtype=torch.int32, device=dev).flip(0).contiguous(), pool=i32([0, 20], dev),
                    kv=torch.randn(n, 2, H, page, D, generator=torch.Generator().manual_seed(1)).to(dev, BF))

    new = torch.ones(B, dtype=torch.int32, device=dev)
    qkv = torch.zeros(B, 3, H, D, dtype=BF, device=dev)

    def step(s):
        p = ops.paged_plan(s["lens"], new, s["table"], s["ring"], s["pool"], page, B)
        ops.paged_write(qkv[:, 1], qkv[:, 2], s["kv"][:, 0], s["kv"][:, 1], p.slots)
        return p, ops.paged_attn(qkv[:, 0], s["kv"][:, 0], s["kv"][:, 1], s["table"], s["lens"], p.q_start, max_q=1, scale=0.125)

    eager, graphed = fresh(), fresh()
    warm = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, out = step(graphed)
    graphed_start = fresh()
    for k in graphed:
        graphed[k].copy_(graphed_start[k])
    for i in range(20):
        qkv.copy_(torch.randn(B, 3, H, D, generator=g).to(dev, BF))
        graph.replay()
        p, want = step(eager)
        torch.cuda.synchronize()
        assert plan.status.item() == 0 and p.status.item() == 0
        assert torch.equal(out, want), i
        for k in eager:
            assert torch.equal(eager[k], graphed[k]), (i, k)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,news,kw", [
    ([1, 17, 40, 130, 333, 700], [1] * 6, dict(max_q=1)),                      # one token, short
    ([1500] * 4, [1] * 4, dict(max_q=1, causal=False)),                         # frames
    ([5001, 3000], [1, 1], dict(max_q=1)),                                      # split keys
    ([300, 90, 500], [5, 9, 30], dict()),                                       # a few tokens
    ([700, 520, 40], [130, 300, 2], dict()),                                    # chunks, and a request with few rows beside them
    ([4100], [70], dict())])                                                    # a chunk with split keys
def test_attn_bf16_is_the_exact_result_rounded_once(dev, D, lens, news, kw):
    """Against the 64-bit result rounded to bf16.  What the kernel holds before its own rounding is off by r: the probabilities by at
    most 2^-16 of themselves (two bf16 pieces, half a step of half a step), fp32 sums by less, and the errors are independent, so that r is
    about 2^-16 |o|.  An element then crosses a border between two bf16 values with probability r / step and is a step off: in the mean
    of squares r * step <= 2^-16 * 2^-7 |o|^2, a norm of 2^-11.5 = 0.09 HALF; twice that is allowed.  Probabilities of one bf16 piece would give
    0.5 HALF."""
    g = torch.Generator().manual_seed(D + len(lens))
    kw = dict(kw)
    causal = kw.pop("causal", True)
    Hq, Hk = 4, 2
    c = Cache(lens, Hk, D, 64, BF, g)
    start = [0]
    for n in news:
        start.append(start[-1] + n)
    q = torch.randn(start[-1], Hq, D, generator=g).to(BF)
    kp, vp = c.views(dev)
    got = ops.paged_attn(q.to(dev), kp, vp, c.table.to(dev), i32(lens, dev), i32(start, dev), scale=D ** -0.5, causal=causal, **kw).cpu().double()
    want = torch.cat([attn_ref(q[start[b]:start[b + 1]], c.k[b], c.v[b], D ** -0.5, causal, BF)[0] for b in range(len(lens))])
    assert (got - want.to(BF).double()).norm() <= 0.2 * HALF[BF] * want.norm()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 20, 200])
def test_attn_infinite_values_with_equal_weights(dev, dtype, D, n):
    """Queries of zeros weigh all keys alike, with a probability before normalisation of exactly 1: both infinities come through, together
    they are NaN, and the other columns are the mean."""
    g = torch.Generator().manual_seed(22)
    lens = [700, 400]
    c = Cache(lens, 1, D, 32, dtype, g)
    kp, vp = c.views(dev)
    q = torch.zeros(2 * n, 2, D, dtype=dtype)
    inf = float("inf")
    for key, d, v in ((3, 0, inf), (100, 1, -inf), (7, 2, inf), (199, 2, -inf), (64, D - 1, inf)):
        vp[c.table[0, key // 32].item(), 0, key % 32, d] = v
    got = ops.paged_attn(q.to(dev), kp, vp, c.table.to(dev), i32(lens, dev), i32([0, n, 2 * n], dev), scale=1.0).cpu().double()
    rows = got[:n]
    assert (rows[:, :, 0] == inf).all() and (rows[:, :, 1] == -inf).all() and rows[:, :, 2].isnan().all() and (rows[:, :, D - 1] == inf).all()
    for b, keep in ((0, list(range(3, D - 1))), (1, list(range(D)))):
        o, bound = attn_ref(q[b * n:(b + 1) * n], c.k[b], c.v[b], 1.0, True, dtype)
        assert ((got[b * n:(b + 1) * n] - o).abs() <= bound)[:, :, keep].all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("hit", [4599, 1000])
def test_attn_infinite_values_in_a_split_context(dev, dtype, D, hit):
    """A visible infinite value gives an infinity in its column, whether the keys are split or not, and whichever split it stands in."""
    g = torch.Generator().manual_seed(21)
    L = 4600
    c = Cache([L], 1, D, 64, dtype, g)
    kp, vp = c.views(dev)
    q = torch.randn(1, 2, D, generator=g).to(dtype)
    splits = _lib.load().avsr_paged_attn_workspace_bytes(ops._dt(q), 1, 1, 2, 1, D, 1, L) // (4 * 2 * (D + 2))
    assert splits > 1 and splits % 8                           # the join runs in groups of eight
    vp[c.table[0, hit // 64].item(), 0, hit % 64, 5] = float("inf")
    o, bound = attn_ref(q, c.k[0], c.v[0], D ** -0.5, True, dtype)
    for mk in (L, 512):
        got = ops.paged_attn(q.to(dev), kp, vp, c.table.to(dev), i32([L], dev), i32([0, 1], dev), max_q=1, max_k=mk, scale=D ** -0.5).cpu().double()
        assert (got[:, :, 5] == float("inf")).all(), mk
        keep = [d for d in range(D) if d != 5]
        assert ((got - o).abs() <= bound)[:, :, keep].all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_attn_c_entry_takes_the_workspace_it_asks_for(dev, dtype, D):
    """Bounds for any step of a server (max_q far above the rows of this one): the entry works in what the query said, and gives what it
    gives with tight bounds."""
    g = torch.Generator().manual_seed(D)
    lens, Hq, Hk, lib = [5000, 8000, 17, 900], 32, 8, _lib.load()
    c = Cache(lens, Hk, D, 64, dtype, g)
    kp, vp = c.views(dev)
    q, table = torch.randn(4, Hq, D, generator=g).to(dtype).to(dev), c.table.to(dev)
    held, start = i32(lens, dev), i32([0, 1, 2, 3, 4], dev)
    want = ops.paged_attn(q, kp, vp, table, held, start, max_q=4, max_k=8000, scale=D ** -0.5)
    dt, out = ops._dt(q), torch.zeros_like(q)
    size = lib.avsr_paged_attn_workspace_bytes(dt, 4, 4, Hq, Hk, D, 448, 8000)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
    rc = lib.avsr_paged_attn(torch.cuda.current_stream().cuda_stream, dt, q.data_ptr(), Hq * D, D, kp.data_ptr(), kp.stride(0), kp.stride(1), vp.data_ptr(),
                             vp.stride(0), vp.stride(1), table.data_ptr(), table.stride(0), table.shape[1], held.data_ptr(), start.data_ptr(),
                             out.data_ptr(), Hq * D, D, 4, 4, Hq, Hk, D, 64, kp.shape[0], 448, 8000, D ** -0.5, 1, ws.data_ptr(), size)
    assert rc == 0 and torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,news,page", [([1500, 1100], [130, 70], 16), ([2500, 64, 2100], [100, 40, 1], 16), ([4300], [150], 32)])
def test_attn_chunks_over_long_tables(dev, dtype, D, lens, news, page):
    """Chunks of requests with more than 64 entries in the block table, keys split and not.  The bound of every element grows with the
    length; as a whole, the result is the exact one to HALF / sqrt(3) (a uniform rounding of a value at the lower end of its octave) and
    fp32 noise of 2^-16, while one key of 4300 is a part of 1 / sqrt(4300) = 0.015 in it."""
    got = attend_and_check(dev, lens, news, 4, 2, D, page, dtype, True, seed=31)
    g = torch.Generator().manual_seed(31)
    c = Cache(lens, 2, D, page, dtype, g)
    start = [sum(news[:b]) for b in range(len(news) + 1)]
    q = torch.randn(start[-1] + 3, 4, 2 * D, generator=g).to(dtype)[:, :, D:]
    want = torch.cat([attn_ref(q[start[b]:start[b + 1]], c.k[b], c.v[b], D ** -0.5, True, dtype)[0] for b in range(len(lens))])
    assert (got.double() - want).norm() <= (0.6 * HALF[dtype] + 2.0 ** -16) * want.norm()
