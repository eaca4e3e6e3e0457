"""Refusals of the serving operators, all before anything is launched, and their layouts and restatements on the CPU."""
import ctypes

import pytest
import torch

from mocov2_whisper_flamingo_amd import _lib, ops
from tests.serving_ref import plan_ref, up

I32 = torch.int32


def z(*shape, dtype=I32):
    return torch.zeros(shape, dtype=dtype)


def test_everything_needs_the_gpu():
    pages = z(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(_lib.AvsrHipError):
        ops.paged_plan(z(2), z(2), z(2, 3), z(4), z(2), 16, 8)
    with pytest.raises(_lib.AvsrHipError):
        ops.paged_write(z(3, 2, 64, dtype=torch.bfloat16), z(3, 2, 64, dtype=torch.bfloat16), pages, pages, z(3))
    with pytest.raises(_lib.AvsrHipError):
        ops.paged_attn(z(3, 2, 64, dtype=torch.bfloat16), pages, pages, z(2, 3), z(2), z(3))
    with pytest.raises(_lib.AvsrHipError):
        ops.w4_matmul(z(2, 40, dtype=torch.float32), ops.w4_pack(z(5, 40), torch.ones(5, 2), 32))
    with pytest.raises(_lib.AvsrHipError):
        ops.embed_tokens_at(z(2, dtype=torch.int64), z(5, 8, dtype=torch.float32), z(5, 8, dtype=torch.float32), z(2))


@pytest.mark.parametrize("change", [
    dict(lens=z(3)), dict(new=z(2, dtype=torch.int64)), dict(table=z(3, 3)), dict(table=z(2, 0)), dict(table=z(3, 2).t()),
    dict(pool=z(3)), dict(ring=z(0)), dict(page=24), dict(page=512), dict(tokens=0), dict(lens_out=z(3)), dict(pool_out=z(1)),
    dict(lens=z(4)[::2]), dict(lens=z(0), new=z(0))])
def test_plan_refuses(change):
    a = dict(lens=z(2), new=z(2), table=z(2, 3), ring=z(4), pool=z(2), page=16, tokens=8, lens_out=None, pool_out=None)
    a.update(change)
    with pytest.raises(ValueError):
        ops.paged_plan(a["lens"], a["new"], a["table"], a["ring"], a["pool"], a["page"], a["tokens"], lens_out=a["lens_out"],
                       pool_out=a["pool_out"])


@pytest.mark.parametrize("change", [
    dict(k=z(3, 2, 32, dtype=torch.float32)), dict(k=z(3, 1, 64, dtype=torch.float32)), dict(k=z(2, 2, 64, dtype=torch.float32)),
    dict(slots=z(4)), dict(slots=z(3, dtype=torch.int64)), dict(v_pages=z(3, 2, 16, 64, dtype=torch.float32)),
    dict(k=z(3, 64, 2, dtype=torch.float32).transpose(1, 2)), dict(k_pages=z(4, 16, 2, 64, dtype=torch.float32).transpose(1, 2)),
    dict(k_pages=z(4, 2, 8, 64, dtype=torch.float32), v_pages=z(4, 2, 8, 64, dtype=torch.float32))])
def test_write_refuses(change):
    a = dict(k=z(3, 2, 64, dtype=torch.float32), v=z(3, 2, 64, dtype=torch.float32), k_pages=z(4, 2, 16, 64, dtype=torch.float32),
             v_pages=z(4, 2, 16, 64, dtype=torch.float32), slots=z(3))
    a.update(change)
    with pytest.raises(ValueError):
        ops.paged_write(**a)


def test_types_are_refused():
    pages = z(4, 2, 16, 64, dtype=torch.float32)
    rows = z(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        ops.paged_write(rows, rows, pages, pages, z(3))
    with pytest.raises(TypeError):
        ops.paged_write(rows.half(), rows.half(), pages, pages, z(3))
    with pytest.raises(ValueError):
        ops.paged_attn(rows, pages, pages, z(2, 3), z(2), z(3))
    with pytest.raises(TypeError):
        ops.w4_matmul(z(2, 40, dtype=torch.float32), ops.w4_pack(z(5, 40), torch.ones(5, 2), 32), out_dtype=torch.float16)


@pytest.mark.parametrize("change", [
    dict(q=z(3, 3, 64, dtype=torch.float32)), dict(q=z(3, 2, 128, dtype=torch.float32)), dict(q=z(3, 128, dtype=torch.float32)),
    dict(lens=z(3)), dict(q_start=z(2)), dict(table=z(2, 3, dtype=torch.int64)), dict(max_q=0), dict(max_k=0),
    dict(out=z(3, 2, 64, dtype=torch.bfloat16)), dict(out=z(2, 2, 64, dtype=torch.float32))])
def test_attn_refuses(change):
    pages = z(4, 2, 16, 64, dtype=torch.float32)
    a = dict(q=z(3, 2, 64, dtype=torch.float32), k_pages=pages, v_pages=pages, table=z(2, 3), lens=z(2), q_start=z(3))
    a.update(change)
    with pytest.raises(ValueError):
        ops.paged_attn(**a)


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_attn_refuses_a_scale_that_is_not_finite(scale):
    pages = z(4, 2, 16, 64, dtype=torch.float32)
    with pytest.raises(ValueError):
        ops.paged_attn(z(3, 2, 64, dtype=torch.float32), pages, pages, z(2, 3), z(2), z(3), scale=scale)
    p = 4096
    assert _lib.load().avsr_paged_attn(None, 1, p, 256, 64, p, 4096, 1024, p, 4096, 1024, p, 3, 3, p, p, p, 256, 64, 3, 2, 4, 2, 64, 16, 9, 1, 40,
                                       scale, 1, None, 0) == -1


def test_w4_refuses():
    w = ops.w4_pack(z(5, 40), torch.ones(5, 2), 32)
    x = z(2, 40, dtype=torch.float32)
    for call in (lambda: ops.w4_pack(z(5, 40), torch.ones(5, 1), 32), lambda: ops.w4_pack(z(5, 40) + 8, torch.ones(5, 2), 32),
                 lambda: ops.w4_pack(z(5, 40) - 9, torch.ones(5, 2), 32), lambda: ops.w4_pack(z(5, 40), torch.ones(5, 3), 16),
                 lambda: ops.w4_pack(x, torch.ones(2, 2), 32), lambda: ops.w4_quantize(z(5, 40)), lambda: ops.w4_quantize(x, 48),
                 lambda: ops.w4_matmul(x[:, :39], w), lambda: ops.w4_matmul(x, w._replace(N=17)), lambda: ops.w4_matmul(x, w._replace(group=64)),
                 lambda: ops.w4_matmul(x, w, bias=z(4, dtype=torch.float32)), lambda: ops.w4_matmul(x, w, bias=z(5)),
                 lambda: ops.w4_matmul(x, w, act=ops.ACT_RELU_AFTER_RESIDUAL), lambda: ops.w4_matmul(x, w, residual=z(2, 4, dtype=torch.float32)),
                 lambda: ops.w4_matmul(x, w, residual=z(2, 5, dtype=torch.bfloat16)), lambda: ops.w4_matmul(x, w, out=z(3, 5, dtype=torch.float32)),
                 lambda: ops.w4_matmul(z(40, 2, dtype=torch.float32).t(), w)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_w4_weights_and_scales_have_to_be_finite(bad):
    w = torch.ones(3, 40)
    w[1, 7] = bad
    with pytest.raises(ValueError, match="finite"):
        ops.w4_quantize(w, 32)
    with pytest.raises(ValueError, match="finite"):
        ops.w4_pack(z(3, 40), w[:, 6:8], 32)


def test_c_entries_refuse_before_they_launch():
    """Status codes of calls whose pointers are never read: -1 for what cannot be, -2 for what is not built."""
    lib = _lib.load()
    p = 4096                                     # an aligned address that is never followed
    plan = lambda B=2, page=16, width=3, ld=3, n=4, tokens=8, ws=p, lens=p: lib.avsr_paged_plan(
        None, lens, p, p, ld, width, p, n, p, B, page, tokens, p, p, p, p, p, p, ws)
    assert plan(lens=None) == -1 and plan(B=0) == -1 and plan(ld=2) == -1 and plan(tokens=0) == -1 and plan(n=0) == -1
    assert plan(B=5000, ws=None) == -1 and lib.avsr_paged_plan_workspace_bytes(5000, 8, 4) > 0
    assert plan(page=17) == -2 and plan(page=8) == -2 and plan(n=1 << 27) == -2 and plan(width=1 << 27, ld=1 << 27) == -2
    write = lambda it=1, ot=1, k=p, ldk=128, D=64, page=16, slots=p, n=4: lib.avsr_paged_write(
        None, it, ot, k, ldk, 64, p, 128, 64, p, 2048, 1024, p, 2048, 1024, slots, 3, 2, D, page, n)
    assert write(k=None) == -1 and write(slots=None) == -1 and write(it=1, ot=0) == -1 and write(it=2) == -1
    assert write(D=96) == -2 and write(page=48) == -2 and write(ldk=130) == -2 and write(k=p + 2) == -2 and write(n=1 << 27) == -2
    attn = lambda dt=1, q=p, N=3, B=2, Hq=4, Hk=2, D=64, page=16, ldq=256, mq=1, ws=None, wb=0, width=3: lib.avsr_paged_attn(
        None, dt, q, ldq, 64, p, 4096, 1024, p, 4096, 1024, p, width, width, p, p, p, 256, 64, N, B, Hq, Hk, D, page, 9, mq, 40, 1.0, 1, ws, wb)
    assert attn(q=None) == -1 and attn(B=0) == -1 and attn(Hq=3) == -1 and attn(mq=0) == -1 and attn(dt=7) == -1 and attn(N=-1) == -1
    assert attn(D=80) == -2 and attn(page=20) == -2 and attn(ldq=258) == -2 and attn(q=p + 8) == -2 and attn(N=1 << 29) == -2
    long = lambda ws, wb: lib.avsr_paged_attn(None, 1, p, 256, 64, p, 4096, 1024, p, 4096, 1024, p, 999, 999, p, p, p, 256, 64, 2, 2, 4, 2, 64,
                                              16, 9, 1, 15984, 1.0, 1, ws, wb)
    need = lib.avsr_paged_attn_workspace_bytes(1, 2, 2, 4, 2, 64, 1, 15984)
    assert need > 0 and long(None, 0) == -1 and long(p, need - 1) == -1
    w4 = lambda xt=1, ot=1, x=p, ldx=64, group=32, act=0, ldy=32, packed=p, K=64: lib.avsr_w4_matmul(
        None, xt, ot, x, ldx, packed, p, group, None, act, None, 0, p, ldy, 2, 32, K)
    assert w4(x=None) == -1 and w4(xt=3) == -1 and w4(ot=3) == -1 and w4(ldx=63) == -1 and w4(ldy=31) == -1 and w4(act=3) == -1
    assert w4(group=16) == -2 and w4(packed=p + 4) == -2 and w4(K=0) == -1
    assert lib.avsr_embed_tokens_at(None, 0, p, p, p, None, p, 2, 64, 10, 10, 1.0, None) == -1
    assert lib.avsr_embed_tokens_at(None, 0, p, p, p, p, p, 2, 66, 10, 10, 1.0, None) == -2


@pytest.mark.parametrize("N,K,group", [(5, 40, 32), (16, 128, 64), (33, 300, 128), (1, 1, 32)])
def test_w4_layout(N, K, group):
    """Every nibble and scale stands where the header puts it; what pads the tiles is nibble 8 and scale 0."""
    g = torch.Generator().manual_seed(N)
    q = torch.randint(-8, 8, (N, K), generator=g)
    s = torch.rand(N, up(K, group), generator=g).to(torch.bfloat16)
    w = ops.w4_pack(q, s, group)
    assert tuple(w.packed.shape) == (up(N, 16), up(K, 128), 4, 16, 4) and tuple(w.scales.shape) == (up(N, 16), up(K, 128) * 128 // group, 16)
    for n in range(up(N, 16) * 16):
        for k in range(up(K, 128) * 128):
            word = int(w.packed[n // 16, k // 128, k // 8 % 4, n % 16, k // 32 % 4]) & 0xFFFFFFFF
            e = k % 8
            nib = (word >> (4 * (e // 2) + 16 * (e % 2))) & 15
            inside = n < N and k < K
            assert nib == (int(q[n, k]) + 8 if inside else 8)
            sc = float(w.scales[n // 16, k // group, n % 16])
            assert sc == (float(s[n, k // group]) if n < N and k // group < s.shape[1] else 0.0)


def test_w4_quantize_rounds_to_nearest():
    g = torch.Generator().manual_seed(3)
    w = torch.randn(7, 100, generator=g)
    w[2, 32:64] = 0
    p = ops.w4_quantize(w, 32)
    s = torch.stack([p.scales[0, :, i] for i in range(7)]).float()
    for n in range(7):
        for k in range(100):
            word = int(p.packed[0, 0, k // 8 % 4, n, k // 32 % 4]) & 0xFFFFFFFF
            q = ((word >> (4 * (k % 8 // 2) + 16 * (k % 2))) & 15) - 8
            sc = float(s[n, k // 32])
            # half a step of the grid; the scale's own rounding may push the largest value 7 * 2^-8 steps beyond 7
            assert abs(float(w[n, k]) - q * sc) <= (0.5 + 1e-6) * sc
    assert float(s[2, 1]) == 0.0


def test_plan_restatement_keeps_every_page_once():
    """The oracle's own bookkeeping: over random steps the pages in tables and ring are a permutation of all pages."""
    import random
    rng = random.Random(5)
    B, page, width, n = 6, 16, 5, 20
    lens, table, ring, pool = [0] * B, [[-1] * width for _ in range(B)], list(range(n)), [0, n]
    for step in range(200):
        new = [rng.choice([-1, 0, 1, 1, 17, 40]) for _ in range(B)]
        r = plan_ref(lens, new, table, ring, pool, page, 64)
        if r["status"]:
            assert r["slots"] == [-1] * 64
        lens, table, ring, pool = r["lens"], r["table"], r["ring"], r["pool"]
        held = [table[b][j] for b in range(B) for j in range(up(lens[b], page))]
        free = [ring[(pool[0] + i) % n] for i in range(pool[1])]
        assert sorted(held + free) == list(range(n))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [0, 1])
def test_attn_workspace_of_a_general_bound(dtype, D):
    """A bound for any step (max_q above the rows of this one) asks for what the tight one does, and fewer keys never for more: what the
    query says is enough for the call, whatever it knows besides."""
    size = _lib.load().avsr_paged_attn_workspace_bytes
    for N, B, Hq, Hk, k in ((4, 4, 32, 8, 8000), (1, 1, 20, 20, 4000), (8, 3, 12, 12, 1500), (70, 2, 16, 4, 30000), (2, 2, 7, 1, 700)):
        tight = size(dtype, N, B, Hq, Hk, D, N, k)
        assert tight > 0
        for q in (N + 1, 65, 448, 1 << 40):
            if q > N:
                assert size(dtype, N, B, Hq, Hk, D, q, k) == tight
        most = 0
        for fewer in range(1, k + 1, 37):
            here = size(dtype, N, B, Hq, Hk, D, 1, fewer)
            assert here >= most
            most = here


@pytest.mark.parametrize("scale", [torch.tensor(3.4e38), -torch.tensor(3.4e38), torch.tensor(1e300, dtype=torch.float64)])
def test_w4_scales_have_to_stay_finite_in_bf16(scale):
    """Finite in the caller's type, but beyond the largest bf16 value (3.39e38): they would be infinite in the packed weights."""
    s = torch.ones(3, 2, dtype=scale.dtype)
    s[1, 1] = scale
    with pytest.raises(ValueError, match="finite"):
        ops.w4_pack(z(3, 40), s, 32)
    s[1, 1] = scale.sign() * 3.38e38
    assert torch.isfinite(ops.w4_pack(z(3, 40), s, 32).scales).all()
