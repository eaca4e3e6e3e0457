"""The Whisper decoder served to requests of different lengths (paged cache, 4-bit weights) against the CPU oracle."""
import random

import pytest
import torch

import oracle
from mocov2_whisper_flamingo_amd import PagedKVCache, WhisperConfig, WhisperModel, _lib, ops
from tests.helpers import max_err, seed_module

pytestmark = pytest.mark.gpu
TOL = {torch.float32: 1e-3, torch.bfloat16: 2e-2}
VOCAB = 503


def model(dev, seed=31, d=128, heads=2):
    cfg = WhisperConfig(d_model=d, decoder_layers=2, decoder_attention_heads=heads, vocab_size=VOCAB, max_target_positions=448)
    m = WhisperModel(cfg)
    sd = seed_module(m, seed)
    return m.to(dev).decoder, sd, cfg


def unpack(w):
    """fp32 [N, K] values of a W4Weight."""
    T, C = w.packed.shape[:2]
    place = torch.tensor([0, 16, 4, 20, 8, 24, 12, 28], dtype=torch.int32)
    q = (torch.bitwise_right_shift(w.packed.cpu()[..., None], place) & 15) - 8
    q = q.view(T, C, 4, 16, 4, 8).permute(0, 3, 1, 4, 2, 5).reshape(T * 16, -1, w.group).float()
    s = w.scales.cpu().float().permute(0, 2, 1).reshape(T * 16, -1, 1)
    return (q * s).view(T * 16, -1)[:w.N, :w.K]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("page_size,frames", [(16, True), (64, True), (32, False)])
def test_requests_that_come_and_go(dev, dtype, page_size, frames):
    """A random schedule over four places: prompts, tokens, waiting, ends, new requests in their places.  Every hidden state is the
    one the oracle gives for that position of the request's own sequence, and at the end all pages are free again."""
    dec, sd, cfg = model(dev)
    rng, g = random.Random(7), torch.Generator().manual_seed(3)
    R, Te = 4, 50
    cache = dec.new_paged_cache(R, page_size=page_size, max_tokens=192, frames=Te if frames else None, dtype=dtype)
    seqs, encs, states = [None] * R, [None] * R, [None] * R
    served = 0
    for step in range(26):
        fresh = [r for r in range(R) if seqs[r] is None and rng.random() < 0.7]
        if fresh:
            te = rng.randint(1, Te)
            enc = torch.randn(len(fresh), te, cfg.d_model, generator=g)
            if frames:
                dec.paged_admit(cache, fresh, enc.to(dev))
            for i, r in enumerate(fresh):
                seqs[r], encs[r], states[r] = [], enc[i:i + 1], []
        new, ids = [0] * R, []
        for r in range(R):
            if seqs[r] is None:
                continue
            if not seqs[r]:
                new[r] = rng.choice([1, 3, 20, 70])
            else:
                new[r] = rng.choice([0, 1, 1, 1, 1, 5, -1]) if len(seqs[r]) < 150 else -1
            if new[r] > 0:
                t = [rng.randrange(3, VOCAB) for _ in range(new[r])]
                seqs[r] += t
                ids += t
        h, plan = dec.paged_step(cache, torch.tensor(ids, dtype=torch.int64, device=dev), new)
        assert h.shape == (len(ids), cfg.d_model)
        at = 0
        for r in range(R):
            if new[r] > 0:
                states[r].append(h[at:at + new[r]].float().cpu())
                at += new[r]
            elif new[r] < 0:
                ref = oracle.whisper_decoder(sd, "decoder.", torch.tensor([seqs[r]]), encs[r] if frames else None, 2)[0]
                assert max_err(torch.cat(states[r]), ref) < TOL[dtype], (step, r)
                served += 1
                if frames:
                    dec.paged_end(cache, [r])
                seqs[r] = None
    assert served >= 3
    live = [r for r in range(R) if seqs[r]]
    for r in live:
        ref = oracle.whisper_decoder(sd, "decoder.", torch.tensor([seqs[r]]), encs[r] if frames else None, 2)[0]
        assert max_err(torch.cat(states[r]), ref) < TOL[dtype]
    dec.paged_end(cache, range(R))
    for part in (cache.tokens, cache.frames):
        if part is not None:
            n = part.ring.numel()
            head, count = part.pool.tolist()
            assert count == n and sorted(part.ring.tolist()) == list(range(n)) and part.lens.tolist() == [0] * R
    assert cache.bad.item() == 0


def test_a_step_that_does_not_fit_changes_nothing(dev):
    dec, sd, cfg = model(dev)
    cache = dec.new_paged_cache(2, pages=4, page_size=16, max_tokens=48)
    ids = torch.arange(3, 43, device=dev)
    dec.paged_step(cache, ids[:40], [20, 20])
    state = lambda: [t.tolist() for t in (cache.tokens.lens, cache.tokens.table, cache.tokens.ring, cache.tokens.pool)]
    before = state()
    with pytest.raises(_lib.AvsrHipError, match="free pages"):
        dec.paged_step(cache, ids[:14], [1, 13])
    with pytest.raises(_lib.AvsrHipError, match="outgrows"):
        dec.paged_step(cache, ids[:29], [29, 0])
    with pytest.raises(IndexError):
        dec.paged_step(cache, torch.tensor([5, VOCAB], device=dev), [1, 1])
    with pytest.raises(IndexError):
        dec.paged_step(cache, torch.tensor([-1, 5], device=dev), [1, 1])
    for bad in (([1], ids[:1]), ([1, 1], ids[:3]), ([2, -1], ids[:1])):
        with pytest.raises(ValueError):
            dec.paged_step(cache, bad[1], bad[0])
    with pytest.raises(ValueError):
        dec.paged_step(cache, ids[:2].view(1, 2), [1, 1])
    with pytest.raises(ValueError):
        dec.paged_admit(cache, [0], torch.zeros(1, 4, cfg.d_model, device=dev))
    assert state() == before
    h, _ = dec.paged_step(cache, ids[:0], [-1, 0])
    assert h.shape == (0, cfg.d_model) and cache.tokens.lens.tolist() == [0, 20]
    for kw in (dict(max_tokens=449), dict(page_size=256), dict(max_tokens=40, page_size=32), dict(page_size=24)):
        with pytest.raises(ValueError):
            dec.new_paged_cache(2, **kw)
    two = dec.new_paged_cache(2, frames=8, frame_pages=1, page_size=16, max_tokens=48)
    enc = torch.randn(2, 8, cfg.d_model, device=dev)
    with pytest.raises(_lib.AvsrHipError, match="free pages"):
        dec.paged_admit(two, [0, 1], enc)
    dec.paged_admit(two, [1], enc[:1])
    for which in ([1], [1, 0], [0, 0], [2], [-1]):
        with pytest.raises(ValueError):
            dec.paged_admit(two, which, enc[:len(which)])
    with pytest.raises(ValueError):
        PagedKVCache(1, 1, 1, pages=0, max_tokens=16)


def test_frames_that_cannot_be_admitted_take_no_pages(dev):
    """Encoder output of another width, on another device, or without frames."""
    dec, sd, cfg = model(dev)
    cache = dec.new_paged_cache(2, frames=32, page_size=16)
    for bad in (torch.zeros(1, 8, cfg.d_model + 8, device=dev), torch.zeros(1, 8, cfg.d_model), torch.zeros(1, 0, cfg.d_model, device=dev)):
        with pytest.raises(ValueError):
            dec.paged_admit(cache, [0], bad)
    with pytest.raises(_lib.AvsrHipError, match="outgrows"):
        dec.paged_admit(cache, [0], torch.zeros(1, 33, cfg.d_model, device=dev))
    assert cache.frames.lens.tolist() == [0, 0] and cache.frames.pool.tolist() == [0, 4]
    dec.paged_admit(cache, [0, 1], torch.zeros(2, 32, cfg.d_model, device=dev))
    assert cache.frames.pool.tolist() == [0, 0]


def test_greedy_ragged_is_greedy_for_each_prompt(dev):
    dec, sd, cfg = model(dev, seed=23)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(3, VOCAB, (n,), generator=g).tolist() for n in (1, 7, 3, 40)]
    enc = torch.randn(4, 50, cfg.d_model, generator=g)
    want = [dec.greedy(torch.tensor([p], device=dev), enc[i:i + 1].to(dev), 12, dtype=torch.float32)[0].tolist() for i, p in enumerate(prompts)]
    assert dec.greedy_ragged(prompts, enc.to(dev), 12, dtype=torch.float32, page_size=16) == want
    eos = want[1][9]                                       # ends prompt 1 early, others perhaps
    want = [dec.greedy(torch.tensor([p], device=dev), enc[i:i + 1].to(dev), 12, eos_token_id=eos, dtype=torch.float32)[0].tolist()
            for i, p in enumerate(prompts)]
    got = dec.greedy_ragged(prompts, enc.to(dev), 12, eos_token_id=eos, dtype=torch.float32)
    assert got == want and len(got[1]) <= 10
    assert dec.greedy_ragged(prompts[:1], enc[:1].to(dev), 0, dtype=torch.float32) == prompts[:1]
    with pytest.raises(ValueError):
        dec.greedy_ragged([[]], enc[:1].to(dev), 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group,head", [(32, False), (128, True)])
def test_quantized_decoder(dev, dtype, group, head):
    """With 4-bit weights the decoder is the oracle on the weights those bits stand for: one pass, incremental, paged; and back."""
    dec, sd, cfg = model(dev, seed=41)
    g = torch.Generator().manual_seed(6)
    ids, enc = torch.randint(3, VOCAB, (2, 12), generator=g), torch.randn(2, 30, cfg.d_model, generator=g)
    full = dec(ids.to(dev), encoder_hidden_states=enc.to(dev), dtype=dtype)[0].float().cpu()
    assert dec.quantize(group, head=head) is dec
    q, s = dict(sd), 64 ** -0.5
    pk = dec._pack(dtype)
    for i, lw in enumerate(pk["layers"]):
        pre, D = f"decoder.layers.{i}.", cfg.d_model
        assert all(isinstance(lw[n], ops.W4Weight) for n in ("wqkv", "wo", "wq_x", "wo_x", "wfc1", "wfc2"))
        wqkv = unpack(lw["wqkv"])
        for j, n in enumerate(("q_proj", "k_proj", "v_proj")):
            q[pre + f"self_attn.{n}.weight"] = wqkv[j * D:(j + 1) * D] / (s if j == 0 else 1.0)
        q[pre + "self_attn.out_proj.weight"] = unpack(lw["wo"])
        q[pre + "encoder_attn.q_proj.weight"] = unpack(lw["wq_x"]) / s
        q[pre + "encoder_attn.out_proj.weight"] = unpack(lw["wo_x"])
        q[pre + "fc1.weight"], q[pre + "fc2.weight"] = unpack(lw["wfc1"]), unpack(lw["wfc2"])
        for n in ("self_attn.q_proj", "encoder_attn.q_proj", "fc1", "fc2"):
            w, o = q[pre + n + ".weight"], sd[pre + n + ".weight"]
            assert 0.02 < ((w - o).norm() / o.norm()).item() < 0.2          # 4 bits: really rounded, and near
    ref = oracle.whisper_decoder(q, "decoder.", ids, enc, 2)
    h = dec(ids.to(dev), encoder_hidden_states=enc.to(dev), dtype=dtype)[0]
    assert max_err(h, ref) < TOL[dtype]
    cache = dec.new_cache(2, enc.to(dev), dtype, max_tokens=16)
    parts = [dec.decode_step(ids[:, :8].to(dev), cache)] + [dec.decode_step(ids[:, t:t + 1].to(dev), cache) for t in range(8, 12)]
    assert max_err(torch.cat(parts, 1), ref) < TOL[dtype]
    paged = dec.new_paged_cache(2, frames=30, dtype=dtype)
    dec.paged_admit(paged, [0, 1], enc.to(dev))
    a, _ = dec.paged_step(paged, torch.cat([ids[0, :8], ids[1, :3]]).to(dev), [8, 3])
    b, _ = dec.paged_step(paged, torch.cat([ids[0, 8:], ids[1, 3:]]).to(dev), [4, 9])
    assert max_err(torch.cat([a[:8], b[:4]]), ref[0]) < TOL[dtype] and max_err(torch.cat([a[8:], b[4:]]), ref[1]) < TOL[dtype]
    logits = dec.project_tokens(h)
    w = unpack(dec._proj[1]) if head else sd["decoder.embed_tokens.weight"]
    want = h.float().cpu() @ w.t()
    assert max_err(logits, want) < TOL[dtype] * max(1.0, want.abs().max().item())
    dec.quantize(None)
    assert torch.equal(dec(ids.to(dev), encoder_hidden_states=enc.to(dev), dtype=dtype)[0].float().cpu(), full)
    with pytest.raises(ValueError):
        dec.quantize(48)


@pytest.mark.parametrize("group", [None, 64])
def test_paged_step_captured_and_replayed(dev, group):
    """The serving loop as a graph: one recording decodes a token for each request, whatever their lengths; eager work and
    synchronizations lie between the replays."""
    dec, sd, cfg = model(dev, seed=51)
    dec.quantize(group)
    R = 3
    enc = torch.randn(R, 40, cfg.d_model, generator=torch.Generator().manual_seed(1)).to(dev)

    def start():
        c = dec.new_paged_cache(R, frames=40, page_size=16, max_tokens=64)
        dec.paged_admit(c, range(R), enc)
        dec.paged_step(c, torch.arange(3, 3 + 22, device=dev), [1, 15, 6])
        return c

    graphed, eager = start(), start()
    new, ids = torch.ones(R, dtype=torch.int32, device=dev), torch.full((R,), 5, dtype=torch.int64, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    warm = start()
    with torch.cuda.stream(side):
        dec.paged_step(warm, ids, new, max_new=1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, plan = dec.paged_step(graphed, ids, new, max_new=1)
        nxt = dec.project_tokens(h[None]).view(R, -1)
    for i in range(12):
        if i == 7:
            new.copy_(torch.tensor([1, -1, 1], dtype=torch.int32))      # a request ends: its row of the batch is empty from here on
        if i == 8:
            new.copy_(torch.tensor([1, 0, 1], dtype=torch.int32))
        ids.copy_(torch.randint(3, VOCAB, (R,), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        rows = 3 if i < 7 else 2
        want, p = dec.paged_step(eager, ids, new, max_new=1)
        assert plan.status.item() == 0 and p.status.item() == 0
        assert torch.equal(h[:rows], want[:rows]), i
        assert torch.equal(nxt[:rows], dec.project_tokens(want[None]).view(R, -1)[:rows])
        assert graphed.tokens.lens.tolist() == eager.tokens.lens.tolist()
    assert graphed.bad.item() == 0


def test_calls_that_are_refused_leave_the_cache_as_it_was(dev):
    """Everything that can be wrong with a step is looked at before the cache moves on."""
    dec, sd, cfg = model(dev)
    cache = dec.new_paged_cache(2, page_size=16, max_tokens=48)
    ids = torch.arange(3, 43, device=dev)
    dec.paged_step(cache, ids[:12], [7, 5])
    state = lambda: [t.tolist() for t in (cache.tokens.lens, cache.tokens.table, cache.tokens.ring, cache.tokens.pool)]
    before, one = state(), torch.ones(2, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        dec.paged_step(cache, ids[:2].cpu(), [1, 1])
    with pytest.raises(ValueError):
        dec.paged_step(cache, ids[:2].cpu(), one, max_new=1)
    for bad in (0, -1):
        with pytest.raises(ValueError):
            dec.paged_step(cache, ids[:2], one, max_new=bad)
    for new in (one.cpu(), one.long(), one[:1], torch.ones(3, dtype=torch.int32, device=dev)):
        with pytest.raises(ValueError):
            dec.paged_step(cache, ids[:2], new, max_new=1)
    for other in (model(dev, d=192, heads=3)[0], WhisperModel(WhisperConfig(d_model=128, decoder_layers=3, decoder_attention_heads=2, vocab_size=VOCAB,
                                                                            max_target_positions=448)).to(dev).decoder):
        with pytest.raises(ValueError):
            other.paged_step(cache, ids[:2], [1, 1])
        framed = other.new_paged_cache(2, page_size=16, frames=16)
        with pytest.raises(ValueError):
            dec.paged_admit(framed, [0], torch.zeros(1, 16, cfg.d_model, device=dev))
        assert framed.frames.lens.tolist() == [0, 0]
    assert state() == before
    seq = torch.cat([ids[:7], ids[20:21]]).cpu()
    h, _ = dec.paged_step(cache, ids[20:22], [1, 1])
    ref = oracle.whisper_decoder(sd, "decoder.", seq[None], None, 2)[0]
    assert max_err(h[:1], ref[-1:]) < TOL[torch.bfloat16]


def test_requests_without_frames_are_refused(dev):
    """With a cache for frames, a request that was not admitted (or was not again after its end) has nothing to attend to."""
    dec, sd, cfg = model(dev)
    cache = dec.new_paged_cache(3, frames=20, page_size=16, max_tokens=48)
    enc, ids = torch.randn(1, 20, cfg.d_model, device=dev), torch.arange(3, 10, device=dev)
    dec.paged_admit(cache, [1], enc)
    with pytest.raises(ValueError, match="admit"):
        dec.paged_step(cache, ids[:4], [2, 2, 0])
    assert cache.tokens.lens.tolist() == [0, 0, 0]
    dec.paged_step(cache, ids[:2], [0, 2, 0])
    dec.paged_end(cache, [1])
    with pytest.raises(ValueError, match="admit"):
        dec.paged_step(cache, ids[:2], [0, 2, 0])
    assert cache.tokens.lens.tolist() == [0, 0, 0]
    dec.paged_step(cache, ids[:0], [-1, 0, -1])                 # ends and waits need no frames


@pytest.mark.parametrize("page_size", [16, 64, 128, 256])
@pytest.mark.parametrize("positions", [448, 100])
def test_greedy_ragged_takes_every_page_size(dev, page_size, positions):
    """Also where the positions are no multiple of it; and the limits of the length are those of greedy."""
    cfg = WhisperConfig(d_model=128, decoder_layers=2, decoder_attention_heads=2, vocab_size=VOCAB, max_target_positions=positions)
    m = WhisperModel(cfg)
    seed_module(m, 61)
    dec = m.to(dev).decoder
    g = torch.Generator().manual_seed(8)
    prompts = [torch.randint(3, VOCAB, (n,), generator=g).tolist() for n in (4, positions - 3, positions, 30)]
    enc = torch.randn(4, 30, cfg.d_model, generator=g).to(dev)
    want = [dec.greedy(torch.tensor([p], device=dev), enc[i:i + 1], 9, dtype=torch.float32)[0].tolist() for i, p in enumerate(prompts)]
    got = dec.greedy_ragged(prompts, enc, 9, dtype=torch.float32, page_size=page_size)
    assert got == want and [len(w) for w in want] == [13, positions + 1, positions + 1, 39]
    with pytest.raises(ValueError):
        dec.greedy_ragged([prompts[0], [5] * (positions + 1)], enc[:2], 2, dtype=torch.float32, page_size=page_size)


@pytest.mark.parametrize("most", [0, -1, -5])
def test_greedy_ragged_adds_nothing_for_no_tokens(dev, most):
    dec, sd, cfg = model(dev)
    enc = torch.zeros(2, 16, cfg.d_model, device=dev)
    assert dec.greedy_ragged([[5, 6], [7]], enc, most, dtype=torch.float32) == [[5, 6], [7]]
