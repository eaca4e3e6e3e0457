"""Whisper decoder on the HIP kernels: causal self-attention, cross-attention to
the encoder output and the GELU MLP of every layer, with the checkpoint key
names of ``whisper_model.decoder.*`` (the reference constructs the decoder with
``WhisperModel.from_pretrained`` at models/av_net.py:22 but never calls it; the
arithmetic is HF ``WhisperDecoder`` / ``WhisperDecoderLayer``,
modeling_whisper.py:649-797 / 416-505).

Forward only.  ``forward`` decodes a whole token sequence in one pass (teacher
forcing / scoring); ``new_cache`` + ``decode_step`` decode incrementally with the
self-attention keys / values of earlier tokens kept in a cache (what HF's
``DynamicCache`` holds, hf:649-797 ``past_key_values``), the causal attention
kernel taking the new tokens as the LAST queries of the cached sequence.
``cross_kv`` exposes the per-layer encoder projections so they are computed
once per encoder output.

``new_paged_cache`` + ``paged_admit`` + ``paged_step`` + ``paged_end`` serve requests
of different lengths that come and go: a step takes each request's new tokens (a
prompt, one token, none) as rows of one ragged batch over a cache in pages;
``greedy_ragged`` decodes a list of prompts that way.  ``quantize`` keeps the
layers' weights in 4 bits.
"""
import torch
import torch.nn as nn

from . import ops
from .paged_cache import PagedKVCache
from .whisper_encoder import _Attention


def _linear(x, w, **kw):
    """x @ w^T with the epilogue of ``ops.gemm_nt``, for a weight matrix or its 4-bit form."""
    return ops.w4_matmul(x, w, **kw) if isinstance(w, ops.W4Weight) else ops.gemm_nt(x, w, **kw)


class PagedDecoderCache:
    """What a server keeps for its requests: ``tokens`` (self-attention), ``frames`` (cross-attention, or None), and ``bad``, an int32
    GPU flag that a token id or position outside the embedding tables sets."""

    def __init__(self, tokens, frames, dtype, device):
        self.tokens, self.frames, self.dtype = tokens, frames, dtype
        self.bad = torch.zeros(1, dtype=torch.int32, device=device)


class _DecoderLayer(nn.Module):
    def __init__(self, d):
        super().__init__()
        self.self_attn = _Attention(d)
        self.self_attn_layer_norm = nn.LayerNorm(d)
        self.encoder_attn = _Attention(d)
        self.encoder_attn_layer_norm = nn.LayerNorm(d)
        self.fc1 = nn.Linear(d, 4 * d)
        self.fc2 = nn.Linear(4 * d, d)
        self.final_layer_norm = nn.LayerNorm(d)


class WhisperDecoder(nn.Module):
    def __init__(self, cfg):
        super().__init__()
        self.cfg = cfg
        d = cfg.d_model
        self.embed_tokens = nn.Embedding(cfg.vocab_size, d)
        self.embed_positions = nn.Embedding(cfg.max_target_positions, d)
        self.layers = nn.ModuleList([_DecoderLayer(d) for _ in range(cfg.decoder_layers)])
        self.layer_norm = nn.LayerNorm(d)
        self._packed = None
        self._proj = None
        self._w4 = None            # (group, with the vocabulary) of quantize()

    # ---- weight packing -------------------------------------------------
    def _versions(self, dtype):
        return (dtype, self._w4, sum(p._version for p in self.parameters()), next(self.parameters()).data_ptr())

    def _pack(self, dtype):
        """Per weight version: q/k/v of the self-attention fused into one [3D, D] matrix, k/v of the
        cross-attention into one [2D, D] matrix (k_proj has no bias), the head_dim**-0.5 query scaling folded
        into W_q and b_q (0.125: exact)."""
        key = self._versions(dtype)
        if self._packed is not None and self._packed[0] == key:
            return self._packed[1]
        d = self.cfg.d_model
        if d // self.cfg.decoder_attention_heads != 64:
            raise ValueError("attention kernels are built for head_dim 64")
        s = 64 ** -0.5
        f32 = lambda t: t.detach().float().contiguous()
        cd = lambda t: t.detach().to(dtype).contiguous()
        ln = lambda m: (f32(m.weight), f32(m.bias))
        pk = {"tok": f32(self.embed_tokens.weight), "pos": f32(self.embed_positions.weight),
              "lnf": ln(self.layer_norm), "layers": []}
        for L in self.layers:
            a, x = L.self_attn, L.encoder_attn
            zb = torch.zeros_like(a.q_proj.bias)
            pk["layers"].append({
                "ln1": ln(L.self_attn_layer_norm),
                "wqkv": cd(torch.cat([a.q_proj.weight.detach() * s, a.k_proj.weight.detach(), a.v_proj.weight.detach()], 0)),
                "bqkv": f32(torch.cat([a.q_proj.bias.detach() * s, zb, a.v_proj.bias.detach()], 0)),
                "wo": cd(a.out_proj.weight), "bo": f32(a.out_proj.bias),
                "lnx": ln(L.encoder_attn_layer_norm),
                "wq_x": cd(x.q_proj.weight.detach() * s), "bq_x": f32(x.q_proj.bias.detach() * s),
                "wkv_x": cd(torch.cat([x.k_proj.weight.detach(), x.v_proj.weight.detach()], 0)),
                "bkv_x": f32(torch.cat([zb, x.v_proj.bias.detach()], 0)),
                "wo_x": cd(x.out_proj.weight), "bo_x": f32(x.out_proj.bias),
                "ln2": ln(L.final_layer_norm),
                "wfc1": cd(L.fc1.weight), "bfc1": f32(L.fc1.bias),
                "wfc2": cd(L.fc2.weight), "bfc2": f32(L.fc2.bias),
            })
            if self._w4 is not None:
                lw = pk["layers"][-1]
                lw["wqkv"] = torch.cat([a.q_proj.weight.detach() * s, a.k_proj.weight.detach(), a.v_proj.weight.detach()], 0)
                lw["wq_x"] = x.q_proj.weight.detach() * s
                lw["wo"], lw["wo_x"] = a.out_proj.weight, x.out_proj.weight
                lw["wfc1"], lw["wfc2"] = L.fc1.weight, L.fc2.weight
                for name in ("wqkv", "wo", "wq_x", "wo_x", "wfc1", "wfc2"):
                    lw[name] = ops.w4_quantize(lw[name], self._w4[0])
        self._packed = (key, pk)
        return pk

    # ---- forward ----------------------------------------------------------
    @torch.no_grad()
    def cross_kv(self, encoder_hidden_states, dtype=torch.bfloat16):
        """Per-layer [B, Te, 2D] key|value projections of the encoder output (k_proj / v_proj of
        ``encoder_attn``): what HF keeps in the cross-attention half of its cache."""
        pk = self._pack(dtype)
        B, Te, D = encoder_hidden_states.shape
        e = encoder_hidden_states
        e = (e if (e.dtype == dtype and e.is_contiguous()) else ops.cast(e.contiguous(), dtype)).view(B * Te, D)
        return [ops.gemm_nt(e, lw["wkv_x"], bias=lw["bkv_x"]).view(B, Te, 2 * D) for lw in pk["layers"]]

    @torch.no_grad()
    def forward(self, input_ids, attention_mask=None, encoder_hidden_states=None, dtype=torch.bfloat16, cross_kv=None):
        """input_ids int64 [B, T] (T <= max_target_positions); ``attention_mask`` [B, T] with 0 on padding
        tokens (keys of the self-attention only, as HF builds its causal mask); ``encoder_hidden_states``
        [B, Te, D] or ``cross_kv`` from :meth:`cross_kv`; with neither the cross-attention is skipped
        (hf:474).  Returns ``([B, T, D] in the compute dtype,)`` = ``last_hidden_state``."""
        cfg = self.cfg
        if input_ids.dim() != 2:
            raise ValueError("input_ids must be [batch, tokens]")
        B, T = input_ids.shape
        if T > cfg.max_target_positions:
            raise ValueError(f"{T} decoder tokens exceed max_target_positions={cfg.max_target_positions}")
        pk = self._pack(dtype)
        H, D = cfg.decoder_attention_heads, cfg.d_model
        use_mfma = dtype == torch.bfloat16
        xs = ops.embed_tokens(input_ids, pk["tok"], pk["pos"])           # fp32 residual stream [B*T, D]
        km = None if attention_mask is None else (attention_mask == 0).to(torch.uint8).contiguous()
        if cross_kv is None and encoder_hidden_states is not None:
            cross_kv = self.cross_kv(encoder_hidden_states, dtype)
        for i, lw in enumerate(pk["layers"]):
            h = ops.layernorm_fwd(xs, *lw["ln1"], out_dtype=dtype)
            qkv = _linear(h, lw["wqkv"], bias=lw["bqkv"]).view(B, T, 3 * D)
            o = ops.attn_fwd(qkv[:, :, :D], qkv[:, :, D:2 * D], qkv[:, :, 2 * D:], H, key_mask=km, scale=1.0,
                             use_mfma=use_mfma, causal=True)
            _linear(o.view(B * T, D), lw["wo"], bias=lw["bo"], residual=xs, out=xs)
            if cross_kv is not None:
                kv = cross_kv[i]
                h = ops.layernorm_fwd(xs, *lw["lnx"], out_dtype=dtype)
                q = _linear(h, lw["wq_x"], bias=lw["bq_x"]).view(B, T, D)
                o = ops.attn_fwd(q, kv[:, :, :D], kv[:, :, D:], H, scale=1.0, use_mfma=use_mfma)
                _linear(o.view(B * T, D), lw["wo_x"], bias=lw["bo_x"], residual=xs, out=xs)
            h = ops.layernorm_fwd(xs, *lw["ln2"], out_dtype=dtype)
            f = _linear(h, lw["wfc1"], bias=lw["bfc1"], act=ops.ACT_GELU)
            _linear(f, lw["wfc2"], bias=lw["bfc2"], residual=xs, out=xs)
        out = ops.layernorm_fwd(xs, *pk["lnf"], out_dtype=dtype)
        return (out.view(B, T, D),)

    @torch.no_grad()
    def new_cache(self, batch, encoder_hidden_states=None, dtype=torch.bfloat16, max_tokens=None, device=None):
        """An empty decoding state for ``batch`` sequences: per-layer [B, max_tokens, 2D] key|value buffers
        (filled front to back by :meth:`decode_step`) and the encoder projections."""
        cfg = self.cfg
        n = cfg.max_target_positions if max_tokens is None else int(max_tokens)
        if n > cfg.max_target_positions:
            raise ValueError(f"max_tokens exceeds max_target_positions={cfg.max_target_positions}")
        device = device or self.embed_tokens.weight.device
        return {"len": 0, "dtype": dtype,
                "kv": [torch.empty((batch, n, 2 * cfg.d_model), dtype=dtype, device=device) for _ in self.layers],
                "cross": None if encoder_hidden_states is None else self.cross_kv(encoder_hidden_states, dtype)}

    @torch.no_grad()
    def decode_step(self, input_ids, cache):
        """Appends ``input_ids`` [B, t] (one token per call in greedy decoding, or a whole prompt) to the
        sequences in ``cache`` and returns their hidden states [B, t, D]: the same values ``forward`` gives
        for these positions of the full sequence (no padding mask: every cached token is attended)."""
        cfg = self.cfg
        dtype = cache["dtype"]
        B, T = input_ids.shape
        past = cache["len"]
        if past + T > cache["kv"][0].shape[1]:
            raise ValueError("decoding past the cache's max_tokens")
        pk = self._pack(dtype)
        H, D = cfg.decoder_attention_heads, cfg.d_model
        use_mfma = dtype == torch.bfloat16
        xs = ops.embed_tokens(input_ids, pk["tok"], pk["pos"], past=past)
        for i, lw in enumerate(pk["layers"]):
            h = ops.layernorm_fwd(xs, *lw["ln1"], out_dtype=dtype)
            qkv = _linear(h, lw["wqkv"], bias=lw["bqkv"]).view(B, T, 3 * D)
            kv = cache["kv"][i]
            for b in range(B):                                  # this step's keys | values behind the cached ones
                ops.cast_rows(qkv[b, :, D:], kv[b, past:past + T])
            seen = kv[:, :past + T]
            if B > 1 and past + T < kv.shape[1]:                # the kernel's batch stride is Tk rows: pack the filled part
                seen = seen.contiguous()
            o = ops.attn_fwd(qkv[:, :, :D], seen[:, :, :D], seen[:, :, D:], H, scale=1.0, use_mfma=use_mfma, causal=True)
            _linear(o.view(B * T, D), lw["wo"], bias=lw["bo"], residual=xs, out=xs)
            if cache["cross"] is not None:
                ckv = cache["cross"][i]
                h = ops.layernorm_fwd(xs, *lw["lnx"], out_dtype=dtype)
                q = _linear(h, lw["wq_x"], bias=lw["bq_x"]).view(B, T, D)
                o = ops.attn_fwd(q, ckv[:, :, :D], ckv[:, :, D:], H, scale=1.0, use_mfma=use_mfma)
                _linear(o.view(B * T, D), lw["wo_x"], bias=lw["bo_x"], residual=xs, out=xs)
            h = ops.layernorm_fwd(xs, *lw["ln2"], out_dtype=dtype)
            f = _linear(h, lw["wfc1"], bias=lw["bfc1"], act=ops.ACT_GELU)
            _linear(f, lw["wfc2"], bias=lw["bfc2"], residual=xs, out=xs)
        cache["len"] = past + T
        return ops.layernorm_fwd(xs, *pk["lnf"], out_dtype=dtype).view(B, T, D)

    @torch.no_grad()
    def greedy(self, prompt_ids, encoder_hidden_states, max_new_tokens, eos_token_id=None, dtype=torch.bfloat16):
        """Greedy decoding with the tied output projection: returns int64 [B, prompt + generated] (stops early
        when every sequence has produced ``eos_token_id``)."""
        B, P = prompt_ids.shape
        cache = self.new_cache(B, encoder_hidden_states, dtype, max_tokens=min(self.cfg.max_target_positions, P + max_new_tokens))
        out = [prompt_ids]
        h = self.decode_step(prompt_ids, cache)
        done = torch.zeros(B, dtype=torch.bool, device=prompt_ids.device)
        for _ in range(max_new_tokens):
            logits = self.project_tokens(h[:, -1:, :].contiguous())
            nxt = ops.argmax_rows(logits.view(B, -1)).view(B, 1)
            out.append(nxt)
            if eos_token_id is not None:
                done |= nxt.view(B) == eos_token_id
                if bool(done.all()):
                    break
            if cache["len"] >= cache["kv"][0].shape[1]:
                break
            h = self.decode_step(nxt, cache)
        return torch.cat(out, dim=1)

    @torch.no_grad()
    def project_tokens(self, hidden, out_dtype=torch.float32):
        """Vocabulary logits with the tied output projection of HF ``WhisperForConditionalGeneration``
        (``proj_out.weight`` is ``embed_tokens.weight``, no bias): [B, T, D] -> [B, T, vocab]."""
        w4 = self._w4 is not None and self._w4[1]
        key = (hidden.dtype, w4 and self._w4, self.embed_tokens.weight._version, self.embed_tokens.weight.data_ptr())
        if self._proj is None or self._proj[0] != key:
            w = self.embed_tokens.weight.detach()
            self._proj = (key, ops.w4_quantize(w, self._w4[0]) if w4 else w.to(hidden.dtype).contiguous())
        B, T, D = hidden.shape
        return _linear(hidden.reshape(B * T, D), self._proj[1], out_dtype=out_dtype).view(B, T, -1)

    # ---- 4-bit weights ------------------------------------------------------
    def quantize(self, group=64, head=False):
        """Keeps the layers' projections and MLPs (and with ``head`` the tied vocabulary projection) as 4-bit weights with a scale per
        ``group`` columns (``ops.w4_quantize``: nearest), for every call from here on; ``group=None`` goes back to full weights.  The
        parameters themselves, the encoder's key / value projections and the embeddings stay as they are."""
        if group is not None and group not in ops.W4_GROUPS:
            raise ValueError(f"group must be one of {ops.W4_GROUPS} or None")
        self._w4 = None if group is None else (group, bool(head))
        self._packed = self._proj = None
        return self

    # ---- requests of different lengths ---------------------------------------
    def new_paged_cache(self, requests, *, pages=None, page_size=64, max_tokens=None, frames=None, frame_pages=None, dtype=torch.bfloat16,
                        device=None):
        """An empty cache for ``requests`` requests of up to ``max_tokens`` tokens over ``pages`` pages (default: enough for all of them).
        ``max_tokens`` is a multiple of the page size, so that the plan keeps to it: max_target_positions at most, which is also the
        default; where that is no multiple (448 with pages of 128 or 256), it has to be given.  ``frames``: most encoder frames of a
        request, over ``frame_pages`` pages; None: no cross-attention."""
        most = self.cfg.max_target_positions
        n = most if max_tokens is None else int(max_tokens)
        if n > most or n < 1 or n % page_size:
            raise ValueError(f"max_tokens must be given as a multiple of the page size {page_size}, up to max_target_positions={most}")
        return self._paged_cache(requests, n, pages, page_size, frames, frame_pages, dtype, device)

    def _paged_cache(self, requests, n, pages, page_size, frames, frame_pages, dtype, device):
        """Without the check: a caller that keeps to max_target_positions itself may have its last page reach beyond."""
        cfg = self.cfg
        device = device or self.embed_tokens.weight.device
        H, D = cfg.decoder_attention_heads, cfg.d_model // cfg.decoder_attention_heads
        make = lambda most, count: PagedKVCache(len(self.layers), requests, H, D, max_tokens=most, page_size=page_size, dtype=dtype, device=device,
                                                pages=requests * -(-most // page_size) if count is None else count)
        return PagedDecoderCache(make(n, pages), None if frames is None else make(int(frames), frame_pages), dtype, device)

    def _own_cache(self, cache):
        """Refuses a cache that was made for another decoder, before anything of it moves on."""
        H, kv = self.cfg.decoder_attention_heads, cache.tokens.kv
        if len(kv) != len(self.layers) or tuple(kv[0].shape[2::2]) != (H, self.cfg.d_model // H):
            raise ValueError("the cache is another decoder's: its layers, heads or head size differ")
        if self.embed_tokens.weight.device != cache.bad.device:
            raise ValueError("the cache is not on the decoder's device")

    @torch.no_grad()
    def paged_admit(self, cache, requests, encoder_hidden_states):
        """Encoder output [n, Te, D] of the n given requests (ascending, none of which holds frames) into the cache's frames.  Raises
        with nothing changed on what does not fit: its width, its device, or the free pages."""
        if cache.frames is None:
            raise ValueError("the cache was made without frames")
        requests = [int(r) for r in requests]
        self._own_cache(cache)
        n, Te, D = encoder_hidden_states.shape
        if D != self.cfg.d_model or encoder_hidden_states.device != cache.bad.device or Te == 0:
            raise ValueError(f"paged_admit expects encoder output [n, frames, {self.cfg.d_model}] on the cache's device")
        if len(requests) != n or n == 0 or any(b <= a for a, b in zip(requests, requests[1:])) or requests[0] < 0 or requests[-1] >= cache.frames.requests:
            raise ValueError("paged_admit expects one ascending request index per encoder output")
        if bool((cache.frames.lens[requests] != 0).any()):
            raise ValueError("a request that holds frames has to end first (paged_end)")
        new = [0] * cache.frames.requests
        for r in requests:
            new[r] = Te
        kvs = self.cross_kv(encoder_hidden_states, cache.dtype)      # what can fail here comes before the pages are taken
        plan = cache.frames.plan(torch.tensor(new, dtype=torch.int32, device=cache.bad.device), n * Te)
        cache.frames.check(plan)
        H = self.cfg.decoder_attention_heads
        for i, kv in enumerate(kvs):
            kv = kv.view(n * Te, 2 * D)
            cache.frames.write(i, kv[:, :D].unflatten(1, (H, -1)), kv[:, D:].unflatten(1, (H, -1)), plan)

    @torch.no_grad()
    def paged_step(self, cache, input_ids, new, max_new=None):
        """One step of a server.  ``new``: tokens each request adds (0: it waits, -1: it ends and gives its tokens' pages back; its frames
        go with :meth:`paged_end`); ``input_ids`` int64 [N]: these tokens, request after request.  Returns their hidden states [N, D],
        the values :meth:`forward` gives for these positions of each request's sequence, and the step's plan.

        ``new`` as a list is checked: the call waits for the GPU, and raises, with nothing changed, on ids outside the vocabulary, on
        a step that does not fit, and (with a cache for frames) on tokens of a request that was not admitted.  As an int32 GPU tensor it
        is taken as it is, and the call can be recorded in a HIP graph (``max_new``: at most so many new tokens of one request; default
        N): ``plan.status`` and ``cache.bad`` say whether it went well; rows behind the last token hold nothing, but their ids are looked
        up too, so any of the vocabulary stands there; whether a request holds frames is the caller's to know
        (``cache.frames.lens``): without any it attends to nothing."""
        cfg, dtype, tok = self.cfg, cache.dtype, cache.tokens
        H, D, dev = cfg.decoder_attention_heads, cfg.d_model, cache.bad.device
        # all that can be wrong is looked at here: the plan below moves the cache on
        if input_ids.dim() != 1 or input_ids.dtype != torch.int64 or input_ids.device != dev:
            raise ValueError("input_ids must be int64 [tokens] on the cache's device")
        self._own_cache(cache)
        N = input_ids.shape[0]
        checked = not torch.is_tensor(new)
        if checked:
            new = [int(n) for n in new]
            if len(new) != tok.requests or sum(max(n, 0) for n in new) != N:
                raise ValueError(f"new must give each of the {tok.requests} requests its share of the {N} tokens")
            if N and bool(((input_ids < 0) | (input_ids >= cfg.vocab_size)).any()):
                raise IndexError("token id out of range for the embedding table")
            if N and cache.frames is not None and any(n > 0 and not held for n, held in zip(new, cache.frames.lens.tolist())):
                raise ValueError("a request that adds tokens holds no frames: paged_admit first")
            max_new = max(new)
            new = torch.tensor(new, dtype=torch.int32, device=dev)
        elif new.dtype != torch.int32 or new.shape != tok.lens.shape or new.device != dev or not new.is_contiguous():
            raise ValueError(f"new must be a contiguous int32 tensor of {tok.requests} values on the cache's device")
        elif max_new is not None and max_new < 1:
            raise ValueError("max_new must be positive")
        pk = self._pack(dtype)
        plan = tok.plan(new, max(N, 1))
        if checked:
            tok.check(plan)
        if N == 0:
            return torch.empty((0, D), dtype=dtype, device=dev), plan
        heads = lambda t: t.unflatten(1, (H, -1))
        xs = ops.embed_tokens_at(input_ids, pk["tok"], pk["pos"], plan.positions, bad=cache.bad)
        for i, lw in enumerate(pk["layers"]):
            h = ops.layernorm_fwd(xs, *lw["ln1"], out_dtype=dtype)
            qkv = _linear(h, lw["wqkv"], bias=lw["bqkv"])
            tok.write(i, heads(qkv[:, D:2 * D]), heads(qkv[:, 2 * D:]), plan)
            o = tok.attend(i, heads(qkv[:, :D]), plan.q_start, max_q=max_new)
            _linear(o.view(N, D), lw["wo"], bias=lw["bo"], residual=xs, out=xs)
            if cache.frames is not None:
                h = ops.layernorm_fwd(xs, *lw["lnx"], out_dtype=dtype)
                q = _linear(h, lw["wq_x"], bias=lw["bq_x"])
                o = cache.frames.attend(i, heads(q), plan.q_start, max_q=max_new, causal=False)
                _linear(o.view(N, D), lw["wo_x"], bias=lw["bo_x"], residual=xs, out=xs)
            h = ops.layernorm_fwd(xs, *lw["ln2"], out_dtype=dtype)
            f = _linear(h, lw["wfc1"], bias=lw["bfc1"], act=ops.ACT_GELU)
            _linear(f, lw["wfc2"], bias=lw["bfc2"], residual=xs, out=xs)
        return ops.layernorm_fwd(xs, *pk["lnf"], out_dtype=dtype), plan

    @torch.no_grad()
    def paged_end(self, cache, requests):
        """The given requests end: their pages, of tokens and frames, go back to the pools."""
        new = [0] * cache.tokens.requests
        for r in requests:
            if not 0 <= int(r) < len(new):
                raise ValueError(f"no request {r}")
            new[int(r)] = -1
        new = torch.tensor(new, dtype=torch.int32, device=cache.bad.device)
        for part in (cache.tokens, cache.frames):
            if part is not None:
                part.plan(new, 1)

    @torch.no_grad()
    def greedy_ragged(self, prompts, encoder_hidden_states, max_new_tokens, eos_token_id=None, dtype=torch.bfloat16, page_size=64):
        """Greedy decoding of prompts of different lengths (lists of token ids, none empty) in one ragged batch: each prompt's list with
        what was generated, up to ``max_new_tokens``, its own ``eos_token_id`` or max_target_positions cached tokens.  A request that is done
        gives its tokens' pages back in the next step."""
        R, most = len(prompts), self.cfg.max_target_positions
        out = [[int(t) for t in p] for p in prompts]
        if R == 0 or any(not 0 < len(p) <= most for p in out):
            raise ValueError(f"greedy_ragged expects prompts of 1 to max_target_positions={most} tokens")
        if max_new_tokens < 1:
            return out
        dev = encoder_hidden_states.device
        cache = self._paged_cache(R, most, None, page_size, encoder_hidden_states.shape[1], None, dtype, dev)
        self.paged_admit(cache, range(R), encoder_hidden_states)
        ids, new, left = [t for p in out for t in p], [len(p) for p in out], [max_new_tokens] * R
        while any(n > 0 for n in new):
            h, _ = self.paged_step(cache, torch.tensor(ids, dtype=torch.int64, device=dev), new)
            live = [r for r in range(R) if new[r] > 0]
            last = torch.tensor(new, device=dev).clamp_min(0).cumsum(0)[live] - 1
            nxt = ops.argmax_rows(self.project_tokens(h[last][:, None]).view(len(live), -1)).tolist()
            ids, new = [], [0] * R
            for r, t in zip(live, nxt):
                out[r].append(t)
                left[r] -= 1
                done = left[r] == 0 or t == eos_token_id or len(out[r]) > most
                new[r] = -1 if done else 1
                ids += [] if done else [t]
        return out
