"""Time per decoded token of the Whisper decoder: the rectangular cache, the paged cache, the paged cache replayed from a HIP graph,
and that with 4-bit weights.  Random weights; B requests after a 4-token prompt over 1500 encoder frames.

  python3 scripts/bench_serving.py [--whisper small] [--batch 8] [--tokens 64]"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from mocov2_whisper_flamingo_amd import WhisperConfig, WhisperDecoder  # noqa: E402


def timed(step, n):
    step()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(n):
        step()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) / n * 1e6


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--whisper", default="small")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--tokens", type=int, default=64)
    a = ap.parse_args()
    dev, B, n = torch.device("cuda:0"), a.batch, a.tokens
    cfg = WhisperConfig.from_name(a.whisper)
    dec = WhisperDecoder(cfg).to(dev)
    enc = torch.randn(B, 1500, cfg.d_model, device=dev)
    prompt = torch.randint(3, 1000, (B, 4), device=dev)
    one = prompt[:, :1].contiguous()
    cache = dec.new_cache(B, enc, max_tokens=n + 8)
    dec.decode_step(prompt, cache)
    print(f"{a.whisper} x {B}: rectangular cache {timed(lambda: dec.project_tokens(dec.decode_step(one, cache)), n):9.1f} us a step", flush=True)

    def paged():
        c = dec.new_paged_cache(B, frames=1500)
        dec.paged_admit(c, range(B), enc)
        dec.paged_step(c, prompt.reshape(-1), [4] * B)
        return c

    new, ids = torch.ones(B, dtype=torch.int32, device=dev), one.reshape(-1).contiguous()
    c = paged()
    print(f"{a.whisper} x {B}: paged             {timed(lambda: dec.project_tokens(dec.paged_step(c, ids, new, max_new=1)[0][None]), n):9.1f} us a step", flush=True)
    for group in (None, 64):
        dec.quantize(group, head=True)
        c = paged()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            dec.project_tokens(dec.paged_step(c, ids, new, max_new=1)[0][None])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h, plan = dec.paged_step(c, ids, new, max_new=1)
            dec.project_tokens(h[None])
        print(f"{a.whisper} x {B}: paged, recorded{', 4 bits' if group else '        '} {timed(graph.replay, n):7.1f} us a step", flush=True)
        assert plan.status.item() == 0 and c.bad.item() == 0


if __name__ == "__main__":
    main()
