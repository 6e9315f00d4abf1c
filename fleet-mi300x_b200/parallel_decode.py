"""Parallel samples of one prompt on an 8-bit cache: the 8-bit rows, the windowed step and the page
operations together, as a server uses them.

    python -m fleet-mi300x_b200.parallel_decode [--layers 27] [--prompt 4000] [--samples 8]
                                                [--steps 64] [--window 0] [--sinks 0] [--bits 8]

(from the repository root, on a GPU). For a stack of attention layers with random weights:

  1. the prompt's raw kv_a rows go into request 0's pages of every layer (rows_to_pages);
  2. the other samples become copies of request 0 (PagePool.fork): shared full pages;
  3. every step reserves a page where a sample needs one, then replays one CUDA graph of all
     layers' attention blocks (LayerStackGraph, mode "block"), which appends and attends;
  4. half the samples end early (release), the pool is compacted, and a second graph, over the first
     entries of the block table and the row counts, decodes the others to the end: a released request has
     no page to store a row in, so a graph that steps it would report that.

It prints the time per step, the pages held at the end and what the samples that are left would hold
without sharing.
"""
from __future__ import annotations

import argparse
import json

import torch

from .attention import MlaDecodeAttention, device_rope_tables
from .cache import PagedLatentCache, PagedLatentCache8
from .config import ModelConfig
from .graph import LayerStackGraph
from .handoff import rows_to_pages
from .native import PAGE_SIZE
from .pool import PagePool
from .workloads import make_layer_weights


def run(layers: int = 27, prompt: int = 4000, samples: int = 8, steps: int = 64, window: int = 0, sinks: int = 0,
        bits: int = 8, device: str = "cuda") -> dict:
    """One run; returns what main() prints, and the final hidden states ("h")."""
    cfg, dev = ModelConfig(), torch.device(device)
    blocks = -(-(prompt + steps) // PAGE_SIZE)
    n_pages = blocks + samples * (steps // PAGE_SIZE + 3)
    cos, sin = device_rope_tables(cfg, prompt + steps + 1, dev)
    table = torch.zeros(samples, blocks, dtype=torch.int32, device=dev)
    lens = torch.zeros(samples, dtype=torch.int32, device=dev)
    caches, runners = [], []
    for layer in range(layers):
        if bits == 8:
            own = PagedLatentCache8(n_pages, samples, blocks, device=dev)
            caches.append(PagedLatentCache8.from_tensors(own.pages, own.scales, table, lens))
        else:
            own = PagedLatentCache(n_pages, samples, blocks, device=dev)
            caches.append(PagedLatentCache.from_tensors(own.pages, table, lens))
        runners.append(MlaDecodeAttention(cfg, make_layer_weights(layer, device=dev), cos, sin, window=window, sinks=sinks))
    pool = PagePool(caches)

    # the prompt, in request 0
    lens[0] = prompt
    pool.reserve(0, [0])
    g = torch.Generator(device=dev).manual_seed(1)
    starts = [0] + [prompt] * samples
    for cache, runner in zip(caches, runners):
        kv_a = torch.randn(prompt, cfg.kv_lora_rank + cfg.qk_rope, generator=g, device=dev).to(torch.bfloat16)
        rows_to_pages(cache, kv_a, starts, raw=True, norm_w=runner.norm_w, cos=cos, sin=sin)
    pool.fork([0] * (samples - 1), range(1, samples))

    live = samples if samples == 1 else samples // 2  # that decode to the end
    pool.reserve(1)
    h0 = torch.randn(samples, cfg.hidden, generator=g, device=dev).to(torch.bfloat16)
    norms = [torch.ones(cfg.hidden, dtype=torch.bfloat16, device=dev)] * layers
    kw = dict(mode="block", in_norms=norms, advance=True)
    stack = LayerStackGraph(runners, caches, h=h0, **kw)
    some = [PagedLatentCache8.from_tensors(c.pages, c.scales, table[:live], lens[:live]) if bits == 8 else
            PagedLatentCache.from_tensors(c.pages, table[:live], lens[:live]) for c in caches]
    rest = stack if live == samples else LayerStackGraph(runners, some, h=h0[:live], **kw)
    decoding, left = None, torch.arange(live, dtype=torch.int32, device=dev)  # None: every request
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    for step in range(steps):
        if step == steps // 2 and live < samples:
            pool.release(range(live, samples))
            pool.compact()
            stack, decoding = rest, left
        pool.reserve(1, decoding)
        stack.replay()
    end.record()
    stack.synchronize()
    pool.raise_pending()
    return {
        "layers": layers, "prompt": prompt, "samples": samples, "steps": steps, "window": window, "sinks": sinks,
        "bits": bits, "us_per_step": begin.elapsed_time(end) * 1e3 / steps, "pages_held": n_pages - pool.free_pages(),
        "pages_unshared": live * blocks, "page_bytes": caches[0].pages[0].numel() * caches[0].pages.element_size(),
        "rows": lens.tolist(), "h": stack.h,
    }


def main(argv: list[str] | None = None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("layers", 27), ("prompt", 4000), ("samples", 8), ("steps", 64), ("window", 0), ("sinks", 0),
                        ("bits", 8)):
        ap.add_argument(f"--{name}", type=int, default=value)
    got = run(**vars(ap.parse_args(argv)))
    got.pop("h")
    print(json.dumps(got))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
