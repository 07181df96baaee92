"""A small decoder on the quantized linears and the paged cache: how the pieces of ``paged`` run together.

Random weights, pre-norm blocks (RMSNorm, rotary attention whose query heads share key/value heads, GELU MLP), greedy
answers. Every linear comes from ``flux_dit.linear_factory``, so the same model runs W4A4 or bf16. Prompts of any
lengths go in together, in chunks; then every step takes one token of each sequence. With a ``budget`` each layer's keys
are cut back to the most attended whenever a sequence has outgrown it by a page:

    python -m gen_worker_amd.decoder --kind w4a4 --prompts 300,17,120 --tokens 64 --budget 128
"""

from __future__ import annotations

import argparse
import time
from dataclasses import dataclass
from typing import Optional, Sequence

import torch
from torch import Tensor, nn

from .flux_dit import _rms, linear_factory
from .paged import PagedBatch, PagedCache, PagedError, rotary_table


@dataclass
class DecoderConfig:
    vocab: int = 2048
    layers: int = 4
    hidden: int = 1024
    heads: int = 16
    kv_heads: int = 4
    head_dim: int = 64
    mlp: int = 4096
    rot: int = 64            # rotated channels of a head
    interleaved: bool = False
    positions: int = 8192    # of the rotary tables
    scaling: str = "none"    # of the tables, for longer contexts (``paged.rotary_table``)
    factor: float = 1.0
    original: int = 0


class DecoderBlock(nn.Module):
    def __init__(self, cfg: DecoderConfig, make, seed: int, device) -> None:
        super().__init__()
        self.cfg = cfg
        width = (cfg.heads + 2 * cfg.kv_heads) * cfg.head_dim
        self.qkv = make(cfg.hidden, width, seed)
        self.out = make(cfg.heads * cfg.head_dim, cfg.hidden, seed + 1)
        self.fc1, self.fc2 = make(cfg.hidden, cfg.mlp, seed + 2, gelu=True), make(cfg.mlp, cfg.hidden, seed + 3)
        for name in ("norm1", "norm2"):
            self.register_buffer(name, torch.ones(cfg.hidden, device=device, dtype=torch.bfloat16))

    def heads_of(self, x: Tensor) -> tuple[Tensor, Tensor, Tensor]:
        """Queries, keys and values of normed rows: column slices of the fused projection."""
        cfg = self.cfg
        y = self.qkv(_rms(x, self.norm1)).view(x.shape[0], -1, cfg.head_dim)
        return y[:, :cfg.heads], y[:, cfg.heads:cfg.heads + cfg.kv_heads], y[:, cfg.heads + cfg.kv_heads:]

    def rest(self, x: Tensor, attended: Tensor) -> Tensor:
        x = x + self.out(attended.reshape(x.shape[0], -1))
        return x + self.fc2(self.fc1(_rms(x, self.norm2)))

    def forward(self, x: Tensor, batch: PagedBatch, cache: PagedCache, cos: Tensor, sin: Tensor) -> Tensor:
        q, k, v = self.heads_of(x)
        q = cache.write(batch, q, k, v, cos, sin, interleaved=self.cfg.interleaved)
        return self.rest(x, cache.attend(batch, q)[0])


class PagedDecoder(nn.Module):
    def __init__(self, cfg: DecoderConfig, kind: str = "w4a4", device="cuda", seed: int = 0, rank: int = 32) -> None:
        super().__init__()
        self.cfg = cfg
        make = linear_factory(kind, device, rank)
        self.blocks = nn.ModuleList(DecoderBlock(cfg, make, seed + 16 * i, device) for i in range(cfg.layers))
        g = torch.Generator(device=device).manual_seed(seed + 7)
        self.register_buffer("embed", torch.randn(cfg.vocab, cfg.hidden, generator=g, device=device).to(torch.bfloat16))
        self.register_buffer("norm", torch.ones(cfg.hidden, device=device, dtype=torch.bfloat16))
        cos, sin = rotary_table(cfg.positions, cfg.rot, scaling=cfg.scaling, factor=cfg.factor, original=cfg.original,
                                device=device)
        self.register_buffer("cos", cos)
        self.register_buffer("sin", sin)

    def caches(self, pages: int, page_size: int = 16, weights: bool = False) -> list[PagedCache]:
        """A pool for each layer under one bookkeeping (the first's)."""
        first = PagedCache(pages, page_size, self.cfg.kv_heads, self.cfg.head_dim, device=self.embed.device,
                           weights=weights)
        return [first] + [first.twin() for _ in range(self.cfg.layers - 1)]

    @torch.no_grad()
    def forward(self, tokens: Tensor, batch: PagedBatch, caches: list[PagedCache]) -> Tensor:
        """Logits [sequences, vocab] after each sequence's last new token (each has one at least); ``tokens``: the
        batch's, packed."""
        x = self.embed[tokens]
        for block, cache in zip(self.blocks, caches):
            x = block(x, batch, cache, self.cos, self.sin)
        last = x[batch.q_start[1:].long() - 1]
        return (_rms(last, self.norm) @ self.embed.t()).float()

    @torch.no_grad()
    def generate(self, prompts: Sequence[Sequence[int]], new_tokens: int, *, budget: Optional[int] = None,
                 recent: int = 16, chunk: int = 512, page_size: int = 16) -> list[list[int]]:
        """Greedy answers of ``new_tokens`` tokens to each prompt, all in one batch. ``budget``: keys a layer keeps of a
        sequence, the last ``recent`` among them."""
        if not prompts or not all(len(p) for p in prompts) or new_tokens < 1:
            raise PagedError("generate: every prompt needs a token, and the answer one")
        if max(len(p) for p in prompts) + new_tokens > self.cfg.positions:
            raise PagedError(f"generate: more than {self.cfg.positions} positions")
        held = [len(p) + new_tokens for p in prompts]
        if budget is not None:
            held = [min(n, budget + page_size + max(chunk, 1)) for n in held]
        pages = sum(-(-n // page_size) + 1 for n in held) + (len(prompts) * -(-(budget or 0) // page_size))
        caches = self.caches(pages, page_size, weights=budget is not None)
        first, dev = caches[0], self.embed.device
        seqs = [first.add() for _ in prompts]
        logits = torch.empty(len(prompts), self.cfg.vocab, device=dev)
        done = 0
        while done < max(len(p) for p in prompts):
            part = [list(p[done:done + chunk]) for p in prompts]
            here = [i for i, p in enumerate(part) if p]
            batch = first.extend([seqs[i] for i in here], [len(part[i]) for i in here])
            packed = torch.tensor([t for i in here for t in part[i]], device=dev)
            logits[torch.tensor(here, device=dev)] = self(packed, batch, caches)
            self._cut(first, seqs, budget, recent, page_size)
            done += chunk
        answer = [logits.argmax(-1)]
        for _ in range(new_tokens - 1):
            batch = first.extend(seqs, [1] * len(seqs))
            answer.append(self(answer[-1], batch, caches).argmax(-1))
            self._cut(first, seqs, budget, recent, page_size)
        return torch.stack(answer, 1).tolist()

    @staticmethod
    def _cut(first: PagedCache, seqs: list[int], budget: Optional[int], recent: int, page_size: int) -> None:
        if budget is not None:
            long = [s for s in seqs if first.length(s) > budget + page_size]
            if long:
                first.evict(long, budget, min(recent, budget))


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--kind", choices=("w4a4", "bf16"), default="w4a4")
    ap.add_argument("--prompts", default="300,17,120", help="prompt lengths")
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--budget", type=int, default=None, help="keys a layer keeps of a sequence")
    ap.add_argument("--layers", type=int, default=4)
    a = ap.parse_args()
    model = PagedDecoder(DecoderConfig(layers=a.layers), a.kind)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, model.cfg.vocab, (int(n),), generator=g).tolist() for n in a.prompts.split(",")]
    for run in ("warm-up", "timed"):
        torch.cuda.synchronize()
        t = time.perf_counter()
        answers = model.generate(prompts, a.tokens, budget=a.budget)
        torch.cuda.synchronize()
        t = time.perf_counter() - t
    for p, x in zip(prompts, answers):
        print(f"{len(p)} tokens -> {x[:12]}{' ...' if len(x) > 12 else ''}")
    print(f"{len(prompts)} sequences x {a.tokens} tokens in {1e3 * t:.1f} ms ({1e3 * t / a.tokens:.2f} ms a step)")


if __name__ == "__main__":
    main()
