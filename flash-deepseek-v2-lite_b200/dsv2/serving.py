"""What an engine that serves many requests keeps: a paged 4-bit latent cache and the requests'
low-rank adapters.

PagedCache4 holds one 4-bit cache per layer (latent4_cache in dsv2.ops), the requests' page
tables and the ring of free pages; PagePlan is one step's plan over it (a decode step of one
token per request, or a chunk of prompt tokens).  Adapters holds every layer's low-rank
adapters of the query + latent projection and of the output projection.

    cache = PagedCache4(layers=27, requests=32, max_len=4096, page_size=64, device="cuda")
    engine = DecodeEngine(model, 32, 4096, kv_format="int4")      # makes its own
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import ops


class PagedCache4:
    """Pages of the 4-bit latent cache of `layers` layers, shared by `requests` requests of up
    to max_len tokens.  pages: the pool's size (default: enough for every request at max_len)."""

    def __init__(self, layers: int, requests: int, max_len: int, page_size: int, device, pages: int | None = None):
        if page_size <= 0 or page_size % ops.L4_BLOCK_TOKENS:
            raise ValueError(f"page_size {page_size} (a positive multiple of {ops.L4_BLOCK_TOKENS})")
        self.requests, self.page_size = requests, page_size
        self.width = math.ceil(max_len / page_size)
        self.pages = requests * self.width if pages is None else int(pages)
        if self.pages <= 0:
            raise ValueError("the pool needs at least one page")
        self.cache = ops.latent4_cache(self.pages, page_size, device, layers=layers)
        # an entry that was never given names no page: a length that claims it is flagged, not served from page 0
        self.block_table = torch.full((requests, self.width), -1, device=device, dtype=torch.int32)
        self.free_ring = torch.arange(self.pages, device=device, dtype=torch.int32)
        self.ring = torch.tensor([0, self.pages], device=device, dtype=torch.int64)

    def reset(self) -> None:
        """Give every page back (all requests start over)."""
        self.free_ring.copy_(torch.arange(self.pages, device=self.free_ring.device, dtype=torch.int32))
        self.ring.copy_(torch.tensor([0, self.pages], dtype=torch.int64))
        self.block_table.fill_(-1)


class PagePlan:
    """Buffers of a step's page plan: `capacity` token rows over the cache's requests.  missed counts
    the rows that an engine's steps could not serve since clear(): they have kept their length and
    token (dsv2.ops.lm_head_argmax), also in steps replayed from a graph."""

    def __init__(self, paged: PagedCache4, capacity: int, new: torch.Tensor | None = None):
        dev = paged.block_table.device
        self.paged = paged
        self.new = torch.ones(paged.requests, device=dev, dtype=torch.int32) if new is None else new
        self.buf = ops.page_plan_buffers(paged.requests, capacity, dev)
        self.buf["ring_out"] = paged.ring           # the ring advances in place
        self.missed = torch.zeros(1, device=dev, dtype=torch.int32)

    def run(self, cached: torch.Tensor) -> None:
        """Append `new` tokens to the requests that hold `cached` ones (int32 / int64 [requests])."""
        p = self.paged
        ops.page_plan(cached=cached, new=self.new, block_table=p.block_table, free_ring=p.free_ring, ring_in=p.ring,
                      page_size=p.page_size, **self.buf)

    @property
    def slots(self) -> torch.Tensor:
        return self.buf["slots"]

    @property
    def positions(self) -> torch.Tensor:
        return self.buf["positions"]

    @property
    def token_row(self) -> torch.Tensor:
        return self.buf["token_row"]

    def check(self) -> None:
        """Raise if the last step, or an engine's step since clear(), could not serve every request
        (synchronises)."""
        n, m = int(self.buf["counts"][3]), int(self.missed)
        if n or m:
            raise RuntimeError(f"page plan: {n} request(s) got no pages in the last step, {m} token row(s) since the count "
                               f"was cleared ({self.paged.pages} pages of {self.paged.page_size} tokens)")

    def clear(self) -> None:
        """Forget the steps that could not serve every request."""
        self.missed.zero_()
        self.buf["counts"].zero_()


@dataclass
class LayerAdapters:
    qkva_a: torch.Tensor   # [adapters, rank, 2048] bf16
    qkva_b: torch.Tensor   # [adapters, 3648, rank]
    o_a: torch.Tensor      # [adapters, rank, 2048]
    o_b: torch.Tensor      # [adapters, 2048, rank]


@dataclass
class Adapters:
    """Low-rank adapters of every layer's query + latent projection and output projection:
    y = W x + scales[i] * B_i (A_i x).  ids: the adapter of every request (-1: none), on the
    device, changed in place between steps."""
    layers: list[LayerAdapters]
    ranks: torch.Tensor    # [adapters] int32
    scales: torch.Tensor   # [adapters] fp32
    ids: torch.Tensor      # [requests] int32

    @property
    def rank(self) -> int:
        return int(self.layers[0].qkva_a.shape[1])


def random_adapters(n_layers: int, n_adapters: int, rank: int, requests: int, device, seed: int = 0,
                    std: float = 0.02) -> Adapters:
    """Seeded adapters for benchmarks and tests (A ~ N(0, 1 / k), B ~ N(0, std^2)); request r has
    adapter r % (n_adapters + 1) - 1, so every so many requests have none."""
    g = torch.Generator(device=device).manual_seed(seed)

    def bf(*shape, s):
        return (torch.randn(*shape, generator=g, device=device) * s).to(torch.bfloat16)
    layers = [LayerAdapters(qkva_a=bf(n_adapters, rank, 2048, s=2048 ** -0.5), qkva_b=bf(n_adapters, 3648, rank, s=std),
                            o_a=bf(n_adapters, rank, 2048, s=2048 ** -0.5), o_b=bf(n_adapters, 2048, rank, s=std))
              for _ in range(n_layers)]
    return Adapters(layers=layers, ranks=torch.full((n_adapters,), rank, device=device, dtype=torch.int32),
                    scales=torch.ones(n_adapters, device=device),
                    ids=(torch.arange(requests, device=device) % (n_adapters + 1) - 1).to(torch.int32))
