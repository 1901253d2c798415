"""A serving loop's KV cache in 64-token pages, kept on the device (not in the reference): the page pools of several
layers in 8 bits, one block table for all of them, and the free pages.

    cache = PagedCache(layers=32, pages=40000, Hkv=8, D=128, requests=64, tokens=32768, rows=8192, fmt="e4m3")
    cache.step(new_lens, drop=finished)          # int32 [requests]: tokens each request brings; bool [requests]: it is over
    for l in range(32):
        cache.write(l, k, v)                     # bf16 [rows, Hkv, D], request b's rows from cache.starts[b] on
        out = cache.decode(l, q, scale)["out"]   # q [requests, Hq, D]; every request's tokens, new ones included

Nothing synchronises: a step can be captured in a HIP graph and replayed. What is allocated after the construction comes from
torch's allocator: decode's outputs and split partials, and in a step of more than 4096 rows page_map's workspace. cache.short
(int32 [1], on the device) counts the requests that the last step had no pages or rows for: their rows are not written, they
keep the tokens they had, and a caller that admits requests without counting pages reads it now and then."""

from __future__ import annotations

import torch

from . import kvskip as K

PAGE = 64
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class PagedCache:
    """fmt: "e4m3" or "int8", with a power-of-two scale for each page and head, grown as rows need it (ext.cache_write).
    requests: rows of the block table; tokens: the most of one request; rows: the most new tokens of a step. (Not over
    bf16 pages: their pass takes a request of no tokens for one of one, and would read a page that it does not hold.)"""

    def __init__(self, layers: int, pages: int, Hkv: int, D: int, requests: int, tokens: int, rows: int, fmt: str = "e4m3",
                 device="cuda"):
        if fmt not in FORMATS:
            raise ValueError(f"fmt in {sorted(FORMATS)} (got {fmt!r})")
        if not 1 <= requests <= 256:
            raise ValueError(f"requests in 1..256, a decode batch's bound (got {requests})")
        i32 = dict(dtype=torch.int32, device=device)
        self.T = (tokens + PAGE - 1) // PAGE * PAGE
        self.pools = [[torch.zeros(pages, Hkv, PAGE, D, dtype=FORMATS[fmt], device=device) for _ in "kv"]
                      for _ in range(layers)]
        self.scales = [[torch.zeros(pages, Hkv, device=device) for _ in "kv"] for _ in range(layers)]
        self.lens = torch.zeros(requests, **i32)
        self.held = torch.zeros(requests, **i32)
        self.block_table = torch.full((requests, self.T // PAGE), -1, **i32)
        self.free_pages = torch.arange(pages, **i32)
        self.free_count = torch.full((1,), pages, **i32)
        self.slot_map = torch.full((rows,), -1, **i32)
        self.starts = torch.zeros(requests + 1, **i32)
        self.short = torch.zeros(1, **i32)

    def step(self, new_lens: torch.Tensor, drop: torch.Tensor | None = None):
        """Makes room for the step's new tokens (int32 [requests]; a negative number takes a request's last tokens off, down to
        none); a request whose rows pass the map's `rows`, or for which there are no pages, gets none, keeps the tokens it
        had and counts in `short`. The requests that drop marks (bool [requests]) end first, and give
        their pages back, but for those that the place's next request fills at once. Updates lens, block_table, slot_map
        and starts."""
        for t, ty in ((new_lens, torch.int32), (drop, torch.bool)):
            if t is not None and (t.dtype != ty or t.shape != self.lens.shape or not t.is_contiguous() or not t.is_cuda
                                  or t.device != self.lens.device):
                raise RuntimeError("step: new_lens int32 [requests], drop bool [requests], contiguous on the cache's device")
        if drop is not None:
            self.lens.masked_fill_(drop, 0)
        self.lens.add_(new_lens)
        K.ext().page_map(self.lens, new_lens, self.held, self.block_table, self.free_pages, self.free_count, self.slot_map,
                         self.starts, self.short, lens_out=self.lens)

    def write(self, layer: int, k: torch.Tensor, v: torch.Tensor):
        """The step's keys and values of a layer, bf16 [n, Hkv, D] with n rows, at most the map's (rows past starts' last are
        left out), into their pages."""
        K.ext().cache_write(k, v, self.slot_map[:k.shape[0]], *self.pools[layer], *self.scales[layer])

    def decode(self, layer: int, q: torch.Tensor, scale: float, **kw) -> dict:
        """kvskip.decode of one query a request [requests, Hq, D] over its tokens. An empty request's row is
        zeros (lse -inf)."""
        k, v = self.pools[layer]
        ks, vs = self.scales[layer]
        return K.decode(q, k, v, scale, seq_lens=self.lens, block_table=self.block_table, T=self.T, k_scale=ks, v_scale=vs,
                        **kw)
