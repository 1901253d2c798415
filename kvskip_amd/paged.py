"""A serving loop's KV cache in 64-token pages, kept on the device (not in the reference): the page pools of several
layers in 8 bits, one block table for all of them, and the free pages.

    cache = PagedCache(layers=32, pages=40000, Hkv=8, D=128, requests=64, tokens=32768, rows=8192, fmt="e4m3")
    cache.step(new_lens, drop=finished)          # int32 [requests]: tokens each request brings; bool [requests]: it is over
    for l in range(32):
        cache.write(l, k, v)                     # bf16 [rows, Hkv, D], request b's rows from cache.starts[b] on
        out = cache.decode(l, q, scale)["out"]   # q [requests, Hq, D]; every request's tokens, new ones included

A step whose requests bring prompts, or parts of them, attends with all of its rows instead:

    cache.step(new_lens)
    plan = cache.plan(rows, Hq)                  # rows: at least the step's new tokens; once for all layers
    for l in range(32):
        q, k = ext.norm_rope(q, k, plan.positions, inv_freq, q_weight, k_weight)   # q [rows, Hq, D], k [rows, Hkv, D]
        cache.write(l, k, v)
        out = cache.attend(l, q, scale, plan)["out"]        # [rows, Hq, D]

Prefixes that requests share (an instruction, a document) are held once, in pages of their own that no step moves:

    cache = PagedCache(..., shared=(8192,))      # the capacity of each, in tokens
    plan = cache.plan_prefix(0, n, Hq)           # its own n rows, as a prompt; per layer cache.write_prefix(l, 0, k, v), attend
    cache.shared_of.zero_()                      # int32 [requests]: the prefix that each request is behind, -1 none

Nothing synchronises: a step can be captured in a HIP graph and replayed. What is allocated after the construction comes from
torch's allocator: decode's outputs and split partials, in a step of more than 4096 rows page_map's workspace, a plan's
workspace (50 KB for 256 single tokens, 1 to 3 MB for 32768 rows), and attend's outputs and partial results: up to 137 MB at 128
dims, and in a cache with shared prefixes 8 * rows * Hq * D bytes more (1.1 GB at 32768 rows of 32 heads of 128 dims), whether
or not a request is behind one. cache.short
(int32 [1], on the device) counts the requests that the last step had no pages or rows for: their rows are not written, they
keep the tokens they had, and a caller that admits requests without counting pages reads it now and then."""

from __future__ import annotations

import torch

from . import kvskip as K

PAGE = 64
FORMATS = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


class PagedCache:
    """fmt: "e4m3" or "int8", with a power-of-two scale for each page and head, grown as rows need it (ext.cache_write).
    requests: rows of the block table; tokens: the most of one request; rows: the most new tokens of a step; shared: the
    capacity of each shared prefix, in tokens, beside `pages`. (Not over
    bf16 pages: their pass takes a request of no tokens for one of one, and would read a page that it does not hold.)"""

    def __init__(self, layers: int, pages: int, Hkv: int, D: int, requests: int, tokens: int, rows: int, fmt: str = "e4m3",
                 device="cuda", shared=()):
        if fmt not in FORMATS:
            raise ValueError(f"fmt in {sorted(FORMATS)} (got {fmt!r})")
        if not 1 <= requests <= 256:
            raise ValueError(f"requests in 1..256, a decode batch's bound (got {requests})")
        if any(n < 1 for n in shared):
            raise ValueError(f"shared: the capacity of each prefix, in tokens (got {tuple(shared)})")
        i32 = dict(dtype=torch.int32, device=device)
        first = [pages]                                # each shared prefix's first page, after those that steps move
        for n in shared:
            first.append(first[-1] + (n + PAGE - 1) // PAGE)
        self.T = (tokens + PAGE - 1) // PAGE * PAGE
        self.pools = [[torch.zeros(first[-1], Hkv, PAGE, D, dtype=FORMATS[fmt], device=device) for _ in "kv"]
                      for _ in range(layers)]
        self.scales = [[torch.zeros(first[-1], Hkv, device=device) for _ in "kv"] for _ in range(layers)]
        self.lens = torch.zeros(requests, **i32)
        self.held = torch.zeros(requests, **i32)
        self.block_table = torch.full((requests, self.T // PAGE), -1, **i32)
        self.free_pages = torch.arange(pages, **i32)
        self.free_count = torch.full((1,), pages, **i32)
        self.slot_map = torch.full((rows,), -1, **i32)
        self.starts = torch.zeros(requests + 1, **i32)
        self.short = torch.zeros(1, **i32)
        self.Hkv, self.shared = Hkv, tuple(shared)
        self.shared_table = self.shared_lens = self.shared_of = None
        if self.shared:
            self.shared_first = tuple(first[:-1])
            at = torch.arange(max(b - a for a, b in zip(first, first[1:])), **i32)
            self.shared_table = torch.stack([torch.where(at < b - a, at + a, -1) for a, b in zip(first, first[1:])]).to(torch.int32)
            self.shared_lens = torch.zeros(len(self.shared), **i32)
            self.shared_of = torch.full((requests,), -1, **i32)

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
        """kvskip.decode of one query a request [requests, Hq, D] over its own tokens; attend() is the call
        for requests behind shared prefixes. An empty request's row is zeros (lse -inf)."""
        k, v = self.pools[layer]
        ks, vs = self.scales[layer]
        return K.decode(q, k, v, scale, seq_lens=self.lens, block_table=self.block_table, T=self.T, k_scale=ks, v_scale=vs,
                        **kw)

    def plan(self, rows: int, Hq: int, max_rows: int = 0, window: int = 0, prefix_lens: torch.Tensor | None = None):
        """The plan of attend() for the last step's rows (kvskip.attend_plan), once for all layers that share a window; rows:
        those of the q that attend() will be given. Rows past the step's come back as zeros, and of a step with more only the
        first `rows` are attended; what those of a request that the
        step did not serve come back as means nothing. max_rows: the most rows that one request is expected to bring (0: all)."""
        return K.attend_plan(self.starts, self.lens, rows, self.block_table, Hq, self.Hkv, max_rows, window, prefix_lens,
                             self.shared_table, self.shared_lens, self.shared_of)

    def attend(self, layer: int, q: torch.Tensor, scale: float, plan, **kw) -> dict:
        """kvskip.attend of the plan's rows [rows, Hq, D] over their requests' tokens and the prefix that each is behind."""
        return K.attend(q, *self.pools[layer], scale, plan, *self.scales[layer], **kw)

    def plan_prefix(self, prefix: int, n: int, Hq: int, window: int = 0):
        """Shared prefix `prefix` has n tokens from now on; the plan of attend() for its own n rows, from position 0 on: all of a
        prefix in one call."""
        if not (0 <= prefix < len(self.shared) and 1 <= n <= self.shared[prefix]):
            raise ValueError(f"prefix in 0..{len(self.shared) - 1}, n in 1..its capacity (got {prefix}, {n})")
        self.shared_lens[prefix].fill_(n)
        starts = torch.arange(2, dtype=torch.int32, device=self.lens.device) * n
        return K.attend_plan(starts, starts[1:], n, self.shared_table[prefix:prefix + 1], Hq, self.Hkv, 0, window)

    def write_prefix(self, layer: int, prefix: int, k: torch.Tensor, v: torch.Tensor):
        """A layer's keys and values of a shared prefix, bf16 [n, Hkv, D], from its first token on, into its pages."""
        if not (0 <= prefix < len(self.shared) and k.shape[0] <= self.shared[prefix]):
            raise ValueError(f"prefix in 0..{len(self.shared) - 1}, rows up to its capacity (got {prefix}, {k.shape[0]})")
        at = self.shared_first[prefix] * PAGE
        slots = torch.arange(at, at + k.shape[0], dtype=torch.int32, device=self.lens.device)
        K.ext().cache_write(k, v, slots, *self.pools[layer], *self.scales[layer])
