"""The work of a serving loop that keeps its KV cache in 64-token pages of 8 bits, as cases that can be timed and checked.

A case names an operator, its sizes and its types:

  pages   a step's block tables and slot map from the requests' lengths (ext.page_map): finished requests give their
          pages back, running and admitted ones take theirs from the free list
  write   a step's new keys and values into the pages that the slot map names (ext.cache_write), into e4m3 or int8
          pages with a scale for each page and head, or into bf16 pages
  decode  one layer's decode attention over a cache held in e4m3 or int8 with a scale for each block and head
          (kvskip.decode with k_scale, v_scale): contiguous or paged, one length or many, every block or lists of them

Head shapes are those that the framework's configurations and kernels have (32 / 8 heads of 64 or 128 dims, 28 / 4, and
the other group sizes that are taken). Contexts run from a short prompt to 128k tokens, batches from one request to some
hundreds.
"""

import math

import torch

BLOCK = 64
QMAX = {"e4m3": 448.0, "int8": 127.0}
MOST_TOKENS = 32 * 8 * 65536          # tokens x KV heads of the largest listed decode, of 128 dims
MOST_ROWS = 131072                    # new rows of the largest listed step
HEADS = [(32, 8, 64), (32, 8, 128), (32, 8, 128), (28, 4, 128), (16, 8, 128), (8, 8, 128), (64, 8, 128), (16, 2, 64),
         (32, 2, 128)]

own = False


def listed():
    return [
        # a decode step of a small batch: one new token a request, now and then a new page
        dict(name="pages_decode", kind="pages", B=24, T=9001, chunk=1, admit=0.0, finish=0.05, tight=False),
        # a busy server's step: some requests end, some come in with prompts, the others decode
        dict(name="pages_mixed", kind="pages", B=257, T=32000, chunk=2048, admit=0.1, finish=0.1, tight=False),
        # the largest: a batch of long prompts taken in at once, and not enough pages for all of them
        dict(name="pages_prefill", kind="pages", B=64, T=4096, chunk=4096, admit=1.0, finish=0.0, tight=True),
        # the new token of each request of a batch, keys and values as slices of the fused projection's output
        dict(name="write_decode", kind="write", fmt="e4m3", B=64, Hq=32, Hkv=8, D=128, T=9001, prompt=False, fused=True),
        # prompts of a batch, odd lengths, 64-dim heads
        dict(name="write_int8", kind="write", fmt="int8", B=7, Hq=32, Hkv=8, D=64, T=2111, prompt=True, fused=False),
        # long prompts
        dict(name="write_prompts", kind="write", fmt="e4m3", B=8, Hq=32, Hkv=8, D=128, T=8192, prompt=True, fused=True),
        # the smallest decode: the first answers of a chat on a small model
        dict(name="decode_short", kind="decode", fmt="e4m3", B=1, Hq=32, Hkv=8, D=64, T=200, paged=False, ragged=False,
             frac=1.0, stats=False),
        # one request at 32k: the shape that the framework's benchmark is quoted on
        dict(name="decode_32k", kind="decode", fmt="e4m3", B=1, Hq=32, Hkv=8, D=128, T=32768, paged=False, ragged=False,
             frac=1.0, stats=False),
        # the same with 35% of the blocks listed and the statistics that a planner reads, in int8
        dict(name="decode_lists", kind="decode", fmt="int8", B=1, Hq=32, Hkv=8, D=128, T=32768, paged=False, ragged=False,
             frac=0.35, stats=True),
        # a serving batch of requests of very different lengths over pages, 7 query heads per KV head
        dict(name="decode_pages_g7", kind="decode", fmt="int8", B=16, Hq=28, Hkv=4, D=128, T=32000, paged=True,
             ragged=True, frac=1.0, stats=False),
        # the same over 64-dim heads in e4m3, odd lengths
        dict(name="decode_pages_d64", kind="decode", fmt="e4m3", B=24, Hq=32, Hkv=8, D=64, T=20011, paged=True,
             ragged=True, frac=1.0, stats=False),
        # the largest: a full batch at 64k
        dict(name="decode_large", kind="decode", fmt="e4m3", B=32, Hq=32, Hkv=8, D=128, T=65536, paged=False,
             ragged=False, frac=1.0, stats=False),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "decode", "write", "write", "pages"])
    if kind == "pages":
        c = dict(kind=kind, B=_spread(rng, 1, 512), T=_spread(rng, 64, 131072),
                 chunk=rng.choice([1, 1, _spread(rng, 2, 4096)]), admit=rng.choice([0.0, 0.1, 1.0]),
                 finish=rng.choice([0.0, 0.1]), tight=rng.random() < 0.25)
        while sum(_step(c)[1]) > MOST_ROWS:
            c["chunk"] = max(1, c["chunk"] // 2)
        return c
    Hq, Hkv, D = rng.choice(HEADS)
    c = dict(kind=kind, fmt=rng.choice(["e4m3", "int8"]), Hq=Hq, Hkv=Hkv, D=D)
    if kind == "write":
        c.update(prompt=rng.random() < 0.6, fused=rng.random() < 0.5, B=_spread(rng, 1, 256), T=_spread(rng, 16, 16384))
        if rng.random() < 0.2:
            c["fmt"] = "bf16"
        while c["prompt"] and c["B"] * c["T"] * Hkv * D > 8 * 8192 * 8 * 128 or c["B"] * c["T"] > MOST_ROWS * 8:
            if c["B"] > 1:
                c["B"] -= max(1, c["B"] // 4)
            else:
                c["T"] = c["T"] * 3 // 4
        return c
    c.update(B=_spread(rng, 1, 64), T=_spread(rng, 64, 131072), paged=rng.random() < 0.5, ragged=rng.random() < 0.5,
             frac=rng.choice([1.0, 1.0, round(rng.uniform(0.1, 0.6), 2)]), stats=rng.random() < 0.3)
    while c["B"] * c["T"] * Hkv > MOST_TOKENS or c["B"] * c["T"] > 32 * 65536:
        if c["B"] > 1:
            c["B"] -= max(1, c["B"] // 4)
        else:
            c["T"] = c["T"] * 3 // 4
    return c


# ---------------------------------------------------------------- lengths (a case's own, whatever the seed)

def _host(c):
    return torch.Generator().manual_seed(1000003 * c["B"] + c["T"])


def _pages_of(n):
    return (n + BLOCK - 1) // BLOCK


def _step(c):
    """A step's requests: lengths after it, new tokens and pages held before it, as lists. A finished request has length
    0 and still holds its pages; an admitted one holds none and brings a prompt of up to `chunk` tokens; the others take
    up to `chunk` tokens when every request is admitted, else one."""
    g = _host(c)
    u = torch.rand(c["B"], 3, generator=g, dtype=torch.float64).tolist()
    lens, new, held = [], [], []
    for role, x, y in u:
        n = max(1, int(round(c["T"] ** (0.6 + 0.4 * x))))
        if role < c["finish"]:
            lens.append(0), new.append(0), held.append(_pages_of(n))
        elif role < c["finish"] + c["admit"]:
            a = max(1, min(c["T"], int(c["chunk"] * (0.25 + 0.75 * y))))
            lens.append(a), new.append(a), held.append(0)
        else:
            lens.append(n), new.append(1), held.append(_pages_of(n - 1))
    return lens, new, held


def _lengths(c):
    """Lengths of a decode batch: T, or log-uniform in [T / 16, T] with one of them T."""
    if not c["ragged"]:
        return [c["T"]] * c["B"]
    g = _host(c)
    x = torch.rand(c["B"], generator=g, dtype=torch.float64).tolist()
    n = [max(1, int(round(c["T"] * 16.0 ** -y))) for y in x]
    n[int(torch.randint(0, c["B"], (1,), generator=g))] = c["T"]
    return n


def _rows(c):
    """A write's requests: (first position, new rows) each: a prompt from position 0, or one token at a later one."""
    x = torch.rand(c["B"], generator=_host(c), dtype=torch.float64).tolist()
    if c["prompt"]:
        return [(0, max(1, int(c["T"] * (0.5 + 0.5 * y)))) for y in x]
    return [(int(c["T"] * y), 1) for y in x]


# ---------------------------------------------------------------- inputs

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _values(g, *shape):
    """Keys or values: N(0, 1), one channel in sixteen four times as large, each block (the axis before the last two) by
    a factor of its own, as activations have them."""
    x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
    x *= torch.where(torch.arange(shape[-1], device="cuda") % 16 == 5, 4.0, 1.0)
    if len(shape) > 2:
        x *= torch.exp2(torch.rand(*shape[:-2], 1, 1, generator=g, device="cuda") * 2 - 1)
    return x.to(torch.bfloat16).float()


def _pow2(amax, qmax):
    """The smallest power of two s with amax <= qmax s (0 for 0)."""
    m, e = torch.frexp(amax.double() / qmax)
    s = torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e).clamp(min=-126))
    return torch.where(amax > 0, s, torch.zeros_like(s)).float()


def _codes(x, scale, fmt):
    """x / scale in the cache's type (0 where the scale is 0)."""
    y = torch.where(scale > 0, x / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(x))
    if fmt == "int8":
        return y.round().clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn)


def _cache(g, lead, D, fmt, most=2 ** 25):
    """A cache of blocks [*lead, BLOCK, D] in 8 bits and its scales [*lead], made in pieces. e4m3: a power of two a block,
    as the framework writes them; int8: amax / 127, as a program that brings its own scales has them."""
    n = math.prod(lead)
    codes = torch.empty(n, BLOCK, D, dtype=torch.int8 if fmt == "int8" else torch.float8_e4m3fn, device="cuda")
    scales = torch.empty(n, dtype=torch.float32, device="cuda")
    step = max(1, most // (BLOCK * D))
    for i in range(0, n, step):
        x = _values(g, min(step, n - i), BLOCK, D)
        amax = x.abs().amax((-1, -2))
        s = _pow2(amax, QMAX[fmt]) if fmt == "e4m3" else amax / 127.0
        codes[i:i + step] = _codes(x, s[:, None, None], fmt)
        scales[i:i + step] = s
    return codes.view(*lead, BLOCK, D), scales.view(*lead)


def _tables(c, lens, seed, extra=16):
    """Random pages for the lengths: the block table [B, pages of T] (0 past a sequence's end) and the page count."""
    need = [_pages_of(n) for n in lens]
    total = sum(need) + extra
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.zeros(c["B"], max(1, _pages_of(c["T"] + 1)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, total


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(case=c)
    i32 = dict(dtype=torch.int32, device="cuda")
    if c["kind"] == "pages":
        lens, new, held = _step(c)
        width = _pages_of(c["T"]) + 1
        need = sum(max(0, _pages_of(n) - h) for n, h in zip(lens, held))
        free = max(1, need * 3 // 4 if c["tight"] else need + 16)
        total = sum(held) + free
        order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        table = torch.full((c["B"], width), -1, dtype=torch.int32)
        at = 0
        for b, h in enumerate(held):
            table[b, :h] = order[at:at + h]
            at += h
        pool = torch.full((total,), -1, dtype=torch.int32)
        pool[:free] = order[at:]
        rows = _pages_of(max(1, sum(new))) * BLOCK            # the step's rows are padded to whole blocks
        s.update(lens=torch.tensor(lens, **i32), new=torch.tensor(new, **i32), held=torch.tensor(held, **i32),
                 table=table.cuda(), free=pool.cuda(), count=torch.tensor([free], **i32),
                 slots=torch.empty(rows, **i32), held_out=torch.empty(c["B"], **i32), count_out=torch.empty(1, **i32))
        return s
    if c["kind"] == "write":
        Hq, Hkv, D, fmt = c["Hq"], c["Hkv"], c["D"], c["fmt"]
        rows = _rows(c)
        table, total = _tables(c, [p + n for p, n in rows], seed)
        slots = torch.cat([table[b, torch.arange(p, p + n) // BLOCK] * BLOCK + torch.arange(p, p + n) % BLOCK
                           for b, (p, n) in enumerate(rows)]).to(torch.int32)
        N = slots.numel()
        if c["fused"]:
            qkv = _values(g, N, Hq + 2 * Hkv, D).to(torch.bfloat16)
            s["k"], s["v"] = qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
        else:
            s["k"], s["v"] = _values(g, N, Hkv, D).to(torch.bfloat16), _values(g, N, Hkv, D).to(torch.bfloat16)
        s["slots"] = slots.cuda()
        for x in ("k", "v"):
            if fmt == "bf16":
                s[x + "_pool"] = _values(g, total, Hkv, BLOCK, D).to(torch.bfloat16)
                s[x + "_scale"] = None
                continue
            # what the pages hold before: the rows below each request's position, with the scale that those asked for
            old = _values(g, total, Hkv, BLOCK, D)
            fill = torch.zeros(total, dtype=torch.long)
            for b, (p, _) in enumerate(rows):
                fill[table[b, :p // BLOCK].long()] = BLOCK
                fill[table[b, p // BLOCK].long()] = p % BLOCK
            old *= (torch.arange(BLOCK) < fill[:, None]).cuda()[:, None, :, None]
            s[x + "_scale"] = _pow2(old.abs().amax((-1, -2)), QMAX[fmt])
            s[x + "_pool"] = _codes(old, s[x + "_scale"][..., None, None], fmt)
        return s
    B, Hq, Hkv, D, T, fmt = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"], c["fmt"]
    lens = _lengths(c)
    s["scale"] = 1.0 / math.sqrt(D)
    s["host_lens"] = lens
    s["lens"] = torch.tensor(lens, **i32) if c["ragged"] else None
    s["q"] = torch.randn(B, Hq, D, generator=g, device="cuda").to(torch.bfloat16)
    nb = _pages_of(T)
    if c["paged"]:
        table, total = _tables(c, lens, seed)
        s["table"] = table[:, :nb].contiguous().cuda()
        for x in ("k", "v"):
            s[x], s[x + "_scale"] = _cache(g, (total, Hkv), D, fmt)
    else:
        cap = nb + 8                                           # the blocks of a growing cache's buffer
        for x in ("k", "v"):
            codes, s[x + "_scale"] = _cache(g, (B, Hkv, cap), D, fmt)
            s[x] = codes.view(B, Hkv, cap * BLOCK, D)[:, :, :T]
    if c["frac"] < 1.0:
        keep = torch.rand(B, Hkv, nb, generator=g, device="cuda") < c["frac"]
        keep[..., 0] = True
        for b, n in enumerate(lens):                           # the newest two; none past the sequence's end
            keep[b, :, max(0, _pages_of(n) - 2):] = True
            keep[b, :, _pages_of(n):] = False
        s["keep"] = keep
        if own:
            from kvskip_amd import kvskip as K

            s["plan"] = K.make_plan(keep)
    return s


# ---------------------------------------------------------------- the operators in elementary torch operations

def _plain_pages(s):
    lens, new, held, table, free = (s[x].long() for x in ("lens", "new", "held", "table", "free"))
    width, rows = table.shape[1], s["slots"].numel()
    n = lens.clamp(min=0)
    a = torch.minimum(new.clamp(min=0), n)
    fits = n <= width * BLOCK
    need = torch.where(fits, (n + BLOCK - 1) // BLOCK, held)
    give, take = (held - need).clamp(min=0), (need - held).clamp(min=0)
    col = torch.arange(width, device=n.device)[None]
    out = (col >= need[:, None]) & (col < held[:, None])       # pages given back, request by request
    at = s["count"].long() + torch.cumsum(out.flatten().long(), 0).view_as(out) - 1
    stack = torch.cat([free, free.new_zeros(1)])
    stack[torch.where(out, at, torch.full_like(at, free.numel()))] = table
    stack = stack[:-1]
    avail = s["count"].long() + give.sum()
    before = torch.cumsum(take, 0) - take
    served = fits & ((take == 0) | (before + take <= avail))
    held_out = torch.where(served, need, held)
    fresh = (col >= held[:, None]) & (col < held_out[:, None])
    kth = before[:, None] + col - held[:, None]
    full = torch.where(fresh, stack[(avail - 1 - kth).clamp(0, free.numel() - 1)], table)
    starts = torch.cat([a.new_zeros(1), torch.cumsum(a, 0)])
    i = torch.arange(rows, device=n.device)
    b = (i[:, None] >= starts[None, 1:]).sum(1)
    live = b < n.numel()
    b = b.clamp(max=n.numel() - 1)
    pos = n[b] - a[b] + i - starts[b]
    page = full[b, (pos // BLOCK).clamp(0, width - 1)]
    good = live & served[b] & (page >= 0) & (page < free.numel())
    slots = torch.where(good, page * BLOCK + pos % BLOCK, torch.full_like(pos, -1))
    i32 = torch.int32
    return dict(slots=slots.to(i32), starts=starts.to(i32), short=(~served).sum().to(i32).view(1), table=full.to(i32),
                free=stack.to(i32), held=held_out.to(i32), count=(avail - (take * served).sum()).to(i32).view(1))


def _plain_write(s, x):
    rows, slots, pool = s[x], s["slots"].long(), s[x + "_pool"]
    page, row = slots // BLOCK, slots % BLOCK
    if s["case"]["fmt"] == "bf16":
        pool = pool.clone()
        pool[page, :, row] = rows
        return pool, None
    fmt, total = s["case"]["fmt"], pool.shape[0]
    y = rows.float()
    amax = y.new_zeros(total, pool.shape[1]).index_reduce_(0, page, y.abs().amax(-1), "amax")
    anew = torch.zeros(total, dtype=torch.bool, device=y.device)
    anew[page[row == 0]] = True
    was = torch.where(anew[:, None], torch.zeros_like(amax), s[x + "_scale"])
    touched = torch.zeros_like(anew)
    touched[page] = True
    scale = torch.where(amax > QMAX[fmt] * was, _pow2(amax, QMAX[fmt]), was)
    scale = torch.where(touched[:, None], scale, s[x + "_scale"])
    # the rows that are there keep their codes, or are held in the larger scale
    grown = touched[:, None] & (scale != was) & ~anew[:, None]
    again = _codes(pool.float() * was[..., None, None], scale[..., None, None].expand(*was.shape, 1, 1), fmt)
    codes = torch.where(grown[..., None, None], again.view(torch.uint8), pool.view(torch.uint8))
    codes[page, :, row] = _codes(y, scale[page][..., None], fmt).view(torch.uint8)
    return codes.view(pool.dtype), scale


def _plain_decode(s):
    c = s["case"]
    Hkv, D, T, nb = c["Hkv"], c["D"], c["T"], _pages_of(c["T"])
    G = c["Hq"] // Hkv
    res = dict(out=[], lse=[], blk_max=[], blk_sum=[])
    for b, n in enumerate(s["host_lens"]):
        m = _pages_of(n)
        if c["paged"]:
            pages = s["table"][b, :m].long()
            k, v = ((s[x].view(torch.uint8)[pages].view(s[x].dtype).float() * s[x + "_scale"][pages][..., None, None])
                    .transpose(0, 1).reshape(Hkv, m * BLOCK, D)[:, :n] for x in ("k", "v"))
        else:
            k, v = (s[x][b, :, :n].float() * s[x + "_scale"][b, :, :m].repeat_interleave(BLOCK, 1)[:, :n, None]
                    for x in ("k", "v"))
        sc = torch.matmul(s["q"][b].float().view(Hkv, G, D), k.transpose(1, 2).contiguous()) * s["scale"]
        if "keep" in s:
            on = s["keep"][b, :, :m].repeat_interleave(BLOCK, 1)[:, None, :n]
            sc = torch.where(on, sc, torch.full_like(sc, -math.inf))
        top = sc.amax(-1, keepdim=True)
        e = torch.exp(sc - top)
        z = e.sum(-1, keepdim=True)
        res["out"].append((torch.matmul(e, v.contiguous()) / z).reshape(c["Hq"], D).to(torch.bfloat16))
        res["lse"].append((top + torch.log(z)).reshape(c["Hq"]))
        if c["stats"]:
            full = sc.new_full((Hkv, G, nb * BLOCK), -math.inf)
            full[..., :n] = sc
            full = full.view(c["Hq"], nb, BLOCK)
            mx = full.amax(-1)
            base = torch.where(mx == -math.inf, torch.zeros_like(mx), mx)
            res["blk_max"].append(mx)
            res["blk_sum"].append(torch.exp(full - base[..., None]).sum(-1))
    return {x: torch.stack(t) for x, t in res.items() if t}


# ---------------------------------------------------------------- the calls

def run(state):
    s, c = state, state["case"]
    if not own:
        if c["kind"] == "pages":
            return _plain_pages(s)
        if c["kind"] == "write":
            (kp, ks), (vp, vs) = _plain_write(s, "k"), _plain_write(s, "v")
            return dict(k=kp, v=vp) if ks is None else dict(k=kp, v=vp, k_scale=ks, v_scale=vs)
        return _plain_decode(s)
    from kvskip_amd import ext, kvskip as K

    if c["kind"] == "pages":
        # the state before stays as it was (the new counts go to buffers of their own), so a step can be planned again
        slots, starts, short = ext.page_map(s["lens"], s["new"], s["held"], s["table"], s["free"], s["count"], s["slots"],
                                            held_out=s["held_out"], free_count_out=s["count_out"])
        return dict(slots=slots, starts=starts, short=short, table=s["table"], free=s["free"], held=s["held_out"],
                    count=s["count_out"])
    if c["kind"] == "write":
        ext.cache_write(s["k"], s["v"], s["slots"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"])
        res = dict(k=s["k_pool"], v=s["v_pool"])
        return res if c["fmt"] == "bf16" else dict(res, k_scale=s["k_scale"], v_scale=s["v_scale"])
    paged = dict(block_table=s["table"], T=c["T"]) if c["paged"] else {}
    r = K.decode(s["q"], s["k"], s["v"], s["scale"], plan=s.get("plan"), stats=c["stats"], seq_lens=s["lens"],
                 k_scale=s["k_scale"], v_scale=s["v_scale"], **paged)
    return {x: r[x] for x in ("out", "lse", "blk_max", "blk_sum") if x in r}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    if c["kind"] == "pages":
        lens, new, held = _step(c)
        taken = sum(max(0, _pages_of(n) - h) for n, h in zip(lens, held))
        given = sum(max(0, h - _pages_of(n)) for n, h in zip(lens, held))
        # lengths, new tokens and pages held in, pages held and starts out; a free page read and put into its table; a
        # page given back; the page of a row that falls into a page held before; a slot a row
        rows = sum(new)
        return dict(bytes=20 * c["B"] + 8 * (taken + given) + 4 * rows // BLOCK + 4 * c["B"] + 4 * rows, flops=0)
    Hq, Hkv, D = c["Hq"], c["Hkv"], c["D"]
    if c["kind"] == "write":
        n = sum(a for _, a in _rows(c))
        pages = sum(_pages_of(p + a) - p // BLOCK for p, a in _rows(c))
        one = 2 if c["fmt"] == "bf16" else 1
        scales = 0 if c["fmt"] == "bf16" else 2 * 8 * pages * Hkv
        return dict(bytes=2 * n * Hkv * D * (2 + one) + 4 * n + scales, flops=0)
    toks = sum(_lengths(c)) * c["frac"]
    blocks = sum(_pages_of(n) for n in _lengths(c)) * c["frac"]
    extra = blocks * 4 * (1 if c["paged"] else 0) + (blocks * Hkv * 4 if c["frac"] < 1.0 else 0)
    stats = 8 * c["B"] * Hq * _pages_of(c["T"]) if c["stats"] else 0
    return dict(bytes=2 * toks * Hkv * D + 8 * blocks * Hkv + c["B"] * Hq * (4 * D + 4) + extra + stats,
                flops=4 * Hq * D * toks)


# ---------------------------------------------------------------- 64 bits

def _exact_pages(c, s):
    lens, new, held, table, free = (s[x].tolist() for x in ("lens", "new", "held", "table", "free"))
    count, width = int(s["count"]), len(table[0])
    total = len(free)
    need = [(n + 63) // 64 for n in lens]
    for b, h in enumerate(held):                               # given back first, in order
        for j in range(need[b], h):
            free[count] = table[b][j]
            count += 1
    slots, starts, short, broke = [], [0], 0, False
    kept = list(held)
    for b, h in enumerate(held):
        want = need[b] - h
        okay = need[b] <= width and (want <= 0 or (not broke and want <= count))
        if okay:
            for j in range(h, need[b]):
                count -= 1
                table[b][j] = free[count]
            kept[b] = need[b]
        else:
            short += 1
            broke = broke or need[b] <= width
        first = lens[b] - new[b]
        slots += [table[b][p // 64] * 64 + p % 64 if okay else -1 for p in range(first, lens[b])]
        starts.append(starts[-1] + new[b])
    assert all(x < total * 64 for x in slots)
    slots += [-1] * (s["slots"].numel() - len(slots))
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return dict(slots=t(slots), starts=t(starts), short=t([short]), table=t(table), free=t(free), held=t(kept),
                count=t([count]))


def _nearest(x, fmt):
    """Codes (as bytes) of the representable values nearest to x, ties to the even code."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127).to(torch.int8).view(torch.uint8)
    grid = torch.arange(127, dtype=torch.uint8, device=x.device).view(torch.float8_e4m3fn).double()
    mid = (grid[1:] + grid[:-1]) / 2
    a = x.abs()
    up, down = torch.searchsorted(mid, a, right=True), torch.searchsorted(mid, a)
    code = torch.where(up == down, up, torch.where(up % 2 == 0, up, down)).clamp(max=126)
    return torch.where(torch.signbit(x), code + 128, code).to(torch.uint8)


def _exact_write(s, x, fmt):
    slots = s["slots"].long()
    pool = s[x + "_pool"].clone()
    if fmt == "bf16":
        flat = pool.transpose(1, 2).reshape(-1, *pool.shape[1::2])
        flat[slots] = s[x]
        return flat.view(pool.shape[0], BLOCK, pool.shape[1], pool.shape[3]).transpose(1, 2).contiguous(), None
    scale = s[x + "_scale"].clone()
    bytes_ = pool.view(torch.uint8)
    pages, which = torch.unique(slots // BLOCK, return_inverse=True)
    for i in range(0, len(pages), 256):                        # some pages at a time, whole, in 64 bits
        mine = (which >= i) & (which < i + 256)
        pg, w, r = pages[i:i + 256], which[mine] - i, slots[mine] % BLOCK
        new = torch.zeros(len(pg), pool.shape[1], BLOCK, pool.shape[3], dtype=torch.float64, device="cuda")
        new[w, :, r] = s[x][mine].double()
        is_new = torch.zeros(len(pg), BLOCK, dtype=torch.bool, device="cuda")
        is_new[w, r] = True
        old_scale = scale[pg].double() * (~is_new[:, :1]).double()
        amax = new.abs().amax((-1, -2))
        ratio = amax / QMAX[fmt]
        want = torch.exp2(torch.ceil(torch.log2(torch.where(ratio > 0, ratio, torch.ones_like(ratio)))).clamp(min=-126))
        got = torch.where((ratio > 0) & (ratio > old_scale), want, old_scale)
        old = bytes_[pg].view(pool.dtype).double()
        safe = torch.where(got > 0, got, torch.ones_like(got))[..., None, None]
        moved = _nearest(old * old_scale[..., None, None] / safe, fmt)
        keep = ((got == old_scale) | is_new[:, :1])[..., None, None]
        res = torch.where(keep, bytes_[pg], moved)
        bytes_[pg] = torch.where(is_new[:, None, :, None], _nearest(new / safe, fmt), res)
        scale[pg] = got.float()
    return pool, scale


def _exact_decode(c, s):
    B, Hq, Hkv, D, T = c["B"], c["Hq"], c["Hkv"], c["D"], c["T"]
    G, nb = Hq // Hkv, _pages_of(T)
    f64 = dict(dtype=torch.float64, device="cuda")
    res = dict(out=torch.zeros(B, Hq, D, **f64), lse=torch.full((B, Hq), -math.inf, **f64),
               blk_max=torch.full((B, Hq, nb), -math.inf, **f64), blk_sum=torch.zeros(B, Hq, nb, **f64))
    for b, n in enumerate(s["host_lens"]):
        m = _pages_of(n)
        for h in range(Hkv):
            def rows(x):
                if c["paged"]:
                    pg = s["table"][b, :m].long()
                    codes, sc = s[x].view(torch.uint8)[pg, h].view(s[x].dtype), s[x + "_scale"][pg, h]
                else:
                    flat = s[x].view(torch.uint8) if s[x].dtype != torch.int8 else s[x]
                    codes = torch.zeros(m * BLOCK, D, dtype=flat.dtype, device="cuda")
                    codes[:n] = flat[b, h, :n]
                    codes, sc = codes.view(s[x].dtype).view(m, BLOCK, D), s[x + "_scale"][b, h, :m]
                return codes.double() * sc.double()[:, None, None]
            hq = slice(h * G, h * G + G)
            sc = torch.einsum("gd,mtd->gmt", s["q"][b, hq].double(), rows("k")) * s["scale"]
            sc.view(G, m * BLOCK)[:, n:] = -math.inf
            if "keep" in s:
                sc.masked_fill_(~s["keep"][b, h, None, :m, None], -math.inf)
            lse = torch.logsumexp(sc.view(G, -1), -1)
            res["lse"][b, hq] = lse
            res["out"][b, hq] = torch.einsum("gmt,mtd->gd", torch.exp(sc - lse[:, None, None]), rows("v"))
            mx = sc.amax(-1)
            res["blk_max"][b, hq, :m] = mx
            res["blk_sum"][b, hq, :m] = torch.exp(sc - mx.clamp(min=-1e300)[..., None]).sum(-1)
    if not c["stats"]:
        del res["blk_max"], res["blk_sum"]
    return res


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "pages":
        return _exact_pages(c, s)
    if c["kind"] == "write":
        (kp, ks), (vp, vs) = _exact_write(s, "k", c["fmt"]), _exact_write(s, "v", c["fmt"])
        return dict(k=kp, v=vp) if ks is None else dict(k=kp, v=vp, k_scale=ks, v_scale=vs)
    return _exact_decode(c, s)
