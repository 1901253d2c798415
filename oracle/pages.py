"""Oracle of the paged 8-bit cache (float64, CPU): a step's block tables and slot map, rows into pages, and the values
that pages stand for. Test infrastructure only (see oracle/__init__.py)."""

from __future__ import annotations

import math

import torch

BLOCK = 64
QMAX = {"e4m3": 448.0, "int8": 127.0}


def page_map(lens, new, held, table, free, count, rows, whole=False):
    """kvskip_page_map on lists: (slots, starts, short, table, free, held_out, count_out); whole: with lens_out, the lengths
    after the step last."""
    table, free, kept = [list(r) for r in table], list(free), list(held)
    width, pages = len(table[0]), len(free)
    n = [max(x, 0) for x in lens]
    a = [min(max(x, 0), y) for x, y in zip(new, n)]
    need = [math.ceil(x / BLOCK) for x in n]
    over, before, at = [False] * len(n), [y - x for x, y in zip(a, n)], 0
    for b in range(len(n) if whole else 0):
        if lens[b] < 0 < new[b]:                  # a sum of 32 bits that passed 31
            over[b], before[b], at = True, (lens[b] - new[b] + 2 ** 31) % 2 ** 32 - 2 ** 31, rows + 1
        elif a[b] > 0:
            at += a[b]
            over[b] = at > rows
    for b, h in enumerate(held):
        if need[b] <= width and not over[b]:
            for j in range(need[b], h):
                free[count] = table[b][j]
                count += 1
    slots, starts, short, out_of_pages, n_after = [], [0], 0, False, list(n)
    for b, h in enumerate(held):
        want = max(need[b] - h, 0)
        fits = need[b] <= width and not over[b]
        if fits and want > 0 and (out_of_pages or want > count):
            out_of_pages = True
        served = fits and (want == 0 or not out_of_pages)
        if served:
            for j in range(h, need[b]):
                count -= 1
                table[b][j] = free[count]
            kept[b] = need[b]
        else:
            short += 1
            n_after[b] = before[b]
        for p in range(n[b] - a[b], n[b]):
            if len(slots) >= rows:
                break
            page = table[b][p // BLOCK] if served else -1
            slots.append(page * BLOCK + p % BLOCK if 0 <= page < pages else -1)
        starts.append(starts[-1] + (rows + 1 if whole and lens[b] < 0 < new[b] else min(a[b], rows + 1)))
    slots += [-1] * (rows - len(slots))
    res = slots[:rows], starts, short, table, free, kept, count
    return (*res, n_after) if whole else res


def pow2_scale(amax: float, fmt: str) -> float:
    """The smallest power of two s >= 2^-126 with amax <= qmax s (0 for 0)."""
    if amax == 0:
        return 0.0
    e = math.frexp(amax / QMAX[fmt])[1]           # amax / qmax < 2^e (both exact in 64 bits to well below the bound)
    return 2.0 ** max(e - 1 if amax <= QMAX[fmt] * 2.0 ** (e - 1) else e, -126)


def encode(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """x (float64, in units of the scale) as codes (uint8 bytes): nearest, ties to even, at most the largest code;
    NaN 0x7f (e4m3; the sign is not part of it) or 0 (int8)."""
    if fmt == "int8":
        return torch.nan_to_num(x, nan=0.0, posinf=127.0, neginf=-127.0).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    grid = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    mid = (grid[1:] + grid[:-1]) / 2
    a = x.abs().nan_to_num(nan=0.0, posinf=448.0).contiguous()
    up, down = torch.searchsorted(mid, a, right=True), torch.searchsorted(mid, a)
    code = torch.where(up == down, up, torch.where(up % 2 == 0, up, down))
    code = torch.where(torch.signbit(x), code + 128, code)
    return torch.where(torch.isnan(x), torch.full_like(code, 127), code).to(torch.uint8)


def decode_values(codes: torch.Tensor, fmt: str) -> torch.Tensor:
    """uint8 bytes as float64."""
    return (codes.view(torch.int8) if fmt == "int8" else codes.view(torch.float8_e4m3fn)).double()


def cache_write(rows, slots, codes, scales, fmt):
    """kvskip_cache_write of keys or values, in place: rows [N, Hkv, D] (any float type), slots list, codes uint8
    [P, Hkv, 64, D], scales fp32 [P, Hkv]. Runs of at most 64 rows of one page, one after another."""
    P, Hkv = codes.shape[:2]
    N, i = len(slots), 0
    page = [s // BLOCK if 0 <= s < P * BLOCK else -1 for s in slots]
    x = rows.double()
    while i < N:
        if page[i] < 0:
            i += 1
            continue
        j = i
        while j < N and page[j] == page[i] and j - i < BLOCK:
            j += 1
        last = {slots[t] % BLOCK: t for t in range(i, j)}
        for h in range(Hkv):
            new = torch.stack([x[t, h] for t in last.values()])
            mag = new.abs().nan_to_num(nan=0.0, posinf=float(torch.finfo(torch.bfloat16).max))
            amax = float(mag.max())
            was = float(scales[page[i], h])
            if 0 in last or not (0 < was < math.inf):
                was = 0.0
            now = pow2_scale(amax, fmt) if amax > float(torch.tensor(QMAX[fmt] * was).float()) else was   # (the product in fp32)
            if now != was and 0 not in last:
                others = [r for r in range(BLOCK) if r not in last]
                codes[page[i], h, others] = encode(decode_values(codes[page[i], h, others].clone(), fmt) * was / now, fmt)
            codes[page[i], h, list(last)] = encode(new / now if now > 0 else new * 0.0, fmt)
            scales[page[i], h] = now
        i = j
