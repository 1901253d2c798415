"""Attention of a step's rows over 8-bit pages and rotation of heads, from their definitions in 64 bits on the CPU (the checks
of kvskip_attend and kvskip_norm_rope)."""

from __future__ import annotations

import math

import torch

PAGE = 64


def positions(starts, lens, rows, shared_lens=None, shared_of=None):
    """Each row's position, -1 of a row that no request brings: a request's last token is in row starts[b + 1] - 1, there or not."""
    pos = [-1] * rows
    if all(a <= b for a, b in zip(starts, starts[1:])):
        for b, n in enumerate(lens):
            s0, s1 = (min(max(x, 0), rows) for x in starts[b:b + 2])
            base = _base(shared_lens, shared_of, b)
            for i in range(s0, s1):
                pos[i] = base + max(n, 0) - min(starts[b + 1], 1 << 28) + i
    return pos


def _base(shared_lens, shared_of, b):
    return max(shared_lens[shared_of[b]], 0) if shared_of is not None and 0 <= shared_of[b] < len(shared_lens) else 0


def _keys(pool, scale, table, n, h):
    """The first n keys (or values) of a table row for KV head h, 64 bits, and which of them a page of the pool holds."""
    m = (n + PAGE - 1) // PAGE
    pages = table[:m].long()
    held = (pages >= 0) & (pages < pool.shape[0])
    at = torch.where(held, pages, torch.zeros_like(pages))
    codes = pool.view(torch.uint8)[at, h].view(pool.dtype).double() * scale[at, h].double()[:, None, None]
    return (codes.reshape(m * PAGE, pool.shape[-1])[:n], held.repeat_interleave(PAGE)[:n],
            scale[at, h].double().abs().repeat_interleave(PAGE)[:n])


def attend(q, k, v, k_scale, v_scale, scale, starts, lens, block_table, softcap=0.0, slopes=None, window=0, prefix_lens=None,
           shared_table=None, shared_lens=None, shared_of=None):
    """out [rows, Hq, D], lse [rows, Hq], and what errors are measured by: mass, the sum of softmax(s) |v|; reach [rows, Hq], the
    largest sum of |q| |k| times |scale|; grain, the largest softmax(s) |v's scale| times the sum of |v's codes|. Tensors on the
    CPU, lengths as lists."""
    rows, Hq, D = q.shape
    Hkv = k.shape[1]
    G = Hq // Hkv
    out = torch.zeros(rows, Hq, D, dtype=torch.float64)
    mass = torch.zeros(rows, Hq, D, dtype=torch.float64)
    lse = torch.full((rows, Hq), -math.inf, dtype=torch.float64)
    reach = torch.zeros(rows, Hq, dtype=torch.float64)
    grain = torch.zeros(rows, Hq, D, dtype=torch.float64)
    pos = positions(starts, lens, rows, shared_lens, shared_of)
    for b, n in enumerate(lens):
        s0, s1 = (min(max(x, 0), rows) for x in starts[b:b + 2])
        if s1 <= s0:
            continue
        base = _base(shared_lens, shared_of, b)
        pre = 0 if prefix_lens is None else prefix_lens[b]
        p = torch.tensor(pos[s0:s1])[:, None]
        j = torch.arange(base + max(n, 0))[None]
        on = j <= p
        if window:
            on &= j > p - window
        on |= j < pre
        for h in range(Hkv):
            kk, held, _ = _keys(k, k_scale, block_table[b], max(n, 0), h)
            vv, _, vs = _keys(v, v_scale, block_table[b], max(n, 0), h)
            if base:
                k0, h0, _ = _keys(k, k_scale, shared_table[shared_of[b]], base, h)
                v0, _, s0_ = _keys(v, v_scale, shared_table[shared_of[b]], base, h)
                kk, vv, held, vs = torch.cat([k0, kk]), torch.cat([v0, vv]), torch.cat([h0, held]), torch.cat([s0_, vs])
            vs = vs.nan_to_num(0.0, 0.0, 0.0)
            code = (vv.abs() / torch.where(vs > 0, vs, torch.ones_like(vs))[:, None]).nan_to_num(0.0, 0.0, 0.0)
            for g in range(h * G, h * G + G):
                x = q[s0:s1, g].double()
                see = on & held
                s = (x @ kk.T) * scale
                a = (x.abs() @ kk.abs().T) * abs(scale)
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if slopes is not None:
                    s = s - slopes[g].double() * (p - j).abs()
                    a = a + slopes[g].double().abs() * (p - j).abs()
                s = torch.where(see, s, torch.full_like(s, -math.inf))
                reach[s0:s1, g] = torch.where(see, a, torch.zeros_like(a)).nan_to_num(0.0, 0.0, 0.0).amax(-1) if j.numel() else 0.0
                seen = see.any(-1)
                if not j.numel():
                    continue
                z = torch.logsumexp(s, -1)
                w = torch.where(see, torch.exp(s - z[:, None]), torch.zeros_like(s))
                # (what a row does not see does not reach it, whatever it is)
                o = _sum(w, vv, see)
                lse[s0:s1, g] = torch.where(seen, z, torch.full_like(z, -math.inf))
                out[s0:s1, g] = torch.where(seen[:, None], o, torch.zeros_like(o))
                top = (w * vs).nan_to_num(0.0).amax(-1, keepdim=True)
                grain[s0:s1, g] = top * (see.double() @ code)
                mass[s0:s1, g] = torch.where(seen[:, None], _sum(w, vv.abs(), see), torch.zeros_like(o)).nan_to_num(0.0)
    return out, lse, mass, reach, grain


def _sum(w, v, see):
    bad = v.isnan()
    o = w @ torch.where(bad, torch.zeros_like(v), v)
    return torch.where((see.double() @ bad.double()) > 0, torch.full_like(o, math.nan), o)


def norm_rope(x, positions, inv_freq, weight=None, eps=1e-6, sections=None, pairs=False, mscale=1.0):
    """One of q, k [rows, heads, D] rotated, in 64 bits."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    if positions is None:
        return y
    half = inv_freq.numel()
    pos = positions.reshape(-1, x.shape[0]).double()
    axis = [a for a, n in enumerate(sections or [half]) for _ in range(n)]
    out = y.clone()
    for i in range(half):
        t = (pos[axis[i]] * inv_freq[i].double())[:, None]
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + half)
        out[..., a] = mscale * (y[..., a] * torch.cos(t) - y[..., b] * torch.sin(t))
        out[..., b] = mscale * (y[..., b] * torch.cos(t) + y[..., a] * torch.sin(t))
    return out
