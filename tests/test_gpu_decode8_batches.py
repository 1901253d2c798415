"""GPU: ragged decode attention over a cache held in 8 bits for batches of 65 to 256 sequences (kvskip_decode8), most of them
short or empty and one long: results against the oracle in 64 bits, and the split budget that such a batch gets."""

import math
import random

import pytest
import torch

from cache8_side import cache, typed
from kvskip_amd import kvskip as K
from kvskip_amd import workloads as W
from test_gpu_decode8 import _check_ragged, _cpu

pytestmark = pytest.mark.gpu


class Batch:
    """Contiguous caches of T tokens, the long sequence's T, the others' up to 200 and a quarter of them empty."""

    def __init__(self, B, Hq, Hkv, D, T, fmt, seed):
        rng = random.Random(seed)
        self.B, self.Hq, self.Hkv, self.D, self.T, self.fmt, self.scale = B, Hq, Hkv, D, T, fmt, D ** -0.5
        self.lens = [0 if rng.random() < 0.25 else rng.randrange(1, 201) for _ in range(B)]
        self.lens[rng.randrange(64, B)] = T
        self.lens[0], self.lens[B - 1 if self.lens[B - 1] != T else B - 2] = 0, 0
        self.q = torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
        self.kc, self.ks, self.k = cache((B, Hkv), T, D, fmt, seed + 1)
        self.vc, self.vs, self.v = cache((B, Hkv), T, D, fmt, seed + 2)
        past = torch.arange(T)[None] >= torch.tensor(self.lens)[:, None]
        for c in (self.kc, self.vc):
            c.masked_fill_(past[:, None, :, None], 0x7f)

    def decode(self, **kw):
        return K.decode(self.q.cuda(), typed(self.kc, self.fmt), typed(self.vc, self.fmt), self.scale, k_scale=self.ks.cuda(),
                        v_scale=self.vs.cuda(), seq_lens=torch.tensor(self.lens, dtype=torch.int32, device="cuda"),
                        stats=True, out_f32=True, **kw)


def _check(c, r, keep=None):
    """The long sequence, those at the borders of 64 and some others against the oracle; all of the empty ones."""
    rows = {c.lens.index(c.T), *(b for b in (0, 1, 63, 64, 65, 127, 128, 129, 191, 192, 255, c.B - 2, c.B - 1) if b < c.B)}
    rows = sorted(rows | set(random.Random(c.B).sample(range(c.B), 16)))
    some = Batch.__new__(Batch)
    some.__dict__.update(c.__dict__, q=c.q[rows], k=c.k[rows], v=c.v[rows])
    _check_ragged(some, {x: t[rows] if torch.is_tensor(t) else t for x, t in r.items()}, [c.lens[b] for b in rows],
                  None if keep is None else keep[rows], stats=True)
    empty = [b for b, n in enumerate(c.lens) if n == 0]
    assert not r["out"][empty].any() and (r["lse"][empty] == -math.inf).all() and (r["blk_max"][empty] == -math.inf).all()
    assert torch.isfinite(r["out_f32"]).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("B,Hq,Hkv,D", [(65, 4, 2, 64), (128, 4, 1, 128), (129, 7, 1, 64), (256, 2, 2, 64), (256, 16, 1, 64)])
def test_dense(gpu, fmt, B, Hq, Hkv, D):
    c = Batch(B, Hq, Hkv, D, 1500, fmt, B + Hq)
    for S in (None, 2, 7):
        _check(c, _cpu(c.decode(num_splits=S)))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("B,Hq,Hkv,D", [(65, 8, 4, 64), (128, 4, 4, 64), (130, 8, 4, 64), (256, 14, 2, 64), (256, 3, 3, 64)])
def test_lists(gpu, fmt, B, Hq, Hkv, D):
    """Lists, of all KV heads cut together (up to 512 of them) or by KV head; S 40: a grid that queues."""
    c = Batch(B, Hq, Hkv, D, 900, fmt, B + Hq)
    nb = math.ceil(900 / 64)
    keep = W.random_block_list(B, Hkv, nb, 0.5, 6, local=0)
    for b, n in enumerate(c.lens):
        keep[b, :, math.ceil(n / 64):] = False
    for S in (None, 2, 40):
        _check(c, _cpu(c.decode(num_splits=S, plan=K.make_plan(keep.cuda()))), keep)


@pytest.mark.parametrize("Hkv", [1, 2, 4, 8, 16, 32])
@pytest.mark.parametrize("B", [16, 64, 72, 96, 128, 200, 256])
def test_split_budget(gpu, B, Hkv):
    """A batch with more than an even share of work for every CU: S is at least seven eighths of a workgroup a CU, and the grid's
    S + B slots a KV head are whole workgroups a CU (but where S is at its most, 256)."""
    T, D = 32768, 64
    kp = torch.zeros(1, Hkv, 64, D, dtype=torch.int8, device="cuda")
    sc = torch.ones(1, Hkv, device="cuda")
    q = torch.zeros(B, Hkv, D, dtype=torch.bfloat16, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    lens[B - 1] = 64
    table = torch.zeros(B, T // 64, dtype=torch.int32, device="cuda")
    r = K.decode(q, kp, kp, 1.0, k_scale=sc, v_scale=sc, seq_lens=lens, block_table=table, T=T)
    S, cus = r["num_splits"], K.num_sms()
    assert S == 256 or (8 * S * Hkv >= 7 * cus and (S + B) * Hkv % cus == 0)
    assert not r["out"].any() and torch.isinf(r["lse"][:-1]).all() and torch.isfinite(r["lse"][-1]).all()
