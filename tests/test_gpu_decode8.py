"""GPU: decode attention over a cache held in 8 bits (kvskip_decode8) against the oracle in 64 bits on the values that
codes and scales stand for; the bounds are derived in cache8_side.check_out. Bytes that a pass must not read (rows past
a sequence's end, unlisted blocks, unused pages) hold NaN (e4m3) or the largest code under a huge scale (int8)."""

import math

import pytest
import torch

from cache8_side import cache, check_out, check_stats, typed
from kvskip_amd import ext as E
from kvskip_amd import kvskip as K
from kvskip_amd import workloads as W
from oracle import attention as O

pytestmark = pytest.mark.gpu

FMTS = ["e4m3", "int8"]


def _q(B, Hq, D, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(B, Hq, D, generator=g).to(torch.bfloat16)


def _cpu(r):
    return {x: t.cpu() if torch.is_tensor(t) else t for x, t in r.items()}


def _poison(codes, fmt, where):
    codes[where] = 0x7f
    return codes


class Case:
    """A contiguous cache in buffers of `cap` tokens, poisoned past T, with its values."""

    def __init__(self, B, Hq, Hkv, D, T, fmt, seed, cap=None):
        self.B, self.Hq, self.Hkv, self.D, self.T, self.fmt = B, Hq, Hkv, D, T, fmt
        self.scale = D ** -0.5
        self.q = _q(B, Hq, D, seed)
        self.kc, self.ks, self.k = cache((B, Hkv), T, D, fmt, seed + 1)
        self.vc, self.vs, self.v = cache((B, Hkv), T, D, fmt, seed + 2)
        self.cap = cap or T + 70

    def views(self):
        def put(c):
            buf = torch.full((self.B, self.Hkv, self.cap, self.D), 0x7f, dtype=torch.uint8)
            buf[:, :, :self.T] = c
            return typed(buf, self.fmt)[:, :, :self.T]
        return put(self.kc), put(self.vc)

    def scales(self):
        def put(s):                                   # rows longer than the blocks, as a growing cache has them
            buf = torch.full((self.B, self.Hkv, s.shape[-1] + 3), 1e30)
            buf[..., :s.shape[-1]] = s
            return buf.cuda()
        return put(self.ks), put(self.vs)

    def decode(self, **kw):
        k, v = self.views()
        ks, vs = self.scales()
        return K.decode(self.q.cuda(), k, v, self.scale, k_scale=ks, v_scale=vs, **kw)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("B,Hq,Hkv,D,T,S", [
    (1, 8, 8, 128, 1, 1), (1, 32, 8, 64, 63, 1), (2, 8, 2, 128, 64, 2), (1, 32, 8, 128, 65, None),
    (1, 32, 8, 64, 200, None), (3, 28, 4, 128, 1000, 5), (2, 6, 2, 64, 777, 3), (1, 5, 1, 128, 4097, 16),
    (2, 16, 2, 64, 2048, 4), (1, 64, 4, 128, 1537, 7), (1, 12, 1, 64, 513, 2), (1, 32, 2, 128, 300, 1),
    (4, 16, 8, 128, 129, 256),
])
def test_dense(gpu, fmt, B, Hq, Hkv, D, T, S):
    c = Case(B, Hq, Hkv, D, T, fmt, 11 * T + Hq)
    r = _cpu(c.decode(num_splits=S, out_f32=True, stats=True))
    ds = check_out(r, O.decode(c.q, c.k, c.v, c.scale), c.q, c.k, c.v, c.scale)
    check_stats(r, c.q, c.k, c.scale, ds)
    r2 = _cpu(c.decode(num_splits=S, out_f32=True))
    assert torch.equal(r["out_f32"], r2["out_f32"]) and torch.equal(r["lse"], r2["lse"])


@pytest.mark.parametrize("fmt", FMTS)
def test_token_major_strides(gpu, fmt):
    """[B, T, Hkv, D] buffers seen as [B, Hkv, T, D], scales [B, nb, Hkv] copied to block rows of another stride."""
    c = Case(2, 8, 4, 128, 333, fmt, 5)
    k, v = (typed(x.transpose(1, 2).contiguous(), fmt).transpose(1, 2) for x in (c.kc, c.vc))
    ks = torch.full((4, 2, c.ks.shape[-1] + 1), 3.0)
    ks[..., :-1] = c.ks.transpose(0, 1)
    r = _cpu(K.decode(c.q.cuda(), k, v, c.scale, k_scale=ks.cuda().transpose(0, 1), v_scale=c.vs.cuda(), num_splits=3))
    check_out(r, O.decode(c.q, c.k, c.v, c.scale), c.q, c.k, c.v, c.scale)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 14, 2), (128, 16, 1)])
@pytest.mark.parametrize("S", [1, 6])
def test_lists(gpu, fmt, D, Hq, Hkv, S):
    c = Case(2, Hq, Hkv, D, 1500, fmt, 3 + S)
    nb = 24
    keep = W.random_block_list(2, Hkv, nb, 0.3, 9, local=1)
    keep[1, 0] = False                                  # a list with nothing in it
    keep[0, Hkv - 1] = False
    keep[0, Hkv - 1, nb - 1] = True                     # the newest block alone
    drop = ~keep.repeat_interleave(64, 2)[:, :, :1500]
    _poison(c.kc, fmt, drop)
    _poison(c.vc, fmt, drop)
    r = _cpu(c.decode(plan=K.make_plan(keep.cuda()), stats=True, num_splits=S, out_f32=True))
    clean = lambda x: torch.where(drop[..., None], torch.zeros_like(x), x)
    k, v = clean(c.k), clean(c.v)
    ds = check_out(r, O.decode(c.q, k, v, c.scale, keep=keep), c.q, k, v, c.scale, keep=keep)
    check_stats(r, c.q, k, c.scale, ds, keep=keep)


def test_lists_with_entries_outside(gpu):
    """Entries outside [0, nb) read nothing; the other entries count."""
    c = Case(1, 4, 1, 64, 300, "e4m3", 1)
    idx = torch.tensor([[[-7, 1, 3, 99, 2 ** 30]]], dtype=torch.int32).cuda()
    cnt = torch.tensor([[5]], dtype=torch.int32).cuda()
    k, v = c.views()
    ks, vs = c.scales()
    keep = torch.zeros(1, 1, 5, dtype=torch.bool)
    keep[..., [1, 3]] = True
    for S in (1, 2, 5):
        out, lse, m, s, o32 = E.decode8(c.q.cuda(), k, v, ks, vs, c.scale, idx, cnt, True, S, True)
        r = dict(out=out.cpu(), lse=lse.cpu(), out_f32=o32.cpu(), blk_max=m.cpu(), blk_sum=s.cpu())
        ds = check_out(r, O.decode(c.q, c.k, c.v, c.scale, keep=keep), c.q, c.k, c.v, c.scale, keep=keep)
        check_stats(r, c.q, c.k, c.scale, ds, keep=keep)


def _ragged_ref(c, lens, keep=None):
    """The oracle sequence by sequence: values, and the dictionary that check_out takes, row by row."""
    for b, n in enumerate(lens):
        n = min(max(n, 0), c.T)
        yield b, n, c.q[b:b + 1], c.k[b:b + 1, :, :n], c.v[b:b + 1, :, :n], (None if keep is None else
                                                                           keep[b:b + 1, :, :math.ceil(n / 64)])


def _check_ragged(c, r, lens, keep=None, stats=False):
    for b, n, q, k, v, kp in _ragged_ref(c, lens, keep):
        row = {x: r[x][b:b + 1] for x in ("out", "lse", "out_f32") if x in r}
        if n == 0:
            assert not row["out"].any() and torch.isinf(row["lse"]).all() and (row["lse"] < 0).all()
            ds = torch.zeros(1, c.Hq, dtype=torch.float64)
        else:
            ds = check_out(row, O.decode(q, k, v, c.scale, keep=kp), q, k, v, c.scale, keep=kp, what=(b, n))
        if stats:
            nb = math.ceil(n / 64)
            st = {x: r[x][b:b + 1, :, :nb] for x in ("blk_max", "blk_sum")}
            if n:
                check_stats(st, q, k, c.scale, ds, keep=kp, what=(b, n))
            assert torch.isinf(r["blk_max"][b, :, nb:]).all() and not r["blk_sum"][b, :, nb:].any()


LENS = [0, 1, 63, 64, 65, 700, 1400, 10 ** 6, -3]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 7, 1)])
@pytest.mark.parametrize("S", [2, 40])
def test_ragged(gpu, fmt, D, Hq, Hkv, S):
    c = Case(len(LENS), Hq, Hkv, D, 1400, fmt, 7)
    for b, n in enumerate(LENS):
        _poison(c.kc[b], fmt, (slice(None), slice(min(max(n, 0), 1400), None)))
        _poison(c.vc[b], fmt, (slice(None), slice(min(max(n, 0), 1400), None)))
    lens = torch.tensor(LENS, dtype=torch.int32).cuda()
    r = _cpu(c.decode(seq_lens=lens, num_splits=S, stats=True, out_f32=True))
    _check_ragged(c, r, LENS, stats=True)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("lp", [0, 1])
@pytest.mark.parametrize("Hq,Hkv", [(8, 2), (14, 2)])
def test_ragged_lists(gpu, fmt, lp, Hq, Hkv):
    lens = [0, 5, 640, 1300, 1400]
    c = Case(5, Hq, Hkv, 128, 1400, fmt, 23)
    keep = W.random_block_list(5, Hkv, 22, 0.4, 2, local=0)
    for b, n in enumerate(lens):
        keep[b, :, math.ceil(n / 64):] = False
    keep[3, 1] = False
    past = keep.clone()
    past[2, 0, 15] = True                               # an entry past the sequence's end: an empty block
    p = K.make_plan(past.cuda())
    k, v = c.views()
    ks, vs = c.scales()
    out, lse, m, s, o32 = E.decode8(c.q.cuda(), k, v, ks, vs, c.scale, p.block_idx, p.block_cnt, True, 9, True,
                                    torch.tensor(lens, dtype=torch.int32).cuda(), list_partition=lp)
    r = dict(out=out.cpu(), lse=lse.cpu(), out_f32=o32.cpu(), blk_max=m.cpu(), blk_sum=s.cpu())
    _check_ragged(c, r, lens, keep, stats=True)


def _paginate(c, lens, seed, extra=4):
    """Pools and scales of the case's tokens in random pages, poison elsewhere, and the table (-1 past each end)."""
    need = [math.ceil(n / 64) for n in lens]
    P = sum(need) + extra
    perm = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).tolist()
    kp, vp = (torch.full((P, c.Hkv, 64, c.D), 0x7f, dtype=torch.uint8) for _ in range(2))
    ks, vs = (torch.full((P, c.Hkv), math.nan) for _ in range(2))
    table = torch.full((c.B, max(need) + 2), -1, dtype=torch.int32)
    i = 0
    for b, n in enumerate(lens):
        for j in range(need[b]):
            pg, rows = perm[i], min(64, n - 64 * j)
            i += 1
            kp[pg, :, :rows], vp[pg, :, :rows] = c.kc[b, :, 64 * j:64 * j + rows], c.vc[b, :, 64 * j:64 * j + rows]
            ks[pg], vs[pg] = c.ks[b, :, j], c.vs[b, :, j]
            table[b, j] = pg
    return typed(kp, c.fmt), typed(vp, c.fmt), ks.cuda(), vs.cuda(), table.cuda()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("D,Hq,Hkv", [(128, 8, 2), (64, 8, 1)])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_pages_same_bits(gpu, fmt, D, Hq, Hkv, ragged, masked):
    lens = [900, 64, 1, 333] if ragged else [900] * 3
    c = Case(len(lens), Hq, Hkv, D, 900, fmt, 31)
    kp, vp, ks, vs, table = _paginate(c, lens, 3)
    kw = dict(num_splits=5, stats=True, out_f32=True)
    if ragged:
        kw["seq_lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
    if masked:
        keep = W.random_block_list(c.B, Hkv, 15, 0.5, 6, local=0)
        for b, n in enumerate(lens):
            keep[b, :, math.ceil(n / 64):] = False
        kw["plan"] = K.make_plan(keep.cuda())
    r = _cpu(K.decode(c.q.cuda(), kp, vp, c.scale, block_table=table, T=900, k_scale=ks, v_scale=vs, **kw))
    ref = _cpu(c.decode(**kw))
    for x in ("out", "out_f32", "lse", "blk_max", "blk_sum"):
        assert torch.equal(r[x], ref[x]), x


def test_bad_pages_are_empty_blocks(gpu):
    c = Case(1, 4, 2, 128, 400, "e4m3", 2)
    kp, vp, ks, vs, table = _paginate(c, [400], 1)
    table[0, 2], table[0, 5] = -4, kp.shape[0]
    keep = torch.ones(1, 2, 7, dtype=torch.bool)
    keep[..., [2, 5]] = False
    for S in (1, 3):
        r = _cpu(K.decode(c.q.cuda(), kp, vp, c.scale, block_table=table, T=400, k_scale=ks, v_scale=vs, num_splits=S,
                          stats=True, out_f32=True))
        ds = check_out(r, O.decode(c.q, c.k, c.v, c.scale, keep=keep), c.q, c.k, c.v, c.scale, keep=keep)
        check_stats(r, c.q, c.k, c.scale, ds, keep=keep)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("kind", ["dense", "lists", "pages", "pages_lists"])
def test_streams_longer_than_a_gather(gpu, fmt, kind):
    """Wavefronts of more than 64 and more than 128 blocks (their items are gathered 64 at a time)."""
    T = 33333
    c = Case(1, 4, 1, 64, T, fmt, 77)
    nb = math.ceil(T / 64)
    kw, keep = dict(num_splits=1, out_f32=True, stats=True), None
    if "lists" in kind:
        keep = W.random_block_list(1, 1, nb, 0.9, 4)
        kw["plan"] = K.make_plan(keep.cuda())
    if "pages" in kind:
        kp, vp, ks, vs, table = _paginate(c, [T], 8)
        r = K.decode(c.q.cuda(), kp, vp, c.scale, block_table=table, T=T, k_scale=ks, v_scale=vs, **kw)
    else:
        r = c.decode(**kw)
    r = _cpu(r)
    ds = check_out(r, O.decode(c.q, c.k, c.v, c.scale, keep=keep), c.q, c.k, c.v, c.scale, keep=keep)
    check_stats(r, c.q, c.k, c.scale, ds, keep=keep)


def test_every_code(gpu):
    """Each of the finite codes alone: one token, so out is the code times the scale, rounded once."""
    for fmt in FMTS:
        codes = torch.arange(256, dtype=torch.uint8)
        if fmt == "e4m3":
            codes = codes[(codes & 127) != 127]
        n = codes.numel()
        vc = codes.view(n, 1, 1, 1).expand(n, 1, 1, 64).contiguous()
        ks = torch.ones(n, 1, 1)
        vs = torch.full((n, 1, 1), 0.3)
        r = K.decode(_q(n, 2, 64, 1).cuda(), typed(torch.zeros_like(vc), fmt), typed(vc, fmt), 1.0, k_scale=ks.cuda(),
                     v_scale=vs.cuda(), out_f32=True)
        from oracle import pages as OPG

        want = OPG.decode_values(codes, fmt) * float(vs[0])
        got = r["out_f32"].double().cpu()[:, 0, 0]
        # the value is exact in fp16; its weight times the scale is rounded to fp16 (2^-11), the rest is fp32
        assert ((got - want).abs() <= (2.0 ** -11 + 2.0 ** -20) * want.abs()).all(), fmt
        r = K.decode(_q(n, 2, 64, 1).cuda(), typed(torch.zeros_like(vc), fmt), typed(vc, fmt), 1.0, k_scale=ks.cuda(),
                     v_scale=torch.full((n, 1, 1), 0.25).cuda(), out_f32=True)
        assert torch.equal(r["out_f32"].double().cpu()[:, 0, 0], OPG.decode_values(codes, fmt) * 0.25), fmt


def test_query_range(gpu):
    """Queries from 2^-60 to 2^60, and one with a largest element that hides small ones."""
    c = Case(1, 4, 1, 64, 130, "int8", 4)
    q = c.q.clone()
    for g, e in enumerate((-60, -20, 20, 60)):
        q[0, g] = (q[0, g].double() * 2.0 ** e).to(torch.bfloat16)
    q[0, 2, 5] = 2.0 ** 20
    k, v = c.views()
    ks, vs = c.scales()
    for scale in (2.0 ** -20, 1e-4, 2.0 ** 30):
        one = q if scale < 1e-3 else q * 2.0 ** -70
        r = _cpu(K.decode(one.cuda(), k, v, scale, k_scale=ks, v_scale=vs, out_f32=True, num_splits=1))
        A = (O.scores(one.double().abs(), c.k.abs(), scale)).amax()
        if float(A) * 72 * 2.0 ** -24 < 1:              # else the scores' own rounding decides (fp32 has no more)
            check_out(r, O.decode(one, c.k, c.v, scale), one, c.k, c.v, scale, what=scale)
        assert torch.isfinite(r["out_f32"]).all()


@pytest.mark.parametrize("fmt", FMTS)
def test_query_not_finite(gpu, fmt):
    """An infinity or NaN in a head's query makes that head NaN, and no other."""
    c = Case(1, 4, 1, 64, 200, fmt, 3)
    for bad in (math.inf, -math.inf, math.nan):
        c.q = _q(1, 4, 64, 3)
        c.q[0, 2, 60] = bad
        for S in (1, 2):
            r = _cpu(c.decode(num_splits=S, out_f32=True))
            assert torch.isnan(r["out_f32"][0, 2]).all() and torch.isnan(r["lse"][0, 2])
            assert torch.isfinite(r["out_f32"][0, [0, 1, 3]]).all()


def test_split_counts(gpu):
    """The counts made up natively: one split up to 8 blocks (12 of 64 dims), then three blocks each while every split has a CU, then
    kvskip.num_splits_for's; a ragged batch's fill whole workgroups per CU."""
    for B, Hq, Hkv, D, T in ((1, 8, 8, 64, 300), (1, 16, 2, 128, 513), (1, 32, 8, 128, 9000), (3, 14, 2, 64, 5000)):
        c = Case(B, Hq, Hkv, D, T, "int8", 1)
        nb = math.ceil(T / 64)
        keep = W.random_block_list(B, Hkv, nb, 0.3, 2)
        p = K.make_plan(keep.cuda())
        for n, r in ((nb, c.decode()), (p.max_cnt, c.decode(plan=p))):
            thin = math.ceil(n / 3)
            assert r["num_splits"] == (1 if n <= (12 if D == 64 else 8) else thin if thin * B * Hkv <= K.num_sms() else
                                       K.num_splits_for(B * Hkv, n))
        S = c.decode(seq_lens=torch.full((B,), T, dtype=torch.int32, device="cuda"))["num_splits"]
        assert 2 <= S <= max(2, (B * nb + 1) // 2) and (S == (B * nb + 1) // 2 or (S + B) * Hkv % K.num_sms() == 0 or S == 2)
        with pytest.raises(RuntimeError, match="num_splits in 1..256"):
            c.decode(num_splits=257)


def test_refusals_on_the_device(gpu):
    c = Case(2, 8, 2, 64, 130, "e4m3", 1)
    k, v = c.views()
    ks, vs = c.scales()
    q = c.q.cuda()
    call = lambda q=q, k=k, v=v, ks=ks, vs=vs, **kw: K.decode(q, k, v, 1.0, k_scale=ks, v_scale=vs, **kw)
    for kw, msg in ((dict(k=k.view(torch.uint8)), "float8_e4m3fn or int8"), (dict(v=v.view(torch.int8)), "one type"),
                    (dict(k=k[..., :-1]), "shape mismatch|16-byte"), (dict(k=k[:, :, :-1]), "shape mismatch"),
                    (dict(ks=ks[:, :, :2]), r"ceil\(T / 64\)"), (dict(ks=ks.double()), "fp32"), (dict(ks=ks[0]), "ceil"),
                    (dict(ks=ks.cpu()), "one device"), (dict(q=q[:, :7]), "multiple of Hkv"),
                    (dict(seq_lens=torch.ones(2, device="cuda")), "int32"),
                    (dict(block_table=torch.zeros(2, 3, dtype=torch.int32, device="cuda")), "T .tokens"),
                    (dict(block_table=torch.zeros(2, 3, dtype=torch.int32, device="cuda"), T=130), "page pools")):
        with pytest.raises(RuntimeError, match=msg):
            call(**kw)


def test_scale_range(gpu):
    """Blocks whose scales differ by 2^80 (a block of zeros with scale 0 among them), and a NaN in one head's block."""
    c = Case(1, 2, 2, 128, 512, "e4m3", 6)
    f = torch.exp2(torch.tensor([0., -60., -40., -20., 3., 10., 20., 0.]))
    c.vs, c.v = c.vs * f, c.v * f.double().repeat_interleave(64)[None, None, :, None]
    c.vs[..., 7] = 0
    c.v[:, :, 448:] = 0
    c.ks[..., 3] = 0
    c.k[:, :, 192:256] = 0
    r = _cpu(c.decode(out_f32=True, num_splits=2))
    check_out(r, O.decode(c.q, c.k, c.v, c.scale), c.q, c.k, c.v, c.scale)
    c.vc[0, 1, 100, 9] = 0x7f
    r = _cpu(c.decode(out_f32=True, num_splits=2))
    bad = torch.isnan(r["out_f32"])
    assert bad[0, 1, 9] and bad.sum() == 1


def test_offsets_past_32_bits(gpu):
    """A list of blocks at the end of a 5 GB head of a contiguous cache, and a page at the end of a 5 GB pool."""
    T, D = 40_000_000, 128
    nb = math.ceil(T / 64)
    c = Case(1, 2, 1, D, 256, "int8", 8)
    buf = torch.empty(1, 1, T, D, dtype=torch.int8, device="cuda")
    ks, vs = (torch.ones(1, 1, nb, device="cuda") for _ in range(2))
    blocks = [0, 262145, nb - 2, nb - 1]                 # 262145: past 2^31 bytes
    for i, blk in enumerate(blocks):
        buf[0, 0, blk * 64:blk * 64 + 64] = typed(c.kc[0, 0, 64 * i:64 * i + 64], "int8")
        ks[0, 0, blk], vs[0, 0, blk] = c.ks[0, 0, i], c.ks[0, 0, i]
    idx = torch.tensor(blocks, dtype=torch.int32, device="cuda").view(1, 1, 4)
    cnt = torch.tensor([[4]], dtype=torch.int32, device="cuda")
    ref = O.decode(c.q, c.k, c.k, c.scale)
    out, lse, *_ = E.decode8(c.q.cuda(), buf, buf, ks, vs, c.scale, idx, cnt, num_splits=2)
    check_out(dict(out=out.cpu(), lse=lse.cpu()), ref, c.q, c.k, c.k, c.scale)
    pool = buf.view(nb, 1, 64, D)
    table = torch.tensor([blocks], dtype=torch.int32, device="cuda")
    out, lse, *_ = E.decode8(c.q.cuda(), pool, pool, ks.view(nb, 1), vs.view(nb, 1), c.scale, num_splits=2,
                             block_table=table, T=256)
    check_out(dict(out=out.cpu(), lse=lse.cpu()), ref, c.q, c.k, c.k, c.scale)


def test_streams_and_graphs(gpu):
    """On a stream of its own, and captured: every replay gives the eager call's bits, new inputs included."""
    c = Case(2, 8, 2, 128, 700, "e4m3", 12)
    k, v = c.views()
    ks, vs = c.scales()
    q = c.q.cuda()
    lens = torch.tensor([700, 130], dtype=torch.int32, device="cuda")
    call = lambda: K.decode(q, k, v, c.scale, k_scale=ks, v_scale=vs, seq_lens=lens, stats=True)
    want = call()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        r = call()
    st.synchronize()
    assert torch.equal(r["out"], want["out"]) and torch.equal(r["lse"], want["lse"])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = call()
    for i in range(4):
        if i == 2:
            q.copy_(_q(2, 8, 128, 99).cuda())
            lens.copy_(torch.tensor([0, 700], dtype=torch.int32))
            want = call()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x in ("out", "lse", "blk_max", "blk_sum"):
            assert torch.equal(r[x], want[x]), (i, x)
